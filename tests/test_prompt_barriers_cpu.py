"""A model of the barriers of prompt_tc_kernel (csrc/kdnn_prompt.cu) on the CPU: loader, product warp, softmax warps and the two warps that look
through the values of steps with masked places, in random interleavings, with copies that land in any order. A wait is for a parity, so it has to
begin in the phase that it means or in the one behind it; the model checks that, what lies in a stage when it is read, and that all roles end."""
import os
import random

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Bar:
    def __init__(self, count):
        self.count, self.pending, self.phase = count, 0, 0

    def arrive(self):
        self.pending += 1
        if self.pending == self.count:
            self.pending, self.phase = 0, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def model(n0, n1, low, high, stages, tiles, rng, landing):
    steps = max(n0, n1)
    is_edge = [j < low or j >= high for j in range(steps)]
    before = [sum(is_edge[:j]) for j in range(steps + 1)]
    full, empty = [Bar(1) for _ in range(stages)], [Bar(1) for _ in range(stages)]
    q_full, s_full, p_full, o_full = ([Bar(c) for _ in range(2)] for c in (1, 1, 4, 1))
    asked, clean = [Bar(1) for _ in range(5)], [Bar(2) for _ in range(5)]
    in_flight, commits, holds = [], [], [None] * stages

    def wait(bar, phase):
        """For the completion of `phase`, by its parity."""
        assert bar.phase in (phase, phase + 1), "a parity that says something else"
        while not bar.passes(phase & 1):
            yield

    def loader():
        q_full[0].arrive()
        for i in range(2 * steps):
            if i >= stages:
                yield from wait(empty[i % stages], i // stages - 1)
            in_flight.append(i)
            if i == 0 and n1 > 0:
                q_full[1].arrive()
            yield

    def products():
        yield from wait(full[0], 0)
        yield from wait(q_full[0], 0)
        commits.append(s_full[0])
        if n1 > 0:
            yield from wait(q_full[1], 0)
            commits.append(s_full[1])
        commits.append(empty[0])
        for j in range(steps):
            v, k = 2 * j + 1, 2 * j + 2
            yield from wait(full[v % stages], v // stages)
            assert holds[v % stages] == v
            if j + 1 < steps and is_edge[j + 1]:
                asked[before[j + 1]].arrive()
            if is_edge[j]:
                yield from wait(clean[before[j]], 0)
            keys = False
            for x in range(tiles):
                n = n1 if x else n0
                if j >= n:
                    continue
                yield from wait(p_full[x], j)
                if j + 1 == n:
                    commits.append(o_full[x])
                else:
                    if not keys:
                        yield from wait(full[k % stages], k // stages)
                        assert holds[k % stages] == k
                    keys = True
                    commits.append(s_full[x])
                yield
            commits.append(empty[v % stages])
            if keys:
                commits.append(empty[k % stages])

    def softmax(x):
        for j in range(n1 if x else n0):
            yield from wait(s_full[x], j)
            yield
            p_full[x].arrive()
        if (n1 if x else n0) > 0:
            yield from wait(o_full[x], 0)

    def looking():
        for j in range(steps):
            if is_edge[j]:
                v = 2 * j + 1
                if j > 0:
                    yield from wait(asked[before[j]], 0)
                yield from wait(full[v % stages], v // stages)
                assert holds[v % stages] == v
                yield
                assert holds[v % stages] == v
                clean[before[j]].arrive()

    roles = [loader(), products(), looking(), looking()] + [softmax(x) for x in range(tiles) for _ in range(4)]
    for _ in range(400000):
        if not (roles or in_flight or commits):
            return
        c = rng.random()
        if in_flight and c < landing:
            i = in_flight.pop(-1 if rng.random() < 0.7 else rng.randrange(len(in_flight)))
            holds[i % stages] = i
            full[i % stages].arrive()
        elif commits and c < landing + 0.2:
            commits.pop(0).arrive()
        elif roles:
            role = rng.choice(roles)
            try:
                next(role)
            except StopIteration:
                roles.remove(role)
    raise AssertionError("a role waits without end")


@pytest.mark.parametrize("stages", [2, 5])
@pytest.mark.parametrize("landing", [0.01, 0.05, 0.4])
def test_every_wait_means_its_phase(stages, landing):
    rng = random.Random(stages)
    for _ in range(400):
        tiles = rng.choice([1, 2])
        n0 = rng.randrange(1, 12)
        n1 = 0 if tiles == 1 else rng.choice([0, n0, n0 + 1, n0 + 2])
        steps = max(n0, n1)
        model(n0, n1, min(rng.randrange(3), steps), max(0, steps - rng.randrange(4)), stages, tiles, rng, landing)


def test_steps_with_masked_places():
    """The bounds that the kernel takes its steps from, against every key and row: no step with a key that some row does not see is left
    out, and there are five at the most."""
    rng = random.Random(7)
    for _ in range(20000):
        tokens, tiles = 128 // rng.choice([1, 2, 3, 4, 5, 8, 20, 64, 128]), rng.choice([1, 2])
        n = rng.choice([1, 2, rng.randrange(1, 60), rng.randrange(1, 3000)])
        window = rng.choice([0, 1, 2, rng.randrange(1, 300), rng.randrange(1, 4000), 2 ** 31 - 1])
        t0 = rng.randrange(-(-n // (tiles * tokens))) * tiles * tokens
        beg = max(0, t0 - window + 1) if window else 0
        end0, end1 = min(n, t0 + tokens), min(n, t0 + tiles * tokens)
        last = max(end0, end1) - 1
        steps = -(-(last + 1 - beg) // 128)
        all_lo = last + 1 - window if window else 0
        low, high = max(int((all_lo - beg + 127) / 128), 0), (t0 - beg + 1) // 128
        edges = [j for j in range(steps) if j < low or j >= high]
        assert len(edges) == (steps if low >= high else low + steps - high) <= 5
        assert edges == [e if e < low or low >= high else e - low + high for e in range(len(edges))]
        for j in set(range(steps)) - set(edges):
            for key in (beg + 128 * j, beg + 128 * j + 127):
                assert all(key <= r and (not window or key > r - window) for r in (t0, last))


def test_the_model_is_of_this_kernel():
    """The lines that the model restates."""
    src = open(os.path.join(ROOT, "dnn-for-kokkos_b200", "csrc", "kdnn_prompt.cu")).read()
    for line in ("if ((j + 1 < low || j + 1 >= high) && j + 1 < steps && lane == 0) mbar_arrive(v_asked(cleaned + here));",
                 "if (here && !(ok = wait(v_clean(cleaned++), 0))) break;",
                 "const int j = step_of(e), fill = 2 * j + 1, st = fill % L::kStages",
                 "const int low = max((all_lo - beg + kPtKeys - 1) / kPtKeys, 0), high = (t0 - beg + 1) / kPtKeys;",
                 "auto step_of = [&](int e) { return e < low || low >= high ? e : e - low + high; };"):
        assert line in src, line
