"""Tensor memory and programmatic launches: a kernel that takes tensor memory has it before it lets the next kernel onto the SMs. The other
way round a CTA of the next kernel could take the columns first and keep them until the grid that waits for them is done."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "dnn-for-kokkos_b200", "csrc")


def kernels_with_tensor_memory():
    for name in sorted(os.listdir(CSRC)):
        src = open(os.path.join(CSRC, name)).read()
        starts = [m.start() for m in re.finditer(r"__global__", src)] + [len(src)]
        for lo, hi in zip(starts, starts[1:]):
            if "tcgen05.alloc" in src[lo:hi]:
                yield name, src[lo:hi]


def test_tensor_memory_comes_before_the_next_kernel():
    found = list(kernels_with_tensor_memory())
    assert {n for n, _ in found} == {"kdnn_prompt.cu", "kdnn_split.cuh", "kdnn_tc.cuh"}
    for name, body in found:
        assert "pdl_chain_entry" not in body, name
        assert body.count("pdl_launch_dependents()") == 1, name
        assert body.index("tcgen05.alloc") < body.index("relinquish_alloc_permit") < body.index("pdl_launch_dependents()"), name
