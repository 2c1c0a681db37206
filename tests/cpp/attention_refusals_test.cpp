// Views that the attention operators of the C++ layer (include/KokkosDNN_B200.hpp) must refuse before anything is launched: strides, shapes
// and caches that the C ABI cannot see. Runs without a device (every pointer is a fake one), so a call whose views are right ends in
// std::runtime_error and one that is refused in std::invalid_argument. Exit code 0 = all checks passed.
#include <Kokkos_Core.hpp>
#include <cuda_runtime.h>

#include <cstdio>
#include <stdexcept>

#include "KokkosDNN_B200.hpp"

namespace {
struct Dev {};
int failures = 0;

template <class T, int R>
struct View {
  size_t n[R] = {}, s[R] = {}, p = 0;
  T* data() const { return reinterpret_cast<T*>(p); }
  size_t extent(int i) const { return n[i]; }
  size_t stride(int i) const { return s[i]; }
};
template <class T, int R, class... N>
View<T, R> make(N... n) {
  static size_t places = 0;      // 4 TiB apart per view, another start per type
  View<T, R> v{{static_cast<size_t>(n)...}, {}, (++places << 42) + (size_t(sizeof...(N)) << 36) + (size_t(R * 8 + sizeof(T)) << 30)};
  size_t at = 1;
  for (int i = R - 1; i >= 0; at *= v.n[i--]) v.s[i] = at;
  return v;
}
template <class T, int R>
View<T, R> with_stride(View<T, R> v, int i, size_t stride) { v.s[i] = stride; return v; }
template <class T, int R>
View<T, R> with_extent(View<T, R> v, int i, size_t n) { v.n[i] = n; return v; }
template <class T>
View<T, 2> left(View<T, 2> v) { v.s[0] = 1; v.s[1] = v.n[0]; return v; }

struct Plan { View<int32_t, 1> row_start, first, lens, state, slots; View<int32_t, 2> writes; size_t page; };
struct Cache { View<int8_t, 4> k, v; View<float, 2> k_scale, v_scale; };

template <class F>
int outcome(F f) {   // 0: accepted, 1: refused, 2: another error (no device)
  try { f(); } catch (const std::invalid_argument&) { return 1; } catch (const std::runtime_error&) { return 2; }
  return 0;
}
#define REFUSED(call) do { if (outcome([&] { call; }) != 1) { std::printf("NOT REFUSED %d: %s\n", __LINE__, #call); ++failures; } } while (0)
#define PASSED_ON(call) do { if (outcome([&] { call; }) != 2) { std::printf("NOT PASSED ON %d: %s\n", __LINE__, #call); ++failures; } } while (0)
}  // namespace

int main() {
  namespace B = KokkosDNN::B200;
  Dev sp;
  int devices = 0;
  if (cudaGetDeviceCount(&devices) == cudaSuccess && devices > 0) { std::printf("run without a device\n"); return 2; }
  const size_t S = 3, N = 10, H = 4, KV = 2, D = 64, page = 16, pages = 9, cols = 4;
  const auto fresh = make<int32_t, 1>(S), lens = make<int32_t, 1>(S), ring = make<int32_t, 1>(pages), state = make<int32_t, 1>(size_t(4));
  const auto table = make<int32_t, 2>(S, cols);
  const Plan plan{make<int32_t, 1>(S + 1), make<int32_t, 1>(S), make<int32_t, 1>(S), make<int32_t, 1>(size_t(4)), make<int32_t, 1>(N),
                  make<int32_t, 2>(kdnn_b200_kv_writes(N, S, page), size_t(4)), page};
  const Cache cache{make<int8_t, 4>(pages, KV, page, D), make<int8_t, 4>(pages, KV, page, D), make<float, 2>(pages, KV), make<float, 2>(pages, KV)};
  const auto q = make<float, 3>(N, H, D), k = make<float, 3>(N, KV, D), out = make<float, 3>(N, H, D);
  const auto ws = make<uint8_t, 1>(size_t(1) << 32);
  const auto rs = plan.row_start;

  // ---- right as they are
  PASSED_ON(B::kv_plan(sp, fresh, lens, table, ring, state, plan));
  PASSED_ON(B::kv_append(sp, k, k, plan, cache));
  PASSED_ON(B::kv_attention(sp, q, plan, table, cache, out, 1.f, 0, ws));
  PASSED_ON(B::prompt_attention(sp, q, k, k, rs, out, 1.f, 0));
  // ---- plan
  auto odd_plan = [&](int which) {
    Plan p = plan;
    switch (which) {
      case 0: p.row_start.s[0] = 2; break;
      case 1: p.first.s[0] = 2; break;
      case 2: p.lens.s[0] = 3; break;
      case 3: p.state.s[0] = 2; break;
      case 4: p.slots.s[0] = 2; break;
      case 5: p.writes = left(p.writes); break;
      case 6: p.writes.n[1] = 3; break;
      case 7: p.row_start.n[0] = S; break;
      case 8: p.lens.n[0] = S - 1; break;
      default: p.state.n[0] = 3;
    }
    return p;
  };
  for (int i = 0; i < 10; ++i) {
    REFUSED(B::kv_plan(sp, fresh, lens, table, ring, state, odd_plan(i)));
    REFUSED(B::kv_append(sp, k, k, odd_plan(i), cache));
    REFUSED(B::kv_attention(sp, q, odd_plan(i), table, cache, out, 1.f, 0, ws));
  }
  REFUSED(B::kv_plan(sp, with_stride(fresh, 0, 2), lens, table, ring, state, plan));
  REFUSED(B::kv_plan(sp, fresh, with_stride(lens, 0, 2), table, ring, state, plan));
  REFUSED(B::kv_plan(sp, fresh, lens, with_stride(with_stride(table, 1, 2), 0, 2 * cols), ring, state, plan));
  REFUSED(B::kv_plan(sp, fresh, lens, left(table), ring, state, plan));
  REFUSED(B::kv_plan(sp, fresh, lens, table, with_stride(ring, 0, 2), state, plan));
  REFUSED(B::kv_plan(sp, fresh, lens, table, ring, with_stride(state, 0, 2), plan));
  // ---- rows
  auto apart = [](View<float, 3> v) { v.s[0] *= 2; v.s[1] *= 2; v.s[2] = 2; return v; };
  REFUSED(B::kv_append(sp, apart(k), k, plan, cache));
  REFUSED(B::kv_append(sp, k, apart(k), plan, cache));
  REFUSED(B::kv_attention(sp, apart(q), plan, table, cache, out, 1.f, 0, ws));
  REFUSED(B::kv_attention(sp, q, plan, table, cache, apart(out), 1.f, 0, ws));
  REFUSED(B::kv_attention(sp, q, plan, with_stride(with_stride(table, 1, 2), 0, 2 * cols), cache, out, 1.f, 0, ws));
  REFUSED(B::kv_attention(sp, q, plan, table, cache, out, 1.f, 0, with_stride(ws, 0, 2)));
  REFUSED(B::kv_attention(sp, with_extent(q, 0, N + 1), plan, table, cache, with_extent(out, 0, N + 1), 1.f, 0, ws));
  REFUSED(B::prompt_attention(sp, apart(q), k, k, rs, out, 1.f, 0));
  REFUSED(B::prompt_attention(sp, q, apart(k), k, rs, out, 1.f, 0));
  REFUSED(B::prompt_attention(sp, q, k, apart(k), rs, out, 1.f, 0));
  REFUSED(B::prompt_attention(sp, q, k, k, rs, apart(out), 1.f, 0));
  REFUSED(B::prompt_attention(sp, q, k, k, with_stride(rs, 0, 2), out, 1.f, 0));
  // ---- caches
  auto odd_cache = [&](int which) {
    Cache c = cache;
    switch (which) {
      case 0: c.k_scale.n[0] = pages - 1; break;
      case 1: c.v_scale.n[1] = KV - 1; break;
      case 2: c.v.n[0] = pages - 2; break;
      case 3: c.v.n[3] = D / 2; break;
      case 4: c.k_scale = left(c.k_scale); break;
      case 5: c.v_scale.s[0] = KV + 1; break;
      case 6: c.k.s[0] *= 2; break;
      default: c.v.s[3] = 2;
    }
    return c;
  };
  for (int i = 0; i < 8; ++i) {
    REFUSED(B::kv_append(sp, k, k, plan, odd_cache(i)));
    REFUSED(B::kv_attention(sp, q, plan, table, odd_cache(i), out, 1.f, 0, ws));
  }
  if (failures == 0) std::printf("attention refusals: all checks passed\n");
  return failures != 0;
}
