// Drives the attention operators of the C++ layer (include/KokkosDNN_B200.hpp) with Kokkos-style views: a prompt of two sequences is
// planned, attended to and cached, then one decode step runs over the cache; results are checked against plain loops in double.
// Exit code 0 = all checks passed.
#include <Kokkos_Core.hpp>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <random>
#include <stdexcept>
#include <vector>

#include "KokkosDNN_B200.hpp"

namespace {
struct Dev {};
int failures = 0;
#define CHECK(cond) do { if (!(cond)) { std::printf("FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); ++failures; } } while (0)

// a dense device tensor with the members that the layer asks of a view
template <class T, int R>
struct View {
  T* p = nullptr;
  size_t n[R] = {};
  T* data() const { return p; }
  size_t extent(int i) const { return n[i]; }
  size_t stride(int i) const { size_t s = 1; for (int k = R - 1; k > i; --k) s *= n[k]; return s; }
  size_t size() const { return n[0] * stride(0); }
};
template <class T, int R, class... N>
View<T, R> make(N... n) {
  View<T, R> v{nullptr, {static_cast<size_t>(n)...}};
  cudaMalloc(reinterpret_cast<void**>(&v.p), v.size() * sizeof(T) + 16);
  cudaMemset(v.p, 0, v.size() * sizeof(T) + 16);
  return v;
}
template <class T, int R> void put(const View<T, R>& v, const std::vector<T>& h) { cudaMemcpy(v.p, h.data(), h.size() * sizeof(T), cudaMemcpyHostToDevice); }
template <class T, int R> std::vector<T> get(const View<T, R>& v) {
  std::vector<T> h(v.size());
  cudaMemcpy(h.data(), v.p, h.size() * sizeof(T), cudaMemcpyDeviceToHost);
  return h;
}
struct Plan { View<int32_t, 1> row_start, first, lens, state, slots; View<int32_t, 2> writes; size_t page; };
struct Cache { View<int8_t, 4> k, v; View<float, 2> k_scale, v_scale; };
Plan make_plan(size_t seqs, size_t rows, size_t page) {
  return Plan{make<int32_t, 1>(seqs + 1), make<int32_t, 1>(seqs), make<int32_t, 1>(seqs), make<int32_t, 1>(4), make<int32_t, 1>(rows),
              make<int32_t, 2>(kdnn_b200_kv_writes(rows, seqs, page), size_t(4)), page};
}

// o = softmax(scale q . k) v over `keys` rows of k and v (row pitch KV * D)
void attend(const float* q, const double* k, const double* v, int keys, int D, size_t pitch, double scale, double* o) {
  std::vector<double> s(keys);
  double top = -1e300, sum = 0;
  for (int j = 0; j < keys; ++j) {
    s[j] = 0;
    for (int d = 0; d < D; ++d) s[j] += q[d] * k[j * pitch + d];
    s[j] *= scale;
    top = std::fmax(top, s[j]);
  }
  for (int d = 0; d < D; ++d) o[d] = 0;
  for (int j = 0; j < keys; ++j) {
    const double p = std::exp(s[j] - top);
    sum += p;
    for (int d = 0; d < D; ++d) o[d] += p * v[j * pitch + d];
  }
  for (int d = 0; d < D; ++d) o[d] /= sum;
}
}  // namespace

int main() {
  namespace B = KokkosDNN::B200;
  Dev space;
  const size_t S = 2, H = 4, KV = 2, D = 64, page = 16, pages = 9, cols = 4;
  const std::vector<int32_t> prompt = {19, 33};
  const size_t rows = 52;
  const float scale = 0.125f;
  auto lens = make<int32_t, 1>(S), fresh = make<int32_t, 1>(S), ring = make<int32_t, 1>(pages), state = make<int32_t, 1>(size_t(4));
  auto table = make<int32_t, 2>(S, cols);
  put(ring, std::vector<int32_t>{8, 1, 6, 3, 0, 5, 2, 7, 4});
  put(state, std::vector<int32_t>{0, 9, 0, 0});
  put(fresh, prompt);
  Cache cache{make<int8_t, 4>(pages, KV, page, D), make<int8_t, 4>(pages, KV, page, D), make<float, 2>(pages, KV), make<float, 2>(pages, KV)};
  std::mt19937 rng(5);
  std::normal_distribution<float> nd(0.f, 1.f);
  auto random = [&](const View<float, 3>& v) {
    std::vector<float> h(v.size());
    for (auto& x : h) x = nd(rng);
    put(v, h);
    return h;
  };

  // ---- the prompts
  Plan plan = make_plan(S, rows, page);
  auto q = make<float, 3>(rows, H, D), k = make<float, 3>(rows, KV, D), v = make<float, 3>(rows, KV, D), out = make<float, 3>(rows, H, D);
  const auto hq = random(q), hk = random(k), hv = random(v);
  B::kv_plan(space, fresh, lens, table, ring, state, plan);
  CHECK((get(plan.row_start) == std::vector<int32_t>{0, 19, 52}));
  CHECK((get(plan.lens) == prompt));
  CHECK((get(table) == std::vector<int32_t>{8, 1, 0, 0, 6, 3, 0, 0}));      // two and three pages in the ring's order, the third is page 0
  B::prompt_attention(space, q, k, v, plan.row_start, out, scale, 0);
  B::kv_append(space, k, v, plan, cache);
  const std::vector<double> dk(hk.begin(), hk.end()), dv(hv.begin(), hv.end());
  const auto ho = get(out);
  double worst = 0;
  for (size_t b = 0, r0 = 0; b < S; r0 += prompt[b++])
    for (int i = 0; i < prompt[b]; ++i)
      for (size_t h = 0; h < H; ++h) {
        double o[64];
        attend(&hq[((r0 + i) * H + h) * D], &dk[(r0 * KV + h / 2) * D], &dv[(r0 * KV + h / 2) * D], i + 1, D, KV * D, scale, o);
        for (size_t d = 0; d < D; ++d) worst = std::fmax(worst, std::fabs(o[d] - ho[((r0 + i) * H + h) * D + d]));
      }
  CHECK(worst < 2e-5);      // fp32 sums of at most 33 products with values of a few units

  // ---- a decode step in place of the pool
  Plan one = make_plan(S, S, page);
  lens = plan.lens;
  one.lens = lens;
  state = plan.state;
  one.state = state;
  put(fresh, std::vector<int32_t>{1, 1});
  auto q1 = make<float, 3>(S, H, D), k1 = make<float, 3>(S, KV, D), v1 = make<float, 3>(S, KV, D), o1 = make<float, 3>(S, H, D);
  const auto hq1 = random(q1);
  random(k1);
  random(v1);
  auto ws = make<uint8_t, 1>(kdnn_b200_kv_attention_workspace_bytes(S, S, H, KV, D));
  B::kv_plan(space, fresh, lens, table, ring, state, one);
  B::kv_append(space, k1, v1, one, cache);
  B::kv_attention(space, q1, one, table, cache, o1, scale, 0, ws);
  CHECK((get(lens) == std::vector<int32_t>{20, 34}));
  const auto t = get(table);
  const auto ck = get(cache.k), cv = get(cache.v);
  const auto sk = get(cache.k_scale), sv = get(cache.v_scale);
  const auto h1 = get(o1);
  worst = 0;
  for (size_t b = 0; b < S; ++b) {
    const int len = b ? 34 : 20;
    std::vector<double> kk(len * KV * D), vv(len * KV * D);
    for (int j = 0; j < len; ++j)
      for (size_t g = 0; g < KV; ++g)
        for (size_t d = 0; d < D; ++d) {
          const size_t pg = t[b * cols + j / page], at = ((pg * KV + g) * page + j % page) * D + d;
          kk[(j * KV + g) * D + d] = ck[at] * double(sk[pg * KV + g]);
          vv[(j * KV + g) * D + d] = cv[at] * double(sv[pg * KV + g]);
        }
    for (size_t h = 0; h < H; ++h) {
      double o[64];
      attend(&hq1[(b * H + h) * D], &kk[(h / 2) * D], &vv[(h / 2) * D], len, D, KV * D, scale, o);
      for (size_t d = 0; d < D; ++d) worst = std::fmax(worst, std::fabs(o[d] - h1[(b * H + h) * D + d]));
    }
  }
  CHECK(worst < 2e-5);

  // ---- refusals
  auto throws = [](auto f) {
    try { f(); } catch (const std::invalid_argument&) { return true; }
    return false;
  };
  auto small = make<uint8_t, 1>(size_t(256));
  CHECK(throws([&] { B::kv_attention(space, q1, one, table, cache, o1, scale, 0, small); }));
  CHECK(throws([&] { B::kv_append(space, k, v, one, cache); }));
  CHECK(throws([&] { B::kv_attention(space, q1, one, table, cache, out, scale, 0, ws); }));
  CHECK(throws([&] { B::prompt_attention(space, q, k1, v, plan.row_start, out, scale, 0); }));
  CHECK(throws([&] { B::prompt_attention(space, q, k, v, plan.row_start, q, scale, 0); }));
  CHECK(throws([&] { B::kv_plan(space, fresh, lens, table, ring, fresh, one); }));
  CHECK(cudaDeviceSynchronize() == cudaSuccess && kdnn_b200_device_status() == 0);
  if (failures == 0) std::printf("attention: all checks passed\n");
  return failures != 0;
}
