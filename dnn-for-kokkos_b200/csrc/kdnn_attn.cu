// Causal grouped attention: over the paged 8-bit cache (kdnn_b200_kv_attention) and over packed prompts
// (kdnn_b200_prompt_attention).
#include "kdnn_common.cuh"

namespace kdnn {

// The sequence of row r: largest b with row_start[b] <= r, or -1 where r lies outside all of them.
__device__ __forceinline__ int seq_of_row(const int32_t* row_start, int seqs, int r) {
  if (r < row_start[0] || r >= row_start[seqs]) return -1;
  int lo = 0, hi = seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (row_start[mid] <= r) lo = mid; else hi = mid;
  }
  return lo;
}

// One CTA of four warps per (row, head): a warp takes every fourth token, a lane every 32nd element; running maximum and
// sum per warp, joined at the end.
template <class ST, bool PAGED>
__global__ void __launch_bounds__(128) attn_row_kernel(AttnArgs a, const int8_t* kc, const int8_t* vc, const float* ks,
                                                       const float* vs, int pages, int page) {
  pdl_chain_entry();
  const int r = blockIdx.x, h = blockIdx.y, D = a.dim, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = seq_of_row(a.row_start, a.seqs, r);
  if (b < 0) return;
  const int g = h / (a.heads / a.kv_heads);
  const int i = r - a.row_start[b];
  const int pos = PAGED ? a.first[b] + i : i;
  const int end = PAGED ? min(pos + 1, a.lens[b]) : pos + 1;
  const int beg = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const ST* q = static_cast<const ST*>(a.q) + static_cast<size_t>(r) * a.ldq + static_cast<size_t>(h) * a.hdq;
  float qv[8], o[8], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    qv[e] = e * 32 + lane < D ? to_f32(q[e * 32 + lane]) : 0.0f;
    o[e] = 0.0f;
  }
  for (int t = beg + w; t < end; t += 4) {
    float kv[8], vv[8];
    if (PAGED) {
      const int j = t / page;
      const int pg = j < a.cols ? a.table[static_cast<size_t>(b) * a.ldt + j] : -1;
      if (pg < 0 || pg >= pages) continue;
      const size_t ph = static_cast<size_t>(pg) * a.kv_heads + g, at = (ph * page + t % page) * D;
      const float s0 = ks[ph], s1 = vs[ph];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = e * 32 + lane;
        kv[e] = d < D ? static_cast<float>(kc[at + d]) * s0 : 0.0f;
        vv[e] = d < D ? static_cast<float>(vc[at + d]) * s1 : 0.0f;
      }
    } else {
      const size_t row = static_cast<size_t>(a.row_start[b]) + t;
      const ST* k = static_cast<const ST*>(a.k) + row * a.ldk + static_cast<size_t>(g) * a.hdk;
      const ST* v = static_cast<const ST*>(a.v) + row * a.ldv + static_cast<size_t>(g) * a.hdv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = e * 32 + lane;
        kv[e] = d < D ? to_f32(k[d]) : 0.0f;
        vv[e] = d < D ? to_f32(v[d]) : 0.0f;
      }
    }
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += qv[e] * kv[e];
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s), f = mn == -INFINITY ? 0.0f : expf(m - mn), p = mn == -INFINITY ? 0.0f : expf(s - mn);
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f + p * vv[e];
    m = mn;
  }
  __shared__ float sm[4], sl[4], so[4][256];
  if (lane == 0) { sm[w] = m; sl[w] = l; }
#pragma unroll
  for (int e = 0; e < 8; ++e) so[w][e * 32 + lane] = o[e];
  __syncthreads();
  const float mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  float f[4], sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[k] = sm[k] == -INFINITY ? 0.0f : expf(sm[k] - mx);
    sum += f[k] * sl[k];
  }
  ST* out = static_cast<ST*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.hdo;
  for (int d = threadIdx.x; d < D; d += 128) {
    const float v = f[0] * so[0][d] + f[1] * so[1][d] + f[2] * so[2][d] + f[3] * so[3][d];
    store_scalar(out + d, sum != 0.0f ? v / sum : 0.0f);
  }
}

template <bool PAGED>
static cudaError_t launch_rows(const AttnArgs& a, const kdnn_b200_kv_cache* c, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.rows), static_cast<unsigned>(a.heads));
  const int8_t *k = c ? c->k : nullptr, *v = c ? c->v : nullptr;
  const float *ks = c ? c->k_scale : nullptr, *vs = c ? c->v_scale : nullptr;
  const int pages = c ? static_cast<int>(c->pages) : 0, page = c ? static_cast<int>(c->page) : 0;
  return a.scalar == KDNN_F32 ? launch_chained(attn_row_kernel<float, PAGED>, grid, dim3(128), 0, st, a, k, v, ks, vs, pages, page)
                              : launch_chained(attn_row_kernel<__nv_bfloat16, PAGED>, grid, dim3(128), 0, st, a, k, v, ks, vs, pages, page);
}

cudaError_t prompt_attention_launch(const AttnArgs& a, cudaStream_t st) { return launch_rows<false>(a, nullptr, st); }

}  // namespace kdnn
