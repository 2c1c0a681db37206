// Causal grouped attention over the paged 8-bit cache (kdnn_b200_kv_attention).
//
// For a query row q of kv head g, with codes k_j, v_j and power-of-two page scales a_j, b_j:
//   s_j = scale log2(e) a_j (q . k_j),  out = sum_j 2^s_j b_j v_j / sum_j 2^s_j.
// HBM-bound: every cached byte is read once by one warp and used for all query rows of its group, 8 NT at a time.
//  * A unit is (sequence, kv head, tile of 8 NT query rows); its tokens are cut into tiles of 16 (a page holds whole ones).
//    The tiles of all units form one line; each warp takes an equal run of it, so a long context is split over as many
//    warps as a batch of short ones. Runs that end inside a unit leave partial sums, joined in a fixed order: within a
//    CTA through shared memory, between CTAs by kv_join_kernel.
//  * A lane fetches exactly the 16-byte pieces that its own matrix fragments come from, with cp.async into its own slots
//    of shared memory: deep queues without registers, no barriers, no bank conflicts, cache layout untouched.
//  * S^T = K q^T and O^T = V^T P^T on mma.sync m16n8k16 (fp16 in, fp32 sums): tokens, then channels, are the 16 rows, the
//    query rows the 8 columns, so a group of 8 heads wastes nothing. Codes become fp16 exactly (1024 + code + 128 by a
//    byte permutation, minus 1152); k order and channel order are permuted the same way on both sides of a product.
//  * Weights: 2^(s + log2 b - m), one running reference for the values and one for the sum of weights, so that scales
//    that lie far apart lose neither. References are whole numbers and move only when a score passes them by 8 (weights
//    stay below 2^15 in fp16; every rescale is exact).
//  * fp32 activations: q and the weights enter as two fp16 parts each (22 bits), and every tile's product is added to the sums
//    by fp32 additions (the tensor core cuts instead of rounding).
#include "kdnn_common.cuh"

#include <algorithm>

namespace kdnn {

constexpr int kKvWarps = 8;
constexpr float kLowest = -3.402823466e38f;
constexpr float kTop = 7.0f;        // weights are 2^(kTop + s - m): at most 2^15
constexpr int kLeast = 4;           // tiles that a warp takes at least

template <int DM>
struct KvShape {
  static constexpr int kKInstr = 2 * (DM / 64);                       // 16-byte pieces of K per lane and tile
  static constexpr int kVInstr = 4 * (DM >= 128 ? DM / 128 : 1);      // pieces of V (8 bytes for DM = 64)
  static constexpr int kVPiece = DM == 64 ? 8 : 16;
  static constexpr int kStageBytes = kKInstr * 512 + kVInstr * 32 * kVPiece;
};
// one partial sum: O [8 NT][DM], then m (values), m (sum), sum per row
template <int DM, int NT>
struct KvPart {
  static constexpr int kRows = 8 * NT;
  static constexpr int kFloats = kRows * (DM + 4);
};

struct KvArgs {
  AttnArgs a;
  const int8_t *k, *v;
  const float *ks, *vs;
  int pages, pshift;
  float* parts;      // [CTA][2 kKvWarps + 2][KvPart::kFloats]: its warps' pieces, then its own two
  int4* joins;       // [CTA]: the unit that begins in this CTA and ends in a later one: {CTAs that follow, b, unit, 0}
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) { return __byte_perm(a, b, s); }
// two biased codes per half2: (1024 + u) - 1152 = code
__device__ __forceinline__ uint32_t code_pair(uint32_t u, uint32_t sel) {
  const uint32_t m = prmt(u, 0x64646464u, sel);
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(m), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float half_low(uint32_t v) { return __half2float(__ushort_as_half(static_cast<unsigned short>(v & 0xFFFFu))); }
__device__ __forceinline__ float half_high(uint32_t v) { return __half2float(__ushort_as_half(static_cast<unsigned short>(v >> 16))); }
template <int N>
__device__ __forceinline__ void fetch(uint32_t dst, const void* src, int bytes) {   // bytes 0: zeros
  if (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}

// What sequence b asks for: rows, token tiles [lo, hi) that some row of it can see (at least one, so that every row is written).
struct SeqWork {
  int row0, n, first, len, lo, tiles, row_tiles;
};
template <int NT>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int pshift, int b) {
  SeqWork s;
  s.row0  = max(a.row_start[b], 0);
  s.n     = max(min(a.row_start[b + 1], a.rows) - s.row0, 0);
  s.first = min(max(a.first[b], 0), 0x7fffffff - a.rows);
  s.len   = min(max(a.lens[b], 0), a.cols << pshift);   // nothing lies behind the table's pages
  const int end = static_cast<int>(min(static_cast<long long>(s.len), static_cast<long long>(s.first) + s.n));
  s.lo = a.window > 0 ? max(s.first - a.window + 1, 0) >> 4 : 0;
  s.tiles = s.n > 0 ? max(((end + 15) >> 4) - s.lo, 1) : 0;
  const int G = a.heads / a.kv_heads;
  s.row_tiles = static_cast<int>((static_cast<long long>(s.n) * G + 8 * NT - 1) / (8 * NT));
  return s;
}

// Tiles of the sequences before each one, for all threads of the CTA; at[seqs] is their sum.
template <int NT>
__device__ __forceinline__ void line_of(const AttnArgs& a, int pshift, long long* at) {
  __shared__ long long s_warp[kKvWarps];
  const int T = kKvWarps * 32, per = (a.seqs + T - 1) / T, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int b0 = min(a.seqs, static_cast<int>(threadIdx.x) * per), b1 = min(a.seqs, b0 + per);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) {
    const SeqWork s = seq_work<NT>(a, pshift, b);
    at[b] = sum;
    sum += static_cast<long long>(s.tiles) * s.row_tiles * a.kv_heads;
  }
  long long inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) s_warp[w] = inc;
  __syncthreads();
  long long base = inc - sum, all = 0;
#pragma unroll
  for (int i = 0; i < kKvWarps; ++i) {
    if (i < w) base += s_warp[i];
    all += s_warp[i];
  }
  for (int b = b0; b < b1; ++b) at[b] += base;
  if (threadIdx.x == 0) at[a.seqs] = all;
  __syncthreads();
}

// One warp, query row r of a unit: the n partial sums that of(k) names (nullptr: none) as one, in that order; to the result, or as a
// partial sum to `to`.
template <class ST, int DM, int NT, class Of>
__device__ __forceinline__ void join_row(const AttnArgs& a, const SeqWork& s, int unit, int r, int lane, int n, Of of, float* to) {
  using Pt = KvPart<DM, NT>;
  constexpr int W = DM >= 128 ? 4 : 2, V = DM / (32 * W);     // W neighbouring channels per lane, V times
  float mz = kLowest, ml = kLowest, l = 0.0f, o[V][W];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) o[i][e] = 0.0f;
#pragma unroll 4
  for (int k = 0; k < n; ++k) {
    const float* part = of(k);
    if (part == nullptr) continue;
    const float4 m = __ldcg(reinterpret_cast<const float4*>(part + Pt::kRows * DM + r * 4));
    float x[V][W];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (W == 4) *reinterpret_cast<float4*>(x[i]) = __ldcg(reinterpret_cast<const float4*>(part + r * DM + 128 * i + 4 * lane));
      else *reinterpret_cast<float2*>(x[i]) = __ldcg(reinterpret_cast<const float2*>(part + r * DM + 2 * lane));
    }
    const float nz = fmaxf(mz, m.x), nl = fmaxf(ml, m.y);
    const float f0 = ex2(mz - nz), f1 = ex2(m.x - nz);
    l = l * ex2(ml - nl) + m.z * ex2(m.y - nl);
    mz = nz;
    ml = nl;
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int e = 0; e < W; ++e) o[i][e] = o[i][e] * f0 + x[i][e] * f1;
  }
  if (to != nullptr) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (W == 4) *reinterpret_cast<float4*>(to + r * DM + 128 * i + 4 * lane) = *reinterpret_cast<float4*>(o[i]);
      else *reinterpret_cast<float2*>(to + r * DM + 2 * lane) = *reinterpret_cast<float2*>(o[i]);
    }
    if (lane == 0) *reinterpret_cast<float4*>(to + Pt::kRows * DM + r * 4) = make_float4(mz, ml, l, 0.0f);
    return;
  }
  const int G = a.heads / a.kv_heads, kvh = unit / s.row_tiles, f = (unit - kvh * s.row_tiles) * 8 * NT + r;
  if (f >= s.n * G) return;
  const int i0 = f / G;
  ST* out = static_cast<ST*>(a.out) + static_cast<size_t>(s.row0 + i0) * a.ldo + static_cast<size_t>(kvh * G + f - i0 * G) * a.hdo;
  const float y = l != 0.0f ? ex2(mz - ml - kTop) / l : 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int d = 128 * i + W * lane + e;
      if (d < a.dim) store_scalar(out + d, y != 0.0f ? o[i][e] * y : 0.0f);
    }
}

template <class ST, int DM, int NT, int STAGES>
__global__ void __launch_bounds__(kKvWarps * 32, NT == 1 && DM <= 128 ? 2 : 1) kv_attention_kernel(KvArgs p) {
  using Sh = KvShape<DM>;
  using Pt = KvPart<DM, NT>;
  constexpr int PARTS = sizeof(ST) == 4 ? 2 : 1;
  constexpr int KS = DM / 16;                       // k steps of S, and m tiles of O
  pdl_chain_entry();
  extern __shared__ __align__(16) uint8_t sm[];
  const AttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int G = a.heads / a.kv_heads, D = a.dim, page = 1 << p.pshift;
  long long* at = reinterpret_cast<long long*>(sm);
  uint8_t* ring = sm + ((static_cast<size_t>(a.seqs + 1) * 8 + 127) & ~size_t(127));
  __shared__ float4 s_meta[kKvWarps][STAGES];
  __shared__ int4 s_seg[2 * kKvWarps];              // pieces of this CTA's warps: {b, unit, 1, .}; z 0: none
  line_of<NT>(a, p.pshift, at);
  const long long total = at[a.seqs];
  // warps that take a run: all of a CTA's where there is enough for them, else fewer in every CTA
  const int ctas = gridDim.x;
  const int wpc  = static_cast<int>(max(1LL, min(static_cast<long long>(kKvWarps), (total + static_cast<long long>(kLeast) * ctas - 1) / (static_cast<long long>(kLeast) * ctas))));
  const long long workers = max(1LL, min(static_cast<long long>(wpc) * ctas, (total + kLeast - 1) / kLeast));
  auto start_of = [&](long long i) { return i >= workers ? total : total * i / workers; };
  const long long my0 = static_cast<long long>(blockIdx.x) * wpc;
  const long long cta0 = start_of(my0), cta1 = start_of(my0 + wpc);
  long long pos = w < wpc ? start_of(my0 + w) : 0;
  const long long end = w < wpc ? start_of(my0 + w + 1) : 0, begin = pos;
  if (lane < 2) s_seg[2 * w + lane] = make_int4(0, 0, 0, 0);

  const uint32_t my_ring = smem_u32(ring) + static_cast<uint32_t>(w) * STAGES * Sh::kStageBytes;
  const uint32_t my_k = my_ring + lane * 16, my_v = my_ring + Sh::kKInstr * 512 + lane * Sh::kVPiece;

  float acc[NT][KS][4];        // O^T: m tile t = 2 word + half of word: rows d = 16 g + 2 t + {0 (c0, c1), 1 (c2, c3)}
  float mz[NT][2], ml[NT][2], l[NT][2];
  // where a lane's channels lie: DM = 64: 8 g + 2 t; 128: 16 g + 2 t; 256: 16 g + 2 t (t < 8), 128 + 16 g + 2 (t - 8)
  int b = 0;
  SeqWork s{};
  long long in_b = 0;          // tiles of sequence b before pos
  if (pos < end) {
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] <= pos) lo = mid; else hi = mid;
    }
    b = lo;
    s = seq_work<NT>(a, p.pshift, b);
    in_b = pos - at[b];
  }
  while (pos < end) {
    while (in_b >= static_cast<long long>(s.tiles) * s.row_tiles * a.kv_heads) {
      in_b = 0;
      s = seq_work<NT>(a, p.pshift, ++b);
    }
    const int unit = static_cast<int>(in_b / s.tiles), tile = static_cast<int>(in_b - static_cast<long long>(unit) * s.tiles);
    const int take = static_cast<int>(min(static_cast<long long>(s.tiles - tile), end - pos));
    const int kvh = unit / s.row_tiles, rt = unit - kvh * s.row_tiles;
    const int f0 = rt * 8 * NT, fn = min(8 * NT, s.n * G - f0);            // query rows of the unit: token f / G, head f % G
    // tiles that some row of the unit sees
    const int p_lo = s.first + f0 / G, p_hi = s.first + (f0 + fn - 1) / G;
    const int u_hi = min(s.len, p_hi + 1), u_lo = a.window > 0 ? max(p_lo - a.window + 1, 0) : 0;
    const int t_beg = max(s.lo + tile, u_lo >> 4), t_end = min(s.lo + tile + take, (u_hi + 15) >> 4);

    // ---- queue of tiles
    int chunk = -1, c_pg = -1;
    float c_ks = 0.0f, c_ev = -INFINITY;
    auto issue = [&](int t) {
      if (t < t_end) {
        const int j = (t << 4) >> p.pshift;
        if (chunk < 0 || j - chunk >= 32) {       // the next 32 pages: a page and its scales per lane
          chunk = j;
          const int jj = j + lane;
          c_pg = -1;
          if (jj < a.cols && (static_cast<long long>(jj) << p.pshift) < u_hi) c_pg = a.table[static_cast<size_t>(b) * a.ldt + jj];
          if (c_pg >= p.pages) c_pg = -1;
          if (c_pg >= 0) {
            const size_t ph = static_cast<size_t>(c_pg) * a.kv_heads + kvh;
            c_ks = p.ks[ph];
            const uint32_t vb = __float_as_uint(p.vs[ph]);
            c_ev = vb == 0u ? -INFINITY : static_cast<float>(static_cast<int>((vb >> 23) & 0xFFu) - 127);
          }
        }
        const int pg = __shfl_sync(0xffffffffu, c_pg, j - chunk);
        const float ks = __shfl_sync(0xffffffffu, c_ks, j - chunk), ev = __shfl_sync(0xffffffffu, c_ev, j - chunk);
        const int st = t % STAGES;
        if (lane == 0) s_meta[w][st] = make_float4(ks, ev, pg >= 0 ? 1.0f : 0.0f, 0.0f);
        const size_t base = ((static_cast<size_t>(max(pg, 0)) * a.kv_heads + kvh) * page + ((t << 4) & (page - 1))) * D;
        const bool there = pg >= 0;
        const uint32_t kd = my_k + st * Sh::kStageBytes, vd = my_v + st * Sh::kStageBytes;
#pragma unroll
        for (int i = 0; i < Sh::kKInstr; ++i) {
          const int tok = 4 * (g >> 1) + (g & 1) + 2 * (i & 1), d = 16 * c + 64 * (i >> 1);
          fetch<16>(kd + i * 512, p.k + base + tok * D + (d < D ? d : 0), there && d < D ? 16 : 0);
        }
#pragma unroll
        for (int i = 0; i < Sh::kVInstr; ++i) {
          const int tok = 4 * c + (i & 3), d = DM == 64 ? 8 * g : 16 * g + 128 * (i >> 2);
          fetch<Sh::kVPiece>(vd + i * 32 * Sh::kVPiece, p.v + base + tok * D + (d < D ? d : 0), there && d < D ? Sh::kVPiece : 0);
        }
      }
      fetch_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(t_beg + i);

    // ---- the unit's query rows
    uint32_t qf[PARTS][NT][KS][2];
    float rsc[NT][2];
    int hi[NT][2], lo[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int f = min(nt * 8 + g, fn - 1) + f0;
      const int i = f / G;
      const ST* q = static_cast<const ST*>(a.q) + static_cast<size_t>(s.row0 + i) * a.ldq + static_cast<size_t>(kvh * G + f - i * G) * a.hdq;
      const bool vec = (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
      float x[DM / 4];
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < DM / 64; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float t[8] = {0, 0, 0, 0, 0, 0, 0, 0};
          const int d = 64 * k + 16 * c + 8 * h;
          if (d < D) load8<ST>(q, static_cast<size_t>(d), vec, t);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[k * 16 + h * 8 + e] = t[e];
            amax = fmaxf(amax, fabsf(t[e]));
          }
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the row's largest value is taken to [2^7, 2^8)
      const int e = amax > 0.0f ? max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100) : 0;
      const float to = __uint_as_float(static_cast<uint32_t>(7 - e + 127) << 23);
      const float back = __uint_as_float(static_cast<uint32_t>(e - 7 + 127) << 23);
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v0 = x[4 * j + 2 * h] * to, v1 = x[4 * j + 2 * h + 1] * to;
          qf[0][nt][j][h] = half_pair(v0, v1);
          if (PARTS == 2) qf[PARTS - 1][nt][j][h] = half_pair(v0 - half_low(qf[0][nt][j][h]), v1 - half_high(qf[0][nt][j][h]));
        }
      const float r = a.scale * 1.4426950408889634f * back;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        rsc[nt][h] = __shfl_sync(0xffffffffu, r, (2 * c + h) * 4);
        const int fr = f0 + min(nt * 8 + 2 * c + h, fn - 1), ps = s.first + fr / G;
        hi[nt][h] = min(s.len, ps + 1);
        lo[nt][h] = a.window > 0 ? ps - a.window + 1 : 0;
        mz[nt][h] = ml[nt][h] = kLowest;
        l[nt][h] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) acc[nt][j][e2] = 0.0f;
    }
    // tokens below in_hi and from in_lo on are seen by every row
    const int in_hi = min(s.len, p_lo + 1), in_lo = a.window > 0 ? p_hi - a.window + 1 : 0;

    for (int t = t_beg; t < t_end; ++t) {
      issue(t + STAGES - 1);
      fetch_wait<STAGES - 1>();
      __syncwarp();
      const int st = t % STAGES;
      const float4 meta = s_meta[w][st];
      // ---- S^T
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < DM / 64; ++k) {
        const uint4 k0 = lds128(my_k + st * Sh::kStageBytes + (2 * k) * 512), k1 = lds128(my_k + st * Sh::kStageBytes + (2 * k + 1) * 512);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u0 = w0[j] ^ 0x80808080u, u1 = w1[j] ^ 0x80808080u;
          const uint32_t a0 = code_pair(u0, 0x4140), a2 = code_pair(u0, 0x4342), a1 = code_pair(u1, 0x4140), a3 = code_pair(u1, 0x4342);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PARTS; ++pt) mma16816(sc[nt], a0, a1, a2, a3, qf[pt][nt][4 * k + j][0], qf[pt][nt][4 * k + j][1]);
        }
      }
      // ---- scores: token tau(g) (e = 0, 1) and tau(g) + 2 (e = 2, 3) against the rows 2 c, 2 c + 1
      const int t0 = (t << 4) + 4 * (g >> 1) + (g & 1);
      const bool edge = (t << 4) + 16 > in_hi || (t << 4) < in_lo || meta.z == 0.0f;
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = sc[nt][e] * rsc[nt][e & 1] * meta.x;
          if (edge) {
            const int tok = t0 + (e & 2);
            if (tok >= hi[nt][e & 1] || tok < lo[nt][e & 1] || meta.z == 0.0f) v = -INFINITY;
          }
          sc[nt][e] = v;
          over |= v > ml[nt][e & 1] + 8.0f || v + meta.y > mz[nt][e & 1] + 8.0f;
        }
      if (__any_sync(0xffffffffu, over)) {     // a reference moves: both, for every row
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(sc[nt][h], sc[nt][2 + h]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float nl = fmaxf(ml[nt][h], ceilf(top)), nz = fmaxf(mz[nt][h], ceilf(top) + meta.y);
            l[nt][h] *= ex2(ml[nt][h] - nl);
            const float f = ex2(mz[nt][h] - nz);
            ml[nt][h] = nl;
            mz[nt][h] = nz;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              acc[nt][j][h] *= f;
              acc[nt][j][2 + h] *= f;
            }
          }
      }
      uint32_t pf[PARTS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float wv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          l[nt][e & 1] += ex2(sc[nt][e] - ml[nt][e & 1]);
          wv[e] = ex2(sc[nt][e] + (meta.y + kTop) - mz[nt][e & 1]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t x = half_pair(wv[2 * h], wv[2 * h + 1]);
          pf[0][nt][h] = transposed(x);
          if (PARTS == 2) pf[PARTS - 1][nt][h] = transposed(half_pair(wv[2 * h] - half_low(x), wv[2 * h + 1] - half_high(x)));
        }
      }
      // ---- O^T
#pragma unroll
      for (int k = 0; k < (DM >= 128 ? DM / 128 : 1); ++k) {
        uint32_t v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t ad = my_v + st * Sh::kStageBytes + (4 * k + i) * 32 * Sh::kVPiece;
          if (DM == 64) {
            const uint2 x = lds64(ad);
            v[i][0] = x.x; v[i][1] = x.y; v[i][2] = v[i][3] = 0u;
          } else {
            const uint4 x = lds128(ad);
            v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
          }
        }
#pragma unroll
        for (int wi = 0; wi < (DM == 64 ? 2 : 4); ++wi) {
          uint32_t u[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) u[i] = v[i][wi] ^ 0x80808080u;
#pragma unroll
          for (int hw = 0; hw < 2; ++hw) {     // channels 4 wi + 2 hw, + 1
            const uint32_t x01 = prmt(u[0], u[1], hw ? 0x7362 : 0x5140), x23 = prmt(u[2], u[3], hw ? 0x7362 : 0x5140);
            const uint32_t a0 = code_pair(x01, 0x4140), a1 = code_pair(x01, 0x4342), a2 = code_pair(x23, 0x4140), a3 = code_pair(x23, 0x4342);
            const int j = 8 * k + 2 * wi + hw;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (PARTS == 1) {
                mma16816(acc[nt][j], a0, a1, a2, a3, pf[0][nt][0], pf[0][nt][1]);
              } else {
                float o[4] = {0, 0, 0, 0};
                mma16816(o, a0, a1, a2, a3, pf[0][nt][0], pf[0][nt][1]);
                mma16816(o, a0, a1, a2, a3, pf[PARTS - 1][nt][0], pf[PARTS - 1][nt][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][j][e] += o[e];
              }
            }
          }
        }
      }
    }
    fetch_wait<0>();
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 4);
        l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 8);
        l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 16);
      }
    const bool whole = take == s.tiles;
    if (whole) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int fr = nt * 8 + 2 * c + h;
          if (fr >= fn) continue;
          const int i = (f0 + fr) / G;
          ST* o = static_cast<ST*>(a.out) + static_cast<size_t>(s.row0 + i) * a.ldo + static_cast<size_t>(kvh * G + f0 + fr - i * G) * a.hdo;
          const float f = l[nt][h] != 0.0f ? ex2(mz[nt][h] - ml[nt][h] - kTop) / l[nt][h] : 0.0f;
#pragma unroll
          for (int j = 0; j < KS; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = DM == 64 ? 8 * g + 2 * j + e : 128 * (j >> 3) + 16 * g + 2 * (j & 7) + e;
              if (d < D) store_scalar(o + d, f != 0.0f ? acc[nt][j][2 * e + h] * f : 0.0f);
            }
        }
    } else {
      // at most two pieces in a run: of a unit that began before it (or at its start), and of one that goes on behind it
      const int slot = 2 * w + (pos == begin ? 0 : 1);
      float* part = p.parts + (static_cast<size_t>(blockIdx.x) * (2 * kKvWarps + 2) + slot) * Pt::kFloats;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int fr = nt * 8 + 2 * c + h;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            const int d = DM == 64 ? 8 * g + 2 * j : 128 * (j >> 3) + 16 * g + 2 * (j & 7);
            *reinterpret_cast<float2*>(part + fr * DM + d) = make_float2(acc[nt][j][h], acc[nt][j][2 + h]);
          }
          if (g == 0) *reinterpret_cast<float4*>(part + Pt::kRows * DM + fr * 4) = make_float4(mz[nt][h], ml[nt][h], l[nt][h], 0.0f);
        }
      if (lane == 0) s_seg[slot] = make_int4(b, unit, 1, 0);
    }
    pos += take;
    in_b += take;
  }

  // ---- pieces of one unit that this CTA's warps hold are joined, a row per warp
  __syncthreads();
  const float* mine = p.parts + static_cast<size_t>(blockIdx.x) * (2 * kKvWarps + 2) * Pt::kFloats;
  int4 goes_on = make_int4(0, 0, 0, 0);
  for (int i = 0; i < 2 * kKvWarps;) {
    const int4 seg = s_seg[i];
    if (seg.z == 0) {
      ++i;
      continue;
    }
    int n = i + 1;      // the unit's pieces follow one another, with unused places between them
    for (int k = i + 1; k < 2 * kKvWarps; ++k) {
      const int4 o = s_seg[k];
      if (o.z != 0 && (o.x != seg.x || o.y != seg.y)) break;
      if (o.z != 0) n = k + 1;
    }
    const SeqWork u = seq_work<NT>(a, p.pshift, seg.x);
    const long long u0 = at[seg.x] + static_cast<long long>(seg.y) * u.tiles, u1 = u0 + u.tiles;
    const bool whole = u0 >= cta0 && u1 <= cta1;
    float* to = p.parts + (static_cast<size_t>(blockIdx.x) * (2 * kKvWarps + 2) + 2 * kKvWarps + (u0 < cta0 ? 0 : 1)) * Pt::kFloats;
    for (int r = w; r < 8 * NT; r += kKvWarps)
      join_row<ST, DM, NT>(a, u, seg.y, r, lane, n - i, [&](int k) {
        return s_seg[i + k].z != 0 ? mine + static_cast<size_t>(i + k) * Pt::kFloats : nullptr; }, whole ? nullptr : to);
    if (u0 >= cta0 && u1 > cta1) {      // the CTA of its last tile
      long long x = (u1 - 1) * workers / total;
      while (start_of(x + 1) <= u1 - 1) ++x;
      while (start_of(x) > u1 - 1) --x;
      goes_on = make_int4(static_cast<int>(x / wpc) - static_cast<int>(blockIdx.x), seg.x, seg.y, 0);
    }
    i = n;
  }
  if (threadIdx.x == 0) p.joins[blockIdx.x] = goes_on;
}

// Units that several CTAs share, joined by the one they begin in: a row per warp.
template <class ST, int DM, int NT>
__global__ void __launch_bounds__(NT * 256) kv_join_kernel(KvArgs p) {
  using Pt = KvPart<DM, NT>;
  pdl_chain_entry();
  const int4 job = p.joins[blockIdx.x];
  if (job.x <= 0) return;
  const SeqWork u = seq_work<NT>(p.a, p.pshift, job.y);
  const int first = blockIdx.x;
  join_row<ST, DM, NT>(p.a, u, job.z, threadIdx.x >> 5, threadIdx.x & 31, job.x + 1, [&](int k) {
    return p.parts + (static_cast<size_t>(first + k) * (2 * kKvWarps + 2) + 2 * kKvWarps + (k == 0 ? 1 : 0)) * Pt::kFloats; },
    nullptr);
}

template <class ST, int DM, int NT, int STAGES>
static cudaError_t launch_kv(const KvArgs& p, int ctas, cudaStream_t st) {
  const size_t ring = static_cast<size_t>(kKvWarps) * STAGES * KvShape<DM>::kStageBytes;
  const size_t smem = ((static_cast<size_t>(p.a.seqs + 1) * 8 + 127) & ~size_t(127)) + ring;
  static SmemAttrOnce once;
  cudaError_t e = set_max_smem_once(once, kv_attention_kernel<ST, DM, NT, STAGES>, static_cast<int>(ring + 8193 * 8 + 128));
  if (e == cudaSuccess)
    e = launch_chained(kv_attention_kernel<ST, DM, NT, STAGES>, dim3(ctas), dim3(kKvWarps * 32), smem, st, p);
  if (e == cudaSuccess) e = launch_chained(kv_join_kernel<ST, DM, NT>, dim3(ctas), dim3(NT * 256), 0, st, p);
  return e;
}

int device_sm_count();
static int kv_dm(size_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Query rows per unit: the group's rows of one sequence fill one tile of 8 or two. Two tiles share the conversion of every
// code, but halve the warps that an SM holds.
static int kv_nt(size_t rows, size_t seqs, size_t heads, size_t kv_heads, int dm) {
  return dm == 256 || (rows + seqs - 1) / seqs * (heads / kv_heads) <= 8 ? 1 : 2;
}
static int kv_ctas(int nt, int dm) { return device_sm_count() * (nt == 1 && dm <= 128 ? 2 : 1); }
static size_t kv_part_floats(int nt, int dm) { return static_cast<size_t>(8 * nt) * (dm + 4); }

// The same for every number of rows: the workspace of a prompt serves the decode steps behind it.
size_t kv_attention_workspace_bytes(size_t, size_t, size_t, size_t, size_t dim) {
  const int dm = kv_dm(dim);
  size_t most = 0;
  for (int nt = 1; nt <= (dm == 256 ? 1 : 2); ++nt) {
    const size_t ctas = static_cast<size_t>(kv_ctas(nt, dm));
    most = std::max(most, ((ctas * 16 + 255) & ~size_t(255)) + ((ctas * (2 * kKvWarps + 2) * kv_part_floats(nt, dm) * 4 + 255) & ~size_t(255)));
  }
  return most;
}

cudaError_t kv_attention_launch(const AttnArgs& a, const kdnn_b200_kv_cache* c, void* ws, cudaStream_t st) {
  const int dm = kv_dm(c->dim), nt = kv_nt(a.rows, a.seqs, a.heads, a.kv_heads, dm), ctas = kv_ctas(nt, dm);
  int shift = 4;
  while ((1u << shift) < c->page) ++shift;
  KvArgs p{a, c->k, c->v, c->k_scale, c->v_scale, static_cast<int>(c->pages), shift,
           reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + ((static_cast<size_t>(ctas) * 16 + 255) & ~size_t(255))),
           static_cast<int4*>(ws)};
  auto go = [&](auto scalar) {
    using ST = decltype(scalar);
    if (dm == 64) return nt == 1 ? launch_kv<ST, 64, 1, 6>(p, ctas, st) : launch_kv<ST, 64, 2, 8>(p, ctas, st);
    if (dm == 128) return nt == 1 ? launch_kv<ST, 128, 1, 3>(p, ctas, st) : launch_kv<ST, 128, 2, 4>(p, ctas, st);
    return launch_kv<ST, 256, 1, 2>(p, ctas, st);
  };
  return a.scalar == KDNN_F32 ? go(float{}) : go(__nv_bfloat16{});
}

}  // namespace kdnn
