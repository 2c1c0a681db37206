// Causal grouped attention over the paged 8-bit cache (kdnn_b200_kv_attention).
//
// For a query row q of kv head g, with codes k_j, v_j and power-of-two page scales a_j, b_j:
//   s_j = scale log2(e) a_j (q . k_j),  out = sum_j 2^s_j b_j v_j / sum_j 2^s_j.
// HBM-bound: every cached byte is read once by one warp and used for all query rows of its group, 8 NT at a time.
//  * A unit is (sequence, kv head, tile of 8 NT query rows); its tokens are cut into tiles of 16 (a page holds whole ones).
//    The tiles of all units form one line; each warp takes an equal run of it, so a long context is split over as many
//    warps as a batch of short ones. Runs that end inside a unit leave partial sums, joined in a fixed order: within a
//    CTA through shared memory, between CTAs by kv_join_kernel.
//  * Calls of few units and short contexts, where launches and dependent loads are all, give each unit a cluster of eight CTAs, whose
//    pieces meet in distributed shared memory: one launch, no workspace (one sequence of 1900 tokens: 9.4 us, 14.3 with the join).
//  * Each warp has its own queue of tiles in shared memory, filled by cp.async: bytes in flight without registers, no barrier
//    between warps, no bank conflicts, and the cache keeps plain rows. What a fetch instruction covers matters: eight neighbouring lanes
//    a whole 128-byte line is the fast form (lanes of a quarter warp on four rows took 1.3 times as long for the same bytes).
//  * S^T = K q^T and O^T = V^T P^T on mma.sync m16n8k16 (fp16 in, fp32 sums): tokens, then channels, are the 16 rows, the
//    query rows the 8 columns, so a group of 8 heads wastes nothing. For S a code + 128 is an fp16 number by its bits alone (a
//    multiple of 2^-24), and the sums start from -128 sum(q); for O, whose sums run over the whole context, codes become
//    fp16 exactly (1024 + code + 128 by a byte permutation, minus 1152). k order and channel order are permuted the same way on both sides of a product.
//  * Weights: 2^(s + log2 b - m), one running reference for the values and one for the sum of weights, so that scales
//    that lie far apart lose neither sum. References are whole numbers and move only when a score passes them by 8 (every rescale is
//    exact). The product's weights stay below 2^15 in fp16, whose smallest step is 2^-24: a weight times its page's value scale is off by
//    2^-31 of the row's largest such product at the most, beside fp16's 11 bits, and vanishes below that.
//  * fp32 activations: q and the weights enter as two fp16 parts each (22 bits, on the same grid of 2^-24), and every tile's product is
//    added to the sums by fp32 additions (the tensor core cuts instead of rounding).
#include "kdnn_common.cuh"

#include <string.h>

#include <algorithm>

namespace kdnn {

constexpr int kKvWarps = 8;
constexpr float kLowest = -3.402823466e38f;
constexpr float kTop = 7.0f;        // weights are 2^(kTop + s - m): at most 2^15
constexpr int kSwitch = 4;          // what going to another unit costs a warp, in tiles: each unit's place in the line is that much longer
constexpr int kKnown = 1024;        // sequences whose lengths a CTA keeps in shared memory
constexpr int kLeast = 2;           // tiles that a warp takes at least

// A stage of a warp's queue: 16 tokens x DM codes of K, then of V, fetched as 16-byte pieces, eight neighbouring lanes a
// 128-byte line. Pieces are placed so that neither the writes nor the fragment reads (lane = 4 g + c) meet in a bank:
//   K, DM >= 128: piece ^ 4 (row & 1), read as pieces c + 4 k of the rows tau(g), tau(g) + 2
//   V, DM >= 128: piece ^ 2 (row / 4 % 4), read as pieces g + 8 k of the rows 4 c + i
//   V, DM = 64: row ^ (row / 4 % 2), piece ^ 2 (row / 8), read as 8 bytes at 8 g of the rows 4 c + i
template <int DM>
struct KvShape {
  static constexpr int kPieces = DM / 16, kRows = 32 / kPieces, kInstr = 16 / kRows;   // pieces of a row; rows of a fetch; fetches of K
  static constexpr int kStageBytes = 2 * 16 * DM;
  static __device__ __forceinline__ uint32_t k_put(int row, int piece) {
    return row * DM + (DM >= 128 ? piece ^ ((row & 1) << 2) : piece) * 16;
  }
  static __device__ __forceinline__ uint32_t v_put(int row, int piece) {
    return DM >= 128 ? row * DM + (piece ^ (((row >> 2) & 3) << 1)) * 16 : (row ^ ((row >> 2) & 1)) * DM + (piece ^ (((row >> 3) & 1) << 1)) * 16;
  }
};
// one partial sum: the accumulators of O^T in register order ([NT][DM / 16] x 32 lanes x 4), then per row {m (values), m (sum), sum, 0}
template <int DM, int NT>
struct KvPart {
  static constexpr int kTiles = NT * DM / 16;
  static constexpr int kRefs = kTiles * 128, kFloats = kRefs + 8 * NT * 4;
};

struct KvArgs {
  AttnArgs a;
  const int8_t *k, *v;
  const float *ks, *vs;
  int pages, pshift;
  float* parts;      // [CTA][kKvWarps + 2][KvPart::kFloats]: pieces that its warps put down before the end of their runs, then its own two
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
__device__ __forceinline__ void fetch(uint32_t dst, const void* src, int bytes) {   // bytes 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// What sequence b asks for: rows, token tiles [lo, lo + tiles) that some row of it can see (at least one, so that every row is
// written); `line` is a unit's length in the line of tiles.
struct SeqWork {
  int row0, n, first, len, lo, tiles, line, row_tiles;
};
__device__ __forceinline__ int4 seq_lengths(const AttnArgs& a, int pshift, int b) {
  const int row0 = max(a.row_start[b], 0);
  return make_int4(row0, max(min(a.row_start[b + 1], a.rows) - row0, 0), min(max(a.first[b], 0), 0x7fffffff - a.rows),
                   min(max(a.lens[b], 0), a.cols << pshift));      // nothing lies behind the table's pages
}
template <int NT>
__device__ __forceinline__ int row_tiles_of(int n, int G) {
  return static_cast<int>((static_cast<long long>(n) * G + 8 * NT - 1) / (8 * NT));
}
template <int NT>
__device__ __forceinline__ SeqWork seq_work(const AttnArgs& a, int G, int4 v) {
  SeqWork s;
  s.row0 = v.x; s.n = v.y; s.first = v.z; s.len = v.w;
  const int end = min(s.len, s.first + s.n);      // (first <= INT_MAX - rows)
  s.lo = a.window > 0 ? max(s.first - a.window + 1, 0) >> 4 : 0;
  s.tiles = s.n > 0 ? max(((end + 15) >> 4) - s.lo, 1) : 0;
  s.line = s.tiles + kSwitch;
  s.row_tiles = row_tiles_of<NT>(s.n, G);
  return s;
}

// The line before each sequence, for all threads of the CTA; at[seqs] is all of it. The first sequences' lengths stay in `known`.
template <int NT>
__device__ __forceinline__ void line_of(const AttnArgs& a, int G, int pshift, long long* at, int4* known) {
  __shared__ long long s_warp[kKvWarps];
  const int T = kKvWarps * 32, per = (a.seqs + T - 1) / T, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int b0 = min(a.seqs, static_cast<int>(threadIdx.x) * per), b1 = min(a.seqs, b0 + per);
  long long sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int4 v = seq_lengths(a, pshift, b);
    if (b < kKnown) known[b] = v;
    const SeqWork s = seq_work<NT>(a, G, v);
    at[b] = sum;
    sum += static_cast<long long>(s.line) * s.row_tiles * a.kv_heads;
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

// at[seqs + 1], known[min(seqs, kKnown)]
__host__ __device__ inline uint32_t kv_lists_bytes(int seqs) {
  return (((static_cast<uint32_t>(seqs + 1) * 8 + 15) & ~15u) + static_cast<uint32_t>(seqs < kKnown ? seqs : kKnown) * 16 + 127) & ~127u;
}

// First channel of m tile j of O^T for a lane: its accumulators are channels d (0, 1) and d + 1 (2, 3) of the rows 2 c (0, 2), 2 c + 1 (1, 3).
template <int DM>
__device__ __forceinline__ int channel_of(int j, int g) {
  return DM == 64 ? 8 * g + 2 * j : 128 * (j >> 3) + 16 * g + 2 * (j & 7);
}
// Where row fr of a unit (first flattened row f0) goes.
template <class ST>
__device__ __forceinline__ ST* out_row(const AttnArgs& a, const SeqWork& s, int kvh, int G, int f) {
  const int i = f / G;
  return static_cast<ST*>(a.out) + static_cast<size_t>(s.row0 + i) * a.ldo + static_cast<size_t>(kvh * G + f - i * G) * a.hdo;
}
__device__ __forceinline__ void store_pair(float* p, float x, float y) { p[0] = x; p[1] = y; }
__device__ __forceinline__ void store_pair(__nv_bfloat16* p, float x, float y) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
  if ((reinterpret_cast<uintptr_t>(p) & 3u) == 0) {
    *reinterpret_cast<__nv_bfloat162*>(p) = v;
  } else {
    p[0] = v.x;
    p[1] = v.y;
  }
}

// One warp, m tile j of row tile nt of a unit: its n partial sums (of(k) names the k-th) as one, in that order; to the result, or
// as a partial sum to `to`. Loads of eight pieces are in flight at once.
template <class ST, int DM, int NT, bool HERE, class Of>
__device__ __forceinline__ void join_tile(const AttnArgs& a, const SeqWork& s, int unit, int nt, int j, int n, Of of, float* to) {
  using Pt = KvPart<DM, NT>;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int at = ((nt * (DM / 16) + j) * 32 + lane) * 4, ref = Pt::kRefs + (nt * 8 + 2 * c) * 4;
  float mz[2] = {kLowest, kLowest}, ml[2] = {kLowest, kLowest}, l[2] = {0.0f, 0.0f};
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int k0 = 0; k0 < n; k0 += 8) {
    float4 x[8], m[8][2];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float* part = of(min(k0 + k, n - 1));
      auto get = [&](int i) {       // pieces of this CTA may lie in shared memory
        return HERE ? *reinterpret_cast<const float4*>(part + i) : __ldcg(reinterpret_cast<const float4*>(part + i)); };
      x[k] = get(at);
      m[k][0] = get(ref);
      m[k][1] = get(ref + 4);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k0 + k >= n) break;
      float f0[2], f1[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float nz = fmaxf(mz[h], m[k][h].x), nl = fmaxf(ml[h], m[k][h].y);
        f0[h] = ex2(mz[h] - nz);
        f1[h] = ex2(m[k][h].x - nz);
        l[h] = l[h] * ex2(ml[h] - nl) + m[k][h].z * ex2(m[k][h].y - nl);
        mz[h] = nz;
        ml[h] = nl;
      }
      o.x = o.x * f0[0] + x[k].x * f1[0];
      o.y = o.y * f0[1] + x[k].y * f1[1];
      o.z = o.z * f0[0] + x[k].z * f1[0];
      o.w = o.w * f0[1] + x[k].w * f1[1];
    }
  }
  if (to != nullptr) {
    *reinterpret_cast<float4*>(to + at) = o;
    if (j == 0 && g == 0) {
      *reinterpret_cast<float4*>(to + ref) = make_float4(mz[0], ml[0], l[0], 0.0f);
      *reinterpret_cast<float4*>(to + ref + 4) = make_float4(mz[1], ml[1], l[1], 0.0f);
    }
    return;
  }
  const int G = a.heads / a.kv_heads, kvh = unit / s.row_tiles, f = (unit - kvh * s.row_tiles) * 8 * NT + nt * 8 + 2 * c;
  const int d = channel_of<DM>(j, g);
  if (d >= a.dim) return;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (f + h >= s.n * G) continue;
    const float y = l[h] != 0.0f ? ex2(mz[h] - ml[h] - kTop) / l[h] : 0.0f;
    const float u = h ? o.y : o.x, v = h ? o.w : o.z;
    store_pair(out_row<ST>(a, s, kvh, G, f + h) + d, y != 0.0f ? u * y : 0.0f, y != 0.0f ? v * y : 0.0f);
  }
}

// Short calls: a cluster of kCluster CTAs for one unit, whose pieces meet in distributed shared memory, without a second kernel.
constexpr int kCluster = 8, kShort = 16384;
// The unit of cluster `index`, by every warp for itself; false: there is none.
template <int NT>
__device__ __forceinline__ bool unit_of_cluster(const AttnArgs& a, int G, int pshift, int index, int& b, int& unit, SeqWork& s) {
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < a.seqs; b0 += 32) {
    const int mine = b0 + lane;
    const int4 v = mine < a.seqs ? seq_lengths(a, pshift, mine) : make_int4(0, 0, 0, 0);
    const int units = v.y > 0 ? row_tiles_of<NT>(v.y, G) * a.kv_heads : 0;
    int inc = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const unsigned here = __ballot_sync(0xffffffffu, index >= inc - units && index < inc);
    if (here != 0) {
      const int src = __ffs(here) - 1;
      b = b0 + src;
      unit = index - __shfl_sync(0xffffffffu, inc - units, src);
      s = seq_work<NT>(a, G, make_int4(__shfl_sync(0xffffffffu, v.x, src), __shfl_sync(0xffffffffu, v.y, src),
                                       __shfl_sync(0xffffffffu, v.z, src), __shfl_sync(0xffffffffu, v.w, src)));
      return true;
    }
    index -= __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}
__device__ __forceinline__ void cluster_meet() { asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory"); }
__device__ __forceinline__ const float* of_rank(const float* p, int rank) {      // the same place in another CTA of the cluster
  uint64_t r;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(r) : "l"(p), "r"(rank));
  return reinterpret_cast<const float*>(r);
}

// FULL: dim == DM (piece addresses are immediate offsets). CLUSTER: a unit per cluster, else equal runs of the line per warp.
template <class ST, int DM, int NT, int STAGES, bool FULL, bool CLUSTER>
__global__ void __launch_bounds__(kKvWarps * 32, NT == 1 && DM <= 128 ? 2 : 1) kv_attention_kernel(KvArgs p) {
  using Sh = KvShape<DM>;
  using Pt = KvPart<DM, NT>;
  constexpr int PARTS = sizeof(ST) == 4 ? 2 : 1;
  constexpr int KS = DM / 16;                       // k steps of S, and m tiles of O
  static_assert(Pt::kFloats * 4 <= STAGES * Sh::kStageBytes, "a piece fits where the queue was");
  pdl_chain_entry();
  extern __shared__ __align__(16) uint8_t sm[];
  const AttnArgs& a = p.a;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  const int G = a.heads / a.kv_heads, D = FULL ? DM : a.dim, page = 1 << p.pshift;
  long long* at = reinterpret_cast<long long*>(sm);
  int4* known = reinterpret_cast<int4*>(sm + ((static_cast<uint32_t>(a.seqs + 1) * 8 + 15) & ~15u));
  const uint32_t ring = smem_u32(sm) + (CLUSTER ? 0u : kv_lists_bytes(a.seqs));
  __shared__ int s_order[kKvWarps][2 * kKvWarps];
  __shared__ int4 s_seg[2 * kKvWarps];              // pieces of this CTA's warps: {b, unit, 1, in the queue's place}; z 0: none
  if (!CLUSTER) line_of<NT>(a, G, p.pshift, at, known);
  auto work_of = [&](int b) { return seq_work<NT>(a, G, b < kKnown ? known[b] : seq_lengths(a, p.pshift, b)); };
  // Runs: every warp takes one while there are kLeast tiles for it; with fewer, the first CTAs' warps do. (Several runs per warp, the later
  // ones by CTAs that follow on the SMs that finish early, cost more than the SMs' different bandwidths: 122 us against 98 for
  // three contexts of 131071.)
  struct Runs {
    long long total, share;
    int workers, longer;      // the first `longer` ones take one tile more
    __device__ __forceinline__ Runs(long long all) : total(all) {
      workers = static_cast<int>(max(1LL, min(static_cast<long long>(kKvWarps) * gridDim.x, (all + kLeast - 1) / kLeast)));
      share   = all < 0x7fffffffLL ? static_cast<int>(all) / workers : all / workers;
      longer  = static_cast<int>(all - share * workers);
    }
    __device__ __forceinline__ long long start(int i) const { return i >= workers ? total : share * i + min(i, longer); }
    __device__ __forceinline__ int of(long long x) const {      // the run that tile x lies in
      const long long cut = (share + 1) * longer;
      return static_cast<int>(x < cut ? x / (share + 1) : longer + (x - cut) / share);
    }
  };
  int b = 0;
  SeqWork s{};
  long long in_b = 0;          // tiles of sequence b before pos
  long long pos = 0, end = 0;
  int cluster_unit = 0, workers = 0;
  const int rank = static_cast<int>(blockIdx.x) % kCluster;
  if (CLUSTER) {
    if (!unit_of_cluster<NT>(a, G, p.pshift, static_cast<int>(blockIdx.x) / kCluster, b, cluster_unit, s)) return;   // (all of the cluster)
    workers = min(kCluster * kKvWarps, (s.tiles + kLeast - 1) / kLeast);
    const int i = rank * kKvWarps + w, share = s.tiles / workers, longer = s.tiles - share * workers;
    end  = i < workers ? share + (i < longer ? 1 : 0) : 0;
    in_b = static_cast<long long>(cluster_unit) * s.line + kSwitch + share * i + min(i, longer);
  } else {
    const Runs runs(at[a.seqs]);
    pos = runs.start(blockIdx.x * kKvWarps + w);
    end = runs.start(blockIdx.x * kKvWarps + w + 1);
  }
  bool first_piece = true;      // of the run
  if (lane < 2) s_seg[2 * w + lane] = make_int4(0, 0, 0, 0);

  const uint32_t my_ring = ring + static_cast<uint32_t>(w) * STAGES * Sh::kStageBytes;
  // the pieces this lane fetches: row lr + i kRows, piece lc; and where it reads
  const int lr = lane / Sh::kPieces, lc = lane % Sh::kPieces;
  const int lane_at = lr * D + (FULL || lc * 16 < D ? lc * 16 : 0), lane_bytes = FULL || lc * 16 < D ? 16 : 0;
  const int tau = 4 * (g >> 1) + (g & 1), dk = 16 * c;

  float acc[NT][KS][4];
  float mz[NT][2], ml[NT][2], l[NT][2];

  if (!CLUSTER && pos < end) {
    int lo = 0, hi = a.seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (at[mid] <= pos) lo = mid; else hi = mid;
    }
    b = lo;
    s = work_of(b);
    in_b = pos - at[b];
  }
  while (pos < end) {
    while (!CLUSTER && in_b >= static_cast<long long>(s.line) * s.row_tiles * a.kv_heads) {
      in_b = 0;
      s = work_of(++b);
    }
    const int unit = in_b < 0x7fffffffLL ? static_cast<int>(in_b) / s.line : static_cast<int>(in_b / s.line);
    const int place = static_cast<int>(in_b - static_cast<long long>(unit) * s.line);
    const int run = static_cast<int>(min(static_cast<long long>(s.line - place), end - pos));
    const bool first_of_run = first_piece;
    first_piece = false;
    pos += run;
    in_b += run;
    const int tile = max(place - kSwitch, 0), take = place + run - kSwitch - tile;
    if (take <= 0) continue;      // the run ends before the unit's first tile
    const int kvh = s.row_tiles == 1 ? unit : unit / s.row_tiles, rt = unit - kvh * s.row_tiles;
    const int f0 = rt * 8 * NT, fn = min(8 * NT, s.n * G - f0);            // query rows of the unit: token f / G, head f % G
    // tiles that some row of the unit sees
    const int p_lo = s.first + f0 / G, p_hi = s.first + (f0 + fn - 1) / G;
    const int u_hi = min(s.len, p_hi + 1), u_lo = a.window > 0 ? max(p_lo - a.window + 1, 0) : 0;
    const int t_beg = max(s.lo + tile, u_lo >> 4), t_end = min(s.lo + tile + take, (u_hi + 15) >> 4);

    // ---- the unit's query rows are requested
    constexpr int QW = DM / 4 * sizeof(ST) / 16;      // 16-byte words of a lane's share of a row
    uint4 raw[NT][QW];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int f = min(nt * 8 + g, fn - 1) + f0, i = f / G;
      const ST* q = static_cast<const ST*>(a.q) + static_cast<size_t>(s.row0 + i) * a.ldq + static_cast<size_t>(kvh * G + f - i * G) * a.hdq;
      constexpr int PER = 16 / sizeof(ST);            // elements of a word
      const bool vec = (reinterpret_cast<uintptr_t>(q) & 15u) == 0;
#pragma unroll
      for (int k = 0; k < QW; ++k) {
        const int d = 64 * (k / (16 / PER)) + dk + PER * (k % (16 / PER));
        raw[nt][k] = make_uint4(0u, 0u, 0u, 0u);
        if (d < D) {
          if (vec) {
            raw[nt][k] = *reinterpret_cast<const uint4*>(q + d);
          } else {
            ST v[PER];
#pragma unroll
            for (int e = 0; e < PER; ++e) v[e] = q[d + e];
            memcpy(&raw[nt][k], v, 16);
          }
        }
      }
    }

    // ---- queue of tiles. The next 32 pages and their scales are held one per lane; those of the 32 before stay for the
    // tiles that are still in the queue.
    int chunk = -32, c_pg = -1, o_chunk = -32, o_pg = -1;
    float c_ks = 0.0f, c_vs = 0.0f, o_ks = 0.0f, o_vs = 0.0f;
    const int8_t *kp = p.k, *vp = p.v;
    int there = 0, in_stage = 0;
    auto issue = [&](int t) {
      if (t < t_end) {
        const int off = (t << 4) & (page - 1);
        if (off == 0 || t == t_beg) {
          const int j = (t << 4) >> p.pshift;
          if (j - chunk >= 32) {
            o_chunk = chunk; o_pg = c_pg; o_ks = c_ks; o_vs = c_vs;
            chunk = j;
            const int jj = j + lane;
            c_pg = -1;
            if (jj < a.cols && (static_cast<long long>(jj) << p.pshift) < u_hi) c_pg = a.table[static_cast<size_t>(b) * a.ldt + jj];
            if (c_pg >= p.pages || c_pg < 0) {
              c_pg = -1;
            } else {
              const size_t ph = static_cast<size_t>(c_pg) * a.kv_heads + kvh;
              c_ks = p.ks[ph];
              c_vs = p.vs[ph];
            }
          }
          const int pg = __shfl_sync(0xffffffffu, c_pg, j - chunk);
          there = pg >= 0 ? lane_bytes : 0;
          const size_t base = ((static_cast<size_t>(max(pg, 0)) * a.kv_heads + kvh) * page + off) * D + lane_at;
          kp = p.k + base;
          vp = p.v + base;
        } else {
          kp += 16 * D;
          vp += 16 * D;
        }
        const uint32_t kd = my_ring + in_stage * Sh::kStageBytes, vd = kd + 16 * DM;
#pragma unroll
        for (int i = 0; i < Sh::kInstr; ++i) fetch(kd + Sh::k_put(lr + i * Sh::kRows, lc), kp + i * Sh::kRows * D, there);
#pragma unroll
        for (int i = 0; i < Sh::kInstr; ++i) fetch(vd + Sh::v_put(lr + i * Sh::kRows, lc), vp + i * Sh::kRows * D, there);
      }
      fetch_commit();
      if (++in_stage == STAGES) in_stage = 0;
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(t_beg + i);

    // ---- query rows as fp16 fragments
    uint32_t qf[PARTS][NT][KS][2];
    float rsc[NT][2], bias[NT][2];      // factor of a row's scores; 128 sum(q) in their units: products are with code + 128
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[DM / 4];
      float amax = 0.0f;
#pragma unroll
      for (int k = 0; k < QW; ++k) {
        constexpr int PER = 16 / sizeof(ST);
        ST v[PER];
        memcpy(v, &raw[nt][k], 16);
#pragma unroll
        for (int e = 0; e < PER; ++e) {
          x[k * PER + e] = to_f32(v[e]);
          amax = fmaxf(amax, fabsf(x[k * PER + e]));
        }
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // the row's largest value is taken to [2^7, 2^8)
      const int e = amax > 0.0f ? max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100) : 0;
      const float to = __uint_as_float(static_cast<uint32_t>(7 - e + 127) << 23);
      const float back = __uint_as_float(static_cast<uint32_t>(e - 7 + 127) << 23);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float v0 = x[4 * j + 2 * h] * to, v1 = x[4 * j + 2 * h + 1] * to;
          const uint32_t u = half_pair(v0, v1);
          qf[0][nt][j][h] = u;
          sum += half_low(u) + half_high(u);
          if (PARTS == 2) {
            const uint32_t r = half_pair(v0 - half_low(u), v1 - half_high(u));
            qf[PARTS - 1][nt][j][h] = r;
            sum += half_low(r) + half_high(r);
          }
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float r = a.scale * 1.4426950408889634f * back;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        rsc[nt][h]  = __shfl_sync(0xffffffffu, r, (2 * c + h) * 4) * 16777216.0f;
        bias[nt][h] = __shfl_sync(0xffffffffu, sum, (2 * c + h) * 4) * -0x1p-17f;
        mz[nt][h] = ml[nt][h] = kLowest;
        l[nt][h] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < KS; ++j)
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) acc[nt][j][e2] = 0.0f;
    }
    // tiles [in_lo, in_hi) are seen whole by every row
    const int in_hi = min(s.len, p_lo + 1) >> 4, in_lo = a.window > 0 ? (max(p_hi - a.window + 1, 0) + 15) >> 4 : 0;

    int stage = 0;
    bool gone = false;                                   // the page is not there
    float ev = 0.0f;                                     // log2 of its value scale
    float rk[NT][2], az[NT][2], lim[NT][2];              // score factor, exponent offset of the weights, where a reference moves
    auto refs = [&]() {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          az[nt][h]  = ev + kTop - mz[nt][h];
          lim[nt][h] = fminf(ml[nt][h], mz[nt][h] - ev) + 8.0f;
        }
    };
    for (int t = t_beg; t < t_end; ++t) {
      __syncwarp();             // the stage that the next fetch goes to has been read
      issue(t + STAGES - 1);
      fetch_wait<STAGES - 1>();
      __syncwarp();             // everybody's pieces are there
      if (((t << 4) & (page - 1)) == 0 || t == t_beg) {   // another page
        const int j = (t << 4) >> p.pshift;
        const bool old = j < chunk;
        const int src = j - (old ? o_chunk : chunk);
        gone = __shfl_sync(0xffffffffu, old ? o_pg : c_pg, src) < 0;
        const float ks = __shfl_sync(0xffffffffu, old ? o_ks : c_ks, src);
        const uint32_t vb = __float_as_uint(__shfl_sync(0xffffffffu, old ? o_vs : c_vs, src));
        ev = vb == 0u ? -INFINITY : static_cast<float>(static_cast<int>((vb >> 23) & 0xFFu) - 127);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) rk[nt][h] = rsc[nt][h] * ks;
        refs();
      }
      const uint32_t kd = my_ring + stage * Sh::kStageBytes, vd = kd + 16 * DM;
      if (++stage == STAGES) stage = 0;
      // ---- S^T: codes + 128 as fp16 by their bits (whole multiples of 2^-24)
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nt][e] = bias[nt][e & 1];
#pragma unroll
      for (int k = 0; k < DM / 64; ++k) {
        const uint4 k0 = lds128(kd + Sh::k_put(tau, c + 4 * k)), k1 = lds128(kd + Sh::k_put(tau + 2, c + 4 * k));
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u0 = w0[j] ^ 0x80808080u, u1 = w1[j] ^ 0x80808080u;
          const uint32_t a0 = prmt(u0, 0u, 0x4140), a2 = prmt(u0, 0u, 0x4342), a1 = prmt(u1, 0u, 0x4140), a3 = prmt(u1, 0u, 0x4342);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int pt = 0; pt < PARTS; ++pt) mma16816(sc[nt], a0, a1, a2, a3, qf[pt][nt][4 * k + j][0], qf[pt][nt][4 * k + j][1]);
        }
      }
      // ---- scores: token tau(g) (e = 0, 1) and tau(g) + 2 (e = 2, 3) against the rows 2 c, 2 c + 1
      const bool edge = t >= in_hi || t < in_lo || gone;
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[nt][e] *= rk[nt][e & 1];
      if (edge) {
        const int t0 = (t << 4) + 4 * (g >> 1) + (g & 1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int ps = s.first + (f0 + min(nt * 8 + 2 * c + h, fn - 1)) / G;
            const int hi = gone ? 0 : min(s.len, ps + 1), lo = a.window > 0 ? ps - a.window + 1 : 0;
            if (t0 >= hi || t0 < lo) sc[nt][h] = -INFINITY;
            if (t0 + 2 >= hi || t0 + 2 < lo) sc[nt][2 + h] = -INFINITY;
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) over |= fmaxf(sc[nt][h], sc[nt][2 + h]) > lim[nt][h];
      if (__any_sync(0xffffffffu, over)) {     // a reference moves: both, for every row
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fmaxf(sc[nt][h], sc[nt][2 + h]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float nl = fmaxf(ml[nt][h], ceilf(top)), nz = fmaxf(mz[nt][h], ceilf(top) + ev);
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
        refs();
      }
      uint32_t pf[PARTS][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float wv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          l[nt][e & 1] += ex2(sc[nt][e] - ml[nt][e & 1]);
          wv[e] = ex2(sc[nt][e] + az[nt][e & 1]);
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
          const uint32_t ad = vd + Sh::v_put(4 * c + i, DM == 64 ? g >> 1 : g + 8 * k) + (DM == 64 ? 8 * (g & 1) : 0);
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
    if (take == s.tiles) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int fr = nt * 8 + 2 * c + h;
          if (fr >= fn) continue;
          ST* o = out_row<ST>(a, s, kvh, G, f0 + fr);
          const float f = l[nt][h] != 0.0f ? ex2(mz[nt][h] - ml[nt][h] - kTop) / l[nt][h] : 0.0f;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            const int d = channel_of<DM>(j, g);
            if (FULL || d < D) store_pair(o + d, f != 0.0f ? acc[nt][j][h] * f : 0.0f, f != 0.0f ? acc[nt][j][2 + h] * f : 0.0f);
          }
        }
    } else {
      // at most two pieces in a run: of a unit that began before it (or at its start), and of one that goes on behind it
      // (the last one lies where the warp's queue was)
      const int slot = 2 * w + (first_of_run ? 0 : 1);
      float* part = pos == end ? reinterpret_cast<float*>(sm + (my_ring - smem_u32(sm)))
                               : p.parts + (static_cast<size_t>(blockIdx.x) * (kKvWarps + 2) + w) * Pt::kFloats;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int j = 0; j < KS; ++j)
          *reinterpret_cast<float4*>(part + ((nt * KS + j) * 32 + lane) * 4) = make_float4(acc[nt][j][0], acc[nt][j][1], acc[nt][j][2], acc[nt][j][3]);
        if (g == 0) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float4*>(part + Pt::kRefs + (nt * 8 + 2 * c + h) * 4) = make_float4(mz[nt][h], ml[nt][h], l[nt][h], 0.0f);
        }
      }
      if (lane == 0) s_seg[slot] = make_int4(b, unit, 1, pos == end);
    }
  }

  if (CLUSTER) {      // the CTA's pieces, in its warps' order, then the cluster's, in its CTAs' order; an m tile per warp
    if (workers == 1) return;
    const float* queues = reinterpret_cast<const float*>(sm + (ring - smem_u32(sm)));
    float* piece = reinterpret_cast<float*>(sm + kKvWarps * STAGES * Sh::kStageBytes);
    const int held = min(workers - rank * kKvWarps, kKvWarps), ctas = (workers + kKvWarps - 1) / kKvWarps;
    __syncthreads();
    if (held > 0)
      for (int x = w; x < Pt::kTiles; x += kKvWarps)
        join_tile<ST, DM, NT, true>(a, s, cluster_unit, x / KS, x % KS, held, [&](int k) { return queues + k * (STAGES * Sh::kStageBytes / 4); }, piece);
    cluster_meet();
    for (int x = rank + kCluster * w; x < Pt::kTiles; x += kCluster * kKvWarps)
      join_tile<ST, DM, NT, true>(a, s, cluster_unit, x / KS, x % KS, ctas, [&](int k) { return of_rank(piece, k); }, nullptr);
    cluster_meet();      // nobody's memory goes before it has been read
    return;
  }
  // ---- pieces of one unit that this CTA's warps hold are joined, an m tile per warp
  __syncthreads();
  const Runs runs(at[a.seqs]);
  const long long cta0 = runs.start(blockIdx.x * kKvWarps), cta1 = runs.start((blockIdx.x + 1) * kKvWarps);
  const float* mine = p.parts + static_cast<size_t>(blockIdx.x) * (kKvWarps + 2) * Pt::kFloats;
  const float* queues = reinterpret_cast<const float*>(sm + (ring - smem_u32(sm)));
  int4 goes_on = make_int4(0, 0, 0, 0);
  const int4 seg = lane < 2 * kKvWarps ? s_seg[lane] : make_int4(0, 0, 0, 0);
  for (unsigned left = __ballot_sync(0xffffffffu, seg.z != 0); left != 0;) {
    const int i = __ffs(left) - 1, ub = __shfl_sync(0xffffffffu, seg.x, i), uu = __shfl_sync(0xffffffffu, seg.y, i);
    const unsigned group = __ballot_sync(0xffffffffu, seg.z != 0 && seg.x == ub && seg.y == uu);
    left &= ~group;
    if ((group >> lane) & 1u) s_order[w][__popc(group & ((1u << lane) - 1u))] = lane;
    __syncwarp();
    const SeqWork u = work_of(ub);
    const long long u1 = at[ub] + static_cast<long long>(uu + 1) * u.line, u0 = u1 - u.tiles;
    float* to = p.parts + (static_cast<size_t>(blockIdx.x) * (kKvWarps + 2) + kKvWarps + (u0 < cta0 ? 0 : 1)) * Pt::kFloats;
    for (int x = w; x < Pt::kTiles; x += kKvWarps)
      join_tile<ST, DM, NT, true>(a, u, uu, x / KS, x % KS, __popc(group), [&](int k) {
        const int at = s_order[w][k];
        return s_seg[at].w ? queues + (at >> 1) * (STAGES * Sh::kStageBytes / 4) : mine + (at >> 1) * Pt::kFloats; },
                            u0 >= cta0 && u1 <= cta1 ? nullptr : to);
    if (u0 >= cta0 && u1 > cta1) {      // how many CTAs further its last tile is
      goes_on = make_int4(runs.of(u1 - 1) / kKvWarps - static_cast<int>(blockIdx.x), ub, uu, 0);
    }
    __syncwarp();
  }
  if (threadIdx.x == 0) p.joins[blockIdx.x] = goes_on;
}

// Units that several CTAs share, joined by the one they begin in: an m tile per SPLIT warps, which take a stretch of the pieces each and meet
// in shared memory where there are many.
template <class ST, int DM, int NT, int SPLIT>
__global__ void __launch_bounds__(NT * DM * 2 * SPLIT) kv_join_kernel(KvArgs p) {
  using Pt = KvPart<DM, NT>;
  pdl_chain_entry();
  const int4 job = __ldcg(p.joins + blockIdx.x);
  if (job.x <= 0) return;
  const SeqWork u = seq_work<NT>(p.a, p.a.heads / p.a.kv_heads, seq_lengths(p.a, p.pshift, job.y));
  const float* first = p.parts + (static_cast<size_t>(blockIdx.x) * (kKvWarps + 2) + kKvWarps) * Pt::kFloats;
  const int w = threadIdx.x >> 5, x = w % Pt::kTiles, pieces = job.x + 1;
  auto piece = [&](int k) { return first + (static_cast<size_t>(k) * (kKvWarps + 2) + (k == 0 ? 1 : 0)) * Pt::kFloats; };
  if (SPLIT == 1 || pieces <= 8 * SPLIT) {
    if (SPLIT == 1 || w < Pt::kTiles) join_tile<ST, DM, NT, false>(p.a, u, job.z, x / (DM / 16), x % (DM / 16), pieces, piece, nullptr);
    return;
  }
  __shared__ __align__(16) float s_part[SPLIT][SPLIT > 1 ? Pt::kFloats : 4];
  const int part = w / Pt::kTiles, k0 = pieces * part / SPLIT, k1 = pieces * (part + 1) / SPLIT;
  join_tile<ST, DM, NT, false>(p.a, u, job.z, x / (DM / 16), x % (DM / 16), k1 - k0, [&](int k) { return piece(k0 + k); }, s_part[part]);
  __syncthreads();
  if (part == 0) join_tile<ST, DM, NT, true>(p.a, u, job.z, x / (DM / 16), x % (DM / 16), SPLIT, [&](int k) { return s_part[k]; }, nullptr);
}

template <class ST, int DM, int NT, int STAGES, bool FULL>
static cudaError_t launch_kv(const KvArgs& p, int ctas, bool few, cudaStream_t st) {
  const size_t ring = static_cast<size_t>(kKvWarps) * STAGES * KvShape<DM>::kStageBytes;
  const size_t smem = kv_lists_bytes(p.a.seqs) + ring;
  static SmemAttrOnce once;
  cudaError_t e = set_max_smem_once(once, kv_attention_kernel<ST, DM, NT, STAGES, FULL, false>, static_cast<int>(ring + kv_lists_bytes(8192)));
  if (e == cudaSuccess)
    e = launch_chained(kv_attention_kernel<ST, DM, NT, STAGES, FULL, false>, dim3(ctas), dim3(kKvWarps * 32), smem, st, p);
  if (e != cudaSuccess) return e;
  if constexpr (NT == 1 && DM <= 128)
    if (few) return launch_chained(kv_join_kernel<ST, DM, NT, 4>, dim3(ctas), dim3(NT * DM * 8), 0, st, p);
  return launch_chained(kv_join_kernel<ST, DM, NT, 1>, dim3(ctas), dim3(NT * DM * 2), 0, st, p);
}
template <class ST, int DM, int STAGES>
static cudaError_t launch_kv_cluster(const KvArgs& p, int units, cudaStream_t st) {
  const size_t smem = static_cast<size_t>(kKvWarps) * STAGES * KvShape<DM>::kStageBytes + KvPart<DM, 1>::kFloats * 4;
  static SmemAttrOnce once;
  const cudaError_t e = set_max_smem_once(once, kv_attention_kernel<ST, DM, 1, STAGES, true, true>, static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  return launch_chained_cluster(kv_attention_kernel<ST, DM, 1, STAGES, true, true>, dim3(units * kCluster), dim3(kKvWarps * 32), smem, kCluster, st, p);
}
template <class ST, int DM, int NT, int STAGES>
static cudaError_t launch_kv_dim(const KvArgs& p, int ctas, bool few, cudaStream_t st) {
  return p.a.dim == DM ? launch_kv<ST, DM, NT, STAGES, true>(p, ctas, few, st) : launch_kv<ST, DM, NT, STAGES, false>(p, ctas, few, st);
}

int device_sm_count();
static int kv_dm(size_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Query rows per unit: the group's rows of one sequence fill one tile of 8 or two. Two tiles share the conversion of every
// code, but halve the warps that an SM holds.
static int kv_nt(size_t rows, size_t seqs, size_t heads, size_t kv_heads, int dm) {
  return dm == 256 || (rows + seqs - 1) / seqs * (heads / kv_heads) <= 8 ? 1 : 2;
}
static int kv_ctas(int nt, int dm) { return device_sm_count() * (nt == 1 && dm <= 128 ? 2 : 1); }
static size_t kv_part_floats(int nt, int dm) { return static_cast<size_t>(8 * nt) * (dm + 4); }   // KvPart::kFloats

// The same for every number of rows: the workspace of a prompt serves the decode steps behind it.
size_t kv_attention_workspace_bytes(size_t, size_t, size_t, size_t, size_t dim) {
  const int dm = kv_dm(dim);
  size_t most = 0;
  for (int nt = 1; nt <= (dm == 256 ? 1 : 2); ++nt) {
    const size_t ctas = static_cast<size_t>(kv_ctas(nt, dm));
    most = std::max(most, ((ctas * 16 + 255) & ~size_t(255)) + ((ctas * (kKvWarps + 2) * kv_part_floats(nt, dm) * 4 + 255) & ~size_t(255)));
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
  // A cluster per unit while all of them are resident at once (clusters of eight fill 7/4 of a CTA per SM: 32 units took 7.5 us where
  // 10.7 are usual, 36 took 12.7 against 10.9) and the table has room for kShort tokens of a sequence at most. 8 kv heads of 128, one
  // sequence, us with clusters and without: 60 tokens 6.7 and 10.2, 1900 tokens 9.5 and 14.3, 16384 tokens 20.7 and 30.1, 32768
  // tokens 35.0 and 33.5 (64 CTAs of the 148 SMs then have too little bandwidth).
  const long long groups = a.heads / a.kv_heads, units = std::min<long long>(a.rows, a.rows * groups / 8 + a.seqs) * a.kv_heads;
  const bool clusters = nt == 1 && a.seqs <= 64 && (a.dim == 64 || a.dim == 128) && units * kCluster * 4 <= 7LL * device_sm_count() &&
                        (static_cast<long long>(a.cols) << shift) <= kShort;
  // Units of 32 pieces and more: four warps join an m tile (one kv head, 65536 tokens: 40 us, 95 with one; 8 kv heads 43 and 50; with many
  // units the larger CTAs cost up to 2 us: 64 sequences of 8192 tokens 72.8 and 70.3).
  const bool few = units * 32 <= ctas;
  auto go = [&](auto scalar) {
    using ST = decltype(scalar);
    if (clusters && dm == 64) return launch_kv_cluster<ST, 64, 6>(p, static_cast<int>(units), st);
    if (clusters) return launch_kv_cluster<ST, 128, 3>(p, static_cast<int>(units), st);
    if (dm == 64) return nt == 1 ? launch_kv_dim<ST, 64, 1, 6>(p, ctas, few, st) : launch_kv_dim<ST, 64, 2, 8>(p, ctas, few, st);
    if (dm == 128) return nt == 1 ? launch_kv_dim<ST, 128, 1, 3>(p, ctas, few, st) : launch_kv_dim<ST, 128, 2, 4>(p, ctas, few, st);
    return launch_kv_dim<ST, 256, 1, 2>(p, ctas, few, st);
  };
  return a.scalar == KDNN_F32 ? go(float{}) : go(__nv_bfloat16{});
}

}  // namespace kdnn
