// The paged 8-bit key / value cache: page plan of a step (block table, slot map, page writes) and the write of new
// rows. No counterpart in the reference's hot path; its int8 cache is src/KokkosDNN_KVCache.hpp.
//
// A page holds `page` tokens of every head as int8 codes [head][token][dim] and one power-of-two scale per head for
// keys and one for values: x = code * scale. A power of two makes every operation of the cache exact but the rounding
// of a code itself, so the same rows give the same cache on any machine, a page whose scale has to grow moves its
// older codes by a shift, and the attention kernel applies scales without error.
#include "kdnn_common.cuh"

#include <algorithm>

namespace kdnn {

// ---- page plan ------------------------------------------------------------------------------------------
// Per sequence b, cached tokens L, fresh tokens n (negative: the sequence has ended and gives its pages back):
//   row_start = min(cumsum max(n, 0), rows), m = its difference; have = ceil(L / page);
//   need = min(ceil((L + m) / page), cols) - have; pages are handed out in sequence order while there are any:
//   got = clamp(available - sum of the needs before, 0, need); stored = min(m, (have + got) page - L).
// Everything is a prefix sum over the sequences followed by independent entries, so each CTA forms the sums for itself in
// shared memory and writes its share of the entries. Where lens / state are updated in place, a large plan's CTAs are one cluster, whose
// barrier lies between the last read of them and their new values; else there are as many CTAs as there is work for.
constexpr int kPlanCluster = 8, kPlanCtas = 64;

struct PlanArgs {
  const int32_t *fresh, *lens, *state;
  int32_t *table, *ring, *row_start, *first, *lens_out, *state_out, *slots;
  int4* writes;
  size_t ldt;
  int B, shift, rows, cols, pages, most;   // pages of 1 << shift tokens
  bool in_place;                           // lens_out / state_out overlap lens / state
};

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
}
// Exclusive sum over the block's threads of one 64-bit value each; `total` comes back to everybody.
template <int THREADS>
__device__ __forceinline__ long long block_exclusive(long long v, long long* warps, long long& total) {
  constexpr int W = THREADS / 32;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  auto scan = [&](long long x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += u;
    }
    return x;
  };
  const long long inc = scan(v);
  __syncthreads();   // the sums of the call before have been read
  if (lane == 31) warps[w] = inc;
  __syncthreads();
  const long long all = scan(lane < W ? warps[lane] : 0);
  total = __shfl_sync(0xffffffffu, all, W - 1);
  const long long base = __shfl_sync(0xffffffffu, all, w == 0 ? 0 : w - 1);
  return (w == 0 ? 0 : base) + inc - v;
}

// Largest b with at[b] <= x, for at[0] = 0 <= x < at[n]
__device__ __forceinline__ int upper_of(const int* at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_plan_kernel(PlanArgs a) {
  pdl_chain_entry();
  extern __shared__ int sm[];
  __shared__ long long s_warps[THREADS / 32];
  const int B = a.B, shift = a.shift, page = 1 << shift;
  int* rs   = sm;              // [B + 1] first row of a sequence
  int* tk   = rs + B + 1;      // [B + 1] pages taken before it
  int* gv   = tk + B + 1;      // [B + 1] pages given back before it
  int* wr   = gv + B + 1;      // [B + 1] page writes before it
  int* len  = wr + B + 1;      // [B] tokens it holds (of an ended one: what it gives back)
  int* stor = len + B;         // [B] fresh tokens that get a slot; -1: ended
  const int per = (B + THREADS - 1) / THREADS, b0 = min(B, static_cast<int>(threadIdx.x) * per), b1 = min(B, b0 + per);
  int head = a.state[0];
  const int avail = max(0, min(a.pages, a.state[1]));
  if (head < 0 || head >= a.pages) head = ((head % a.pages) + a.pages) % a.pages;
  const int tail = head + avail >= a.pages ? head + avail - a.pages : head + avail;

  long long n = 0, total, all;
  for (int b = b0; b < b1; ++b) {
    const int f = a.fresh[b];
    stor[b] = f;
    len[b]  = max(0, static_cast<int>(min(static_cast<long long>(a.lens[b]), static_cast<long long>(a.cols) * page)));
    n += max(f, 0);
  }
  long long at = block_exclusive<THREADS>(n, s_warps, all);
  for (int b = b0; b < b1; ++b) {
    rs[b] = static_cast<int>(min(at, static_cast<long long>(a.rows)));
    at += max(stor[b], 0);
  }
  if (threadIdx.x == 0) rs[B] = static_cast<int>(min(all, static_cast<long long>(a.rows)));
  __syncthreads();

  auto held  = [&](int b) { return (len[b] + page - 1) >> shift; };
  auto wants = [&](int b) {
    if (stor[b] < 0) return 0;
    const long long to = static_cast<long long>(len[b]) + (rs[b + 1] - rs[b]);
    return static_cast<int>(min((to + page - 1) >> shift, static_cast<long long>(a.cols))) - held(b);
  };
  long long need = 0, back = 0;
  for (int b = b0; b < b1; ++b) {
    need += wants(b);
    back += stor[b] < 0 ? held(b) : 0;
  }
  long long take = block_exclusive<THREADS>(need, s_warps, total), give = block_exclusive<THREADS>(back, s_warps, total);
  const int given = static_cast<int>(min(total, static_cast<long long>(a.pages)));
  long long put = 0, kept = 0;
  for (int b = b0; b < b1; ++b) {
    const int w = wants(b), h = held(b);
    const long long left = avail - take;
    const int got = static_cast<int>(left <= 0 ? 0 : left < w ? left : w);
    tk[b] = static_cast<int>(min(take, static_cast<long long>(avail)));
    gv[b] = static_cast<int>(min(give, static_cast<long long>(a.pages)));
    take += w;
    if (stor[b] < 0) {
      give += h;
      continue;
    }
    const int st = static_cast<int>(min(static_cast<long long>(rs[b + 1] - rs[b]), static_cast<long long>(h + got) * page - len[b]));
    stor[b] = st;
    kept += st;
    put += st > 0 ? ((len[b] + st - 1) >> shift) - (len[b] >> shift) + 1 : 0;
  }
  long long stored;
  block_exclusive<THREADS>(kept, s_warps, stored);
  long long w0 = block_exclusive<THREADS>(put, s_warps, total);
  const int touched = static_cast<int>(min(total, static_cast<long long>(a.most)));
  for (int b = b0; b < b1; ++b) {
    wr[b] = static_cast<int>(min(w0, static_cast<long long>(a.most)));
    w0 += stor[b] > 0 ? ((len[b] + stor[b] - 1) >> shift) - (len[b] >> shift) + 1 : 0;
  }
  if (threadIdx.x == THREADS - 1) {
    tk[B] = static_cast<int>(min(take, static_cast<long long>(avail)));
    gv[B] = given;
    wr[B] = touched;
  }
  __syncthreads();
  const int taken = tk[B];

  auto ring_at = [&](int from, int i) { return from + i >= a.pages ? from + i - a.pages : from + i; };   // i <= pages
  // the j-th page of sequence b: what the table holds, or the ring's next ones
  auto page_of = [&](int b, int j) {
    const int h = held(b);
    return j < h ? a.table[static_cast<size_t>(b) * a.ldt + j] : a.ring[ring_at(head, tk[b] + j - h)];
  };
  const int step = static_cast<int>(gridDim.x) * THREADS, me = static_cast<int>(blockIdx.x) * THREADS + threadIdx.x;
  const int rows = rs[B];
  // four rows per search; a page is looked up where it changes
  const bool wide = (reinterpret_cast<uintptr_t>(a.slots) & 15u) == 0;
  for (int r0 = me * 4; r0 < a.rows; r0 += step * 4) {
    int out[4] = {-1, -1, -1, -1};
    if (r0 < rows) {
      int b = upper_of(rs, B, r0), at_b = -1, at_j = -1, pg = -1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = r0 + k;
        if (r >= rows) break;
        while (r >= rs[b + 1]) ++b;
        const int i = r - rs[b];
        if (i < stor[b]) {
          const int pos = len[b] + i, j = pos >> shift;
          if (b != at_b || j != at_j) {
            pg = page_of(b, j);
            at_b = b;
            at_j = j;
          }
          if (pg >= 0 && pg < a.pages) out[k] = (pg << shift) + (pos & (page - 1));
        }
      }
    }
    if (wide && r0 + 4 <= a.rows) *reinterpret_cast<int4*>(a.slots + r0) = make_int4(out[0], out[1], out[2], out[3]);
    else
      for (int k = 0; k < 4 && r0 + k < a.rows; ++k) a.slots[r0 + k] = out[k];
  }
  for (int w = me; w < a.most; w += step) {
    int4 e = make_int4(0, 0, 0, 0);
    if (w < touched) {
      const int b = upper_of(wr, B, w), j = (len[b] >> shift) + w - wr[b];
      const int lo = max(j << shift, len[b]);
      const int hi = static_cast<int>(min((static_cast<long long>(j) + 1) << shift, static_cast<long long>(len[b]) + stor[b]));
      e = make_int4(rs[b] + lo - len[b], hi - lo, page_of(b, j), lo - (j << shift));
    }
    a.writes[w] = e;
  }
  for (int p = me; p < taken; p += step) {
    const int b = upper_of(tk, B, p);
    a.table[static_cast<size_t>(b) * a.ldt + held(b) + p - tk[b]] = a.ring[ring_at(head, p)];
  }
  for (int p = me; p < given; p += step) {
    const int b = upper_of(gv, B, p);
    a.ring[ring_at(tail, p)] = a.table[static_cast<size_t>(b) * a.ldt + p - gv[b]];
  }
  if (a.in_place && gridDim.x > 1) cluster_sync_all(); else __syncthreads();
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < B; b += THREADS) {
      const bool ended = stor[b] < 0;
      a.row_start[b] = rs[b];
      a.first[b]     = ended ? 0 : len[b];
      a.lens_out[b]  = ended ? 0 : len[b] + stor[b];
    }
    if (threadIdx.x == 0) {
      a.row_start[B]   = rows;
      a.state_out[0]   = ring_at(head, taken) % a.pages;
      a.state_out[1]   = avail - taken + given;
      a.state_out[2]   = static_cast<int>(min(all - stored, 0x7fffffffLL));
      a.state_out[3]   = touched;
    }
  }
}

template <int THREADS>
static cudaError_t launch_plan(const PlanArgs& a, unsigned ctas, cudaStream_t st) {
  static SmemAttrOnce once;
  const cudaError_t e = set_max_smem_once(once, kv_plan_kernel<THREADS>, (6 * 8192 + 4) * 4);
  if (e != cudaSuccess) return e;
  const size_t smem = (6 * static_cast<size_t>(a.B) + 4) * 4;
  if (a.in_place && ctas > 1) return launch_chained_cluster(kv_plan_kernel<THREADS>, dim3(ctas), dim3(THREADS), smem, ctas, st, a);
  return launch_chained(kv_plan_kernel<THREADS>, dim3(ctas), dim3(THREADS), smem, st, a);
}
static bool overlap(const int32_t* x, const int32_t* y, size_t n) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
  return a < b + n * 4 && b < a + n * 4;
}

cudaError_t kv_plan_launch(const int32_t* fresh, const int32_t* lens, const int32_t* state, int32_t* table, size_t ldt, size_t cols,
                           int32_t* ring, size_t pages, size_t B, size_t page, size_t rows, int32_t* row_start, int32_t* first,
                           int32_t* lens_out, int32_t* state_out, int32_t* slots, int32_t* writes, size_t most, cudaStream_t st) {
  int shift = 4;
  while ((size_t(1) << shift) < page) ++shift;
  PlanArgs a{fresh, lens, state, table, ring, row_start, first, lens_out, state_out, slots, reinterpret_cast<int4*>(writes), ldt,
             static_cast<int>(B), shift, static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(pages),
             static_cast<int>(most), overlap(lens, lens_out, B) || overlap(state, state_out, 4)};
  // one CTA of 256 threads while each has a few entries (a decode step of 64 sequences: 6.7 us, 12.6 with 1024 threads), else large ones
  // (134 000 rows of 200 sequences: 9.3 us, on a cluster of eight 16)
  const size_t work = rows / 4 + most;
  if (work + B <= 1024) return launch_plan<256>(a, 1, st);
  return launch_plan<1024>(a, a.in_place ? kPlanCluster : static_cast<unsigned>(std::min<size_t>(kPlanCtas, work / 1024 + 1)), st);
}

// ---- new rows into the cache ---------------------------------------------------------------------------------
struct AppendArgs {
  const void* x[2];        // keys, values [rows][heads][dim]
  size_t ld[2], hd[2];     // row and head pitch in elements
  int8_t* codes[2];
  float* scale[2];
  const int4* writes;
  int rows, pages, heads, page, dim;
};

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float pow2_of(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }
// The smallest power of two s with amax <= 127 s, at least 2^-100; 0 for 0. 127 / 128 of the next power of two is the
// mantissa 0x7E0000.
__device__ __forceinline__ float scale_for(float amax) {
  if (!(amax > 0.0f)) return 0.0f;
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 127 - 6 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return pow2_of(max(e, -100));
}
// x / s for a power of two s (inv = 1 / s), to the nearest code; infinities are the largest code, NaN is 0.
__device__ __forceinline__ int code_of(float x, float inv) {
  const float q = rintf(__fmul_rn(x, inv));
  return q != q ? 0 : static_cast<int>(fminf(fmaxf(q, -127.0f), 127.0f));
}

// T threads per job, a job being (page write, head, key or value): the rows are read once and kept in registers where they fit (8 T pieces
// of 8 elements), the largest of them gives the page's scale, then they are rounded and written.
// Bound by memory for prompts; for a decode step by the chain entry -> rows and old scale -> codes.
template <class XT, int T>
__global__ void __launch_bounds__(T < 128 ? 128 : T) kv_append_kernel(AppendArgs a, long long jobs) {
  pdl_chain_entry();
  constexpr int JOBS = T < 128 ? 128 / T : 1;      // jobs of a CTA: a warp each, or the whole CTA for one
  static_assert(T == 32 || T >= 128, "a job is a warp's or a CTA's");
  const long long job = static_cast<long long>(blockIdx.x) * JOBS + threadIdx.x / T;
  if (job >= jobs) return;
  const unsigned place = static_cast<unsigned>(job >> 1), entry = place / static_cast<unsigned>(a.heads);
  const int t = threadIdx.x % T, h = static_cast<int>(place - entry * a.heads);
  const bool z = job & 1;
  const int4 e = a.writes[entry];
  const int row0 = e.x, count = e.y, pg = e.z, off = e.w;
  // an entry without rows, or one that does not name a place of the cache
  if (count <= 0 || row0 < 0 || row0 > a.rows - count || pg < 0 || pg >= a.pages || off < 0 || off > a.page - count) return;
  const int D = a.dim;
  const size_t ld = z ? a.ld[1] : a.ld[0], ph = static_cast<size_t>(pg) * a.heads + h;
  const XT* x = static_cast<const XT*>(z ? a.x[1] : a.x[0]) + static_cast<size_t>(row0) * ld + static_cast<size_t>(h) * (z ? a.hd[1] : a.hd[0]);
  int8_t* codes = (z ? a.codes[1] : a.codes[0]) + ph * a.page * D;
  float* scale = (z ? a.scale[1] : a.scale[0]) + ph;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | (ld * sizeof(XT))) & 15u) == 0;
  const int per_row = D / 8, work = count * per_row;
  const float old = off > 0 ? *scale : 0.0f;
  float v[8][8], amax = 0.0f;
  auto read = [&](int i0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + t + k * T;
      if (i < work) load8<XT>(x + static_cast<size_t>(i / per_row) * ld, static_cast<size_t>(i % per_row) * 8, vec, v[k]);
    }
  };
  for (int i0 = 0; i0 < work; i0 += 8 * T) {
    read(i0);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (i0 + t + k * T < work) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float m = fabsf(v[k][j]);
          if (m <= 3.402823466e38f) amax = fmaxf(amax, m);   // finite values alone
        }
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (T > 32) {
    __shared__ float s_max[T / 32];
    if ((t & 31) == 0) s_max[t >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < T / 32; ++k) amax = fmaxf(amax, s_max[k]);
  }
  const float s = fmaxf(old, scale_for(amax)), inv = s > 0.0f ? 1.0f / s : 0.0f;
  if (off > 0 && old != s) {   // the page's scale grows: older codes follow
    const float ratio = __fmul_rn(old, inv);
    for (int i = t; i < off * D / 16; i += T) {
      uint4 w = reinterpret_cast<uint4*>(codes)[i];
      uint32_t* u = &w.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          r |= (static_cast<uint32_t>(code_of(static_cast<float>(static_cast<int8_t>(u[k] >> (8 * j))), ratio)) & 0xFFu) << (8 * j);
        u[k] = r;
      }
      reinterpret_cast<uint4*>(codes)[i] = w;
    }
  }
  uint2* mine = reinterpret_cast<uint2*>(codes + static_cast<size_t>(off) * D);
  for (int i0 = 0; i0 < work; i0 += 8 * T) {
    if (work > 8 * T) read(i0);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + t + k * T;
      if (i >= work) break;
      uint32_t r[2] = {0u, 0u};
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j >> 2] |= (static_cast<uint32_t>(code_of(v[k][j], inv)) & 0xFFu) << (8 * (j & 3));
      mine[i] = make_uint2(r[0], r[1]);
    }
  }
  if (t == 0) *scale = s;
}

template <class XT>
static cudaError_t launch_append(const AppendArgs& a, size_t most, cudaStream_t st) {
  const long long jobs = static_cast<long long>(most) * a.heads * 2;
  // a warp per job where a page gets a few rows, else as many threads as hold a page of rows
  const int T = a.rows < 8 * static_cast<long long>(most) ? 32 : a.page * a.dim <= 8192 ? 128 : a.page * a.dim <= 16384 ? 256 : 512;
  const long long ctas = T == 32 ? (jobs + 3) / 4 : jobs;
  if (ctas > 0x7fffffffLL || jobs > 0x1ffffffffLL) return cudaErrorInvalidConfiguration;
  const dim3 grid(static_cast<unsigned>(ctas));
  switch (T) {
    case 32: return launch_chained(kv_append_kernel<XT, 32>, grid, dim3(128), 0, st, a, jobs);
    case 128: return launch_chained(kv_append_kernel<XT, 128>, grid, dim3(128), 0, st, a, jobs);
    case 256: return launch_chained(kv_append_kernel<XT, 256>, grid, dim3(256), 0, st, a, jobs);
    default: return launch_chained(kv_append_kernel<XT, 512>, grid, dim3(512), 0, st, a, jobs);
  }
}

cudaError_t kv_append_launch(const void* k, size_t ldk, size_t hdk, const void* v, size_t ldv, size_t hdv, int scalar, size_t rows,
                             const int32_t* writes, size_t most, const kdnn_b200_kv_cache* c, cudaStream_t st) {
  AppendArgs a{{k, v}, {ldk, ldv}, {hdk, hdv}, {c->k, c->v}, {c->k_scale, c->v_scale}, reinterpret_cast<const int4*>(writes),
               static_cast<int>(rows), static_cast<int>(c->pages), static_cast<int>(c->kv_heads), static_cast<int>(c->page),
               static_cast<int>(c->dim)};
  return scalar == KDNN_F32 ? launch_append<float>(a, most, st) : launch_append<__nv_bfloat16>(a, most, st);
}

}  // namespace kdnn
