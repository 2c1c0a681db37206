// Causal grouped attention over packed prompts (kdnn_b200_prompt_attention).
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2(e),  m a running reference.
//
// prompt_tc_kernel (bf16, 16-byte aligned rows): 128 query rows of one kv head, a few tokens times the
// heads of the group, are the M of a tcgen05 product, so a group shares every key and value that is fetched and a short
// prompt fills its tile. A CTA owns two such tiles (one, where heads are over 128) and walks the keys 128 at a time: TMA brings keys and values (five stages
// in turn, two for heads over 128), S = Q K^T lands in TMEM, a warpgroup per tile turns it into weights (a thread owns a row: no shuffles) and
// writes them back as bf16 over the scores, O += P V accumulates in TMEM. While one tile's scores go through the exponentials,
// the tensor cores work for the other. The reference m moves, and O is rescaled, only when a score passes it by 2^8.
// Weights are rounded to bf16 (2^-8 each, averaged over the keys); sums and references are fp32.
// A product reads masked values with weight 0, so infinities or NaN there would reach the sum. Masked places lie in a few tiles of keys alone (the
// last three of a CTA at the most and, with a window, the first two). There two warps look through the values while the weights are on their
// way, put 0 where one is not finite and note its key; rows that do see it add it to their result at the end. (8150 tokens with NaN in the rows
// behind them: 0.49 ms, as without; 221 ms when rows that had met one were computed again from their own keys. It costs 1 % and
// up to 2 %: 12 ragged prompts 63.1 us in turn with 62.3, a window of 512 over 4096 tokens 65.9 with 65.3, 77 tokens 6.4 with 6.5.)
//
// prompt_tile_kernel (fp32, any alignment, any scale): 64 query rows against 32 keys in shared memory, tf32 products of two parts each.
#include "kdnn_tc.cuh"

#include "kdnn_ring.cuh"

namespace kdnn {

cudaError_t moe_status_ptr(int** out);

// ---- which sequence and which part of it a CTA works on ---------------------------------------------------------------
struct PromptItem {
  int row0, n, part;   // first row and rows of the sequence, index of the part (the last parts, with the most keys, come first)
};
// `per`: rows of a part; item: this CTA's. All THREADS threads; false: there is no such item.
template <int THREADS>
__device__ __forceinline__ bool find_item(const AttnArgs& a, long long per, int item, PromptItem& it) {
  __shared__ int s_warp[THREADS / 32];
  __shared__ int4 s_found;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long left = item;
  for (int b0 = 0; b0 < a.seqs; b0 += THREADS) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int row0 = 0, n = 0;
    if (b < a.seqs) {
      row0 = max(a.row_start[b], 0);
      n = max(min(a.row_start[b + 1], a.rows) - row0, 0);
    }
    const int parts = static_cast<int>((n + per - 1) / per);
    int inc = parts;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    if (lane == 31) s_warp[w] = inc;
    __syncthreads();
    int base = 0, total = 0;
    for (int k = 0; k < THREADS / 32; ++k) {
      if (k < w) base += s_warp[k];
      total += s_warp[k];
    }
    const long long at = left - (base + inc - parts);
    if (at >= 0 && at < parts) s_found = make_int4(row0, n, parts - 1 - static_cast<int>(at), 0);
    __syncthreads();
    if (left < total) {
      const int4 f = s_found;
      it = PromptItem{f.x, f.y, f.z};
      return true;
    }
    left -= total;
  }
  return false;
}

// ---- fp32 tiles -----------------------------------------------------------------------------------------------------------
// S = Q K^T and O = P V on mma.sync m16n8k8 with tf32 operands in two parts, x = hi + lo: hi is x rounded to eleven bits, lo the rest
// cut to eleven, and hi hi + hi lo + lo hi leaves out 2^-21 of a product at most (bf16 values are one part). The products' own sums drop
// bits without rounding, so no more than four products with hi hi meet in one before it goes to an fp32 register by an ordinary sum.
// Values from 2^64 on, infinities and NaN among them, are not taken apart (what the lower parts bring could then overflow against the
// rest): a tile that holds one is computed by single FMAs, which leave masked keys out.
// The order of channels within 16 (of a product over them) and of keys within 8 is such that fragments are 16-byte loads and
// the scores' accumulators are the weights' operand.
constexpr int kTileM = 64, kTileN = 32, kTileWarps = kTileM / 16;
constexpr float kTileDown = 0x1p-40f;
template <int DM, int GROUPS>
struct TileShape {
  static constexpr int kKeys = kTileN * GROUPS, kThreads = kTileWarps * 32 * GROUPS;
  static constexpr int kKPitch = DM + 16, kVPitch = DM + 4, kKv = kKeys * (kKPitch + kVPitch);   // no two lanes of a load in a bank
  static constexpr int kFloats = kTileM * kKPitch + 2 * kKv;
  static_assert(GROUPS == 1 || kTileWarps * 32 * (DM / 2 + 4) <= kKv, "a group's sums fit where its keys were");
};
__device__ __forceinline__ void tile_fetch(float* dst, const void* src, bool there) {   // 16 bytes, zeros where there is nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void mma1688(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TWO>
__device__ __forceinline__ void in_parts(float x, uint32_t& hi, uint32_t& lo) {
  if (TWO) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) & 0xFFFFE000u;
  } else {
    hi = __float_as_uint(x);
    lo = 0u;
  }
}
__device__ __forceinline__ bool beyond_parts(float4 x) {
  auto size = [](float v) { return __float_as_int(v) & 0x7FFFFFFF; };
  return max(max(size(x.x), size(x.y)), max(size(x.z), size(x.w))) >= 0x5F800000;
}

// Four channels of a row; channels behind D are 0.
template <class ST>
__device__ __forceinline__ float4 four_of(const ST* p, int d, int D) {
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (d < D) load4<ST>(p, static_cast<size_t>(d), (reinterpret_cast<uintptr_t>(p) & (4 * sizeof(ST) - 1)) == 0, v);
  return make_float4(v[0], v[1], v[2], v[3]);
}

// GROUPS groups of warps hold the same rows and take kTileN keys each of what is fetched at a time.
// Warp w of a group holds the rows 16 w + g and + 8 (lane = 4 g + c): keys 8 j + 2 c, + 1 of the scores, channels 32 i + 8 c .. + 7 of the result.
template <class ST, int DM, int GROUPS>
__global__ void __launch_bounds__(kTileWarps * 32 * GROUPS, GROUPS == 2 ? 128 / DM : DM == 64 ? 3 : DM == 128 ? 2 : 1) prompt_tile_kernel(AttnArgs a) {
  using S = TileShape<DM, GROUPS>;
  constexpr int THREADS = S::kThreads;
  constexpr bool TWO = sizeof(ST) == 4;
  pdl_chain_entry();
  extern __shared__ __align__(16) float sf[];
  float *sq = sf, *kv = sq + kTileM * S::kKPitch;
  const int g = blockIdx.x % a.kv_heads, G = a.heads / a.kv_heads, D = a.dim;
  const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % kTileWarps, group = threadIdx.x / (kTileWarps * 32), lg = lane >> 2, lc = lane & 3;
  PromptItem it;
  // a part of a sequence: the tokens whose query rows (token, head of the group) fill a tile, or one token of a larger group
  const int tokens = max(kTileM / G, 1), splits = (tokens * G + kTileM - 1) / kTileM;
  const int idx = blockIdx.x / a.kv_heads;
  if (!find_item<THREADS>(a, tokens, idx / splits, it)) return;
  const int f0 = (idx % splits) * kTileM;             // first flattened row inside the part
  const int tok0 = it.part * tokens;
  const int fn = min(min(tokens, it.n - tok0) * G - f0, kTileM);
  if (fn <= 0) return;

  auto q_at = [&](int r) { return f0 + min(r, fn - 1); };
  bool odd_q = false;
  for (int i = threadIdx.x; i < kTileM * (DM / 4); i += THREADS) {
    const int r = i / (DM / 4), d = (i % (DM / 4)) * 4, f = q_at(r), t = f / G;
    const ST* q = static_cast<const ST*>(a.q) + static_cast<size_t>(it.row0 + tok0 + t) * a.ldq + static_cast<size_t>(g * G + f - t * G) * a.hdq;
    const float4 x = four_of<ST>(q, d, D);
    odd_q |= beyond_parts(x);
    *reinterpret_cast<float4*>(sq + r * S::kKPitch + d) = x;
  }
  int hi[2], lo[2];
  float m[2], l[2];
  float o[DM / 8][4];          // [4 i + e]: channels 32 i + 8 c + e and + 4 of row g, then of row g + 8
  // Set by the first tile that holds values from 2^64 on: from there on all weights are kTileDown times as large, so that their sums stay finite.
  // (Kept here, as there is no register left: 1500 tokens, 16 / 8 heads of 64 151 us, 160 with a flag in one.)
  __shared__ int s_large;
  if (threadIdx.x == 0) s_large = 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int pos = tok0 + q_at(16 * w + lg + 8 * r) / G;
    hi[r] = pos + 1;
    lo[r] = a.window > 0 ? pos - a.window + 1 : 0;
    m[r] = -INFINITY;
    l[r] = 0.0f;
  }
#pragma unroll
  for (int i = 0; i < DM / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  const int p_lo = tok0 + f0 / G, p_hi = tok0 + (f0 + fn - 1) / G;
  const int k_beg = a.window > 0 ? max(0, p_lo - a.window + 1) : 0, k_end = p_hi + 1;
  // keys that some row of this warp sees, and those that all of them see
  const int w_lo = tok0 + q_at(16 * w) / G, w_hi = tok0 + q_at(16 * w + 15) / G;
  const int see_beg = a.window > 0 ? w_lo - a.window + 1 : 0, all_beg = a.window > 0 ? w_hi - a.window + 1 : 0;
  const float c = a.scale * 1.4426950408889634f;
  // this thread's share of a tile: rows r0 + RP i, four channels at d0
  constexpr int RP = THREADS * 4 / DM, EACH = S::kKeys / RP;
  const int r0 = threadIdx.x / (DM / 4), d0 = (threadIdx.x % (DM / 4)) * 4;
  const ST* kbase = static_cast<const ST*>(a.k) + static_cast<size_t>(it.row0) * a.ldk + static_cast<size_t>(g) * a.hdk;
  const ST* vbase = static_cast<const ST*>(a.v) + static_cast<size_t>(it.row0) * a.ldv + static_cast<size_t>(g) * a.hdv;
  // fp32 rows on 16 bytes: fetched asynchronously; others loaded one by one
  const bool async = TWO && ((reinterpret_cast<uintptr_t>(kbase) | reinterpret_cast<uintptr_t>(vbase)) & 15u) == 0 && ((a.ldk | a.ldv) & 3u) == 0;
  auto share = [&](int buf) { return kv + buf * S::kKv + r0 * S::kKPitch + d0; };
  auto share_v = [&](int buf) { return kv + buf * S::kKv + S::kKeys * S::kKPitch + r0 * S::kVPitch + d0; };
  auto request = [&](int k0, int buf) {      // a key behind the last one is 0
    float *tk = share(buf), *tv = share_v(buf);
    if (async) {
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int row = k0 + r0 + RP * i;
        const bool there = row < k_end && d0 < D;
        const size_t at = there ? row : 0;
        tile_fetch(tk + RP * i * S::kKPitch, kbase + at * a.ldk + (there ? d0 : 0), there);
        tile_fetch(tv + RP * i * S::kVPitch, vbase + at * a.ldv + (there ? d0 : 0), there);
      }
    } else {
#pragma unroll 4
      for (int i = 0; i < EACH; ++i) {
        const int row = k0 + r0 + RP * i;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
        if (row < k_end) {
          x = four_of<ST>(kbase + static_cast<size_t>(row) * a.ldk, d0, D);
          y = four_of<ST>(vbase + static_cast<size_t>(row) * a.ldv, d0, D);
        }
        *reinterpret_cast<float4*>(tk + RP * i * S::kKPitch) = x;
        *reinterpret_cast<float4*>(tv + RP * i * S::kVPitch) = y;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  request(k_beg, 0);
  for (int at = k_beg, buf = 0; at < k_end; at += S::kKeys, buf ^= 1) {
    __syncthreads();      // the tile before has been used
    if (at + S::kKeys < k_end) {
      request(at + S::kKeys, buf ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    bool odd = odd_q;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      odd |= beyond_parts(*reinterpret_cast<const float4*>(share(buf) + RP * i * S::kKPitch));
      odd |= beyond_parts(*reinterpret_cast<const float4*>(share_v(buf) + RP * i * S::kVPitch));
    }
    odd = __syncthreads_or(odd);
    if (odd) {
      const bool first = s_large == 0;
      __syncthreads();      // everybody has read it
      s_large = 1;
      if (first) {
#pragma unroll
        for (int i = 0; i < DM / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] *= kTileDown;
        l[0] *= kTileDown;
        l[1] *= kTileDown;
      }
    }
    const bool large = s_large != 0;
    const int k0 = at + group * kTileN;      // this group's keys
    if (k0 > w_hi || k0 + kTileN <= see_beg) continue;
    const float *sk = kv + buf * S::kKv + group * kTileN * S::kKPitch;
    const float* sv = kv + buf * S::kKv + S::kKeys * S::kKPitch + group * kTileN * S::kVPitch;
    const float *qr = sq + (16 * w + lg) * S::kKPitch, *kr = sk + lg * S::kKPitch;
    // ---- scores
    float s[kTileN / 8][4];
#pragma unroll
    for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.0f;
    if (!odd) {
      float low[kTileN / 8][4];       // what the lower parts bring
#pragma unroll
      for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) low[j][e] = 0.0f;
#pragma unroll 2
      for (int d = 0; d < DM; d += 32) {
        float top[kTileN / 8][4];
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[j][e] = 0.0f;
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
          const float4 x0 = *reinterpret_cast<const float4*>(qr + d + h + 4 * lc), x1 = *reinterpret_cast<const float4*>(qr + 8 * S::kKPitch + d + h + 4 * lc);
          uint32_t ah[2][4], al[2][4];
          in_parts<TWO>(x0.x, ah[0][0], al[0][0]); in_parts<TWO>(x1.x, ah[0][1], al[0][1]);
          in_parts<TWO>(x0.y, ah[0][2], al[0][2]); in_parts<TWO>(x1.y, ah[0][3], al[0][3]);
          in_parts<TWO>(x0.z, ah[1][0], al[1][0]); in_parts<TWO>(x1.z, ah[1][1], al[1][1]);
          in_parts<TWO>(x0.w, ah[1][2], al[1][2]); in_parts<TWO>(x1.w, ah[1][3], al[1][3]);
#pragma unroll
          for (int j = 0; j < kTileN / 8; ++j) {
            const float4 y = *reinterpret_cast<const float4*>(kr + 8 * j * S::kKPitch + d + h + 4 * lc);
            uint32_t bh[4], bl[4];
            in_parts<TWO>(y.x, bh[0], bl[0]); in_parts<TWO>(y.y, bh[1], bl[1]);
            in_parts<TWO>(y.z, bh[2], bl[2]); in_parts<TWO>(y.w, bh[3], bl[3]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              mma1688(top[j], ah[u], bh[2 * u], bh[2 * u + 1]);
              if (TWO) {
                mma1688(low[j], ah[u], bl[2 * u], bl[2 * u + 1]);
                mma1688(low[j], al[u], bh[2 * u], bh[2 * u + 1]);
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] += top[j][e];
      }
      if (TWO) {
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] += low[j][e];
      }
    } else {
      for (int d = 0; d < DM; ++d) {
        const float x0 = qr[d], x1 = qr[8 * S::kKPitch + d];
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float y = sk[(8 * j + 2 * lc + e) * S::kKPitch + d];
            s[j][e] += x0 * y;
            s[j][2 + e] += x1 * y;
          }
      }
    }
    // ---- weights
    const bool edge = k0 + kTileN > w_lo + 1 || k0 < all_beg;
    float top[2] = {-INFINITY, -INFINITY}, f[2], ref[2];
#pragma unroll
    for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = e >> 1, key = k0 + 8 * j + 2 * lc + (e & 1);
        s[j][e] *= c;
        if (edge && (key >= hi[r] || key < lo[r])) s[j][e] = -INFINITY;
        top[r] = fmaxf(top[r], s[j][e]);
      }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float nm = fmaxf(m[r], top[r]);
      ref[r] = nm == -INFINITY ? 0.0f : nm;
      f[r] = exp2f(m[r] - ref[r]);
      m[r] = nm;
      l[r] *= f[r];
    }
#pragma unroll
    for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = exp2f(s[j][e] - ref[e >> 1]);
        if (large) s[j][e] *= kTileDown;
        l[e >> 1] += s[j][e];
      }
#pragma unroll
    for (int i = 0; i < DM / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] *= f[e >> 1];
    // ---- O += P V
    if (!odd) {
      uint32_t ph[kTileN / 8][4], pl[kTileN / 8][4];      // rows g, g + 8 at key 2 c, then at key 2 c + 1
#pragma unroll
      for (int j = 0; j < kTileN / 8; ++j) {
        in_parts<true>(s[j][0], ph[j][0], pl[j][0]); in_parts<true>(s[j][2], ph[j][1], pl[j][1]);
        in_parts<true>(s[j][1], ph[j][2], pl[j][2]); in_parts<true>(s[j][3], ph[j][3], pl[j][3]);
      }
#pragma unroll
      for (int i = 0; i < DM / 32; ++i) {
        float top[4][4], low[4][4];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[n][e] = low[n][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j) {
          const float* vr = sv + (8 * j + 2 * lc) * S::kVPitch + 32 * i + 4 * lg;
          const float4 x = *reinterpret_cast<const float4*>(vr), y = *reinterpret_cast<const float4*>(vr + S::kVPitch);
          const float v0[4] = {x.x, x.y, x.z, x.w}, v1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            uint32_t h0, h1, l0, l1;
            in_parts<TWO>(v0[n], h0, l0);
            in_parts<TWO>(v1[n], h1, l1);
            mma1688(top[n], ph[j], h0, h1);
            mma1688(low[n], pl[j], h0, h1);
            if (TWO) mma1688(low[n], ph[j], l0, l1);
          }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * i + n][e] += top[n][e] + low[n][e];
      }
    } else {
      for (int cc = 0; cc < 4; ++cc)
#pragma unroll
        for (int j = 0; j < kTileN / 8; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 8 * j + 2 * cc + e, key = k0 + row;
            const float p0 = __shfl_sync(0xffffffffu, s[j][e], (lane & 28) + cc), p1 = __shfl_sync(0xffffffffu, s[j][2 + e], (lane & 28) + cc);
            const bool in0 = key < hi[0] && key >= lo[0], in1 = key < hi[1] && key >= lo[1];
#pragma unroll
            for (int i = 0; i < DM / 32; ++i)
#pragma unroll
              for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const float v = sv[row * S::kVPitch + 32 * i + 8 * lc + 4 * h + n];
                  if (in0) o[4 * i + n][h] += p0 * v;
                  if (in1) o[4 * i + n][2 + h] += p1 * v;
                }
          }
    }
  }
  if (GROUPS == 2) {      // the second group's sums join the first one's
    float* other = kv + w * 32 * (DM / 2 + 4) + lane;
    __syncthreads();
    if (group == 1) {
#pragma unroll
      for (int i = 0; i < DM / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) other[32 * (4 * i + e)] = o[i][e];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        other[32 * (DM / 2 + r)] = m[r];
        other[32 * (DM / 2 + 2 + r)] = l[r];
      }
    }
    __syncthreads();
    if (group == 1) return;
    float f0[2], f1[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float m1 = other[32 * (DM / 2 + r)], nm = fmaxf(m[r], m1), ref = nm == -INFINITY ? 0.0f : nm;
      f0[r] = exp2f(m[r] - ref);
      f1[r] = exp2f(m1 - ref);
      l[r] = l[r] * f0[r] + other[32 * (DM / 2 + 2 + r)] * f1[r];
    }
#pragma unroll
    for (int i = 0; i < DM / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = o[i][e] * f0[e >> 1] + other[32 * (4 * i + e)] * f1[e >> 1];
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int fr = 16 * w + lg + 8 * r;
    if (fr >= fn) continue;
    const int fl = f0 + fr, t = fl / G;
    ST* out = static_cast<ST*>(a.out) + static_cast<size_t>(it.row0 + tok0 + t) * a.ldo + static_cast<size_t>(g * G + fl - t * G) * a.hdo;
#pragma unroll
    for (int i = 0; i < DM / 32; ++i) {
      const int d = 32 * i + 8 * lc;
      if (d >= D) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 4; ++n) store_scalar(out + d + 4 * h + n, o[4 * i + n][2 * r + h] / l[r]);
    }
  }
}

template <class ST, int DM, int GROUPS>
static cudaError_t launch_tile(const AttnArgs& a, unsigned ctas, cudaStream_t st) {
  using S = TileShape<DM, GROUPS>;
  static SmemAttrOnce once;
  const cudaError_t e = set_max_smem_once(once, prompt_tile_kernel<ST, DM, GROUPS>, S::kFloats * 4);
  if (e != cudaSuccess) return e;
  return launch_chained(prompt_tile_kernel<ST, DM, GROUPS>, dim3(ctas), dim3(S::kThreads), S::kFloats * 4, st, a);
}
// Two groups of warps share a tile's keys where a call has few CTAs, so that its longest rows decide: up to three per SM for heads of up to 64 (two such
// CTAs fit an SM), up to two and a half for heads of up to 128 (one fits, two of one group). fp32, us with two groups and with one:
//   heads of 64: 152 CTAs (600 tokens) 49 and 51, 376 (1500) 143 and 153, 392 (three of 500) 65 and 74, 392 (twelve of 100) 35 and 29, 752 (1500) 219 and 213
//   heads of 128: 152 CTAs 78 and 89, 304 (2400) 304 and 382, 304 (1200) 173 and 204, 368 (2900) 464 and 478, 376 (1500) 264 and 260,
//   392 (three of 500) 127 and 115, 416 (four of 200) 78 and 74, 604 (1200) 321 and 282; short prompts alone lose: 240 (twelve of 100) 45 and 39
template <class ST>
static cudaError_t launch_tiles(const AttnArgs& a, cudaStream_t st) {
  const int G = a.heads / a.kv_heads;
  const long long tokens = std::max(kTileM / G, 1), splits = (tokens * G + kTileM - 1) / kTileM;
  const long long all = std::min<long long>(a.rows, a.rows / tokens + a.seqs) * splits * a.kv_heads;
  if (all > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  const unsigned ctas = static_cast<unsigned>(all);
  if constexpr (sizeof(ST) == 4) {
    if (a.dim <= 128 && 2 * all <= (a.dim <= 64 ? 6LL : 5LL) * device_sm_count()) return a.dim <= 64 ? launch_tile<ST, 64, 2>(a, ctas, st) : launch_tile<ST, 128, 2>(a, ctas, st);
  }
  if (a.dim <= 64) return launch_tile<ST, 64, 1>(a, ctas, st);
  return a.dim <= 128 ? launch_tile<ST, 128, 1>(a, ctas, st) : launch_tile<ST, 256, 1>(a, ctas, st);
}

// ---- tcgen05 tiles ----------------------------------------------------------------------------------------------------------
constexpr int kPtKeys = 128, kPtEdges = 5;
// Weights are 2^(score - reference - kPtDown), so that sums of values near the largest number stay finite (up to 2^16 keys whose scores are all
// 2^8 above the reference, 2^24 at it); in return values below 2^-102 lose bits.
constexpr float kPtDown = 24.0f;
constexpr uint32_t kPtHalf = 128 * 128;     // 128 rows of 64 channels, 128-byte swizzle

// TILES: query tiles of a CTA. Two share every key and value and keep the tensor cores busy in turn; one is for calls that would leave SMs idle.
template <int DM, int TILES>
struct PtLayout {
  static constexpr int kThreads = 128 * TILES + 128, kWarpTma = 4 * TILES, kWarpMma = kWarpTma + 1, kStages = DM == 256 ? 2 : 5;
  static constexpr uint32_t kColumns = DM == 256 ? 512 : 256 * TILES;   // TMEM: scores of the tiles (the weights take the first half of the
  static constexpr uint32_t kO = 128 * TILES;                   // same columns), then their sums
  static constexpr uint32_t kOperand = (DM / 64) * kPtHalf;     // 128 rows x DM channels
  static constexpr uint32_t q = 0, kv = q + TILES * kOperand, bar = kv + kStages * kOperand;   // kv: keys and values in turn
  static constexpr uint32_t total = bar + 512 + 1024;           // + slack for the 1024-byte alignment of the base
  static_assert(total <= 232448 && 128 * TILES + TILES * DM <= kColumns, "one CTA's shared memory and TMEM");
};

struct alignas(64) PromptParams {
  CUtensorMap q, k, v;
  AttnArgs a;
  int G, tokens;     // heads of a group; tokens of a tile (tokens * G <= 128 rows)
  float c;           // scale * log2(e), positive
  int* status;
};

__device__ __forceinline__ void pt_load(uint32_t dst, const CUtensorMap* map, int d, int h, int row, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(d), "r"(h), "r"(row), "r"(bar)
      : "memory");
}
// rows of 128 bytes, 128-byte swizzle, eight rows per 1024-byte atom: K-major operand (channels inner, reduced) ...
__device__ __forceinline__ uint64_t pt_desc_k(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// ... and MN-major (channels inner, keys reduced): the next 64 channels one half further, the next eight keys one atom further
__device__ __forceinline__ uint64_t pt_desc_mn(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (uint64_t(kPtHalf >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// D = F32, A = B = bf16, M = 128
__device__ __forceinline__ constexpr uint32_t pt_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
      : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(0)
      : "memory");
}
__device__ __forceinline__ void pt_ld32(uint32_t t, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
        "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
        "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
        "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(t));
}
__device__ __forceinline__ void pt_st32(uint32_t t, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(t), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
      "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void pt_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ bool pt_elect() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ float pt_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pt_bf2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two bf16 values: the top bit of each half says that its exponent is all ones (infinity or NaN)
__device__ __forceinline__ uint32_t pt_ones(uint32_t v) { return (v & 0x7FFF7FFFu) + 0x00800080u; }
__device__ __forceinline__ uint32_t pt_odd(uint4 v) { return (pt_ones(v.x) | pt_ones(v.y) | pt_ones(v.z) | pt_ones(v.w)) & 0x80008000u; }
__device__ __forceinline__ uint32_t pt_odd_mask(uint32_t v) { return ((pt_ones(v) & 0x80008000u) >> 15) * 0xFFFFu; }
__device__ __forceinline__ uint32_t pt_finite(uint32_t v) { return v & ~pt_odd_mask(v); }      // 0 in its place
__device__ __forceinline__ bool pt_all_nan(uint4 v) {
  auto nan = [](uint32_t x) { return (x & 0x7FFF7FFFu) + 0x007F007Fu; };
  return (nan(v.x) & nan(v.y) & nan(v.z) & nan(v.w) & 0x80008000u) == 0x80008000u;
}
__device__ __forceinline__ uint32_t pt_add_odd(uint32_t x, uint32_t v) {      // x + what of v is not finite
  const uint32_t o = v & pt_odd_mask(v);
  return pt_bf2(__uint_as_float(x << 16) + __uint_as_float(o << 16), __uint_as_float(x & 0xFFFF0000u) + __uint_as_float(o & 0xFFFF0000u));
}

__device__ __forceinline__ void pt_add_zero(uint32_t& sum, uint32_t v) {      // sum + 0 v
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(v), "r"(0u));
}
struct PromptOdd { int row0, t0, beg, low, high, edges, end0, end1; };      // where a CTA's noted keys lie

template <int DM, int TILES>
__global__ void __launch_bounds__(128 * TILES + 128, 1) prompt_tc_kernel(const __grid_constant__ PromptParams p) {
  using L = PtLayout<DM, TILES>;
  extern __shared__ __align__(1024) uint8_t pt_raw[];
  const uint32_t base = (smem_u32(pt_raw) + 1023u) & ~1023u;
  uint8_t* smem = pt_raw + (base - smem_u32(pt_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnArgs& a = p.a;

  const uint32_t bars = base + L::bar;
  auto q_full  = [&](int x) { return bars + 8u * x; };
  auto full    = [&](int s) { return bars + 16u + 8u * s; };
  auto empty   = [&](int s) { return bars + 56u + 8u * s; };
  auto s_full  = [&](int x) { return bars + 96u + 8u * x; };
  auto p_full  = [&](int x) { return bars + 112u + 8u * x; };
  auto o_full  = [&](int x) { return bars + 128u + 8u * x; };
  const uint32_t mma_end = bars + 144u;
  // The e-th step with masked places: its values come next to their stage (v_asked), and have been looked through (v_clean). One phase each.
  auto v_asked = [&](int e) { return bars + 176u + 8u * e; };
  auto v_clean = [&](int e) { return bars + 216u + 8u * e; };
  uint32_t* tmem_slot      = reinterpret_cast<uint32_t*>(smem + L::bar + 152);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::bar + 156);
  RingArmed* ring_end      = reinterpret_cast<RingArmed*>(smem + L::bar + 160);   // what the TMA warp armed last
  uint32_t* odd_any        = reinterpret_cast<uint32_t*>(smem + L::bar + 256);
  uint32_t* odd_keys       = reinterpret_cast<uint32_t*>(smem + L::bar + 260);    // a bit per key of the tiles that hold masked places
  if (threadIdx.x == 0) {
    for (const CUtensorMap* m : {&p.q, &p.k, &p.v}) asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full(i), 1);
      mbar_init(s_full(i), 1);
      mbar_init(p_full(i), 4);
      mbar_init(o_full(i), 1);
    }
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(full(i), 1);
      mbar_init(empty(i), 1);
    }
    mbar_init(mma_end, 1);
    *abort_flag = 0;
    *ring_end = RingArmed();
    fence_barrier_init();
    fence_proxy_async();
  } else if (warp == 1) {
    if (lane < 2 * kPtEdges) mbar_init(v_asked(lane), lane < kPtEdges ? 1 : 2);      // (v_clean right behind)
    if (lane <= 4 * kPtEdges) odd_any[lane] = 0u;
    fence_barrier_init();
  }
  pdl_wait();
  const int g = blockIdx.x % a.kv_heads;
  PromptItem it;
  if (!find_item<L::kThreads>(a, TILES * p.tokens, blockIdx.x / a.kv_heads, it)) return;   // (its barriers publish the ones above)
  // tokens [t0, t0 + tokens) and [t0 + tokens, ...) of the sequence; keys from `beg` on, 128 at a time
  const int t0 = it.part * TILES * p.tokens;
  const int beg = a.window > 0 ? max(0, t0 - a.window + 1) : 0;
  const int end0 = min(it.n, t0 + p.tokens), end1 = min(it.n, t0 + TILES * p.tokens);
  const int n0 = (end0 - beg + kPtKeys - 1) / kPtKeys, n1 = TILES == 2 && end1 > end0 ? (end1 - beg + kPtKeys - 1) / kPtKeys : 0;
  const int steps = max(n0, n1);
  // Keys in [all_lo, t0] are seen by every row. Steps with others: the first `low` and those from `high` on, kPtEdges at the most (keys from beg on
  // that lie before all_lo are fewer than 256, and so are those behind t0).
  const int all_lo = a.window > 0 ? max(end0, end1) - a.window : 0;
  const int low = max((all_lo - beg + kPtKeys - 1) / kPtKeys, 0), high = (t0 - beg + 1) / kPtKeys;
  const int edges = low >= high ? steps : low + steps - high;
  auto step_of = [&](int e) { return e < low || low >= high ? e : e - low + high; };      // the e-th of them

  // The TMA warp's copies: queries, then keys 0, values 0, keys 1, ... The first ones need no room made and start at once.
  RingArmed armed;
  auto load = [&](uint32_t dst, const CUtensorMap* map, int head, int row, uint32_t bytes, uint32_t bar) {
    mbar_expect_tx(bar, bytes * (DM / 64));
    for (int d = 0; d < DM; d += 64) pt_load(dst + (d / 64) * kPtHalf, map, d, head, row, bar);
  };
  auto load_queries = [&](int x) {
    load(base + L::q + x * L::kOperand, &p.q, g * p.G, it.row0 + t0 + x * p.tokens, static_cast<uint32_t>(p.tokens * p.G) * 128u, q_full(x));
    armed.arm(L::kStages + x, 0);
  };
  auto load_keys = [&](int i, int st, uint32_t ph) {
    load(base + L::kv + st * L::kOperand, i & 1 ? &p.v : &p.k, g, it.row0 + beg + (i >> 1) * kPtKeys, kPtHalf, full(st));
    armed.arm(st, ph);
  };
  if (warp == L::kWarpMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(L::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    // The kernel behind this one may come onto the SMs when every CTA has said so or is done. A CTA says so when it has its tensor memory and not
    // before: a CTA of that kernel that took the columns first would keep them until this grid is done, and this one would wait for them
    // without end. (Said at the top, with the allocation before it, every CTA began with the allocation's time: 12 ragged prompts 63.9 us, 62.7.)
    pdl_launch_dependents();
  } else if (warp == L::kWarpTma) {
    if (lane == 0) {
      load_queries(0);
      for (int i = 0; i < min(L::kStages, 2 * steps); ++i) {
        load_keys(i, i, 0);
        if (i == 0 && n1 > 0) load_queries(1);
      }
    }
    __syncwarp();
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_slot;

  // Bounded wait of a whole warp; the vote makes the verdict uniform.
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    for (uint32_t i = 0; i < (1u << 21); ++i) {
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
      if ((i & 31u) == 31u && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
    *abort_flag = 1;
    return false;
  };
  bool ok = true;

  // Registers go where the scores are: 2 x 128 threads of 224 and 128 of 56 are the 64512 that the launch holds (168 each). (One tile alone
  // needs no split: 217 a thread, 255 for wide heads.)
  if (warp < L::kWarpTma) {
    if (TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    // ------------------------------------------------------------------ scores -> weights (a thread owns a row)
    const int x = warp >> 2, row = (warp & 3) * 32 + lane, n = x ? n1 : n0;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + x * 128, to = tmem + lanes + L::kO + x * 128;
    if (n > 0) {
      const int t = row / p.G, h = row - t * p.G, first = t0 + x * p.tokens;
      const int last = (x ? end1 : end0) - 1;
      const bool live = t < p.tokens && first + t <= last;
      const int pos = min(first + t, last);
      const int hi = pos + 1, lo = a.window > 0 ? pos - a.window + 1 : 0;
      const int in_hi = first + 1, in_lo = a.window > 0 ? last - a.window + 1 : 0;   // seen by every row
      const float c = p.c;
      float m = -INFINITY;
      float2 l2 = make_float2(0.0f, 0.0f);
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = wait(s_full(x), j & 1))) break;
        tc_after();
        float s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) pt_ld32(ts + 32 * i, s[i]);
        tc_wait_ld();
        const int k0 = beg + j * kPtKeys;
        if (k0 + kPtKeys > in_hi || k0 < in_lo) {
          // a warp's rows are a few neighbouring tokens: of four blocks of 32 keys, their limits lie in one or two
          const int rh = hi - k0, rl = lo - k0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (__any_sync(0xffffffffu, rh < 32 * i + 32 || rl > 32 * i)) {
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * i + e >= rh || 32 * i + e < rl) s[i][e] = -INFINITY;
            }
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top[i] = s[i][0];
#pragma unroll
          for (int e = 1; e < 31; e += 2) top[i] = fmaxf(fmaxf(top[i], s[i][e]), s[i][e + 1]);
          top[i] = fmaxf(top[i], s[i][31]);
        }
        const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const bool moves = m == -INFINITY ? mx != -INFINITY : (mx - m) * c > 8.0f;
        if (__any_sync(0xffffffffu, moves)) {
          const float f = moves ? (m == -INFINITY ? 0.0f : pt_ex2((m - mx) * c)) : 1.0f;
          if (moves) m = mx;
          l2.x *= f;
          l2.y *= f;
          if (j > 0) {      // (the product of step j - 1 came before the scores of this one)
#pragma unroll
            for (int i = 0; i < DM / 32; ++i) {
              float o[32];
              pt_ld32(to + 32 * i, o);
              tc_wait_ld();
              uint32_t u[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(o[e] * f);
              pt_st32(to + 32 * i, u);
            }
          }
        }
        const float nm = m == -INFINITY ? 0.0f : -m * c - kPtDown;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float2 y = ffma2(make_float2(s[2 * i + (e >> 4)][2 * (e & 15)], s[2 * i + (e >> 4)][2 * (e & 15) + 1]), make_float2(c, c), make_float2(nm, nm));
            const float2 pr = make_float2(pt_ex2(y.x), pt_ex2(y.y));
            l2 = fadd2(l2, pr);
            w[e] = pt_bf2(pr.x, pr.y);
          }
          pt_st32(ts + 32 * i, w);
        }
        pt_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(x));
      }
      if (ok) ok = wait(o_full(x), 0);
      if (ok) {
        tc_after();
        const float inv = 1.0f / (l2.x + l2.y);
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(it.row0 + pos) * a.ldo + static_cast<size_t>(g * p.G + h) * a.hdo;
#pragma unroll
        for (int i = 0; i < DM / 32; ++i) {
          float o[32];
          pt_ld32(to + 32 * i, o);
          tc_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pt_bf2(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
            if (live && 32 * i + e < a.dim) *reinterpret_cast<uint4*>(out + 32 * i + e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    }
  } else if (TILES == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  }
  if (warp == L::kWarpTma) {
    // ------------------------------------------------------------------ keys and values behind the first ones
    if (lane == 0) {
      auto wait1 = [&](uint32_t bar, uint32_t parity) -> bool {
        for (uint32_t i = 0; i < (1u << 21); ++i) {
          if (mbar_try_wait(bar, parity)) return true;
          if ((i & 31u) == 31u && *abort_flag != 0) return false;
        }
        *abort_flag = 1;
        return false;
      };
      uint32_t ph = 1;
      for (int i = L::kStages, st = 0; i < 2 * steps; ++i) {
        if (!(ok = wait1(empty(st), ph ^ 1u))) break;
        load_keys(i, st, ph);
        if (++st == L::kStages) { st = 0; ph ^= 1u; }
      }
      *ring_end = armed;
    }
    __syncwarp();
  } else if (warp == L::kWarpMma) {
    // ------------------------------------------------------------------ products
    auto scores = [&](int x, int st) {
      if (pt_elect()) {
        const uint32_t qa = base + L::q + x * L::kOperand, ka = base + L::kv + st * L::kOperand;
#pragma unroll
        for (int k = 0; k < DM / 16; ++k)
          pt_mma_ss(tmem + x * 128, pt_desc_k(qa + (k >> 2) * kPtHalf + (k & 3) * 32), pt_desc_k(ka + (k >> 2) * kPtHalf + (k & 3) * 32),
                    pt_idesc(kPtKeys, false), k != 0);
        tc_commit(s_full(x));
      }
      __syncwarp();
    };
    auto sums = [&](int x, int st, bool more, bool last) {
      if (pt_elect()) {
        const uint32_t va = base + L::kv + st * L::kOperand;
#pragma unroll
        for (int k = 0; k < kPtKeys / 16; ++k)
          pt_mma_ts(tmem + L::kO + x * 128, tmem + x * 128 + 8 * k, pt_desc_mn(va + k * 2048), pt_idesc(DM, true), more || k != 0);
        if (last) tc_commit(o_full(x));
      }
      __syncwarp();
    };
    auto done = [&](uint32_t bar) {
      if (pt_elect()) tc_commit(bar);
      __syncwarp();
    };
    struct Stage { int at; uint32_t ph; } ks = {0, 0}, vs = {1, 0};
    auto two_on = [&](Stage& s) {
      s.at += 2;
      if (s.at >= L::kStages) { s.at -= L::kStages; s.ph ^= 1u; }
    };
    ok = wait(full(0), 0) && wait(q_full(0), 0);
    if (ok) {
      tc_after();
      scores(0, 0);
      if (n1 > 0) {
        ok = wait(q_full(1), 0);
        if (ok) scores(1, 0);
      }
      done(empty(0));
    }
    two_on(ks);
    int cleaned = 0;
    for (int j = 0; j < steps && ok; ++j) {
      if (!(ok = wait(full(vs.at), vs.ph))) break;
      const bool here = j < low || j >= high;
      if ((j + 1 < low || j + 1 >= high) && j + 1 < steps && lane == 0) mbar_arrive(v_asked(cleaned + here));
      if (here && !(ok = wait(v_clean(cleaned++), 0))) break;
      bool keys = false;       // the next step's keys are there
      for (int x = 0; x < TILES && ok; ++x) {
        const int n = x ? n1 : n0;
        if (j >= n) continue;
        if (!(ok = wait(p_full(x), j & 1))) break;
        tc_after();
        sums(x, vs.at, j > 0, j + 1 == n);
        if (j + 1 < n) {
          if (!keys && !(ok = wait(full(ks.at), ks.ph))) break;
          keys = true;
          scores(x, ks.at);
        }
      }
      if (!ok) break;
      done(empty(vs.at));
      if (keys) done(empty(ks.at));
      two_on(vs);
      two_on(ks);
    }
  } else if (warp > L::kWarpMma) {
    // ------------------------------------------------------------------ values of the tiles with masked places: none that is not finite
    // (the two warps take eight rows at a time; the swizzle keeps a row's pieces in the row)
    constexpr int HALVES = DM / 64;
    const int tid = static_cast<int>(threadIdx.x) - (L::kWarpMma + 1) * 32, last = max(end0, end1) - 1;
    for (int e = 0; e < edges; ++e) {
      // A parity tells a stage's next copy from the one before it, not from the one before that: the wait for the values of step j begins when the
      // product warp is at step j - 1, which has used what lay in their stage before them (the keys of step j - 2, with two stages the values of
      // j - 1), and they stay until they have been looked through.
      const int j = step_of(e), fill = 2 * j + 1, st = fill % L::kStages, k0 = beg + j * kPtKeys;
      if (j > 0) {      // behind all the steps between, each of which has the time of a wait: parked, so that two warps do not poll beside the exponentials
        ok = false;
        for (long long i = 0; i < (j + 1LL) << 16; ++i) {
          if ((ok = __all_sync(0xffffffffu, mbar_try_wait_hint(v_asked(e), 0, 20000u)))) break;
          if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        }
        if (!ok) *abort_flag = 1;
      }
      if (!(ok = ok && wait(full(st), (fill / L::kStages) & 1))) break;
      uint4* values = reinterpret_cast<uint4*>(smem + L::kv + st * L::kOperand) + tid;
      const int r_beg = j < low ? 0 : max(t0 + 1 - k0, 0) & ~7, r_end = j >= high ? kPtKeys : min(all_lo - k0, kPtKeys);
      uint32_t sum[2] = {0u, 0u};      // 0 v + 0 v + ...: NaN where one is not finite
#pragma unroll DM == 256 ? 1 : 2
      for (int r0 = r_beg; r0 < r_end; r0 += 8) {
        uint4 v[HALVES];
#pragma unroll
        for (int i = 0; i < HALVES; ++i) v[i] = values[i * 1024 + r0 * 8];
#pragma unroll
        for (int i = 0; i < HALVES; ++i) {
          pt_add_zero(sum[0], v[i].x);
          pt_add_zero(sum[1], v[i].y);
          pt_add_zero(sum[0], v[i].z);
          pt_add_zero(sum[1], v[i].w);
        }
      }
      if (pt_ones(sum[0] | sum[1]) & 0x80008000u) {
        *reinterpret_cast<PromptOdd*>(smem + L::bar + 352) = PromptOdd{it.row0, t0, beg, low, high, edges, end0, end1};
        *odd_any = 1u;
#pragma unroll 1
        for (int r0 = r_beg; r0 < r_end; r0 += 8)
#pragma unroll 1
          for (int i = 0; i < HALVES; ++i) {
            const uint4 v = values[i * 1024 + r0 * 8];
            if (pt_odd(v) == 0u) continue;
            values[i * 1024 + r0 * 8] = make_uint4(pt_finite(v.x), pt_finite(v.y), pt_finite(v.z), pt_finite(v.w));
            const int r = r0 + (tid >> 3);
            if (k0 + r <= last) atomicOr(odd_keys + 4 * e + (r >> 5), 1u << (r & 31));      // some row sees it
          }
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(v_clean(e));
    }
  }
  if (!ok && lane == 0) atomicExch(p.status, KDNN_ERR_DEVICE_WAIT);
  tc_before();
  __syncthreads();
  if (*abort_flag) {
    // some role gave up: the copies and products still in flight end (bounded) before the CTA gives its memory back
    if (warp == L::kWarpTma && lane == 0)
      ring_drain(*ring_end, L::kStages + 2, 1u << 14, [&](int s, uint32_t parity) {
        return mbar_try_wait(s < L::kStages ? full(s) : q_full(s - L::kStages), parity); });
    if (warp == L::kWarpMma && pt_elect()) {
      tc_commit(mma_end);
      mbar_wait_bounded(mma_end, 0u, 1u << 16);
    }
    __syncthreads();
  }
  if (warp == L::kWarpMma)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::kColumns) : "memory");
  if (warp < L::kWarpTma && *odd_any != 0u) {
    // Values that are not finite and were taken out: rows that see them get them now, a thread its row (written above).
    const PromptOdd o = *reinterpret_cast<const PromptOdd*>(smem + L::bar + 352);
    const int x = warp >> 2, row = (warp & 3) * 32 + lane, t = row / p.G, h = row - t * p.G, pos = o.t0 + x * p.tokens + t;
    if (t >= p.tokens || pos >= (x ? o.end1 : o.end0)) return;
    const int lo = a.window > 0 ? pos - a.window + 1 : 0;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(o.row0 + pos) * a.ldo + static_cast<size_t>(g * p.G + h) * a.hdo;
    const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(a.v) + static_cast<size_t>(o.row0) * a.ldv + static_cast<size_t>(g) * a.hdv;
#pragma unroll 1
    for (int d = 0; d < a.dim; d += 8) {
      uint4 y = *reinterpret_cast<const uint4*>(out + d);
#pragma unroll 1
      for (int b = 0; b < 4 * o.edges; ++b)
#pragma unroll 1
        for (uint32_t bits = pt_all_nan(y) ? 0u : odd_keys[b]; bits != 0; bits &= bits - 1) {
          const int e = b >> 2, key = o.beg + (e < o.low || o.low >= o.high ? e : e - o.low + o.high) * kPtKeys + 32 * (b & 3) + __ffs(bits) - 1;
          if (key < lo || key > pos) continue;
          const uint4 z = *reinterpret_cast<const uint4*>(v + static_cast<size_t>(key) * a.ldv + d);
          y = make_uint4(pt_add_odd(y.x, z.x), pt_add_odd(y.y, z.y), pt_add_odd(y.z, z.z), pt_add_odd(y.w, z.w));
          if (pt_all_nan(y)) break;
        }
      *reinterpret_cast<uint4*>(out + d) = y;
    }
  }
}

static bool encode_heads(CUtensorMap* map, const void* x, size_t ld, size_t hd, int rows, int heads, int dim, int box_heads, int box_rows) {
  TcEncodeFn fn = tc_encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[3]    = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(hd) * 2, static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[3]     = {64u, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[3]    = {1u, 1u, 1u};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DM, int TILES>
static cudaError_t launch_tc(const PromptParams& p, cudaStream_t st) {
  using L = PtLayout<DM, TILES>;
  static SmemAttrOnce once;
  const cudaError_t e = set_max_smem_once(once, prompt_tc_kernel<DM, TILES>, static_cast<int>(L::total));
  if (e != cudaSuccess) return e;
  const long long parts = std::min<long long>(p.a.rows, p.a.rows / (TILES * p.tokens) + p.a.seqs), ctas = parts * p.a.kv_heads;
  if (ctas > 0x7fffffffLL) return cudaErrorInvalidConfiguration;
  return launch_chained(prompt_tc_kernel<DM, TILES>, dim3(static_cast<unsigned>(ctas)), dim3(L::kThreads), L::total, st, p);
}
// One tile per CTA while all of them find an SM of their own (a prompt of 77 tokens, 32 / 8 heads: 7.6 us against 9.6 when it was chosen, 6.7
// now), else two (with one, 8192 tokens took 605 us against 500). Heads over 128 leave room for one: queries and two operands
// of 64 KB (4096 tokens, 8 / 4 heads of 256: 79 us, 870 TFLOP/s).
template <int DM>
static cudaError_t launch_tiles_tc(const PromptParams& p, cudaStream_t st) {
  const long long tiles = static_cast<long long>(std::min(p.a.rows, p.a.rows / p.tokens + p.a.seqs)) * p.a.kv_heads;
  return tiles <= device_sm_count() ? launch_tc<DM, 1>(p, st) : launch_tc<DM, 2>(p, st);
}

cudaError_t prompt_attention_launch(const AttnArgs& a, cudaStream_t st) {
  if (a.scalar == KDNN_F32) return launch_tiles<float>(a, st);
  const int G = a.heads / a.kv_heads;
  const size_t pitches = a.ldq | a.hdq | a.ldk | a.hdk | a.ldv | a.hdv | a.ldo | a.hdo;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                          reinterpret_cast<uintptr_t>(a.out);
  // TMA wants 16-byte pitches; the kernel's maximum is one of products, so the scale has to be positive
  if (G <= 128 && pitches % 8 == 0 && bases % 16 == 0 && a.scale > 1e-30f && a.scale < 1e30f) {
    PromptParams p;
    p.a = a;
    p.G = G;
    p.tokens = 128 / G;
    p.c = a.scale * 1.4426950408889634f;
    const cudaError_t e = moe_status_ptr(&p.status);
    if (e != cudaSuccess) return e;
    if (encode_heads(&p.q, a.q, a.ldq, a.hdq, a.rows, a.heads, a.dim, G, p.tokens) &&
        encode_heads(&p.k, a.k, a.ldk, a.hdk, a.rows, a.kv_heads, a.dim, 1, kPtKeys) &&
        encode_heads(&p.v, a.v, a.ldv, a.hdv, a.rows, a.kv_heads, a.dim, 1, kPtKeys))
      return a.dim <= 64 ? launch_tiles_tc<64>(p, st) : a.dim <= 128 ? launch_tiles_tc<128>(p, st) : launch_tc<256, 1>(p, st);
  }
  return launch_tiles<__nv_bfloat16>(a, st);
}

}  // namespace kdnn
