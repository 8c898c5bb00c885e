// Attention over a paged cache of keys and values held in 4 bits (layout: kv4_cache.cu):
//   out = sum_t p_t (s_v[t] code_v[t] + m_v[t]) / sum_t p_t,
//   p_t = exp(scale * q . (s_k[t] code_k[t] + m_k[t])) over the tokens that the query sees.
//
// The codes go into the tensor cores as they are, as small exact fp16 numbers (codes_lower below); the
// factors are taken out of q and of the results.  Scale and minimum of a token leave the products:
//   q . k_t = s_k (q . code) + m_k sum(q)            sum_t p_t v_t = sum_t (p_t s_v) code + sum_t p_t m_v
// Queries are brought to fp16 by a power of two per row (exact for 16-bit types; fp32 queries travel as two
// fp16 planes, hi + lo, 22 bits).  p_t s_v is held in fp16 relative to the running maximum of (score +
// exponent of s_v), so that it lies in [0, 2) 2^14 whatever the scales are: in two planes for fp32 and fp16,
// whose outputs then are as exact as their rounding, in one (2^-11 of each weight at most) for bf16, whose
// outputs are rounded eight times as coarsely.  The second plane and codes that are not subnormal numbers (below)
// cost 32 % on 64 x 8192 cached tokens of 8 heads (149 us for 113).  Sums, maxima and the output stay in fp32.
//
// mma.m16n8k16 with the tokens (scores) or the channels (output) as the 16 rows and eight query rows as
// the columns: S^T = K Q^T, O^T = V^T P^T.  One step of a conversation has as many query rows per
// key head as query heads share it, mostly 1 to 8, which fills the narrow side.  All operands come
// straight from global memory into the registers of the thread that multiplies them: which channel is
// which column of an MMA is free as long as both operands agree, so a thread takes consecutive bytes.
// More rows are more blocks, next to each other, which meet the codes in L2 (16 rows over 64 x 8192 tokens,
// bf16: 212 us, as two groups of eight in one block 291).
//
// Bound: dependent instructions of few warps (22 of a warp per cached token and head; issue 56 %, DRAM 47 %), then
// HBM (d + 8 bytes per cached token and head).  64 sequences of up to 8192 tokens, 8 key heads of 128, bf16: 113 us, 3.8 TB/s;
// one of 131072, 4 heads: 27 us.  The cache of one sequence and head is split over `splits` blocks and the warps of
// each; partial results (numerator, sum, maximum) are joined by kv4_join_kernel in a fixed order.  Not better: tiles
// of 64 tokens, five blocks an SM.
#include <float.h>

#include <type_traits>

#include "kv4.cuh"

namespace modiff {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kQueries = 8;               // query rows of a block
constexpr int kTile = 32;                 // tokens a warp takes at a time
constexpr int kSub = kTile / 16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kExponentBias = 47.0f;    // of the exponents of s_v in the running maximum, see there
constexpr int kMaxSplits = 256;
constexpr int kBlocksPerSm = 4;           // of the single-token kernel: 128 registers a thread

__device__ inline void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values held by the warp as an MMA fragment
__device__ inline uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// An infinite scale or minimum of a key becomes NaN, so that rows that see it are NaN: its score might be -inf, which
// would hide the key.  (inf 0 + inf; finite numbers stay as they are.)
__device__ inline uint32_t nan_unless_finite(uint32_t params) {
  const __half2 h = *reinterpret_cast<const __half2*>(&params);
  const __half2 r = __hfma2(h, __float2half2_rn(0.0f), h);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Two channels of four codes out of a word: `even` the low halves of two bytes 16 bits apart, as n unit,
// `odd` the high halves, as 16 n unit.  For bf16 unit is 2^-24 and the masked bits are the subnormal
// numbers; the even ones of the upper bytes come from a subtraction (exact), because logic instructions,
// of half the rate of additions, are what this kernel has most of.  The tensor cores align the products
// of subnormal numbers as if they had a leading bit, which leaves sums of them some 17 bits: fp16 and fp32 take
// unit 1 (0x6400 | x is the number 1024 + x), and n - 8 for n, so that sums over tokens or channels do not
// meet a large common part that the minima take out again (the accumulation truncates).
__device__ inline uint32_t half_minus(uint32_t v, float c) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(c));
  return *reinterpret_cast<const uint32_t*>(&d);
}
template <bool SUBNORMAL>
__device__ inline void codes_lower(uint32_t w, uint32_t& even, uint32_t& odd) {
  even = w & 0x000f000fu;
  odd = w & 0x00f000f0u;
  if (!SUBNORMAL) {
    even = half_minus(even | 0x64006400u, 1024.0f + 8.0f);
    odd = half_minus(odd | 0x64006400u, 1024.0f + 16.0f * 8.0f);
  }
}
template <bool SUBNORMAL>
__device__ inline void codes_upper(uint32_t w, uint32_t& even, uint32_t& odd) {
  const uint32_t t = __byte_perm(w, 0, 0x4341);
  if (SUBNORMAL) {
    odd = t & 0x00f000f0u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&t), *reinterpret_cast<const __half2*>(&odd));
    even = *reinterpret_cast<const uint32_t*>(&d);
  } else {
    codes_lower<false>(t, even, odd);
  }
}

template <typename T, int D>
constexpr int smem_bytes() {
  constexpr int planes = sizeof(T) == 4 ? 2 : 1;
  const int q = (D / 16) * 32 * 8 * planes;               // query fragments
  const int o = kWarps * kQueries * (D + 4) * 4;                 // the warps' outputs, joined at the end
  return q > o ? q : o;
}

// One block: eight query rows (query, head of the group) of one sequence and key head, one part of
// the tokens.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, D > 128 ? 2 : kBlocksPerSm)
kv4_attention_kernel(const Kv4Attention p) {
  constexpr int P = sizeof(T) == 4 ? 2 : 1;       // fp16 planes of q
  constexpr bool kCoarse = std::is_same_v<T, __nv_bfloat16>;
  constexpr int W = kCoarse ? 1 : 2;              // fp16 planes of the weights
  constexpr float kUnit = kCoarse ? 0x1p-24f : 1.0f;  // what a code of 1 is to the tensor cores
  constexpr int R = kQueries;
  constexpr int KW = D / 32;                      // words of a key row that a thread holds
  constexpr int VW = D / 64;                      // words of a value row that a thread holds
  constexpr bool kAllValues = D <= 128;  // registers for a whole tile's values
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float row_a[R], row_b[R];            // factor of a score, sum of the scaled query
  __shared__ float join_m[kWarps][R], join_l[kWarps][R], join_s[kWarps][R];

  if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, j = lane & 3;
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  const int rt = id % p.row_tiles;
  id /= p.row_tiles;
  const int head = id % p.c.heads, b = id / p.c.heads;
  const int row0 = rt * R;
  const int rows_here = min(R, p.count * p.group - row0);
  const int32_t* table = p.table + (int64_t)b * p.max_pages;
  const int length = min(max(__ldg(p.lengths + b), 0), p.max_pages * p.c.page_size);

  const int pos_lo = length - p.count + row0 / p.group;
  const int pos_hi = length - p.count + (row0 + rows_here - 1) / p.group;
  const TileRange range = tiles_of<kTile>(p, length, pos_lo, pos_hi);
  const int t_begin = (int)((int64_t)range.count * split / p.splits);
  const int t_end = (int)((int64_t)range.count * (split + 1) / p.splits);

  constexpr int kRow = D / 2;                     // bytes of a token's codes
  const uint8_t* k_lane = p.c.k_codes + g * kRow + j * (D / 8);
  const uint8_t* v_lane = p.c.v_codes + 2 * j * kRow + g * (D / 16);
  const uint32_t* kp_lane = reinterpret_cast<const uint32_t*>(p.c.k_params) + g;
  const uint32_t* vp_lane = reinterpret_cast<const uint32_t*>(p.c.v_params) + g;

  // Rows of the cache where the two pieces of 16 tokens of a tile begin; -1: not there.  Pages of whole
  // tiles are looked up once.
  const bool whole_pages = p.c.page_size % kTile == 0;
  auto place = [&](int t0, int64_t (&base)[kSub]) {
    if (whole_pages) {
      const int64_t first = kv4_place(p.c, table, p.max_pages, t0, head);
#pragma unroll
      for (int u = 0; u < kSub; ++u) base[u] = first >= 0 && t0 + 16 * u < length ? first + 16 * u : -1;
    } else {
#pragma unroll
      for (int u = 0; u < kSub; ++u)
        base[u] = t0 + 16 * u < length ? kv4_place(p.c, table, p.max_pages, t0 + 16 * u, head) : -1;
    }
  };
  // Pieces that are not there are read from the cache's beginning, and masked.
  uint32_t kw[kSub][2][KW], kp[kSub][2];
  auto load_keys = [&](const int64_t (&base)[kSub]) {
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int64_t at = base[u] < 0 ? 0 : base[u];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        load_words<4 * KW>(k_lane + at * kRow + 8 * e * kRow, kw[u][e]);
        kp[u][e] = __ldg(kp_lane + at + 8 * e);
      }
    }
  };

  int64_t base[kSub];
  int ti = t_begin + warp;
  if (ti < t_end) {
    place(range.tile(ti) * kTile, base);
    load_keys(base);
  }

  // ---- queries: one warp per row, brought to fp16 by a power of two, laid out as MMA fragments
  uint32_t* q_frag = reinterpret_cast<uint32_t*>(smem);       // [plane][k step][lane][2]
  for (int r = warp; r < R; r += kWarps) {
    float x[D / 32];
    uint32_t top = 0;                             // largest magnitude, by its bits: a NaN is above infinity
    float sum = 0.0f;
    const int rr = row0 + r;
    const bool real = r < rows_here;
    int member;
    const int token = p.by_group.divmod(rr, member);
    const T* src = static_cast<const T*>(p.q) + (int64_t)b * p.qb + (int64_t)token * p.qt +
                   (int64_t)(head * p.group + member) * p.qh;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      x[e] = real ? to_f32<T>(src[lane + 32 * e]) : 0.0f;
      top = max(top, __float_as_uint(fabsf(x[e])));
      sum += x[e];
    }
    for (int o = 16; o > 0; o >>= 1) {
      top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    // power of two that brings the largest element to [2^14, 2^15) (a subnormal one less far); in two
    // factors, for fp32's range
    const bool finite = top < 0x7f800000u;
    int e2 = 0;
    if (top > 0 && finite) e2 = 141 - (int)(top >> 23);
    const float f1 = __int_as_float((127 + e2 / 2) << 23), f2 = __int_as_float((127 + e2 - e2 / 2) << 23);
    if (lane == 0) {
      // score = a (s_k (q' . code') + m_k b) with q' the scaled query and code' = code * unit
      // (not a number for a query that is not finite: its scores may all be -inf, which stands for hidden)
      row_a[r] = (finite ? p.scale2 / kUnit : __int_as_float(0x7fc00000)) * __int_as_float((127 - e2 / 2) << 23) * __int_as_float((127 - (e2 - e2 / 2)) << 23);
      row_b[r] = sum * f1 * f2 * kUnit;
    }
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      const int ch = lane + 32 * e;
      // thread j of an MMA holds channels [j D/4, (j + 1) D/4): word w, nibble n of them
      const int tj = ch / (D / 4), w = ch % (D / 4) / 8, n = ch % 8;
      const int step = 2 * w + ((n >> 1) & 1), reg = n & 1, half_at = n >> 2;
      float v = x[e] * f1 * f2;
      if (n & 1) v *= 0.0625f;
      __half* dst = reinterpret_cast<__half*>(
          &q_frag[(step * 32 + r * 4 + tj) * 2 + reg]) + half_at;
      const __half hi = __float2half_rn(v);
      *dst = hi;
      if (P == 2) dst[(D / 16) * 32 * 2 * 2] = __float2half_rn(v - __half2float(hi));
    }
  }
  __syncthreads();

  float o[D / 16][4];
  float m_run[2];
  uint64_t l_run, s_run, ra, rb;   // pairs: query rows 2j and 2j + 1 of the eight
  int pos[2];
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  const int r = 2 * j;
  l_run = s_run = 0ull;
  ra = pack2(row_a[r], row_a[r + 1]);
  rb = pack2(row_b[r], row_b[r + 1]);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    m_run[e] = -INFINITY;
    pos[e] = length - p.count + (row0 + r + e) / p.group;
  }
  for (; ti < t_end; ti += kWarps) {
    const int t0 = range.tile(ti) * kTile;
    bool whole = true;
#pragma unroll
    for (int u = 0; u < kSub; ++u) whole &= base[u] >= 0;
    // does every row see every token?
    whole &= t0 + kTile <= length;
    if (p.causal) whole &= t0 + kTile <= pos_lo + 1;
    if (p.window > 0) whole &= t0 > pos_hi - p.window || t0 + kTile <= p.sinks;

    // ---- this tile's values are on their way while the scores are multiplied
    uint32_t vw[kAllValues ? kSub : 1][4][VW], vp[kSub][2];
    auto load_values = [&](int u) {
      const int64_t at = base[u] < 0 ? 0 : base[u];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        load_words<4 * VW>(v_lane + at * kRow + ((e & 1) + 8 * (e >> 1)) * kRow, vw[kAllValues ? u : 0][e]);
    };
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int64_t at = base[u] < 0 ? 0 : base[u];
#pragma unroll
      for (int e = 0; e < 2; ++e) vp[u][e] = __ldg(vp_lane + at + 8 * e);
      if (kAllValues) load_values(u);
    }

    // ---- scores, in units of 1 / a
    float s[kSub][4];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[u][e] = 0.0f;
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint2 qf[P];
#pragma unroll
        for (int pl = 0; pl < P; ++pl)
          qf[pl] = *reinterpret_cast<const uint2*>(
              &q_frag[((pl * (D / 16) + 2 * w + h) * 32 + lane) * 2]);
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          uint32_t e0, o0, e1, o1;
          if (h) {
            codes_upper<kCoarse>(kw[u][0][w], e0, o0);
            codes_upper<kCoarse>(kw[u][1][w], e1, o1);
          } else {
            codes_lower<kCoarse>(kw[u][0][w], e0, o0);
            codes_lower<kCoarse>(kw[u][1][w], e1, o1);
          }
#pragma unroll
          for (int pl = 0; pl < P; ++pl)
            mma_f16(s[u], e0, e1, o0, o1, qf[pl].x, qf[pl].y);
        }
      }
    float2 kf[kSub][2], vf[kSub][2];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        kf[u][e] = half_values(nan_unless_finite(kp[u][e]));
        vf[u][e] = half_values(vp[u][e]);
        if (!kCoarse) {                           // the minimum that belongs to n - 8
          kf[u][e].y = fmaf(8.0f, kf[u][e].x, kf[u][e].y);
          vf[u][e].y = fmaf(8.0f, vf[u][e].x, vf[u][e].y);
        }
        if (!whole && (base[u] < 0 || t0 + 16 * u + g + 8 * e >= length))   // not there: whatever was read
          kf[u][e] = vf[u][e] = make_float2(0.0f, 0.0f);
      }

    // ---- the next tile's keys
    int64_t here[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) here[u] = base[u];
    if (ti + kWarps < t_end) {
      place(range.tile(ti + kWarps) * kTile, base);
      load_keys(base);
    }

    // ---- softmax: scores in units of log2, reference = running maximum of score + exponent of s_v
    uint32_t pw[W][kSub][2];                  // weights times s_v, fp16 pairs
    float top[2] = {-INFINITY, -INFINITY};
    uint64_t x[kSub][2];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[u][e] = fma2(pack2(s[u][2 * e], s[u][2 * e + 1]), pack2(kf[u][e].x, kf[u][e].x),
                       mul2(pack2(kf[u][e].y, kf[u][e].y), rb));
        // 32 + the exponent field of the fp16 scale, as a float: its true exponent + 47 (less for subnormal
        // scales, which then only leave the weights some of their room)
        const float ev = __uint_as_float(((vp[u][e] << 8) & 0x007c0000u) | 0x42000000u);
        float2 r = unpack2(fma2(x[u][e], ra, pack2(ev, ev)));
        if (!whole) {
          const int t = t0 + 16 * u + g + 8 * e;
          const bool there = here[u] >= 0 && t < length;
          if (!(there && sees(p, t, pos[0]))) r.x = -INFINITY;
          if (!(there && sees(p, t, pos[1]))) r.y = -INFINITY;
        }
        top[0] = fmaxf(top[0], r.x);
        top[1] = fmaxf(top[1], r.y);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
      top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 16));
    }
    if (top[0] > m_run[0] || top[1] > m_run[1]) {
      float alpha[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const bool more = top[c] > m_run[c];
        alpha[c] = more ? exp2_fast(m_run[c] - top[c]) : 1.0f;      // 0 while nothing was seen
        m_run[c] = more ? top[c] : m_run[c];
      }
      const uint64_t a2 = pack2(alpha[0], alpha[1]);
      l_run = mul2(l_run, a2);
      s_run = mul2(s_run, a2);
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[i][0] *= alpha[0];
        o[i][1] *= alpha[1];
        o[i][2] *= alpha[0];
        o[i][3] *= alpha[1];
      }
    }
    const uint64_t ref = pack2(m_run[0] == -INFINITY ? 0.0f : kExponentBias - m_run[0],
                               m_run[1] == -INFINITY ? 0.0f : kExponentBias - m_run[1]);
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 a = unpack2(fma2(x[u][e], ra, ref));
        float2 w = make_float2(exp2_fast(a.x), exp2_fast(a.y));
        float vx = vf[u][e].x * 16384.0f, vx1 = vx, vy = vf[u][e].y, vy1 = vy;
        if (!whole) {
          // a hidden token's scale and minimum may be anything: its weight of 0 must not meet them
          const int t = t0 + 16 * u + g + 8 * e;
          const bool there = here[u] >= 0 && t < length;
          if (!(there && sees(p, t, pos[0]))) { w.x = 0.0f; vx = vy = 0.0f; }
          if (!(there && sees(p, t, pos[1]))) { w.y = 0.0f; vx1 = vy1 = 0.0f; }
        }
        const uint64_t w2 = pack2(w.x, w.y);
        l_run = add2(l_run, w2);
        s_run = fma2(w2, pack2(vy, vy1), s_run);
        const float2 q = unpack2(mul2(w2, pack2(vx, vx1)));
        const uint32_t h = half_pair(q.x, q.y);
        pw[0][u][e] = h;
        if (W == 2) {
          const float2 f = half_values(h);
          pw[W - 1][u][e] = half_pair(q.x - f.x, q.y - f.y);
        }
      }

    // ---- output
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      if (!kAllValues) {
        const int64_t at = here[u] < 0 ? 0 : here[u];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          load_words<4 * VW>(v_lane + at * kRow + ((e & 1) + 8 * (e >> 1)) * kRow, vw[0][e]);
      }
      const auto& vu = vw[kAllValues ? u : 0];
      uint32_t b0[W], b1[W];
#pragma unroll
      for (int pl = 0; pl < W; ++pl) {
        b0[pl] = transpose8(pw[pl][u][0]);
        b1[pl] = transpose8(pw[pl][u][1]);
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t z0 = __byte_perm(vu[0][w], vu[1][w], h ? 0x7632 : 0x5410);
          const uint32_t z1 = __byte_perm(vu[2][w], vu[3][w], h ? 0x7632 : 0x5410);
#pragma unroll
          for (int h2 = 0; h2 < 2; ++h2) {
            uint32_t e0, o0, e1, o1;
            if (h2) {
              codes_upper<kCoarse>(z0, e0, o0);
              codes_upper<kCoarse>(z1, e1, o1);
            } else {
              codes_lower<kCoarse>(z0, e0, o0);
              codes_lower<kCoarse>(z1, e1, o1);
            }
            float(&acc)[4] = o[4 * w + 2 * h + h2];
            if constexpr (sizeof(T) == 4) {
              // The tensor cores cut off what they add: over thousands of tokens that is 1e-5 of the sum, so
              // sixteen tokens' products are added to the others by rounding additions.
              float part[4] = {};
#pragma unroll
              for (int pl = 0; pl < W; ++pl) mma_f16(part, e0, o0, e1, o1, b0[pl], b1[pl]);
              const float2 lo = unpack2(add2(pack2(acc[0], acc[1]), pack2(part[0], part[1])));
              const float2 hi = unpack2(add2(pack2(acc[2], acc[3]), pack2(part[2], part[3])));
              acc[0] = lo.x; acc[1] = lo.y; acc[2] = hi.x; acc[3] = hi.y;
            } else {
#pragma unroll
              for (int pl = 0; pl < W; ++pl) mma_f16(acc, e0, o0, e1, o1, b0[pl], b1[pl]);
            }
          }
        }
    }
  }

  // ---- the warps' results joined: numerators in units of 2^m
#pragma unroll
  for (int sh = 4; sh < 32; sh <<= 1) {
    l_run = add2(l_run, __shfl_xor_sync(0xffffffffu, l_run, sh));
    s_run = add2(s_run, __shfl_xor_sync(0xffffffffu, s_run, sh));
  }
  if (g == 0) {
    const int r = 2 * j;
    const float2 l = unpack2(l_run), sm = unpack2(s_run);
    join_m[warp][r] = m_run[0];
    join_m[warp][r + 1] = m_run[1];
    join_l[warp][r] = l.x;
    join_l[warp][r + 1] = l.y;
    join_s[warp][r] = sm.x;
    join_s[warp][r + 1] = sm.y;
  }
  __syncthreads();                                            // also: the query fragments are read
  float* o_sh = reinterpret_cast<float*>(smem);               // [warp][row][D + 4]
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float* dst = o_sh + (size_t)(warp * R + 2 * j + c) * (D + 4) + g * (D / 8) + 2 * i;
      dst[0] = o[i][c] * (0x1p-14f / kUnit);
      dst[1] = o[i][2 + c] * (0x1p-18f / kUnit);        // codes of odd channels stood for 16 n
    }
  __syncthreads();
  for (int idx = threadIdx.x; idx < rows_here * (D / 4); idx += kThreads) {
    const int r = idx / (D / 4), c4 = idx % (D / 4) * 4;
    float m = join_m[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, join_m[w][r]);
    float l = 0.0f, acc[4] = {};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = join_m[w][r] == -INFINITY ? 0.0f : exp2_fast(join_m[w][r] - m);
      const float4 v = *reinterpret_cast<const float4*>(o_sh + (size_t)(w * R + r) * (D + 4) + c4);
      const float ms = join_s[w][r];
      l = fmaf(f, join_l[w][r], l);
      acc[0] = fmaf(f, v.x + ms, acc[0]);
      acc[1] = fmaf(f, v.y + ms, acc[1]);
      acc[2] = fmaf(f, v.z + ms, acc[2]);
      acc[3] = fmaf(f, v.w + ms, acc[3]);
    }
    const int rr = row0 + r;
    const int64_t out_row = ((int64_t)b * p.count + rr / p.group) * p.heads + head * p.group + rr % p.group;
    if (p.splits == 1) {
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;          // a row that sees nothing is 0
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= inv;
      store_f32<T, 4>(static_cast<T*>(p.out) + out_row * D + c4, acc);
    } else {
      const int64_t at = split * p.rows + out_row;
      store_f32<float, 4>(p.part + at * D + c4, acc);
      if (c4 == 0) {
        float* lm = p.part + (int64_t)p.splits * p.rows * D;
        lm[at] = l;
        lm[(int64_t)p.splits * p.rows + at] = m;
      }
    }
  }
}

// The splits' partial results of one row joined: weights first, then the numerators, four channels a
// thread, the splits dealt out to kGroups groups of threads whose sums are added in order.
constexpr int kJoinThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads)
kv4_join_kernel(const float* __restrict__ part, T* __restrict__ out, int64_t rows, int splits) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float weight[kMaxSplits];
  __shared__ float sh[32];
  __shared__ float4 acc_sh[kGroups][kLanes];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = blockIdx.x;
  const float* l_at = part + (int64_t)splits * rows * D + row;
  const float* m_at = l_at + (int64_t)splits * rows;
  float m = -INFINITY, ms = -INFINITY, l = 0.0f;
  if (threadIdx.x < splits) {                          // splits <= kJoinThreads
    m = ms = m_at[threadIdx.x * rows];
    l = l_at[threadIdx.x * rows];
  }
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kJoinThreads / 32; ++i) m = fmaxf(m, sh[i]);
  // a part without a maximum saw nothing, or only scores that are not numbers: its sum says which
  const float f = ms == -INFINITY ? 0.0f : exp2_fast(ms - m);
  if (threadIdx.x < splits) weight[threadIdx.x] = f;
  l = ms == -INFINITY ? l : f * l;
  l = block_sum(l, sh);                                // a barrier inside: the weights are there
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (group < kGroups) {
#pragma unroll 4
    for (int s = group; s < splits; s += kGroups) {
      const float w = weight[s];
      const float4 v = *reinterpret_cast<const float4*>(part + (s * rows + row) * D + 4 * lane);
      acc.x = fmaf(w, v.x, acc.x);
      acc.y = fmaf(w, v.y, acc.y);
      acc.z = fmaf(w, v.z, acc.z);
      acc.w = fmaf(w, v.w, acc.w);
    }
    acc_sh[group][lane] = acc;
  }
  __syncthreads();
  if (threadIdx.x < kLanes) {
    float v[4] = {};
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const float4 a = acc_sh[i][threadIdx.x];
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= inv;
    store_f32<T, 4>(out + row * D + 4 * threadIdx.x, v);
  }
}

// Parts of the tokens of one sequence and key head: one round of blocks over all SMs if there are few of
// them, else two, so that sequences of other lengths even out (64 sequences of up to 8192 tokens, us for 1 : 2 :
// 3 : 4 rounds, 117 : 113 : 116 : 120; 200 of 2000 88 : 87 : 109 : 108), but one of the many-row kernel, whose
// blocks take 8 us to begin and end (32 sequences of 1000 tokens, 24 rows, 43 : 67).  Every part at least `least`
// tokens: a tile for every warp (2000 tokens of 8 heads, 128 : 512 tokens a part, 7.4 : 10.4; 131072 of 4 heads
// 27.2 : 27.2), two tiles of the many-row kernel (100 queries, 4000 tokens, 256 : 1024, 33 : 49); fewer than four
// parts are not worth the second launch (200 tokens 7.2 split, 6.9 not).  The lengths are on the device, so the
// table's width stands for the longest.
int splits_for(int64_t units, int max_tokens, bool many) {
  const int64_t slots = (int64_t)(many ? 1 : kBlocksPerSm) * device_sms();
  const int least = many ? 256 : kTile * kWarps;
  const int64_t want = many || 2 * units <= slots ? slots / units : ceil_div64(2 * slots, units);
  const int64_t most = max_tokens < 4 * least ? 1 : max_tokens / least;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : (s > kMaxSplits ? kMaxSplits : s));
}

struct Plan {
  int row_tiles, splits;
  bool tc;                              // the tensor-core kernel for many rows
  int64_t blocks;
};
Plan plan_of(const modiff_kv4_cache* c, int batch, int count, int heads, int max_pages, int window, int sinks,
             int dtype) {
  Plan pl;
  const int rows = count * (heads / c->heads);
  pl.tc = kv4_tc_wanted(rows, c->dim, dtype);
  const int tile = pl.tc ? kv4_tc_rows() : kQueries;
  pl.row_tiles = ceil_div(rows, tile);
  const int64_t units = (int64_t)batch * c->heads * pl.row_tiles;
  int64_t tokens = (int64_t)max_pages * c->page_size;
  if (window > 0 && (int64_t)window + sinks + tile < tokens) tokens = (int64_t)window + sinks + tile;
  pl.splits = splits_for(units, (int)tokens, pl.tc);
  pl.blocks = units * pl.splits;
  return pl;
}

template <typename T, int D>
int join(const Kv4Attention& p, cudaStream_t s) {
  if (p.splits == 1) return MODIFF_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.rows);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MODIFF_CUDA(cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, D>, (const float*)p.part, static_cast<T*>(p.out), p.rows,
                                 p.splits));
  return MODIFF_OK;
}

template <typename T, int D>
int launch_attention(const Kv4Attention& p, int64_t blocks, cudaStream_t s) {
  constexpr int smem = smem_bytes<T, D>();
  static SmemLimit limit;
  MODIFF_CUDA(raise_smem_limit(kv4_attention_kernel<T, D>, smem, limit));
  kv4_attention_kernel<T, D><<<(unsigned)blocks, kThreads, smem, s>>>(p);
  MODIFF_LAUNCH_CHECK("kv4_attention_kernel");
  return join<T, D>(p, s);
}

template <typename T, int D>
int by_rows(const Kv4Attention& p, const Plan& pl, int dtype, cudaStream_t s) {
  if (pl.tc) {
    const int rc = kv4_launch_tc(p, dtype, s);
    return rc ? rc : join<T, D>(p, s);
  }
  return launch_attention<T, D>(p, pl.blocks, s);
}

int check_shape(const modiff_kv4_cache* c, int batch, int count, int heads) {
  MODIFF_CHECK_ARG(batch >= 0 && count >= 0 && heads > 0, "bad shape");
  MODIFF_CHECK_ARG(heads % c->heads == 0, "%d query heads for %d key heads", heads, c->heads);
  MODIFF_CHECK_ARG((int64_t)count * heads <= 0x3fffffff, "too many query rows");
  return MODIFF_OK;
}

}  // namespace
}  // namespace modiff

using namespace modiff;

extern "C" int64_t modiff_kv4_attention_bytes(const modiff_kv4_cache* cache, int batch, int count, int heads,
                                              int max_pages, int window, int sinks, int dtype) {
  if (!cache || !dtype_ok(dtype) || cache->heads <= 0 || batch <= 0 || count <= 0 || check_shape(cache, batch, count, heads)) return 0;
  const Plan pl = plan_of(cache, batch, count, heads, max_pages, window, sinks, dtype);
  if (pl.splits == 1) return 0;
  return 4ll * pl.splits * batch * count * heads * (cache->dim + 2);
}

extern "C" int modiff_kv4_attention(const void* q, int64_t q_seq, int64_t q_token, int64_t q_head,
                                    const modiff_kv4_cache* cache, const int32_t* table, const int32_t* lengths, void* out, int batch, int count,
                                    int heads, int max_pages, float scale, int causal, int window, int sinks,
                                    int dtype, void* workspace, void* stream) {
  int rc = kv4_check(cache, table, lengths, batch, max_pages);
  if (rc) return rc;
  rc = check_shape(cache, batch, count, heads);
  if (rc) return rc;
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(window >= 0 && sinks >= 0, "negative window or sinks");
  MODIFF_CHECK_ARG(causal || window == 0, "a window needs causal positions");
  if (batch == 0 || count == 0) return MODIFF_OK;
  MODIFF_CHECK_ARG(q && out, "NULL pointer argument");
  const int size = dtype_bytes(dtype);
  MODIFF_CHECK_ARG((uintptr_t)q % size == 0 && (uintptr_t)out % 16 == 0, "misaligned tensor");
  const Plan pl = plan_of(cache, batch, count, heads, max_pages, window, sinks, dtype);
  MODIFF_CHECK_ARG(pl.blocks <= 0x7fffffff, "too many query rows");
  MODIFF_CHECK_ARG(pl.splits == 1 || (workspace && (uintptr_t)workspace % 16 == 0), "NULL or misaligned workspace");
  Kv4Attention p;
  p.q = q;
  p.qb = q_seq; p.qt = q_token; p.qh = q_head;
  p.q_vec = (((uintptr_t)q | (uintptr_t)((q_seq | q_token | q_head) * size)) & 15) == 0;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.c = kv4_pages(cache);
  p.table = table; p.lengths = lengths;
  p.batch = batch; p.count = count; p.heads = heads; p.group = heads / cache->heads;
  p.by_group = FastDiv(p.group);
  p.max_pages = max_pages;
  p.splits = pl.splits; p.row_tiles = pl.row_tiles;
  // positions and windows are subtracted in 32 bits; none of the cache's tokens is 2^30 back
  constexpr int kFar = 1 << 30;
  p.causal = causal;
  p.window = window < kFar ? window : kFar;
  p.sinks = sinks < kFar ? sinks : kFar;
  p.scale2 = scale * kLog2e;
  p.rows = (int64_t)batch * count * heads;
  cudaStream_t st = (cudaStream_t)stream;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    switch (cache->dim) {
      case 64: return by_rows<T, 64>(p, pl, dtype, st);
      case 128: return by_rows<T, 128>(p, pl, dtype, st);
      case 192: return by_rows<T, 192>(p, pl, dtype, st);
      default: return by_rows<T, 256>(p, pl, dtype, st);
    }
  });
}
