// Attention over the 4-bit cache for many query rows per key head (prompts and pieces of them), on the
// 5th-generation tensor cores.  fp16 and bf16 tensors; fp16 results are as exact as those of kv4_attention.cu.
//
// A block owns 256 query rows (query, head of the group) of one sequence and key head, as two groups of
// 128, and walks the keys in tiles of 128 that both groups share:
//   four warps each read the codes of keys and of values through the page table and write them as fp16 operands of
//   an MMA (128-byte swizzle; a key's channels stay in its row, which is K-major for the scores and N-major for the
//   output; eight channels of a word lie in the order 0 4 1 5 2 6 3 7, in which they come out of it, and so do the
//   queries');
//   one warp issues S = Q K^T into tensor memory (128 columns a group) and O += P V, with P read from
//   tensor memory, where the softmax has put it in place of S;
//   four softmax warps a group, a thread per row, no exchange between threads: maximum, then weights.
//   O is rescaled only when a row's maximum has grown by more than 2^10.
// While one group's softmax runs the tensor pipe works for the other.
//
// What the operands are:
//   bf16 calls  s code + m, rounded to fp16 once (2^-11 of it at most), for keys and values; weights in fp16, in units
//               of 2^(reference - 5), at most 2^15.  So a score is off by up to scale 2^-11 sum |q k|, one weight by
//               2^-11.  Beside the rounding of bf16 outputs (1.66e-3 of them in the mean) that is little while scores
//               are not large: 1.77e-3 in all on the case below.
//   fp16 calls  codes as the exact numbers n - 8, scales and minima outside the products (kExact):
//                 score = s (q . (n - 8)) + (m + 8 s) sum(q),  sum_t p v = sum_t (p s) (n - 8) + sum_t p (m + 8 s),
//               p s as two fp16 numbers (22 bits) relative to the largest score + exponent of s.  Half as many products
//               again and twice the softmax's instructions: 423 us where bf16 takes 257, for errors of the output's
//               own rounding (2.1e-4); with bf16's operands they were 4e-4 to 8.6e-4, and 2.6e-3 where scores reach 60.
//
// Queries are brought to fp16 by a power of two per row (exact).  A key whose scale or minimum is not finite is
// NaN, and so are its scores; such a value is replaced by zero and makes the rows that see it NaN, so that rows
// that do not see it never meet it.
//
// Bound (bf16): tensor pipe and exponentials alike, 2048 cycles a tile of 128 keys and 256 rows of 128 channels.  4
// pieces of 1000 queries over up to 8000 tokens, window 2048, 32 / 8 heads of 128, bf16: 255 us, of which 34 are
// the blocks' beginnings and ends, 32 the steps with hidden keys; without exponentials, maxima and dequantisation
// it would be 178: what is left are the roles' waits for each other.  What it took: one group of warps for loading
// and weighing 447, loaders of their own 310, half tiles of 64 keys with the next scores multiplied meanwhile 299,
// queries laid out in 16-byte chunks 274, masks out of the steps that need none 264, by bit 255.  Not better:
// exponentials before the maximum is known (278), scores fetched a step ahead by four loader warps (323), one
// straight copy of the step for each kind of mask (281, spills).
#include <type_traits>

#include "kv4.cuh"
#include "tc_common.cuh"

namespace modiff {

int read_device_status_kv4(int* status, int reset) { return read_status_this_unit(status, reset); }

namespace {

constexpr int kKeys = 128;                  // keys of a tile
constexpr int kHalf = 64;                   // keys of one softmax step
constexpr int kRows = 256;                  // query rows of a block
constexpr int kLoaders = 4;                 // warps 0 .. 3 keys, 4 .. 7 values; softmax 8 .. 15; MMAs 16
constexpr int kSoftmaxWarp = 8, kMmaWarp = 16;
constexpr int kThreads = 32 * 20;           // the last three warps only complete the MMA warp's group
// Registers: 96 a thread at launch, dealt out anew by group of four warps.
constexpr int kRegsAtLaunch = 96, kRegsMma = 56;
template <bool EXACT> constexpr int kRegsLoad = EXACT ? 64 : 72;
template <bool EXACT> constexpr int kRegsSoftmax = EXACT ? 144 : 136;
static_assert(5 * kRegsAtLaunch >= 2 * kRegsLoad<false> + 2 * kRegsSoftmax<false> + kRegsMma &&
                  5 * kRegsAtLaunch >= 2 * kRegsLoad<true> + 2 * kRegsSoftmax<true> + kRegsMma, "register split");
constexpr int kChunk = kKeys * 128;         // bytes of 128 rows of 64 channels
constexpr float kGrowth = 10.0f;            // of a row's maximum, in powers of two, before O is rescaled
// Weights (times the scale of their value, in fp16 calls) are at most 2^15, kGrowth included.
template <bool EXACT> constexpr float kRoom = EXACT ? 4.0f : 5.0f;
constexpr int kBitSlots = 4;

// fp16 x fp16 -> fp32; descriptors as low words and the high word they share.  A from shared or tensor memory.
__device__ inline void tc_mma_f16_lo(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                     uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ inline void tc_mma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                     uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ inline void tc_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
// Instruction descriptor of kind::f16 with fp16 operands and fp32 accumulation; B K-major or N-major.
__host__ __device__ inline uint32_t make_idesc_f16(int m, int n, bool b_n_major) {
  return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Operand whose rows of 128 bytes are steps of K (N-major): 64-element pieces of N `kChunk` apart, groups of
// eight rows 1024 bytes apart.
__device__ inline uint64_t make_n_major_desc(uint32_t saddr) {
  uint64_t d = make_smem_desc(saddr);
  d &= ~((uint64_t)0x3fff << 16);
  d |= (uint64_t)(kChunk >> 4) << 16;
  return d;
}

__device__ inline __half2 as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ inline uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }

// One word of eight codes as fp16 values s code + m.  1024 + n is the fp16 number 0x6400 | n, and 1024 + 16 n
// that of the other half of a byte; taking 1024 (and the factor) out again is exact.
template <bool CLAMP>
__device__ inline uint4 dequantise(uint32_t w, __half2 s, __half2 m) {
  const __half2 k1024 = as_half2(0x64006400u), k16th = as_half2(0x2c002c00u), k64 = as_half2(0xd400d400u);   // 1024, 1/16, -64
  __half2 v[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = i ? w >> 8 : w;
    v[2 * i] = __hfma2(__hsub2(as_half2((x & 0x000f000fu) | 0x64006400u), k1024), s, m);
    v[2 * i + 1] = __hfma2(__hfma2(as_half2((x & 0x00f000f0u) | 0x64006400u), k16th, k64), s, m);
  }
  if (CLAMP) {
    // s rounded up can carry the largest code past fp16's range
    const __half2 top = as_half2(0x7bff7bffu), low = as_half2(0xfbfffbffu);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmin2(__hmax2(v[i], low), top);
  }
  return make_uint4(as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3]));
}

// One word of eight codes as the numbers n - 8.
__device__ inline uint4 centred(uint32_t w) {
  const __half2 k1032 = as_half2(0x64086408u), k16th = as_half2(0x2c002c00u), k72 = as_half2(0xd480d480u);   // 1032, 1/16, -72
  __half2 v[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t x = i ? w >> 8 : w;
    v[2 * i] = __hsub2(as_half2((x & 0x000f000fu) | 0x64006400u), k1032);
    v[2 * i + 1] = __hfma2(as_half2((x & 0x00f000f0u) | 0x64006400u), k16th, k72);
  }
  return make_uint4(as_u32(v[0]), as_u32(v[1]), as_u32(v[2]), as_u32(v[3]));
}

// A row of codes into its place of an operand tile.
template <int D, bool EXACT>
__device__ inline void store_row(uint8_t* tile, int row, const uint32_t (&w)[D / 8], uint32_t params, bool there) {
  const __half2 sm = as_half2(params);
  const __half2 s = __low2half2(sm), m = __high2half2(sm);
  const float2 f = half_values(params);
  const bool edge = fabsf(f.y) > 65000.0f || fabsf(fmaf(15.0f, f.x, f.y)) > 65000.0f;
  uint8_t* base = tile + row * 128;
  auto place = [&](int i) { return reinterpret_cast<uint4*>(base + (i >> 3) * kChunk + (((i & 7) ^ (row & 7)) << 4)); };
  if (EXACT) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *place(i) = centred(w[i]);
  } else if (!there) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *place(i) = make_uint4(0u, 0u, 0u, 0u);
  } else if (edge) {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *place(i) = dequantise<true>(w[i], s, m);
  } else {
#pragma unroll
    for (int i = 0; i < D / 8; ++i) *place(i) = dequantise<false>(w[i], s, m);
  }
}

// the largest of three; a NaN is passed over
__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ inline void tc_ld16(uint32_t taddr, int (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}

// low bits [0, n) of a word, n clamped to 0 .. 32
__device__ inline uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u); }

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
kv4_attention_tc_kernel(const Kv4Attention p) {
  constexpr int kQTile = 128 * D * 2, kKvTile = kKeys * D * 2;
  constexpr bool kExact = std::is_same_v<T, __half>;
  extern __shared__ __align__(1024) uint8_t smem[];          // Q [2], K [2], V [2]
  __shared__ __align__(8) uint64_t bar_k_full[2], bar_k_empty[2], bar_v_full[2], bar_v_empty[2];
  __shared__ __align__(8) uint64_t bar_s_full[2][2], bar_p_ready[2][2], bar_pv[2][2], bar_bits[kBitSlots];   // [group][half]
  __shared__ __align__(16) uint32_t there_sh[kBitSlots][4], bad_sh[kBitSlots][4];   // tokens that exist; values that are not finite
  // kExact: of a tile's keys the scale and minimum, of its values the scale's exponent, scale and minimum
  __shared__ __align__(16) float factor_sh[kExact ? kBitSlots : 1][5][kExact ? kKeys : 4];
  __shared__ float row_a[kRows], row_b[kExact ? kRows : 1];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_sh;
  uint8_t* q_sh = smem;
  uint8_t* k_sh = smem + 2 * kQTile;
  uint8_t* v_sh = k_sh + 2 * kKvTile;

  if (p.splits > 1) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int id = blockIdx.x;
  const int split = id % p.splits;
  id /= p.splits;
  // the last rows of a causal call have the most keys: they start first
  const int rt = p.row_tiles - 1 - id % p.row_tiles;
  id /= p.row_tiles;
  const int head = id % p.c.heads, b = id / p.c.heads;
  const int row0 = rt * kRows;
  const int rows_here = min(kRows, p.count * p.group - row0);
  const bool two = rows_here > 128;
  const int32_t* table = p.table + (int64_t)b * p.max_pages;
  const int length = min(max(__ldg(p.lengths + b), 0), p.max_pages * p.c.page_size);
  const int pos_lo = length - p.count + row0 / p.group;
  const int pos_hi = length - p.count + (row0 + rows_here - 1) / p.group;
  const TileRange range = tiles_of<kKeys>(p, length, pos_lo, pos_hi);
  const int t_begin = (int)((int64_t)range.count * split / p.splits);
  const int tiles = (int)((int64_t)range.count * (split + 1) / p.splits) - t_begin;

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_k_full[i]), kLoaders);
      mbar_init(smem_u32(&bar_k_empty[i]), 1);
      mbar_init(smem_u32(&bar_v_full[i]), kLoaders);
      mbar_init(smem_u32(&bar_v_empty[i]), 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_u32(&bar_s_full[i][h]), 1);
        mbar_init(smem_u32(&bar_p_ready[i][h]), 4);
        mbar_init(smem_u32(&bar_pv[i][h]), 1);
      }
    }
    for (int i = 0; i < kBitSlots; ++i) mbar_init(smem_u32(&bar_bits[i]), kExact ? 2 * kLoaders : kLoaders);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // ---- queries: D / 8 lanes a row, eight channels (a chunk of the operand) each; a warp's loads are all on
  // their way before the first is looked at
  const float sign = p.scale2 < 0.0f ? -1.0f : 1.0f;           // the scale's sign goes into the queries
  constexpr int kLanes = D / 8, kPass = kThreads / kLanes, kBatch = (kRows + kPass - 1) / kPass;
  const int q_row = threadIdx.x / kLanes, chunk = threadIdx.x % kLanes;
  Pack<T, 8> raw[kBatch];
  const T* q_lane = static_cast<const T*>(p.q) + (int64_t)b * p.qb + (int64_t)(head * p.group) * p.qh + 8 * chunk;
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int r = q_row + u * kPass;
    if (r < rows_here) {
      int member;
      const int token = p.by_group.divmod(row0 + r, member);
      const T* src = q_lane + token * p.qt + member * p.qh;
      if (p.q_vec) {
        raw[u] = *reinterpret_cast<const Pack<T, 8>*>(src);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[u].v[e] = src[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) raw[u].v[e] = from_f32<T>(0.0f);
    }
  }
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int r = q_row + u * kPass;
    float x[8];
    uint32_t top = 0;                             // largest magnitude, by its bits: a NaN is above infinity
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = to_f32<T>(raw[u].v[e]);
      top = max(top, __float_as_uint(fabsf(x[e])));
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    // power of two that brings the largest element to [2^14, 2^15) (a subnormal one less far); in two
    // factors, for bf16's range
    const bool finite = top < 0x7f800000u;
    int e2 = 0;
    if (top > 0 && finite) e2 = 141 - (int)(top >> 23);
    const float f1 = sign * __int_as_float((127 + e2 / 2) << 23), f2 = __int_as_float((127 + e2 - e2 / 2) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * f1 * f2;
    float sum = 0.0f;
    if constexpr (kExact) {
      sum = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (r < kRows) {
      if (kExact && chunk == 0) row_b[kExact ? r : 0] = sum;
      // divided by both (powers of two, exactly); not a number for a query that is not finite: its scores may all
      // be -inf, which stands for hidden
      if (chunk == 0)
        row_a[r] = (finite ? fabsf(p.scale2) : __int_as_float(0x7fc00000)) * __int_as_float((127 - e2 / 2) << 23) * __int_as_float((127 - (e2 - e2 / 2)) << 23);
      *reinterpret_cast<uint4*>(q_sh + (r >> 7) * kQTile + (chunk >> 3) * kChunk + (r & 127) * 128 +
                                (((chunk & 7) ^ (r & 7)) << 4)) =
          make_uint4(half_pair(x[0], x[4]), half_pair(x[1], x[5]), half_pair(x[2], x[6]), half_pair(x[3], x[7]));
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;

  if (warp < kSoftmaxWarp) {
    // ------------------------------------------------------------ keys (warps 0 .. 3), values (4 .. 7)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad<kExact>));
    const bool value = warp >= kLoaders;
    const int key = threadIdx.x & 127;
    const uint8_t* codes = value ? p.c.v_codes : p.c.k_codes;
    const uint32_t* params = reinterpret_cast<const uint32_t*>(value ? p.c.v_params : p.c.k_params);
    uint8_t* stages = value ? v_sh : k_sh;
    const uint32_t empty0 = smem_u32(value ? &bar_v_empty[0] : &bar_k_empty[0]);
    const uint32_t full0 = smem_u32(value ? &bar_v_full[0] : &bar_k_full[0]);
    uint32_t w[D / 8], sm = 0;
    int64_t place = -1;
    auto load = [&](int i) {
      const int t = range.tile(t_begin + i) * kKeys + key;
      place = t < length ? kv4_place(p.c, table, p.max_pages, t, head) : -1;
      const int64_t a = place < 0 ? 0 : place;                 // what is not there is read from the beginning
      load_words<D / 2>(codes + a * (D / 2), w);
      sm = __ldg(params + a);
    };
    if (tiles > 0) load(0);
    for (int i = 0; i < tiles; ++i) {
      const int st = i & 1, slot = i % kBitSlots;
      if (!mbar_wait(empty0 + 8 * st, ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag)) break;
      bool there = place >= 0;
      // exponent field of all ones: infinity or NaN
      const bool bad = there && ((sm & 0x7c00u) == 0x7c00u || (sm & 0x7c000000u) == 0x7c000000u);
      if (!value && bad) sm = 0x7fff7fffu;                     // its scores are NaN, not what an infinity clamps to
      if (value) {
        const uint32_t there_bits = __ballot_sync(0xffffffffu, there), bad_bits = __ballot_sync(0xffffffffu, bad);
        if (lane == 0) {
          there_sh[slot][warp - kLoaders] = there_bits;
          bad_sh[slot][warp - kLoaders] = bad_bits;
        }
        there = there && !bad;
      }
      if constexpr (kExact) {
        // what n - 8 stands for is scale (n - 8) + (minimum + 8 scale)
        const float2 f = there ? half_values(sm) : make_float2(0.0f, 0.0f);
        float* to = &factor_sh[slot][value ? 3 : 0][key];
        to[0] = f.x;
        to[kKeys] = fmaf(8.0f, f.x, f.y);
        if (value) to[-kKeys] = (float)((int)((sm >> 10) & 31u) - 15);   // f.x is below 2^(that + 1)
      }
      if (value || kExact) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_bits[slot]));
      }
      store_row<D, kExact>(stages + st * kKvTile, key, w, sm, there);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(full0 + 8 * st);
      if (i + 1 < tiles) load(i + 1);
    }
    __syncwarp();
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMAs
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsMma));
    if (warp == kMmaWarp) {
      // This warp's instructions are the critical path (about five cycles each beside the other warps): the
      // descriptors' low words are added to 32-bit constants, waits that come together are one.
      const uint32_t idesc_s = make_idesc_f16(128, kHalf, false), idesc_o = make_idesc_f16(128, D, true);
      const uint32_t q_lo = (uint32_t)make_smem_desc(smem_u32(q_sh)), desc_hi = (uint32_t)(make_smem_desc(0) >> 32);
      const uint32_t k_lo = (uint32_t)make_smem_desc(smem_u32(k_sh)), v_lo = (uint32_t)make_n_major_desc(smem_u32(v_sh));
      // every lane its own barrier and parity, until all have seen theirs
      auto wait_all = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
      };
      // scores of half h of the keys in stage st, into the group's buffer of that half
      auto scores = [&](int g, int h, int st) {
        const uint32_t a = q_lo + (uint32_t)(g * (kQTile >> 4)), kd = k_lo + (uint32_t)(st * (kKvTile >> 4) + h * (kHalf * 128 >> 4));
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tc_mma_f16_lo(tmem_base + (uint32_t)(128 * g + kHalf * h), a + (uint32_t)(c * (kChunk >> 4) + 2 * k),
                          kd + (uint32_t)(c * (kChunk >> 4) + 2 * k), desc_hi, idesc_s, c > 0 || k > 0 ? 1u : 0u);
        tc_commit(smem_u32(&bar_s_full[g][h]));
      };
      auto products = [&](int g, int h, int st, uint32_t accumulate) {
        const uint32_t vd = v_lo + (uint32_t)(st * (kKvTile >> 4) + h * (kHalf * 128 >> 4));
#pragma unroll
        for (int k = 0; k < (kExact ? 2 : 1) * kHalf / 16; ++k)
          tc_mma_f16_ta(tmem_base + (uint32_t)(256 + 128 * g), tmem_base + (uint32_t)(128 * g + kHalf * h + 8 * k),
                        vd + (uint32_t)(k % (kHalf / 16) * (16 * 128 >> 4)), desc_hi, idesc_o, k > 0 ? 1u : accumulate);
        tc_commit(smem_u32(&bar_pv[g][h]));
      };
      const uint32_t k_full0 = smem_u32(&bar_k_full[0]), v_full0 = smem_u32(&bar_v_full[0]);
      bool ok = tiles > 0 && wait_all(k_full0, 0);
      if (ok) {
        tc_fence_after();
        if (elect_one()) {
          scores(0, 0, 0);
          if (two) scores(1, 0, 0);
          scores(0, 1, 0);
          if (two) scores(1, 1, 0);
          tc_commit(smem_u32(&bar_k_empty[0]));
        }
        __syncwarp();
      }
      for (int i = 0; i < tiles && ok; ++i) {
        const int st = i & 1;
        const bool more = i + 1 < tiles;
#pragma unroll
        for (int hg = 0; hg < 4; ++hg) {
          const int h = hg >> 1, g = hg & 1;
          if (!ok || (g == 1 && !two)) continue;
          uint32_t bar = smem_u32(&bar_p_ready[g][h]), parity = (uint32_t)i & 1u;
          if (hg == 0) {
            if (lane & 1) { bar = v_full0 + 8 * st; parity = (uint32_t)(i >> 1) & 1u; }
            if (more && (lane & 2)) { bar = k_full0 + 8 * (st ^ 1); parity = (uint32_t)((i + 1) >> 1) & 1u; }
          }
          ok = wait_all(bar, parity);
          if (!ok) continue;
          tc_fence_after();
          if (elect_one()) {
            products(g, h, st, i > 0 || h > 0 ? 1u : 0u);
            if (more) scores(g, h, st ^ 1);
            if (h == 1 && (g == 1 || !two)) {
              tc_commit(smem_u32(&bar_v_empty[st]));
              if (more) tc_commit(smem_u32(&bar_k_empty[st ^ 1]));
            }
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax, output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax<kExact>));
    const int g = (warp - kSoftmaxWarp) >> 2, quarter = warp & 3;
    const int r = 128 * g + 32 * quarter + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t t_s = t_lane + (uint32_t)(128 * g), t_o = t_lane + (uint32_t)(256 + 128 * g);
    if (g == 0 || two) {
      const float ra = row_a[r];
      const uint64_t ra2 = pack2(ra, ra);
      const float rb = kExact ? row_b[kExact ? r : 0] : 0.0f;
      const uint64_t rb2 = pack2(rb, rb);
      const int pos = length - p.count + (row0 + r) / p.group;
      float m_ref = -INFINITY;                                 // the row's reference, in units of log2
      uint64_t l2 = 0ull, s2 = 0ull;                           // sums of even and odd columns; kExact: of weights times minima
      bool ok = true, poisoned = false;
      for (int step = 0; step < 2 * tiles; ++step) {
        const int i = step >> 1, h = step & 1, slot = i % kBitSlots;
        const int t0 = range.tile(t_begin + i) * kKeys + kHalf * h;
        ok = mbar_wait(smem_u32(&bar_s_full[g][h]), (uint32_t)i & 1u, abort_flag) &&
             (h == 1 || mbar_wait(smem_u32(&bar_bits[slot]), (uint32_t)(i / kBitSlots) & 1u, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const uint32_t t_sh = t_s + (uint32_t)(kHalf * h);
        int v[kHalf];
        tc_ld32(t_sh, reinterpret_cast<int(&)[32]>(v[0]));
        tc_ld32(t_sh + 32, reinterpret_cast<int(&)[32]>(v[32]));
        const uint2 there = *reinterpret_cast<const uint2*>(&there_sh[slot][2 * h]);
        const uint2 bad = *reinterpret_cast<const uint2*>(&bad_sh[slot][2 * h]);
        bool whole = (there.x & there.y) == 0xffffffffu && (bad.x | bad.y) == 0;
        if (p.causal) whole &= t0 + kHalf <= pos_lo + 1;
        if (p.window > 0) whole &= t0 > pos_hi - p.window || t0 + kHalf <= p.sinks;
        // the keys that this row sees, one bit each; where that is not all of them the scores are left as they
        // are and passed over below
        whole = __all_sync(0xffffffffu, whole) != 0;
        uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
        if (!whole) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int tb = t0 + 32 * c;
            vis[c] = c ? there.y : there.x;
            if (p.causal) vis[c] &= low_bits(pos - tb + 1);
            if (p.window > 0) vis[c] &= ~low_bits(pos - p.window + 1 - tb) | low_bits(p.sinks - tb);
            poisoned |= (vis[c] & (c ? bad.y : bad.x)) != 0;
          }
        }
        // factors of four columns, as two pairs
        auto factors = [&](int which, int j) {
          return *reinterpret_cast<const ulonglong2*>(&factor_sh[kExact ? slot : 0][which][kExact ? kHalf * h + j : 0]);
        };
        tc_wait_ld();
        float top = -INFINITY, top2 = -INFINITY;
        auto largest = [&](auto all) {
          auto seen = [&](int j, float x) { return decltype(all)::value || (vis[j >> 5] >> (j & 31) & 1u) ? x : -INFINITY; };
#pragma unroll
          for (int j = 0; j < kHalf; j += 4) {
            float2 a = make_float2(__int_as_float(v[j]), __int_as_float(v[j + 1]));
            float2 b = make_float2(__int_as_float(v[j + 2]), __int_as_float(v[j + 3]));
            if constexpr (kExact) {
              // the scores, in place of the codes' products; the largest of score + exponent of the value's scale
              const ulonglong2 ks = factors(0, j), km = factors(1, j), ev = factors(2, j);
              const uint64_t xa = fma2(pack2(a.x, a.y), ks.x, mul2(km.x, rb2));
              const uint64_t xb = fma2(pack2(b.x, b.y), ks.y, mul2(km.y, rb2));
              a = unpack2(xa);
              b = unpack2(xb);
              v[j] = __float_as_int(a.x); v[j + 1] = __float_as_int(a.y);
              v[j + 2] = __float_as_int(b.x); v[j + 3] = __float_as_int(b.y);
              a = unpack2(fma2(xa, ra2, ev.x));
              b = unpack2(fma2(xb, ra2, ev.y));
            }
            top = max3(seen(j, a.x), seen(j + 1, a.y), top);
            top2 = max3(seen(j + 2, b.x), seen(j + 3, b.y), top2);
          }
        };
        if (whole) largest(std::true_type());
        else largest(std::false_type());
        top = fmaxf(top, top2);
        const float m_new = kExact || top == -INFINITY ? top : top * ra;
        const bool grow = m_new > m_ref + kGrowth || (m_ref == -INFINITY && m_new > -INFINITY);
        if (__any_sync(0xffffffffu, grow)) {
          // nothing was seen before: nothing to rescale, the sum and O are 0
          const bool rescale = grow && m_ref > -INFINITY;
          const float alpha = rescale ? exp2_fast(m_ref - m_new) : 1.0f;
          if (grow) m_ref = m_new;
          l2 = mul2(l2, pack2(alpha, alpha));
          if (kExact) s2 = mul2(s2, pack2(alpha, alpha));
          if (__any_sync(0xffffffffu, rescale)) {
            // O may be rewritten once the products of the step before are in it; those of two steps before
            // are, this step's scores were multiplied behind them
            ok = mbar_wait(smem_u32(&bar_pv[g][h ^ 1]), (uint32_t)((step - 1) >> 1) & 1u, abort_flag);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              int o[16];
              tc_ld16(t_o + c, o);
              tc_wait_ld();
              uint32_t w[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(__int_as_float(o[j]) * alpha);
              tc_st16(t_o + c, w);
            }
          }
        }
        // ---- weights, in place of the scores: two fp16 a column; a hidden key's score of -inf gives 0.  kExact: times
        // the scales of the values, the rounded numbers first, what the rounding left behind them
        const float ref = m_ref == -INFINITY ? 0.0f : kRoom<kExact> - m_ref;
        const uint64_t ref2 = pack2(ref, ref);
        uint32_t w[kHalf / 2], rest[kExact ? kHalf / 2 : 16];
        auto weigh = [&](auto all) {
          ulonglong2 vs = {}, vm = {};
#pragma unroll
          for (int j = 0; j < kHalf; j += 2) {
            if (kExact && j % 4 == 0) { vs = factors(3, j); vm = factors(4, j); }
            float2 a = unpack2(fma2(pack2(__int_as_float(v[j]), __int_as_float(v[j + 1])), ra2, ref2));
            if (!decltype(all)::value) {
              if (!(vis[j >> 5] >> (j & 31) & 1u)) a.x = -INFINITY;
              if (!(vis[j >> 5] >> (j & 31) & 2u)) a.y = -INFINITY;
            }
            const float2 e = make_float2(exp2_fast(a.x), exp2_fast(a.y));
            const uint64_t e2 = pack2(e.x, e.y);
            l2 = add2(l2, e2);
            if constexpr (kExact) {
              s2 = fma2(e2, j % 4 == 0 ? vm.x : vm.y, s2);
              const float2 q = unpack2(mul2(e2, j % 4 == 0 ? vs.x : vs.y));
              w[j / 2] = half_pair(q.x, q.y);
              const float2 f = half_values(w[j / 2]);
              rest[j / 2] = half_pair(q.x - f.x, q.y - f.y);
            } else {
              w[j / 2] = half_pair(e.x, e.y);
            }
          }
        };
        if (whole) weigh(std::true_type());
        else weigh(std::false_type());
        tc_st16(t_sh, reinterpret_cast<uint32_t(&)[16]>(w[0]));
        tc_st16(t_sh + 16, reinterpret_cast<uint32_t(&)[16]>(w[16]));
        if constexpr (kExact) {
          tc_st16(t_sh + 32, reinterpret_cast<uint32_t(&)[16]>(rest[0]));
          tc_st16(t_sh + 48, reinterpret_cast<uint32_t(&)[16]>(rest[16]));
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_p_ready[g][h]));
      }
      const float2 lp = unpack2(l2);
      float l = lp.x + lp.y;
      const float2 sp = unpack2(s2);
      const float minima = sp.x + sp.y;
      if (poisoned) l = __int_as_float(0x7fc00000);
      if (ok && tiles > 0) ok = mbar_wait(smem_u32(&bar_pv[g][1]), (uint32_t)(tiles - 1) & 1u, abort_flag);
      if (ok) {
        tc_fence_after();
        const int rr = row0 + r;
        const bool real = r < rows_here;
        const int64_t out_row = ((int64_t)b * p.count + rr / p.group) * p.heads + head * p.group + rr % p.group;
        const int64_t at = split * p.rows + out_row;
        const float inv = p.splits > 1 ? 1.0f : (l != 0.0f ? 1.0f / l : 0.0f);   // a row that sees nothing is 0
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          int v[32];
          if (tiles > 0) {
            tc_ld32(t_o + c, v);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
          if (real) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              float o[8];
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                // a row that sees nothing has no weights, whatever its products are
                const float y = __int_as_float(v[8 * w + (((n & 3) << 1) | (n >> 2))]);
                const float x = (kExact ? y + minima : y) * inv;
                o[n] = m_ref == -INFINITY && l == 0.0f ? 0.0f : x;
              }
              if (p.splits > 1) store_f32<float, 8>(p.part + at * D + c + 8 * w, o);
              else store_f32<T, 8>(static_cast<T*>(p.out) + out_row * D + c + 8 * w, o);
            }
          }
        }
        if (p.splits > 1 && real) {
          float* lm = p.part + (int64_t)p.splits * p.rows * D;
          lm[at] = l;
          lm[(int64_t)p.splits * p.rows + at] = m_ref == -INFINITY ? -INFINITY : m_ref - kRoom<kExact>;
        }
      }
    }
    __syncwarp();
  }

  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

template <typename T, int D>
int launch(const Kv4Attention& p, cudaStream_t s) {
  constexpr int smem = 2 * 128 * D * 2 + 4 * kKeys * D * 2;
  static SmemLimit limit;
  MODIFF_CUDA(raise_smem_limit(kv4_attention_tc_kernel<T, D>, smem, limit));
  // the split waits for registers: they have to be there from the launch on
  static const int regs = [] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kv4_attention_tc_kernel<T, D>) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs != kRegsAtLaunch) return set_error(MODIFF_ERR_UNSUPPORTED, "kernel built with %d registers", regs);
  const int64_t blocks = (int64_t)p.batch * p.c.heads * p.row_tiles * p.splits;
  kv4_attention_tc_kernel<T, D><<<(unsigned)blocks, kThreads, smem, s>>>(p);
  MODIFF_LAUNCH_CHECK("kv4_attention_tc_kernel");
  return MODIFF_OK;
}

}  // namespace

// From 41 rows per key head on (bf16, us, kv4_attention.cu : this kernel; 4 sequences of up to 8000 tokens, 8 key
// heads: 24 rows 30 : 45, 32 rows 38 : 45, 48 rows 51 : 46; 64 of 8192 tokens, 32 rows 373 : 405), in fp16 from 49 on
// (the same: 40 rows 65 : 68, 48 rows 68 : 69, 52 rows 89 : 69, 64 rows 92 : 69; 64 of 8192 tokens, 40 rows 654 : 712,
// 48 rows 767 : 711; 2 of 1500 tokens, 64 channels, 52 rows 12.5 : 16, 96 rows 16.7 : 18).
bool kv4_tc_wanted(int rows, int dim, int dtype) {
  return dtype != MODIFF_FP32 && dim <= 128 && rows > (dtype == MODIFF_BF16 ? 40 : 48);
}
int kv4_tc_rows() { return kRows; }

int kv4_launch_tc(const Kv4Attention& p, int dtype, cudaStream_t s) {
  if (dtype == MODIFF_FP16) return p.c.dim == 64 ? launch<__half, 64>(p, s) : launch<__half, 128>(p, s);
  return p.c.dim == 64 ? launch<__nv_bfloat16, 64>(p, s) : launch<__nv_bfloat16, 128>(p, s);
}

}  // namespace modiff
