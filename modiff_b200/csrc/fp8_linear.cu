// Linear layers in 8-bit floating point (e4m3) with one fp32 scale for each block of 128:
//   rows     s_x[m][b] = max |x[m][128 b ..]| (1 / 448) (1 where that is 0),  code = e4m3(x / s_x)
//   weights  s_w[n / 128][b] likewise over a 128 x 128 block
//   y[m][n] = sum_b s_x[m][b] s_w[n / 128][b] (sum over the block of code_x code_w)  (+ bias[n])
// Products and sums inside a block are exact codes multiplied by tcgen05.mma kind::f8f6f4 into fp32
// tensor memory; the block's sum is drained, scaled and added in fp32 registers, so that a scale
// meets only its own block.
#include <cuda_fp8.h>

#include "fp8.cuh"

namespace modiff {

int read_device_status_fp8(int* status, int reset) { return read_status_this_unit(status, reset); }

namespace {

constexpr int kBlock = kFp8Block;
constexpr int kMostRows = 0x7fffff00;          // sizes are rounded up to tiles in 32 bits
constexpr float kInvE4m3Max = 1.0f / 448.0f;   // the scale is a product with this fp32 number

__device__ inline void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// four values, already divided by their scale, as four e4m3 codes (round to nearest even)
__device__ inline uint32_t e4m3_x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ inline float block_scale(float top) {
  // an infinity or NaN in the block stays one in its scale
  const float s = __fmul_rn(top, kInvE4m3Max);
  return s == 0.0f ? 1.0f : s;
}
__device__ inline float larger_or_nan(float a, float b) { return (a > b || isnan(a)) ? a : b; }

// ---------------------------------------------------------------- quantisers
struct QuantParams {
  const void* x;
  int64_t x_pitch;
  uint8_t* codes;
  int64_t code_pitch;
  float* scale;
  int64_t scale_pitch;
  int64_t rows;
  int k, blocks;
  FastDiv by_group;                         // groups of four blocks of a row
};

// Largest magnitude of the elements in a word (or a float): as integers, where a NaN is above infinity.
template <typename T> __device__ inline uint32_t magnitude_max(uint32_t top, uint32_t w) {
  if constexpr (sizeof(T) == 4) return max(top, w & 0x7fffffffu);
  else return __vmaxu2(top, w & 0x7fff7fffu);
}
template <typename T> __device__ inline float magnitude_value(uint32_t top) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(top);
  else {
    const uint16_t h = (uint16_t)max(top & 0xffffu, top >> 16);
    return to_f32<T>(*reinterpret_cast<const T*>(&h));
  }
}
// The two elements of a word of 16-bit values, or of two fp32 words.
template <typename T> __device__ inline float2 pair_of(const uint32_t* w, int i) {
  if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else return make_float2(to_f32<T>(reinterpret_cast<const T*>(w)[2 * i]), to_f32<T>(reinterpret_cast<const T*>(w)[2 * i + 1]));
}

// Eight lanes own a block of 128 channels of one row, 16 each; a warp does four neighbouring blocks of ROWS
// neighbouring rows, whose scales of a block it writes as one access.  All loads come first.  Bound: HBM,
// size + 1 bytes an element.  16384 x 5120 bf16: 40.5 us, 6.2 TB/s (97.8 with the compiler's divisions).
template <typename T> constexpr int kQuantRows = sizeof(T) == 4 ? 2 : 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const QuantParams p) {
  constexpr int kRows = kQuantRows<T>, kWords = 16 * sizeof(T) / 4;
  // a linear layer behind this kernel may bring its weights in meanwhile; it waits before it reads rows
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 7;
  int group;
  const int64_t row0 = (int64_t)kRows * p.by_group.divmod(blockIdx.x * 8 + (threadIdx.x >> 5), group);
  const int blk = group * 4 + ((threadIdx.x >> 3) & 3);
  const int c0 = blk * kBlock + 16 * lane;
  const bool live = blk < p.blocks && row0 < p.rows;
  uint32_t w[kRows][kWords];
  if constexpr (VEC) {
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const T* src = static_cast<const T*>(p.x) + (row0 + u) * p.x_pitch + c0;
      const bool here = live && row0 + u < p.rows && c0 < p.k;
      if (here && c0 + 16 <= p.k) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
          w[u][4 * i] = v.x; w[u][4 * i + 1] = v.y; w[u][4 * i + 2] = v.z; w[u][4 * i + 3] = v.w;
        }
      } else {
        T* t = reinterpret_cast<T*>(w[u]);
#pragma unroll
        for (int e = 0; e < 16; ++e) t[e] = here && c0 + e < p.k ? src[e] : from_f32<T>(0.0f);
      }
    }
  } else {
    // rows that do not start on 16 bytes: neighbouring lanes load neighbouring elements, shared memory deals
    // them out (the layer 13578 x 1660 -> 135, bf16: 62 us with every lane at its own 16, 33 so)
    __shared__ __align__(16) T staged[8][kRows][4 * kBlock];
    T(&mine)[kRows][4 * kBlock] = staged[threadIdx.x >> 5];
    const int w0 = group * 4 * kBlock + (threadIdx.x & 31);
#pragma unroll
    for (int u = 0; u < kRows; ++u) {
      const T* src = static_cast<const T*>(p.x) + (row0 + u) * p.x_pitch;
      const bool here = row0 + u < p.rows;
#pragma unroll
      for (int i = 0; i < 4 * kBlock / 32; ++i)
        mine[u][32 * i + (threadIdx.x & 31)] = here && w0 + 32 * i < p.k ? src[w0 + 32 * i] : from_f32<T>(0.0f);
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < kRows; ++u)
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(&mine[u][16 * (threadIdx.x & 31) + i * (16 / sizeof(T))]);
        w[u][4 * i] = v.x; w[u][4 * i + 1] = v.y; w[u][4 * i + 2] = v.z; w[u][4 * i + 3] = v.w;
      }
  }
  float scale[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kWords; ++i) top = magnitude_max<T>(top, w[u][i]);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = magnitude_max<T>(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float s = block_scale(magnitude_value<T>(top));
    scale[u] = s;
    if (!live || row0 + u >= p.rows) continue;
    uint32_t codes[4];
    if (s > 1e-25f && s < 1e25f) {
      uint64_t r2, ms2;
      const float r = __frcp_rn(s);
      asm("mov.b64 %0, {%1, %1};" : "=l"(r2) : "f"(r));
      asm("mov.b64 %0, {%1, %1};" : "=l"(ms2) : "f"(-s));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = pair_of<T>(w[u], 2 * i), b = pair_of<T>(w[u], 2 * i + 1);
        const float2 qa = divide_pair(a.x, a.y, r2, ms2), qb = divide_pair(b.x, b.y, r2, ms2);
        codes[i] = e4m3_x4(qa.x, qa.y, qb.x, qb.y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = pair_of<T>(w[u], 2 * i), b = pair_of<T>(w[u], 2 * i + 1);
        codes[i] = e4m3_x4(__fdiv_rn(a.x, s), __fdiv_rn(a.y, s), __fdiv_rn(b.x, s), __fdiv_rn(b.y, s));
      }
    }
    if (c0 < p.k)                                // up to the next multiple of 16, zeros from k on
      *reinterpret_cast<uint4*>(p.codes + (row0 + u) * p.code_pitch + c0) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  }
  if (lane == 0 && live) {
    float* dst = p.scale + blk * p.scale_pitch + row0;         // the pitch covers whole groups of four rows
    store_f32<float, kRows>(dst, scale);
  }
}

// One block of 256 threads per 128 x 128 block of a weight matrix (once per weight version).
template <typename T>
__global__ void __launch_bounds__(256)
fp8_pack_weight_kernel(const T* __restrict__ w, int64_t w_pitch, int n, int k, uint8_t* __restrict__ codes,
                       int64_t code_pitch, float* __restrict__ scale, int64_t scale_pitch) {
  __shared__ float sh[8];
  const int c = blockIdx.x * kBlock + (threadIdx.x & 127);
  const int r0 = blockIdx.y * kBlock + (threadIdx.x >> 7);
  float top = 0.0f;
  if (c < k)
    for (int r = r0; r < n && r < (int)(blockIdx.y + 1) * kBlock; r += 2)
      top = larger_or_nan(fabsf(to_f32<T>(w[r * w_pitch + c])), top);
  for (int o = 16; o > 0; o >>= 1) top = larger_or_nan(__shfl_xor_sync(0xffffffffu, top, o), top);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = larger_or_nan(sh[i], top);
  const float s = block_scale(top);
  if (threadIdx.x == 0) scale[blockIdx.y * scale_pitch + blockIdx.x] = s;
  if (c < code_pitch)
    for (int r = r0; r < n && r < (int)(blockIdx.y + 1) * kBlock; r += 2) {
      const float q = c < k ? __fdiv_rn(to_f32<T>(w[r * w_pitch + c]), s) : 0.0f;
      codes[r * code_pitch + c] = (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
    }
}

// ---------------------------------------------------------------- few rows
// Weights as the 128 rows of the MMA, up to TN tokens as its columns, the channels split over a
// cluster of CTAs whose partial sums meet through distributed shared memory in rank order.  Bound:
// the weights' bytes; four stages of (16 KB + 128 TN) are in flight per CTA.  64 x 8192 x 8192, codes to bf16: 14.9 us,
// 4.6 TB/s.
//
// FUSED (a few rows): the epilogue warps quantise the rows' part of the CTA's channels themselves, straight
// into the swizzled shared-memory layout of an MMA operand, while the weights are on their way: one
// launch and no workspace.  Operand rows beyond the last token hold whatever was there; only columns of
// the result that nobody stores depend on them.
constexpr int kStages = 4;
constexpr int kScaleChunk = 8;              // channel blocks whose scales a warp keeps at a time
constexpr int kATile = 128 * kBlock;
constexpr int kFusedRows = 16;              // columns of the fused kernel's MMA
constexpr int kFusedBlocks = 16;            // channel blocks of one CTA that it can hold

// epilogue warps: four own the 128 weight rows; from 64 tokens on two such sets share the columns
template <int TN> constexpr int kRowsWarps = TN >= 64 ? 8 : 4;
template <int TN> constexpr int kRowsThreads = 64 + 32 * kRowsWarps<TN>;
template <int TN, bool FUSED> constexpr int rows_smem() {
  return FUSED ? kStages * kATile + kFusedBlocks * (TN * kBlock + TN * 4)
               : kStages * (kATile + TN * kBlock) + 4 * kScaleChunk * TN * 4;
}

__device__ inline float4 ld_cluster_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

// One row's block of 128 channels by one warp, four channels a lane.
template <typename T>
__device__ inline void load_block(const Fp8Params& p, int row, int kb, int lane, float (&x)[4]) {
  const int c0 = kb * kBlock + 4 * lane;
  const T* src = static_cast<const T*>(p.x) + (int64_t)row * p.x_pitch + c0;
  if (p.x_vec && c0 + 4 <= p.k) {
    load_f32<T, 4>(src, x);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = c0 + e < p.k ? to_f32<T>(src[e]) : 0.0f;
  }
}

template <typename T, int TN, bool FUSED>
__global__ void __launch_bounds__(kRowsThreads<TN>)
fp8_linear_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                       const __grid_constant__ Fp8Params p) {
  constexpr int kBTile = TN * kBlock;
  constexpr int kStageBytes = FUSED ? kATile : kATile + kBTile;
  constexpr int kCols = TN < 32 ? 32 : TN;
  constexpr int kEpiWarps = kRowsWarps<TN>;
  constexpr int kOwn = TN / (kEpiWarps / 4);                   // columns of an epilogue warp
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kStages], bar_empty[kStages], bar_acc_full[2], bar_acc_empty[2], bar_x;
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_sh;
  const uint32_t ring = smem_u32(smem_raw);
  const uint32_t x_tiles = ring + kStages * kStageBytes;       // FUSED: [block][TN rows of 128 bytes, swizzled]

  if (threadIdx.x == 0) {
    abort_sh = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), kEpiWarps);
    }
    mbar_init(smem_u32(&bar_x), kEpiWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_sh)),
                 "r"((uint32_t)(2 * kCols))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;

  const int rank = blockIdx.x % p.split;
  const int nt = blockIdx.x / p.split;
  const int tok0 = blockIdx.y * TN;
  const int kb0 = (int)((int64_t)p.kb * rank / p.split), kb1 = (int)((int64_t)p.kb * (rank + 1) / p.split);

  uint64_t acc[kOwn / 2];                                      // pairs of columns
#pragma unroll
  for (int j = 0; j < kOwn / 2; ++j) acc[j] = 0ull;
  const int col0 = warp >= 2 ? ((warp - 2) >> 2) * kOwn : 0;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      // the weights do not depend on the kernel before this one, the rows' codes do
      const int ahead = min(kStages, kb1 - kb0);
      for (int i = 0; i < ahead; ++i) {
        const uint32_t full = smem_u32(&bar_full[i]);
        mbar_arrive_expect_tx(full, kStageBytes);
        tma_load_2d(ring + i * kStageBytes, &map_w, full, (kb0 + i) * kBlock, nt * 128);
      }
      if (!FUSED) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        for (int i = 0; i < ahead; ++i)
          tma_load_2d(ring + i * kStageBytes + kATile, &map_x, smem_u32(&bar_full[i]), (kb0 + i) * kBlock, tok0);
      }
      for (int kb = kb0 + kStages; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bar_empty[stage]), phase, abort_flag)) break;
        const uint32_t full = smem_u32(&bar_full[stage]);
        mbar_arrive_expect_tx(full, kStageBytes);
        tma_load_2d(ring + stage * kStageBytes, &map_w, full, kb * kBlock, nt * 128);
        if (!FUSED) tma_load_2d(ring + stage * kStageBytes + kATile, &map_x, full, kb * kBlock, tok0);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_e4m3(128, TN);
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    bool ok = !FUSED || mbar_wait(smem_u32(&bar_x), 0, abort_flag);
    for (int kb = kb0; kb < kb1 && ok; ++kb) {
      ok = mbar_wait(smem_u32(&bar_acc_empty[buf]), bphase ^ 1u, abort_flag) &&
           mbar_wait(smem_u32(&bar_full[stage]), phase, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint64_t adesc = make_smem_desc(ring + stage * kStageBytes);
      const uint64_t bdesc = make_smem_desc(FUSED ? x_tiles + (kb - kb0) * kBTile : ring + stage * kStageBytes + kATile);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kBlock / 32; ++k)
          tc_mma_f8(tmem_base + (uint32_t)(buf * kCols), adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc,
                    k > 0 ? 1u : 0u);
        tc_commit(smem_u32(&bar_empty[stage]));
        tc_commit(smem_u32(&bar_acc_full[buf]));
      }
      __syncwarp();
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
      if (++buf == 2) { buf = 0; bphase ^= 1u; }
    }
  } else {
    const int quarter = warp & 3;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
    // s_x s_w as [block][token]: of all the CTA's blocks (FUSED), or a warp's own copy of the next few
    float* sc = FUSED ? reinterpret_cast<float*>(smem_raw + kStages * kATile + kFusedBlocks * kBTile)
                      : reinterpret_cast<float*>(smem_raw + kStages * kStageBytes) + (warp - 2) * kScaleChunk * kOwn;
    constexpr int kScPitch = FUSED ? TN : kOwn;
    bool ok = true;
    if (FUSED) {
      constexpr int kBatch = 4;                                // blocks whose loads a warp has in flight
      const int here = min(TN, p.rows - tok0), pieces = (kb1 - kb0) * here;
      for (int i0 = warp - 2; i0 < pieces; i0 += kEpiWarps * kBatch) {
        float x[kBatch][4], sw[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kEpiWarps;
          if (i < pieces) {
            load_block<T>(p, tok0 + i % here, kb0 + i / here, lane, x[u]);
            sw[u] = __ldg(p.sw + (int64_t)nt * p.sw_pitch + kb0 + i / here);
          }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int i = i0 + u * kEpiWarps;
          if (i >= pieces) break;
          const int r = i % here, blk = i / here;
          float top = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e) top = larger_or_nan(fabsf(x[u][e]), top);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = larger_or_nan(__shfl_xor_sync(0xffffffffu, top, o), top);
          const float s = block_scale(top);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] = __fdiv_rn(x[u][e], s);
          uint8_t* dst = smem_raw + kStages * kATile + blk * kBTile + r * kBlock + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3);
          *reinterpret_cast<uint32_t*>(dst) = e4m3_x4(x[u][0], x[u][1], x[u][2], x[u][3]);
          if (lane == 0) sc[blk * TN + r] = s * sw[u];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_x));
      ok = mbar_wait(smem_u32(&bar_x), 0, abort_flag);         // the scales of the other warps' rows
    } else {
      asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    int buf = 0;
    uint32_t bphase = 0;
    for (int kb = kb0; kb < kb1 && ok; ++kb) {
      const int at = FUSED ? kb - kb0 : (kb - kb0) % kScaleChunk;
      if (!FUSED && at == 0) {
        __syncwarp();
#pragma unroll
        for (int t = lane; t < kOwn; t += 32)
#pragma unroll
          for (int i = 0; i < kScaleChunk; ++i)
            sc[i * kOwn + t] = tok0 + col0 + t < p.rows && kb + i < kb1
                                   ? p.sx[(int64_t)(kb + i) * p.sx_pitch + tok0 + col0 + t] *
                                         __ldg(p.sw + (int64_t)nt * p.sw_pitch + kb + i)
                                   : 0.0f;
        __syncwarp();
      }
      ok = mbar_wait(smem_u32(&bar_acc_full[buf]), bphase, abort_flag);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + (uint32_t)(buf * kCols + col0);
      constexpr int kPiece = kOwn < 32 ? kOwn : 32;
#pragma unroll
      for (int q = 0; q < kOwn / kPiece; ++q) {
        int v[kPiece];
        if constexpr (kPiece == 16) tc_ld16(t_acc, v); else tc_ld32(t_acc + 32 * q, v);
        tc_wait_ld();
        if (q == kOwn / kPiece - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[buf]));
        }
#pragma unroll
        for (int j = 0; j < kPiece; j += 4) {
          const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(sc + at * kScPitch + kPiece * q + j);
          fma_pair(acc[(kPiece * q + j) / 2], v[j], v[j + 1], f.x);
          fma_pair(acc[(kPiece * q + j) / 2 + 1], v[j + 2], v[j + 3], f.y);
        }
      }
      if (++buf == 2) { buf = 0; bphase ^= 1u; }
    }
    __syncwarp();
  }

  // ---- the cluster's partial sums, then bias and rounding
  const int row = (warp & 3) * 32 + lane;
  const int n = nt * 128 + row;
  const bool epilogue = warp >= 2;
  T* y = static_cast<T*>(p.y);
  float sum[kOwn];
#pragma unroll
  for (int j = 0; j < kOwn / 2; ++j) asm("mov.b64 {%0, %1}, %2;" : "=f"(sum[2 * j]), "=f"(sum[2 * j + 1]) : "l"(acc[j]));
  if (p.split > 1) {
    float* red = reinterpret_cast<float*>(smem_raw);           // [token][128]: the ring is empty by now
    __syncthreads();
    if (epilogue) {
#pragma unroll
      for (int j = 0; j < kOwn; ++j)
        if (tok0 + col0 + j < p.rows) red[(col0 + j) * 128 + row] = sum[j];
    }
    cluster_sync_all();
    if (epilogue) {
      const int here = min(TN, p.rows - tok0);
      const int j0 = here * rank / p.split, j1 = here * (rank + 1) / p.split;
      for (int i = threadIdx.x - 64; i < (j1 - j0) * 32; i += 32 * kEpiWarps) {
        const int j = j0 + (i >> 5), r4 = 4 * (i & 31);
        float4 part[8];                                        // split <= 8: all loads first, then the sum in order
#pragma unroll
        for (int r = 0; r < 8; ++r)
          if (r < p.split) part[r] = ld_cluster_f32x4(map_to_cta(ring + (uint32_t)(j * 128 + r4) * 4, (uint32_t)r));
        float4 t = part[0];
#pragma unroll
        for (int r = 1; r < 8; ++r)
          if (r < p.split) { t.x += part[r].x; t.y += part[r].y; t.z += part[r].z; t.w += part[r].w; }
        const int n4 = nt * 128 + r4;
        float v[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (p.bias && n4 + e < p.n) v[e] += to_f32<T>(static_cast<const T*>(p.bias)[n4 + e]);
        T* dst = y + (int64_t)(tok0 + j) * p.y_pitch + n4;
        if (p.y_vec && n4 + 4 <= p.n) {
          store_f32<T, 4>(dst, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n4 + e < p.n) dst[e] = from_f32<T>(v[e]);
        }
      }
    }
    cluster_sync_all();                                        // nobody leaves while its sums are read
  } else if (epilogue && n < p.n) {
    const float bias = p.bias ? to_f32<T>(static_cast<const T*>(p.bias)[n]) : 0.0f;
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (tok0 + col0 + j < p.rows) y[(int64_t)(tok0 + col0 + j) * p.y_pitch + n] = from_f32<T>(sum[j] + bias);
  }

  __syncwarp();
  if (abort_sh) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);            // let copies in flight land
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)(2 * kCols))
                 : "memory");
  }
}

// Channels split over up to eight CTAs of a cluster while the grid leaves SMs idle (two CTAs share one) and every
// CTA keeps two blocks (64 x 8192 x 8192, us for 2 : 4 : 8 parts, 18.7 : 14.9 : 22.1).
int rows_split(int rows, int n, int kb, int tn) {
  const int64_t tiles = (int64_t)ceil_div(n, 128) * ceil_div(rows, tn);
  int split = 1;
  while (split < 8 && tiles * split < device_sms() && kb >= 4 * split) split *= 2;
  return split;
}

// Rows few enough to be quantised by the CTAs that multiply them, in one launch: every CTA of a column of tiles
// repeats that work.  Device time against two kernels (us): 1 x 4096 x 4096 (8 row blocks a CTA) 7.4 : 7.9, 1 x
// 8192 x 8192 (16) 13.4 : 12.5, 8 x 1024 x 4096 (16) 8.2 : 6.6, 2 x 8192 x 8192 (32) 16.4 : 12.1; the second
// launch and its workspace cost the host about 5 us.
bool fused_wanted(int rows, int k, int n) {
  const int kb = ceil_div(k, kBlock);
  const int blocks = ceil_div(kb, rows_split(rows, n, kb, kFusedRows));
  return rows <= kFusedRows && blocks <= kFusedBlocks && rows * blocks <= 16;
}

template <typename T, int TN, bool FUSED>
int launch_rows(const Fp8Operands& o, Fp8Params p, cudaStream_t s) {
  EncodeTiledFn encode = get_encode_fn();
  if (!encode) return set_error(MODIFF_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
  const int n_tiles = ceil_div(p.n, 128), t_tiles = ceil_div(p.rows, TN);
  MODIFF_CHECK_ARG(t_tiles <= 65535, "too many rows");
  CUtensorMap mw, mx;
  CUresult r = fp8_map(encode, &mw, o.w, o.k, p.n, o.w_pitch, 128);
  if (FUSED) mx = mw;
  if (!FUSED && r == CUDA_SUCCESS) r = fp8_map(encode, &mx, o.x, o.k, p.rows, o.x_pitch, TN);
  if (r != CUDA_SUCCESS) return set_error(MODIFF_ERR_CUDA, "cuTensorMapEncodeTiled(fp8 operands) failed: %d", (int)r);
  p.split = rows_split(p.rows, p.n, p.kb, TN);
  p.y_vec = ((uintptr_t)p.y % (4 * sizeof(T)) | (uintptr_t)(p.y_pitch % 4)) == 0;
  constexpr int smem = rows_smem<TN, FUSED>();
  static SmemLimit limit;
  MODIFF_CUDA(raise_smem_limit(fp8_linear_rows_kernel<T, TN, FUSED>, smem, limit));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * p.split), (unsigned)t_tiles);
  cfg.blockDim = dim3(kRowsThreads<TN>);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = !FUSED && p.x ? 2 : 1;      // right behind this call's own quantiser
  MODIFF_CUDA(cudaLaunchKernelEx(&cfg, fp8_linear_rows_kernel<T, TN, FUSED>, mw, mx, p));
  return MODIFF_OK;
}

int launch_linear(const Fp8Operands& o, const Fp8Params& p, int dtype, cudaStream_t s) {
  if (fp8_pair_wanted(p.rows, p.n)) return fp8_launch_pair(o, p, dtype, s);
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    // the narrowest tile that holds the rows, at most 64 (4096 x 4096, us with the quantiser, tiles of 16 : 32 : 64 :
    // 128: 16 rows 8.7 : 9.0 : 9.7 : 11.5, 33 rows 12.7 : 10.3 : 9.9 : 10.7; 128 x 8192 x 8192 32 : 64 : 128: 34.6 : 25.2 : 27.3)
    if (p.rows <= 16) return launch_rows<T, 16, false>(o, p, s);
    if (p.rows <= 32) return launch_rows<T, 32, false>(o, p, s);
    return launch_rows<T, 64, false>(o, p, s);
  });
}

int check_weight(const uint8_t* w, int64_t w_pitch, const float* w_scale, int64_t w_scale_pitch, const void* bias,
                 const void* y, int64_t y_pitch, int rows, int k, int n, int dtype) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(rows >= 0 && k > 0 && n > 0, "bad shape");
  MODIFF_CHECK_ARG(rows <= kMostRows && k <= kMostRows && n <= kMostRows, "more than %d rows or channels", kMostRows);
  if (rows == 0) return MODIFF_OK;
  const int size = dtype_bytes(dtype);
  MODIFF_CHECK_ARG(w && w_scale && y, "NULL pointer argument");
  MODIFF_CHECK_ARG(w_pitch >= k && w_pitch % 16 == 0 && (uintptr_t)w % 16 == 0,
                   "rows of codes need 16-byte alignment and a pitch that is a multiple of 16");
  MODIFF_CHECK_ARG(w_scale_pitch >= ceil_div(k, kBlock) && y_pitch >= n, "bad pitch");
  MODIFF_CHECK_ARG((uintptr_t)w_scale % 4 == 0 && (((uintptr_t)y | (uintptr_t)bias) % size) == 0, "misaligned tensor");
  return MODIFF_OK;
}

}  // namespace
}  // namespace modiff

using namespace modiff;

// scales of one block of all rows, padded to 16 bytes
static int64_t scale_row(int rows) { return ((int64_t)rows + 3) / 4 * 4; }

static int quantize_rows(const void* x, int64_t x_pitch, int64_t rows, int k, int dtype, uint8_t* codes,
                         int64_t code_pitch, float* scale, int64_t scale_pitch, cudaStream_t s) {
  const int size = dtype_bytes(dtype), blocks = ceil_div(k, kBlock);
  const int groups = ceil_div(blocks, 4), per = size == 4 ? kQuantRows<float> : kQuantRows<__half>;
  QuantParams p{x, x_pitch, codes, code_pitch, scale, scale_pitch, rows, k, blocks, FastDiv(groups)};
  const int64_t warps = ceil_div64(rows, per) * groups;
  MODIFF_CHECK_ARG(warps <= 0x7fffffff - 8, "too many rows");
  const int64_t grid = ceil_div64(warps, 8);
  const bool vec = (((uintptr_t)x | (uintptr_t)(x_pitch * size)) & 15) == 0;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (vec)
      fp8_quantize_kernel<T, true><<<(unsigned)grid, 256, 0, s>>>(p);
    else
      fp8_quantize_kernel<T, false><<<(unsigned)grid, 256, 0, s>>>(p);
    MODIFF_LAUNCH_CHECK("fp8_quantize_kernel");
    return MODIFF_OK;
  });
}

extern "C" int modiff_fp8_quantize(const void* x, int64_t x_pitch, int64_t rows, int k, int dtype, uint8_t* codes,
                                   int64_t code_pitch, float* scale, int64_t scale_pitch, void* stream) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(rows >= 0 && k > 0 && k <= kMostRows, "bad shape");
  if (rows == 0) return MODIFF_OK;
  MODIFF_CHECK_ARG(x && codes && scale, "NULL pointer argument");
  MODIFF_CHECK_ARG(code_pitch >= k && code_pitch % 16 == 0 && (uintptr_t)codes % 16 == 0,
                   "rows of codes need 16-byte alignment and a pitch that is a multiple of 16");
  MODIFF_CHECK_ARG(scale_pitch >= rows && scale_pitch % 4 == 0 && (uintptr_t)scale % 16 == 0,
                   "scales need 16-byte alignment and a pitch that is a multiple of 4");
  MODIFF_CHECK_ARG((uintptr_t)x % dtype_bytes(dtype) == 0, "misaligned tensor");
  return quantize_rows(x, x_pitch, rows, k, dtype, codes, code_pitch, scale, scale_pitch, (cudaStream_t)stream);
}

extern "C" int modiff_fp8_pack_weight(const void* w, int64_t w_pitch, int n, int k, int dtype, uint8_t* codes,
                                      int64_t code_pitch, float* scale, int64_t scale_pitch, void* stream) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(n > 0 && k > 0 && n <= kMostRows && k <= kMostRows, "bad shape");
  MODIFF_CHECK_ARG(w && codes && scale, "NULL pointer argument");
  MODIFF_CHECK_ARG(code_pitch >= k && code_pitch <= round_up(k, 16) && code_pitch % 16 == 0 && (uintptr_t)codes % 16 == 0,
                   "rows of codes need 16-byte alignment and the next multiple of 16 as pitch");
  MODIFF_CHECK_ARG(scale_pitch >= ceil_div(k, kBlock) && (uintptr_t)scale % 4 == 0 &&
                       (uintptr_t)w % dtype_bytes(dtype) == 0, "misaligned tensor");
  const dim3 grid((unsigned)ceil_div(k, kBlock), (unsigned)ceil_div(n, kBlock));
  MODIFF_CHECK_ARG(grid.y <= 65535, "too many weight rows");
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    fp8_pack_weight_kernel<T><<<grid, 256, 0, (cudaStream_t)stream>>>(static_cast<const T*>(w), w_pitch, n, k, codes,
                                                                      code_pitch, scale, scale_pitch);
    MODIFF_LAUNCH_CHECK("fp8_pack_weight_kernel");
    return MODIFF_OK;
  });
}

extern "C" int modiff_fp8_linear(const uint8_t* codes, int64_t code_pitch, const float* scale, int64_t scale_pitch,
                                 const uint8_t* w, int64_t w_pitch, const float* w_scale, int64_t w_scale_pitch,
                                 const void* bias, void* y, int64_t y_pitch, int rows, int k, int n, int dtype,
                                 void* stream) {
  const int rc = check_weight(w, w_pitch, w_scale, w_scale_pitch, bias, y, y_pitch, rows, k, n, dtype);
  if (rc || rows == 0) return rc;
  const int kb = ceil_div(k, kBlock);
  MODIFF_CHECK_ARG(codes && scale, "NULL pointer argument");
  MODIFF_CHECK_ARG(code_pitch >= k && code_pitch % 16 == 0 && (uintptr_t)codes % 16 == 0,
                   "rows of codes need 16-byte alignment and a pitch that is a multiple of 16");
  MODIFF_CHECK_ARG(scale_pitch >= rows && scale_pitch % 4 == 0 && (uintptr_t)scale % 16 == 0,
                   "scales need 16-byte alignment and a pitch that is a multiple of 4");
  const Fp8Params p{scale, scale_pitch, w_scale, w_scale_pitch, bias, y, y_pitch, rows, n, kb, 1, nullptr, 0, k, 0};
  return launch_linear(Fp8Operands{codes, w, code_pitch, w_pitch, k}, p, dtype, (cudaStream_t)stream);
}

extern "C" int64_t modiff_fp8_linear_bytes(int rows, int k, int n) {
  if (rows <= 0 || k <= 0 || n <= 0 || rows > kMostRows || k > kMostRows || n > kMostRows || fused_wanted(rows, k, n)) return 0;
  return (int64_t)rows * round_up(k, 16) + 4ll * scale_row(rows) * ceil_div(k, kBlock);
}

extern "C" int modiff_fp8_linear_x(const void* x, int64_t x_pitch, const uint8_t* w, int64_t w_pitch,
                                   const float* w_scale, int64_t w_scale_pitch, const void* bias, void* y,
                                   int64_t y_pitch, int rows, int k, int n, int dtype, void* workspace,
                                   void* stream) {
  const int rc = check_weight(w, w_pitch, w_scale, w_scale_pitch, bias, y, y_pitch, rows, k, n, dtype);
  if (rc || rows == 0) return rc;
  const int size = dtype_bytes(dtype), kb = ceil_div(k, kBlock);
  MODIFF_CHECK_ARG(x && (uintptr_t)x % size == 0, "NULL or misaligned tensor");
  cudaStream_t s = (cudaStream_t)stream;
  Fp8Params p{nullptr, 0, w_scale, w_scale_pitch, bias, y, y_pitch, rows, n, kb, 1, x, x_pitch, k, 0};
  if (fused_wanted(rows, k, n)) {
    p.x_vec = ((uintptr_t)x % (4 * size) | (uintptr_t)(x_pitch % 4)) == 0;
    const Fp8Operands o{nullptr, w, 0, w_pitch, k};
    return with_dtype(dtype, [&](auto tag) { return launch_rows<decltype(tag), kFusedRows, true>(o, p, s); });
  }
  MODIFF_CHECK_ARG(workspace && (uintptr_t)workspace % 16 == 0, "NULL or misaligned workspace");
  const int64_t kp = round_up(k, 16);
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  float* scale = reinterpret_cast<float*>(codes + rows * kp);
  const int rq = quantize_rows(x, x_pitch, rows, k, dtype, codes, kp, scale, scale_row(rows), s);
  if (rq) return rq;
  p.sx = scale;
  p.sx_pitch = scale_row(rows);
  return launch_linear(Fp8Operands{codes, w, kp, w_pitch, k}, p, dtype, s);
}
