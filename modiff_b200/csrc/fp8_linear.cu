// Linear layers in 8-bit floating point (e4m3) with one fp32 scale for each block of 128:
//   rows     s_x[m][b] = max |x[m][128 b ..]| / 448 (1 where that is 0),  code = e4m3(x / s_x)
//   weights  s_w[n / 128][b] likewise over a 128 x 128 block
//   y[m][n] = sum_b s_x[m][b] s_w[n / 128][b] (sum over the block of code_x code_w)  (+ bias[n])
// Products and sums inside a block are exact codes multiplied by tcgen05.mma kind::f8f6f4 into fp32
// tensor memory; the block's sum is drained, scaled and added in fp32 registers, so that a scale
// meets only its own block.
#include <cuda_fp8.h>

#include "tc_common.cuh"
#include "types.cuh"

namespace modiff {

int read_device_status_fp8(int* status, int reset) { return read_status_this_unit(status, reset); }

namespace {

constexpr int kBlock = 128;                 // channels (and weight rows) of one scale
constexpr float kE4m3Max = 448.0f;

__device__ inline void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4: e4m3 x e4m3 -> fp32, both operands K-major.
__host__ __device__ inline uint32_t make_idesc_e4m3(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// four values, already divided by their scale, as four e4m3 codes (round to nearest even)
__device__ inline uint32_t e4m3_x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ inline float block_scale(float top) {
  // an infinity or NaN in the block stays one in its scale
  return top > 0.0f ? __fdiv_rn(top, kE4m3Max) : (top == 0.0f ? 1.0f : top);
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
  int64_t rows, items;
  int k, blocks;
};

// Sixteen lanes own a block of 128 channels of one row, 8 each.  Bound: HBM, size + 1 bytes an element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
fp8_quantize_kernel(const QuantParams p) {
  const int lane = threadIdx.x & 15;
  const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = item < p.items;
  const int64_t row = live ? item / p.blocks : 0;
  const int blk = live ? (int)(item % p.blocks) : 0;
  const int c0 = blk * kBlock + 8 * lane;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (live && c0 < p.k) {
    const T* src = static_cast<const T*>(p.x) + row * p.x_pitch + c0;
    if (VEC && c0 + 8 <= p.k) {
      load_f32<T, 8>(src, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < p.k) x[e] = to_f32<T>(src[e]);
    }
  }
  float top = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = larger_or_nan(fabsf(x[e]), top);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = larger_or_nan(__shfl_xor_sync(0xffffffffu, top, o), top);
  if (!live) return;
  const float s = block_scale(top);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = __fdiv_rn(x[e], s);
  if (c0 < p.code_pitch) {                       // the pitch is a multiple of 16
    uint2 w;
    w.x = e4m3_x4(x[0], x[1], x[2], x[3]);
    w.y = e4m3_x4(x[4], x[5], x[6], x[7]);
    *reinterpret_cast<uint2*>(p.codes + row * p.code_pitch + c0) = w;
  }
  if (lane == 0) p.scale[row * p.scale_pitch + blk] = s;
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
// the weights' bytes; four stages of (16 KB + 128 TN) are in flight per CTA.
constexpr int kStages = 4;
constexpr int kEpiWarps = 4;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kScaleChunk = 8;              // channel blocks whose scales a warp keeps at a time
constexpr int kATile = 128 * kBlock;

struct LinearParams {
  const float* sx;
  int64_t sx_pitch;
  const float* sw;
  int64_t sw_pitch;
  const void* bias;
  void* y;
  int64_t y_pitch;
  int rows, n, kb, split;
};

template <int TN> constexpr int rows_smem() { return kStages * (kATile + TN * kBlock) + kEpiWarps * kScaleChunk * TN * 4; }

template <typename T, int TN>
__global__ void __launch_bounds__(kThreads)
fp8_linear_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                       const __grid_constant__ LinearParams p) {
  constexpr int kBTile = TN * kBlock;
  constexpr int kStageBytes = kATile + kBTile;
  constexpr int kCols = TN < 32 ? 32 : TN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kStages], bar_empty[kStages], bar_acc_full[2], bar_acc_empty[2];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int abort_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &abort_sh;
  const uint32_t ring = smem_u32(smem_raw);

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

  float acc[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) acc[j] = 0.0f;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1u, abort_flag)) break;
        const uint32_t full = smem_u32(&bar_full[stage]);
        mbar_arrive_expect_tx(full, kStageBytes);
        tma_load_2d(ring + stage * kStageBytes, &map_w, full, kb * kBlock, nt * 128);
        tma_load_2d(ring + stage * kStageBytes + kATile, &map_x, full, kb * kBlock, tok0);
        if (++stage == kStages) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t idesc = make_idesc_e4m3(128, TN);
    int stage = 0, buf = 0;
    uint32_t phase = 0, bphase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(smem_u32(&bar_acc_empty[buf]), bphase ^ 1u, abort_flag)) break;
      if (!mbar_wait(smem_u32(&bar_full[stage]), phase, abort_flag)) break;
      tc_fence_after();
      const uint64_t adesc = make_smem_desc(ring + stage * kStageBytes);
      const uint64_t bdesc = make_smem_desc(ring + stage * kStageBytes + kATile);
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
    float* sc = reinterpret_cast<float*>(smem_raw + kStages * kStageBytes) + (warp - 2) * kScaleChunk * TN;
    int buf = 0;
    uint32_t bphase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int at = (kb - kb0) % kScaleChunk;
      if (at == 0) {                              // s_x s_w of the next blocks, [block][token]
        __syncwarp();
#pragma unroll
        for (int t = lane; t < TN; t += 32)
#pragma unroll
          for (int i = 0; i < kScaleChunk; ++i)
            sc[i * TN + t] = tok0 + t < p.rows && kb + i < kb1
                                 ? __ldg(p.sx + (int64_t)(tok0 + t) * p.sx_pitch + kb + i) *
                                       __ldg(p.sw + (int64_t)nt * p.sw_pitch + kb + i)
                                 : 0.0f;
        __syncwarp();
      }
      if (!mbar_wait(smem_u32(&bar_acc_full[buf]), bphase, abort_flag)) break;
      tc_fence_after();
      const uint32_t t_acc = t_lane + (uint32_t)(buf * kCols);
#pragma unroll
      for (int q = 0; q < kCols / 32; ++q) {
        int v[32];
        tc_ld32(t_acc + 32 * q, v);
        tc_wait_ld();
        if (q == kCols / 32 - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_acc_empty[buf]));
        }
#pragma unroll
        for (int j = 0; j < (TN < 32 ? TN : 32); ++j)
          acc[32 * q + j] = fmaf(__int_as_float(v[j]), sc[at * TN + 32 * q + j], acc[32 * q + j]);
      }
      if (++buf == 2) { buf = 0; bphase ^= 1u; }
    }
    __syncwarp();
  }

  // ---- the cluster's partial sums, then bias and rounding
  const int row = (warp & 3) * 32 + lane;
  const int n = nt * 128 + row;
  const bool epilogue = warp >= 2;
  const float bias = epilogue && p.bias && n < p.n ? to_f32<T>(static_cast<const T*>(p.bias)[n]) : 0.0f;
  T* y = static_cast<T*>(p.y);
  if (p.split > 1) {
    float* red = reinterpret_cast<float*>(smem_raw);           // [token][128]: the ring is empty by now
    __syncthreads();
    if (epilogue) {
#pragma unroll
      for (int j = 0; j < TN; ++j) red[j * 128 + row] = acc[j];
    }
    cluster_sync_all();
    if (epilogue) {
      const int j0 = TN * rank / p.split, j1 = TN * (rank + 1) / p.split;
      for (int j = j0; j < j1 && tok0 + j < p.rows; ++j) {
        float sum = 0.0f;
        for (int r = 0; r < p.split; ++r)
          sum += __int_as_float(ld_cluster_s32(map_to_cta(ring + (uint32_t)(j * 128 + row) * 4, (uint32_t)r)));
        if (n < p.n) y[(int64_t)(tok0 + j) * p.y_pitch + n] = from_f32<T>(sum + bias);
      }
    }
    cluster_sync_all();                                        // nobody leaves while its sums are read
  } else if (epilogue && n < p.n) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      if (tok0 + j < p.rows) y[(int64_t)(tok0 + j) * p.y_pitch + n] = from_f32<T>(acc[j] + bias);
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

CUresult encode_codes(EncodeTiledFn encode, CUtensorMap* m, const void* base, int k, int rows, int64_t pitch,
                      int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)kBlock, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

struct Operands {
  const uint8_t *x, *w;
  int64_t x_pitch, w_pitch;
  int k;
};

template <typename T, int TN>
int launch_rows(const Operands& o, LinearParams& p, EncodeTiledFn encode, cudaStream_t s) {
  const int n_tiles = ceil_div(p.n, 128), t_tiles = ceil_div(p.rows, TN);
  MODIFF_CHECK_ARG(t_tiles <= 65535, "too many rows");
  CUtensorMap mw, mx;
  CUresult r = encode_codes(encode, &mw, o.w, o.k, p.n, o.w_pitch, 128);
  if (r == CUDA_SUCCESS) r = encode_codes(encode, &mx, o.x, o.k, p.rows, o.x_pitch, TN);
  if (r != CUDA_SUCCESS) return set_error(MODIFF_ERR_CUDA, "cuTensorMapEncodeTiled(fp8 operands) failed: %d", (int)r);
  // channels split over up to eight CTAs while the grid leaves SMs idle and every CTA keeps two blocks
  p.split = 1;
  while (p.split < 8 && (int64_t)n_tiles * t_tiles * p.split < device_sms() && p.kb >= 4 * p.split) p.split *= 2;
  constexpr int smem = rows_smem<TN>();
  static SmemLimit limit;
  MODIFF_CUDA(raise_smem_limit(fp8_linear_rows_kernel<T, TN>, smem, limit));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * p.split), (unsigned)t_tiles);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MODIFF_CUDA(cudaLaunchKernelEx(&cfg, fp8_linear_rows_kernel<T, TN>, mw, mx, p));
  return MODIFF_OK;
}

}  // namespace
}  // namespace modiff

using namespace modiff;

extern "C" int modiff_fp8_quantize(const void* x, int64_t x_pitch, int64_t rows, int k, int dtype, uint8_t* codes,
                                   int64_t code_pitch, float* scale, int64_t scale_pitch, void* stream) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(rows >= 0 && k > 0, "bad shape");
  if (rows == 0) return MODIFF_OK;
  MODIFF_CHECK_ARG(x && codes && scale, "NULL pointer argument");
  const int size = dtype_bytes(dtype), blocks = ceil_div(k, kBlock);
  MODIFF_CHECK_ARG(code_pitch >= k && code_pitch % 16 == 0 && (uintptr_t)codes % 16 == 0,
                   "rows of codes need 16-byte alignment and a pitch that is a multiple of 16");
  MODIFF_CHECK_ARG(scale_pitch >= blocks && (uintptr_t)scale % 4 == 0 && (uintptr_t)x % size == 0, "misaligned tensor");
  QuantParams p{x, x_pitch, codes, code_pitch, scale, scale_pitch, rows, rows * blocks, k, blocks};
  const int64_t grid = ceil_div64(p.items, 16);
  MODIFF_CHECK_ARG(grid <= 0x7fffffff, "too many rows");
  const bool vec = (((uintptr_t)x | (uintptr_t)(x_pitch * size)) & 15) == 0;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (vec)
      fp8_quantize_kernel<T, true><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(p);
    else
      fp8_quantize_kernel<T, false><<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>(p);
    MODIFF_LAUNCH_CHECK("fp8_quantize_kernel");
    return MODIFF_OK;
  });
}

extern "C" int modiff_fp8_pack_weight(const void* w, int64_t w_pitch, int n, int k, int dtype, uint8_t* codes,
                                      int64_t code_pitch, float* scale, int64_t scale_pitch, void* stream) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(n > 0 && k > 0, "bad shape");
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
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(rows >= 0 && k > 0 && n > 0, "bad shape");
  if (rows == 0) return MODIFF_OK;
  MODIFF_CHECK_ARG(codes && scale && w && w_scale && y, "NULL pointer argument");
  MODIFF_CHECK_ARG(code_pitch >= k && w_pitch >= k && ((code_pitch | w_pitch) & 15) == 0 &&
                       (((uintptr_t)codes | (uintptr_t)w) & 15) == 0,
                   "rows of codes need 16-byte alignment and a pitch that is a multiple of 16");
  const int kb = ceil_div(k, kBlock), size = dtype_bytes(dtype);
  MODIFF_CHECK_ARG(scale_pitch >= kb && w_scale_pitch >= kb && y_pitch >= n, "bad pitch");
  MODIFF_CHECK_ARG((((uintptr_t)scale | (uintptr_t)w_scale) & 3) == 0 &&
                       (((uintptr_t)y | (uintptr_t)bias) % size) == 0, "misaligned tensor");
  EncodeTiledFn encode = get_encode_fn();
  if (!encode) return set_error(MODIFF_ERR_UNSUPPORTED, "cuTensorMapEncodeTiled is not available");
  LinearParams p{scale, scale_pitch, w_scale, w_scale_pitch, bias, y, y_pitch, rows, n, kb, 1};
  const Operands o{codes, w, code_pitch, w_pitch, k};
  cudaStream_t s = (cudaStream_t)stream;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (rows <= 16) return launch_rows<T, 16>(o, p, encode, s);
    if (rows <= 32) return launch_rows<T, 32>(o, p, encode, s);
    if (rows <= 64) return launch_rows<T, 64>(o, p, encode, s);
    return launch_rows<T, 128>(o, p, encode, s);
  });
}
