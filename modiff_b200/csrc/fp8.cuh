// What the kernels of the 8-bit floating-point linear layers share.
#pragma once

#include "tc_common.cuh"
#include "types.cuh"

namespace modiff {

constexpr int kFp8Block = 128;              // channels (and weight rows) of one scale

struct Fp8Operands {
  const uint8_t *x, *w;                     // e4m3 codes, K-major
  int64_t x_pitch, w_pitch;
  int k;
};

struct Fp8Params {
  const float* sx;                          // [blocks][sx_pitch]: a block's scales of all rows in a row
  int64_t sx_pitch;
  const float* sw;                          // [ceil(n / 128)][sw_pitch]
  int64_t sw_pitch;
  const void* bias;                         // [n] or NULL
  void* y;
  int64_t y_pitch;
  int rows, n, kb, split;
  const void* x;                            // rows that a kernel quantises itself
  int64_t x_pitch;
  int k, x_vec, y_vec;
};

// Kernel for many rows (fp8_linear_pair.cu)
bool fp8_pair_wanted(int rows, int n);
int fp8_launch_pair(const Fp8Operands& o, const Fp8Params& p, int dtype, cudaStream_t s);

namespace {

// Instruction descriptor of kind::f8f6f4: e4m3 x e4m3 -> fp32, both operands K-major.
__host__ __device__ inline uint32_t make_idesc_e4m3(int m, int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
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
// acc += (a, b) * s, two fp32 multiply-adds in one instruction, each rounded as one
__device__ inline void fma_pair(uint64_t& acc, int a, int b, uint64_t s) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(a), "r"(b));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(v), "l"(s));
}

// Rows of codes as 2-D tiles of 128 channels by box_rows, 128-byte swizzle; zeros outside.
inline CUresult fp8_map(EncodeTiledFn encode, CUtensorMap* m, const void* base, int k, int rows, int64_t pitch,
                        int box_rows) {
  cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch};
  cuuint32_t box[2] = {(cuuint32_t)kFp8Block, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

}  // namespace
}  // namespace modiff
