// The paged 4-bit cache as kernels address it.
#pragma once

#include "types.cuh"

namespace modiff {

struct Kv4Pages {
  uint8_t *k_codes, *v_codes;      // [page][head][offset][dim / 2]
  uint16_t *k_params, *v_params;   // fp16 [page][head][offset][2]
  int pages, heads, page_size, dim;
  FastDiv by_page;
};

// One attention call over the cache, as its kernels take it.
struct Kv4Attention {
  const void* q;
  int64_t qb, qt, qh;                     // element strides: sequence, token, head
  void* out;                              // [batch][count][heads][dim]
  float* part;                            // [splits][rows][dim], then sums and maxima [splits][rows] each
  Kv4Pages c;
  const int32_t* table;
  const int32_t* lengths;
  int batch, count, heads, group, max_pages, splits, row_tiles;
  int causal, window, sinks;
  int q_vec;                              // rows of q start on 16 bytes
  FastDiv by_group;
  float scale2;                           // scale * log2(e)
  int64_t rows;                           // batch * count * heads
};

// Whether the tensor-core kernel for many query rows serves a call, and its launch (kv4_attention_tc.cu).
bool kv4_tc_wanted(int rows, int dim, int dtype);
int kv4_tc_rows();                    // query rows of one of its blocks
int kv4_launch_tc(const Kv4Attention& p, int dtype, cudaStream_t s);

int kv4_check(const modiff_kv4_cache* c, const int32_t* table, const int32_t* lengths, int batch, int max_pages);
Kv4Pages kv4_pages(const modiff_kv4_cache* c);

#ifdef __CUDACC__
// Row of a token in the cache's arrays, or -1: a position outside the table or a page number outside
// the cache is never followed.
__device__ inline int64_t kv4_place(const Kv4Pages& c, const int32_t* table_row, int max_pages, int at, int head) {
  if (at < 0) return -1;
  int offset;
  const int slot = c.by_page.divmod(at, offset);
  if (slot >= max_pages) return -1;
  const int page = __ldg(table_row + slot);
  if (page < 0 || page >= c.pages) return -1;
  return ((int64_t)page * c.heads + head) * c.page_size + offset;
}

namespace {

__device__ inline float exp2_fast(float x) {   // hardware exp2, relative error about 2^-22
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ inline uint32_t half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ inline float2 half_values(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

// pairs of fp32 values, one instruction for both
__device__ inline uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ inline float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ inline uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ inline uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ inline uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int BYTES>
__device__ inline void load_words(const uint8_t* src, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES % 16 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src) + i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
    for (int i = 0; i < BYTES / 8; ++i) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(src) + i);
      w[2 * i] = v.x; w[2 * i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(src) + i);
  }
}

// Tiles of TILE tokens that rows at positions [p_lo, p_hi] see any of: `first` tiles from 0 on (the
// sinks), the others from tile `start` on.
struct TileRange {
  int first, start, count;
  __device__ int tile(int i) const { return i < first ? i : start + (i - first); }
};
template <int TILE>
__device__ inline TileRange tiles_of(const Kv4Attention& p, int length, int p_lo, int p_hi) {
  TileRange r;
  const int end = p.causal ? min(length, p_hi + 1) : length;
  int lo = 0, sink_end = 0;
  if (p.window > 0) {
    lo = max(0, p_lo - p.window + 1);
    sink_end = min(min(p.sinks, lo), max(end, 0));
  }
  r.first = (sink_end + TILE - 1) / TILE;
  r.start = max(lo / TILE, r.first);
  const int last = end > 0 ? (end + TILE - 1) / TILE : 0;
  r.count = r.first + max(0, last - r.start);
  return r;
}

__device__ inline bool sees(const Kv4Attention& p, int t, int pos) {
  if (p.causal && t > pos) return false;
  return p.window <= 0 || t > pos - p.window || t < p.sinks;
}


}  // namespace
#endif

}  // namespace modiff
