// Writing and reading back a paged cache of keys and values held in 4 bits.
//
// A token's d channels of one head x have, in fp32 and rounded to fp16,
//   m = fp16(min x),  s = fp16((max x - min x) (1 / 15))      (a product with the fp32 number 1 / 15)
// and the codes round((x - m) / s) in 0 .. 15 (all 0 where s is 0); values beyond +-65504 count as
// +-65504, a NaN makes the whole row NaN.  Every step is one correctly rounded fp32 operation, so the
// bits are those of the same formula written with tensor operations.
//
// Layout: codes uint8 [page][head][offset][d / 2], channel 2i in the low and 2i + 1 in the high half of
// byte i; params fp16 [page][head][offset][2] = (s, m).  Position t of sequence b is at offset t %
// page_size of page table[b][t / page_size]; a page number outside the cache is not followed.
//
// Bound: HBM, one read of the new tokens and one write of d / 2 + 4 bytes per row, close behind it instruction
// issue; launch latency for a step of single tokens (4 us).  LANES lanes own a row, 8 channels each, of the key and
// of the value, in registers between the extremes and the codes.  4 x 2048 tokens of 8 heads of 128, fp16: 17.4 us,
// 2.5 TB/s (21.1 with extremes in fp32, 35.4 with the compiler's divisions and 64-bit indexes as well); reading
// them back as fp32 13.7 us, 5.5 TB/s, nearly all of it writes (20.5 with two accesses of a lane side by side).
#include <type_traits>

#include "kv4.cuh"

namespace modiff {
namespace {

constexpr int kThreads = 128;
constexpr int64_t kMostRows = 0x7fffffff - kThreads;   // rows of one call: their numbers are 32-bit

struct AppendParams {
  const void *k, *v;
  int64_t kb, kt, kh, vb, vt, vh;     // element strides: sequence, token, head
  Kv4Pages c;
  const int32_t* table;
  const int32_t* lengths;
  int count, max_pages, rows;         // batch * count * heads
  FastDiv by_heads, by_count;
};

// Smaller and larger of two numbers, a NaN if either is one.
__device__ inline float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ inline float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Extremes of a row whose channels LANES lanes hold eight each; 16-bit values two at a time, and between
// lanes both extremes as one word (the smaller of the values and of their negatives).
template <typename T, int LANES>
__device__ inline void extremes(const Pack<T, 8>& x, bool mine, float& low, float& high) {
  if constexpr (sizeof(T) == 4) {
    low = INFINITY; high = -INFINITY;
    if (mine) {
      low = high = x.v[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) { low = min_nan(low, x.v[e]); high = max_nan(high, x.v[e]); }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      low = min_nan(low, __shfl_xor_sync(0xffffffffu, low, o));
      high = max_nan(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
  } else {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* w = reinterpret_cast<const T2*>(x.v);
    T2 both;
    both.x = both.y = from_f32<T>(INFINITY);
    if (mine) {
      const T2 lo = __hmin2_nan(__hmin2_nan(w[0], w[1]), __hmin2_nan(w[2], w[3]));
      const T2 hi = __hneg2(__hmax2_nan(__hmax2_nan(w[0], w[1]), __hmax2_nan(w[2], w[3])));
      T2 a, b;
      a.x = lo.x; a.y = hi.x; b.x = lo.y; b.y = hi.y;
      both = __hmin2_nan(a, b);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) both = __hmin2_nan(both, __shfl_xor_sync(0xffffffffu, both, o));
    low = to_f32<T>(both.x);
    high = -to_f32<T>(both.y);
  }
}

// Eight values as codes; the scale and minimum of their row.
template <typename T, int LANES>
__device__ inline uint32_t encode(const Pack<T, 8>& in, bool mine, __half2& params) {
  float low, high;
  extremes<T, LANES>(in, mine, low, high);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(in.v[e]);
  if (low < -65504.0f || high > 65504.0f) {
    low = fminf(fmaxf(low, -65504.0f), 65504.0f);
    high = fminf(fmaxf(high, -65504.0f), 65504.0f);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
  }
  const __half s = __float2half_rn(__fmul_rn(__fsub_rn(high, low), 1.0f / 15.0f)), m = __float2half_rn(low);
  params = __halves2half2(s, m);
  const float sf = __half2float(s), mf = __half2float(m);
  if (!(sf > 0.0f)) return 0;
  // s is a fp16 number above 0: nothing under- or overflows where the code is not 0 anyway
  const float inv = __frcp_rn(sf);
  const uint64_t r = pack2(inv, inv), minus_s = pack2(-sf, -sf), minus_m = pack2(-mf, -mf);
  // adding 1.5 2^23 rounds to an integer, ties to even, and leaves it in the low bits
  const uint64_t bias = pack2(12582912.0f, 12582912.0f);
  uint32_t packed = 0;
#pragma unroll
  for (int e = 6; e >= 0; e -= 2) {
    const float2 d = unpack2(add2(pack2(x[e], x[e + 1]), minus_m));
    const float2 q = divide_pair(d.x, d.y, r, minus_s);
    const float2 n = unpack2(add2(pack2(fminf(fmaxf(q.x, 0.0f), 15.0f), fminf(fmaxf(q.y, 0.0f), 15.0f)), bias));
    packed = (packed << 4) + __float_as_uint(n.y);
    packed = (packed << 4) + __float_as_uint(n.x);
  }
  // what 0x4b400000 of each of the eight adds up to, modulo 2^32
  return packed - (0x4b400000u + 0xb4000000u + 0x40000000u);
}

template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv4_append_kernel(const AppendParams p) {
  const int lane = threadIdx.x % LANES;
  const int row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  bool live = row < p.rows;
  int head = 0, i = 0, b = 0;
  if (live) b = p.by_heads.divmod(p.by_count.divmod(row, i), head);
  const bool mine = live && 8 * lane < p.c.dim;
  Pack<T, 8> x[2];
  if (mine) {                         // on their way before the page number is known
    const T* src[2] = {static_cast<const T*>(p.k) + (b * p.kb + i * p.kt + head * p.kh) + 8 * lane,
                       static_cast<const T*>(p.v) + (b * p.vb + i * p.vt + head * p.vh) + 8 * lane};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (VEC) {
        x[u] = *reinterpret_cast<const Pack<T, 8>*>(src[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[u].v[e] = src[u][e];
      }
    }
  }
  int64_t place = -1;
  if (live)
    place = kv4_place(p.c, p.table + (int64_t)b * p.max_pages, p.max_pages, max(__ldg(p.lengths + b), 0) - p.count + i,
                      head);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    __half2 sm;
    const uint32_t packed = encode<T, LANES>(x[u], mine, sm);
    if (!mine || place < 0) continue;
    *reinterpret_cast<uint32_t*>((u ? p.c.v_codes : p.c.k_codes) + place * (p.c.dim / 2) + 4 * lane) = packed;
    if (lane == 0) reinterpret_cast<__half2*>(u ? p.c.v_params : p.c.k_params)[place] = sm;
  }
}

struct ReadParams {
  Kv4Pages c;
  const int32_t* table;
  const int32_t* lengths;
  void *k, *v;                        // [batch][count][heads][dim]
  int count, max_pages, rows;         // batch * count * heads
  FastDiv by_heads, by_count;
};

// A lane's stores are 16 bytes next to its neighbour's: eight channels of 16-bit values, four of fp32 twice.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const ReadParams p) {
  constexpr int E = 16 / sizeof(T), kPieces = 8 / E;
  using Codes = std::conditional_t<E == 8, uint32_t, uint16_t>;
  const int lane = threadIdx.x % LANES;
  const int row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  if (row >= p.rows) return;
  int head, i;
  const int b = p.by_heads.divmod(p.by_count.divmod(row, i), head);
  const int64_t place = kv4_place(p.c, p.table + (int64_t)b * p.max_pages, p.max_pages,
                                  max(__ldg(p.lengths + b), 0) - p.count + i, head);
  const int64_t to = (((int64_t)b * p.count + i) * p.c.heads + head) * p.c.dim;
  uint32_t w[2][kPieces] = {};
  float2 sm[2] = {};
  if (place >= 0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint8_t* codes = (u ? p.c.v_codes : p.c.k_codes) + place * (p.c.dim / 2);
#pragma unroll
      for (int q = 0; q < kPieces; ++q)
        if (const int c = (q * LANES + lane) * E; c < p.c.dim) w[u][q] = *reinterpret_cast<const Codes*>(codes + c / 2);
      sm[u] = __half22float2(reinterpret_cast<const __half2*>(u ? p.c.v_params : p.c.k_params)[place]);
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      const int c = (q * LANES + lane) * E;
      if (c >= p.c.dim) continue;
      float x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = fmaf((float)((w[u][q] >> (4 * e)) & 15u), sm[u].x, sm[u].y);
      store_f32<T, E>(static_cast<T*>(u ? p.v : p.k) + to + c, x);
    }
}

template <typename T, int LANES>
int launch_append(const AppendParams& p, bool vec, cudaStream_t s) {
  const unsigned blocks = (unsigned)ceil_div(p.rows, kThreads / LANES);
  if (vec)
    kv4_append_kernel<T, LANES, true><<<blocks, kThreads, 0, s>>>(p);
  else
    kv4_append_kernel<T, LANES, false><<<blocks, kThreads, 0, s>>>(p);
  MODIFF_LAUNCH_CHECK("kv4_append_kernel");
  return MODIFF_OK;
}

template <typename T, int LANES>
int launch_read(const ReadParams& p, cudaStream_t s) {
  kv4_read_kernel<T, LANES><<<(unsigned)ceil_div(p.rows, kThreads / LANES), kThreads, 0, s>>>(p);
  MODIFF_LAUNCH_CHECK("kv4_read_kernel");
  return MODIFF_OK;
}

}  // namespace

int kv4_check(const modiff_kv4_cache* c, const int32_t* table, const int32_t* lengths, int batch, int max_pages) {
  MODIFF_CHECK_ARG(c && c->k_codes && c->k_params && c->v_codes && c->v_params, "NULL cache pointer");
  MODIFF_CHECK_ARG(table && lengths, "NULL pointer argument");
  MODIFF_CHECK_ARG((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15) == 0 &&
                       (((uintptr_t)c->k_params | (uintptr_t)c->v_params) & 3) == 0 &&
                       (((uintptr_t)table | (uintptr_t)lengths) & 3) == 0,
                   "misaligned cache, table or lengths");
  MODIFF_CHECK_ARG(c->pages > 0 && c->heads > 0, "empty cache");
  MODIFF_CHECK_ARG(c->page_size > 0 && c->page_size % 16 == 0, "page size %d: a multiple of 16 is served",
                   c->page_size);
  MODIFF_CHECK_ARG(c->dim >= 64 && c->dim <= 256 && c->dim % 64 == 0,
                   "head width %d: 64, 128, 192 and 256 are served", c->dim);
  MODIFF_CHECK_ARG(batch >= 0 && max_pages > 0, "bad batch or table");
  MODIFF_CHECK_ARG((int64_t)max_pages * c->page_size <= 1 << 30, "table of more than 2^30 tokens");
  return MODIFF_OK;
}

Kv4Pages kv4_pages(const modiff_kv4_cache* c) {
  Kv4Pages p;
  p.k_codes = c->k_codes; p.v_codes = c->v_codes;
  p.k_params = c->k_params; p.v_params = c->v_params;
  p.pages = c->pages; p.heads = c->heads; p.page_size = c->page_size; p.dim = c->dim;
  p.by_page = FastDiv(c->page_size);
  return p;
}

}  // namespace modiff

using namespace modiff;

extern "C" int modiff_kv4_append(const modiff_kv4_cache* cache, const void* k, int64_t k_seq, int64_t k_token,
                                 int64_t k_head, const void* v, int64_t v_seq, int64_t v_token, int64_t v_head,
                                 const int32_t* table,
                                 const int32_t* lengths, int batch, int count, int max_pages, int dtype,
                                 void* stream) {
  int rc = kv4_check(cache, table, lengths, batch, max_pages);
  if (rc) return rc;
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(k && v, "NULL pointer argument");
  MODIFF_CHECK_ARG(count >= 0, "negative token count");
  if (batch == 0 || count == 0) return MODIFF_OK;
  AppendParams p;
  p.k = k; p.v = v;
  p.kb = k_seq; p.kt = k_token; p.kh = k_head;
  p.vb = v_seq; p.vt = v_token; p.vh = v_head;
  p.c = kv4_pages(cache);
  p.table = table; p.lengths = lengths;
  p.count = count; p.max_pages = max_pages;
  const int64_t rows = (int64_t)batch * count * cache->heads;
  MODIFF_CHECK_ARG((int64_t)batch * count <= kMostRows && rows <= kMostRows, "too many tokens");
  p.rows = (int)rows;
  p.by_heads = FastDiv(cache->heads);
  p.by_count = FastDiv(count);
  const int size = dtype_bytes(dtype);
  const uintptr_t align = (uintptr_t)k | (uintptr_t)v |
                          (uintptr_t)((p.kb | p.kt | p.kh | p.vb | p.vt | p.vh) * size);
  MODIFF_CHECK_ARG(align % size == 0, "misaligned tensor");
  const bool vec = align % 16 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (cache->dim == 64) return launch_append<T, 8>(p, vec, st);
    if (cache->dim == 128) return launch_append<T, 16>(p, vec, st);
    return launch_append<T, 32>(p, vec, st);
  });
}

extern "C" int modiff_kv4_read(const modiff_kv4_cache* cache, const int32_t* table, const int32_t* lengths,
                               int batch, int count, int max_pages, void* k, void* v, int dtype, void* stream) {
  int rc = kv4_check(cache, table, lengths, batch, max_pages);
  if (rc) return rc;
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(count >= 0, "negative token count");
  if (batch == 0 || count == 0) return MODIFF_OK;
  MODIFF_CHECK_ARG(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, "NULL or misaligned output");
  ReadParams p;
  p.c = kv4_pages(cache);
  p.table = table; p.lengths = lengths;
  p.k = k; p.v = v;
  p.count = count; p.max_pages = max_pages;
  const int64_t rows = (int64_t)batch * count * cache->heads;
  MODIFF_CHECK_ARG((int64_t)batch * count <= kMostRows && rows <= kMostRows, "too many tokens");
  p.rows = (int)rows;
  p.by_heads = FastDiv(cache->heads);
  p.by_count = FastDiv(count);
  cudaStream_t st = (cudaStream_t)stream;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    if (cache->dim == 64) return launch_read<T, 8>(p, st);
    if (cache->dim == 128) return launch_read<T, 16>(p, st);
    return launch_read<T, 32>(p, st);
  });
}
