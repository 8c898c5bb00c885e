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
// Bound: HBM, one read of the new tokens and one write of d / 2 + 4 bytes per row (and launch latency
// for a step of single tokens).  LANES lanes own a row, 8 channels each, in registers between the
// extremes and the codes.
#include "kv4.cuh"

namespace modiff {
namespace {

constexpr int kThreads = 256;

struct AppendParams {
  const void *k, *v;
  int64_t kb, kt, kh, vb, vt, vh;     // element strides: sequence, token, head
  Kv4Pages c;
  const int32_t* table;
  const int32_t* lengths;
  int batch, count, max_pages;
  int64_t rows;                       // batch * count * heads
};

template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(kThreads)
kv4_append_kernel(const AppendParams p) {
  const int lane = threadIdx.x % LANES;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool value = item >= p.rows;
  const int64_t row = value ? item - p.rows : item;
  bool live = row < p.rows;
  const int head = live ? (int)(row % p.c.heads) : 0;
  const int64_t bt = live ? row / p.c.heads : 0;
  const int i = (int)(bt % p.count), b = (int)(bt / p.count);
  const int at = live ? max(__ldg(p.lengths + b), 0) - p.count + i : -1;
  const int64_t place = kv4_place(p.c, p.table + (int64_t)b * p.max_pages, p.max_pages, at, head);
  live = live && place >= 0;
  const bool mine = live && 8 * lane < p.c.dim;

  float x[8];
  float low = INFINITY, high = -INFINITY;
  bool bad = false;
  if (mine) {
    const T* src = static_cast<const T*>(value ? p.v : p.k) +
                   (value ? b * p.vb + i * p.vt + head * p.vh : b * p.kb + i * p.kt + head * p.kh) + 8 * lane;
    if (VEC) {
      load_f32<T, 8>(src, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(src[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      bad |= isnan(x[e]);
      x[e] = fminf(fmaxf(x[e], -65504.0f), 65504.0f);
      low = fminf(low, x[e]);
      high = fmaxf(high, x[e]);
    }
  }
  int any = bad;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    any |= __shfl_xor_sync(0xffffffffu, any, o);
  }
  if (!mine) return;
  const __half s = __float2half_rn(any ? __int_as_float(0x7fc00000) : __fmul_rn(__fsub_rn(high, low), 1.0f / 15.0f));
  const __half m = __float2half_rn(any ? __int_as_float(0x7fc00000) : low);
  const float sf = __half2float(s), mf = __half2float(m);
  uint32_t packed = 0;
  if (sf > 0.0f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], mf), sf)), 0.0f), 15.0f);
      packed |= (uint32_t)q << (4 * e);
    }
  }
  uint8_t* codes = value ? p.c.v_codes : p.c.k_codes;
  *reinterpret_cast<uint32_t*>(codes + place * (p.c.dim / 2) + 4 * lane) = packed;
  if (lane == 0) {
    __half2* params = reinterpret_cast<__half2*>(value ? p.c.v_params : p.c.k_params);
    params[place] = __halves2half2(s, m);
  }
}

struct ReadParams {
  Kv4Pages c;
  const int32_t* table;
  const int32_t* lengths;
  void *k, *v;                        // [batch][count][heads][dim]
  int batch, count, max_pages;
  int64_t items;                      // batch * count * heads * dim / 8
};

template <typename T>
__global__ void __launch_bounds__(kThreads)
kv4_read_kernel(const ReadParams p) {
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (item >= 2 * p.items) return;
  const bool value = item >= p.items;
  const int64_t local = value ? item - p.items : item;
  const int chunks = p.c.dim / 8;
  const int chunk = (int)(local % chunks);
  const int64_t row = local / chunks;
  const int head = (int)(row % p.c.heads);
  const int64_t bt = row / p.c.heads;
  const int i = (int)(bt % p.count), b = (int)(bt / p.count);
  const int at = max(__ldg(p.lengths + b), 0) - p.count + i;
  const int64_t place = kv4_place(p.c, p.table + (int64_t)b * p.max_pages, p.max_pages, at, head);
  float x[8] = {};
  if (place >= 0) {
    const uint8_t* codes = value ? p.c.v_codes : p.c.k_codes;
    const __half2* params = reinterpret_cast<const __half2*>(value ? p.c.v_params : p.c.k_params);
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + place * (p.c.dim / 2) + 4 * chunk);
    const float2 sm = __half22float2(params[place]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((w >> (4 * e)) & 15u), sm.x, sm.y);
  }
  store_f32<T, 8>(static_cast<T*>(value ? p.v : p.k) + row * p.c.dim + 8 * chunk, x);
}

template <typename T, int LANES>
int launch_append(const AppendParams& p, bool vec, cudaStream_t s) {
  const int64_t blocks = ceil_div64(2 * p.rows, kThreads / LANES);
  MODIFF_CHECK_ARG(blocks <= 0x7fffffff, "too many tokens");
  if (vec)
    kv4_append_kernel<T, LANES, true><<<(unsigned)blocks, kThreads, 0, s>>>(p);
  else
    kv4_append_kernel<T, LANES, false><<<(unsigned)blocks, kThreads, 0, s>>>(p);
  MODIFF_LAUNCH_CHECK("kv4_append_kernel");
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
  p.batch = batch; p.count = count; p.max_pages = max_pages;
  p.rows = (int64_t)batch * count * cache->heads;
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
  p.batch = batch; p.count = count; p.max_pages = max_pages;
  p.items = (int64_t)batch * count * cache->heads * (cache->dim / 8);
  const int64_t blocks = ceil_div64(2 * p.items, kThreads);
  MODIFF_CHECK_ARG(blocks <= 0x7fffffff, "too many tokens");
  return with_dtype(dtype, [&](auto tag) {
    kv4_read_kernel<decltype(tag)><<<(unsigned)blocks, kThreads, 0, (cudaStream_t)stream>>>(p);
    MODIFF_LAUNCH_CHECK("kv4_read_kernel");
    return MODIFF_OK;
  });
}
