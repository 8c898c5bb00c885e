// Root-mean-square norm of every head of the queries and keys, and the rotation of their positions,
// in one pass:
//   y = x / sqrt(mean(x^2) + eps) * w       over a head's d channels, in fp32
//   (a, b) -> (a cos - b sin, b cos + a sin)  for the pairs of its first 2 * half channels, pair i with
//   row `position` and column i of the tables; pairs are (i, half + i), or (2i, 2i + 1) interleaved;
// one rounding to the tensors' type at the end.
//
// Bound: HBM, every value read and written once.  A group of lanes owns one token's row of one head:
// a lane holds V pairs (two accesses of V elements), so that both members of a pair meet in one
// thread and only the sum of squares crosses lanes.  A group walks several heads of its token with
// the angles and weights in registers, loads of all of them issued first.  65536 tokens, 16 heads of 40, fp32:
// 69 us, 5.0 TB/s; one token 2.6 us.
#include "types.cuh"

namespace modiff {
namespace {

constexpr int kThreads = 128;

struct NormRopeSide {
  const void* x;
  void* y;
  int64_t x_token, x_head, y_token, y_head;   // element strides
  const float* w;                             // [d] or NULL
  int heads;
  FastDiv groups;                             // of `step` heads, per token
};

struct NormRopeParams {
  NormRopeSide q, k;
  const float* cos;
  const float* sin;
  const void* positions;     // int32 / int64 [tokens], or NULL: row = token
  int64_t tokens, table_rows;
  int items_q, items;
  int pos64, d, half, units, rot_units;
  float eps;
};

// STEP heads of one token per group of LANES lanes; a lane owns NU units of V pairs.
template <typename T, int V, int NU, int LANES, int STEP, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads)
qk_norm_rope_kernel(const NormRopeParams p) {
  const int lane = threadIdx.x % LANES;
  const int item = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool is_q = item < p.items_q;
  const NormRopeSide& s = is_q ? p.q : p.k;
  const bool live = item < p.items;
  int group = 0;
  const int64_t token = live ? s.groups.divmod(is_q ? item : item - p.items_q, group) : 0;
  const int head0 = group * STEP;
  const int heads = live ? min(STEP, s.heads - head0) : 0;

  int64_t row = token;
  if (p.positions && live)
    row = p.pos64 ? static_cast<const int64_t*>(p.positions)[token]
                  : (int64_t)static_cast<const int32_t*>(p.positions)[token];
  const bool inside = row >= 0 && row < p.table_rows;   // no row of the tables: the result is NaN

  int first[NU], second[NU];
  bool mine[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int unit = lane + u * LANES;
    mine[u] = unit < p.units;
    if (INTERLEAVED) {
      first[u] = 2 * V * unit;
      second[u] = first[u] + V;
    } else if (unit < p.rot_units) {
      first[u] = V * unit;
      second[u] = p.half + V * unit;
    } else {
      first[u] = 2 * p.half + 2 * V * (unit - p.rot_units);
      second[u] = first[u] + V;
    }
  }

  Pack<T, V> a[STEP][NU], b[STEP][NU];
  const T* x = static_cast<const T*>(s.x) + token * s.x_token + (int64_t)head0 * s.x_head;
#pragma unroll
  for (int h = 0; h < STEP; ++h)
#pragma unroll
    for (int u = 0; u < NU; ++u)
      if (h < heads && mine[u]) {
        a[h][u] = *reinterpret_cast<const Pack<T, V>*>(x + h * s.x_head + first[u]);
        b[h][u] = *reinterpret_cast<const Pack<T, V>*>(x + h * s.x_head + second[u]);
      }

  float co[NU][V], si[NU][V], wa[NU][V], wb[NU][V];
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    const int unit = lane + u * LANES;
#pragma unroll
    for (int i = 0; i < V; ++i) { co[u][i] = 1.0f; si[u][i] = 0.0f; wa[u][i] = wb[u][i] = 1.0f; }
    if (live && mine[u]) {
      if (unit < p.rot_units && inside) {
        load_f32<float, V>(p.cos + row * p.half + V * unit, co[u]);
        load_f32<float, V>(p.sin + row * p.half + V * unit, si[u]);
      }
      if (s.w) {
        load_f32<float, V>(s.w + first[u], wa[u]);
        load_f32<float, V>(s.w + second[u], wb[u]);
      }
    }
  }

  T* y = static_cast<T*>(s.y) + token * s.y_token + (int64_t)head0 * s.y_head;
#pragma unroll
  for (int h = 0; h < STEP; ++h) {
    float sum = 0.0f;
    if (h < heads) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
        if (mine[u]) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float f = to_f32<T>(a[h][u].v[i]), g = to_f32<T>(b[h][u].v[i]);
            sum = fmaf(f, f, sum);
            sum = fmaf(g, g, sum);
          }
        }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (h >= heads) continue;
    float rstd = 1.0f / sqrtf(sum / (float)p.d + p.eps);
    if (!inside) rstd = __int_as_float(0x7fc00000);
#pragma unroll
    for (int u = 0; u < NU; ++u)
      if (mine[u]) {
        float e[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          e[i] = to_f32<T>(a[h][u].v[i]) * rstd * wa[u][i];
          e[V + i] = to_f32<T>(b[h][u].v[i]) * rstd * wb[u][i];
        }
        Pack<T, V> ya, yb;
        if (INTERLEAVED) {
          float z[2 * V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            z[2 * i] = e[2 * i] * co[u][i] - e[2 * i + 1] * si[u][i];
            z[2 * i + 1] = e[2 * i + 1] * co[u][i] + e[2 * i] * si[u][i];
          }
#pragma unroll
          for (int i = 0; i < V; ++i) { ya.v[i] = from_f32<T>(z[i]); yb.v[i] = from_f32<T>(z[V + i]); }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ya.v[i] = from_f32<T>(e[i] * co[u][i] - e[V + i] * si[u][i]);
            yb.v[i] = from_f32<T>(e[V + i] * co[u][i] + e[i] * si[u][i]);
          }
        }
        *reinterpret_cast<Pack<T, V>*>(y + h * s.y_head + first[u]) = ya;
        *reinterpret_cast<Pack<T, V>*>(y + h * s.y_head + second[u]) = yb;
      }
  }
}

template <typename T, int V, int NU, int LANES, bool IL>
int launch(NormRopeParams& p, cudaStream_t stream) {
  constexpr int kGroups = kThreads / LANES;
  auto plan = [&](int step) -> int64_t {
    const int qg = p.q.heads ? ceil_div(p.q.heads, step) : 1, kg = p.k.heads ? ceil_div(p.k.heads, step) : 1;
    p.q.groups = FastDiv(qg);
    p.k.groups = FastDiv(kg);
    const int64_t items_q = p.q.heads ? p.tokens * qg : 0, items = items_q + (p.k.heads ? p.tokens * kg : 0);
    p.items_q = (int)items_q;
    p.items = (int)items;
    return items;
  };
  // Several heads of a token per group once every SM still gets eight blocks (32 + 8 heads of 128, bf16, us for one
  // : four heads a group: 300 tokens 3.6 : 4.2, 1000 tokens 7.3 : 6.7, 16000 tokens 92 : 73).
  constexpr int kStep = NU == 1 ? 4 : 1;
  const bool wide = kStep > 1 && plan(kStep) >= 8ll * device_sms() * kGroups;
  const int64_t items = plan(wide ? kStep : 1);
  MODIFF_CHECK_ARG(items <= 0x7fffffff - kGroups, "too many tokens");
  const unsigned blocks = (unsigned)ceil_div64(items, kGroups);
  if (wide)
    qk_norm_rope_kernel<T, V, NU, LANES, kStep, IL><<<blocks, kThreads, 0, stream>>>(p);
  else
    qk_norm_rope_kernel<T, V, NU, LANES, 1, IL><<<blocks, kThreads, 0, stream>>>(p);
  MODIFF_LAUNCH_CHECK("qk_norm_rope_kernel");
  return MODIFF_OK;
}

template <typename T, int V, bool IL>
int by_lanes(NormRopeParams& p, cudaStream_t s) {
  constexpr int kNu = V >= 4 ? 1 : (V == 2 ? 2 : 4);   // d <= 256: at most 128 / V units
  if (p.units <= 4) return launch<T, V, 1, 4, IL>(p, s);
  if (p.units <= 8) return launch<T, V, 1, 8, IL>(p, s);
  if (p.units <= 16) return launch<T, V, 1, 16, IL>(p, s);
  if (p.units <= 32) return launch<T, V, 1, 32, IL>(p, s);
  return launch<T, V, kNu, 32, IL>(p, s);
}

}  // namespace
}  // namespace modiff

using namespace modiff;

extern "C" int modiff_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, void* q_out, int64_t q_out_token,
                                   int64_t q_out_head, int q_heads, const void* k, int64_t k_token,
                                   int64_t k_head, void* k_out, int64_t k_out_token, int64_t k_out_head, int k_heads, const float* q_weight, const float* k_weight,
                                   const float* cos, const float* sin, int64_t table_rows,
                                   const void* positions, int positions64, int64_t tokens, int d,
                                   int rot, int interleaved, float eps, int dtype, void* stream) {
  MODIFF_CHECK_ARG(dtype_ok(dtype), "unknown element type %d", dtype);
  MODIFF_CHECK_ARG(tokens >= 0 && q_heads >= 0 && k_heads >= 0, "negative size");
  MODIFF_CHECK_ARG(d >= 2 && d <= 256 && d % 2 == 0, "head width %d: an even number up to 256 is served", d);
  MODIFF_CHECK_ARG(rot >= 0 && rot <= d && rot % 2 == 0, "rotated channels %d of %d", rot, d);
  MODIFF_CHECK_ARG(rot == 0 || (cos && sin), "NULL table");
  MODIFF_CHECK_ARG(q_heads == 0 || (q && q_out), "NULL pointer argument");
  MODIFF_CHECK_ARG(k_heads == 0 || (k && k_out), "NULL pointer argument");
  MODIFF_CHECK_ARG(positions || rot == 0 || table_rows >= tokens, "tables of %lld rows for %lld tokens",
                   (long long)table_rows, (long long)tokens);
  MODIFF_CHECK_ARG((uintptr_t)positions % (positions64 ? 8 : 4) == 0, "misaligned positions");
  if (tokens == 0 || q_heads + k_heads == 0) return MODIFF_OK;

  NormRopeParams p = {};
  p.q = NormRopeSide{q, q_out, q_token, q_head, q_out_token, q_out_head, q_weight, q_heads, FastDiv()};
  p.k = NormRopeSide{k, k_out, k_token, k_head, k_out_token, k_out_head, k_weight, k_heads, FastDiv()};
  p.cos = cos;
  p.sin = sin;
  p.positions = rot ? positions : nullptr;
  p.pos64 = positions64;
  p.tokens = tokens;
  p.table_rows = rot ? table_rows : tokens;
  p.d = d;
  p.half = rot / 2;
  p.eps = eps;

  // pairs per access: 16 bytes where widths, strides and addresses allow, else fewer
  const int size = dtype_bytes(dtype);
  uintptr_t align = 0;
  for (const NormRopeSide* s : {&p.q, &p.k})
    if (s->heads)
      align |= (uintptr_t)s->x | (uintptr_t)s->y |
               (uintptr_t)((s->x_token | s->x_head | s->y_token | s->y_head) * size);
  // tables and weights are read as v fp32 values at a time: at most 16 bytes each
  uintptr_t align4 = (uintptr_t)p.q.w | (uintptr_t)p.k.w;
  if (rot) align4 |= (uintptr_t)cos | (uintptr_t)sin;
  MODIFF_CHECK_ARG(align4 % 4 == 0, "misaligned table or weight");
  int v = 16 / size;
  while (v > 1 && (align4 % (v >= 4 ? 16 : 4 * v) != 0 || align % (v * size) != 0 || (interleaved ? rot % (2 * v) != 0 || d % (2 * v) != 0
                                                           : p.half % v != 0 || (d - rot) % (2 * v) != 0)))
    v /= 2;
  MODIFF_CHECK_ARG(align % size == 0, "misaligned tensor");
  p.units = d / 2 / v;
  p.rot_units = p.half / v;
  cudaStream_t st = (cudaStream_t)stream;
  return with_dtype(dtype, [&](auto tag) {
    using T = decltype(tag);
    auto go = [&](auto il) {
      constexpr bool IL = decltype(il)::value;
      if constexpr (sizeof(T) == 2) {
        if (v == 8) return by_lanes<T, 8, IL>(p, st);
      }
      if (v >= 4) return by_lanes<T, 4, IL>(p, st);
      if (v == 2) return by_lanes<T, 2, IL>(p, st);
      return by_lanes<T, 1, IL>(p, st);
    };
    return interleaved ? go(std::true_type()) : go(std::false_type());
  });
}
