// Norms of queries and keys per head with the rotation by position in the same pass, and the append of keys and values to
// a paged cache.
//
// Programs (a head's row x of D elements, token t at position p = positions[t], rotary[p] = cos | sin of R / 2 angles each):
//   qk_norm_rope      q_out = rotate(norm(q), p), k_out = rotate(norm(k), p)
//   paged_kv_append   q_out = rotate(norm(q), p); k_cache[page, h, i] = rotate(norm(k), p) and v_cache[page, h, i] = v at
//                     slots[t] = page * PAGE + i
//   norm(x) = x / sqrt(mean(x^2) + eps) * weight (the _norm entries; the others leave it out)
//   rotate  pairs (i, i + R/2) or (2i, 2i + 1) of the first R elements: a cos - b sin, b cos + a sin
//
// All sums and products are in f32 and every result is rounded once.  A token whose slot is outside the cache (-1: padding)
// is not stored; one whose position is outside the table gets NaN, as there is no angle for it.
//
// A row is held by D / 8 lanes, 16 bytes each: the norm is one sum over them, and the partner of a pair (i, i + R/2) lies
// R / 16 lanes away in the same group, so a row is read once, and all that leaves the registers is the result.
#include <cstring>

#include "common.cuh"

namespace ib200 {
namespace {

constexpr int THREADS = 256;

struct RotateParams {
  const uint16_t *q, *k, *v;
  const int32_t* positions;
  const int64_t* slots;
  const float* rotary;
  const uint16_t *q_weight, *k_weight;
  uint16_t *q_out, *k_out;             // k_out: [T, HK, D], or the key cache
  uint16_t* v_out;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;   // strides in elements
  int64_t table_rows, slot_count;
  uint32_t rows;                       // T * heads of a token
  uint32_t heads, q_heads, k_heads;    // of a token: queries, keys (and values)
  int rotary_dim, page_shift;
  float eps;
};

// Eight 16-bit elements as floats and back
template <typename T>
__device__ __forceinline__ void widen(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = Elem<T>::to_float(uint16_t(w[i]));
    x[2 * i + 1] = Elem<T>::to_float(uint16_t(w[i] >> 16));
  }
}
template <typename T>
__device__ __forceinline__ uint4 narrow(const float (&x)[8]) {
  return make_uint4(Elem<T>::pack2(x[0], x[1]), Elem<T>::pack2(x[2], x[3]), Elem<T>::pack2(x[4], x[5]),
                    Elem<T>::pack2(x[6], x[7]));
}

template <typename T, int D, bool NORM, bool NEIGHBOURS, bool CACHE>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const RotateParams p) {
  constexpr int LANES = D / 8;                       // of a row
  programmatic_begin();
  const int lane = threadIdx.x & 31, chunk = lane % LANES;
  const uint32_t at = blockIdx.x * uint32_t(THREADS / LANES) + threadIdx.x / LANES;
  const bool live = at < p.rows;                     // (all lanes stay for the exchanges)
  const uint32_t token = live ? at / p.heads : 0, head = live ? at - token * p.heads : 0;
  const bool is_q = head < p.q_heads, is_v = CACHE && head >= p.q_heads + p.k_heads;
  const uint32_t h = is_q ? head : head - p.q_heads - (is_v ? p.k_heads : 0);
  const uint16_t* row = is_q   ? p.q + token * p.q_token + h * p.q_head
                        : is_v ? p.v + token * p.v_token + h * p.v_head
                               : p.k + token * p.k_token + h * p.k_head;
  programmatic_wait();
  const uint4 raw = live ? ldg_stream_v4(row + 8 * chunk) : make_uint4(0, 0, 0, 0);
  const int64_t position = __ldg(p.positions + token);
  const bool known = position >= 0 && position < p.table_rows;
  const float* angles = p.rotary + (known ? position : 0) * p.rotary_dim;
  const int half = p.rotary_dim / 2, first = 8 * chunk;
  const bool turned = known && !is_v && first < p.rotary_dim;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  if (turned) {
    // angles of this lane's pairs: eight from its place in its half on, or those of four neighbours
    const int from = NEIGHBOURS ? first / 2 : first < half ? first : first - half;
#pragma unroll
    for (int i = 0; i < (NEIGHBOURS ? 4 : 8); i += 4) {
      const float4 cc = __ldg(reinterpret_cast<const float4*>(angles + from + i));
      const float4 ss = __ldg(reinterpret_cast<const float4*>(angles + half + from + i));
      c[i] = cc.x, c[i + 1] = cc.y, c[i + 2] = cc.z, c[i + 3] = cc.w;
      s[i] = ss.x, s[i + 1] = ss.y, s[i + 2] = ss.z, s[i + 3] = ss.w;
    }
  }
  float x[8];
  widen<T>(raw, x);
  if (NORM) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (!is_v) {
      const float scale = rsqrtf(sum * (1.f / D) + p.eps);
      float w[8];
      widen<T>(__ldg(reinterpret_cast<const uint4*>((is_q ? p.q_weight : p.k_weight) + first)), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * scale * w[i];
    }
  }
  float y[8];
  if (NEIGHBOURS) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
      y[2 * i + 1] = x[2 * i + 1] * c[i] + x[2 * i] * s[i];
    }
  } else {
    const int step = half / 8;                       // lanes between the halves of a pair
    const int partner = first < half ? lane + step : lane - step;
    const float sign = first < half ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_sync(0xffffffffu, x[i], turned ? partner : lane);
      y[i] = turned ? x[i] * c[i] + sign * (other * s[i]) : x[i];
    }
  }
  if (!known && !is_v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __int_as_float(0x7fc00000);
  }
  if (!live) return;
  const uint4 out = is_v ? raw : narrow<T>(y);
  if (is_q || !CACHE) {
    uint16_t* to = is_q ? p.q_out + (size_t(token) * p.q_heads + h) * D : p.k_out + (size_t(token) * p.k_heads + h) * D;
    *reinterpret_cast<uint4*>(to + first) = out;
    return;
  }
  const int64_t slot = __ldg(p.slots + token);
  if (slot < 0 || slot >= p.slot_count) return;
  const int64_t page = slot >> p.page_shift, inside = slot & ((int64_t(1) << p.page_shift) - 1);
  uint16_t* to = (is_v ? p.v_out : p.k_out) + (((page * p.k_heads + h) << p.page_shift) + inside) * D;
  *reinterpret_cast<uint4*>(to + first) = out;
}

template <typename T, int D, bool NORM, bool CACHE>
int launch(const RotateParams& p, bool neighbours, cudaStream_t stream) {
  constexpr uint32_t PER_CTA = THREADS / (D / 8);
  auto kernel = neighbours ? rotate_kernel<T, D, NORM, true, CACHE> : rotate_kernel<T, D, NORM, false, CACHE>;
  const uint32_t grid = (p.rows + PER_CTA - 1) / PER_CTA;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel), CACHE ? "rotate_kernel into pages" : "rotate_kernel",
                         int(grid), THREADS, 0, 1);
  const cudaError_t e = launch_programmatic(kernel, dim3(grid), dim3(THREADS), 0, stream, 1, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

// Checks what both programs share and fills the parameters in.
int prepare(RotateParams& p, const View3& q, const View3& k, const View1& positions, const View2& rotary, const View3& q_out,
            const View1* q_weight, const View1* k_weight, int32_t eps_bits, int32_t pairs) {
  const int64_t T = q.d0, D = q.d2;
  if (T < 0 || q.d1 <= 0 || k.d1 <= 0 || k.d0 != T || k.d2 != D || positions.d0 != T || q_out.d0 != T || q_out.d1 != q.d1 ||
      q_out.d2 != D)
    return INTENT_B200_ERR_SHAPE;
  if (D != 64 && D != 128) return INTENT_B200_ERR_UNSUPPORTED;
  if (rotary.d1 < 16 || rotary.d1 > D || rotary.d1 % 16 != 0 || pairs < 0 || pairs > 1) return INTENT_B200_ERR_UNSUPPORTED;
  if (!rows16(q) || !rows16(k) || !contiguous(positions) || !contiguous(rotary) || !contiguous(q_out))
    return INTENT_B200_ERR_LAYOUT;
  if (!aligned16(q.p) || !aligned16(k.p) || !aligned16(rotary.p) || !aligned16(q_out.p)) return INTENT_B200_ERR_LAYOUT;
  if (T > 0 && (!q.p || !k.p || !positions.p || !q_out.p || (!rotary.p && rotary.d0 > 0))) return INTENT_B200_ERR_NULL;
  if (q_weight) {
    if (q_weight->d0 != D || k_weight->d0 != D) return INTENT_B200_ERR_SHAPE;
    if (!contiguous(*q_weight) || !contiguous(*k_weight) || !aligned16(q_weight->p) || !aligned16(k_weight->p))
      return INTENT_B200_ERR_LAYOUT;
    if (!q_weight->p || !k_weight->p) return INTENT_B200_ERR_NULL;
    p.q_weight = static_cast<const uint16_t*>(q_weight->p);
    p.k_weight = static_cast<const uint16_t*>(k_weight->p);
  }
  p.q = static_cast<const uint16_t*>(q.p);
  p.k = static_cast<const uint16_t*>(k.p);
  p.positions = static_cast<const int32_t*>(positions.p);
  p.rotary = static_cast<const float*>(rotary.p);
  p.q_out = static_cast<uint16_t*>(q_out.p);
  p.q_token = q.s0, p.q_head = q.s1, p.k_token = k.s0, p.k_head = k.s1;
  p.table_rows = rotary.d0;
  p.rotary_dim = int(rotary.d1);
  p.q_heads = uint32_t(q.d1), p.k_heads = uint32_t(k.d1);
  std::memcpy(&p.eps, &eps_bits, sizeof(float));
  return INTENT_B200_OK;
}

int count_rows(RotateParams& p, int64_t tokens, int64_t heads) {
  if (heads > (1 << 20) || tokens > ((int64_t(1) << 31) - 1) / heads) return INTENT_B200_ERR_UNSUPPORTED;
  p.heads = uint32_t(heads);
  p.rows = uint32_t(tokens * heads);
  return INTENT_B200_OK;
}

template <typename T>
int norm_rope(const View3& q, const View3& k, const View1& positions, const View2& rotary, const View1* q_weight,
              const View1* k_weight, const View3& q_out, const View3& k_out, int32_t eps_bits, int32_t pairs,
              cudaStream_t stream) {
  RotateParams p = {};
  int status = prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
  if (status != INTENT_B200_OK) return status;
  if (k_out.d0 != k.d0 || k_out.d1 != k.d1 || k_out.d2 != k.d2) return INTENT_B200_ERR_SHAPE;
  if (!contiguous(k_out) || !aligned16(k_out.p)) return INTENT_B200_ERR_LAYOUT;
  if ((status = count_rows(p, q.d0, q.d1 + k.d1)) != INTENT_B200_OK) return status;
  if (p.rows == 0) return INTENT_B200_OK;
  if (!k_out.p) return INTENT_B200_ERR_NULL;
  p.k_out = static_cast<uint16_t*>(k_out.p);
  if (q_weight) return q.d2 == 128 ? launch<T, 128, true, false>(p, pairs, stream) : launch<T, 64, true, false>(p, pairs, stream);
  return q.d2 == 128 ? launch<T, 128, false, false>(p, pairs, stream) : launch<T, 64, false, false>(p, pairs, stream);
}

template <typename T>
int append(const View3& q, const View3& k, const View3& v, const View1& positions, const View1& slots, const View2& rotary,
           const View1* q_weight, const View1* k_weight, const View4& k_cache, const View4& v_cache, const View3& q_out,
           int32_t eps_bits, int32_t pairs, cudaStream_t stream) {
  RotateParams p = {};
  int status = prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
  if (status != INTENT_B200_OK) return status;
  const int64_t page = k_cache.d2;
  if (v.d0 != k.d0 || v.d1 != k.d1 || v.d2 != k.d2 || slots.d0 != q.d0 || k_cache.d0 < 0 || k_cache.d1 != k.d1 ||
      k_cache.d3 != k.d2 || v_cache.d0 != k_cache.d0 || v_cache.d1 != k_cache.d1 || v_cache.d2 != page || v_cache.d3 != k_cache.d3)
    return INTENT_B200_ERR_SHAPE;
  if (page < 16 || page > 256 || (page & (page - 1)) != 0 || k_cache.d0 > (int64_t(1) << 40) / page)
    return INTENT_B200_ERR_UNSUPPORTED;
  if (!rows16(v) || !contiguous(slots) || !contiguous(k_cache) || !contiguous(v_cache) || !aligned16(v.p) ||
      !aligned16(k_cache.p) || !aligned16(v_cache.p))
    return INTENT_B200_ERR_LAYOUT;
  if ((status = count_rows(p, q.d0, q.d1 + 2 * k.d1)) != INTENT_B200_OK) return status;
  if (p.rows == 0) return INTENT_B200_OK;
  if (!v.p || !slots.p || (k_cache.d0 > 0 && (!k_cache.p || !v_cache.p))) return INTENT_B200_ERR_NULL;
  p.v = static_cast<const uint16_t*>(v.p);
  p.v_token = v.s0, p.v_head = v.s1;
  p.slots = static_cast<const int64_t*>(slots.p);
  p.k_out = static_cast<uint16_t*>(k_cache.p);
  p.v_out = static_cast<uint16_t*>(v_cache.p);
  p.slot_count = k_cache.d0 * page;
  while ((int64_t(1) << p.page_shift) < page) ++p.page_shift;
  if (q_weight) return q.d2 == 128 ? launch<T, 128, true, true>(p, pairs, stream) : launch<T, 64, true, true>(p, pairs, stream);
  return q.d2 == 128 ? launch<T, 128, false, true>(p, pairs, stream) : launch<T, 64, false, true>(p, pairs, stream);
}

}  // namespace
}  // namespace ib200

#define IB200_ROTATE_ENTRIES(NAME, TYPE)                                                                                   \
  extern "C" int intent_b200_qk_rope_##NAME(INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW1(a2),           \
                                            INTENT_B200_VIEW2(a3), INTENT_B200_VIEW3(a4), INTENT_B200_VIEW3(a5),           \
                                            int32_t pairs, void* stream) {                                                 \
    return ib200::norm_rope<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW1_ARG(a2), IB200_VIEW2_ARG(a3),      \
                                  nullptr, nullptr, IB200_VIEW3_ARG(a4), IB200_VIEW3_ARG(a5), 0, pairs,                    \
                                  static_cast<cudaStream_t>(stream));                                                      \
  }                                                                                                                        \
  extern "C" int intent_b200_qk_norm_rope_##NAME(INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW1(a2),      \
                                                 INTENT_B200_VIEW2(a3), INTENT_B200_VIEW1(a4), INTENT_B200_VIEW1(a5),      \
                                                 INTENT_B200_VIEW3(a6), INTENT_B200_VIEW3(a7), int32_t eps_bits,           \
                                                 int32_t pairs, void* stream) {                                            \
    const ib200::View1 qw = IB200_VIEW1_ARG(a4), kw = IB200_VIEW1_ARG(a5);                                                 \
    return ib200::norm_rope<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW1_ARG(a2), IB200_VIEW2_ARG(a3), &qw, \
                                  &kw, IB200_VIEW3_ARG(a6), IB200_VIEW3_ARG(a7), eps_bits, pairs,                          \
                                  static_cast<cudaStream_t>(stream));                                                      \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_kv_append_##NAME(                                                                       \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW4(a6), INTENT_B200_VIEW4(a7), INTENT_B200_VIEW3(a8), int32_t pairs,           \
      void* stream) {                                                                                                      \
    return ib200::append<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),         \
                               IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), nullptr, nullptr, IB200_VIEW4_ARG(a6),            \
                               IB200_VIEW4_ARG(a7), IB200_VIEW3_ARG(a8), 0, pairs, static_cast<cudaStream_t>(stream));     \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_kv_append_norm_##NAME(                                                                  \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW1(a6), INTENT_B200_VIEW1(a7), INTENT_B200_VIEW4(a8), INTENT_B200_VIEW4(a9),   \
      INTENT_B200_VIEW3(a10), int32_t eps_bits, int32_t pairs, void* stream) {                                             \
    const ib200::View1 qw = IB200_VIEW1_ARG(a6), kw = IB200_VIEW1_ARG(a7);                                                 \
    return ib200::append<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),         \
                               IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), &qw, &kw, IB200_VIEW4_ARG(a8),                    \
                               IB200_VIEW4_ARG(a9), IB200_VIEW3_ARG(a10), eps_bits, pairs,                                 \
                               static_cast<cudaStream_t>(stream));                                                         \
  }
IB200_ROTATE_ENTRIES(f16, __half)
IB200_ROTATE_ENTRIES(bf16, __nv_bfloat16)
