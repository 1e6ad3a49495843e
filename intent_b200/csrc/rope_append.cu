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
// Bound by instructions before it is bound by HBM, so a row costs few of them.  It is held by D / (2 PIECE) lanes in two pieces;
// with pairs (i, i + R/2) the pieces of a rotated lane lie R/2 apart, so that both elements of a pair and their angle are in one
// lane and nothing but the norm's sum is exchanged.  Several rows of one kind (queries, keys, values) of one token share what does
// not depend on the row: weight times cosine and weight times sine, worked out once, turn a row into two packed operations per
// two elements, one more scales it by the norm.  Calls of few rows take one row per group of lanes, as there the latency counts
// (64 tokens alone: 13.0 us, with four rows 14.2).
//
// Measured on one B200: append of 8192 tokens, 32 + 8 + 8 heads of 128, norm, bf16: 42.5 us, 4.8 TB/s (with the angles read for
// every row 66; pieces of eight elements 45; two rows per group 45, eight 42); 6001 tokens, heads of 64, no norm, f16: 11.2 us.
// One token, 6.4 us, is the host's time for a call.
#include "common.cuh"
#include "rotate.cuh"

namespace ib200 {
namespace {

template <typename T, int D, bool NORM, bool NEIGHBOURS, bool CACHE, int ROWS>
__global__ void __launch_bounds__(ROTATE_THREADS) rotate_kernel(const RotateParams p) {
  programmatic_begin();
  rotate_rows<T, D, NORM, NEIGHBOURS, CACHE, ROWS>(p, blockIdx.x);
}

template <typename T, int D, bool NORM, bool CACHE, int ROWS>
int launch(const RotateParams& p, bool neighbours, cudaStream_t stream) {
  constexpr uint32_t PER_CTA = ROTATE_THREADS / (D / (2 * PIECE_OF));
  auto kernel = neighbours ? rotate_kernel<T, D, NORM, true, CACHE, ROWS> : rotate_kernel<T, D, NORM, false, CACHE, ROWS>;
  const uint32_t groups = (p.q_heads + ROWS - 1) / ROWS + (CACHE ? 2 : 1) * ((p.k_heads + ROWS - 1) / ROWS);
  const uint32_t grid = (p.tokens * groups + PER_CTA - 1) / PER_CTA;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel),
                         ROWS == 1 ? "rotate_kernel a row per group" : "rotate_kernel several rows per group", int(grid), ROTATE_THREADS, 0, 1);
  const cudaError_t e = launch_programmatic(kernel, dim3(grid), dim3(ROTATE_THREADS), 0, stream, 1, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

template <typename T, bool CACHE>
int choose(const RotateParams& p, int64_t dim, bool neighbours, cudaStream_t stream) {
  const bool many = p.tokens * (p.q_heads + (CACHE ? 2 : 1) * p.k_heads) >= MANY;
#define IB200_ROTATE(D_, NORM_)                                                        \
  (many ? launch<T, D_, NORM_, CACHE, SHARED_ROWS>(p, neighbours, stream)              \
        : launch<T, D_, NORM_, CACHE, 1>(p, neighbours, stream))
  if (p.q_weight) return dim == 128 ? IB200_ROTATE(128, true) : IB200_ROTATE(64, true);
  return dim == 128 ? IB200_ROTATE(128, false) : IB200_ROTATE(64, false);
#undef IB200_ROTATE
}

template <typename T>
int norm_rope(const View3& q, const View3& k, const View1& positions, const View2& rotary, const View1* q_weight,
              const View1* k_weight, const View3& q_out, const View3& k_out, int32_t eps_bits, int32_t pairs,
              cudaStream_t stream) {
  RotateParams p = {};
  int status = rotate_prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
  if (status != INTENT_B200_OK) return status;
  if (k_out.d0 != k.d0 || k_out.d1 != k.d1 || k_out.d2 != k.d2) return INTENT_B200_ERR_SHAPE;
  if (!contiguous(k_out) || !aligned16(k_out.p)) return INTENT_B200_ERR_LAYOUT;
  if ((status = rotate_set_rows(p, q.d0, q.d1 + k.d1)) != INTENT_B200_OK) return status;
  if (p.tokens == 0) return INTENT_B200_OK;
  if (!k_out.p) return INTENT_B200_ERR_NULL;
  p.k_out = static_cast<uint16_t*>(k_out.p);
  return choose<T, false>(p, q.d2, pairs, stream);
}

template <typename T>
int append(const View3& q, const View3& k, const View3& v, const View1& positions, const View1& slots, const View2& rotary,
           const View1* q_weight, const View1* k_weight, const View4& k_cache, const View4& v_cache, const View3& q_out,
           int32_t eps_bits, int32_t pairs, cudaStream_t stream) {
  RotateParams p = {};
  int status = rotate_prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
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
  if ((status = rotate_set_rows(p, q.d0, q.d1 + 2 * k.d1)) != INTENT_B200_OK) return status;
  if (p.tokens == 0) return INTENT_B200_OK;
  if (!v.p || !slots.p || (k_cache.d0 > 0 && (!k_cache.p || !v_cache.p))) return INTENT_B200_ERR_NULL;
  p.v = static_cast<const uint16_t*>(v.p);
  p.v_token = v.s0, p.v_head = v.s1;
  p.slots = static_cast<const int64_t*>(slots.p);
  p.k_out = static_cast<uint16_t*>(k_cache.p);
  p.v_out = static_cast<uint16_t*>(v_cache.p);
  p.slot_count = k_cache.d0 * page;
  while ((int64_t(1) << p.page_shift) < page) ++p.page_shift;
  return choose<T, true>(p, q.d2, pairs, stream);
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
