// Norms of queries and keys per head with the rotation by position in the same pass, and the append of keys and values to
// a paged cache.
//
// Programs (a head's row x of D elements, token t at position p = positions[t], rotary[p] = cos | sin of R / 2 angles each):
//   qk_norm_rope      q_out = rotate(norm(q), p), k_out = rotate(norm(k), p)
//   paged_kv_append   q_out = rotate(norm(q), p); k_cache[page, h, i] = rotate(norm(k), p) and v_cache[page, h, i] = v at
//                     slots[t] = page * PAGE + i
//   norm(x) = x / sqrt(mean(x^2) + eps) * weight (the _norm entries; the others leave it out)
//   rotate  pairs (i, i + R/2) or (2i, 2i + 1) of the first R elements: a cos - b sin, b cos + a sin
//   paged_kv_append_int4   the same with a cache in 4 bits: keys, not rounded before, and values in groups of GROUP elements as
//                          m + s n:  m = min and s = (max - min) / 15, rounded to the type,  n = nearest((x - m) / s) in 0 .. 15
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
#include <cstring>

#include "common.cuh"
#include "paged.cuh"

namespace ib200 {
namespace {

constexpr int THREADS = 256;
constexpr int PIECE_OF = 4;             // elements of a lane's piece of a row, of which it has two
constexpr int SHARED_ROWS = 4;          // rows of a group in calls of many rows
constexpr uint32_t MANY = 20000;        // rows from which on a call has many

struct RotateParams {
  const uint16_t *q, *k, *v;
  const int32_t* positions;
  const int64_t* slots;
  const float* rotary;
  const uint16_t *q_weight, *k_weight;
  uint16_t *q_out, *k_out;             // k_out: [T, HK, D], or the key cache
  uint16_t* v_out;
  uint32_t *k_codes, *v_codes;         // caches in 4 bits: eight codes a word
  uint32_t *k_scales, *v_scales;       // and scale | minimum of every group
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;   // strides in elements
  int64_t table_rows, slot_count;
  uint32_t tokens, q_heads, k_heads;                           // k_heads: keys' and values'
  int rotary_dim, page_shift;
  float eps;
};

struct float8 {
  float v[8];
};

// A piece of a row: PIECE 16-bit elements
template <int PIECE>
struct Piece {
  uint32_t w[PIECE / 2];
};
template <int PIECE, bool STREAM>
__device__ __forceinline__ Piece<PIECE> load_piece(const uint16_t* from) {
  Piece<PIECE> d;
  if constexpr (PIECE == 8) {
    const uint4 v = STREAM ? ldg_stream_v4(from) : __ldg(reinterpret_cast<const uint4*>(from));
    d.w[0] = v.x, d.w[1] = v.y, d.w[2] = v.z, d.w[3] = v.w;
  } else {
    const uint2 v = STREAM ? ldg_stream_v2(from) : __ldg(reinterpret_cast<const uint2*>(from));
    d.w[0] = v.x, d.w[1] = v.y;
  }
  return d;
}
template <int PIECE>
__device__ __forceinline__ void store_piece(uint16_t* to, const Piece<PIECE>& v) {
  if constexpr (PIECE == 8) *reinterpret_cast<uint4*>(to) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  else *reinterpret_cast<uint2*>(to) = make_uint2(v.w[0], v.w[1]);
}

__device__ __forceinline__ float least(float a, float b) {      // NaN if any is
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float largest(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// Eight neighbouring elements of a row, which has D / 8 lanes, as codes; `scales`: scale | minimum of their group.  The codes are those
// of a division rounded to f32: the quotient by the rounded reciprocal gets its remainder added (P. Markstein, Computation of
// elementary functions on the IBM RISC System/6000 processor, 1990), so halves, which are common among 16-bit values, go to
// the even code.  A group with something that is no finite number is NaN.
template <typename T, int GROUP>
__device__ __forceinline__ uint32_t quantise(const float (&x)[8], uint32_t& scales) {
  float low = x[0], high = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) low = least(low, x[e]), high = largest(high, x[e]);
#pragma unroll
  for (int d = 1; d < GROUP / 8; d *= 2) {
    low = least(low, __shfl_xor_sync(0xffffffffu, low, d));
    high = largest(high, __shfl_xor_sync(0xffffffffu, high, d));
  }
  constexpr float PART = 1.f / 15.f;
  scales = Elem<T>::pack2(fmaf(high, PART, -low * PART), low);      // (the difference itself may exceed the type)
  const float m = Elem<T>::to_float(uint16_t(scales >> 16));
  // (a scale that was rounded up must not take the upper end out of the type: the next lower one)
  const float upper = fmaf(15.f, Elem<T>::to_float(uint16_t(scales)), m);
  if (!(fabsf(Elem<T>::to_float(Elem<T>::from_float(upper))) < __int_as_float(0x7f800000)) && high < __int_as_float(0x7f800000)) --scales;
  const float s = Elem<T>::to_float(uint16_t(scales));
  const bool finite = fabsf(s) < __int_as_float(0x7f800000) && fabsf(m) < __int_as_float(0x7f800000);
  if (!finite) scales = 0x7fff7fffu;
  // (powers of two that keep the reciprocal a normal number)
  const float by = std::is_same<T, __half>::value ? 1.f : s < 0x1p-60f ? 0x1p64f : s > 0x1p60f ? 0x1p-64f : 1.f;
  const float divisor = s * by, inverse = finite && s > 0.f ? __frcp_rn(divisor) : 0.f, origin = -m * by;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float d = fmaf(x[e], by, origin), q = d * inverse;
    const float n = fminf(fmaxf(fmaf(fmaf(-q, divisor, d), inverse, q), 0.f), 15.f);
    // (added to 1.5 * 2^23 a number is rounded to a whole one in the lowest bits)
    codes += (__float_as_uint(n + 12582912.f) - 0x4b400000u) << (4 * e);
  }
  return codes;
}

// GROUP: elements of a group of a cache in 4 bits; 0: a cache of 16-bit elements, or none
template <typename T, int D, bool NORM, bool NEIGHBOURS, bool CACHE, int ROWS, int GROUP>
__global__ void __launch_bounds__(THREADS) rotate_kernel(const RotateParams p) {
  constexpr int PIECE = PIECE_OF, PAIRS = PIECE / 2, LANES = D / (2 * PIECE);   // lanes of a row
  programmatic_begin();
  const int lane = threadIdx.x & 31, j = lane % LANES;
  // groups of a token: of its queries, its keys, its values
  const uint32_t q_groups = (p.q_heads + ROWS - 1) / ROWS, k_groups = (p.k_heads + ROWS - 1) / ROWS;
  const uint32_t groups = q_groups + (CACHE ? 2 : 1) * k_groups;
  const uint32_t at = blockIdx.x * uint32_t(THREADS / LANES) + threadIdx.x / LANES;
  const bool live = at < p.tokens * groups;          // (all lanes stay for the norms' sums)
  const uint32_t token = live ? at / groups : 0, group = at - token * groups;
  const bool is_q = group < q_groups, is_v = CACHE && group >= q_groups + k_groups;
  const uint32_t first = (is_q ? group : group - q_groups - (is_v ? k_groups : 0)) * ROWS;
  const uint32_t rows = live ? min((is_q ? p.q_heads : p.k_heads) - first, uint32_t(ROWS)) : 0;
  const int half = p.rotary_dim / 2;
  const bool turned = 2 * PIECE * j < p.rotary_dim;
  // this lane's two pieces of a row
  const int low = (NEIGHBOURS || !turned ? 2 : 1) * PIECE * j, high = NEIGHBOURS || !turned ? low + PIECE : half + low;
  const int64_t step = is_q ? p.q_head : is_v ? p.v_head : p.k_head;
  const uint16_t* from = (is_q ? p.q + token * p.q_token : is_v ? p.v + token * p.v_token : p.k + token * p.k_token) + first * step;
  programmatic_wait();

  Piece<PIECE> raw[ROWS][2];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    raw[i][0] = raw[i][1] = Piece<PIECE>{};
    if (i < rows) {
      raw[i][0] = load_piece<PIECE, true>(from + i * step + low);
      raw[i][1] = load_piece<PIECE, true>(from + i * step + high);
    }
  }
  // A row that is put in 4 bits changes its pieces of lanes for eight neighbouring elements each.
  constexpr bool EXCHANGED = GROUP > 0 && !NEIGHBOURS;
  __shared__ __align__(16) float exchange[EXCHANGED ? THREADS / LANES : 1][EXCHANGED ? D : 4];
  // (all of a warp's lanes stay for the groups' minima, if it has such rows)
  const bool quantised = GROUP > 0 && __any_sync(0xffffffffu, live && !is_q);
  const int64_t position = __ldg(p.positions + token);
  const bool known = position >= 0 && position < p.table_rows;
  uint16_t* to;                                      // the group's first row
  int64_t next = D;                                  // elements from one row to the next
  bool kept = true;
  int64_t place = 0;                                 // of the group's first row among the cache's
  if (CACHE && !is_q) {
    const int64_t slot = __ldg(p.slots + token);
    kept = slot >= 0 && slot < p.slot_count;
    const int64_t row = (((slot >> p.page_shift) * p.k_heads + first) << p.page_shift) + (slot & ((int64_t(1) << p.page_shift) - 1));
    place = kept ? row : 0;
    to = GROUP > 0 ? nullptr : (is_v ? p.v_out : p.k_out) + (kept ? row * D : 0);
    next = int64_t(D) << p.page_shift;
  } else {
    to = (is_q ? p.q_out + size_t(token) * p.q_heads * D : p.k_out + size_t(token) * p.k_heads * D) + size_t(first) * D;
  }
  if (GROUP == 0 && is_v) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
      if (i < rows && kept) {
        store_piece(to + i * next + low, raw[i][0]);
        store_piece(to + i * next + high, raw[i][1]);
      }
  }

  // What an element is multiplied with, and what its partner is for it: weight times cosine, weight times (minus) sine.
  uint64_t own[2][PAIRS], cross[2][PAIRS];
  {
    float c[PIECE], s[PIECE];                        // of this lane's PIECE pairs
#pragma unroll
    for (int e = 0; e < PIECE; ++e) c[e] = known ? 1.f : __int_as_float(0x7fc00000), s[e] = 0.f;
    if (known && turned && !is_v) {
      const float* angles = p.rotary + position * p.rotary_dim + PIECE * j;
#pragma unroll
      for (int e = 0; e < PIECE; e += 4) {
        const float4 cosine = __ldg(reinterpret_cast<const float4*>(angles + e));
        const float4 sine = __ldg(reinterpret_cast<const float4*>(angles + half + e));
        c[e] = cosine.x, c[e + 1] = cosine.y, c[e + 2] = cosine.z, c[e + 3] = cosine.w;
        s[e] = sine.x, s[e + 1] = sine.y, s[e + 2] = sine.z, s[e + 3] = sine.w;
      }
    }
    float w[2][PIECE];
    if (NORM) {
      const uint16_t* weight = is_q ? p.q_weight : p.k_weight;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const Piece<PIECE> v = load_piece<PIECE, false>(weight + (side ? high : low));
#pragma unroll
        for (int e = 0; e < PIECE; ++e) w[side][e] = Elem<T>::to_float(uint16_t(v.w[e / 2] >> (16 * (e & 1))));
      }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        float a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // element 2 e + i of the piece: its pair among the lane's, its partner
          const int pair = NEIGHBOURS ? side * PAIRS + e : 2 * e + i;
          const float sign = (NEIGHBOURS ? i : side) ? 1.f : -1.f;
          const float mine = NORM ? w[side][2 * e + i] : 1.f;
          const float partner = NORM ? (NEIGHBOURS ? w[side][2 * e + 1 - i] : w[1 - side][2 * e + i]) : 1.f;
          a[i] = mine * c[pair];
          b[i] = sign * (partner * s[pair]);
        }
        own[side][e] = two(a[0], a[1]);
        cross[side][e] = two(b[0], b[1]);
      }
  }
  const bool partly = p.rotary_dim < D;

#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    uint64_t x[2][PAIRS];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int e = 0; e < PAIRS; ++e)
        x[side][e] = two(Elem<T>::to_float(uint16_t(raw[i][side].w[e])), Elem<T>::to_float(uint16_t(raw[i][side].w[e] >> 16)));
    uint64_t scale = 0;
    if (NORM) {
      uint64_t squares = mul_two(x[0][0], x[0][0]);
#pragma unroll
      for (int e = 1; e < 2 * PAIRS; ++e) squares = fma_two(x[e / PAIRS][e % PAIRS], x[e / PAIRS][e % PAIRS], squares);
      const float2 both = apart(squares);
      float sum = both.x + both.y;
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float r = rsqrtf(sum * (1.f / D) + p.eps);
      scale = two(r, r);
    }
    const bool stored = i < rows && kept && !(GROUP == 0 && is_v);
    if (!stored && !quantised) continue;
    uint64_t turned_row[2][PAIRS];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) {
        uint64_t partner;
        if (NEIGHBOURS) {
          const float2 v = apart(x[side][e]);
          partner = two(v.y, v.x);
        } else {
          partner = x[1 - side][e];
        }
        if (partly && !turned) partner = 0;          // (what is not rotated has none, and may be infinite)
        uint64_t y = fma_two(x[side][e], own[side][e], mul_two(partner, cross[side][e]));
        if (NORM) y = mul_two(y, scale);
        turned_row[side][e] = GROUP > 0 && is_v ? x[side][e] : y;
      }
    if (stored && (GROUP == 0 || is_q)) {
      Piece<PIECE> out[2];
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int e = 0; e < PAIRS; ++e) {
          const float2 v = apart(turned_row[side][e]);
          out[side].w[e] = Elem<T>::pack2(v.x, v.y);
        }
      store_piece(to + i * next + low, out[0]);
      store_piece(to + i * next + high, out[1]);
    }
    if constexpr (GROUP > 0) {
      if (!quantised) continue;
      float8 row;
      if constexpr (EXCHANGED) {
        float* mine = exchange[threadIdx.x / LANES];
        __syncwarp();                                // (the row before has been read)
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const float2 a = apart(turned_row[side][0]), b = apart(turned_row[side][1]);
          *reinterpret_cast<float4*>(mine + (side ? high : low)) = make_float4(a.x, a.y, b.x, b.y);
        }
        __syncwarp();
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const float4 v = *reinterpret_cast<const float4*>(mine + 8 * j + 4 * side);
          row.v[4 * side] = v.x, row.v[4 * side + 1] = v.y, row.v[4 * side + 2] = v.z, row.v[4 * side + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = apart(turned_row[e / 2][e % 2]);
          row.v[2 * e] = v.x, row.v[2 * e + 1] = v.y;
        }
      }
      uint32_t scales;
      const uint32_t codes = quantise<T, GROUP>(row.v, scales);
      if (stored && !is_q) {
        const int64_t at_row = place + (int64_t(i) << p.page_shift);
        (is_v ? p.v_codes : p.k_codes)[at_row * (D / 8) + j] = codes;
        if (j % (GROUP / 8) == 0) (is_v ? p.v_scales : p.k_scales)[at_row * (D / GROUP) + j / (GROUP / 8)] = scales;
      }
    }
  }
}

template <typename T, int D, bool NORM, bool CACHE, int ROWS, int GROUP>
int launch(const RotateParams& p, bool neighbours, cudaStream_t stream) {
  constexpr uint32_t PER_CTA = THREADS / (D / (2 * PIECE_OF));
  auto kernel = neighbours ? rotate_kernel<T, D, NORM, true, CACHE, ROWS, GROUP> : rotate_kernel<T, D, NORM, false, CACHE, ROWS, GROUP>;
  const uint32_t groups = (p.q_heads + ROWS - 1) / ROWS + (CACHE ? 2 : 1) * ((p.k_heads + ROWS - 1) / ROWS);
  const uint32_t grid = (p.tokens * groups + PER_CTA - 1) / PER_CTA;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel),
                         ROWS == 1 ? "rotate_kernel a row per group" : "rotate_kernel several rows per group", int(grid), THREADS, 0, 1);
  const cudaError_t e = launch_programmatic(kernel, dim3(grid), dim3(THREADS), 0, stream, 1, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

template <typename T, bool CACHE, int GROUP = 0>
int choose(const RotateParams& p, int64_t dim, bool neighbours, cudaStream_t stream) {
  const bool many = p.tokens * (p.q_heads + (CACHE ? 2 : 1) * p.k_heads) >= MANY;
#define IB200_ROTATE(D_, NORM_)                                                        \
  (many ? launch<T, D_, NORM_, CACHE, SHARED_ROWS, GROUP>(p, neighbours, stream)       \
        : launch<T, D_, NORM_, CACHE, 1, GROUP>(p, neighbours, stream))
  if constexpr (GROUP == 128) return p.q_weight ? IB200_ROTATE(128, true) : IB200_ROTATE(128, false);
  else if (p.q_weight) return dim == 128 ? IB200_ROTATE(128, true) : IB200_ROTATE(64, true);
  else return dim == 128 ? IB200_ROTATE(128, false) : IB200_ROTATE(64, false);
#undef IB200_ROTATE
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

int set_rows(RotateParams& p, int64_t tokens, int64_t heads) {
  if (heads > (1 << 20) || tokens > ((int64_t(1) << 31) - 1) / heads) return INTENT_B200_ERR_UNSUPPORTED;
  p.tokens = uint32_t(tokens);
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
  if ((status = set_rows(p, q.d0, q.d1 + k.d1)) != INTENT_B200_OK) return status;
  if (p.tokens == 0) return INTENT_B200_OK;
  if (!k_out.p) return INTENT_B200_ERR_NULL;
  p.k_out = static_cast<uint16_t*>(k_out.p);
  return choose<T, false>(p, q.d2, pairs, stream);
}

// The same for a cache in 4 bits
template <typename T>
int append_int4(const View3& q, const View3& k, const View3& v, const View1& positions, const View1& slots, const View2& rotary,
                const View1* q_weight, const View1* k_weight, const View4& k_codes, const View4& k_scales, const View4& v_codes,
                const View4& v_scales, const View3& q_out, int32_t group, int32_t eps_bits, int32_t pairs, cudaStream_t stream) {
  RotateParams p = {};
  int status = prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
  if (status != INTENT_B200_OK) return status;
  if (v.d0 != k.d0 || v.d1 != k.d1 || v.d2 != k.d2 || slots.d0 != q.d0) return INTENT_B200_ERR_SHAPE;
  status = check_int4(k_codes, k_scales, v_codes, v_scales, k.d1, k.d2, group);
  if (status != INTENT_B200_OK) return status;
  if (!rows16(v) || !contiguous(slots) || !aligned16(v.p)) return INTENT_B200_ERR_LAYOUT;
  if ((status = set_rows(p, q.d0, q.d1 + 2 * k.d1)) != INTENT_B200_OK) return status;
  if (p.tokens == 0) return INTENT_B200_OK;
  if (!v.p || !slots.p || (k_codes.d0 > 0 && (!k_codes.p || !v_codes.p || !k_scales.p || !v_scales.p))) return INTENT_B200_ERR_NULL;
  p.v = static_cast<const uint16_t*>(v.p);
  p.v_token = v.s0, p.v_head = v.s1;
  p.slots = static_cast<const int64_t*>(slots.p);
  p.k_codes = static_cast<uint32_t*>(k_codes.p), p.v_codes = static_cast<uint32_t*>(v_codes.p);
  p.k_scales = static_cast<uint32_t*>(k_scales.p), p.v_scales = static_cast<uint32_t*>(v_scales.p);
  p.slot_count = k_codes.d0 * k_codes.d2;
  while ((int64_t(1) << p.page_shift) < k_codes.d2) ++p.page_shift;
  return group == 32 ? choose<T, true, 32>(p, q.d2, pairs, stream)
       : group == 64 ? choose<T, true, 64>(p, q.d2, pairs, stream) : choose<T, true, 128>(p, q.d2, pairs, stream);
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
  if ((status = set_rows(p, q.d0, q.d1 + 2 * k.d1)) != INTENT_B200_OK) return status;
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

#define IB200_APPEND_INT4_ENTRIES(NAME, TYPE)                                                                              \
  extern "C" int intent_b200_paged_kv_append_int4_##NAME(                                                                  \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW4(a6), INTENT_B200_VIEW4(a7), INTENT_B200_VIEW4(a8), INTENT_B200_VIEW4(a9),   \
      INTENT_B200_VIEW3(a10), int32_t group, int32_t pairs, void* stream) {                                                \
    return ib200::append_int4<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),    \
                                    IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), nullptr, nullptr, IB200_VIEW4_ARG(a6),       \
                                    IB200_VIEW4_ARG(a7), IB200_VIEW4_ARG(a8), IB200_VIEW4_ARG(a9), IB200_VIEW3_ARG(a10),   \
                                    group, 0, pairs, static_cast<cudaStream_t>(stream));                                   \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_kv_append_norm_int4_##NAME(                                                             \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW1(a6), INTENT_B200_VIEW1(a7), INTENT_B200_VIEW4(a8), INTENT_B200_VIEW4(a9),   \
      INTENT_B200_VIEW4(a10), INTENT_B200_VIEW4(a11), INTENT_B200_VIEW3(a12), int32_t group, int32_t eps_bits,             \
      int32_t pairs, void* stream) {                                                                                       \
    const ib200::View1 qw = IB200_VIEW1_ARG(a6), kw = IB200_VIEW1_ARG(a7);                                                 \
    return ib200::append_int4<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),    \
                                    IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), &qw, &kw, IB200_VIEW4_ARG(a8),               \
                                    IB200_VIEW4_ARG(a9), IB200_VIEW4_ARG(a10), IB200_VIEW4_ARG(a11), IB200_VIEW3_ARG(a12), \
                                    group, eps_bits, pairs, static_cast<cudaStream_t>(stream));                            \
  }
IB200_APPEND_INT4_ENTRIES(f16, __half)
IB200_APPEND_INT4_ENTRIES(bf16, __nv_bfloat16)
