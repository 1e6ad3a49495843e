// Norms of rows and their rotation by position, for the kernels that rotate queries and keys (rope_append.cu, append_int4.cu).
#pragma once

#include <cstring>

#include "common.cuh"

namespace ib200 {

constexpr int ROTATE_THREADS = 256;
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

// Checks what both programs share and fills the parameters in.
inline int rotate_prepare(RotateParams& p, const View3& q, const View3& k, const View1& positions, const View2& rotary, const View3& q_out,
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

inline int rotate_set_rows(RotateParams& p, int64_t tokens, int64_t heads) {
  if (heads > (1 << 20) || tokens > ((int64_t(1) << 31) - 1) / heads) return INTENT_B200_ERR_UNSUPPORTED;
  p.tokens = uint32_t(tokens);
  return INTENT_B200_OK;
}

#ifdef __CUDACC__

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

// The rows of one block of ROTATE_THREADS.  QUERIES: there are no others.
template <typename T, int D, bool NORM, bool NEIGHBOURS, bool CACHE, int ROWS, bool QUERIES = false>
__device__ __forceinline__ void rotate_rows(const RotateParams& p, uint32_t block) {
  constexpr int PIECE = PIECE_OF, PAIRS = PIECE / 2, LANES = D / (2 * PIECE);   // lanes of a row
  const int lane = threadIdx.x & 31, j = lane % LANES;
  // groups of a token: of its queries, its keys, its values
  const uint32_t q_groups = (p.q_heads + ROWS - 1) / ROWS, k_groups = (p.k_heads + ROWS - 1) / ROWS;
  const uint32_t groups = QUERIES ? q_groups : q_groups + (CACHE ? 2 : 1) * k_groups;
  const uint32_t at = block * uint32_t(ROTATE_THREADS / LANES) + threadIdx.x / LANES;
  const bool live = at < p.tokens * groups;          // (all lanes stay for the norms' sums)
  const uint32_t token = live ? at / groups : 0, group = at - token * groups;
  const bool is_q = QUERIES || group < q_groups, is_v = CACHE && group >= q_groups + k_groups;
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
  const int64_t position = __ldg(p.positions + token);
  const bool known = position >= 0 && position < p.table_rows;
  uint16_t* to;                                      // the group's first row
  int64_t next = D;                                  // elements from one row to the next
  bool kept = true;
  if (CACHE && !is_q) {
    const int64_t slot = __ldg(p.slots + token);
    kept = slot >= 0 && slot < p.slot_count;
    const int64_t row = (((slot >> p.page_shift) * p.k_heads + first) << p.page_shift) + (slot & ((int64_t(1) << p.page_shift) - 1));
    to = (is_v ? p.v_out : p.k_out) + (kept ? row * D : 0);
    next = int64_t(D) << p.page_shift;
  } else {
    to = (is_q ? p.q_out + size_t(token) * p.q_heads * D : p.k_out + size_t(token) * p.k_heads * D) + size_t(first) * D;
  }
  if (is_v) {
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
    if (i >= rows || !kept || is_v) continue;
    Piece<PIECE> out[2];
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
        const float2 v = apart(y);
        out[side].w[e] = Elem<T>::pack2(v.x, v.y);
      }
    store_piece(to + i * next + low, out[0]);
    store_piece(to + i * next + high, out[1]);
  }
}

#endif  // __CUDACC__

}  // namespace ib200
