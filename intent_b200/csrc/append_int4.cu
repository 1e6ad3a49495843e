// Append of keys and values to a paged cache in 4 bits, with the norms and the rotation of queries and keys (paged_kv_append_int4).
//
// Queries are those of paged_kv_append (rotate.cuh).  A group of GROUP consecutive elements x of a head's key, after its norm and
// rotation and not rounded before, or of its value, is held as
//   m = min x,   s = (max x - min x) / 15, both rounded to the 16-bit type,   n = nearest((x - m) / s), the even one of two, in 0 .. 15
// (s the next lower number where m + 15 s would be beyond the type; a group with something that is no finite number is NaN).
//
// A code is off by one as soon as a number next to a half is off by a little, and then by a whole step.  So keys are worked out in 64
// bits where f32 does not decide (in f32 alone three of a million codes were others, now they are those of the definition).
// Values have no arithmetic before: their minima are exact, their codes' quotients are in 64 bits (55.2 us below; with f32, in which
// the difference to a minimum 2^16 times as large or as small is rounded, 54.4).
//
// A lane has eight neighbouring elements of a row.  The partners of a key's elements in pairs (i, i + R/2) are another lane's; it reads
// them once more from the first-level cache and works out its own half of each pair.  Blocks have keys, values or queries; in
// calls of many rows two rows of keys or values, and four of queries, share what does not depend on the row.
//
// Measured on one B200: 8192 tokens, 32 + 8 + 8 heads of 128, norm, bf16, with paged_kv_read_int4 of them 55 us (floor 33), of which the
// read is 9, queries take 20 alone, keys 12 and values 6: bound by instructions, two thirds of the issue slots.  All keys in 64
// bits 59; keys' blocks ahead of the others 63; with four rows of keys and 102 registers 76.  (With norms and several rows a group the
// 64 registers do not hold everything: 40 to 48 bytes are spilled.)
#include "common.cuh"
#include "paged.cuh"
#include "rotate.cuh"

namespace ib200 {
namespace {

constexpr int THREADS = ROTATE_THREADS;
constexpr int CACHE_ROWS = 2;           // keys or values of a group in calls of many rows

// The smaller and the larger of two; NaN if one is (f32), which is looked for apart (f64)
__device__ __forceinline__ float least_of(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float largest_of(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ double least_of(double a, double b) { return a < b ? a : b; }
__device__ __forceinline__ double largest_of(double a, double b) { return a > b ? a : b; }

// The quotients of eight numbers by a scale s, rounded to whole numbers from 0 to 15, in 64 bits: the difference to the minimum of two
// 16-bit numbers can have more bits than f32 has, and a half and a little is not a half.  The product with the rounded reciprocal gets
// its remainder added, which makes it the quotient as a division rounds it (P. Markstein, Computation of elementary functions on the
// IBM RISC System/6000 processor, 1990): halves, common among 16-bit numbers, are halves.  So are those of keys: what is zero stays
// zero, and -m / s is a quotient of 16-bit numbers.  Added to 1.5 * 2^52 a number is rounded in the lowest bits.
template <typename F>
__device__ __forceinline__ uint32_t codes_of(const F (&x)[8], float scale, float minimum) {
  const double s = scale, m = minimum, inverse = scale > 0.f ? __drcp_rn(s) : 0.;
  uint32_t codes = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double d = double(x[e]) - m, q = d * inverse;
    double quotient = fma(fma(-q, s, d), inverse, q);
    // (where the rounding of a key's minimum is many scales, it may be far out; a value's minimum is not rounded)
    if (std::is_same<F, double>::value) quotient = quotient < 0. ? 0. : quotient > 15. ? 15. : quotient;
    codes |= uint32_t(min(__double2loint(quotient + 6755399441055744.), 15)) << (4 * e);
  }
  return codes;
}

// Eight neighbouring elements of a row as codes; `scales`: scale | minimum of their group, which all of its lanes know
template <typename T, int GROUP, typename F>
__device__ __forceinline__ uint32_t quantise(const F (&x)[8], uint32_t& scales) {
  const float infinity = __int_as_float(0x7f800000);
  F low = x[0], high = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) low = least_of(x[e], low), high = largest_of(x[e], high);
#pragma unroll
  for (int d = 1; d < GROUP / 8; d *= 2) {
    low = least_of(__shfl_xor_sync(0xffffffffu, low, d), low);
    high = largest_of(__shfl_xor_sync(0xffffffffu, high, d), high);
  }
  bool odd = false;                    // something of the group is no number
  if (std::is_same<F, double>::value) {
    F nothing = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) nothing = fma(x[e], F(0), nothing);
    constexpr uint32_t LANES = (1u << (GROUP / 8)) - 1;
    odd = __ballot_sync(0xffffffffu, nothing != 0) >> (threadIdx.x & 31 & ~(GROUP / 8 - 1)) & LANES;
  }
  // (in 64 bits; rounded to the type by way of f32, so that within 2^-25 of the middle between two numbers it may be either)
  scales = Elem<T>::pack2(float((double(high) - double(low)) * (1. / 15.)), float(low));
  const float m = Elem<T>::to_float(uint16_t(scales >> 16));
  float s = Elem<T>::to_float(uint16_t(scales));
  if (odd || !(s < infinity) || !(fabsf(m) < infinity)) {
    scales = 0x7fff7fffu;
    return 0;
  }
  if (!(Elem<T>::to_float(Elem<T>::from_float(fmaf(15.f, s, m))) < infinity)) s = Elem<T>::to_float(uint16_t(--scales));
  return codes_of(x, s, m);
}

// A group of lanes and its rows of one kind of one token
template <int D, int ROWS>
struct Group {
  uint32_t token, first;               // its first head
  int rows;                            // 0: there is none
  int64_t place;                       // of the first row in the cache, in rows
  bool kept;
  __device__ __forceinline__ Group(const RotateParams& p, uint32_t block) {
    const uint32_t groups = (p.k_heads + ROWS - 1) / ROWS, at = block * uint32_t(THREADS / (D / 8)) + threadIdx.x / (D / 8);
    const bool live = at < p.tokens * groups;
    token = live ? at / groups : 0;
    first = (at - token * groups) * ROWS;
    rows = live ? int(min(p.k_heads - first, uint32_t(ROWS))) : 0;
  }
  __device__ __forceinline__ void find(const RotateParams& p) {
    const int64_t slot = __ldg(p.slots + token);
    kept = rows > 0 && slot >= 0 && slot < p.slot_count;
    place = kept ? (((slot >> p.page_shift) * p.k_heads + first) << p.page_shift) + (slot & ((int64_t(1) << p.page_shift) - 1)) : 0;
  }
  template <int GROUP>
  __device__ __forceinline__ void store(const RotateParams& p, int i, int j, uint32_t* codes_to, uint32_t* scales_to, uint32_t codes,
                                        uint32_t scales) const {
    if (!kept || i >= rows) return;
    const int64_t row = place + (int64_t(i) << p.page_shift);
    codes_to[row * (D / 8) + j] = codes;
    if (j % (GROUP / 8) == 0) scales_to[row * (D / GROUP) + j / (GROUP / 8)] = scales;
  }
};

template <typename T, int D, int ROWS, int GROUP>
__device__ __forceinline__ void value_rows(const RotateParams& p, uint32_t block) {
  const int j = threadIdx.x % (D / 8);
  Group<D, ROWS> group(p, block);
  const uint16_t* from = p.v + group.token * p.v_token + group.first * p.v_head + 8 * j;
  programmatic_wait();
  uint4 raw[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) raw[i] = i < group.rows ? ldg_stream_v4(from + i * p.v_head) : make_uint4(0, 0, 0, 0);
  group.find(p);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = Elem<T>::to_float(uint16_t(w[e / 2] >> (16 * (e & 1))));
    uint32_t scales;
    const uint32_t codes = quantise<T, GROUP>(x, scales);
    group.template store<GROUP>(p, i, j, p.v_codes, p.v_scales, codes, scales);
  }
}

// What a lane's eight elements of a key are multiplied with, and what their partners are for them: weight times cosine, weight times
// (minus) sine.
template <typename T, int D, bool NORM, bool NEIGHBOURS, typename F>
struct Turn {
  F own[8], cross[8];
  int mate;                            // first of the partners
  bool turned;
  __device__ __forceinline__ Turn(const RotateParams& p, int j, int64_t position) {
    const int half = p.rotary_dim / 2;
    const bool upper = 8 * j >= half, known = position >= 0 && position < p.table_rows;
    turned = 8 * j < p.rotary_dim;
    mate = NEIGHBOURS || !turned ? 8 * j : upper ? 8 * j - half : 8 * j + half;
    constexpr int ANGLES = NEIGHBOURS ? 4 : 8;
    float c[ANGLES], s[ANGLES];
#pragma unroll
    for (int e = 0; e < ANGLES; ++e) c[e] = known ? 1.f : __int_as_float(0x7fc00000), s[e] = 0.f;
    if (known && turned) {
      const float* angles = p.rotary + position * p.rotary_dim + (NEIGHBOURS ? 4 * j : upper ? 8 * j - half : 8 * j);
#pragma unroll
      for (int e = 0; e < ANGLES; e += 4) {
        const float4 cosine = __ldg(reinterpret_cast<const float4*>(angles + e));
        const float4 sine = __ldg(reinterpret_cast<const float4*>(angles + half + e));
        c[e] = cosine.x, c[e + 1] = cosine.y, c[e + 2] = cosine.z, c[e + 3] = cosine.w;
        s[e] = sine.x, s[e + 1] = sine.y, s[e + 2] = sine.z, s[e + 3] = sine.w;
      }
    }
    uint4 weight = make_uint4(0, 0, 0, 0), partner_weight = weight;
    if (NORM) {
      weight = __ldg(reinterpret_cast<const uint4*>(p.k_weight + 8 * j));
      if (!NEIGHBOURS) partner_weight = __ldg(reinterpret_cast<const uint4*>(p.k_weight + mate));
    }
    const uint32_t w[4] = {weight.x, weight.y, weight.z, weight.w};
    const uint32_t v[4] = {partner_weight.x, partner_weight.y, partner_weight.z, partner_weight.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pair = NEIGHBOURS ? e / 2 : e;
      const F cosine = c[pair], sine = (NEIGHBOURS ? e & 1 : upper) ? s[pair] : -s[pair];
      own[e] = NORM ? cosine * F(Elem<T>::to_float(uint16_t(w[e / 2] >> (16 * (e & 1))))) : cosine;
      const uint32_t of_partner = NEIGHBOURS ? w[e / 2] >> (16 * (1 - (e & 1))) : v[e / 2] >> (16 * (e & 1));
      cross[e] = NORM ? sine * F(Elem<T>::to_float(uint16_t(of_partner))) : sine;
    }
  }
  // the elements of a row before its norm's factor, and their partners
  __device__ __forceinline__ void elements(const uint4& raw, const uint4& partners, F (&x)[8], F (&y)[8]) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w}, v[4] = {partners.x, partners.y, partners.z, partners.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = Elem<T>::to_float(uint16_t(w[e / 2] >> (16 * (e & 1))));
      y[e] = Elem<T>::to_float(uint16_t(NEIGHBOURS ? w[e / 2] >> (16 * (1 - (e & 1))) : v[e / 2] >> (16 * (e & 1))));
      if (NEIGHBOURS && !turned) y[e] = 0;           // (what is not rotated has none, and may be infinite)
    }
  }
};

__device__ __forceinline__ uint4 load_eight(const uint16_t* from, bool there) {
  return there ? __ldg(reinterpret_cast<const uint4*>(from)) : make_uint4(0, 0, 0, 0);
}

// A lane's part of a key in 64 bits, from its row in memory: codes in the lower half, scales in the upper.  (Few rows come here, so
// it is a function of its own.)
template <typename T, int D, bool NORM, bool NEIGHBOURS, int GROUP>
__device__ __noinline__ uint64_t key_in_64_bits(const RotateParams& p, const uint16_t* row, bool there, int64_t position) {
  constexpr int LANES = D / 8;
  const int j = threadIdx.x % LANES;
  const Turn<T, D, NORM, NEIGHBOURS, double> turn(p, j, position);
  double x[8], y[8];
  turn.elements(load_eight(row + 8 * j, there), load_eight(row + turn.mate, there && turn.turned && !NEIGHBOURS), x, y);
  double scale = 1.;
  if (NORM) {
    double sum = x[0] * x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) sum = fma(x[e], x[e], sum);
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    scale = rsqrt(sum * (1. / D) + double(p.eps));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = fma(x[e], turn.own[e], y[e] * turn.cross[e]) * scale;
  uint32_t scales;
  const uint32_t codes = quantise<T, GROUP>(y, scales);
  return codes | uint64_t(scales) << 32;
}

// A number added to this is rounded to a whole one in the lowest bits, from which code_of takes it, cut to 0 .. 15
constexpr float WHOLE = 12582912.f;
__device__ __forceinline__ uint32_t code_of(float sum) {
  return uint32_t(__viaddmin_s32_relu(__float_as_int(sum), -__float_as_int(WHOLE), 15));
}

// Keys in f32 first.  An element is then off by at most DELTA = 2^-20 of |x own| + |partner cross|, times the norm's factor r (the
// sum of squares and r up to 2^-21, five roundings of 2^-24), which is at most the row's largest |own| + |cross| times its largest r |x|.
// (With sqrt(D) in the place of that, which r |x| cannot exceed, four times as many rows were worked out twice: 6 us of 57.)  Where the
// minimum's or the scale's rounding, or a code's, could be another within that, the warp's rows are worked out in 64 bits; so are
// those with something that is no number, with equal elements, and near the ends of the type.
template <typename T, int D, bool NORM, bool NEIGHBOURS, int ROWS, int GROUP>
__device__ __forceinline__ void key_rows(const RotateParams& p, uint32_t block) {
  constexpr int LANES = D / 8;
  const int j = threadIdx.x % LANES;
  Group<D, ROWS> group(p, block);
  const uint16_t* from = p.k + group.token * p.k_token + group.first * p.k_head;
  programmatic_wait();
  const int64_t position = __ldg(p.positions + group.token);
  const Turn<T, D, NORM, NEIGHBOURS, float> turn(p, j, position);
  uint4 raw[ROWS], partners[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    raw[i] = load_eight(from + i * p.k_head + 8 * j, i < group.rows);
    partners[i] = load_eight(from + i * p.k_head + turn.mate, i < group.rows && turn.turned && !NEIGHBOURS);
  }
  group.find(p);
  float most = 0.f;                    // of |own| + |cross|, in the row
#pragma unroll
  for (int e = 0; e < 8; ++e) most = largest_of(most, fabsf(turn.own[e]) + fabsf(turn.cross[e]));
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) most = largest_of(most, __shfl_xor_sync(0xffffffffu, most, d));
  most *= 0x1.001p-20f;                // (and what these products are rounded by)
  uint32_t open = 0;                   // the rows that have to be worked out in 64 bits

#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float x[8], y[8], size = 0.f;
    turn.elements(raw[i], partners[i], x, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) size = largest_of(size, fabsf(x[e]));
#pragma unroll
    for (int d = 1; d < LANES; d *= 2) size = largest_of(size, __shfl_xor_sync(0xffffffffu, size, d));
    float delta = most * size;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], turn.own[e], y[e] * turn.cross[e]);
    if (NORM) {
      float sum = x[0] * x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float scale = rsqrtf(sum * (1.f / D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= scale;
      delta *= scale;
    }
    float low = y[0], high = y[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) low = least_of(y[e], low), high = largest_of(y[e], high);
#pragma unroll
    for (int d = 1; d < GROUP / 8; d *= 2) {
      low = least_of(low, __shfl_xor_sync(0xffffffffu, low, d));
      high = largest_of(high, __shfl_xor_sync(0xffffffffu, high, d));
    }
    const float step = (high - low) * (1.f / 15.f), of_step = fmaf(delta, 2.1f / 15.f, step * 0x1p-21f);
    uint32_t scales = Elem<T>::pack2(step - of_step, low - delta);
    const float s = Elem<T>::to_float(uint16_t(scales)), m = Elem<T>::to_float(uint16_t(scales >> 16));
    bool sure = scales == Elem<T>::pack2(step + of_step, low + delta) && s > 0x1p-60f && s < 0x1p60f &&
                Elem<T>::to_float(Elem<T>::from_float(fmaf(15.f, s, m))) < __int_as_float(0x7f800000);
    // (a quotient is off by DELTA's share and a few roundings of numbers up to 16)
    const float inverse = __fdividef(1.f, s), most_off = 0.5f - fmaf(delta, inverse, 0x1p-17f);
    float off = 0.f;                   // farthest from a whole number
    uint32_t codes = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = (y[e] - m) * inverse, sum = q + WHOLE;
      off = largest_of(off, fabsf(q - (sum - WHOLE)));
      codes |= code_of(sum) << (4 * e);
    }
    // (and none is so far out, by the minimum's rounding, that its whole number is)
    sure = sure && off < most_off && fabsf(low - m) < 1024.f * s && high - m < 1024.f * s;
    if (__any_sync(0xffffffffu, !sure && group.kept && i < group.rows)) open |= 1u << i;
    group.template store<GROUP>(p, i, j, p.k_codes, p.k_scales, codes, scales);
  }
  // (behind the loop, where little has to be kept across the call: 57 -> 56 us)
#pragma unroll 1
  for (int i = 0; open; ++i, open >>= 1) {
    if (!(open & 1)) continue;
    const uint64_t both = key_in_64_bits<T, D, NORM, NEIGHBOURS, GROUP>(p, from + i * p.k_head, i < group.rows, position);
    group.template store<GROUP>(p, i, j, p.k_codes, p.k_scales, uint32_t(both), uint32_t(both >> 32));
  }
}

// Blocks of keys and as many of values, in turn, spread evenly among those of queries: keys are bound by
// instructions, queries by HBM.  `share`: of the blocks, keys' and values', in 2^-32, rounded up.
template <typename T, int D, bool NORM, bool NEIGHBOURS, int ROWS, int GROUP>
__global__ void __launch_bounds__(THREADS, 4) append_int4_kernel(const __grid_constant__ RotateParams p, uint32_t share) {
  constexpr int OF_CACHE = ROWS == 1 ? 1 : CACHE_ROWS;
  programmatic_begin();
  const uint32_t before = __umulhi(blockIdx.x, share);             // keys' and values' blocks ahead of this one
  if (__umulhi(blockIdx.x + 1, share) == before) rotate_rows<T, D, NORM, NEIGHBOURS, false, ROWS, true>(p, blockIdx.x - before);
  else if (before % 2 == 0) key_rows<T, D, NORM, NEIGHBOURS, OF_CACHE, GROUP>(p, before / 2);
  else value_rows<T, D, OF_CACHE, GROUP>(p, before / 2);
}

template <typename T, int D, bool NORM, int ROWS, int GROUP>
int launch(const RotateParams& p, bool neighbours, cudaStream_t stream) {
  auto kernel = neighbours ? append_int4_kernel<T, D, NORM, true, ROWS, GROUP> : append_int4_kernel<T, D, NORM, false, ROWS, GROUP>;
  constexpr uint32_t PER_CTA = THREADS / (D / 8);
  static_assert(D / 8 == D / (2 * PIECE_OF), "lanes of a row of queries");
  constexpr uint32_t OF_CACHE = ROWS == 1 ? 1 : CACHE_ROWS;
  const uint32_t k_blocks = (p.tokens * ((p.k_heads + OF_CACHE - 1) / OF_CACHE) + PER_CTA - 1) / PER_CTA;
  const uint32_t q_blocks = (p.tokens * ((p.q_heads + ROWS - 1) / ROWS) + PER_CTA - 1) / PER_CTA, grid = 2 * k_blocks + q_blocks;
  const uint32_t share = uint32_t((uint64_t(2 * k_blocks) << 32) / grid) + 1;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel),
                         ROWS == 1 ? "append_int4_kernel a row per group" : "append_int4_kernel several rows per group", int(grid), THREADS,
                         0, 1);
  const cudaError_t e = launch_programmatic(kernel, dim3(grid), dim3(THREADS), 0, stream, 1, p, share);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

template <typename T, int D, int GROUP>
int choose(const RotateParams& p, bool neighbours, cudaStream_t stream) {
  const bool many = p.tokens * (p.q_heads + 2 * p.k_heads) >= MANY;
  if (p.q_weight) return many ? launch<T, D, true, SHARED_ROWS, GROUP>(p, neighbours, stream)
                              : launch<T, D, true, 1, GROUP>(p, neighbours, stream);
  return many ? launch<T, D, false, SHARED_ROWS, GROUP>(p, neighbours, stream) : launch<T, D, false, 1, GROUP>(p, neighbours, stream);
}

template <typename T>
int append(const View3& q, const View3& k, const View3& v, const View1& positions, const View1& slots, const View2& rotary,
           const View1* q_weight, const View1* k_weight, const View4& k_codes, const View4& k_scales, const View4& v_codes,
           const View4& v_scales, const View3& q_out, int32_t group, int32_t eps_bits, int32_t pairs, cudaStream_t stream) {
  RotateParams p = {};
  int status = rotate_prepare(p, q, k, positions, rotary, q_out, q_weight, k_weight, eps_bits, pairs);
  if (status != INTENT_B200_OK) return status;
  if (v.d0 != k.d0 || v.d1 != k.d1 || v.d2 != k.d2 || slots.d0 != q.d0) return INTENT_B200_ERR_SHAPE;
  status = check_int4(k_codes, k_scales, v_codes, v_scales, k.d1, k.d2, group);
  if (status != INTENT_B200_OK) return status;
  if (!rows16(v) || !contiguous(slots) || !aligned16(v.p)) return INTENT_B200_ERR_LAYOUT;
  if ((status = rotate_set_rows(p, q.d0, q.d1 + 2 * k.d1)) != INTENT_B200_OK) return status;
  if (p.tokens == 0) return INTENT_B200_OK;
  if (!v.p || !slots.p || (k_codes.d0 > 0 && (!k_codes.p || !v_codes.p || !k_scales.p || !v_scales.p))) return INTENT_B200_ERR_NULL;
  p.v = static_cast<const uint16_t*>(v.p);
  p.v_token = v.s0, p.v_head = v.s1;
  p.slots = static_cast<const int64_t*>(slots.p);
  p.k_codes = static_cast<uint32_t*>(k_codes.p), p.v_codes = static_cast<uint32_t*>(v_codes.p);
  p.k_scales = static_cast<uint32_t*>(k_scales.p), p.v_scales = static_cast<uint32_t*>(v_scales.p);
  p.slot_count = k_codes.d0 * k_codes.d2;
  while ((int64_t(1) << p.page_shift) < k_codes.d2) ++p.page_shift;
  if (q.d2 == 64) return group == 32 ? choose<T, 64, 32>(p, pairs, stream) : choose<T, 64, 64>(p, pairs, stream);
  return group == 32   ? choose<T, 128, 32>(p, pairs, stream)
         : group == 64 ? choose<T, 128, 64>(p, pairs, stream) : choose<T, 128, 128>(p, pairs, stream);
}

}  // namespace
}  // namespace ib200

#define IB200_APPEND_INT4_ENTRIES(NAME, TYPE)                                                                              \
  extern "C" int intent_b200_paged_kv_append_int4_##NAME(                                                                  \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW4(a6), INTENT_B200_VIEW4(a7), INTENT_B200_VIEW4(a8), INTENT_B200_VIEW4(a9),   \
      INTENT_B200_VIEW3(a10), int32_t group, int32_t pairs, void* stream) {                                                \
    return ib200::append<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),         \
                               IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), nullptr, nullptr, IB200_VIEW4_ARG(a6),            \
                               IB200_VIEW4_ARG(a7), IB200_VIEW4_ARG(a8), IB200_VIEW4_ARG(a9), IB200_VIEW3_ARG(a10),        \
                               group, 0, pairs, static_cast<cudaStream_t>(stream));                                        \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_kv_append_norm_int4_##NAME(                                                             \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW3(a1), INTENT_B200_VIEW3(a2), INTENT_B200_VIEW1(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW1(a6), INTENT_B200_VIEW1(a7), INTENT_B200_VIEW4(a8), INTENT_B200_VIEW4(a9),   \
      INTENT_B200_VIEW4(a10), INTENT_B200_VIEW4(a11), INTENT_B200_VIEW3(a12), int32_t group, int32_t eps_bits,             \
      int32_t pairs, void* stream) {                                                                                       \
    const ib200::View1 qw = IB200_VIEW1_ARG(a6), kw = IB200_VIEW1_ARG(a7);                                                 \
    return ib200::append<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW3_ARG(a1), IB200_VIEW3_ARG(a2), IB200_VIEW1_ARG(a3),         \
                               IB200_VIEW1_ARG(a4), IB200_VIEW2_ARG(a5), &qw, &kw, IB200_VIEW4_ARG(a8),                    \
                               IB200_VIEW4_ARG(a9), IB200_VIEW4_ARG(a10), IB200_VIEW4_ARG(a11), IB200_VIEW3_ARG(a12),      \
                               group, eps_bits, pairs, static_cast<cudaStream_t>(stream));                                 \
  }
IB200_APPEND_INT4_ENTRIES(f16, __half)
IB200_APPEND_INT4_ENTRIES(bf16, __nv_bfloat16)
