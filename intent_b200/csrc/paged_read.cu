// Keys and values of given tokens out of a paged cache in 4 bits (paged_kv_read_int4):
//   k[t, h, i] = m + s * n of the code n at slots[t], of the scale s and the minimum m of its group, in f32 and rounded once; v alike
// A slot outside the cache (-1) gives a row of zeros.
//
// Bound by HBM, and by what it writes: 2 D bytes a row for D / 2 + 4 D / GROUP read.  A thread turns eight codes of keys and eight of
// values of two rows into 16 bytes each (65536 tokens, 8 heads of 128, bf16: with one row 73 us, with two 59 - 61, with four 60; 5.6 TB/s).
#include "common.cuh"
#include "paged.cuh"

namespace ib200 {
namespace {

constexpr int THREADS = 256;
constexpr int ROWS = 2;                  // of a thread

struct ReadParams {
  const int64_t* slots;
  const uint32_t *k_codes, *k_scales, *v_codes, *v_scales;
  uint4 *k, *v;
  int64_t slot_count;
  uint32_t tokens, heads;
  int page_shift;
};

// (2^23 + n has n in its lowest bits: no conversion)
template <typename T>
__device__ __forceinline__ uint4 values_of(uint32_t codes, uint32_t scales) {
  const float s = Elem<T>::to_float(uint16_t(scales)), m = Elem<T>::to_float(uint16_t(scales >> 16));
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float low = __uint_as_float(lop3_and_or(codes >> (8 * e), 15u, 0x4b000000u)) - 8388608.f;
    const float high = __uint_as_float(lop3_and_or(codes >> (8 * e + 4), 15u, 0x4b000000u)) - 8388608.f;
    w[e] = Elem<T>::pack2(fmaf(low, s, m), fmaf(high, s, m));
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(THREADS) read_kernel(const ReadParams p) {
  constexpr uint32_t PIECES = D / 8;
  programmatic_begin();
  const uint32_t lane_piece = threadIdx.x % PIECES, rows = p.tokens * p.heads;
  const uint32_t first = blockIdx.x * (THREADS / PIECES * ROWS) + threadIdx.x / PIECES;
  programmatic_wait();
  uint32_t codes[ROWS][2], scales[ROWS][2];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const uint32_t row = first + i * (THREADS / PIECES);
    codes[i][0] = codes[i][1] = scales[i][0] = scales[i][1] = 0;
    if (row >= rows) continue;
    const uint32_t token = row / p.heads, head = row - token * p.heads;
    const int64_t slot = __ldg(p.slots + token);
    if (slot < 0 || slot >= p.slot_count) continue;
    const int64_t place = (((slot >> p.page_shift) * p.heads + head) << p.page_shift) + (slot & ((int64_t(1) << p.page_shift) - 1));
    const int64_t code = place * PIECES + lane_piece, scale = place * (D / GROUP) + lane_piece / (GROUP / 8);
    codes[i][0] = __ldg(p.k_codes + code), scales[i][0] = __ldg(p.k_scales + scale);
    codes[i][1] = __ldg(p.v_codes + code), scales[i][1] = __ldg(p.v_scales + scale);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const uint32_t row = first + i * (THREADS / PIECES);
    if (row >= rows) continue;
    __stcs(p.k + size_t(row) * PIECES + lane_piece, values_of<T>(codes[i][0], scales[i][0]));
    __stcs(p.v + size_t(row) * PIECES + lane_piece, values_of<T>(codes[i][1], scales[i][1]));
  }
}

template <typename T, int D, int GROUP>
int launch(const ReadParams& p, cudaStream_t stream) {
  auto kernel = read_kernel<T, D, GROUP>;
  constexpr uint32_t PER_CTA = THREADS / (D / 8) * ROWS;
  const uint32_t grid = (p.tokens * p.heads + PER_CTA - 1) / PER_CTA;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel), "read_kernel", int(grid), THREADS, 0, 1);
  const cudaError_t e = launch_programmatic(kernel, dim3(grid), dim3(THREADS), 0, stream, 1, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

template <typename T>
int read(const View1& slots, const View4& k_codes, const View4& k_scales, const View4& v_codes, const View4& v_scales, const View3& k,
         const View3& v, int32_t group, cudaStream_t stream) {
  const int64_t tokens = slots.d0, heads = k.d1, dim = k.d2;
  if (tokens < 0 || k.d0 != tokens || heads <= 0 || v.d0 != tokens || v.d1 != heads || v.d2 != dim) return INTENT_B200_ERR_SHAPE;
  if (dim != 64 && dim != 128) return INTENT_B200_ERR_UNSUPPORTED;
  const int status = check_int4(k_codes, k_scales, v_codes, v_scales, heads, dim, group);
  if (status != INTENT_B200_OK) return status;
  if (!contiguous(slots) || !contiguous(k) || !contiguous(v) || !aligned16(k.p) || !aligned16(v.p)) return INTENT_B200_ERR_LAYOUT;
  if (heads > (1 << 20) || tokens > ((int64_t(1) << 31) - 1) / heads) return INTENT_B200_ERR_UNSUPPORTED;
  if (tokens == 0) return INTENT_B200_OK;
  if (!slots.p || !k.p || !v.p || (k_codes.d0 > 0 && (!k_codes.p || !k_scales.p || !v_codes.p || !v_scales.p)))
    return INTENT_B200_ERR_NULL;
  ReadParams p = {};
  p.slots = static_cast<const int64_t*>(slots.p);
  p.k_codes = static_cast<const uint32_t*>(k_codes.p), p.v_codes = static_cast<const uint32_t*>(v_codes.p);
  p.k_scales = static_cast<const uint32_t*>(k_scales.p), p.v_scales = static_cast<const uint32_t*>(v_scales.p);
  p.k = static_cast<uint4*>(k.p), p.v = static_cast<uint4*>(v.p);
  p.slot_count = k_codes.d0 * k_codes.d2;
  p.tokens = uint32_t(tokens), p.heads = uint32_t(heads);
  while ((int64_t(1) << p.page_shift) < k_codes.d2) ++p.page_shift;
  if (dim == 64) return group == 32 ? launch<T, 64, 32>(p, stream) : launch<T, 64, 64>(p, stream);
  return group == 32 ? launch<T, 128, 32>(p, stream) : group == 64 ? launch<T, 128, 64>(p, stream) : launch<T, 128, 128>(p, stream);
}

}  // namespace
}  // namespace ib200

#define IB200_READ_ENTRIES(NAME, TYPE)                                                                                     \
  extern "C" int intent_b200_paged_kv_read_int4_##NAME(                                                                    \
      INTENT_B200_VIEW1(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW4(a3), INTENT_B200_VIEW4(a4),   \
      INTENT_B200_VIEW3(a5), INTENT_B200_VIEW3(a6), int32_t group, void* stream) {                                         \
    return ib200::read<TYPE>(IB200_VIEW1_ARG(a0), IB200_VIEW4_ARG(a1), IB200_VIEW4_ARG(a2), IB200_VIEW4_ARG(a3),           \
                             IB200_VIEW4_ARG(a4), IB200_VIEW3_ARG(a5), IB200_VIEW3_ARG(a6), group,                         \
                             static_cast<cudaStream_t>(stream));                                                           \
  }
IB200_READ_ENTRIES(f16, __half)
IB200_READ_ENTRIES(bf16, __nv_bfloat16)
