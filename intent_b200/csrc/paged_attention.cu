// Entries of attention over a paged cache: argument checks and the choice of the kernel.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>

#include "paged.cuh"

namespace ib200 {
namespace {

constexpr float kInt4Scale = 0x1p50f;     // (scores over a cache in 4 bits are in a unit of their own)

int device_sms() {
  int device = 0, sms = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return sms;
}

// Which kernel takes a sequence goes by its rows (new tokens x query heads of a key head).  Those of one tile, up to sixteen
// rows, are bound by HBM in the rows kernel; with more rows it reads and multiplies the cache once for every tile.  us for 64
// sequences of up to 4000 tokens, 32 heads of 128 on 8 key heads, 1 / 4 / 8 / 16 new tokens each: rows 98 / 103 / 189 / 345, chunk
// 146 / 146 / 147 / 146; one sequence of 8000: rows 14 / 17 / 20 / 30, chunk 24 throughout.  With heads of 64 two tiles still are
// (64 heads on 8, 4 / 8 new tokens: rows 105 / 185, chunk 128 / 130).
// The host knows the number of all rows only, so a call may need both kernels, each for its sequences (`few`):
//  * more rows than one tile each on average: the chunk kernel, in calls of many sequences beside the rows kernel for those of
//    one tile (20 single tokens beside 4 chunks of up to 500: 169 -> 160 us, with tiles of eight 144; of few sequences the two
//    launches cost more than that: 3 prompts 120 -> 128);
//  * no more: the rows kernel, and the chunk kernel for those of more than two tiles.  768 tokens beside 255 single ones (up to
//    8192, as above): 1375 us by the rows kernel alone, 802 by both; 2000 beside 199 (16 heads on 16): 1175 and 618; 128 beside
//    64: 163 and 135.  Where no sequence turns out to have so many, that costs a launch that finds nothing to do: 64 of 4 tokens 111
//    and 118.  So it is left out where it can win little: the rows that one sequence may have, if each has a token, times the
//    tokens that they may walk through, up to MOST.  us without and with it: 49 tokens beside 15 single ones of up to 4096 (0.8 M)
//    62 and 66, of up to 16384 (3.2 M) 189 and 139; 60 beside 63 of up to 4096 (1.0 M) 132 and 128; 22 beside 6 of up to 65536
//    (5.8 M) 306 and 212; and if there is no long one 16 of 4 tokens 40 and 47, 64 of 2 of up to 300 26 and 31, 4 of 4 of up to
//    65536 105 and 113.
// A cache in 4 bits is read four times as fast, and more of the time goes to what both kernels do with its codes: the rows kernel's
// tiles are worth it for more rows.  us for the 64 sequences of up to 4000 tokens, 1 / 4 / 8 new ones each, bf16, groups of 64: rows
// 40 / 83 / 130, from four on with the 12 of a launch that finds nothing to do; 16, by the chunk kernel, 155 (4 to 16 all take it 146 -
// 155).  Heads of 64: rows 29 / 47 / 77, 16 of them 126, chunk 130; 8 of up to 16000: rows 28 / 54 / 78, chunk 89.  (8 new ones
// in f16 151; groups of 32 179, f16 210, where the chunk kernel would be faster: the limits are the same for all groups and types, as
// what a call's workspace holds is asked for without them.  MOST is that of 16-bit elements.)
struct Choice {
  int tile_rows;           // of the rows kernel; 0: it is not needed
  int few;                 // rows up to which a sequence is its
  bool chunks;             // the chunk kernel is needed
};
Choice choose(int64_t tokens, int64_t batch, int64_t group, int64_t dim, int64_t capacity, int64_t window, bool may_chunk, bool int4) {
  constexpr int FEW = 16, MANY = 8, MOST = 1 << 20;
  // rows per sequence, on average, up to which a call is the rows kernel's; a sequence's rows up to which it is beside others
  const int all_few = int4 ? (dim == 64 ? 4 * FEW : 2 * FEW) : dim == 64 ? 2 * FEW : FEW;
  const int one_few = int4 ? (dim == 64 ? 4 * FEW : 3 * FEW) : 2 * FEW;
  const int64_t rows = tokens * group, most = tokens < batch ? rows : (tokens - batch + 1) * group;
  const bool usual = rows <= all_few * batch;
  const bool narrow = rows <= FEW / 2 * batch || (!usual && group <= FEW / 2);
  Choice c;
  const int64_t reach = window > 0 ? std::min(capacity, window + most / group) : capacity;   // tokens that its rows may walk through
  c.chunks = may_chunk && !(usual && (most <= one_few || most * reach <= MOST));
  c.few = !c.chunks ? std::numeric_limits<int>::max() : usual ? one_few : batch < MANY ? 0 : narrow ? FEW / 2 : FEW;
  if (c.few < group) c.few = 0;            // (no sequence has so few)
  c.tile_rows = c.few == 0 ? 0 : narrow ? FEW / 2 : FEW;
  return c;
}
int64_t workspace_bytes_of(int64_t dim, bool chunks) {
  return kPagedHeader + paged_rows_parts_bytes(dim) + (chunks ? paged_chunk_parts_bytes(dim) : 0);
}

// A cache of 16-bit elements, or in 4 bits (its scales and the elements of a group of them)
struct CacheViews {
  const View4 &k, &v;
  const View4 *k_scales, *v_scales;
  int32_t group;
};

template <typename T>
int attend(const View3& q, const CacheViews& cache, const View2& table, const View1* offsets, const View1& lengths, const View3& out,
           int32_t scale_bits, int32_t window, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  const View4 &k_cache = cache.k, &v_cache = cache.v;
  const bool int4 = cache.k_scales != nullptr;
  const int64_t tokens = q.d0, heads = q.d1, dim = q.d2, pages = k_cache.d0, k_heads = k_cache.d1, page = k_cache.d2;
  const int64_t batch = lengths.d0;
  if (tokens < 0 || batch < 0 || heads <= 0 || k_heads <= 0 || heads % k_heads != 0 || v_cache.d0 != pages ||
      v_cache.d1 != k_heads || v_cache.d2 != page || (!int4 && (k_cache.d3 != dim || v_cache.d3 != dim)) || table.d0 != batch ||
      out.d0 != tokens || out.d1 != heads || out.d2 != dim || (offsets ? offsets->d0 != batch + 1 : tokens != batch))
    return INTENT_B200_ERR_SHAPE;
  if (dim != 64 && dim != 128) return INTENT_B200_ERR_UNSUPPORTED;
  if (page < 16 || page > 256 || (page & (page - 1)) != 0 || window < 0) return INTENT_B200_ERR_UNSUPPORTED;
  if (int4) {
    const int status = check_int4(k_cache, *cache.k_scales, v_cache, *cache.v_scales, k_heads, dim, cache.group);
    if (status != INTENT_B200_OK) return status;
  }
  constexpr int64_t kMost = (int64_t(1) << 31) - 1, kHalf = int64_t(1) << 30;   // (differences of positions are 32 bits, too)
  if (heads > 4096 || batch > (1 << 24) || tokens > kHalf / heads || pages > kMost / (k_heads * page) || table.d1 > kHalf / page)
    return INTENT_B200_ERR_UNSUPPORTED;
  float scale;
  std::memcpy(&scale, &scale_bits, sizeof(float));
  if (scale == 0.f) scale = 1.f / std::sqrt(float(dim));
  if (!(scale > 0.f) || std::isinf(scale) || (int4 && scale > kInt4Scale)) return INTENT_B200_ERR_UNSUPPORTED;
  if (!rows16(q) || !contiguous(k_cache) || !contiguous(v_cache) || !contiguous(table) || !contiguous(lengths) ||
      !contiguous(out) || (offsets && !contiguous(*offsets)) || !aligned16(q.p) || !aligned16(k_cache.p) ||
      !aligned16(v_cache.p) || !aligned16(out.p))
    return INTENT_B200_ERR_LAYOUT;
  if (tokens == 0 || batch == 0) return INTENT_B200_OK;
  if (!q.p || !out.p || !lengths.p || (offsets && !offsets->p)) return INTENT_B200_ERR_NULL;
  if (pages == 0 || table.d1 == 0) {     // no token anywhere
    if (observe_sink()) return INTENT_B200_OK;
    return cuda_status(cudaMemsetAsync(out.p, 0, size_t(tokens * heads * dim) * 2, stream));
  }
  if (!k_cache.p || !v_cache.p || !table.p || (int4 && (!cache.k_scales->p || !cache.v_scales->p))) return INTENT_B200_ERR_NULL;
  PagedParams p = {};
  p.q = static_cast<const uint16_t*>(q.p);
  p.q_token = q.s0, p.q_head = q.s1;
  p.out = static_cast<uint16_t*>(out.p);
  p.page_table = static_cast<const int32_t*>(table.p);
  p.offsets = offsets ? static_cast<const int32_t*>(offsets->p) : nullptr;
  p.lengths = static_cast<const int32_t*>(lengths.p);
  p.tokens = int(tokens), p.batch = int(batch), p.q_heads = int(heads), p.k_heads = int(k_heads);
  p.group = int(heads / k_heads);
  p.table_width = int(table.d1), p.pages = int(pages), p.capacity = int(table.d1 * page);
  while ((int64_t(1) << p.page_shift) < page) ++p.page_shift;
  p.window = window < p.capacity ? window : 0;   // (a query that sees as many tokens as there may be sees all)
  p.scale = scale * 1.44269504f;         // log2(e): the exponentials are powers of two
  const Choice choice = choose(tokens, batch, p.group, dim, p.capacity, p.window, offsets && paged_chunk_takes(p), int4);
  p.few = choice.few;
  if (!workspace || workspace_bytes < workspace_bytes_of(dim, choice.chunks)) return INTENT_B200_ERR_WORKSPACE;
  if (!aligned16(workspace)) return INTENT_B200_ERR_LAYOUT;
  const int sms = device_sms();
  if (sms <= 0) return INTENT_B200_ERR_CUDA;

  p.status = static_cast<int*>(workspace);
  p.joins = static_cast<unsigned char*>(workspace) + kPagedRowsJoins;
  p.parts = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kPagedHeader);
  const WorkspaceTurn turn(workspace);
  const int grid = std::min(sms, kPagedCtas);
  PagedParams chunk = p;
  const Int4Cache codes = {k_cache.p, int4 ? cache.k_scales->p : nullptr, v_cache.p, int4 ? cache.v_scales->p : nullptr, cache.group};
  if (choice.tile_rows > 0) {
    const int four = tokens * p.group <= 4 * batch ? 4 : choice.tile_rows;     // (rows of a tile; its parts are laid out as of eight)
    const int status = int4 ? paged_rows_int4<T>(p, dim, four, codes, grid, stream)
                            : paged_rows<T>(p, dim, choice.tile_rows, k_cache.p, v_cache.p, grid, stream);
    if (status != INTENT_B200_OK) return status;
  }
  if (choice.chunks) {
    chunk.joins = static_cast<unsigned char*>(workspace) + kPagedChunkJoins;
    chunk.parts += paged_rows_parts_bytes(dim) / int64_t(sizeof(float));
    chunk.half_tokens = paged_chunk_half_tokens(p);
    const int status = int4 ? paged_chunk_int4<T>(chunk, dim, codes, grid, stream)
                            : paged_chunk<T>(chunk, dim, k_cache.p, v_cache.p, grid, stream);
    if (status != INTENT_B200_OK) return status;
  }
  return paged_join<T>(p, choice.tile_rows, chunk, choice.chunks, dim, grid, stream);
}

}  // namespace
}  // namespace ib200

extern "C" int64_t intent_b200_paged_attention_workspace_bytes(int64_t dim, int32_t single) {
  return ib200::workspace_bytes_of(dim, !single);
}
namespace ib200 {
namespace {
int64_t call_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t dim, int64_t capacity,
                             int64_t window, bool int4) {
  if (tokens <= 0 || batch <= 0 || k_heads <= 0 || q_heads < k_heads || q_heads > 4096 || capacity < 0 || window < 0) return 0;
  const int64_t group = q_heads / k_heads;
  PagedParams p = {};
  p.tokens = p.q_heads = 1, p.group = int(group);      // (what its strides may rule out asks for less)
  return workspace_bytes_of(dim, choose(tokens, batch, group, dim, capacity, window, paged_chunk_takes(p), int4).chunks);
}
}  // namespace
}  // namespace ib200

// The same for one call of paged_attention (of paged_attention_int4): with few rows it needs as much as single tokens do.
extern "C" int64_t intent_b200_paged_attention_call_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads,
                                                                    int64_t dim, int64_t capacity, int64_t window) {
  return ib200::call_workspace_bytes(tokens, batch, q_heads, k_heads, dim, capacity, window, false);
}
extern "C" int64_t intent_b200_paged_attention_int4_call_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads,
                                                                         int64_t dim, int64_t capacity, int64_t window) {
  return ib200::call_workspace_bytes(tokens, batch, q_heads, k_heads, dim, capacity, window, true);
}

// Reads the status word at the head of a workspace after synchronising `stream`, and clears it.
extern "C" int intent_b200_paged_attention_workspace_status(void* workspace, int64_t workspace_bytes, void* stream) {
  if (!workspace || workspace_bytes < ib200::kPagedHeader) return INTENT_B200_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int value = 0;
  cudaError_t e = cudaStreamSynchronize(s);
  if (e == cudaSuccess) e = cudaMemcpy(&value, workspace, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && value != 0) {
    e = cudaMemsetAsync(workspace, 0, size_t(ib200::kPagedHeader), s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  return e == cudaSuccess ? value : ib200::cuda_status(e);
}

#define IB200_PAGED_TAIL int32_t window, void *workspace, int64_t workspace_bytes, void *stream
#define IB200_PAGED_ENTRIES(NAME, TYPE)                                                                                    \
  extern "C" int intent_b200_paged_attention_##NAME(                                                                       \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW2(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW1(a5), INTENT_B200_VIEW3(a6), int32_t scale_bits, IB200_PAGED_TAIL) {                                \
    const ib200::View4 k = IB200_VIEW4_ARG(a1), v = IB200_VIEW4_ARG(a2);                                                   \
    const ib200::View1 offsets = IB200_VIEW1_ARG(a4);                                                                      \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), {k, v, nullptr, nullptr, 0}, IB200_VIEW2_ARG(a3), &offsets,            \
                               IB200_VIEW1_ARG(a5), IB200_VIEW3_ARG(a6), scale_bits, window, workspace, workspace_bytes,   \
                               static_cast<cudaStream_t>(stream));                                                         \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_decode_attention_##NAME(                                                                \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW2(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW3(a5), int32_t scale_bits, IB200_PAGED_TAIL) {                                                       \
    const ib200::View4 k = IB200_VIEW4_ARG(a1), v = IB200_VIEW4_ARG(a2);                                                   \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), {k, v, nullptr, nullptr, 0}, IB200_VIEW2_ARG(a3), nullptr,             \
                               IB200_VIEW1_ARG(a4), IB200_VIEW3_ARG(a5), scale_bits, window, workspace, workspace_bytes,   \
                               static_cast<cudaStream_t>(stream));                                                         \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_attention_int4_##NAME(                                                                  \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW4(a3), INTENT_B200_VIEW4(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW1(a6), INTENT_B200_VIEW1(a7), INTENT_B200_VIEW3(a8), int32_t group,           \
      int32_t scale_bits, IB200_PAGED_TAIL) {                                                                              \
    const ib200::View4 k = IB200_VIEW4_ARG(a1), ks = IB200_VIEW4_ARG(a2), v = IB200_VIEW4_ARG(a3), vs = IB200_VIEW4_ARG(a4); \
    const ib200::View1 offsets = IB200_VIEW1_ARG(a6);                                                                      \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), {k, v, &ks, &vs, group}, IB200_VIEW2_ARG(a5), &offsets,                \
                               IB200_VIEW1_ARG(a7), IB200_VIEW3_ARG(a8), scale_bits, window, workspace, workspace_bytes,   \
                               static_cast<cudaStream_t>(stream));                                                         \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_decode_attention_int4_##NAME(                                                           \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW4(a3), INTENT_B200_VIEW4(a4),   \
      INTENT_B200_VIEW2(a5), INTENT_B200_VIEW1(a6), INTENT_B200_VIEW3(a7), int32_t group, int32_t scale_bits,              \
      IB200_PAGED_TAIL) {                                                                                                  \
    const ib200::View4 k = IB200_VIEW4_ARG(a1), ks = IB200_VIEW4_ARG(a2), v = IB200_VIEW4_ARG(a3), vs = IB200_VIEW4_ARG(a4); \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), {k, v, &ks, &vs, group}, IB200_VIEW2_ARG(a5), nullptr,                 \
                               IB200_VIEW1_ARG(a6), IB200_VIEW3_ARG(a7), scale_bits, window, workspace, workspace_bytes,   \
                               static_cast<cudaStream_t>(stream));                                                         \
  }
IB200_PAGED_ENTRIES(f16, __half)
IB200_PAGED_ENTRIES(bf16, __nv_bfloat16)
