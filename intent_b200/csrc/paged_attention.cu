// Entries of attention over a paged cache: argument checks and the choice of the kernel.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <limits>

#include "paged.cuh"

namespace ib200 {
namespace {

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
struct Choice {
  int tile_rows;           // of the rows kernel; 0: it is not needed
  int few;                 // rows up to which a sequence is its
  bool chunks;             // the chunk kernel is needed
};
Choice choose(int64_t tokens, int64_t batch, int64_t group, int64_t dim, int64_t capacity, int64_t window, bool may_chunk) {
  constexpr int FEW = 16, MANY = 8, MOST = 1 << 20;
  const int64_t rows = tokens * group, most = tokens < batch ? rows : (tokens - batch + 1) * group;
  const bool usual = rows <= (dim == 64 ? 2 * FEW : FEW) * batch;
  const bool narrow = rows <= FEW / 2 * batch || (!usual && group <= FEW / 2);
  Choice c;
  const int64_t reach = window > 0 ? std::min(capacity, window + most / group) : capacity;   // tokens that its rows may walk through
  c.chunks = may_chunk && !(usual && (most <= 2 * FEW || most * reach <= MOST));
  c.few = !c.chunks ? std::numeric_limits<int>::max() : usual ? 2 * FEW : batch < MANY ? 0 : narrow ? FEW / 2 : FEW;
  if (c.few < group) c.few = 0;            // (no sequence has so few)
  c.tile_rows = c.few == 0 ? 0 : narrow ? FEW / 2 : FEW;
  return c;
}
int64_t workspace_bytes_of(int64_t dim, bool chunks) {
  return kPagedHeader + paged_rows_parts_bytes(dim) + (chunks ? paged_chunk_parts_bytes(dim) : 0);
}

template <typename T>
int attend(const View3& q, const View4& k_cache, const View4& v_cache, const View2& table, const View1* offsets,
           const View1& lengths, const View3& out, int32_t scale_bits, int32_t window, void* workspace, int64_t workspace_bytes,
           cudaStream_t stream) {
  const int64_t tokens = q.d0, heads = q.d1, dim = q.d2, pages = k_cache.d0, k_heads = k_cache.d1, page = k_cache.d2;
  const int64_t batch = lengths.d0;
  if (tokens < 0 || batch < 0 || heads <= 0 || k_heads <= 0 || heads % k_heads != 0 || k_cache.d3 != dim || v_cache.d0 != pages ||
      v_cache.d1 != k_heads || v_cache.d2 != page || v_cache.d3 != dim || table.d0 != batch || out.d0 != tokens ||
      out.d1 != heads || out.d2 != dim || (offsets ? offsets->d0 != batch + 1 : tokens != batch))
    return INTENT_B200_ERR_SHAPE;
  if (dim != 64 && dim != 128) return INTENT_B200_ERR_UNSUPPORTED;
  if (page < 16 || page > 256 || (page & (page - 1)) != 0 || window < 0) return INTENT_B200_ERR_UNSUPPORTED;
  constexpr int64_t kMost = (int64_t(1) << 31) - 1, kHalf = int64_t(1) << 30;   // (differences of positions are 32 bits, too)
  if (heads > 4096 || batch > (1 << 24) || tokens > kHalf / heads || pages > kMost / (k_heads * page) || table.d1 > kHalf / page)
    return INTENT_B200_ERR_UNSUPPORTED;
  float scale;
  std::memcpy(&scale, &scale_bits, sizeof(float));
  if (scale == 0.f) scale = 1.f / std::sqrt(float(dim));
  if (!(scale > 0.f) || std::isinf(scale)) return INTENT_B200_ERR_UNSUPPORTED;
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
  if (!k_cache.p || !v_cache.p || !table.p) return INTENT_B200_ERR_NULL;
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
  const Choice choice = choose(tokens, batch, p.group, dim, p.capacity, p.window, offsets && paged_chunk_takes(p));
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
  if (choice.tile_rows > 0) {
    const int status = paged_rows<T>(p, dim, choice.tile_rows, k_cache.p, v_cache.p, grid, stream);
    if (status != INTENT_B200_OK) return status;
  }
  if (choice.chunks) {
    chunk.joins = static_cast<unsigned char*>(workspace) + kPagedChunkJoins;
    chunk.parts += paged_rows_parts_bytes(dim) / int64_t(sizeof(float));
    chunk.half_tokens = paged_chunk_half_tokens(p);
    const int status = paged_chunk<T>(chunk, dim, k_cache.p, v_cache.p, grid, stream);
    if (status != INTENT_B200_OK) return status;
  }
  return paged_join<T>(p, choice.tile_rows, chunk, choice.chunks, dim, grid, stream);
}

}  // namespace
}  // namespace ib200

extern "C" int64_t intent_b200_paged_attention_workspace_bytes(int64_t dim, int32_t single) {
  return ib200::workspace_bytes_of(dim, !single);
}
// The same for one call of paged_attention: with few rows it needs as much as single tokens do.
extern "C" int64_t intent_b200_paged_attention_call_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads,
                                                                    int64_t dim, int64_t capacity, int64_t window) {
  if (tokens <= 0 || batch <= 0 || k_heads <= 0 || q_heads < k_heads || q_heads > 4096 || capacity < 0 || window < 0) return 0;
  const int64_t group = q_heads / k_heads;
  ib200::PagedParams p = {};
  p.tokens = p.q_heads = 1, p.group = int(group);      // (what its strides may rule out asks for less)
  return ib200::workspace_bytes_of(dim, ib200::choose(tokens, batch, group, dim, capacity, window, ib200::paged_chunk_takes(p)).chunks);
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

#define IB200_PAGED_ENTRIES(NAME, TYPE)                                                                                    \
  extern "C" int intent_b200_paged_attention_##NAME(                                                                       \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW2(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW1(a5), INTENT_B200_VIEW3(a6), int32_t scale_bits, int32_t window, void* workspace,                   \
      int64_t workspace_bytes, void* stream) {                                                                             \
    const ib200::View1 offsets = IB200_VIEW1_ARG(a4);                                                                      \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW4_ARG(a1), IB200_VIEW4_ARG(a2), IB200_VIEW2_ARG(a3),         \
                               &offsets, IB200_VIEW1_ARG(a5), IB200_VIEW3_ARG(a6), scale_bits, window, workspace,          \
                               workspace_bytes, static_cast<cudaStream_t>(stream));                                        \
  }                                                                                                                        \
  extern "C" int intent_b200_paged_decode_attention_##NAME(                                                                \
      INTENT_B200_VIEW3(a0), INTENT_B200_VIEW4(a1), INTENT_B200_VIEW4(a2), INTENT_B200_VIEW2(a3), INTENT_B200_VIEW1(a4),   \
      INTENT_B200_VIEW3(a5), int32_t scale_bits, int32_t window, void* workspace, int64_t workspace_bytes, void* stream) { \
    return ib200::attend<TYPE>(IB200_VIEW3_ARG(a0), IB200_VIEW4_ARG(a1), IB200_VIEW4_ARG(a2), IB200_VIEW2_ARG(a3),         \
                               nullptr, IB200_VIEW1_ARG(a4), IB200_VIEW3_ARG(a5), scale_bits, window, workspace,           \
                               workspace_bytes, static_cast<cudaStream_t>(stream));                                        \
  }
IB200_PAGED_ENTRIES(f16, __half)
IB200_PAGED_ENTRIES(bf16, __nv_bfloat16)
