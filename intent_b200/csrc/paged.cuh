// What the kernels of attention over a paged cache share.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace ib200 {

constexpr int kPagedCtas = 160;            // most CTAs of a launch
// The workspace: status word; descriptions of the tile that each CTA leaves to others, those of the rows kernel, then those of the
// chunk kernel; parts of the rows kernel, then those of the chunk kernel
constexpr int64_t kPagedEntry = 24;        // bytes of a description, at most
constexpr int64_t kPagedRowsJoins = 64, kPagedChunkJoins = kPagedRowsJoins + kPagedEntry * kPagedCtas, kPagedHeader = 8192;
static_assert(kPagedChunkJoins + kPagedEntry * kPagedCtas <= kPagedHeader, "room ahead of the parts");

struct PagedParams {
  const uint16_t* q;                 // [T, HQ, D] at these strides (elements)
  int64_t q_token, q_head;
  uint16_t* out;                     // [T, HQ, D]
  const int32_t* page_table;         // [B, table_width]
  const int32_t* offsets;            // [B + 1] rows of q of every sequence; null: row b is sequence b's only one
  const int32_t* lengths;            // [B] tokens in the cache, the new ones among them
  int tokens, batch, q_heads, k_heads, group, table_width;
  int pages, page_shift, capacity;   // capacity: tokens that a row of the page table can name
  int window;                        // tokens that a query sees, its own among them; 0 = all
  float scale;                       // of the scores, times log2(e)
  int* status;                       // head of the workspace
  void* joins;                       // a kernel's own
  float* parts;
  int half_tokens;                   // chunks: tokens of half a tile
  int few;                           // rows of queries per key head up to which a sequence is the rows kernel's; those with more
                                     // are the chunk kernel's (either may get all: INT_MAX, 0)
};

// Checks of a cache in 4 bits: codes [PAGES, HK, PAGE, D / 2] of 8 bits, scales [PAGES, HK, PAGE, 2 D / GROUP] of the 16-bit type.
inline int check_int4(const View4& k_codes, const View4& k_scales, const View4& v_codes, const View4& v_scales, int64_t heads,
                      int64_t dim, int32_t group) {
  if (group != 32 && group != 64 && group != 128) return INTENT_B200_ERR_UNSUPPORTED;
  if (group > dim) return INTENT_B200_ERR_UNSUPPORTED;
  const int64_t pages = k_codes.d0, page = k_codes.d2;
  for (const View4* v : {&k_codes, &v_codes, &k_scales, &v_scales})
    if (v->d0 != pages || pages < 0 || v->d1 != heads || v->d2 != page) return INTENT_B200_ERR_SHAPE;
  if (k_codes.d3 * 2 != dim || v_codes.d3 * 2 != dim || k_scales.d3 * group != 2 * dim || v_scales.d3 * group != 2 * dim)
    return INTENT_B200_ERR_SHAPE;
  if (page < 16 || page > 256 || (page & (page - 1)) != 0 || pages > (int64_t(1) << 40) / page) return INTENT_B200_ERR_UNSUPPORTED;
  for (const View4* v : {&k_codes, &v_codes, &k_scales, &v_scales})
    if (!contiguous(*v) || !aligned16(v->p)) return INTENT_B200_ERR_LAYOUT;
  return INTENT_B200_OK;
}

#ifdef __CUDACC__

template <bool B>
using Bool = std::integral_constant<bool, B>;

struct TokenSpan {
  int begin, count;
};
// rows of q of a sequence; offsets that make no sense are cut to the rows there are
__device__ __forceinline__ TokenSpan span_of(const PagedParams& p, int b) {
  if (!p.offsets) return {b, 1};
  const int begin = min(max(__ldg(p.offsets + b), 0), p.tokens);
  return {begin, min(max(__ldg(p.offsets + b + 1), begin), p.tokens) - begin};
}

// Places of a CTA, of a line of so many; negative where a CTA has no count for them.  (The line is in 64 bits: 2^20 new tokens of 64
// heads on 8 are 2^30 places.  Within a CTA places are counted from its first one, in 32.)
__device__ __forceinline__ int share_of(long long line) {
  constexpr int MOST = 0x3fffffff;
  if (line <= MOST) return (int(line) + int(gridDim.x) - 1) / int(gridDim.x);
  const long long share = (line + gridDim.x - 1) / gridDim.x;
  return share <= MOST ? int(share) : -1;
}
__device__ __forceinline__ int divide(long long a, long long b) {     // for quotients of 31 bits
  return (a | b) >> 31 == 0 ? int(unsigned(a) / unsigned(b)) : int(a / b);
}

// The factor of a row whose weights add up to nothing: zero where it sees no token; where it does, all its scores are -infinity,
// and their softmax is no number.  `row`: of q.
__device__ __forceinline__ float of_nothing(const PagedParams& p, int b, int row) {
  const TokenSpan span = span_of(p, b);
  const int position = min(max(__ldg(p.lengths + b), 0), p.capacity) - span.count + row - span.begin;
  const int from = p.window > 0 ? max(position - p.window + 1, 0) : 0;
#pragma unroll 1
  for (int i = from >> p.page_shift; i <= position >> p.page_shift; ++i) {
    const int page = __ldg(p.page_table + int64_t(b) * p.table_width + i);
    if (page >= 0 && page < p.pages) return __int_as_float(0x7fc00000);
  }
  return 0.f;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x * 0 + sum for a pair of 16-bit numbers: NaN where x is no finite number
template <typename T>
__device__ __forceinline__ uint32_t add_no_numbers(uint32_t x, uint32_t sum) {
  if (std::is_same<T, __half>::value) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
  else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0u));
  return sum;
}

#endif  // __CUDACC__

// few rows per sequence, in tiles of so many (8 or 16; paged_rows.cu)
int64_t paged_rows_parts_bytes(int64_t dim);
template <typename T>
int paged_rows(const PagedParams& p, int64_t dim, int tile_rows, const void* k_cache, const void* v_cache, int grid,
               cudaStream_t stream);

// the same over a cache in 4 bits (paged_rows_int4.cu)
struct Int4Cache {
  const void *k_codes, *k_scales, *v_codes, *v_scales;
  int group;
};
template <typename T>
int paged_rows_int4(const PagedParams& p, int64_t dim, int tile_rows, const Int4Cache& cache, int grid, cudaStream_t stream);

// chunks (paged_chunk.cu)
int64_t paged_chunk_parts_bytes(int64_t dim);
bool paged_chunk_takes(const PagedParams& p);
int paged_chunk_half_tokens(const PagedParams& p);
template <typename T>
int paged_chunk(const PagedParams& p, int64_t dim, const void* k_cache, const void* v_cache, int grid, cudaStream_t stream);
template <typename T>
int paged_chunk_int4(const PagedParams& p, int64_t dim, const Int4Cache& cache, int grid, cudaStream_t stream);

// the parts that paged_rows (tile_rows > 0) and paged_chunk (`chunks`) leave (paged_join.cu)
template <typename T>
int paged_join(const PagedParams& rows, int tile_rows, const PagedParams& chunk, bool chunks, int64_t dim, int grid,
               cudaStream_t stream);

}  // namespace ib200
