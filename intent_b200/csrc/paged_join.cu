// Joins of attention over a paged cache: the parts of the tiles that CTA boundaries cut, added in the CTAs' order.
#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"

namespace ib200 {
namespace {

template <int ROWS>
struct JoinRoom {
  float maxima[kPagedCtas][ROWS], sums[kPagedCtas][ROWS];
};

// A block per CTA in which such a tile begins, a thread per row and four elements (more threads than that are left over).
// What it costs is the latency of dependent reads: all maxima and sums are read at once, then the results of eight parts at a time.
// (When the CTA that finished a tile last did this, one multiprocessor had 16 rows of 16 parts to read: four tokens behind 8000,
// 32 heads on 8, took 31 us a call; with a kernel of its own 17.)
template <typename T, int D, int ROWS>
__device__ __forceinline__ void join_rows(const PagedParams& p, JoinRoom<ROWS>& room) {
  const RowsJoin entry = static_cast<const RowsJoin*>(p.joins)[blockIdx.x];
  const int first = blockIdx.x, count = entry.last_cta - first + 1, r = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
  if (entry.last_cta < 0) return;
  constexpr size_t SIZE = size_t(ROWS) * (D + 2);
  const float infinity = __int_as_float(0x7f800000);
  auto part = [&](int v) { return p.parts + (2 * (first + v) + (v == 0)) * SIZE; };
  for (int i = threadIdx.x; i < count * ROWS; i += blockDim.x) {
    const int v = i / ROWS, row = i % ROWS;
    room.maxima[v][row] = row < entry.rows ? __ldcg(part(v) + ROWS * D + row) : -infinity;
    room.sums[v][row] = row < entry.rows ? __ldcg(part(v) + ROWS * (D + 1) + row) : 0.f;
  }
  __syncthreads();
  if (r >= entry.rows) return;
  float m = -infinity, l = 0.f, x[4] = {};
  for (int v = 0; v < count; ++v) m = fmaxf(m, room.maxima[v][r]);
  const float origin = m == -infinity ? 0.f : m;
#pragma unroll 1
  for (int from = 0; from < count; from += 8) {
    float4 y[8];
#pragma unroll
    for (int v = 0; v < 8; ++v)
      if (from + v < count) y[v] = __ldcg(reinterpret_cast<const float4*>(part(from + v) + r * D) + c);
#pragma unroll
    for (int v = 0; v < 8; ++v) {
      if (from + v >= count) break;
      const float f = exp2_fast(room.maxima[from + v][r] - origin);
      l = fmaf(room.sums[from + v][r], f, l);
      x[0] = fmaf(y[v].x, f, x[0]), x[1] = fmaf(y[v].y, f, x[1]), x[2] = fmaf(y[v].z, f, x[2]), x[3] = fmaf(y[v].w, f, x[3]);
    }
  }
  const int token = (entry.tile_row + r) / p.group, of_group = entry.tile_row + r - token * p.group;
  const float inverse = l == 0.f ? of_nothing(p, entry.sequence, entry.row + token) : 1.f / l;
  *reinterpret_cast<uint2*>(p.out + (int64_t(entry.row + token) * p.q_heads + entry.head * p.group + of_group) * D + 4 * c) =
      make_uint2(Elem<T>::pack2(x[0] * inverse, x[1] * inverse), Elem<T>::pack2(x[2] * inverse, x[3] * inverse));
}

// Block (cta, 32 rows) of 4 D threads, a thread per row and eight elements.  What it costs is the latency of dependent reads (0.5 us
// each): the maxima and sums of all parts are read at once, by all warps, and the results four parts at a time (8 tiles of 16
// parts, 33 tokens behind 7967, a call alone: 39.7 us; with two at a time and sixteen elements per thread 40.4).
template <typename T, int D>
__device__ __forceinline__ void join_chunk(const PagedParams& p, JoinRoom<32>& room) {
  constexpr int WARPS = D / 8;
  const ChunkJoin entry = static_cast<const ChunkJoin*>(p.joins)[blockIdx.x];
  const int first = blockIdx.x, count = entry.last_cta - first + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.y * 32 + lane;
  const int of_half = row % HALF_ROWS, row_token = of_half / p.group, token = row / HALF_ROWS * p.half_tokens + row_token;
  const bool real = row_token < p.half_tokens && token < entry.tokens;
  if (entry.last_cta < 0 || !__any_sync(0xffffffffu, real)) return;    // (all warps have the same rows)
  constexpr size_t SIZE = size_t(2 * HALF_ROWS) * (D + 2);
  const float infinity = __int_as_float(0x7f800000);
  auto part = [&](int v) { return p.parts + (2 * (first + v) + (v == 0)) * SIZE; };
#pragma unroll 4
  for (int v = warp; v < count; v += WARPS) {
    room.maxima[v][lane] = real ? __ldcg(part(v) + 2 * HALF_ROWS * D + row) : -infinity;
    room.sums[v][lane] = real ? __ldcg(part(v) + 2 * HALF_ROWS * (D + 1) + row) : 0.f;
  }
  __syncthreads();
  if (!real) return;
  float m = -infinity, l = 0.f, x[8] = {};
  for (int v = 0; v < count; ++v) m = fmaxf(m, room.maxima[v][lane]);
  const float origin = m == -infinity ? 0.f : m;
#pragma unroll 1
  for (int from = 0; from < count; from += 4) {
    float4 y[4][2];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (from + v < count) y[v][e] = __ldcg(reinterpret_cast<const float4*>(part(from + v)) + (2 * warp + e) * 2 * HALF_ROWS + row);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (from + v >= count) break;
      const float f = exp2_fast(room.maxima[from + v][lane] - origin);
      l = fmaf(room.sums[from + v][lane], f, l);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[4 * e] = fmaf(y[v][e].x, f, x[4 * e]), x[4 * e + 1] = fmaf(y[v][e].y, f, x[4 * e + 1]);
        x[4 * e + 2] = fmaf(y[v][e].z, f, x[4 * e + 2]), x[4 * e + 3] = fmaf(y[v][e].w, f, x[4 * e + 3]);
      }
    }
  }
  const float inverse = l == 0.f ? of_nothing(p, entry.sequence, entry.row + token) : 1.f / l;
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = Elem<T>::pack2(x[2 * e] * inverse, x[2 * e + 1] * inverse);
  uint16_t* to = p.out + (int64_t(entry.row + token) * p.q_heads + entry.head * p.group + of_half - row_token * p.group) * D + 8 * warp;
  *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(ROWS * D / 4) paged_rows_join_kernel(const PagedParams p) {
  __shared__ JoinRoom<ROWS> room;
  programmatic_begin();
  programmatic_wait();
  join_rows<T, D, ROWS>(p, room);
}
template <typename T, int D>
__global__ void __launch_bounds__(4 * D, 1024 / (4 * D)) paged_chunk_join_kernel(const PagedParams p) {
  __shared__ JoinRoom<32> room;
  programmatic_begin();
  programmatic_wait();
  join_chunk<T, D>(p, room);
}
// both, in blocks of their own
constexpr unsigned CHUNK_BLOCKS = 2 * HALF_ROWS / 32;
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(4 * D, 1024 / (4 * D)) paged_joins_kernel(const PagedParams rows, const PagedParams chunk) {
  __shared__ union {
    JoinRoom<32> chunk;
    JoinRoom<ROWS> rows;
  } room;
  programmatic_begin();
  programmatic_wait();
  if (blockIdx.y == CHUNK_BLOCKS) join_rows<T, D, ROWS>(rows, room.rows);
  else join_chunk<T, D>(chunk, room.chunk);
}

template <typename T, int D>
cudaError_t launch(const PagedParams& rows, int tile_rows, const PagedParams& chunk, bool chunks, unsigned grid, cudaStream_t stream) {
  if (!chunks)
    return launch_programmatic(tile_rows == 8 ? paged_rows_join_kernel<T, D, 8> : paged_rows_join_kernel<T, D, 16>, dim3(grid),
                               dim3(unsigned(tile_rows) * D / 4), 0, stream, 1, rows);
  if (tile_rows == 0)
    return launch_programmatic(paged_chunk_join_kernel<T, D>, dim3(grid, CHUNK_BLOCKS), dim3(4 * D), 0, stream, 1, chunk);
  return launch_programmatic(tile_rows == 8 ? paged_joins_kernel<T, D, 8> : paged_joins_kernel<T, D, 16>,
                             dim3(grid, CHUNK_BLOCKS + 1), dim3(4 * D), 0, stream, 1, rows, chunk);
}

}  // namespace

template <typename T>
int paged_join(const PagedParams& rows, int tile_rows, const PagedParams& chunk, bool chunks, int64_t dim, int grid, cudaStream_t stream) {
  if (observe_sink()) return INTENT_B200_OK;
  const cudaError_t e = dim == 128 ? launch<T, 128>(rows, tile_rows, chunk, chunks, unsigned(grid), stream)
                                   : launch<T, 64>(rows, tile_rows, chunk, chunks, unsigned(grid), stream);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}
template int paged_join<__half>(const PagedParams&, int, const PagedParams&, bool, int64_t, int, cudaStream_t);
template int paged_join<__nv_bfloat16>(const PagedParams&, int, const PagedParams&, bool, int64_t, int, cudaStream_t);

}  // namespace ib200
