// What the kernels for few rows of queries share: the line of steps and its cut into equal parts.
#pragma once

#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"

namespace ib200 {

#ifdef __CUDACC__

constexpr float SLACK = 8.f;             // growth of a row's maximum (log2) that its weights are left to absorb

// One sequence's share of the line of steps
struct Sequence {
  int rows;        // query rows of a key head: new tokens x group
  int first_row;   // its first token among all
  int length;      // tokens in the cache
  int first;       // position of its first query
  int low;         // first token that any of its queries sees
  int begin;       // first step
  int steps;       // of a row tile, one at least: a tile without tokens writes zeros
  int tiles;       // row tiles of a key head
};

template <int STEP>
__device__ __forceinline__ Sequence sequence_of(const PagedParams& p, int b, int tile_rows) {
  Sequence s;
  const TokenSpan span = span_of(p, b);
  s.rows = span.count * p.group <= p.few ? span.count * p.group : 0;
  s.first_row = span.begin;
  s.length = min(max(__ldg(p.lengths + b), 0), p.capacity);
  s.first = s.length - span.count;
  s.low = p.window > 0 ? min(max(s.first - p.window + 1, 0), s.length) : 0;
  s.begin = s.low / STEP;
  s.steps = max((s.length + STEP - 1) / STEP - s.begin, 1);
  s.tiles = (s.rows + tile_rows - 1) / tile_rows;
  return s;
}

// Places of a sequence on the line
template <int BEGIN>
__device__ __forceinline__ long long places_of(const PagedParams& p, const Sequence& s) {
  return (long long)s.tiles * p.k_heads * (s.steps + BEGIN);
}

// A step on the line
template <int STEP, int BEGIN>
struct Walk {
  Sequence s;
  int b, head, tile, step;
  // how many places on the next one is
  __device__ __forceinline__ int distance() const { return step + 1 < s.steps ? 1 : 1 + BEGIN; }
  __device__ __forceinline__ void advance(const PagedParams& p, int tile_rows) {
    if (++step < s.steps) return;
    step = 0;
    if (++tile < s.tiles) return;
    tile = 0;
    if (++head < p.k_heads) return;
    head = 0;
    do {
      if (++b >= p.batch) return;
      s = sequence_of<STEP>(p, b, tile_rows);
    } while (s.tiles == 0);
  }
};

// The part of the line that a CTA, or one of its warps, takes
template <int STEP, int BEGIN>
struct Place {
  Walk<STEP, BEGIN> at;    // its first step
  int first, end;          // its place and where the part's places end, counted from the part's first one (first >= end: none)
  int share;               // places of every part
};

// The parts of a line of so many places that WORKERS of every CTA take, one behind the other; negative as in share_of
template <int WORKERS>
__device__ __forceinline__ int share_of_workers(long long line) {
  if (WORKERS == 1) return share_of(line);
  constexpr int MOST = 0x3fffffff / WORKERS;             // (a CTA's places are counted in 32 bits)
  const long long workers = (long long)gridDim.x * WORKERS, share = (line + workers - 1) / workers;
  return share <= MOST ? int(share) : -1;
}

// To be called by all threads of a CTA.  `starts` has room for two 64-bit numbers of every worker (the CTA, or each of its warps),
// `warp_sums` for one a warp.
template <int STEP, int BEGIN, int THREADS, int WORKERS>
__device__ __forceinline__ Place<STEP, BEGIN> place_of(const PagedParams& p, int tile_rows, long long* starts, long long* warp_sums,
                                                       RowsJoin* entry) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, worker = WORKERS == 1 ? 0 : warp;
  Place<STEP, BEGIN> place;
  place.first = place.end = 0;
  const int per_thread = (p.batch + THREADS - 1) / THREADS, mine = tid * per_thread;
  long long sum = 0;
  for (int b = mine; b < min(mine + per_thread, p.batch); ++b) {
    const Sequence s = sequence_of<STEP>(p, b, tile_rows);
    sum += places_of<BEGIN>(p, s);
  }
  long long before = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += v;
  }
  if (lane == 31) warp_sums[warp] = before;
  __syncthreads();
  long long line = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    line += warp_sums[w];
  }
  before -= sum;
  place.share = share_of_workers<WORKERS>(line);
  if (tid == 0) {
    entry->last_cta = -1;
    if (place.share < 0) atomicExch(p.status, INTENT_B200_ERR_SHAPE);
  }
  const long long first_of_cta = (long long)blockIdx.x * WORKERS * place.share;
  if (place.share <= 0 || first_of_cta >= line) return place;
#pragma unroll 1
  for (int i = 0; i < WORKERS; ++i) {
    const long long begin = first_of_cta + (long long)i * place.share;
    if (begin >= before && begin < before + sum) {
      int b = mine;
      long long at = before;
      for (; per_thread > 1; ++b) {
        const Sequence s = sequence_of<STEP>(p, b, tile_rows);
        const long long places = places_of<BEGIN>(p, s);
        if (begin < at + places || b + 1 >= min(mine + per_thread, p.batch)) break;
        at += places;
      }
      starts[2 * i] = b;
      starts[2 * i + 1] = begin - at;                    // place in the sequence
    }
  }
  __syncthreads();
  const long long begin = first_of_cta + (long long)worker * place.share;
  if (begin >= line) return place;
  place.end = int(min((long long)place.share, line - begin));
  Walk<STEP, BEGIN>& first = place.at;
  first.b = int(starts[2 * worker]);
  first.s = sequence_of<STEP>(p, first.b, tile_rows);
  const long long of_sequence = starts[2 * worker + 1];
  const int item = divide(of_sequence, first.s.steps + BEGIN);
  first.step = int(of_sequence - (long long)item * (first.s.steps + BEGIN)) - BEGIN;
  first.head = item / first.s.tiles;
  first.tile = item - first.head * first.s.tiles;
  place.first = max(-first.step, 0);                     // of a step
  first.step = max(first.step, 0);
  return place;
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

#endif  // __CUDACC__

}  // namespace ib200
