// Attention over a paged cache for few rows of queries per sequence and key head: a decode step, or short chunks.
//
// Program (paged_decode_attention; paged_attention for chunks): query row x at position p of a sequence with n new tokens and
// L tokens in the cache (p = L - n + i), over the tokens j with max(0, p - W + 1) <= j <= p (W = 0: no window)
//   o = sum_j softmax_j(scale * x . k_j) * v_j,     zero where there is no such token, NaN where all scores are -infinity
// Token j of sequence b lies in page page_table[b, j / PAGE]; the tokens of a page number outside the cache are not seen.
// All statistics and sums are in f32; the weights of one product with V are rounded to the 16-bit type (relative to a maximum
// that a score may exceed by SLACK before it is raised, so at most 2^8), as the tensor core takes them.
//
// Bound by HBM: a token's keys and values (4 D bytes per key head) are read once for the whole group of query heads that share
// them.  What has to be right for that:
//  * Loads run ahead.  A warp has its own ring of three units of 32 tokens (16 KiB each with D = 128), filled by TMA through
//    128B-swizzled boxes of one page's rows, so that 192 KiB are asked for per SM whatever the warp is computing.
//  * Work is cut evenly, not by sequence.  All steps (32 tokens for each warp) of all (sequence, key head, row tile) form one
//    line, of which every CTA takes the same length; a long sequence is shared by many CTAs and a CTA goes through many short ones
//    while its ring runs on.  A row tile that was cut leaves its parts (maximum, sum, unscaled result) in the workspace,
//    which join_rows puts together in CTA order: the same bits in every launch.
//  * Few instructions per token.  Keys are the tensor core's A operand (16 tokens) and the queries its B operand (eight rows,
//    kept in registers): S^T = K Q^T, then O^T += V^T P^T with V^T from transposing loads and P^T from one movmatrix per
//    eight tokens.  With up to eight query heads per key head nothing is computed for rows that are not there.  A maximum is
//    shared between lanes only when it grows.
//
// Measured on one B200 (6530 GB/s copied): 64 histories of up to 8192 tokens, 32 heads of 128 on 8 key heads, bf16: 181 us, 6.24
// TB/s; 4 of up to 131072 on 4 key heads: 108 us, 5.9 TB/s; 200 of up to 2048, 16 heads of 64: 149 us, 5.9 TB/s.  One history of
// 1000 tokens, 7.9 us: the reads one after another of a launch (lengths, page numbers, keys, parts) and its join.
#include <cstring>

#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "tma.cuh"

namespace ib200 {
namespace {

constexpr int UNIT = 32;                 // tokens of a ring slot
constexpr float SLACK = 8.f;             // growth of a row's maximum (log2) that its weights are left to absorb

template <int D>
struct Ring {
  // Heads of 64 give a warp half the bytes for nearly the same instructions: with four warps, one per scheduler, their latency
  // was what bounded the kernel (200 histories of up to 2048 tokens, 16 heads: 211 us; with eight 149).
  static constexpr int WARPS = D == 128 ? 4 : 8;
  static constexpr int STAGES = 3;
  static constexpr int STEP = UNIT * WARPS;               // tokens of a CTA's step
  static constexpr int HALF = UNIT * 128;                 // 64 elements of every token of a unit
  static constexpr int OPERAND = HALF * (D / 64);         // keys or values of a unit
  static constexpr int SLOT = 2 * OPERAND;
  static constexpr int BYTES = WARPS * STAGES * SLOT;
  // Places on the line ahead of the steps of a tile, for what it costs beside them: with eight warps to put together about a
  // step's time (200 histories of up to 2048 tokens, 16 heads of 64: 154 us without, 149 with one, 151 with two); with four not
  // enough to show (64 histories of up to 8192, 8 heads of 128: 184 us without, 185 with one, 184 with two).
  static constexpr int BEGIN = D == 128 ? 0 : 1;
};

// Places for the warps' parts of a tile: two where there is room
template <int D, int NT>
constexpr int joins() {
  return NT == 2 ? 1 : 2;
}
template <int D, int NT>
constexpr int smem_bytes() {
  return 1024 + Ring<D>::BYTES + joins<D, NT>() * Ring<D>::WARPS * 8 * NT * (D * 4 + 8) +
         Ring<D>::WARPS * Ring<D>::STAGES * 8 + 16 + 8 * Ring<D>::WARPS;
}
static_assert(smem_bytes<128, 2>() <= 227 * 1024 && smem_bytes<128, 1>() <= 227 * 1024 && smem_bytes<64, 2>() <= 227 * 1024,
              "shared memory of a CTA");

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

template <typename T, int D, int NT>
__global__ void __launch_bounds__(32 * Ring<D>::WARPS, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PagedParams p) {
  using R = Ring<D>;
  constexpr int ROWS = 8 * NT, PITCH = D, WARPS = R::WARPS, THREADS = 32 * WARPS, STEP = R::STEP, BEGIN = R::BEGIN;
  extern __shared__ unsigned char smem_raw[];
  programmatic_begin();
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  constexpr int JOINS = joins<D, NT>();
  float* join = reinterpret_cast<float*>(base_ptr + R::BYTES);          // [JOINS][WARPS][ROWS][PITCH]
  float* join_max = join + JOINS * WARPS * ROWS * PITCH;                // [JOINS][WARPS][ROWS]
  float* join_sum = join_max + JOINS * WARPS * ROWS;
  int* shared = reinterpret_cast<int*>(join_sum + JOINS * WARPS * ROWS);   // a number, a 64-bit one, the warps' 64-bit sums
  long long* warp_sums = reinterpret_cast<long long*>(shared + 4);
  const uint32_t bars = smem_u32(warp_sums + WARPS);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = base + warp * R::STAGES * R::SLOT, full = bars + warp * R::STAGES * 8;
  if (lane == 0) {
    for (int s = 0; s < R::STAGES; ++s) mbar_init(full + 8 * s, 1);
    fence_mbar_init();
  }
  programmatic_wait();

  // ---- this CTA's part of the line
  const int per_thread = (p.batch + THREADS - 1) / THREADS, mine = tid * per_thread;
  long long sum = 0;
  for (int b = mine; b < min(mine + per_thread, p.batch); ++b) {
    const Sequence s = sequence_of<STEP>(p, b, ROWS);
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
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += warp_sums[w];
    line += warp_sums[w];
  }
  before -= sum;
  const int share = share_of(line), cta = blockIdx.x;
  RowsJoin* entry = static_cast<RowsJoin*>(p.joins) + cta;
  if (tid == 0) {
    entry->last_cta = -1;
    if (share < 0) atomicExch(p.status, INTENT_B200_ERR_SHAPE);
  }
  const long long begin = (long long)cta * share;
  if (share <= 0 || begin >= line) return;
  const int end = int(min((long long)share, line - begin));            // of this CTA's places, counted from its first one
  if (begin >= before && begin < before + sum) {
    int b = mine;
    long long at = before;
    for (;; ++b) {
      const Sequence s = sequence_of<STEP>(p, b, ROWS);
      const long long places = places_of<BEGIN>(p, s);
      if (begin < at + places || b + 1 >= min(mine + per_thread, p.batch)) break;
      at += places;
    }
    shared[0] = b;
    *reinterpret_cast<long long*>(shared + 2) = begin - at;            // place in the sequence
  }
  __syncthreads();
  Walk<STEP, BEGIN> load;
  load.b = shared[0];
  load.s = sequence_of<STEP>(p, load.b, ROWS);
  {
    const long long place = *reinterpret_cast<const long long*>(shared + 2);
    const int item = divide(place, load.s.steps + BEGIN);
    load.step = int(place - (long long)item * (load.s.steps + BEGIN)) - BEGIN;
    load.head = item / load.s.tiles;
    load.tile = item - load.head * load.s.tiles;
  }
  const int first_place = max(-load.step, 0);            // of a step
  if (first_place >= end) return;
  load.step = max(load.step, 0);
  Walk<STEP, BEGIN> work = load;

  const float infinity = __int_as_float(0x7f800000);
  int loading = first_place, slot_in = 0, slot_out = 0;
  uint32_t parity = 0, present = 0;      // a bit per slot; two bits per unit asked for (its halves), the oldest lowest
  int queued = 0;
  bool ok = true;
  const int boxes = p.page_shift >= 5 ? 1 : 2;           // pages that a unit lies in
  int page[2];                           // of the unit at `load`, asked for one unit ahead; -1: not needed
  auto look_up = [&] {
    const int token = (load.s.begin + load.step) * STEP + warp * UNIT;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = token + i * (UNIT / 2);
      page[i] = -1;
      if (t < load.s.length && t + UNIT / 2 > load.s.low)
        page[i] = __ldg(p.page_table + int64_t(load.b) * p.table_width + (t >> p.page_shift));
    }
  };
  // asks for the unit of this warp at `load`, and goes on
  auto ask = [&] {
    const int token = (load.s.begin + load.step) * STEP + warp * UNIT;
    const bool here[2] = {page[0] >= 0 && page[0] < p.pages, page[1] >= 0 && page[1] < p.pages};
    const bool any = here[0] || here[1];
    if (lane == 0 && any) {
      const uint32_t bar = full + 8 * slot_in, to = ring + slot_in * R::SLOT;
      mbar_expect_tx(bar, boxes == 1 || (here[0] && here[1]) ? R::SLOT : R::SLOT / 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // (a unit in one page is one box, whichever of its halves is needed)
        if (boxes == 1 ? i == 1 : !here[i]) continue;
        const int number = boxes == 1 && !here[0] ? page[1] : page[i], t = token + i * (UNIT / 2);
        const int row = ((number * p.k_heads + load.head) << p.page_shift) + (t & ((1 << p.page_shift) - 1));
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          tma_load_2d(to + c * R::HALF + i * (R::HALF / 2), &map_k, 64 * c, row, bar);
          tma_load_2d(to + R::OPERAND + c * R::HALF + i * (R::HALF / 2), &map_v, 64 * c, row, bar);
        }
      }
    }
    present |= (uint32_t(here[0]) | (uint32_t(here[1]) << 1)) << (2 * queued);
    ++queued;
    if (any) slot_in = slot_in + 1 == R::STAGES ? 0 : slot_in + 1;
    loading += load.distance();
    if (loading < end) {
      load.advance(p, ROWS);
      look_up();
    }
  };
  uint32_t qf[NT][D / 16][2];            // queries as B fragments: k = elements, n = rows
  float o[NT][D / 16][4];                // O^T: elements 16 i + lane / 4 (+ 8) of rows 2 (lane % 4) (+ 1)
  float top[NT][2], weight_sum[NT][2];
  int position[NT][2];                   // of this thread's rows; -1 where there is none
  int least = 0, most = 0;               // positions of the tile's first and last row
  // the queries of the tile at `work`
  auto begin_tile = [&] {
    const int tile_row = work.tile * ROWS, rows = min(ROWS, work.s.rows - tile_row);
    least = work.s.first + tile_row / p.group;
    most = work.s.first + (tile_row + rows - 1) / p.group;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = tile_row + nt * 8 + 2 * (lane & 3) + e;
        position[nt][e] = r < work.s.rows ? work.s.first + r / p.group : -1;
        top[nt][e] = -infinity;
        weight_sum[nt][e] = 0.f;
      }
      const int r = min(tile_row + nt * 8 + (lane >> 2), work.s.rows - 1), token = r / p.group;
      const uint16_t* x = p.q + int64_t(work.s.first_row + token) * p.q_token +
                          int64_t(work.head * p.group + r - token * p.group) * p.q_head;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        qf[nt][i][0] = __ldg(reinterpret_cast<const uint32_t*>(x + 16 * i + 2 * (lane & 3)));
        qf[nt][i][1] = __ldg(reinterpret_cast<const uint32_t*>(x + 16 * i + 8 + 2 * (lane & 3)));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      }
    }
  };
  look_up();
  begin_tile();
  for (int i = 0; i < R::STAGES && loading < end; ++i) ask();
  int turn = 0;                          // place of the join that is next
  for (int at = first_place, next; at < end; at = next) {
    const uint32_t halves = present & 3;
    present >>= 2;
    --queued;
    if (halves) {
      const int token = (work.s.begin + work.step) * STEP + warp * UNIT;
      const uint32_t keys = ring + slot_out * R::SLOT, values = keys + R::OPERAND;
      if (ok) ok = mbar_wait_warp(full + 8 * slot_out, (parity >> slot_out) & 1);
      parity ^= 1u << slot_out;
      slot_out = slot_out + 1 == R::STAGES ? 0 : slot_out + 1;

      float s[NT][2][4], s_odd[NT][2][4];  // S^T: tokens 16 m + lane / 4 (+ 8), rows as in o; of even and odd pieces of 16 elements
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][m][e] = s_odd[nt][m][e] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const int r = 16 * m + (lane & 15), c = 2 * (i & 3) + (lane >> 4);
          uint32_t a[4];
          ldmatrix_x4(a, keys + (i / 4) * R::HALF + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            Elem<T>::mma16816(i & 1 ? s_odd[nt][m] : s[nt][m], a[0], a[1], a[2], a[3], qf[nt][i][0], qf[nt][i][1]);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][m][e] += s_odd[nt][m][e];
      const bool all = halves == 3 && token + UNIT - 1 <= least && (p.window == 0 || token > most - p.window);
      uint32_t counted[2][2] = {};       // pairs of tokens 16 m + 2 (lane % 4) (+ 8) that some row of the tile sees
      if (!all) {
        const int low = p.window > 0 ? max(least - p.window + 1, 0) : 0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const bool there = (halves >> m) & 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = token + 16 * m + (lane >> 2) + 8 * (e >> 1), at_row = position[nt][e & 1];
              if (!there || t > at_row || (p.window > 0 && t <= at_row - p.window)) s[nt][m][e] = -infinity;
            }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // (what lies behind the tile's last token, or was never loaded, may be no number: 0 * NaN is NaN)
            const int t = token + 16 * m + 8 * e + 2 * (lane & 3);
            if (there && t >= low && t <= most) counted[m][e] |= 0xffffu;
            if (there && t + 1 >= low && t + 1 <= most) counted[m][e] |= 0xffff0000u;
          }
        }
      }
      // A row's maximum is raised only when a score exceeds it by more than SLACK: until then no lane has to know the others'.
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float here = fmaxf(fmaxf(s[nt][0][e], s[nt][0][e + 2]), fmaxf(s[nt][1][e], s[nt][1][e + 2]));
          raise |= here * p.scale > top[nt][e] + SLACK;                // (from -inf: any)
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float factor[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float here = fmaxf(fmaxf(s[nt][0][e], s[nt][0][e + 2]), fmaxf(s[nt][1][e], s[nt][1][e + 2]));
#pragma unroll
            for (int d = 4; d < 32; d *= 2) here = fmaxf(here, __shfl_xor_sync(0xffffffffu, here, d));
            const float now = fmaxf(top[nt][e], here * p.scale);
            factor[e] = exp2_fast(top[nt][e] - (now == -infinity ? 0.f : now));
            top[nt][e] = now;
            weight_sum[nt][e] *= factor[e];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][i][e] *= factor[e & 1];
        }
      }
      uint32_t pf[NT][2][2];             // P^T as B fragments
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float origin = top[nt][e] == -infinity ? 0.f : top[nt][e];
          float added = 0.f;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int f = 0; f < 4; f += 2) {
              const float w = exp2_fast(fmaf(s[nt][m][e + f], p.scale, -origin));
              s[nt][m][e + f] = w;
              added += w;
            }
          weight_sum[nt][e] += added;
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          pf[nt][m][0] = movmatrix(Elem<T>::pack2(s[nt][m][0], s[nt][m][1]));
          pf[nt][m][1] = movmatrix(Elem<T>::pack2(s[nt][m][2], s[nt][m][3]));
        }
      }
      auto values_of = [&](auto whole, int m, int i, uint32_t (&a)[4]) {   // elements 16 i of tokens 16 m, as A fragments
        const int r = 16 * m + (lane & 7) + ((lane >> 4) << 3), c = 2 * (i & 3) + ((lane >> 3) & 1);
        ldmatrix_x4_trans(a, values + (i / 4) * R::HALF + r * 128 + ((c ^ (r & 7)) << 4));
        if (!decltype(whole)::value)
#pragma unroll
          for (int e = 0; e < 4; ++e) a[e] &= counted[m][e >> 1];
      };
      auto not_finite = [&] {
        // (a loop that stays one: code that few calls reach has to be fetched when they do)
        uint32_t sum[2] = {};
#pragma unroll 1
        for (int i = 0; i < D / 16; ++i) {
          uint32_t a[4], b[4];
          values_of(Bool<false>{}, 0, i, a);
          values_of(Bool<false>{}, 1, i, b);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            sum[0] = add_no_numbers<T>(a[e], sum[0]);
            sum[1] = add_no_numbers<T>(b[e], sum[1]);
          }
        }
        return __any_sync(0xffffffffu, ((sum[0] | sum[1]) & 0x7fff7fffu) != 0) != 0;
      };
      auto add_values = [&](auto whole) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t a[4];
            values_of(whole, m, i, a);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) Elem<T>::mma16816(o[nt][i], a[0], a[1], a[2], a[3], pf[nt][m][0], pf[nt][m][1]);
          }
      };
      if (all) {
        add_values(Bool<true>{});
      } else if (least == most || !not_finite()) {
        add_values(Bool<false>{});
      } else {
        // Values that are no finite numbers, in tokens that some rows see and others do not: row by row, from what it sees.
#pragma unroll 1
        for (int r = 0; r < ROWS; ++r) {
          const int even = NT == 2 && r >= 8 ? position[NT - 1][0] : position[0][0];
          const int odd = NT == 2 && r >= 8 ? position[NT - 1][1] : position[0][1];
          const int at_row = __shfl_sync(0xffffffffu, r & 1 ? odd : even, (r & 7) >> 1);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint32_t sees[2] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = token + 16 * m + 8 * (e >> 1) + 2 * (lane & 3) + (e & 1);
              if (t <= at_row && (p.window == 0 || t > at_row - p.window)) sees[e >> 1] |= e & 1 ? 0xffff0000u : 0xffffu;
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              uint32_t a[4];
              values_of(Bool<false>{}, m, i, a);
#pragma unroll
              for (int e = 0; e < 4; ++e) a[e] &= sees[e >> 1];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float part[4] = {};
                Elem<T>::mma16816(part, a[0], a[1], a[2], a[3], pf[nt][m][0], pf[nt][m][1]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (nt * 8 + 2 * (lane & 3) + (e & 1) == r) o[nt][i][e] += part[e];
              }
            }
          }
        }
      }
      __syncwarp();                      // every lane is done with the slot
    }
    if (ok && loading < end) ask();      // (a slot that was given up on may still be on its way)

    const bool last_step = work.step + 1 == work.s.steps;
    next = at + work.distance();
    if (!last_step && next < end) {
      ++work.step;
    } else {
      // ---- the warps' parts, then the CTAs'.  There are two places for them in turn: when a warp writes to one of them again,
      // all have passed the barrier of the tile between.
      float* join_here = join + turn * (WARPS * ROWS * PITCH);
      float* max_here = join_max + turn * (WARPS * ROWS);
      float* sum_here = join_sum + turn * (WARPS * ROWS);
      turn ^= JOINS - 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = nt * 8 + 2 * (lane & 3) + e;
          float sum_all = weight_sum[nt][e];
#pragma unroll
          for (int d = 4; d < 32; d *= 2) sum_all += __shfl_xor_sync(0xffffffffu, sum_all, d);
          if (lane < 4) {
            max_here[warp * ROWS + r] = top[nt][e];
            sum_here[warp * ROWS + r] = sum_all;
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            // (pieces of eight elements change places with the row, so that a store meets 32 banks)
            float* to = join_here + (warp * ROWS + r) * PITCH + (lane >> 2);
            to[((2 * i) ^ (lane & 3)) * 8] = o[nt][i][e];
            to[((2 * i + 1) ^ (lane & 3)) * 8] = o[nt][i][e + 2];
          }
        }
      }
      const int tile_row = work.tile * ROWS, rows = min(ROWS, work.s.rows - tile_row), head = work.head;
      const int first_row = work.s.first_row, sequence = work.b;
      const int item_begin = at - work.step, item_end = item_begin + work.s.steps;   // the tile's places, maybe of other CTAs
      if (next < end) {
        work.advance(p, ROWS);
        begin_tile();                    // (its queries are on their way while this tile is put together)
      }
      __syncthreads();
      const bool begins = item_begin >= 0, whole = begins && item_end <= share;
      float* part = p.parts + size_t(2 * cta + begins) * (ROWS * (D + 2));
      auto place = [&](int r) {
        const int token = (tile_row + r) / p.group, of_group = tile_row + r - token * p.group;
        return p.out + (int64_t(first_row + token) * p.q_heads + head * p.group + of_group) * D;
      };
      for (int w = tid; w < rows * (D / 8); w += THREADS) {
        const int r = w / (D / 8), c = w - r * (D / 8);
        float m = -infinity, l = 0.f, x[8] = {};
#pragma unroll
        for (int v = 0; v < WARPS; ++v) m = fmaxf(m, max_here[v * ROWS + r]);
        const float origin = m == -infinity ? 0.f : m;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) {
          const float f = exp2_fast(max_here[v * ROWS + r] - origin);
          l = fmaf(sum_here[v * ROWS + r], f, l);
          const float* from = join_here + (v * ROWS + r) * PITCH + 8 * (c ^ (r >> 1 & 3));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = fmaf(from[e], f, x[e]);
        }
        if (whole) {
          const float inverse = l == 0.f ? of_nothing(p, sequence, first_row + (tile_row + r) / p.group) : 1.f / l;
          *reinterpret_cast<uint4*>(place(r) + 8 * c) =
              make_uint4(Elem<T>::pack2(x[0] * inverse, x[1] * inverse), Elem<T>::pack2(x[2] * inverse, x[3] * inverse),
                         Elem<T>::pack2(x[4] * inverse, x[5] * inverse), Elem<T>::pack2(x[6] * inverse, x[7] * inverse));
        } else {
          float4* to = reinterpret_cast<float4*>(part + r * D + 8 * c);
          to[0] = make_float4(x[0], x[1], x[2], x[3]);
          to[1] = make_float4(x[4], x[5], x[6], x[7]);
          if (c == 0) {
            part[ROWS * D + r] = m;
            part[ROWS * (D + 1) + r] = l;
          }
        }
      }
      if (tid == 0 && !whole && begins) {
        entry->row = first_row;
        entry->head = head;
        entry->tile_row = tile_row;
        entry->rows = rows;
        entry->sequence = sequence;
        entry->last_cta = cta + (item_end - 1) / share;
      }
      if (JOINS == 1) __syncthreads();
    }
  }
  if (!ok) {
    // Nothing may be on its way to a CTA that is gone.  (Which phase a slot is in has not been counted since the wait that gave
    // up: of the two parities the wait for one is for the current phase, the other is over.)
    for (int s = 0; s < R::STAGES; ++s)
      for (int of_phase = 0; of_phase < 2; ++of_phase) mbar_wait_warp(full + 8 * s, of_phase, 64);
    if (lane == 0) atomicExch(p.status, INTENT_B200_ERR_TIMEOUT);
  }
}

template <typename T, int D, int NT>
int launch(const CUtensorMap& map_k, const CUtensorMap& map_v, const PagedParams& p, int grid, cudaStream_t stream) {
  auto kernel = paged_rows_kernel<T, D, NT>;
  constexpr int smem = smem_bytes<D, NT>();
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_status(e);
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel),
                         NT == 1 ? "paged_rows_kernel 8 rows" : "paged_rows_kernel 16 rows", grid, 32 * Ring<D>::WARPS, smem, 1);
  e = launch_programmatic(kernel, dim3(unsigned(grid)), dim3(32 * Ring<D>::WARPS), smem, stream, 1, map_k, map_v, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

}  // namespace

int64_t paged_rows_parts_bytes(int64_t dim) {
  return int64_t(2) * kPagedCtas * 16 * (dim + 2) * int64_t(sizeof(float));
}

template <typename T>
int paged_rows(const PagedParams& p, int64_t dim, int tile_rows, const void* k_cache, const void* v_cache, int grid,
               cudaStream_t stream) {
  CUtensorMap map_k, map_v;
  const uint64_t rows = uint64_t(p.pages) * uint64_t(p.k_heads) << p.page_shift;
  const uint32_t box = p.page_shift >= 5 ? UNIT : UNIT / 2;
  constexpr auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  if (!make_tensor_map_2d(&map_k, type, k_cache, rows, uint64_t(dim), uint64_t(dim) * 2, box, 64,
                          CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&map_v, type, v_cache, rows, uint64_t(dim), uint64_t(dim) * 2, box, 64,
                          CU_TENSOR_MAP_SWIZZLE_128B))
    return INTENT_B200_ERR_CUDA;
  if (dim == 128)
    return tile_rows == 8 ? launch<T, 128, 1>(map_k, map_v, p, grid, stream)
                          : launch<T, 128, 2>(map_k, map_v, p, grid, stream);
  return tile_rows == 8 ? launch<T, 64, 1>(map_k, map_v, p, grid, stream)
                        : launch<T, 64, 2>(map_k, map_v, p, grid, stream);
}
template int paged_rows<__half>(const PagedParams&, int64_t, int, const void*, const void*, int, cudaStream_t);
template int paged_rows<__nv_bfloat16>(const PagedParams&, int64_t, int, const void*, const void*, int, cudaStream_t);

}  // namespace ib200
