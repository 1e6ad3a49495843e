// Attention over a paged cache in 4 bits for few rows of queries per sequence and key head (paged_decode_attention_int4, and
// paged_attention_int4 for short chunks).  The program is that of paged_rows.cu with keys and values m + s n: of a code n (0 .. 15), and of
// the scale s and the minimum m of its group of GROUP elements.
//
// Codes are multiplied as they are, and scales and minima go to the scores and the weights: with the sums over a group g
//   x . k_j = sum_g s_jg (x_g . n_jg) + m_jg sum(x_g)            o = sum_j w_j v_j = sum_g (sum_j (w_j s_jg) n_jg + sum_j w_j m_jg)
// Four bits become operands of the tensor core by being masked where they are: in the lowest or the next four bits of a 16-bit
// word they are n or 16 n times the smallest bf16 (2^-133; an f16 too, 2^-24, in the lowest four), exact numbers for it.  The factor of
// 16 is taken out of the queries (bf16) or the results ahead, so that eight codes cost five instructions; with 2^64 on weight times
// scale and 2^60 on a query no product comes near the ends of f32.  (Queries of 2^67 and more and scales of values of 2^55 and more
// are out of that range, and below f32's smallest normal number, 2^-126, are 2^-57 of s n and 2^-53 of x n.)
//
// All statistics and sums are in f32, or in three bf16 parts that have its bits.  A weight times its scale is rounded to bf16 for the
// product with the codes.  The same rounded numbers times the middle of the codes (8 and 7 in turn) are taken off, and the middle's
// share is added up apart: the rounding is worth what it is for a product with v_j.  For f16 results the product is made with what
// the rounding left over, too, and nothing is taken off.
//
// A product cuts, instead of rounding, what it adds to, and a sum of codes only grows: after 131072 tokens of a row in one warp it
// was too small by a fifth of the result.  So the middle is taken off in every step (bf16), and in every LEVEL-th what the sums of a
// row's group have in common goes to the sum of minima or middles.  What is cut is a part of what is left then (131072 tokens: f16
// results are off by 2.9 10^-4, of which 2.1 are their own rounding, bf16 by 2.4 10^-3 and 1.7; skewed values 2.3 10^-4 and 2.9 10^-3).
//
// With a quarter of the bytes of 16-bit elements there is a quarter of the time, and what all warps of a CTA have to wait for costs
// four times as much.  So the line of steps (as in paged_rows.cu, but of UNIT tokens each) is cut into a share for every warp,
// which goes through its tiles on its own, with a ring of its own, and writes the results of those that it has whole.  Tiles that are
// cut leave at most two parts per warp in shared memory, which are put together once, at the end: the results, or one part of the
// CTA for the join.
//
// Copies are made by the warps that read them (cp.async): a TMA copy needs a lane of its own, and with four of them per step they
// were a quarter of a step's instructions (74 -> 70 us below).
//
// Measured on one B200 (6540 GB/s copied; bf16, 32 heads of 128 on 8, groups of 64): 64 histories of up to 8192 tokens 68 - 71 us, 4.6
// TB/s (floor 49); 4 of up to 131072, 4 key heads, groups of 128 44 us, 3.9 TB/s; 200 of up to 2048, 16 heads of 64, f16, groups of 32
// 81 us, 3.4 TB/s; one of 2000 10.5 us, the reads one after another of two launches.  Bound by what a step of 64 tokens costs beside
// its bytes, 900 instructions on two warps per scheduler, of which the ALU's are the masks (256 of 64 tokens' codes).  Tiles of sixteen
// rows of heads of 128 are out of registers and spill (28 to 136 bytes).
// Tried and not kept: twelve warps with keys and values in slots of their own (more instructions issued, and more of them: 72 us where
// eight warps took 70), steps of 32 or 48 tokens for sixteen or twelve (80, 76), of 32 for tiles of
// sixteen rows (64 sequences of 16 heads of 64 on one: 151 us, 122 with 64), codes asked for in the second-level cache a step
// ahead (73), shifts as products (77), parts joined by the CTA that is done last in place of a launch (70, and 88 for 79 with four
// tokens each).
#include <cstring>

#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "paged_rows.cuh"
#include "tma.cuh"

namespace ib200 {
namespace {

// TILE: rows of queries, 4, 8 or 16.  Tiles of four stand twice among the eight columns of a product, for a group each when weights
// are multiplied by scales: half the work of that (64 histories of up to 8192, groups of 32 / 64: 77 -> 71, 69 -> 65 us).
template <int D, int GROUP, int TILE>
struct Ring {
  static constexpr int NT = TILE == 16 ? 2 : 1;           // columns, in eights
  static constexpr int UNIT = 64;                         // tokens of a ring slot, a step
  static constexpr int PARTS = UNIT / 16;                 // pieces of it that lie in one page in any case
  static constexpr int WARPS = NT == 1 && D == 64 ? 16 : 8;
  static constexpr int STAGES = 2;
  static constexpr int GROUPS = D / GROUP;
  static constexpr int ROW = D / 2;                       // bytes of a token's codes
  static constexpr int CODES = UNIT * ROW, SCALES = UNIT * GROUPS * 4;   // of keys or values of a unit
  static constexpr int SLOT = 2 * (CODES + SCALES);       // keys' codes, values' codes, keys' scales, values' scales
  static constexpr int OF_WARP = STAGES * SLOT, BYTES = WARPS * OF_WARP;
  static constexpr int BEGIN = 1;                         // places on the line ahead of the steps of a tile
  static constexpr int PIECE = 8 * NT * (D + 2) * 4;      // a part of a tile: results, maxima, sums
  static_assert(PIECE <= OF_WARP, "a warp's last part lies in its ring");
};

// What a warp leaves of a tile that it does not have whole
struct Left {
  int there;
  int begin, end;          // the tile's places, counted from the CTA's first one
  int row, head, tile_row, rows, sequence;      // as in RowsJoin
};

template <int D, int GROUP, int TILE>
constexpr int smem_bytes() {
  using R = Ring<D, GROUP, TILE>;
  constexpr int bytes = 128 + R::BYTES + R::WARPS * (R::PIECE + 2 * int(sizeof(Left)) + 8 + 16);
  static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
  return bytes;
}

// 16 bytes to shared memory, past the first-level cache; copies are waited for in groups, in order
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// What the number of a 16-byte chunk of a row of codes is changed by: rows of 64 or 32 bytes, eight of which fill 32 banks
template <int D>
__device__ __forceinline__ int swizzle_of(int row) {
  return D == 128 ? (row >> 1) & 3 : (row >> 2) & 1;
}

template <int N>
struct Words {
  uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> lds(uint32_t addr) {
  Words<N> d;
  if constexpr (N == 1) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(d.w[0]) : "r"(addr));
  else if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(d.w[0]), "=r"(d.w[1]) : "r"(addr));
  else asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(d.w[0]), "=r"(d.w[1]), "=r"(d.w[2]), "=r"(d.w[3]) : "r"(addr));
  return d;
}

using Wide = __nv_bfloat16;              // the type of the weights' product with the codes
constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u;
// The middle of the codes of an even token and of the odd one behind it, 8 and 7, negative, in the same places
constexpr uint32_t LOW_CENTRE = 0x80078008u, HIGH_CENTRE = 0x80708080u;

// What the scores of keys' codes are multiplied with
template <typename T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
  static constexpr float UNIT_OF_SCORES = 0x1p-73f;      // 2^60 * 2^-133
  // the 16-bit pair as an operand for codes in the lowest four bits, and in the next
  __device__ static __forceinline__ uint32_t low(uint32_t x) { return Elem<__nv_bfloat16>::mul2(x, 0x5d805d80u); }     // 2^60
  __device__ static __forceinline__ uint32_t high(uint32_t x) { return Elem<__nv_bfloat16>::mul2(x, 0x5b805b80u); }    // 2^56
  __device__ static __forceinline__ uint32_t odd(uint32_t codes) { return codes & HIGH; }
};
template <>
struct Codes<__half> {
  static constexpr float UNIT_OF_SCORES = 0x1p-24f;
  __device__ static __forceinline__ uint32_t low(uint32_t x) { return x; }
  __device__ static __forceinline__ uint32_t high(uint32_t x) { return x; }
  // (an f16 query divided by 16 might lose bits)
  __device__ static __forceinline__ uint32_t odd(uint32_t codes) { return (codes >> 4) & LOW; }
};

template <typename T, int D, int GROUP, int TILE>
__global__ void __launch_bounds__(32 * Ring<D, GROUP, TILE>::WARPS, 1)
paged_rows_int4_kernel(const Int4Cache cache, const PagedParams p) {
  using R = Ring<D, GROUP, TILE>;
  constexpr int NT = R::NT, ROWS = 8 * NT, WARPS = R::WARPS, THREADS = 32 * WARPS, UNIT = R::UNIT, PARTS = R::PARTS, STEP = UNIT,
                BEGIN = R::BEGIN, GROUPS = R::GROUPS;
  constexpr int CHUNKS = D / 32, OF_GROUP = CHUNKS / GROUPS;            // 16 bytes of a token's codes
  // Columns of a product are the tile's rows, or these twice: then the upper half of the columns has the upper half of the groups.
  constexpr int COPIES = TILE == 4 && GROUPS > 1 ? 2 : 1, COLUMNS = ROWS / COPIES, SETS = GROUPS / COPIES;
  constexpr bool SPLIT = std::is_same<T, __half>::value;                // weights in two bf16 parts
  // Steps after which sums of codes are brought back to nothing on average.  (f16, for whose two products the middle is not taken off
  // before, us of 200 histories of up to 2048, 16 heads of 64 / what results over 131072 tokens in one warp are off by, in 10^-4: 2
  // steps 82.7 / 2.6, 4 81.1 / 2.9, 8 80.3 / 3.8; taken off in every step and 16 of these 85.4 / 2.5, and tiles of sixteen rows 10 - 30 %
  // slower.)
  constexpr int LEVEL = SPLIT ? 4 : 16;
  // The 2^64 of the product with codes, on the weights (f16) or on the scales (bf16, whose minima times 2^64 would leave f32's range).
  constexpr float OF_WEIGHTS = SPLIT ? 64.f : 0.f, UNIT_OF_WEIGHTS = SPLIT ? 0x1p-64f : 1.f, OF_SCALES = SPLIT ? 1.f : 0x1p64f;
  extern __shared__ unsigned char smem_raw[];
  programmatic_begin();
  const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  // a warp's part of the tile that its share begins in; then of the tile that it ends in, in its ring
  float* first_parts = reinterpret_cast<float*>(base_ptr + R::BYTES);
  auto part_of = [&](int w, int which) {
    return which == 0 ? first_parts + w * (R::PIECE / 4) : reinterpret_cast<float*>(base_ptr + w * R::OF_WARP);
  };
  Left* left = reinterpret_cast<Left*>(base_ptr + R::BYTES + WARPS * R::PIECE);          // [WARPS][2]
  long long* starts = reinterpret_cast<long long*>(left + 2 * WARPS);                    // [WARPS][2]: sequence, place in it
  long long* warp_sums = starts + 2 * WARPS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = base + warp * R::OF_WARP;
  programmatic_wait();

  // ---- this warp's part of the line
  RowsJoin* entry = static_cast<RowsJoin*>(p.joins) + blockIdx.x;
  const Place<STEP, BEGIN> start = place_of<STEP, BEGIN, THREADS, WARPS>(p, TILE, starts, warp_sums, entry);
  const int first_place = start.first, end = start.end, origin = warp * start.share;     // origin: the warp's first of the CTA's
  Walk<STEP, BEGIN> load = start.at, work = load;
  if (lane < 2) left[2 * warp + lane].there = 0;

  const float infinity = __int_as_float(0x7f800000);
  int loading = first_place, slot_in = 0, slot_out = 0;
  uint32_t present = 0;                  // PARTS bits per unit asked for, the oldest lowest
  int queued = 0;
  const int box = min(1 << p.page_shift, UNIT);          // tokens of a unit that lie in one page
  int page;                              // of piece lane % PARTS of the unit at `load`, asked for one unit ahead; -1: not needed
  auto look_up = [&] {
    const int t = (load.s.begin + load.step) * UNIT + (lane % PARTS) * 16;
    page = -1;
    if (t < load.s.length && t + 16 > load.s.low)
      page = __ldg(p.page_table + int64_t(load.b) * p.table_width + (t >> p.page_shift));
  };
  // A lane copies 16 bytes at a time of the 512 that a warp does, rows of codes in an order in which eight of them meet 32 banks.
  constexpr int CHUNKS_OF_ROW = R::ROW / 16;
  const int copied_row = lane / CHUNKS_OF_ROW, copied_chunk = lane % CHUNKS_OF_ROW;
  const uint32_t copied = copied_row * R::ROW + ((copied_chunk ^ swizzle_of<D>(copied_row)) << 4);
  const unsigned char *k_codes = static_cast<const unsigned char*>(cache.k_codes) + 16 * lane,
                      *v_codes = static_cast<const unsigned char*>(cache.v_codes) + 16 * lane;
  // asks for the unit of this warp at `load`, and goes on
  auto ask = [&] {
    const int number = page >= 0 && page < p.pages ? page : -1;
    const uint32_t here = __ballot_sync(0xffffffffu, number >= 0) & ((1u << PARTS) - 1);
    const int first = ((load.s.begin + load.step) * UNIT) & ((1 << p.page_shift) - 1);     // in its page
    const uint32_t to = ring + slot_in * R::SLOT;
    if (box == UNIT) {
      // (the pieces that are needed have the same page)
      if (here) {
        const int row = ((__shfl_sync(0xffffffffu, number, __ffs(here) - 1) * p.k_heads + load.head) << p.page_shift) + first;
        const int64_t code = int64_t(row) * R::ROW, scale = int64_t(row) * (GROUPS * 4);
#pragma unroll
        for (int i = 0; i < R::CODES / 512; ++i) {
          copy16(to + copied + 512 * i, k_codes + code + 512 * i);
          copy16(to + R::CODES + copied + 512 * i, v_codes + code + 512 * i);
        }
#pragma unroll
        for (int i = 0; i < (2 * R::SCALES + 511) / 512; ++i) {
          const int at = 512 * i + 16 * lane;            // keys' scales, then values'
          const unsigned char* from = static_cast<const unsigned char*>(at < R::SCALES ? cache.k_scales : cache.v_scales);
          if (at < 2 * R::SCALES) copy16(to + 2 * R::CODES + at, from + scale + (at < R::SCALES ? at : at - R::SCALES));
        }
      }
    } else {
#pragma unroll
      for (int piece = 0; piece < PARTS; ++piece) {
        const int of_piece = __shfl_sync(0xffffffffu, number, piece);
        if (of_piece < 0) continue;
        const int row = ((of_piece * p.k_heads + load.head) << p.page_shift) + ((first + 16 * piece) & ((1 << p.page_shift) - 1));
        const int64_t code = int64_t(row) * R::ROW, scale = int64_t(row) * (GROUPS * 4);
#pragma unroll
        for (int i = 0; i < 16 * R::ROW / 512; ++i) {
          const uint32_t there = to + copied + 16 * piece * R::ROW + 512 * i;
          copy16(there, k_codes + code + 512 * i);
          copy16(there + R::CODES, v_codes + code + 512 * i);
        }
        const unsigned char* from = static_cast<const unsigned char*>(lane < 16 ? cache.k_scales : cache.v_scales) + 16 * (lane % 16);
        if (lane % 16 < 4 * GROUPS)
          copy16(to + 2 * R::CODES + (lane < 16 ? 0 : R::SCALES) + 64 * GROUPS * piece + 16 * (lane % 16), from + scale);
      }
    }
    copies_commit();
    slot_in = slot_in + 1 == R::STAGES ? 0 : slot_in + 1;
    present |= here << (PARTS * queued);
    ++queued;
    loading += load.distance();
    if (loading < end) {
      load.advance(p, TILE);
      look_up();
    }
  };
  uint32_t qf[NT][CHUNKS][4];            // queries as B fragments: elements 32 c + 8 (lane % 4) + {0, 4}, {1, 5}, {2, 6}, {3, 7}
  // Sums of a group's queries in the scores' unit, which its minimum is multiplied with: of this thread's rows (f16), or in three
  // bf16 parts, which have the bits of f32, as a B fragment: elements 0 .. GROUPS - 1 the rounded sums, the next ones what that left
  // over, and from the eighth on what both left.  (With two parts a score is off by 2^-17 of minimum times sum, which can be many
  // times the score where keys have a common offset.)
  constexpr bool BY_PRODUCT = std::is_same<T, __nv_bfloat16>::value;
  float q_sum[NT][2][GROUPS];
  uint32_t q_parts[NT][2];
  float o[NT][CHUNKS][2][4];             // sums of codes: elements 32 c + 4 (lane / 4) + 2 t (+ 1, times 16) of rows 2 (lane % 4) (+ 1)
  const float centre = lane & 4 ? 7.f : 8.f;             // of the codes of this thread's tokens, which are odd or even (bf16)
  const int upper = COPIES == 2 ? (lane & 3) >> 1 : 0;   // this thread's half of the groups
  // Sums of weight times the middle of the codes (f16: times the minimum) of this thread's tokens
  float middle[NT][2][SETS];
  float top[NT][2];
  uint64_t weight_sum[NT];               // of both rows
  int position[NT][2];                   // of this thread's rows; -1 where there is none
  int least = 0, most = 0;               // positions of the tile's first and last row
  const float scale = p.scale / Codes<T>::UNIT_OF_SCORES;
  // the queries of the tile at `work`
  auto begin_tile = [&] {
    const int tile_row = work.tile * TILE, rows = min(TILE, work.s.rows - tile_row);
    least = work.s.first + tile_row / p.group;
    most = work.s.first + (tile_row + rows - 1) / p.group;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = min(tile_row + nt * 8 + (lane >> 2) % COLUMNS, work.s.rows - 1), token = r / p.group;
      const uint16_t* x = p.q + int64_t(work.s.first_row + token) * p.q_token +
                          int64_t(work.head * p.group + r - token * p.group) * p.q_head + 8 * (lane & 3);
      float sums[GROUPS] = {};
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + 32 * c));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sums[c / OF_GROUP] += Elem<T>::to_float(uint16_t(w[e])) + Elem<T>::to_float(uint16_t(w[e] >> 16));
        qf[nt][c][0] = Codes<T>::low(prmt(v.x, v.z, 0x5410));
        qf[nt][c][1] = Codes<T>::high(prmt(v.x, v.z, 0x7632));
        qf[nt][c][2] = Codes<T>::low(prmt(v.y, v.w, 0x5410));
        qf[nt][c][3] = Codes<T>::high(prmt(v.y, v.w, 0x7632));
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][c][t][e] = 0.f;
      }
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 1);
        sums[g] += __shfl_xor_sync(0xffffffffu, sums[g], 2);
        sums[g] *= Codes<T>::UNIT_OF_SCORES;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (!BY_PRODUCT) q_sum[nt][e][g] = __shfl_sync(0xffffffffu, sums[g], 8 * (lane & 3) + 4 * e);
        }
      }
#pragma unroll
      for (int i = 0; i < SETS; ++i) middle[nt][0][i] = middle[nt][1][i] = 0.f;
      if (BY_PRODUCT) {
        uint32_t parts[2][2 * GROUPS] = {};
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          parts[0][g] = Elem<Wide>::from_float(sums[g]);
          const float rest = sums[g] - Elem<Wide>::to_float(uint16_t(parts[0][g]));
          parts[0][GROUPS + g] = Elem<Wide>::from_float(rest);
          parts[1][g] = Elem<Wide>::from_float(rest - Elem<Wide>::to_float(uint16_t(parts[0][GROUPS + g])));
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          q_parts[nt][h] = 0;
#pragma unroll
          for (int i = 0; i < GROUPS; ++i)
            if ((lane & 3) == i) q_parts[nt][h] = parts[h][2 * i] | (parts[h][2 * i + 1] << 16);
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int column = (nt * 8 + 2 * (lane & 3) + e) % COLUMNS, of_thread = tile_row + column;
        position[nt][e] = column < TILE && of_thread < work.s.rows ? work.s.first + of_thread / p.group : -1;
        top[nt][e] = -infinity;
      }
      weight_sum[nt] = 0;
    }
  };
  if (first_place < end) {
    look_up();
    begin_tile();
  }
#pragma unroll
  for (int i = 0; i < R::STAGES; ++i) {
    if (loading < end) ask();
    else copies_commit();                // (every unit of the ring has a group of copies, be it empty)
  }
  for (int at = first_place, next; at < end; at = next) {
    const uint32_t pieces = present & ((1u << PARTS) - 1);
    present >>= PARTS;
    --queued;
    copies_wait<R::STAGES - 1>();
    __syncwarp();
    const uint32_t slot = ring + slot_out * R::SLOT;
    slot_out = slot_out + 1 == R::STAGES ? 0 : slot_out + 1;
    if (pieces) {
      const int token = (work.s.begin + work.step) * UNIT;
      const uint32_t keys = slot, values = keys + R::CODES;
      const uint32_t of_keys = slot + 2 * R::CODES + (lane >> 2) * (GROUPS * 4), of_values = of_keys + R::SCALES;

      float s[NT][PARTS][4];             // S^T: tokens 16 m + lane / 4 (+ 8), rows as in o
#pragma unroll
      for (int m = 0; m < PARTS; ++m) {
        uint32_t codes[2][CHUNKS];       // of tokens 16 m + lane / 4 (+ 8): elements 32 c + 8 (lane % 4) ..
        if constexpr (D == 128) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int r = 16 * m + 8 * h + (lane & 7), c = lane >> 3;
            ldmatrix_x4(codes[h], keys + r * 64 + ((c ^ swizzle_of<D>(lane & 7)) << 4));
          }
        } else {
          const int r = 16 * m + 8 * (lane >> 4) + (lane & 7), c = (lane >> 3) & 1;
          uint32_t all[4];
          ldmatrix_x4(all, keys + r * 32 + ((c ^ swizzle_of<D>(lane & 7)) << 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) codes[e >> 1][e & 1] = all[e];
        }
        float x[NT][GROUPS][4] = {};
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            const uint32_t a = codes[0][c] >> (8 * pair), b = codes[1][c] >> (8 * pair);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              Elem<T>::mma16816(x[nt][c / OF_GROUP], a & LOW, b & LOW, Codes<T>::odd(a), Codes<T>::odd(b), qf[nt][c][2 * pair],
                                qf[nt][c][2 * pair + 1]);
          }
        Words<GROUPS> w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) w[h] = lds<GROUPS>(of_keys + (16 * m + 8 * h) * (GROUPS * 4));
        if (BY_PRODUCT) {
          // minima of tokens 16 m + lane / 4 (+ 8): elements 2 (lane % 4) (+ 1) are groups, in turn
          uint32_t minima[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            minima[h] = GROUPS == 1   ? prmt(w[h].w[0], w[h].w[0], 0x3232)
                        : GROUPS == 2 ? prmt(w[h].w[0], w[h].w[GROUPS > 1], 0x7632)
                                      : (lane & 1) ? prmt(w[h].w[GROUPS / 2], w[h].w[GROUPS - 1], 0x7632)
                                                   : prmt(w[h].w[0], w[h].w[GROUPS > 1], 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][m][e] = 0.f;
            Elem<T>::mma16816(s[nt][m], minima[0], minima[1], minima[0], minima[1], q_parts[nt][0], q_parts[nt][1]);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const float by = Elem<T>::to_float(uint16_t(w[h].w[g])), from = Elem<T>::to_float(uint16_t(w[h].w[g] >> 16));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& sum = s[nt][m][2 * h + e];
                if (!BY_PRODUCT) sum = fmaf(from, q_sum[nt][e][g], g == 0 ? 0.f : sum);
                sum = fmaf(by, x[nt][g][2 * h + e], sum);
              }
          }
        }
      }
      const bool all = pieces == (1u << PARTS) - 1 && token + UNIT - 1 <= least && (p.window == 0 || token > most - p.window);
      uint32_t hidden[NT] = {};          // bit 4 m + e: of s[nt][m][e]
      if (!all) {
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
          const bool there = (pieces >> m) & 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = token + 16 * m + (lane >> 2) + 8 * (e >> 1), at_row = position[nt][e & 1];
              if (!there || t > at_row || (p.window > 0 && t <= at_row - p.window)) {
                s[nt][m][e] = -infinity;
                hidden[nt] |= 1u << (4 * m + e);
              }
            }
        }
      }
      // A row's maximum is raised only when a score exceeds it by more than SLACK: until then no lane has to know the others'.
      bool raise = false;
      float here[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          here[nt][e] = fmaxf(s[nt][0][e], s[nt][0][e + 2]);
#pragma unroll
          for (int m = 1; m < PARTS; ++m) here[nt][e] = fmaxf(here[nt][e], fmaxf(s[nt][m][e], s[nt][m][e + 2]));
          raise |= here[nt][e] * scale > top[nt][e] + SLACK;           // (from -inf: any)
        }
      const bool level = work.step % LEVEL == LEVEL - 1;
      if (__any_sync(0xffffffffu, raise || level)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float factor[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) here[nt][e] = fmaxf(here[nt][e], __shfl_xor_sync(0xffffffffu, here[nt][e], d));
            const float now = fmaxf(top[nt][e], here[nt][e] * scale);
            factor[e] = exp2_fast(top[nt][e] - (now == -infinity ? 0.f : now));
            top[nt][e] = now;
#pragma unroll
            for (int i = 0; i < SETS; ++i) middle[nt][e][i] *= factor[e];
          }
          weight_sum[nt] = mul_two(weight_sum[nt], two(factor[0], factor[1]));
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
              for (int t = 0; t < 2; ++t) o[nt][c][t][e] *= factor[e & 1];
        }
        // What the elements of a row's group have in common goes to `middle`.  (In this branch, which is rarely taken: behind the
        // product with values it cost 3 to 9 %.  Where registers are spilled, whenever it is taken: 8 new tokens for each of 64 sequences,
        // groups of 32, 177 us, 202 with a branch of its own; other tiles are 1 to 2 % faster with that.)
        if (level || SETS * NT > 4) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int g = 0; g < SETS; ++g)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float mean = 0.f;          // of this thread's four elements of a chunk, as codes in the lowest four bits
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                  if (c / OF_GROUP % SETS != g || (COPIES == 2 && c / OF_GROUP / SETS != upper)) continue;
#pragma unroll
                  for (int t = 0; t < 2; ++t) mean += fmaf(o[nt][c][t][e + 2], 0x1p-4f, o[nt][c][t][e]);
                }
#pragma unroll
                for (int d = 4; d < 32; d *= 2) mean += __shfl_xor_sync(0xffffffffu, mean, d);
                mean *= 1.f / GROUP;
                // (an eighth of 2^69 in each of eight lanes)
                middle[nt][e][g] = fmaf(mean * 0x1p66f, 1.f / UNIT_OF_WEIGHTS, middle[nt][e][g]);
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {
                  if (c / OF_GROUP % SETS != g) continue;
#pragma unroll
                  for (int t = 0; t < 2; ++t) o[nt][c][t][e] -= mean, o[nt][c][t][e + 2] = fmaf(mean, -16.f, o[nt][c][t][e + 2]);
                }
              }
        }
      }
      // weights
      const uint64_t scales = two(scale, scale);
      uint64_t origins[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        origins[nt] = two(OF_WEIGHTS - (top[nt][0] == -infinity ? 0.f : top[nt][0]),
                          OF_WEIGHTS - (top[nt][1] == -infinity ? 0.f : top[nt][1]));
      auto add_values = [&](auto whole) {
        float centres[NT][SETS][4] = {}; // (bf16) minus the centre's part of what this step adds to o, in its places
#pragma unroll
        for (int m = 0; m < PARTS; ++m) {
          uint32_t pf[NT][SETS][2], rest[NT][SETS][2];                 // (weights times scales)^T as B fragments
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float2 power = apart(fma_two(two(s[nt][m][e], s[nt][m][e + 1]), scales, origins[nt]));
              s[nt][m][e] = exp2_fast(power.x), s[nt][m][e + 1] = exp2_fast(power.y);
              weight_sum[nt] = add_two(weight_sum[nt], two(s[nt][m][e], s[nt][m][e + 1]));
            }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const Words<SETS> w = lds<SETS>(of_values + (16 * m + 8 * h) * (GROUPS * 4) + upper * (SETS * 4));
#pragma unroll
            for (int g = 0; g < SETS; ++g) {
              const float by = Elem<T>::to_float(uint16_t(w.w[g])), from = Elem<T>::to_float(uint16_t(w.w[g] >> 16));
              const float middle_here = SPLIT ? from : fmaf(centre, by, from), factor = by * OF_SCALES;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float scaled[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  // (what is hidden may be anything, and 0 * NaN is NaN)
                  const bool seen = decltype(whole)::value || !(hidden[nt] >> (4 * m + 2 * h + e) & 1);
                  scaled[e] = seen ? s[nt][m][2 * h + e] * factor : 0.f;
                  if (seen) middle[nt][e][g] = fmaf(s[nt][m][2 * h + e], middle_here, middle[nt][e][g]);
                }
                const uint32_t rounded = Elem<Wide>::pack2(scaled[0], scaled[1]);
                pf[nt][g][h] = movmatrix(rounded);
                if (SPLIT) {
                  const float a = Elem<Wide>::to_float(uint16_t(rounded)), b = Elem<Wide>::to_float(uint16_t(rounded >> 16));
                  rest[nt][g][h] = movmatrix(Elem<Wide>::pack2(scaled[0] - a, scaled[1] - b));
                }
              }
            }
          }
          if (!SPLIT) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int g = 0; g < SETS; ++g) {
                const uint32_t(&f)[2] = pf[nt][g];
                Elem<Wide>::mma16816(centres[nt][g], LOW_CENTRE, HIGH_CENTRE, LOW_CENTRE, HIGH_CENTRE, f[0], f[1]);
              }
          }
#pragma unroll
          for (int pair = 0; pair < CHUNKS / 2; ++pair) {
            // codes of tokens 16 m + 2 (lane % 4) (+ 1; + 8): elements 32 c + 4 (lane / 4) .. of chunks 2 pair and 2 pair + 1
            const int r = 16 * m + (lane & 15), c = 2 * pair + (lane >> 4);
            uint32_t codes[4];
            ldmatrix_x4_trans(codes, values + r * R::ROW + ((c ^ swizzle_of<D>(lane & 7)) << 4));
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                const uint32_t a = codes[2 * i] >> (8 * t), b = codes[2 * i + 1] >> (8 * t);
                const int at_chunk = 2 * pair + i;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const uint32_t(&f)[2] = pf[nt][at_chunk / OF_GROUP % SETS];
                  Elem<Wide>::mma16816(o[nt][at_chunk][t], a & LOW, a & HIGH, b & LOW, b & HIGH, f[0], f[1]);
                  if (SPLIT) {
                    const uint32_t(&left)[2] = rest[nt][at_chunk / OF_GROUP % SETS];
                    Elem<Wide>::mma16816(o[nt][at_chunk][t], a & LOW, a & HIGH, b & LOW, b & HIGH, left[0], left[1]);
                  }
                }
              }
          }
        }
        if (!SPLIT) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
              for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][c][t][e] += centres[nt][c / OF_GROUP % SETS][e];
        }
      };
      if (all) add_values(Bool<true>{});
      else add_values(Bool<false>{});
      __syncwarp();                      // every lane is done with the slot
    }
    if (loading < end) ask();
    else copies_commit();

    const bool last_step = work.step + 1 == work.s.steps;
    next = at + work.distance();
    if (!last_step && next < end) {
      ++work.step;
    } else {
      // ---- the tile's end, or the share's
      const int tile_row = work.tile * TILE, rows = min(TILE, work.s.rows - tile_row);
      const int item_begin = at - work.step, item_end = item_begin + work.s.steps;       // the tile's places, maybe of other warps
      const bool begins = item_begin >= 0, whole = begins && last_step;
      float* part = part_of(warp, begins);
      // (a last part lies in the ring, which nothing is on its way to any more)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = (nt * 8 + 2 * (lane & 3) + e) % COLUMNS;
          float sum_all = e ? apart(weight_sum[nt]).y : apart(weight_sum[nt]).x;
#pragma unroll
          for (int d = 4; d < 32; d *= 2) sum_all += __shfl_xor_sync(0xffffffffu, sum_all, d);
          sum_all *= UNIT_OF_WEIGHTS;
          float constant[SETS];
#pragma unroll
          for (int g = 0; g < SETS; ++g) {
            float m = middle[nt][e][g];
#pragma unroll
            for (int d = 4; d < 32; d *= 2) m += __shfl_xor_sync(0xffffffffu, m, d);
            constant[g] = m * UNIT_OF_WEIGHTS;
          }
          const int token = (tile_row + min(r, rows - 1)) / p.group, of_group = tile_row + min(r, rows - 1) - token * p.group;
          uint16_t* to = p.out + (int64_t(work.s.first_row + token) * p.q_heads + work.head * p.group + of_group) * D + 4 * (lane >> 2);
          float inverse = 1.f;
          if (whole && r < rows) inverse = sum_all == 0.f ? of_nothing(p, work.b, work.s.first_row + token) : 1.f / sum_all;
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            if (COPIES == 2 && c / OF_GROUP / SETS != upper) continue;
            const float from = constant[c / OF_GROUP % SETS];
            const float x[4] = {fmaf(o[nt][c][0][e], 0x1p69f, from), fmaf(o[nt][c][0][e + 2], 0x1p65f, from),
                                fmaf(o[nt][c][1][e], 0x1p69f, from), fmaf(o[nt][c][1][e + 2], 0x1p65f, from)};
            if (whole) {
              if (r < rows)
                *reinterpret_cast<uint2*>(to + 32 * c) =
                    make_uint2(Elem<T>::pack2(x[0] * inverse, x[1] * inverse), Elem<T>::pack2(x[2] * inverse, x[3] * inverse));
            } else {
              // (pieces change places with the row, so that a store meets 32 banks)
              *reinterpret_cast<float4*>(part + r * D + 4 * ((8 * c + (lane >> 2)) ^ (2 * (r >> 1 & 3)))) =
                  make_float4(x[0], x[1], x[2], x[3]);
            }
          }
          if (!whole && lane < 4 / COPIES) {
            part[ROWS * D + r] = top[nt][e];
            part[ROWS * (D + 1) + r] = sum_all;
          }
        }
      }
      if (!whole && lane == 0) {
        Left& mine = left[2 * warp + begins];
        mine.there = 1;
        mine.begin = origin + item_begin, mine.end = origin + item_end;
        mine.row = work.s.first_row, mine.head = work.head, mine.tile_row = tile_row, mine.rows = rows, mine.sequence = work.b;
      }
      if (next < end) {
        work.advance(p, TILE);
        begin_tile();
      }
    }
  }
  // ---- the warps' parts, then the CTAs': of every tile that was cut in this CTA, a thread per row and eight elements
  __syncthreads();
  const int of_cta = WARPS * start.share;
  // Where they begin: with a warp's last part, or the CTA's very first (the first part of another warp goes on with one before).
  uint32_t tiles = __ballot_sync(0xffffffffu, lane < 2 * WARPS && (lane % 2 == 1 || lane == 0) && left[lane].there);
  constexpr int OF_TILE = ROWS * (D / 8);
  for (int at = tid, before = 0; tiles; tiles &= tiles - 1, before += OF_TILE) {
    if (at >= before + OF_TILE) continue;
    const int from = __ffs(tiles) - 1, first = from / 2, w = at - before, r = w / (D / 8), c = w - r * (D / 8);
    at += THREADS;
    const Left item = left[from];
    const bool begins = item.begin >= 0, whole = begins && item.end <= of_cta;
    int count = 1;                       // warps that have a part of it
    while (first + count < WARPS && left[2 * (first + count)].there && left[2 * (first + count)].begin == item.begin) ++count;
    if (r >= item.rows) continue;
    auto part = [&](int v) { return part_of(first + v, v == 0 ? from % 2 : 0); };
    float maxima[WARPS], m = -infinity, l = 0.f, x[8] = {};
#pragma unroll
    for (int v = 0; v < WARPS; ++v) maxima[v] = v < count ? part(v)[ROWS * D + r] : -infinity;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) m = fmaxf(m, maxima[v]);
    const float top_here = m == -infinity ? 0.f : m;
#pragma unroll
    for (int v = 0; v < WARPS; ++v) {
      if (v >= count) break;
      const float f = exp2_fast(maxima[v] - top_here);
      l = fmaf(part(v)[ROWS * (D + 1) + r], f, l);
      const float4* of_row = reinterpret_cast<const float4*>(part(v) + r * D + 8 * (c ^ (r >> 1 & 3)));
      const float4 low = of_row[0], high = of_row[1];
      x[0] = fmaf(low.x, f, x[0]), x[1] = fmaf(low.y, f, x[1]), x[2] = fmaf(low.z, f, x[2]), x[3] = fmaf(low.w, f, x[3]);
      x[4] = fmaf(high.x, f, x[4]), x[5] = fmaf(high.y, f, x[5]), x[6] = fmaf(high.z, f, x[6]), x[7] = fmaf(high.w, f, x[7]);
    }
    if (whole) {
      const int token = (item.tile_row + r) / p.group, of_group = item.tile_row + r - token * p.group;
      const float inverse = l == 0.f ? of_nothing(p, item.sequence, item.row + token) : 1.f / l;
      *reinterpret_cast<uint4*>(p.out + (int64_t(item.row + token) * p.q_heads + item.head * p.group + of_group) * D + 8 * c) =
          make_uint4(Elem<T>::pack2(x[0] * inverse, x[1] * inverse), Elem<T>::pack2(x[2] * inverse, x[3] * inverse),
                     Elem<T>::pack2(x[4] * inverse, x[5] * inverse), Elem<T>::pack2(x[6] * inverse, x[7] * inverse));
    } else {
      float* to_part = p.parts + size_t(2 * blockIdx.x + begins) * (ROWS * (D + 2));
      float4* to = reinterpret_cast<float4*>(to_part + r * D + 8 * c);
      to[0] = make_float4(x[0], x[1], x[2], x[3]);
      to[1] = make_float4(x[4], x[5], x[6], x[7]);
      if (c == 0) {
        to_part[ROWS * D + r] = m;
        to_part[ROWS * (D + 1) + r] = l;
      }
      if (w == 0 && begins) {
        entry->row = item.row;
        entry->head = item.head;
        entry->tile_row = item.tile_row;
        entry->rows = item.rows;
        entry->sequence = item.sequence;
        entry->last_cta = blockIdx.x + (item.end - 1) / of_cta;
      }
    }
  }
}

template <typename T, int D, int GROUP, int TILE>
int launch(const Int4Cache& cache, const PagedParams& p, int grid, cudaStream_t stream) {
  auto kernel = paged_rows_int4_kernel<T, D, GROUP, TILE>;
  constexpr int smem = smem_bytes<D, GROUP, TILE>(), threads = 32 * Ring<D, GROUP, TILE>::WARPS;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_status(e);
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel),
                         TILE == 4   ? "paged_rows_int4_kernel 4 rows"
                         : TILE == 8 ? "paged_rows_int4_kernel 8 rows" : "paged_rows_int4_kernel 16 rows", grid, threads, smem, 1);
  e = launch_programmatic(kernel, dim3(unsigned(grid)), dim3(threads), smem, stream, 1, cache, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

template <typename T, int D, int GROUP>
int launch_rows(const Int4Cache& cache, const PagedParams& p, int tile_rows, int grid, cudaStream_t stream) {
  if constexpr (GROUP < D)
    if (tile_rows == 4) return launch<T, D, GROUP, 4>(cache, p, grid, stream);
  return tile_rows <= 8 ? launch<T, D, GROUP, 8>(cache, p, grid, stream) : launch<T, D, GROUP, 16>(cache, p, grid, stream);
}

}  // namespace

template <typename T>
int paged_rows_int4(const PagedParams& p, int64_t dim, int tile_rows, const Int4Cache& cache, int grid, cudaStream_t stream) {
  if (dim == 64)
    return cache.group == 32 ? launch_rows<T, 64, 32>(cache, p, tile_rows, grid, stream)
                             : launch_rows<T, 64, 64>(cache, p, tile_rows, grid, stream);
  return cache.group == 32   ? launch_rows<T, 128, 32>(cache, p, tile_rows, grid, stream)
         : cache.group == 64 ? launch_rows<T, 128, 64>(cache, p, tile_rows, grid, stream)
                             : launch_rows<T, 128, 128>(cache, p, tile_rows, grid, stream);
}
template int paged_rows_int4<__half>(const PagedParams&, int64_t, int, const Int4Cache&, int, cudaStream_t);
template int paged_rows_int4<__nv_bfloat16>(const PagedParams&, int64_t, int, const Int4Cache&, int, cudaStream_t);

}  // namespace ib200
