// Attention of chunks of new tokens over a paged cache on tcgen05 (paged_attention; the definition is in paged_rows.cu).
//
// A tile of queries is 256 rows: new tokens of one sequence with all query heads that share a key head (row = token x group +
// head), in two halves of 128.  For every step of 128 tokens of the cache and each half
//   S = Q K^T          tcgen05.mma, both operands from shared memory, 128 x 128 f32 in tensor memory
//   P = 2^(S - m)      128 threads, one row each: no exchange between threads; P goes back over S as 16-bit values
//   O += P V           tcgen05.mma, P from tensor memory, V as the cache holds it (N-major)
// Both halves use the same keys and values, and while one half's threads work out exponentials the tensor core has the other
// half's two products to do.  A row's running maximum m is only raised when it grows by more than 8 (a factor of 256, which
// 16-bit weights and f32 sums hold without loss): then O is scaled where it lies.  Every sum uses the m its weights were made
// with, so that the result does not depend on when that is.
//
// The steps of all tiles of all sequences form one line, of which every CTA takes the same length (as in paged_rows.cu); how
// many steps a tile has follows from its last token's position and its first one's window, and the sums of these over the
// tiles of a sequence are evaluated in closed form (sum of floor((a j + b) / m)), so a CTA finds its place in a few divisions.
// Tiles that a CTA boundary cuts leave maximum, sum and unscaled result per part, and join_chunk adds the parts in order.
//
// Keys and values come through a ring of TMA boxes of one page's rows each (128B swizzle, one lane per box); boxes of tokens
// that no query of the tile sees are asked for behind the cache's end, where TMA fills in zeros.
//
// Of a cache in 4 bits (GROUP > 0) codes and scales come by bulk copies, a run of bytes per page, and four warps turn them into the
// operands, numbers of the 16-bit type, in the ring's slots.  Rounding them is what reading the cache back would do.  A pair of codes
// costs four instructions for keys, three for values, whose columns then lie in another order (column_of).  4096 tokens behind 12288
// take 1010 - 1018 us with groups of 32, the same call on 16-bit elements 920.  (With three for keys, too, which would need the
// queries in that order, it is the same time.)  The rows' threads have 208 registers here in place of 224, and 38 to 46 bytes of
// them are spilled.
//
// Measured on one B200: 4096 tokens behind 12288, 32 heads of 128 on 8 key heads, bf16: 0.92 ms, 1.05 PFLOP/s of what the queries
// see, at the power cap (1.6 GHz, 1000 W).  A step takes 3500 cycles there: the tensor core is busy for 58 % of them (a half's two
// products take 1440, as both operands of S come through shared memory), the exponential unit for 59 %; the rest is the chain of
// one half, scores to registers, exponentials (1450), weights back, which two halves do not hide altogether.  With the arithmetic
// on the scores left out the same call takes 0.80 ms.  Tried and not kept: a part of the exponentials by a cubic on the FMA units
// (fewer cycles, the same time at the power cap), two threads per row (0.94 -> 1.04 ms, they have to exchange the maximum every
// step), the maximum looked for only when a sum says so (0.91 -> 0.90 ms, short calls 3 % slower), scores read in two loads with the
// first one's maximum between them (0.91 -> 0.93 ms).
//
// Heads of 64: a step takes 3500 cycles as well (1024 tokens behind 7168, 32 heads on 4 key heads: 111 us).  The products take half
// as long, but a half's chain is what counts: scores into registers 360, maximum 450, weights 1700, handed over and multiplied by V
// 400, the next scores 600.  Not kept for them: weights beside the scores in tensor memory, which takes the products off the chain
// (three prompts with a window 115 -> 123 us, 111 -> 127 with one half's products between the other's two: the halves then do the
// same things at the same time and each takes longer, 3770 cycles a step); a cubic for an eighth or a quarter of the exponentials
// (111 -> 113 and 114).
#include <algorithm>
#include <atomic>
#include <cstddef>
#include <type_traits>

#include "common.cuh"
#include "paged.cuh"
#include "paged_join.cuh"
#include "tma.cuh"
#include "umma.cuh"

namespace ib200 {
namespace {

constexpr int STEP = 128;                  // tokens of a step
// Warps 0..3 and 4..7: a half's rows; 10 .. 13 turn codes of a cache in 4 bits into operands.  What is left only lends registers.
constexpr int LOAD_WARP = 9, MMA_WARP = 8, CONVERT_WARPS = 4;
// Registers of a thread: the launch's, then those of a row's thread (128 scores and more) and of the others.
struct Split {
  int threads, launch, row, other;
};
// (with two warps for the codes, on two of the four schedulers, 4096 tokens behind 12288 took 1129 us, with four 1014)
constexpr Split WIDE = {12 * 32, 168, 224, 56}, INT4 = {16 * 32, 128, 208, 48};
constexpr bool shared_out(const Split& s) { return 256 * s.row + (s.threads - 256) * s.other <= s.threads * s.launch; }
static_assert(shared_out(WIDE) && shared_out(INT4), "the warpgroups share the launch's registers");
constexpr Split split_of(int group) { return group ? INT4 : WIDE; }
// Places on the line ahead of the steps of a tile, for what it costs beside them (four chunks of up to 500 tokens beside 20 single
// ones, 16-bit heads of 128: 149 us without, 142 with one, 137 with two, 136 with three, 137 with four; 33 tokens behind 7967:
// 28.2 without, 26.1 with two; long chunks alike).
constexpr int BEGIN = 2;
constexpr int EARLY = 96;                  // tokens of a step whose weights the products begin with
constexpr float SLACK = 8.f;               // growth of a row's maximum (log2) that its weights are left to absorb

// GROUP: elements of a group of a cache in 4 bits, 0 for one of 16-bit elements
template <int D, int GROUP>
struct Room {
  static constexpr int BOX = STEP * 128;                 // 64 elements of 128 rows
  static constexpr int OPERAND = BOX * (D / 64);
  static constexpr int SLOTS = GROUP ? (D == 128 ? 4 : 8) : D == 128 ? 5 : 10;
  // codes of a step's keys or values, and their scales, on their way to a slot
  static constexpr int GROUPS = GROUP ? D / (GROUP ? GROUP : D) : 0, ROW = D / 2;
  static constexpr int STAGES = GROUP ? (D == 128 ? 3 : 4) : 0, CODES = STEP * ROW, STAGE = CODES + STEP * GROUPS * 4;
  static constexpr int OPERANDS = (2 + SLOTS) * OPERAND, BYTES = OPERANDS + STAGES * STAGE;
};

// Column of an element among eight: values of a cache in 4 bits are put down as they come out of a word, one of its lower four
// codes beside one of its upper.
template <int GROUP>
__host__ __device__ constexpr int column_of(int element) {
  return GROUP == 0 ? element : (element & ~7) + 2 * (element & 3) + (element >> 2 & 1);
}

// ---- the line of steps -----------------------------------------------------------------------------------------------
struct Sequence {
  int count, first_row, length, first;     // new tokens, their first row of q, tokens in the cache, position of the first
  int tiles;                               // of a key head
};

__device__ __forceinline__ Sequence sequence_of(const PagedParams& p, int b) {
  Sequence s;
  const TokenSpan span = span_of(p, b);
  s.count = span.count * p.group > p.few ? span.count : 0;
  s.first_row = span.begin;
  s.length = min(max(__ldg(p.lengths + b), 0), p.capacity);
  s.first = s.length - s.count;
  s.tiles = (s.count + 2 * p.half_tokens - 1) / (2 * p.half_tokens);
  return s;
}

// A tile takes its steps' places on the line and BEGIN more ahead of them, for what it costs beside its steps: queries, the
// steps that hide some of their tokens, the results' way out.

// Steps of tile j: from that of the first token its first query sees to that of its last query's own.  (Of queries ahead of the
// first token, which see nothing, one step each is walked, all of it hidden.)
__device__ __forceinline__ int first_step(const PagedParams& p, const Sequence& s, int j) {
  return p.window > 0 ? max(s.first + 2 * j * p.half_tokens - p.window + 1, 0) / STEP : 0;
}
__device__ __forceinline__ int steps_of(const PagedParams& p, const Sequence& s, int j) {
  const int end = max(s.first, 0) + min(s.count, 2 * (j + 1) * p.half_tokens);
  return (end + STEP - 1) / STEP - first_step(p, s, j);
}

// sum of floor((a j + b) / 128) over j < n, for n < 2^24, by Euclid's algorithm (the reciprocity of such sums: Graham, Knuth,
// Patashnik, Concrete Mathematics, 3.5): the whole parts of a / 128 and b / 128, then the same with the remainder of a as the divisor
__device__ __forceinline__ unsigned long long floor_sum(unsigned n, unsigned a, unsigned b) {
  static_assert(STEP == 128, "the divisor that it begins with");
  unsigned long long sum = (unsigned long long)(n * (n - 1ull) / 2) * (a >> 7) + (unsigned long long)n * (b >> 7);
  a &= 127, b &= 127;
  unsigned m = 128;
  while (true) {
    const unsigned last = a * n + b;                     // (a < 128)
    if (last < m) return sum;
    n = last / m;
    b = last - n * m;
    const unsigned t = m;
    m = a;
    a = t / m;
    sum += (unsigned long long)n * (n - 1ull) / 2 * a;
    a = t - a * m;
    sum += (unsigned long long)n * (b / m);
    b %= m;
  }
}

// Places of tiles 0 .. j - 1 of a key head.
__device__ __forceinline__ long long places_before(const PagedParams& p, const Sequence& s, int j) {
  const int size = 2 * p.half_tokens, start = max(s.first, 0), full = min(j, s.tiles - 1);
  if (j <= 0) return 0;
  unsigned long long sum = full > 0 ? floor_sum(full, size, unsigned(start) + size + STEP - 1) : 0;
  if (j == s.tiles) sum += (unsigned(start) + s.count + STEP - 1) / STEP;
  if (p.window > 0) {
    const int low = s.first - p.window + 1;              // first token that the first tile's first query sees
    const int from = low >= 0 ? 0 : (-low + size - 1) / size;
    if (j > from) sum -= floor_sum(j - from, size, unsigned(low + from * size));
  }
  return (long long)sum + (long long)BEGIN * j;
}

// Goes through the parts of tiles among a CTA's places [0, end); visit(sequence, head, tile, step, steps, all, at) gets the part's
// first step in its tile, how many it has, how many the tile has and the first one's place, and returns whether to go on.
struct Start {
  int b, head, tile, place;
};
template <typename Visit>
__device__ __forceinline__ void walk(const PagedParams& p, const Start& from, int end, Visit visit) {
  int b = from.b, head = from.head, tile = from.tile, place = from.place, at = 0;
  Sequence s = sequence_of(p, b);
  while (true) {
    const int all = steps_of(p, s, tile), places = min(BEGIN + all - place, end - at);
    const int step = max(place - BEGIN, 0), steps = place + places - BEGIN - step;
    if (steps > 0 && !visit(s, b, head, tile, step, steps, all, at + max(BEGIN - place, 0))) return;
    at += places;
    if (at >= end) return;
    place = 0;
    if (++tile < s.tiles) continue;
    tile = 0;
    if (++head < p.k_heads) continue;
    head = 0;
    do {
      if (++b >= p.batch) return;            // (not unless the lengths change under the launch)
      s = sequence_of(p, b);
    } while (s.tiles == 0);
  }
}

// A CTA's share of a tile, as the loading warp leaves it to the others
struct Part {
  int row, head, tokens;   // first row of q, key head, new tokens from there on in the sequence
  int sequence;
  int position;            // of the first of them
  int first, steps;        // steps of 128 tokens
  int step, all, at;       // the first one's number in the tile, the tile's steps, the first one's place among the CTA's
                           // (steps = 0: there are no more)
};

// What a half of a tile sees
struct Half {
  int tokens;              // of it
  int least, most;         // positions of its first and last
  __device__ __forceinline__ Half(const PagedParams& p, int tile_tokens, int position, int half) {
    const int from = half * p.half_tokens;
    tokens = min(max(tile_tokens - from, 0), p.half_tokens);
    least = position + from;
    most = least + tokens - 1;
  }
  // whether any of its queries sees any token of the step that begins with `token`
  __device__ __forceinline__ bool sees(const PagedParams& p, int token) const {
    return tokens > 0 && token <= most && (p.window == 0 || token + STEP > least - p.window + 1);
  }
  // whether all of them see all of it
  __device__ __forceinline__ bool sees_all(const PagedParams& p, int token) const {
    return token + STEP - 1 <= least && (p.window == 0 || token > most - p.window);
  }
};

// ---- tensor memory -----------------------------------------------------------------------------------------------------
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_f16_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  const uint32_t acc = accumulate ? 1u : 0u;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t tmem_load_one(uint32_t taddr) {
  uint32_t v;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(v) : "r"(taddr) : "memory");
  tmem_load_wait();
  return v;
}

__device__ __forceinline__ void tmem_load_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// ---- weights -----------------------------------------------------------------------------------------------------------
// the largest of three; NaN if any is
__device__ __forceinline__ float largest(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Weights of 32 scores, rounded, and what they add up to.
template <typename T>
__device__ __forceinline__ void weigh(const uint32_t (&v)[32], uint64_t scale, uint64_t origin, uint64_t (&sum)[2], uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 x = apart(fma_two(two(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale, origin));
    const float a = exp2_fast(x.x), b = exp2_fast(x.y);
    sum[e & 1] = add_two(sum[e & 1], two(a, b));
    w[e] = Elem<T>::pack2(a, b);
  }
}

// Codes, masked where they are, as numbers m + s * n of the type, rounded once.  A pair of 16-bit words has a code each in its lowest
// four bits (which = 0), in the next (1), or in one word in these and in the other in those (2).
//   bf16  such bits are n or 16 n times the smallest number; a product makes n / 64 of them.  (Scales of 2^122 and more would not do.)
//   f16   beside the bits of 1024 they are 1024 + n or 1024 + 16 n, of which a product and a difference make n.
template <typename T>
struct Codes;
template <>
struct Codes<__nv_bfloat16> {
  __device__ static __forceinline__ uint32_t scale(uint32_t s) { return Elem<__nv_bfloat16>::mul2(s, 0x42804280u); }
  template <int WHICH>
  __device__ static __forceinline__ uint32_t number(uint32_t codes, uint32_t s, uint32_t m) {
    constexpr uint32_t MASK = WHICH == 0 ? 0x000f000fu : WHICH == 1 ? 0x00f000f0u : 0x00f0000fu;
    constexpr uint32_t BY = WHICH == 0 ? 0x7f007f00u : WHICH == 1 ? 0x7d007d00u : 0x7d007f00u;       // 2^127, 2^123
    return Elem<__nv_bfloat16>::fma2(Elem<__nv_bfloat16>::mul2(codes & MASK, BY), s, m);
  }
};
template <>
struct Codes<__half> {
  __device__ static __forceinline__ uint32_t scale(uint32_t s) { return s; }
  template <int WHICH>
  __device__ static __forceinline__ uint32_t number(uint32_t codes, uint32_t s, uint32_t m) {
    constexpr uint32_t MASK = WHICH == 0 ? 0x000f000fu : WHICH == 1 ? 0x00f000f0u : 0x00f0000fu;
    constexpr uint32_t BY = WHICH == 0 ? 0x3c003c00u : WHICH == 1 ? 0x2c002c00u : 0x2c003c00u;       // 1, 1 / 16
    constexpr uint32_t LESS = WHICH == 0 ? 0xe400e400u : WHICH == 1 ? 0xd400d400u : 0xd400e400u;     // 1024, 64
    return Elem<__half>::fma2(Elem<__half>::fma2(lop3_and_or(codes, MASK, 0x64006400u), BY, LESS), s, m);
  }
};
// eight of them in their order, and by column_of
template <typename T>
__device__ __forceinline__ uint4 numbers_in_order(uint32_t codes, uint32_t s, uint32_t m) {
  return make_uint4(Codes<T>::template number<2>(prmt(codes, 0u, 0x4040), s, m), Codes<T>::template number<2>(prmt(codes, 0u, 0x4141), s, m),
                    Codes<T>::template number<2>(prmt(codes, 0u, 0x4242), s, m), Codes<T>::template number<2>(prmt(codes, 0u, 0x4343), s, m));
}
template <typename T>
__device__ __forceinline__ uint4 numbers_by_column(uint32_t codes, uint32_t s, uint32_t m) {
  return make_uint4(Codes<T>::template number<0>(codes, s, m), Codes<T>::template number<1>(codes, s, m),
                    Codes<T>::template number<0>(codes >> 8, s, m), Codes<T>::template number<1>(codes >> 8, s, m));
}

// What lies behind the operands in shared memory
template <int SLOTS, int THREADS>
struct Shared {
  uint64_t q_full, q_empty, kv_full[SLOTS], kv_empty[SLOTS], s_full[2], p_full[2][2], o_full[2], vote_full[2], part_full[4],
      part_empty[4], products_over, stage_full[4], stage_empty[4];
  long long warp_sums[THREADS / 32];
  Part parts[4];
  long long start, start_head;             // this CTA's first place, counted in the sequence; places of a key head of it
  int start_sequence;
  volatile uint32_t tmem;
  volatile int skip[2];                    // this half's step has been added to O by its threads
  volatile uint32_t vote[2];               // step + 1 in which a warp of the half asked for that
  volatile uint32_t missing[8];            // per step, boxes of pages outside the cache
  volatile uint32_t absent[8];             // and of those, with boxes that no query sees, that were not asked for (4 bits)
};

template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(split_of(GROUP).threads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const Int4Cache cache, const PagedParams p) {
  using R = Room<D, GROUP>;
  constexpr int SLOTS = R::SLOTS, BOXES = D / 64, THREADS = split_of(GROUP).threads;
  using Behind = Shared<SLOTS, THREADS>;
  extern __shared__ unsigned char smem_raw[];
  programmatic_begin();
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t queries = base, ring = base + 2 * R::OPERAND;
  Behind& sh = *reinterpret_cast<Behind*>(base_ptr + R::BYTES);
  const uint32_t bars = base + R::BYTES;
  const uint32_t q_full = bars + offsetof(Behind, q_full), q_empty = bars + offsetof(Behind, q_empty),
                 kv_full = bars + offsetof(Behind, kv_full), kv_empty = bars + offsetof(Behind, kv_empty),
                 s_full = bars + offsetof(Behind, s_full), p_full = bars + offsetof(Behind, p_full),
                 o_full = bars + offsetof(Behind, o_full), vote_full = bars + offsetof(Behind, vote_full),
                 part_full = bars + offsetof(Behind, part_full), part_empty = bars + offsetof(Behind, part_empty),
                 products_over = bars + offsetof(Behind, products_over),
                 stage_full = bars + offsetof(Behind, stage_full), stage_empty = bars + offsetof(Behind, stage_empty);
  const uint32_t stages = base + R::OPERANDS;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    prefetch_tensormap(&map_q);
    if (GROUP == 0) {
      prefetch_tensormap(&map_k);
      prefetch_tensormap(&map_v);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(kv_full + 8 * i, GROUP ? CONVERT_WARPS : 1);
      mbar_init(kv_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 16 * i, 4);         // weights of the first EARLY tokens, then the others
      mbar_init(p_full + 16 * i + 8, 4);
      mbar_init(o_full + 8 * i, 1);
      mbar_init(vote_full + 8 * i, 4);
      sh.vote[i] = 0;
    }
    mbar_init(products_over, 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(part_full + 8 * i, 1);
      mbar_init(part_empty + 8 * i, GROUP ? 9 + CONVERT_WARPS : 9);      // the warps of both halves and the products'
    }
    if (GROUP)
      for (int i = 0; i < R::STAGES; ++i) {
        mbar_init(stage_full + 8 * i, 1);
        mbar_init(stage_empty + 8 * i, CONVERT_WARPS);
      }
    fence_mbar_init();
  }
  if (warp == MMA_WARP) tmem_alloc(bars + offsetof(Behind, tmem), 512);
  programmatic_wait();

  // ---- this CTA's part of the line
  const int per_thread = (p.batch + THREADS - 1) / THREADS, mine = tid * per_thread;
  long long sum = 0, each = 0;
  for (int b = mine; b < min(mine + per_thread, p.batch); ++b) {
    const Sequence s = sequence_of(p, b);
    each = places_before(p, s, s.tiles);
    sum += each * p.k_heads;
  }
  long long before = sum;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long v = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += v;
  }
  if (lane == 31) sh.warp_sums[warp] = before;
  __syncthreads();
  long long line = 0;
#pragma unroll 1
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += sh.warp_sums[w];
    line += sh.warp_sums[w];
  }
  before -= sum;
  const int share = share_of(line), cta = blockIdx.x;
  const long long begin = (long long)cta * share;
  const int end = share > 0 && begin < line ? int(min((long long)share, line - begin)) : 0;   // of this CTA's places, from its first on
  if (end > 0 && begin >= before && begin < before + sum) {
    int b = mine;
    long long at = before, of_head = each;
    for (; per_thread > 1; ++b) {
      const Sequence s = sequence_of(p, b);
      of_head = places_before(p, s, s.tiles);
      if (begin < at + of_head * p.k_heads || b + 1 >= min(mine + per_thread, p.batch)) break;
      at += of_head * p.k_heads;
    }
    sh.start_sequence = b;
    sh.start = begin - at;
    sh.start_head = of_head;
  }
  ChunkJoin* entry = static_cast<ChunkJoin*>(p.joins) + cta;
  if (tid == 0) {
    entry->last_cta = -1;
    if (share < 0) atomicExch(p.status, INTENT_B200_ERR_SHAPE);
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = sh.tmem;
  const uint32_t tmem_s = tmem, tmem_o = tmem + 2 * STEP;              // of both halves, 128 columns apart
  bool ok = true;

  if (end == 0) {
    // nothing to do
  } else if (warp >= MMA_WARP) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(split_of(GROUP).other));
    if (warp == LOAD_WARP) {
      // ------------------------------ loads ---------------------------------------
      Start at_first;
      at_first.b = sh.start_sequence;
      {
        const Sequence s = sequence_of(p, at_first.b);
        at_first.head = divide(sh.start, sh.start_head);
        const long long place = sh.start - at_first.head * sh.start_head;
        int low = 0, high = s.tiles;                                   // places_before(low) <= place < places_before(high)
        while (high - low > 1) {
          const int stride = (high - low + 31) / 32, j = low + lane * stride;
          const int fitting = __popc(__ballot_sync(0xffffffffu, j < high && places_before(p, s, j) <= place));
          low += (fitting - 1) * stride;
          high = min(low + stride, high);
        }
        at_first.tile = low;
        at_first.place = int(place - places_before(p, s, low));
      }
      const int rows = min(1 << p.page_shift, STEP);                   // of a box
      const int boxes = STEP / rows;                                   // of 64 elements of a step
      const int cache_rows = (p.pages * p.k_heads) << p.page_shift;
      uint32_t u = 0, parts = 0, odd = 0;                     // odd: keys asked for whose values were given up on
      walk(p, at_first, end, [&](const Sequence& s, int b, int head, int tile, int step, int steps, int all, int at) {
        const uint32_t place = parts & 3;
        ok = mbar_wait_warp(part_empty + 8 * place, (parts / 4 & 1) ^ 1) && mbar_wait_warp(q_empty, (parts & 1) ^ 1);
        if (!ok) return false;
        const int from = 2 * tile * p.half_tokens, position = s.first + from, tokens = min(s.count - from, 2 * p.half_tokens);
        const int first = first_step(p, s, tile) + step, halves = tokens > p.half_tokens ? 2 : 1;
        if (lane == 0) {
          Part& part = sh.parts[place];
          part.row = s.first_row + from, part.head = head, part.tokens = s.count - from, part.position = position;
          part.sequence = b;
          part.first = first, part.steps = steps, part.step = step, part.all = all, part.at = at;
          mbar_arrive(part_full + 8 * place);
          mbar_expect_tx(q_full, uint32_t(p.half_tokens * p.group * 128 * BOXES * halves));
          for (int half = 0; half < halves; ++half)
            for (int c = 0; c < BOXES; ++c)
              tma_load_3d(queries + half * R::OPERAND + c * R::BOX, &map_q, 64 * c, head * p.group,
                          s.first_row + from + half * p.half_tokens, q_full);
        }
        ++parts;
        // tokens that some query of the tile sees: [low, high)
        const int high = position + tokens, low = p.window > 0 ? max(position - p.window + 1, 0) : 0;
        for (int i = 0; i < steps; ++i, ++u) {
          const int box = lane % boxes, column = lane / boxes, token = (first + i) * STEP + box * rows;
          const bool wanted = token < high && token + rows > low;
          int page = -1;
          if (wanted) page = __ldg(p.page_table + int64_t(b) * p.table_width + (token >> p.page_shift));
          const bool there = page >= 0 && page < p.pages;
          const int row = there ? ((page * p.k_heads + head) << p.page_shift) + (token & ((1 << p.page_shift) - 1)) : cache_rows;
          const uint32_t missing = __ballot_sync(0xffffffffu, wanted && !there && column == 0);
          if constexpr (GROUP > 0) {
            // codes by the lanes of column 0, scales by those of column 1, each one run of bytes
            const uint32_t absent = __ballot_sync(0xffffffffu, !there && column == 0);
            const uint32_t bytes = uint32_t((boxes - __popc(absent)) * rows * (R::ROW + 4 * R::GROUPS));
#pragma unroll
            for (int operand = 0; operand < 2; ++operand) {
              const uint32_t stage = (2 * u + operand) % R::STAGES, turn = (2 * u + operand) / R::STAGES;
              ok = mbar_wait_warp(stage_empty + 8 * stage, (turn & 1) ^ 1);
              if (!ok) {
                odd = operand;
                return false;
              }
              if (lane == 0) {
                if (operand == 0) sh.missing[u & 7] = missing, sh.absent[u & 7] = absent;
                mbar_expect_tx(stage_full + 8 * stage, bytes);
              }
              __syncwarp();
              if (there && column < 2) {
                const uint32_t size = column ? 4 * R::GROUPS : R::ROW;                 // bytes of a token
                const void* from = operand == 0 ? (column ? cache.k_scales : cache.k_codes) : (column ? cache.v_scales : cache.v_codes);
                bulk_load(stages + stage * R::STAGE + column * R::CODES + box * rows * size,
                          static_cast<const unsigned char*>(from) + int64_t(row) * size, rows * size, stage_full + 8 * stage);
              }
              __syncwarp();
            }
          } else {
#pragma unroll
            for (int operand = 0; operand < 2; ++operand) {
              const uint32_t slot = (2 * u + operand) % SLOTS, turn = (2 * u + operand) / SLOTS;
              ok = mbar_wait_warp(kv_empty + 8 * slot, (turn & 1) ^ 1);
              if (!ok) {
                odd = operand;
                return false;
              }
              if (lane == 0) {
                if (operand == 0) sh.missing[u & 7] = missing;
                mbar_expect_tx(kv_full + 8 * slot, R::OPERAND);
              }
              __syncwarp();
              if (column < BOXES)
                tma_load_2d(ring + slot * R::OPERAND + column * R::BOX + box * rows * 128, operand == 0 ? &map_k : &map_v, 64 * column,
                            row, kv_full + 8 * slot);
              __syncwarp();
            }
          }
        }
        return true;
      });
      ok = ok && mbar_wait_warp(part_empty + 8 * (parts & 3), (parts / 4 & 1) ^ 1);
      if (ok && lane == 0) {
        sh.parts[parts & 3].steps = 0;
        mbar_arrive(part_full + 8 * (parts & 3));
      }
      // (also where another warp gave up: no load may be on its way to a CTA that is gone)
      if (parts > 0) mbar_wait_warp(q_full, (parts - 1) & 1);
      const uint32_t loads = 2 * u + odd, last = loads - 1 - lane;
      constexpr uint32_t PLACES = GROUP ? R::STAGES : SLOTS;
      if (lane < min(loads, PLACES)) mbar_wait((GROUP ? stage_full : kv_full) + 8 * (last % PLACES), last / PLACES & 1, 1u << 12);
      __syncwarp();
    } else if (GROUP > 0 && warp > LOAD_WARP && warp <= LOAD_WARP + CONVERT_WARPS) {
      // ------------------------------ codes to numbers ----------------------------
      // A lane turns 32 codes (16 bytes of a row) into four pieces of eight numbers where the products expect them, in an order in
      // which eight lanes meet 32 banks.  Keys' elements lie as the queries' do, values' by column_of.
      if constexpr (GROUP > 0) {
        constexpr int PER_ROW = D / 32, ROWS_AT_ONCE = 32 / PER_ROW, ROWS = STEP / CONVERT_WARPS;
        const int k = lane % PER_ROW, first_row = (warp - LOAD_WARP - 1) * ROWS + lane / PER_ROW;
        const bool swapped = (k & 2) != 0;
        const int shift = min(p.page_shift, 7);
        uint32_t parts = 0, n = 0;                                     // n: operands
        while (ok) {
          const uint32_t place = parts & 3;
          ok = mbar_wait_warp(part_full + 8 * place, parts / 4 & 1);
          if (!ok || sh.parts[place].steps == 0) break;
          const int steps = sh.parts[place].steps;
          ++parts;
          __syncwarp();
          if (lane == 0) mbar_arrive(part_empty + 8 * place);
          for (int i = 0; i < 2 * steps; ++i, ++n) {
            const uint32_t stage = n % R::STAGES, slot = n % SLOTS;
            ok = mbar_wait_warp(stage_full + 8 * stage, n / R::STAGES & 1) && mbar_wait_warp(kv_empty + 8 * slot, (n / SLOTS & 1) ^ 1);
            if (!ok) break;
            const uint32_t absent = sh.absent[(n / 2) & 7];
            const uint32_t codes = stages + stage * R::STAGE, scales = codes + R::CODES + (k * 32 / GROUP) * 4;
            unsigned char* to = base_ptr + (ring - base) + slot * R::OPERAND + (k >> 1) * R::BOX;
            auto convert = [&](auto values) {
#pragma unroll 1                            // (two rows at a time do not fit the registers: 1014 -> 1100 us)
              for (int r = first_row; r < first_row + ROWS; r += ROWS_AT_ONCE) {
                const uint4 v = lds128(codes + r * R::ROW + 16 * k);
                uint32_t pair;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(pair) : "r"(scales + r * (4 * R::GROUPS)));
                if (absent >> (r >> shift) & 1) pair = 0;              // (what is there was left by others)
                const uint32_t s = Codes<T>::scale(prmt(pair, pair, 0x1010)), m = prmt(pair, pair, 0x3232);
                const uint32_t words[4] = {swapped ? v.z : v.x, swapped ? v.w : v.y, swapped ? v.x : v.z, swapped ? v.y : v.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const uint4 out = decltype(values)::value ? numbers_by_column<T>(words[j], s, m) : numbers_in_order<T>(words[j], s, m);
                  const int piece = 4 * (k & 1) + (swapped ? j ^ 2 : j);
                  *reinterpret_cast<uint4*>(to + r * 128 + ((piece ^ (r & 7)) << 4)) = out;
                }
              }
            };
            if (i & 1) convert(Bool<true>{});
            else convert(Bool<false>{});
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(kv_full + 8 * slot);
              mbar_arrive(stage_empty + 8 * stage);
            }
          }
        }
      }
    } else if (warp == MMA_WARP) {
      // ------------------------------ products ------------------------------------
      constexpr uint32_t FORMAT = std::is_same<T, __half>::value ? 0 : 1;
      constexpr uint32_t scores = umma_idesc(1, FORMAT, FORMAT, 0, 0, HALF_ROWS, STEP);
      constexpr uint32_t results = umma_idesc(1, FORMAT, FORMAT, 0, 1, HALF_ROWS, D);
      const bool issue = elect_one();
      const uint64_t query_desc = umma_desc_k_major_sw128(queries), key_desc = umma_desc_k_major_sw128(ring),
                     value_desc = umma_desc_mn_major_sw128(ring, R::BOX);
      constexpr uint64_t UNIT = R::OPERAND / 16, BOX_UNIT = R::BOX / 16;       // in descriptors' 16 bytes
      uint32_t parts = 0, taken[2] = {0, 0};
      bool waiting[2] = {false, false}, begun[2] = {false, false}, mixed[2] = {false, false};
      // Places in the ring: of this step's keys, and of the values of the step before.  What is waited for between the products
      // of two steps leaves the tensor core idle, so all that can be is waited for ahead of the weights.
      uint32_t k_slot = 0, k_turn = 0, v_slot = SLOTS - 1, v_turn = 1;
      bool some = false;                                               // there is a step before
      // adds the values of the step before to a half that has its weights
      auto add = [&](int h) {
        const uint64_t values = value_desc + v_slot * UNIT;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          ok = ok && mbar_wait_warp(p_full + 16 * h + 8 * c, taken[h] & 1);
          if (!ok) return;
          tcgen05_fence_after();
          if (issue && !(mixed[h] && sh.skip[h])) {
#pragma unroll
            for (int k = c * (EARLY / 16); k < (c ? STEP / 16 : EARLY / 16); ++k)   // 16 tokens: 8 columns of P, 16 rows of 128 bytes
              umma_f16_tmem(tmem_o + h * 128, tmem_s + h * STEP + 8 * k, values + uint64_t(128 * k), results, begun[h] || k != 0);
          }
        }
        ++taken[h];
        waiting[h] = false;
        begun[h] = true;
      };
      // the same for a part's last step
      auto finish = [&](int h) {
        if (waiting[h]) add(h);
        if (ok && issue && begun[h]) umma_commit(o_full + 8 * h);
        begun[h] = false;
      };
      while (ok) {
        const uint32_t place = parts & 3;
        ok = mbar_wait_warp(part_full + 8 * place, parts / 4 & 1);
        if (!ok || sh.parts[place].steps == 0) break;
        const int steps = sh.parts[place].steps, first = sh.parts[place].first, tokens = sh.parts[place].tokens,
                  position = sh.parts[place].position;
        __syncwarp();
        if (lane == 0) mbar_arrive(part_empty + 8 * place);
        const Half half[2] = {Half(p, tokens, position, 0), Half(p, tokens, position, 1)};
        for (int i = 0; i < steps; ++i) {
          const int token = (first + i) * STEP;
          const bool sees[2] = {half[0].sees(p, token), half[1].sees(p, token)};
          if (some) ok = mbar_wait_warp(kv_full + 8 * v_slot, v_turn & 1);
          // (ahead of a new tile's first products a half may still have its last results to add)
          if (i > 0) ok = ok && mbar_wait_warp(kv_full + 8 * k_slot, k_turn & 1);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!ok) break;
            if (i == 0) {
              finish(h);
              if (h == 0 && ok) ok = mbar_wait_warp(q_full, parts & 1) && mbar_wait_warp(kv_full + 8 * k_slot, k_turn & 1);
              tcgen05_fence_after();
            } else if (waiting[h]) {
              add(h);
            }
            if (!ok || !sees[h]) continue;
            if (issue) {
#pragma unroll
              for (int k = 0; k < D / 16; ++k)      // 16 elements: 32 bytes of a row of 128
                umma_f16(tmem_s + h * STEP, query_desc + (h * UNIT + (k / 4) * BOX_UNIT + 2 * (k & 3)),
                         key_desc + (k_slot * UNIT + (k / 4) * BOX_UNIT + 2 * (k & 3)), scores, k != 0);
              umma_commit(s_full + 8 * h);
            }
            waiting[h] = true;
            mixed[h] = !half[h].sees_all(p, token);
          }
          if (!ok) break;
          if (issue) {
            if (some) umma_commit(kv_empty + 8 * v_slot);
            umma_commit(kv_empty + 8 * k_slot);
            if (i == steps - 1) umma_commit(q_empty);
          }
          __syncwarp();
          some = true;
          v_slot = k_slot + 1, v_turn = k_turn;
          if (v_slot == SLOTS) v_slot = 0, ++v_turn;
          k_slot = v_slot + 1, k_turn = v_turn;
          if (k_slot == SLOTS) k_slot = 0, ++k_turn;
        }
        ++parts;
      }
      // the last step's values: no slot is asked for again, but nothing may be on its way to a CTA that is gone
      if (some) ok = ok && mbar_wait_warp(kv_full + 8 * v_slot, v_turn & 1);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (ok) finish(h);
      // (also where a warp gave up: no product may be under way in tensor memory that is given back)
      if (issue) umma_commit(products_over);
      __syncwarp();
      mbar_wait_warp(products_over, 0);
    }
  } else {
    // ------------------------------ weights and results --------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(split_of(GROUP).row));
    const int h = warp >> 2, quadrant = warp & 3, row = quadrant * 32 + lane;
    const uint32_t lanes = uint32_t(quadrant * 32) << 16;
    const uint32_t at_s = tmem_s + h * STEP + lanes, at_o = tmem_o + h * 128 + lanes;
    const float infinity = __int_as_float(0x7f800000);
    const int row_token = row / p.group;                               // in the half
    uint32_t u = 0, parts = 0, seen = 0, done = 0, votes = 0;
    while (true) {
      const uint32_t place = parts & 3;
      ok = mbar_wait_warp(part_full + 8 * place, parts / 4 & 1);
      if (!ok || sh.parts[place].steps == 0) break;
      const volatile Part& part = sh.parts[place];
      ++parts;
      const int steps = part.steps, first = part.first, tokens = part.tokens, tile_position = part.position;
      const Half half(p, tokens, tile_position, h);
      const bool real = row_token < half.tokens;
      const int position = real ? half.least + row_token : -1;
      float top = -infinity, weight_sum = 0.f;
      bool begun = false;
      for (int i = 0; i < steps; ++i, ++u) {
        const int token = (first + i) * STEP;
        if (!half.sees(p, token)) continue;
        ok = mbar_wait_warp(s_full + 8 * h, seen & 1);
        ++seen;
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t missing = sh.missing[u & 7];
        const bool mixed = !half.sees_all(p, token), edge = mixed || missing != 0;
        const uint32_t slot = (2 * u + 1) % SLOTS, values = ring + slot * R::OPERAND;
        if (edge) {
          // Values that no query of the tile sees may be anything, and 0 * NaN is NaN: they become zeros.
          ok = mbar_wait_warp(kv_full + 8 * slot, ((2 * u + 1) / SLOTS) & 1);
          if (!ok) break;
          const int tile_high = tile_position + min(tokens, 2 * p.half_tokens);
          const int tile_low = p.window > 0 ? max(tile_position - p.window + 1, 0) : 0;
          unsigned char* mine_row = base_ptr + (values - base) + row * 128;     // (pieces in another order for every row: 32 banks)
          const bool outside = token + row < tile_low || token + row >= tile_high;
          if (outside) {
#pragma unroll 1
            for (int j = 0; j < 8 * BOXES; ++j)
              *reinterpret_cast<uint4*>(mine_row + (j / 8) * R::BOX + 16 * ((j ^ row) & 7)) = make_uint4(0, 0, 0, 0);
            fence_proxy_async();
          }
          // Those that some rows see and others do not have to be finite for the product; where they are not, the rows add
          // them up themselves, each from what it sees.  The warps of the half ask one another, and hear it after the weights.
          uint32_t sum[2] = {0, 0};
          if (mixed && !outside && (token + row > half.least || (p.window > 0 && token + row <= half.most - p.window))) {
#pragma unroll 4
            for (int j = 0; j < 8 * BOXES; ++j) {
              const uint4 x = *reinterpret_cast<const uint4*>(mine_row + (j / 8) * R::BOX + 16 * ((j ^ row) & 7));
              sum[0] = add_no_numbers<T>(x.x, sum[0]);
              sum[1] = add_no_numbers<T>(x.y, sum[1]);
              sum[0] = add_no_numbers<T>(x.z, sum[0]);
              sum[1] = add_no_numbers<T>(x.w, sum[1]);
            }
          }
          if (__any_sync(0xffffffffu, ((sum[0] | sum[1]) & 0x7fff7fffu) != 0) && lane == 0) sh.vote[h] = u + 1;
          __syncwarp();
          if (lane == 0) mbar_arrive(vote_full + 8 * h);
        }
        uint32_t v[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_load_32x32(at_s + 32 * c, v[c]);
        tmem_load_wait();
        if (edge) {
          const int behind = position - token, ahead = p.window > 0 ? behind - p.window : -1;   // seen: (ahead, behind]
          const int shift = min(p.page_shift, 7);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            // bit e: token 32 c + e is seen
            const int last = behind - 32 * c, none = ahead - 32 * c + 1;
            uint32_t shown = last < 0 ? 0u : last >= 31 ? ~0u : (2u << last) - 1;
            shown &= none <= 0 ? ~0u : none >= 32 ? 0u : ~0u << none;
            if (missing >> ((32 * c) >> shift) & 1) shown &= 0xffff0000u;
            if (missing >> ((32 * c + 16) >> shift) & 1) shown &= 0xffffu;
            if (missing == 0 && token + 32 * c + 31 <= half.least && (p.window == 0 || token + 32 * c > half.most - p.window)) continue;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(shown >> e & 1)) v[c][e] = 0xff800000u;
          }
        }
        float most[4] = {-infinity, -infinity, -infinity, -infinity};
#pragma unroll
        for (int e = 0; e < 32; e += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) most[c] = largest(most[c], __uint_as_float(v[c][e]), __uint_as_float(v[c][e + 1]));
        const float now = largest(largest(most[0], most[1], most[2]), most[3], -infinity) * p.scale;
        // (rows that are no query's hold what was in shared memory, or other sequences' queries, maybe no numbers: they ask for nothing)
        const bool raise = real && (!(now <= top + SLACK) || top == -infinity);
        const float factor = raise ? exp2_fast(top - (now == -infinity ? 0.f : now)) : 1.f;
        if (raise) top = now;
        weight_sum *= factor;
        if (begun && __any_sync(0xffffffffu, raise)) {
          // (S was asked for behind the product that adds the step before, so O is whole)
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_load_32x16(at_o + 16 * c, o);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_store_32x16(at_o + 16 * c, o);
          }
        }
        // (a score of +infinity, as one that is no number, makes the row none)
        const float origin = top == -infinity ? 0.f : top == infinity ? top - top : -top;
        const uint64_t scales = two(p.scale, p.scale), origins = two(origin, origin);
        uint64_t added[2] = {0, 0};
        uint32_t w[16];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          weigh<T>(v[c], scales, origins, added, w);
          tmem_store_32x16(at_s + 16 * c, w);
          if (c == EARLY / 32 - 1 && !edge) {
            tmem_store_wait();
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 16 * h);
          }
        }
        const float2 sums[2] = {apart(added[0]), apart(added[1])};
        weight_sum += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
        bool by_hand = false;
        if (edge) {
          ok = mbar_wait_warp(vote_full + 8 * h, votes & 1);
          ++votes;
          if (!ok) break;
          by_hand = sh.vote[h] == u + 1;
          if (by_hand) {
            tmem_store_wait();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_load_32x16(at_o + 16 * c, o);
              tmem_load_wait();
              if (!begun)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = 0;
              const int element = 16 * c, piece = element % 64 / 8;
#pragma unroll 1
              for (int k = 0; k < STEP; ++k) {
                __syncwarp();
                const uint32_t pair = tmem_load_one(at_s + k / 2);
                const float weight = Elem<T>::to_float(uint16_t(k & 1 ? pair >> 16 : pair));
                const int t = token + k;
                if (t > position || (p.window > 0 && t <= position - p.window)) continue;
                const unsigned char* value = base_ptr + (values - base) + element / 64 * R::BOX + k * 128;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint4 x = *reinterpret_cast<const uint4*>(value + (((piece + j) ^ (k & 7)) << 4));
                  const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                  for (int e = 0; e < 8; ++e)
                    o[8 * j + e] = __float_as_uint(fmaf(weight, Elem<T>::to_float(uint16_t(y[e / 2] >> (16 * (e & 1)))),
                                                        __uint_as_float(o[8 * j + e])));
                }
              }
              __syncwarp();
              tmem_store_32x16(at_o + 16 * c, o);
            }
          }
        }
        begun = true;
        if (edge && quadrant == 0 && lane == 0) sh.skip[h] = by_hand;
        tmem_store_wait();
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (edge) mbar_arrive(p_full + 16 * h);
          mbar_arrive(p_full + 16 * h + 8);
        }
      }
      if (!ok) break;

      // ---- the part's end
      if (begun) {
        ok = mbar_wait_warp(o_full + 8 * h, done & 1);
        ++done;
        if (!ok) break;
        tcgen05_fence_after();
      }
      const int all = part.all, tile_at = part.at - part.step, head = part.head, tile_row = part.row, sequence = part.sequence;
      __syncwarp();
      if (lane == 0) mbar_arrive(part_empty + 8 * place);
      const bool whole = steps == all;
      const bool begins = tile_at >= 0;                                // the tile, in this CTA
      if (tid == 0 && !whole && begins) {
        entry->row = tile_row;
        entry->head = head;
        entry->tokens = tokens;
        entry->sequence = sequence;
        entry->last_cta = cta + (tile_at + all - 1) / share;
      }
      float inverse = 0.f;
      if (whole && real)
        inverse = weight_sum == 0.f ? of_nothing(p, sequence, tile_row + h * p.half_tokens + row_token) : 1.f / weight_sum;
      float* to_part = p.parts + size_t(2 * cta + begins) * (2 * HALF_ROWS * (D + 2));
      uint16_t* to = p.out + (int64_t(tile_row + h * p.half_tokens + row_token) * p.q_heads + head * p.group +
                              (row - row_token * p.group)) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (begun) {
          tmem_load_32x32(at_o + 32 * c, o);
          tmem_load_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0;
        }
        if (real && whole) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              x[j] = Elem<T>::pack2(__uint_as_float(o[column_of<GROUP>(e + 2 * j)]) * inverse,
                                    __uint_as_float(o[column_of<GROUP>(e + 2 * j + 1)]) * inverse);
            *reinterpret_cast<uint4*>(to + 32 * c + e) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else if (real) {
          // [D / 4][256 rows][4]: neighbouring threads write neighbouring 16 bytes
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *reinterpret_cast<uint4*>(to_part + ((8 * c + e / 4) * 2 * HALF_ROWS + h * HALF_ROWS + row) * 4) =
                make_uint4(o[column_of<GROUP>(e)], o[column_of<GROUP>(e + 1)], o[column_of<GROUP>(e + 2)], o[column_of<GROUP>(e + 3)]);
        }
        __syncwarp();
      }
      if (!whole && real) {
        to_part[2 * HALF_ROWS * D + h * HALF_ROWS + row] = top;
        to_part[2 * HALF_ROWS * (D + 1) + h * HALF_ROWS + row] = weight_sum;
      }
      tcgen05_fence_before();
      __syncwarp();
    }
  }
  if (!ok && lane == 0) atomicExch(p.status, INTENT_B200_ERR_TIMEOUT);
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

template <typename T, int D, int GROUP>
int launch(const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, const Int4Cache& cache,
           const PagedParams& p, int grid, cudaStream_t stream) {
  constexpr int THREADS = split_of(GROUP).threads;
  auto kernel = paged_chunk_kernel<T, D, GROUP>;
  constexpr int smem = 1024 + Room<D, GROUP>::BYTES + int(sizeof(Shared<Room<D, GROUP>::SLOTS, split_of(GROUP).threads>));
  static_assert(smem <= 227 * 1024, "shared memory of a CTA");
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return cuda_status(e);
  // (the kernel shares the launch's registers out anew, which would wait for ever if there were fewer)
  static std::atomic<int> registers{0};    // (asked for until the answer comes: a call that fails does not decide for those after it)
  if (registers.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes attributes;
    e = cudaFuncGetAttributes(&attributes, kernel);
    if (e != cudaSuccess) return cuda_status(e);
    registers.store(attributes.numRegs, std::memory_order_relaxed);
  }
  if (registers.load(std::memory_order_relaxed) != split_of(GROUP).launch) return INTENT_B200_ERR_UNSUPPORTED;
  if (LaunchFacts* sink = observe_sink())
    return record_launch(sink, reinterpret_cast<const void*>(kernel), GROUP ? "paged_chunk_kernel int4 2 x 128 rows, parts joined"
                                                                                  : "paged_chunk_kernel 2 x 128 rows, parts joined", grid,
                         THREADS, smem, 1);
  e = launch_programmatic(kernel, dim3(unsigned(grid)), dim3(THREADS), smem, stream, 1, map_q, map_k, map_v, cache, p);
  if (e != cudaSuccess) return cuda_status(e);
  note_launch();
  return launch_status();
}

}  // namespace

int64_t paged_chunk_parts_bytes(int64_t dim) {
  return int64_t(2) * kPagedCtas * 2 * HALF_ROWS * (dim + 2) * int64_t(sizeof(float));
}

bool paged_chunk_takes(const PagedParams& p) {
  return p.group <= HALF_ROWS && (p.tokens == 1 || p.q_token > 0) && (p.q_heads == 1 || p.q_head > 0);
}

int paged_chunk_half_tokens(const PagedParams& p) { return HALF_ROWS / p.group; }

namespace {

// 64 elements of the queries of half a tile
template <typename T>
bool map_queries(CUtensorMap* map, const PagedParams& p, int64_t dim) {
  EncodeTiledFn encode = encode_tiled_fn();
  constexpr auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(p.q_heads), cuuint64_t(p.tokens)};
  const cuuint64_t strides[2] = {cuuint64_t(p.q_heads > 1 ? p.q_head : dim) * 2,
                                 cuuint64_t(p.tokens > 1 ? p.q_token : p.q_heads * dim) * 2};
  const cuuint32_t sizes[3] = {64, cuuint32_t(p.group), cuuint32_t(p.half_tokens)}, ones[3] = {1, 1, 1};
  return encode && encode(map, type, 3, const_cast<uint16_t*>(p.q), dims, strides, sizes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

template <typename T>
int paged_chunk(const PagedParams& p, int64_t dim, const void* k_cache, const void* v_cache, int grid, cudaStream_t stream) {
  CUtensorMap map_q, map_k, map_v;
  const uint64_t rows = uint64_t(p.pages) * uint64_t(p.k_heads) << p.page_shift;
  constexpr auto type = std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t box = uint32_t(std::min(1 << p.page_shift, STEP));
  if (!map_queries<T>(&map_q, p, dim) ||
      !make_tensor_map_2d(&map_k, type, k_cache, rows, uint64_t(dim), uint64_t(dim) * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_tensor_map_2d(&map_v, type, v_cache, rows, uint64_t(dim), uint64_t(dim) * 2, box, 64, CU_TENSOR_MAP_SWIZZLE_128B))
    return INTENT_B200_ERR_CUDA;
  const Int4Cache none = {};
  return dim == 128 ? launch<T, 128, 0>(map_q, map_k, map_v, none, p, grid, stream)
                    : launch<T, 64, 0>(map_q, map_k, map_v, none, p, grid, stream);
}
template int paged_chunk<__half>(const PagedParams&, int64_t, const void*, const void*, int, cudaStream_t);
template int paged_chunk<__nv_bfloat16>(const PagedParams&, int64_t, const void*, const void*, int, cudaStream_t);

template <typename T>
int paged_chunk_int4(const PagedParams& p, int64_t dim, const Int4Cache& cache, int grid, cudaStream_t stream) {
  CUtensorMap map;
  if (!map_queries<T>(&map, p, dim)) return INTENT_B200_ERR_CUDA;
  if (dim == 64)
    return cache.group == 32 ? launch<T, 64, 32>(map, map, map, cache, p, grid, stream)
                             : launch<T, 64, 64>(map, map, map, cache, p, grid, stream);
  return cache.group == 32   ? launch<T, 128, 32>(map, map, map, cache, p, grid, stream)
         : cache.group == 64 ? launch<T, 128, 64>(map, map, map, cache, p, grid, stream)
                             : launch<T, 128, 128>(map, map, map, cache, p, grid, stream);
}
template int paged_chunk_int4<__half>(const PagedParams&, int64_t, const Int4Cache&, int, cudaStream_t);
template int paged_chunk_int4<__nv_bfloat16>(const PagedParams&, int64_t, const Int4Cache&, int, cudaStream_t);

}  // namespace ib200
