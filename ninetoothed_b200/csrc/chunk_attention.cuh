// Causal attention of the next pieces of prompts, packed one after another, over the
// paged 8-bit cache that holds them already:
//     s = (q . k_code) * (scale * key_scale[page]),  o = sum_j softmax(s)_j * value_scale[page_j] * v_code_j,
//     lse = ln sum_j exp(s_j)
// Sequence b has the queries offsets[b] .. offsets[b+1] - 1 and lengths[b] cached
// tokens, its last query standing at the last of them.  A query that sees no token gets
// o = 0 and lse = -inf.  All math is base 2 in fp32.
//
// Bound by the tensor cores and, level with them, by the exponentials (a block of 128
// keys costs 256 rows 2048 cycles of either); short pieces by reading the cache once.
//
// Rows of a tile are (query, head of the group) pairs, so that all query heads of a
// key/value head share one pass over its keys: 128 / group queries a tile.  A unit of
// work is a key/value head and two tiles of 128 rows; its blocks of 128 keys, with
// UNIT_STEPS more for its start and end, are steps of one line: sequence by sequence,
// head by head.  The line is cut into equal pieces, one a CTA, so that any mix of
// lengths keeps every SM busy to the end, and a few rows over many keys as well.  Where a
// cut falls into a unit, its pieces leave (o, m, l) in a workspace and a second kernel
// joins them, in the line's order.
//
// Persistent, one CTA an SM, 16 warps:
//   warp 0      tensor memory, and the MMAs from one thread: S_t = Q_t K_j^T, O_t +=
//               P_t V_j with P_t read from tensor memory;
//   warps 1-7   read pages, turn codes into fp16 (exact for both types) and store them
//               into a ring of 5 blocks as the MMAs read them;
//   warps 8-15  softmax, 4 warps a tile, a thread a row; a unit's queries at its start.
// Both operands are fp16: a query row is scaled by a power of two to a largest element in
// [2^14, 2^15), which leaves elements down to 2^-28 of it all their bits, and P is rounded
// to fp16 (11 bits) relative to the largest weight p * value_scale of its row, 2^9 above
// it, so neither scales far apart nor a long tail lose bits that count.  l is kept in two
// floats.  O's fp32 sums in tensor memory take 16 keys a step, and a step loses what is
// less than 2^-24 of the sum so far.
//
// Measured (32 query heads on 8 of 128 elements, e4m3, 64-token pages): two pieces of
// 2048 tokens over 24576 2.03 ms, 780 TFLOP/s; one of 256 over 100000 0.55-0.58 ms, 720-760;
// eight of up to 512 over up to 8192 0.32 ms.  Bound by a block's way through a tile, 3.2 us:
// the softmax's 3500 cycles with 16 warps at 0.43 of the issue rate, then P V and the next
// Q K^T, 850 each where 512 are dense; the seven converting warps wait half of their time.
// Measured and not kept: 3 and 5 converting warps (2.74 and 2.16 ms where 7 took 2.10);
// two buffers of scores of 64-key blocks, so that Q K^T runs ahead (2.79 ms: Q is read
// twice as often); 128 scores in a thread's registers at once (they spill, and the local
// memory left beside 230 KB of shared memory is in L2: 3.36 ms); a unit's blocks dealt to
// both tiles where one holds its rows (170 us where 189 for 16 sequences of 8192 tokens, but
// ragged pieces 385 where 325); the lines of a group's codes fetched into L2 ahead (188).
#pragma once

#include "attention_tc.cuh"
#include "common.cuh"
#include "paged_attention.cuh"
#include "prompt_attention.cuh"
#include "ptx.cuh"

namespace nt {
namespace chunk {

using paged::exp2_fast;
using paged::kLn2;
using paged::log2_fast;
using paged::reference;
using prompt::store_shared16;

struct Problem : paged::Attention {
  IndexArray offsets;
  int64_t tokens;
  int per_tile;  // queries of a tile
  uint8_t *workspace;
};

constexpr int BM = 128, BN = 128, TILES = 2, ROWS = TILES * BM;  // rows of a tile, keys of a block
// What a unit's start and end (its queries, its output) count in the line, in key
// blocks: 8 pieces of up to 512 tokens over up to 8192 took 354 us at 2, 335 at 3, 324 at
// 4, 317 at 5; units of few rows, 6 pieces of up to 300 over up to 4000, 75.2, 75.5, 75.9
// and 76.5; 4 of up to 16 over up to 1000 22.6, 23.6, 22.9 and 23.7.  Steps of a piece at
// least: the last took 32 us at 8, 26 at 4, 23 at 2.
constexpr int UNIT_STEPS = 4, LEAST_STEPS = 2;

// ---------------------------------------------------------------- any layout
// A warp a query row.
template <typename T, typename C>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ Problem p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.tokens * p.heads) return;
  // All sequences' offsets are looked at: among ones out of order the search below may miss
  // sequences, whose tokens would be left out without a word.
  for (int64_t i = row * 32 + (threadIdx.x & 31); i < p.batch; i += p.tokens * p.heads * 32)
    if (p.offsets[i] < 0 || p.offsets[i + 1] < p.offsets[i] || p.offsets[i + 1] > p.tokens)
      record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
  const int64_t token = row / p.heads;
  const int h = (int)(row % p.heads);
  const int64_t b = paged::warp_search(p.batch, token, [&](int64_t i) { return p.offsets[i]; });
  const int64_t q0 = p.offsets[b], n = p.offsets[b + 1] - q0;
  if (q0 < 0 || n < 0 || q0 + n > p.tokens) return;
  if (token < q0 || token >= q0 + n) return;
  const T *q = static_cast<const T *>(p.query) + token * p.q_token + h * p.q_head;
  T *out = static_cast<T *>(p.out) + token * p.o_token + h * p.o_head;
  paged::attend_row<T, C>(p, b, h, paged::cached_length(p, b) - n + 1 + (token - q0), q, out,
                          p.lse ? p.lse + token * p.l_token + h * p.l_head : nullptr);
}

// ---------------------------------------------------------------- the line
// sum of floor((a i + b) / m) for i in [0, n), by the steps of Euclid's algorithm
// (a, b >= 0): pairs of whole numbers under a line, counted again with the axes
// exchanged (floor sums and their reciprocity: Graham, Knuth and Patashnik, Concrete
// Mathematics, 3.5).
__device__ __forceinline__ int64_t floor_sum(int64_t n, int32_t m, int32_t a, int64_t b) {
  int64_t sum = 0;
  while (n > 0) {
    sum += (n - 1) * n / 2 * (a / m);
    a %= m;
    sum += n * (b / m);
    b %= m;
    const int64_t top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const int32_t x = m;
    m = a;
    a = x;
  }
  return sum;
}

// Key blocks of a unit whose last query sees `seen` tokens: one at least.
__device__ __forceinline__ int blocks_of(int seen) { return seen <= 0 ? 1 : (seen - 1) / BN + 1; }

// A sequence: `pairs` units a head, of 2 * per_tile queries each.
struct Sequence {
  int32_t q0, n, length, pairs;
  // false where the offsets are out of order or leave the tensors
  __device__ __forceinline__ bool load(const Problem &p, int64_t b) {
    const int64_t o0 = p.offsets[b], count = p.offsets[b + 1] - o0;
    pairs = 0;
    if (o0 < 0 || count < 0 || o0 + count > p.tokens) {
      record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
      return false;
    }
    q0 = (int32_t)o0;
    n = (int32_t)count;
    length = count > 0 ? paged::cached_length(p, b) : 0;
    pairs = (int32_t)((count + 2 * p.per_tile - 1) / (2 * p.per_tile));
    return true;
  }
  // tokens that the queries before `queries` see
  __device__ __forceinline__ int seen(int queries) const { return length - n + queries; }
  __device__ __forceinline__ int blocks(int pair, int i) const { return blocks_of(seen(min((i + 1) * pair, n))); }
  // steps of a head's units before unit i, i < pairs, and of all
  __device__ __forceinline__ int64_t before(int pair, int64_t i) const {
    const int64_t start = (int64_t)length - n;
    int64_t none = start < 0 ? -start / pair : 0;  // units that see nothing: one block
    if (none > i) none = i;
    return i * UNIT_STEPS + none + floor_sum(i - none, BN, pair, start + (none + 1) * pair + BN - 1);
  }
  __device__ __forceinline__ int64_t steps(int pair) const {
    return before(pair, pairs - 1) + blocks(pair, pairs - 1) + UNIT_STEPS;
  }
};

// A CTA's piece of the line, and where its first unit lies.
struct Piece {
  int64_t total, start, end;  // steps of the line; the piece
  int64_t pos;                // of its first unit
  int64_t batch;              // the unit
  int32_t head, pair;
  int32_t pieces;
};

// Where a role stands in its CTA's piece.  All lanes of a warp walk together; the
// sequences come 32 at a time.
struct Walk {
  Sequence mine, seq;  // of lane i: sequence base + i; the current one
  int64_t base, batch, pos;
  int32_t head, pair;
  __device__ __forceinline__ void window(const Problem &p, int64_t from) {
    base = from;
    mine.pairs = 0;
    const int64_t b = from + (threadIdx.x & 31);
    if (b < p.batch) mine.load(p, b);
  }
  __device__ __forceinline__ void take(int lane) {
    seq.q0 = __shfl_sync(0xffffffffu, mine.q0, lane);
    seq.n = __shfl_sync(0xffffffffu, mine.n, lane);
    seq.length = __shfl_sync(0xffffffffu, mine.length, lane);
    seq.pairs = __shfl_sync(0xffffffffu, mine.pairs, lane);
  }
  __device__ __forceinline__ void begin(const Problem &p, const Piece &piece) {
    batch = piece.batch;
    head = piece.head;
    pair = piece.pair;
    pos = piece.pos;
    window(p, batch);
    take(0);
  }
  __device__ __forceinline__ int blocks(const Problem &p) const { return seq.blocks(2 * p.per_tile, pair); }
  // to the next unit; the caller stops at the piece's end, before the line's
  __device__ __forceinline__ void next(const Problem &p) {
    pos += blocks(p) + UNIT_STEPS;
    if (++pair < seq.pairs) return;
    pair = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    ++batch;
    for (;;) {
      const int at = (int)(batch - base);
      const unsigned some = at < 32 ? __ballot_sync(0xffffffffu, mine.pairs > 0) >> at : 0u;
      if (some) {
        batch += __ffs(some) - 1;
        take((int)(batch - base));
        return;
      }
      batch = base + 32;
      if (batch >= p.batch) {
        seq.pairs = 0;
        return;
      }
      window(p, batch);
    }
  }
};

// A unit's share of a piece.
struct Item {
  int32_t q0, queries;   // first packed query, how many (at most two tiles')
  int32_t limit0, keys;  // keys that the first query sees (may be negative); of the sequence
  int32_t batch, head;
  int32_t from, until, blocks;  // the share's key blocks, of the unit's
  int64_t end;                  // of the unit in the line
  __device__ __forceinline__ void take(const Problem &p, const Piece &piece, const Walk &w) {
    const int pair = 2 * p.per_tile, first = w.pair * pair;
    q0 = w.seq.q0 + first;
    queries = min(w.seq.n - first, pair);
    limit0 = w.seq.length - w.seq.n + 1 + first;
    keys = w.seq.length;
    batch = (int32_t)w.batch;
    head = w.head;
    blocks = w.blocks(p);
    end = w.pos + UNIT_STEPS + blocks;
    from = (int32_t)min(max(piece.start - w.pos - UNIT_STEPS, (int64_t)0), (int64_t)blocks);
    until = (int32_t)min(max(piece.end - w.pos - UNIT_STEPS, (int64_t)0), (int64_t)blocks);
  }
  // the share's end for tile t, whose rows may see fewer keys; `from` or less: none
  __device__ __forceinline__ int until_of(int t, int per_tile) const {
    const int last = min(queries, (t + 1) * per_tile) - 1;
    if (last < t * per_tile) return 0;
    return min(until, blocks_of(min(limit0 + last, keys)));
  }
  __device__ __forceinline__ bool whole() const { return from == 0 && until == blocks; }
};
// The items of a piece, all lanes of a warp together.  Where a walk stands lies in
// memory: in registers it would take them from the roles' loops.
__device__ __noinline__ void begin_items(const Problem &p, const Piece &piece, Walk *w) {
  w->seq.pairs = 0;
  if (piece.start < piece.end) w->begin(p, piece);
}
__device__ __noinline__ bool next_item(const Problem &p, const Piece &piece, Walk *state, Item *item) {
  Walk w = *state;
  bool some = false;
  while (!some && w.seq.pairs > 0 && w.pos < piece.end) {
    item->take(p, piece, w);
    w.next(p);
    some = item->from < item->until;
  }
  *state = w;
  return some;
}
// f(item) is false where a wait gave up.
template <typename F>
__device__ __forceinline__ void each_item(const Problem &p, const Piece &piece, F f) {
  Walk walk;
  Item next;
  begin_items(p, piece, &walk);
  while (next_item(p, piece, &walk, &next)) {
    const Item item = next;  // (a copy that no address is taken of stays in registers)
    if (!f(item)) return;
  }
}

// ---------------------------------------------------------------- shared memory, workspace
constexpr int RING = 5, CONVERTERS = 7, SOFTMAX_WARPS = 8, WARPS = 1 + CONVERTERS + SOFTMAX_WARPS, THREADS = WARPS * 32;
constexpr int GROUPS = BN / 16;  // of 16 tokens in a block: a page's or a part of one
constexpr int TMEM_COLS = 512, SCALE_SLOTS = 4, NOTE_SLOTS = 3;

// What a group's 16 keys share.
struct alignas(16) GroupScale {
  float key, add;  // s = raw * key * (the row's factor) + add (-inf: a page outside the pool)
  float unused, log2_value;
};

template <int DP>  // head_dim padded to 64 or 128
struct Layout {
  static constexpr int ATOMS = DP / 64;         // 128-byte swizzle atoms along the head
  static constexpr int Q_BYTES = BM * DP * 2;   // one Q tile
  static constexpr int KV_BYTES = BN * DP * 2;  // one key or value block
  static constexpr int RING_OFF = TILES * Q_BYTES;
  static constexpr int SCALE_OFF = RING_OFF + RING * KV_BYTES;
  static constexpr int BAR_OFF = SCALE_OFF + SCALE_SLOTS * GROUPS * (int)sizeof(GroupScale);
  static constexpr int PIECE_OFF = BAR_OFF + 256;
  static constexpr int SCAN_OFF = PIECE_OFF + 64;                   // int64 [WARPS + 1]
  static constexpr int STAMP_OFF = SCAN_OFF + 8 * (WARPS + 1);      // int [NOTE_SLOTS][CONVERTERS]
  static constexpr int LOW_OFF = STAMP_OFF + 4 * NOTE_SLOTS * CONVERTERS;  // float [SOFTMAX_WARPS * 32]
  static constexpr int SMEM_BYTES = LOW_OFF + 4 * SOFTMAX_WARPS * 32;
  static_assert(sizeof(Piece) <= 64, "the piece's place");
  static_assert(SMEM_BYTES <= 232448, "shared memory of a CTA");
  // a part in the workspace: o [DP / 4][ROWS] float4, then (m, l, mo) [ROWS] float4
  static constexpr int64_t PART = (int64_t)ROWS * (DP + 4) * 4;
};

// A unit that pieces share, as its first CTA leaves it for the join.
struct alignas(16) Shared {
  int32_t last;  // CTA with its last part, or -1: no such unit
  int32_t q0, queries, head;
};
// The workspace: Shared [CTAs], notes int [CTAs][NOTE_SLOTS][CONVERTERS][128], two parts a
// CTA: of the unit that was begun before its piece, and of the one that goes on after it.
__host__ __device__ constexpr int64_t notes_offset(int64_t ctas) { return ctas * (int64_t)sizeof(Shared); }
__host__ __device__ constexpr int64_t parts_offset(int64_t ctas) {
  return notes_offset(ctas) + ctas * NOTE_SLOTS * CONVERTERS * 128 * 4;
}

template <int DP> struct Control {
  using L = Layout<DP>;
  uint8_t *smem;
  uint32_t base, bars;
  __device__ __forceinline__ explicit Control(uint8_t *s) : smem(s), base(ptx::smem_u32(s)), bars(base + L::BAR_OFF) {}
#define NT_BARRIER __device__ __forceinline__ uint32_t
  // of tile t
  NT_BARRIER q_full(int t) const { return bars + 8u * t; }       // Q_t stored
  NT_BARRIER s_full(int t) const { return bars + 16 + 8u * t; }  // S_t of a key block in tensor memory
  NT_BARRIER p_full(int t) const { return bars + 32 + 8u * t; }  // P_t written, O_t rescaled
  NT_BARRIER o_done(int t) const { return bars + 48 + 8u * t; }  // the item's last P_t V done
  NT_BARRIER o_free(int t) const { return bars + 64 + 8u * t; }  // O_t read out
  // of ring slot s
  NT_BARRIER slot_full(int s) const { return bars + 80 + 8u * s; }
  NT_BARRIER slot_empty(int s) const { return bars + 80 + 8u * RING + 8u * s; }
  // of a block's scales; of an item's notes: read
  NT_BARRIER scale_full(int s) const { return bars + 80 + 16u * RING + 8u * s; }
  NT_BARRIER notes_free(int s) const { return bars + 80 + 16u * RING + 8u * SCALE_SLOTS + 8u * s; }
  NT_BARRIER settled() const { return bars + 80 + 16u * RING + 8u * (SCALE_SLOTS + NOTE_SLOTS); }
#undef NT_BARRIER
  static_assert(80 + 16 * RING + 8 * (SCALE_SLOTS + NOTE_SLOTS + 1) <= 240, "barriers");
  __device__ __forceinline__ volatile uint32_t *tmem_base() const {
    return reinterpret_cast<volatile uint32_t *>(smem + L::BAR_OFF + 240);
  }
  __device__ __forceinline__ volatile int *abort_flag() const {
    return reinterpret_cast<volatile int *>(smem + L::BAR_OFF + 244);
  }
  __device__ __forceinline__ GroupScale *scales(int slot) const {
    return reinterpret_cast<GroupScale *>(smem + L::SCALE_OFF) + slot * GROUPS;
  }
  // items with notes: the number of the item that a converter's notes are of
  __device__ __forceinline__ volatile int *stamp(int slot, int converter) const {
    return reinterpret_cast<volatile int *>(smem + L::STAMP_OFF) + slot * CONVERTERS + converter;
  }
  __device__ __forceinline__ int *notes(const Problem &p, int slot, int converter) const {
    return reinterpret_cast<int *>(p.workspace + notes_offset(gridDim.x)) +
           ((blockIdx.x * NOTE_SLOTS + slot) * CONVERTERS + converter) * 128;
  }
};

// ---------------------------------------------------------------- the cut
// All threads: the CTA's piece, into shared memory.
__device__ __noinline__ void find_piece(const Problem &p, Piece *out, int64_t *scan) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pair = 2 * p.per_tile;
  const int64_t per = ((int64_t)p.batch + THREADS - 1) / THREADS;  // sequences of a thread
  const int64_t b0 = threadIdx.x * per, b1 = min(b0 + per, (int64_t)p.batch);
  Sequence s;
  int64_t mine = 0;
  for (int64_t b = b0; b < b1; ++b)
    if (s.load(p, b) && s.pairs > 0) mine += p.kv_heads * s.steps(pair);
  int64_t up = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += x;
  }
  if (lane == 31) scan[warp] = up;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  before += up - mine;
  const int64_t pieces = max(min(total / LEAST_STEPS, (int64_t)gridDim.x), (int64_t)1);
  const int64_t c = blockIdx.x;
  Piece piece{};
  piece.total = total;
  piece.pieces = (int32_t)pieces;
  piece.start = c < pieces ? total * c / pieces : total;
  piece.end = c < pieces ? total * (c + 1) / pieces : total;
  if (threadIdx.x == 0 && piece.start >= piece.end) *out = piece;
  if (piece.start < piece.end && piece.start >= before && piece.start < before + mine) {
    for (int64_t b = b0; b < b1; ++b) {
      if (!s.load(p, b) || s.pairs == 0) continue;
      const int64_t steps = s.steps(pair);  // of a head
      if (piece.start < before + p.kv_heads * steps) {
        const int64_t into = piece.start - before;
        piece.batch = b;
        piece.head = (int32_t)(into / steps);
        piece.pos = before + piece.head * steps;
        *out = piece;
        break;
      }
      before += p.kv_heads * steps;
    }
  }
  __syncthreads();
  if (warp == 0 && piece.start < piece.end) {
    s.load(p, out->batch);
    const int64_t into = piece.start - out->pos;
    const int64_t i = paged::warp_search(s.pairs, into, [&](int64_t k) { return s.before(pair, k); });
    if (lane == 0) {
      out->pair = (int32_t)i;
      out->pos += s.before(pair, i);
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------- pages to operands
// Four E4M3 codes: the top bit of each byte that is NaN, among others; the codes with 0
// for NaN.
__device__ __forceinline__ uint32_t nan_bits(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }
__device__ __forceinline__ uint32_t without_nan(uint32_t w) { return w & ~(((nan_bits(w) & 0x80808080u) >> 7) * 0xffu); }

// Takes the NaN codes out of a lane's word of a token's value, and notes the first key
// with one for each element of the head.  A full warp; false where a wait gave up.
template <int DP, int LOADS>
__device__ __noinline__ bool take_out(const Control<DP> &c, const Problem &p, uint4 (&x)[LOADS], int item, int key0, int key_step,
                                      int element0) {
  const int lane = threadIdx.x & 31, me = (threadIdx.x >> 5) - 1, slot = item % NOTE_SLOTS;
  int *notes = c.notes(p, slot, me);
  if (*c.stamp(slot, me) != item) {
    if (!ptx::mbar_wait_warp(c.notes_free(slot), ((uint32_t)(item / NOTE_SLOTS) & 1u) ^ 1u, c.abort_flag())) return false;
    for (int d = lane; d < 128; d += 32) notes[d] = INT32_MAX;
    __threadfence();
    __syncwarp();
    if (lane == 0) *c.stamp(slot, me) = item;
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    uint32_t *w = &x[i].x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll 1
      for (int e = 0; e < 4; ++e)
        if ((w[k] >> 8 * e & 0x7fu) == 0x7fu) atomicMin(notes + element0 + k * 4 + e, key0 + i * key_step);
      w[k] = without_nan(w[k]);
    }
  }
  __threadfence();
  return true;
}

// A group of 16 tokens, of which `count` are the sequence's.
struct Group {
  int64_t page;        // as the block table has it (to look at it is to wait for it), then -1: outside the pool
  int32_t at, count;   // the group of the sequence
  int32_t ring, item;  // its keys' place in the ring
  int32_t head;
};

// The groups of the CTA's items are dealt to the warps in turn.  A warp stores a group's
// keys, asks for those of its next, stores its values, asks for the next's values: so two
// loads of 2 KB are always on their way, 28 KB an SM.  Pages' numbers come two groups ahead.
template <typename C, int DP>
__device__ __forceinline__ void convert(const Control<DP> &c, const Problem &p, const Piece &piece) {
  using L = Layout<DP>;
  constexpr int WORDS = DP / 16, KEYS = 32 / WORDS, LOADS = 16 / KEYS;  // 16-byte words of a token; tokens a load of the warp
  const int lane = threadIdx.x & 31, me = (threadIdx.x >> 5) - 1;
  // A quarter warp takes the four words of one 64-element atom of two tokens: its stores
  // of their first halves, and of the second, then meet every bank once.
  const int word = DP == 128 ? (lane & 3) | (lane >> 1 & 4) : lane & 3;
  const int sub = DP == 128 ? (lane >> 2 & 1) | (lane >> 3 & 2) : lane >> 2;
  const bool in_head = word * 16 < p.head_dim;
  const uint32_t base = c.base + L::RING_OFF + (word / 4) * (BN * 128) + sub * 128;
  uint32_t place[2][2];  // of the halves of a word, for a load's even and odd turns
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) place[i][h] = base + i * KEYS * 128 + (((word % 4) * 2 + h) ^ ((i * KEYS + sub) & 7)) * 16;

  auto store = [&](const uint4 (&x)[LOADS], int ring, int at) {
    const uint32_t to = (ring % RING) * L::KV_BYTES + (at % GROUPS) * (16 * 128);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      uint4 lo, hi;
      paged::to_halves<C>(x[i].x, lo.x, lo.y);
      paged::to_halves<C>(x[i].y, lo.z, lo.w);
      paged::to_halves<C>(x[i].z, hi.x, hi.y);
      paged::to_halves<C>(x[i].w, hi.z, hi.w);
      store_shared16(place[i % 2][0] + to + (i / 2) * (2 * KEYS * 128), lo);
      store_shared16(place[i % 2][1] + to + (i / 2) * (2 * KEYS * 128), hi);
    }
    ptx::fence_proxy_async_smem();  // the MMAs read what was written here
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(c.slot_full(ring % RING));
  };
  auto wait_empty = [&](int ring) {
    return ptx::mbar_wait_warp(c.slot_empty(ring % RING), ((uint32_t)(ring / RING) & 1u) ^ 1u, c.abort_flag());
  };
  auto load = [&](uint4 (&x)[LOADS], const Group &g, const uint8_t *codes, int64_t page, int64_t head, int64_t token) {
    const int in_page = g.at - (int)((uint64_t)(uint32_t)g.at * p.page_reciprocal >> 36) * p.page_groups;
    const uint8_t *from = codes + g.page * page + g.head * head + (in_page * 16 + sub) * token + word * 16;
    const int count = g.page < 0 || !in_head ? 0 : g.count - sub;
    if (__all_sync(0xffffffffu, count > 16 - KEYS)) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) x[i] = __ldg(reinterpret_cast<const uint4 *>(from + i * KEYS * token));
    } else {
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        x[i] = i * KEYS < count ? __ldg(reinterpret_cast<const uint4 *>(from + i * KEYS * token)) : make_uint4(0, 0, 0, 0);
    }
  };

  Walk walk;
  Item next_of_walk;
  begin_items(p, piece, &walk);
  bool more = next_item(p, piece, &walk, &next_of_walk);
  Item e = next_of_walk;  // (in registers: no address is taken of it)
  int ring = 0, item = 0, x = me;  // the item's K_0; the next group
  auto ask = [&](Group &g) -> bool {
    while (more && x >= (e.until - e.from) * GROUPS) {
      x -= (e.until - e.from) * GROUPS;
      ring += 2 * (e.until - e.from);
      ++item;
      more = next_item(p, piece, &walk, &next_of_walk);
      e = next_of_walk;
    }
    if (!more) return false;
    g.ring = ring + x / GROUPS * 2;
    g.at = e.from * GROUPS + x;
    g.item = item;
    g.head = e.head;
    g.count = min(max(e.keys - g.at * 16, 0), 16);
    g.page = -1;
    if (g.count > 0) {
      const int64_t column = (int64_t)((uint64_t)(uint32_t)g.at * p.page_reciprocal >> 36);
      const int64_t entry = e.batch * p.table_row_stride + column * p.block_table.stride;
      if (p.block_table.wide) g.page = static_cast<const int64_t *>(p.block_table.data)[entry];
      else g.page = static_cast<const int32_t *>(p.block_table.data)[entry];
    }
    x += CONVERTERS;
    return true;
  };
  uint4 keys[LOADS], values[LOADS];
  float key_scale = 0.f, value_scale = 0.f;
  Group now, next;
  bool has = ask(now), has_next = has && ask(next);
  auto load_keys = [&](Group &g) {
    if (g.page < 0 || g.page >= p.pages) {
      if (g.count > 0) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
      g.page = -1;
    }
    load(keys, g, p.key, p.k_page, p.k_head, p.k_token);
    if (g.page >= 0) {
      key_scale = p.key_scale[g.page * p.ks_page + g.head * p.ks_head];
      value_scale = p.value_scale[g.page * p.vs_page + g.head * p.vs_head];
    }
  };
  if (has) {
    load_keys(now);
    load(values, now, p.value, p.v_page, p.v_head, p.v_token);
  }
#pragma unroll 1
  while (has) {
    const Group g = now;
    if (!wait_empty(g.ring)) return;
    const float scale = value_scale;
    if (lane == 0) {
      const int block = g.ring / 2 % SCALE_SLOTS;
      GroupScale s{p.scale * key_scale, 0.f, 0.f, log2_fast(scale)};
      if (g.page < 0) s = GroupScale{0.f, -INFINITY, 0.f, -INFINITY};
      c.scales(block)[g.at % GROUPS] = s;
      ptx::mbar_arrive(c.scale_full(block));
    }
    store(keys, g.ring, g.at);
    has = has_next;
    now = next;
    if (has) {
      load_keys(now);
      has_next = ask(next);
    }
    if (std::is_same<C, __nv_fp8_e4m3>::value) {
      uint32_t nan = 0;
#pragma unroll
      for (int i = 0; i < LOADS; ++i)
        nan |= nan_bits(values[i].x) | nan_bits(values[i].y) | nan_bits(values[i].z) | nan_bits(values[i].w);
      if (__any_sync(0xffffffffu, (nan & 0x80808080u) != 0)) {
        uint4 box[LOADS];
#pragma unroll
        for (int i = 0; i < LOADS; ++i) box[i] = values[i];
        if (!take_out<DP, LOADS>(c, p, box, g.item, g.at * 16 + sub, KEYS, word * 16)) return;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) values[i] = box[i];
      }
    }
    if (scale == 0.f)  // they stand for 0, however small their weights are kept
#pragma unroll
      for (int i = 0; i < LOADS; ++i) values[i] = make_uint4(0, 0, 0, 0);
    if (!wait_empty(g.ring + 1)) return;
    store(values, g.ring + 1, g.at);
    if (has) load(values, now, p.value, p.v_page, p.v_head, p.v_token);
  }
}

// ---------------------------------------------------------------- MMA issuer
// A full warp; lane 0 issues.  K, V and Q stand in shared memory as 128-byte-swizzled
// tiles of 64 elements.
struct Standing {
  int ring;            // place of the item's K_0
  int blocks[TILES];   // key blocks of tile t so far
  int used[TILES];     // items that had tile t
};

template <int DP>
__device__ __forceinline__ void issue(const Control<DP> &c, const Problem &p, const Piece &piece, uint32_t tmem_base,
                                      Shared &open) {
  using L = Layout<DP>;
  constexpr uint32_t fmt = tc::umma_format<__half>();
  constexpr uint32_t idesc_qk = ptx::f16_idesc(fmt, 0, 0, BM, BN);  // B = keys, K-major
  constexpr uint32_t idesc_pv = ptx::f16_idesc(fmt, 0, 1, BM, DP);  // B = values, MN-major
  const bool issues = (threadIdx.x & 31) == 0;
  auto tmem_s = [&](int t) { return tmem_base + (uint32_t)(t * BN); };
  auto tmem_o = [&](int t) { return tmem_base + (uint32_t)(TILES * BN + t * 128); };
  auto slot_addr = [&](int r) { return c.base + L::RING_OFF + (r % RING) * L::KV_BYTES; };
  auto wait = [&](uint32_t bar, uint32_t parity) { return ptx::mbar_wait_warp(bar, parity, c.abort_flag()); };
  auto wait_slot = [&](int r) { return wait(c.slot_full(r % RING), (uint32_t)(r / RING) & 1u); };
  auto commit = [&](uint32_t bar) {
    if (issues) ptx::mma_commit(bar);
  };
  auto issue_qk = [&](int t, int r) {
    if (!issues) return;
    const uint32_t kb = slot_addr(r);
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const uint32_t qoff = (kk / 4) * (BM * 128) + (kk % 4) * 32, koff = (kk / 4) * (BN * 128) + (kk % 4) * 32;
      ptx::mma_f16_ss(tmem_s(t), ptx::sw128_desc(c.base + t * L::Q_BYTES + qoff, 16, 1024),
                      ptx::sw128_desc(kb + koff, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
    }
    ptx::mma_commit(c.s_full(t));
  };
  auto issue_pv = [&](int t, int r, bool first) {
    if (!issues) return;
    const uint32_t vb = slot_addr(r);
#pragma unroll
    for (int kk = 0; kk < BN / 16; ++kk)
      ptx::mma_f16_ts(tmem_o(t), tmem_s(t) + (uint32_t)(kk * 8), ptx::sw128_desc(vb + kk * 16 * 128, BN * 128, 1024),
                      idesc_pv, (!first || kk > 0) ? 1u : 0u);
  };
  Standing at{};
  each_item(p, piece, [&](const Item &e) {
    if (e.from == 0 && e.until < e.blocks)
      open = Shared{(int32_t)((e.end * piece.pieces - 1) / piece.total), e.q0, e.queries, e.head};
    const int count = e.until - e.from;
    const int n[TILES] = {max(e.until_of(0, p.per_tile) - e.from, 0), max(e.until_of(1, p.per_tile) - e.from, 0)};
    if (!wait_slot(at.ring)) return false;  // K_0
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (n[t] == 0) continue;
      if (!wait(c.q_full(t), (uint32_t)at.used[t] & 1u)) return false;
      ptx::tc_fence_after();
      issue_qk(t, at.ring);
    }
    commit(c.slot_empty(at.ring % RING));
    for (int j = 0; j < count; ++j) {
      const int rv = at.ring + 2 * j + 1, rk = rv + 1;
      if (!wait_slot(rv)) return false;
      const bool next_keys = j + 1 < count;
      bool waited = false;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        if (j >= n[t]) continue;
        // P_t written also means that S_t was read: Q K^T may overwrite it
        if (!wait(c.p_full(t), (uint32_t)(at.blocks[t] + j) & 1u)) return false;
        if (j == 0 && at.used[t] > 0 && !wait(c.o_free(t), (uint32_t)(at.used[t] - 1) & 1u)) return false;
        ptx::tc_fence_after();
        issue_pv(t, rv, j == 0);
        if (j == n[t] - 1) commit(c.o_done(t));
        if (j + 1 < n[t]) {
          if (!waited) {
            if (!wait_slot(rk)) return false;
            waited = true;
            ptx::tc_fence_after();
          }
          issue_qk(t, rk);
        }
      }
      commit(c.slot_empty(rv % RING));
      if (next_keys) {
        // (a block that no tile needs was loaded all the same)
        if (!waited && !wait_slot(rk)) return false;
        commit(c.slot_empty(rk % RING));
      }
    }
    at.ring += 2 * count;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      at.blocks[t] += n[t];
      at.used[t] += n[t] > 0;
    }
    return true;
  });
}

// ---------------------------------------------------------------- queries, softmax, output
// A row's references move only when a block passes them by 2^kLead, so that O is rescaled
// rarely, and P is kept 2^kRise above: its largest, 2^15, stays in fp16's range.
constexpr float kLead = 6.f, kRise = 9.f, kLeastShift = -60.f;
constexpr float kLeastKey = 1.1754943508222875e-38f;  // in place of a key scale of 0: -inf times it is -inf

// A row of Q into shared memory, scaled by 2^e with its largest finite element then in
// [2^14, 2^15); returns 2^-e.  `query` null: zeros.
template <int DP>
__device__ __forceinline__ float store_query(const Control<DP> &c, const Problem &p, int t, int row, const uint16_t *query) {
  using L = Layout<DP>;
  uint32_t w[DP / 2];  // two elements each
  if (p.q_vector) {
#pragma unroll
    for (int x = 0; x < DP / 8; ++x) {
      const uint4 v = query && x * 8 < p.head_dim ? __ldg(reinterpret_cast<const uint4 *>(query) + x) : make_uint4(0, 0, 0, 0);
      w[4 * x] = v.x; w[4 * x + 1] = v.y; w[4 * x + 2] = v.z; w[4 * x + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int x = 0; x < DP / 2; ++x)
      w[x] = query && 2 * x < p.head_dim ? query[2 * x * p.q_dim] | (uint32_t)query[(2 * x + 1) * p.q_dim] << 16 : 0u;
  }
  auto values = [&](uint32_t v) {
    return p.bf16 ? make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u))
                  : __half22float2(*reinterpret_cast<const __half2 *>(&v));
  };
  float top = 0.f;
#pragma unroll
  for (int x = 0; x < DP / 2; ++x) {
    const float2 v = values(w[x]);
    top = fmaxf(top, fmaxf(paged::finite_magnitude(v.x), paged::finite_magnitude(v.y)));
  }
  // 2^(14 - exponent); rows of less than 2^-112 as those of 2^-112
  const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);
  const float factor = __uint_as_float((uint32_t)(paged::Q_TOP - e + 127) << 23);
  const uint32_t to = c.base + t * L::Q_BYTES + row * 128;
#pragma unroll
  for (int x = 0; x < DP / 8; ++x) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = values(w[4 * x + i]);
      h[i] = paged::half2_bits(v.x * factor, v.y * factor);
    }
    store_shared16(to + (x / 8) * (BM * 128) + (((x % 8) ^ (row & 7)) * 16), make_uint4(h[0], h[1], h[2], h[3]));
  }
  return __uint_as_float((uint32_t)(e - paged::Q_TOP + 127) << 23);
}

template <int N> __device__ __forceinline__ void store_output(const Problem &p, int64_t token, int head, int d0, const float (&x)[N]) {
  uint16_t *out = static_cast<uint16_t *>(p.out) + token * p.o_token + (int64_t)head * p.o_head + d0 * p.o_dim;
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    w[i] = p.bf16 ? tc::attn::pack2<__nv_bfloat16>(x[2 * i], x[2 * i + 1]) : tc::attn::pack2<__half>(x[2 * i], x[2 * i + 1]);
  if (p.o_dim == 1 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i)
      reinterpret_cast<uint4 *>(out)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i * p.o_dim] = (uint16_t)(w[i / 2] >> 16 * (i & 1));
  }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// A warp is done with an item's notes; false where a wait gave up.  A tile that has nothing
// in its items would run through them all: a warp arrives for a slot's use only after all
// arrived for the one before, so that a phase is one use by every warp, and what waits for
// it by parity (here and in take_out) is never two phases off.
__device__ __noinline__ bool leave_notes(uint32_t bar, int item, volatile int *abort_flag) {
  if (!ptx::mbar_wait_warp(bar, ((uint32_t)(item / NOTE_SLOTS) & 1u) ^ 1u, abort_flag)) return false;
  __syncwarp();
  if ((threadIdx.x & 31) == 0) ptx::mbar_arrive(bar);
  return true;
}

template <int DP>
__device__ __forceinline__ void attend(const Control<DP> &c, const Problem &p, const Piece &piece, uint32_t tmem_base) {
  using L = Layout<DP>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = (warp - 1 - CONVERTERS) / 4, quarter = warp & 3;
  const int row = quarter * 32 + lane;  // row of the tile = lane of tensor memory
  const int row_query = row / p.group + t * p.per_tile, row_head = row % p.group;
  const bool has_row = row / p.group < p.per_tile;
  const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
  const uint32_t tmem_s = tmem_base + (uint32_t)(t * BN) + lane_base;
  const uint32_t tmem_o = tmem_base + (uint32_t)(TILES * BN + t * 128) + lane_base;
  // what the row's sum of weights has beside l; a register for it would spill others
  volatile float *l_low = reinterpret_cast<volatile float *>(c.smem + L::LOW_OFF) + (warp - 1 - CONVERTERS) * 32 + lane;
  auto arrive_warp = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar);
  };
  int s_turn = 0, o_turn = 0, block0 = 0, items = 0;  // blocks and items of this tile; the item's first block, the item
  each_item(p, piece, [&](const Item &e) {
    const int until = e.until_of(t, p.per_tile), item = items++, first_block = block0;
    block0 += e.until - e.from;
    const bool mine = has_row && row_query < e.queries;
    const int64_t token = e.q0 + row_query;
    const int head = e.head * p.group + row_head;
    float *part = nullptr;
    if (!e.whole())
      part = reinterpret_cast<float *>(p.workspace + parts_offset(gridDim.x) +
                                       (2 * (int64_t)blockIdx.x + (e.from > 0 ? 0 : 1)) * L::PART);
    float4 *stats = reinterpret_cast<float4 *>(part) + ROWS * (DP / 4) + t * BM + row;
    if (until <= e.from) {  // nothing to see in this share
      if (part && mine) *stats = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
      return leave_notes(c.notes_free(item % NOTE_SLOTS), item, c.abort_flag());
    }
    const float factor = store_query<DP>(
        c, p, t, row,
        mine ? static_cast<const uint16_t *>(p.query) + token * p.q_token + (int64_t)head * p.q_head : nullptr);
    ptx::fence_proxy_async_smem();
    arrive_warp(c.q_full(t));
    const int limit = min(e.limit0 + row_query, e.keys);             // keys that the row sees
    const int sure = min(e.limit0 + t * p.per_tile, e.keys);         // that all rows see

    float m = -INFINITY, mo = -INFINITY, l = 0.f;
    *l_low = 0.f;
    for (int j = e.from; j < until; ++j) {
      const int block = first_block + j - e.from, slot = block % SCALE_SLOTS;
      // (for a tile that is items ahead the scales' phase may be two back, which looks the
      // same: they are there with the scores, as a group's are written before its keys)
      if (!ptx::mbar_wait_warp(c.scale_full(slot), (uint32_t)(block / SCALE_SLOTS) & 1u, c.abort_flag())) return false;
      if (!ptx::mbar_wait_warp(c.s_full(t), (uint32_t)s_turn & 1u, c.abort_flag())) return false;
      ++s_turn;
      ptx::tc_fence_after();
      const int seen = limit - j * BN;
      bool move_o;
      float alpha_o, near = 0.f;  // near: the block's part of the sum of weights
      auto take_block = [&](auto with_mask) {
      constexpr bool MASKED = decltype(with_mask)::value;
      // 32 scores at a time, read twice: 128 would fill the registers.  The next are on
      // their way while these are worked on.
      auto ask_scores = [&](int quarter, uint32_t (&s)[32]) { ptx::tmem_ld_32x32b_x32(tmem_s + (uint32_t)(quarter * 32), s); };
      auto mask_scores = [&](int quarter, float (&s)[32]) {
        if constexpr (!MASKED) return;
        const int in_quarter = seen - quarter * 32;
#pragma unroll
        for (int x = 0; x < 32; ++x) s[x] = x < in_quarter ? s[x] : -INFINITY;
      };
      // f(quarter, its scores), the first half's and then the second's
      auto each_quarter = [&](auto f) {
        uint32_t a[32], b[32];
        ask_scores(0, a);
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          ptx::tmem_ld_wait();
          ask_scores(2 * half + 1, b);
          f(2 * half, *reinterpret_cast<float(*)[32]>(&a));
          ptx::tmem_ld_wait();
          if (half == 0) ask_scores(2, a);
          f(2 * half + 1, *reinterpret_cast<float(*)[32]>(&b));
        }
      };
      const GroupScale *scales = c.scales(slot);
      // (a group that the row does not see takes no part, whatever its scales)
      auto unseen = [&](int k) { return MASKED && k * 16 >= seen; };
      auto key_factor = [&](float key, int k) {
        const float f = key * factor;
        return MASKED && (f == 0.f || unseen(k)) ? kLeastKey : f;
      };
      float top_s = -INFINITY, top_w = -INFINITY;
      each_quarter([&](int quarter, float (&s)[32]) {
        mask_scores(quarter, s);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int group = quarter * 2 + k;
          const float4 g = *reinterpret_cast<const float4 *>(scales + group);
          const float *x = s + k * 16;
          const float a = max3(max3(x[0], x[1], x[2]), x[3], x[4]), b = max3(max3(x[5], x[6], x[7]), x[8], x[9]);
          const float d = max3(max3(x[10], x[11], x[12]), x[13], x[14]);
          const float high = fmaf(fmaxf(max3(a, b, d), x[15]), key_factor(g.x, group), g.y);
          top_s = fmaxf(top_s, high);
          top_w = fmaxf(top_w, high + g.w);
        }
      });
      const bool move = top_s > m + kLead;
      move_o = top_w > mo + kLead;
      alpha_o = move_o ? exp2_fast(mo - top_w) : 1.f;
      if (move) {
        const float f = exp2_fast(m - top_s);
        l *= f;
        *l_low *= f;
        m = top_s;
      }
      if (move_o) mo = top_w;
      // P = 2^(s - m + shift) with the group's shift = log2 value_scale + m - mo + kRise, and
      // near takes a group's sum of them times 2^-shift.  Where a group's values are so small
      // that its P would leave fp32, P is kept at 2^kLeastShift: too large, but nothing beside the others.
      const float ref = reference(m), rise = ref - reference(mo) + kRise;
      each_quarter([&](int quarter, float (&s)[32]) {
        mask_scores(quarter, s);
        uint32_t packed[16];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int group = quarter * 2 + k;
          const float4 g = *reinterpret_cast<const float4 *>(scales + group);
          const float by = key_factor(g.x, group);
          float shift = g.w + rise;
          shift = shift < kLeastShift || unseen(group) ? kLeastShift : shift;  // (a NaN scale stays)
          const float add = g.y - ref + shift;
          float sum[4] = {};
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int at = k * 16 + 2 * x;
            const float p0 = exp2_fast(fmaf(s[at], by, add)), p1 = exp2_fast(fmaf(s[at + 1], by, add));
            sum[(2 * x) & 3] += p0;
            sum[(2 * x + 1) & 3] += p1;
            packed[k * 8 + x] = paged::half2_bits(p0, p1);
          }
          near = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), exp2_fast(-shift), near);
        }
        // (P's 16 columns lie among scores that were read before)
        ptx::tmem_st_32x32b_x16(tmem_s + (uint32_t)(quarter * 16), packed);
      });
      };
      if (sure - j * BN < BN) take_block(std::true_type{});
      else take_block(std::false_type{});
      if (j > e.from && __any_sync(0xffffffffu, move_o)) {
        // O_t holds P(j-1) V(j-1): the commit of S_t(j) covers it
#pragma unroll 1
        for (int x = 0; x < DP; x += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32b_x32(tmem_o + (uint32_t)x, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha_o);
          ptx::tmem_st_32x32b_x32(tmem_o + (uint32_t)x, o);
        }
      }
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      arrive_warp(c.p_full(t));
      // l + near, and what fp32 cuts off it: beside a weight of 1, 2^18 weights of 2^-28 were
      // lost 16 at a time (1e-3 of the lse).  (While the MMAs run it takes no time: 2024 us
      // for two pieces of 2048 tokens over 24576, 2018 with one sum.)
      const float both = __fadd_rn(l, near), added = __fsub_rn(both, l);
      *l_low += __fadd_rn(__fsub_rn(l, __fsub_rn(both, added)), __fsub_rn(near, added));
      l = both;
    }
    if (!ptx::mbar_wait_warp(c.o_done(t), (uint32_t)o_turn & 1u, c.abort_flag())) return false;
    ++o_turn;
    ptx::tc_fence_after();
    l += *l_low;
    // (mo: -inf where all values stand for 0)
    const float f = l == 0.f ? 0.f : exp2_fast(reference(mo) - reference(m) - kRise) / l;
#pragma unroll 1
    for (int x = 0; x < DP; x += 32) {
      uint32_t o[32];
      ptx::tmem_ld_32x32b_x32(tmem_o + (uint32_t)x, o);
      ptx::tmem_ld_wait();
      // values' NaN, to the rows that see them
#pragma unroll 1
      for (int w = 0; w < CONVERTERS; ++w) {
        if (*c.stamp(item % NOTE_SLOTS, w) != item) continue;
        const int *notes = c.notes(p, item % NOTE_SLOTS, w) + x;
#pragma unroll
        for (int d = 0; d < 32; ++d)
          if (__ldcg(notes + d) < limit) o[d] = 0x7fc00000u;
      }
      if (mine && !part) {
#pragma unroll
        for (int y = 0; y < 32; y += 16) {
          float v[16];
#pragma unroll
          for (int z = 0; z < 16; ++z) v[z] = __uint_as_float(o[y + z]) * f;
          if (x + y < p.head_dim) store_output<16>(p, token, head, x + y, v);
        }
      } else if (part && mine) {
        float4 *out = reinterpret_cast<float4 *>(part) + (x / 4) * ROWS + t * BM + row;
#pragma unroll
        for (int y = 0; y < 8; ++y)
          out[y * ROWS] = make_float4(__uint_as_float(o[4 * y]), __uint_as_float(o[4 * y + 1]), __uint_as_float(o[4 * y + 2]),
                                      __uint_as_float(o[4 * y + 3]));
      }
    }
    ptx::tc_fence_before();
    arrive_warp(c.o_free(t));
    if (mine && part) *stats = make_float4(m, l, mo, 0.f);
    if (mine && !part && p.lse)
      p.lse[token * p.l_token + (int64_t)head * p.l_head] = l == 0.f ? -INFINITY : (m + log2_fast(l)) * kLn2;
    return leave_notes(c.notes_free(item % NOTE_SLOTS), item, c.abort_flag());
  });
}

template <typename C, int DP>
__global__ void __launch_bounds__(THREADS, 1) attention_kernel(const __grid_constant__ Problem p) {
  using L = Layout<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const Control<DP> c(smem);
  Shared *shared = reinterpret_cast<Shared *>(p.workspace) + blockIdx.x;
  if ((c.base & 1023u) != 0) {  // the swizzle needs it; there is no room to align by hand
    record_error(NT_B200_ERR_INVALID_ARGUMENT);
    wait_prior_grid();
    if (threadIdx.x == 0) shared->last = -1;
    return;
  }
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int t = 0; t < TILES; ++t) {
      ptx::mbar_init(c.q_full(t), 4);  // a warp's lanes arrive as one
      ptx::mbar_init(c.s_full(t), 1);
      ptx::mbar_init(c.p_full(t), 4);
      ptx::mbar_init(c.o_done(t), 1);
      ptx::mbar_init(c.o_free(t), 4);
    }
    for (int s = 0; s < RING; ++s) {
      ptx::mbar_init(c.slot_full(s), GROUPS);
      ptx::mbar_init(c.slot_empty(s), 1);
    }
    for (int s = 0; s < SCALE_SLOTS; ++s) ptx::mbar_init(c.scale_full(s), GROUPS);
    for (int s = 0; s < NOTE_SLOTS; ++s) {
      ptx::mbar_init(c.notes_free(s), SOFTMAX_WARPS);
      for (int w = 0; w < CONVERTERS; ++w) *c.stamp(s, w) = -1;
    }
    ptx::mbar_init(c.settled(), 1);
    *c.abort_flag() = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 0) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t *>(c.tmem_base())), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  wait_prior_grid();
  ptx::tc_fence_before();
  find_piece(p, reinterpret_cast<Piece *>(smem + L::PIECE_OFF), reinterpret_cast<int64_t *>(smem + L::SCAN_OFF));
  ptx::tc_fence_after();
  const Piece &piece = *reinterpret_cast<const Piece *>(smem + L::PIECE_OFF);
  const uint32_t tmem_base = *c.tmem_base();
  if (warp == 0) {
    Shared open{-1, 0, 0, 0};  // the unit that goes on in the next piece, for the join
    issue<DP>(c, p, piece, tmem_base, open);
    if ((threadIdx.x & 31) == 0) *shared = open;
  } else if (warp <= CONVERTERS) {
    convert<C, DP>(c, p, piece);
  } else {
    attend<DP>(c, p, piece, tmem_base);
  }
  allow_dependent_launch();
  ptx::tc_fence_before();
  __syncthreads();
  if (*c.abort_flag()) {
    // after a wait gave up: the MMAs in flight, so that shared and tensor memory are at rest
    if (threadIdx.x == 0) {
      volatile int over = 0;
      ptx::mma_commit(c.settled());
      ptx::mbar_wait(c.settled(), 0, &over, 1000000000ull);
    }
    __syncthreads();
  }
  if (warp == 0) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- join
// Block (a, y): 16 elements of the rows of the unit that CTA a left open; a thread a row.
template <int DP>
__global__ void __launch_bounds__(ROWS) join_kernel(const __grid_constant__ Problem p, int ctas) {
  using L = Layout<DP>;
  wait_prior_grid();
  allow_dependent_launch();
  const Shared s = reinterpret_cast<const Shared *>(p.workspace)[blockIdx.x];
  if (s.last < 0) return;
  const int row = threadIdx.x % BM, t = threadIdx.x / BM;
  const int query = t * p.per_tile + row / p.group;
  if (row / p.group >= p.per_tile || query >= s.queries) return;
  // the parts: this CTA's second, then the first of those after it
  const auto part = [&](int i) {
    return reinterpret_cast<const float4 *>(p.workspace + parts_offset(ctas) +
                                            (i == 0 ? 2 * (int64_t)blockIdx.x + 1 : 2 * ((int64_t)blockIdx.x + i)) * L::PART);
  };
  const int parts = s.last - (int)blockIdx.x + 1;
  constexpr int STATS = ROWS * (DP / 4);
  float top = -INFINITY, top_o = -INFINITY;
  for (int i = 0; i < parts; ++i) {
    const float4 st = part(i)[STATS + threadIdx.x];
    top = fmaxf(top, st.x);
    top_o = fmaxf(top_o, st.z);
  }
  float l = 0.f, o[16] = {};
  for (int i = 0; i < parts; ++i) {
    const float4 *from = part(i);
    const float4 st = from[STATS + threadIdx.x];
    l += st.y * exp2_fast(st.x - reference(top));
    if (st.z == -INFINITY && st.y == 0.f) continue;  // a tile without keys in this part: nothing was written
    const float f = exp2_fast(st.z - reference(top_o));
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float4 v = from[(blockIdx.y * 4 + x) * ROWS + threadIdx.x];
      o[4 * x] = fmaf(v.x, f, o[4 * x]);
      o[4 * x + 1] = fmaf(v.y, f, o[4 * x + 1]);
      o[4 * x + 2] = fmaf(v.z, f, o[4 * x + 2]);
      o[4 * x + 3] = fmaf(v.w, f, o[4 * x + 3]);
    }
  }
  const int64_t token = s.q0 + query;
  const int head = s.head * p.group + row % p.group;
  const float f = l == 0.f ? 0.f : exp2_fast(reference(top_o) - reference(top) - kRise) / l;
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] *= f;
  store_output<16>(p, token, head, blockIdx.y * 16, o);
  if (p.lse && blockIdx.y == 0)
    p.lse[token * p.l_token + (int64_t)head * p.l_head] = l == 0.f ? -INFINITY : (top + log2_fast(l)) * kLn2;
}

template <typename C, int DP> int launch_tiles(const Problem &p, cudaStream_t stream) {
  using L = Layout<DP>;
  cudaError_t e = smem_optin<attention_kernel<C, DP>>(L::SMEM_BYTES);
  if (e != cudaSuccess) return (int)e;
  const int ctas = sm_count();
  const int rc = launch_overlapped(attention_kernel<C, DP>, dim3(ctas), dim3(THREADS), L::SMEM_BYTES, stream, p);
  if (rc != 0) return rc;
  return launch_overlapped(join_kernel<DP>, dim3(ctas, (unsigned)(p.head_dim / 16)), dim3(ROWS), 0, stream, p, ctas);
}

template <typename T, typename C> int launch(const Problem &p, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (p.head_dim <= 128 && p.group <= BM && p.scale > 0.f && p.tokens <= (1 << 30)) {
      if (p.head_dim <= 64) return launch_tiles<C, 64>(p, stream);
      return launch_tiles<C, 128>(p, stream);
    }
  }
  const int64_t blocks = (p.tokens * p.heads + 3) / 4;
  if (blocks > (1LL << 31) - 1) return NT_B200_ERR_INVALID_ARGUMENT;
  rows_kernel<T, C><<<(unsigned)blocks, 128, 0, stream>>>(p);
  return launch_status();
}

}  // namespace chunk
}  // namespace nt

extern "C" int64_t nt_b200_chunk_attention_workspace_size(void) {
  using namespace nt::chunk;
  const int64_t ctas = nt::sm_count();
  return parts_offset(ctas) + 2 * ctas * Layout<128>::PART;
}

extern "C" int nt_b200_chunk_attention(const NtB200ChunkAttentionArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->batch < 0 || a->tokens < 0 || a->heads < 0 || a->table_columns < 0) return NT_B200_ERR_INVALID_ARGUMENT;
  if (!is_float_dtype((int)a->dtype) || !is_index_dtype(a->index_dtype)) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->batch == 0 || a->tokens == 0 || a->heads == 0) return 0;
  const NtB200PagedCache &c = a->cache;
  const int rc = paged::check_cache(c);
  if (rc != 0) return rc;
  if (c.kv_heads == 0 || a->heads % c.kv_heads != 0 || c.head_dim > paged::kMostDim) return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->query || !a->output || !a->lengths || !a->offsets || (a->table_columns > 0 && !a->block_table) || !a->workspace ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0 ||
      a->workspace_bytes < nt_b200_chunk_attention_workspace_size() || a->batch > (1 << 30) || a->heads > (1 << 30) ||
      a->table_columns > (1LL << 40) || !(a->scale == a->scale))
    return NT_B200_ERR_INVALID_ARGUMENT;
  const int wide = a->index_dtype == NT_B200_INT64;
  chunk::Problem p{};
  p.query = a->query;
  p.out = a->output;
  p.lse = a->lse;
  p.key = static_cast<const uint8_t *>(c.key);
  p.value = static_cast<const uint8_t *>(c.value);
  p.key_scale = c.key_scale;
  p.value_scale = c.value_scale;
  p.lengths = {a->lengths, a->lengths_stride, wide};
  p.offsets = {a->offsets, a->offsets_stride, wide};
  p.block_table = {a->block_table, a->block_table_strides[1], wide};
  p.table_row_stride = a->block_table_strides[0];
  p.q_token = a->query_strides[0]; p.q_head = a->query_strides[1]; p.q_dim = a->query_strides[2];
  p.o_token = a->output_strides[0]; p.o_head = a->output_strides[1]; p.o_dim = a->output_strides[2];
  p.l_token = a->lse_strides[0]; p.l_head = a->lse_strides[1];
  p.k_page = c.key_strides[0]; p.k_head = c.key_strides[1]; p.k_token = c.key_strides[2];
  p.v_page = c.value_strides[0]; p.v_head = c.value_strides[1]; p.v_token = c.value_strides[2];
  p.ks_page = c.key_scale_strides[0]; p.ks_head = c.key_scale_strides[1];
  p.vs_page = c.value_scale_strides[0]; p.vs_head = c.value_scale_strides[1];
  p.pages = c.pages;
  const int64_t capacity = a->table_columns * c.page;
  p.capacity = (int)(capacity < paged::MOST_TOKENS ? capacity : paged::MOST_TOKENS);
  p.page_groups = (int)(c.page / 16);
  p.page_reciprocal = ((1ull << 36) + p.page_groups - 1) / p.page_groups;
  p.batch = (int)a->batch; p.heads = (int)a->heads; p.kv_heads = (int)c.kv_heads;
  p.group = (int)(a->heads / c.kv_heads);
  p.head_dim = (int)c.head_dim;
  p.page = (int)c.page;
  p.per_tile = p.group > chunk::BM ? 1 : chunk::BM / p.group;
  p.bf16 = a->dtype == NT_B200_BFLOAT16;
  p.q_vector = p.q_dim == 1 && p.q_token % 8 == 0 && p.q_head % 8 == 0 && rotary::aligned16(p.query);
  p.scale = (float)(a->scale * 1.4426950408889634);
  p.tokens = a->tokens;
  p.workspace = static_cast<uint8_t *>(a->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    if (c.code_dtype == NT_B200_INT8) return chunk::launch<scalar_t, int8_t>(p, s);
    return chunk::launch<scalar_t, __nv_fp8_e4m3>(p, s);
  });
}
