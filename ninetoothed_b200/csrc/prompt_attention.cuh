// Attention over whole prompts packed one after another, grouped heads, causal
// or not:
//     s = scale * (q . k),  o = softmax(s) v,  lse = ln sum exp(s)
// Sequence b has the queries query_offsets[b] .. query_offsets[b+1] - 1 and the
// keys key_offsets[b] .. key_offsets[b+1] - 1; the last query stands at the
// last key, so that a causal query i of nq sees the first nk - nq + 1 + i keys.
// A query that sees none gets o = 0 and lse = -inf.
//
// Bound by the tensor cores and, level with them, by the exponentials: a key
// block of 128 keys costs 256 rows 2048 cycles of dense MMA and 2048 cycles of
// the SM's 16 exponentials a cycle.  Now by a tile's round trip, softmax, then P V
// and the next Q K^T: four causal sequences of 4096 tokens, 32 heads on 8, 128
// bfloat16 elements: 580-630 us, 870-945 TFLOP/s.
//
// Rows of a tile are (query, head of the group) pairs, so that all query heads
// of a key/value head share one pass over its keys: 128 / group queries a tile.
// Persistent, one CTA an SM; an item of work is a key/value head and two tiles
// of 128 rows.  10 warps:
//   warp 0      TMA: an item's Q tiles, then its key and value blocks through a
//               ring of 5 shared-memory slots that runs on across items;
//   warp 1      tensor memory, and the MMAs from one thread: S_t = Q_t K_j^T,
//               O_t += P_t V_j with P_t read from tensor memory;
//   warps 2-9   softmax, 4 warps a tile, a thread a row.
// (Eight warps a tile, two threads a row of 64 keys each with their maxima
// exchanged through shared memory, took 1160 us where this takes 1080 us for
// four sequences of 4096 tokens, 32 heads of 128, not causal: at 96 registers a
// thread they spill.)
//
// The order of items comes from a small kernel before (plan_kernel): items of
// more than half, a quarter, an eighth of the longest item's key blocks, and the
// rest; in each class sequence by sequence, longest first, and head by head, so
// that a head's keys and values stay in L2 while they are used.  CTAs take the
// next item when they are done with one (a counter; warp 0 fetches it an item
// ahead and hands it to the other warps through shared memory), and the last to
// be taken are short.
#pragma once

#include <cuda.h>
#include "attention_tc.cuh"
#include "common.cuh"
#include "paged_attention.cuh"
#include "ptx.cuh"

namespace nt {
namespace prompt {

using paged::exp2_fast;
using paged::kLn2;
using paged::log2_fast;
using paged::reference;

struct Problem {
  const void *q, *k, *v;
  void *o;
  float *lse;  // or null
  IndexArray q_offsets, k_offsets;
  int64_t q_tokens, k_tokens, batch;
  int64_t q_token, q_head, q_dim, k_token, k_head, k_dim, v_token, v_head, v_dim, o_token, o_head, o_dim, l_token, l_head;
  int heads, kv_heads, group, head_dim, causal;
  float scale;  // softmax scale * log2 e
  void *workspace;
};

// A sequence's extents, or false (and the device error word) where its offsets
// are out of order or leave the tensors.
__device__ __forceinline__ bool extents(const Problem &p, int64_t b, int64_t &q0, int64_t &nq, int64_t &k0, int64_t &nk) {
  q0 = p.q_offsets[b];
  k0 = p.k_offsets[b];
  nq = p.q_offsets[b + 1] - q0;
  nk = p.k_offsets[b + 1] - k0;
  if (q0 < 0 || k0 < 0 || nq < 0 || nk < 0 || q0 + nq > p.q_tokens || k0 + nk > p.k_tokens) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return false;
  }
  return true;
}

// ---------------------------------------------------------------- any layout
// A warp a query row: head elements dealt over the lanes, one key at a time.
constexpr int kMostDim = 256;
template <typename T>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ Problem p) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= p.q_tokens * p.heads) return;
  const int64_t token = row / p.heads;
  const int h = (int)(row % p.heads);
  const int64_t b = paged::warp_search(p.batch, token, [&](int64_t i) { return p.q_offsets[i]; });
  int64_t q0, nq, k0, nk;
  if (!extents(p, b, q0, nq, k0, nk) || token < q0 || token >= q0 + nq) return;
  const int64_t limit = p.causal ? nk - nq + 1 + (token - q0) : nk;
  const T *q = static_cast<const T *>(p.q) + token * p.q_token + h * p.q_head;
  const int g = h / p.group;
  constexpr int E = kMostDim / 32;
  float qv[E], acc[E], far[E];  // (sums in two levels, as in the paged kernel)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < p.head_dim ? to_f(q[d * p.q_dim]) : 0.f;
    acc[e] = far[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f, l_far = 0.f;
  for (int64_t t = 0; t < limit; ++t) {
    const T *k = static_cast<const T *>(p.k) + (k0 + t) * p.k_token + g * p.k_head;
    const T *v = static_cast<const T *>(p.v) + (k0 + t) * p.v_token + g * p.v_head;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.head_dim) dot = fmaf(qv[e], to_f(k[(lane + 32 * e) * p.k_dim]), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = dot * p.scale;
    if (s > m) {
      const float alpha = exp2f(m - s);
      m = s;
      l *= alpha;
      l_far *= alpha;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        acc[e] *= alpha;
        far[e] *= alpha;
      }
    }
    const float w = exp2f(s - reference(m));
    l += w;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.head_dim) acc[e] = fmaf(w, to_f(v[(lane + 32 * e) * p.v_dim]), acc[e]);
    if (t % paged::FAR_KEYS == paged::FAR_KEYS - 1) {
      l_far += l;
      l = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        far[e] += acc[e];
        acc[e] = 0.f;
      }
    }
  }
  l += l_far;
  T *out = static_cast<T *>(p.o) + token * p.o_token + h * p.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    if (d < p.head_dim) out[d * p.o_dim] = from_f<T>(limit > 0 ? (acc[e] + far[e]) / l : 0.f);
  }
  if (p.lse && lane == 0) p.lse[token * p.l_token + h * p.l_head] = limit > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------- plan
constexpr int BM = 128, BN = 128;  // rows of a tile, keys of a block

// Two tiles of queries of one sequence.  A sequence's entries of one class are
// `total` from `first` on in the list, latest queries first.
struct alignas(32) Entry {
  int32_t q0, queries;  // first packed query, how many (at most two tiles')
  int32_t k0, keys;     // first packed key, how many the sequence has
  int32_t limit0;       // keys that the first query sees (causal), else `keys`
  int32_t first, total; // of an item: first says which it is
  int32_t head;         // of an item; unused in the list
};
// The workspace: Plan, the entries, then an int32 for each sequence and class and
// one for each item.
struct Plan {
  int32_t count, next, pad[6];  // entries; the next item
};

// Key blocks of the tile whose queries are [t * per_tile, ..) of an entry: up
// to the last key its last query sees, at least one; 0 for a tile without
// queries.
__host__ __device__ __forceinline__ int blocks_of(const Entry &e, int t, int per_tile, bool causal) {
  const int last = (e.queries < (t + 1) * per_tile ? e.queries : (t + 1) * per_tile) - 1;
  if (last < t * per_tile) return 0;
  int seen = causal ? e.limit0 + last : e.keys;
  if (seen > e.keys) seen = e.keys;
  return seen <= 0 ? 1 : (seen + BN - 1) / BN;
}

constexpr int PLAN_THREADS = 1024, CLASSES = 4, BINS = PLAN_THREADS / CLASSES;

// A sequence in the plan: `total` entries, entry i the queries from i * pair on.
struct Span {
  int64_t q0, nq, k0, nk;
  int total, blocks;  // entries; key blocks of the last
  __device__ bool load(const Problem &p, int64_t b, int pair) {
    if (!extents(p, b, q0, nq, k0, nk)) nq = 0;
    total = (int)((uint32_t)(nq + pair - 1) / (uint32_t)pair);  // (at most 2^30 tokens)
    blocks = (int)((uint32_t)(nk + BN - 1) / BN);
    return total > 0;
  }
  // the first entry of class `c` or a lower one, for a longest item of `most`
  // key blocks: those with more than most / 2^(c + 1)
  __device__ int from(const Problem &p, int c, int most, int pair) const {
    if (c == CLASSES - 1) return 0;
    const int least = most >> (c + 1);
    if (!p.causal) return blocks > least ? 0 : total;
    const int64_t before = (int64_t)least * BN - (nk - nq);  // queries that see no more
    return before < 0 ? 0 : before > nq ? total : min((int)((uint32_t)before / (uint32_t)pair), total);
  }
};

// The candidate entries: sequence b owns the candidates from query_offsets[b] /
// pair + b on (pair = queries of two tiles), as many as it can have entries;
// those past its last are empty.  Counting sort of the sequences' classes by
// class and key blocks, then the entries at their class's place.
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const __grid_constant__ Problem p, int64_t candidates,
                                                            int per_tile) {
  __shared__ int bins[CLASSES * BINS];
  __shared__ int warp_sums[PLAN_THREADS / 32];
  __shared__ int most_shared, out_of_order;
  wait_prior_grid();
  allow_dependent_launch();
  const int pair = 2 * per_tile;
  Plan *plan = static_cast<Plan *>(p.workspace);
  Entry *list = reinterpret_cast<Entry *>(plan + 1);
  int32_t *first_of = reinterpret_cast<int32_t *>(list + candidates);  // [batch][CLASSES]
  bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    most_shared = 1;
    out_of_order = 0;
  }
  __syncthreads();
  Span w;
  for (int64_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
    if (!extents(p, b, w.q0, w.nq, w.k0, w.nk)) out_of_order = 1;
    else if (w.load(p, b, pair)) atomicMax(&most_shared, w.blocks);
  }
  __syncthreads();
  if (out_of_order) {  // sequences may overlap and outnumber the candidates: none is taken
    if (threadIdx.x == 0) plan->count = plan->next = 0;
    return;
  }
  const int most = most_shared;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t b = threadIdx.x; b < p.batch; b += PLAN_THREADS) {
      if (!w.load(p, b, pair)) continue;
      int end = w.total;
      for (int c = 0; c < CLASSES; ++c) {
        const int from = w.from(p, c, most, pair);
        int *bin = &bins[c * BINS + (int)((uint32_t)(most - w.blocks) * (BINS - 1) / (uint32_t)most)];
        if (pass == 0) atomicAdd(bin, end - from);
        else first_of[b * CLASSES + c] = atomicAdd(bin, end - from);
        end = from;
      }
    }
    __syncthreads();
    if (pass == 1) break;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = bins[threadIdx.x];
    int up = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += x;
    }
    if (lane == 31) warp_sums[warp] = up;
    __syncthreads();
    int base = 0;
    for (int i = 0; i < warp; ++i) base += warp_sums[i];
    bins[threadIdx.x] = base + up - n;
    if (threadIdx.x == PLAN_THREADS - 1) {
      plan->count = base + up;
      plan->next = 0;
    }
    __syncthreads();
  }
  for (int64_t x = threadIdx.x; x < candidates; x += PLAN_THREADS) {
    int64_t low = 0, high = p.batch;  // the largest b whose first candidate is <= x
    while (high - low > 1) {
      const int64_t mid = (low + high) / 2;
      if ((uint32_t)p.q_offsets[mid] / (uint32_t)pair + mid <= x) low = mid;
      else high = mid;
    }
    if (!w.load(p, low, pair)) continue;
    const int64_t i = x - ((uint32_t)w.q0 / (uint32_t)pair + low);
    if (i < 0 || i >= w.total) continue;
    int c = 0, end = w.total, from = w.from(p, 0, most, pair);
    while (i < from) {
      end = from;
      from = w.from(p, ++c, most, pair);
    }
    const int64_t first = i * pair;
    Entry e{};
    e.q0 = (int32_t)(w.q0 + first);
    e.queries = (int32_t)(w.nq - first < pair ? w.nq - first : pair);
    e.k0 = (int32_t)w.k0;
    e.keys = (int32_t)w.nk;
    e.limit0 = (int32_t)(p.causal ? w.nk - w.nq + 1 + first : w.nk);
    e.first = first_of[low * CLASSES + c];
    e.total = end - from;
    list[e.first + end - 1 - (int)i] = e;
  }
}

// ---------------------------------------------------------------- tensor cores
constexpr int TILES = 2, RING = 5;
constexpr int SOFTMAX_WARPS = 8;
constexpr int THREADS = (2 + SOFTMAX_WARPS) * 32;
constexpr int TMEM_COLS = 512;

template <int DP>  // head_dim padded to 64 or 128
struct Layout {
  static constexpr int ATOMS = DP / 64;         // 128-byte swizzle atoms along the head
  static constexpr int Q_BYTES = BM * DP * 2;   // one Q tile
  static constexpr int KV_BYTES = BN * DP * 2;  // one key or value block
  static constexpr int RING_OFF = TILES * Q_BYTES;
  static constexpr int CTRL_OFF = RING_OFF + RING * KV_BYTES;
  static constexpr int ROWS_OFF = CTRL_OFF + 384;  // ushort2 [BM]: a row's query and head in its tile
  static constexpr int NOTES_OFF = ROWS_OFF + BM * 4;  // uint32 [2][128], see take_out
  static constexpr int SMEM_BYTES = NOTES_OFF + 2 * 128 * 4;
  static_assert(120 + 16 * RING <= 240, "barrier slots");
  static_assert(SMEM_BYTES <= 232448, "shared memory of a CTA");
};

struct Params {
  Problem p;
  int per_tile;        // queries of a tile
  int64_t candidates;  // places in the list
  __device__ __forceinline__ Entry *list() const {
    return reinterpret_cast<Entry *>(static_cast<Plan *>(p.workspace) + 1);
  }
  // an item's predecessor among those that need a second pass
  __device__ __forceinline__ int32_t *chain() const {
    return reinterpret_cast<int32_t *>(list() + candidates) + p.batch * CLASSES;
  }
};

// A masked key's weight is 0, but 0 times an infinity or NaN in its value is NaN
// in the MMA.  An item in which a row's O is not finite is therefore taken a
// second time, after the CTA's other items, without the values that some row does
// not see: of the item's keys those are [lo, keys), of them [hi, keys) and what a
// block holds past `keys` (another sequence's values) are seen by no row.  Warp 1
// zeroes the latter in shared memory before P V; among the former, fewer than the
// item's 256 queries, it looks for elements that are not finite, zeroes those too
// and notes them, and the rows that see them get them back at the end.  Blocks
// before `lo` are left alone: what every row sees is every row's.  Such an item
// takes twice its time; done for every item at once (a warp of its own), the
// search took packed prompts of up to 2048 tokens from 138 to 158 us.
__device__ __forceinline__ int first_unseen(const Entry &e, bool causal) {
  return causal ? min(max(e.limit0, 0), e.keys) : e.keys;
}
__device__ __forceinline__ int first_seen_by_none(const Entry &e, bool causal) {
  return causal ? min(max(e.limit0 + e.queries - 1, 0), e.keys) : e.keys;
}

__device__ __forceinline__ void store_shared16(uint32_t to, const uint4 &v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// What is not finite among an element's values of the keys from lo on, in three
// fields of 9 bits: the first key, counted from lo, with +inf, -inf and NaN; 511:
// none.
constexpr uint32_t kAllFinite = 0x7ffffffu;
__device__ __forceinline__ void note_not_finite(uint32_t *at, float v, uint32_t key) {
  const int shift = v == INFINITY ? 0 : v == -INFINITY ? 9 : 18;
  uint32_t old = *reinterpret_cast<volatile uint32_t *>(at);
  while ((old >> shift & 511u) > key) {
    const uint32_t now = atomicCAS(at, old, (old & ~(511u << shift)) | key << shift);
    if (now == old) break;
    old = now;
  }
}
// What the values noted add to a row that sees `seen` keys from lo on.
__device__ __forceinline__ float noted(uint32_t note, int seen) {
  const float up = (int)(note & 511u) < seen ? INFINITY : 0.f, down = (int)(note >> 9 & 511u) < seen ? -INFINITY : 0.f;
  return (int)(note >> 18 & 511u) < seen ? NAN : up + down;
}

// Takes the values of one block's keys [from, until) that are not finite out of
// shared memory into `notes` (a key's place counted from lo = from - first), and
// zeroes the keys [until, BN); a full warp.  Returns whether there were any; the
// first of an item clears the notes.
template <typename T, int DP>
__device__ __forceinline__ bool take_out(uint32_t block, int from, int until, int first, uint32_t *notes, bool any) {
  constexpr int WORDS = DP / 8, KEYS = 32 / WORDS;  // 16-byte words of a key; keys a step of the warp
  constexpr uint32_t EXPONENT = Elem<T>::is_f16 ? 0x7c00 : 0x7f80;
  constexpr uint32_t ONES = EXPONENT * 0x10001u, CARRY = (0x8000u - EXPONENT) * 0x10001u;
  const int lane = threadIdx.x & 31, word = lane % WORDS;
  block += (word / 8) * (BN * 128);
  auto place = [&](int key) { return block + key * 128 + ((word % 8) ^ (key & 7)) * 16; };
  auto not_finite = [&](const uint4 &x) {  // an exponent of all ones carries into its half's top bit
    return ((((x.x & ONES) + CARRY) | ((x.y & ONES) + CARRY)) | (((x.z & ONES) + CARRY) | ((x.w & ONES) + CARRY))) & 0x80008000u;
  };
#pragma unroll 8
  for (int key = until + lane / WORDS; key < BN; key += KEYS) store_shared16(place(key), make_uint4(0, 0, 0, 0));
  constexpr int AHEAD = 8;
#pragma unroll 1
  for (int k0 = from + lane / WORDS; k0 - lane / WORDS < until; k0 += AHEAD * KEYS) {
    uint4 x[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      x[u] = k0 + u * KEYS < until ? paged::load_shared16(place(k0 + u * KEYS)) : make_uint4(0, 0, 0, 0);
    uint32_t bad = 0;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) bad |= not_finite(x[u]);
    if (!__any_sync(0xffffffffu, bad != 0)) continue;
    if (!any) {
      for (int d = lane; d < DP; d += 32) notes[d] = kAllFinite;
      __syncwarp();
      any = true;
    }
    if (bad == 0) continue;
#pragma unroll 1
    for (int key = k0; key < min(until, k0 + AHEAD * KEYS); key += KEYS) {
      uint4 w = paged::load_shared16(place(key));
      if (not_finite(w) == 0) continue;
      T *v = reinterpret_cast<T *>(&w);
      for (int e = 0; e < 8; ++e) {
        const float value = to_f(v[e]);
        if (fabsf(value) < INFINITY) continue;
        note_not_finite(notes + word * 8 + e, value, (uint32_t)(key - from + first));
        v[e] = from_f<T>(0.f);
      }
      store_shared16(place(key), w);
    }
  }
  return any;
}

// The shared memory beside the tiles: barriers (8 bytes each), items, notes.
template <int DP> struct Control {
  using L = Layout<DP>;
  uint32_t base, ctrl;
  volatile int *abort_flag;
  volatile uint32_t *tmem_base;
  volatile int4 *item_slots;  // [2][2]
  int *again;                 // items that need a second pass, chained through the workspace: the last, or kEnd
  volatile int *notes_taken;  // [2]: the item has notes
  uint32_t *notes;            // [2][128], see take_out
  __device__ __forceinline__ explicit Control(uint8_t *smem) {
    base = ptx::smem_u32(smem);
    ctrl = base + L::CTRL_OFF;
    tmem_base = reinterpret_cast<volatile uint32_t *>(smem + L::CTRL_OFF + 240);
    abort_flag = reinterpret_cast<volatile int *>(smem + L::CTRL_OFF + 244);
    item_slots = reinterpret_cast<volatile int4 *>(smem + L::CTRL_OFF + 288);
    again = reinterpret_cast<int *>(smem + L::CTRL_OFF + 352);
    notes_taken = again + 1;
    notes = reinterpret_cast<uint32_t *>(smem + L::NOTES_OFF);
  }
#define NT_BARRIER __device__ __forceinline__ uint32_t
  // of tile t
  NT_BARRIER q_full(int t) const { return ctrl + 8u * t; }       // Q_t landed
  NT_BARRIER q_free(int t) const { return ctrl + 16 + 8u * t; }  // the item's last Q_t K^T done
  NT_BARRIER s_full(int t) const { return ctrl + 32 + 8u * t; }  // S_t of a key block in tensor memory
  NT_BARRIER p_full(int t) const { return ctrl + 48 + 8u * t; }  // P_t written, O_t rescaled
  NT_BARRIER o_done(int t) const { return ctrl + 64 + 8u * t; }  // the item's last P_t V done
  NT_BARRIER o_free(int t) const { return ctrl + 80 + 8u * t; }  // O_t read out
  // of ring slot s
  NT_BARRIER slot_full(int s) const { return ctrl + 96 + 8u * s; }
  NT_BARRIER slot_empty(int s) const { return ctrl + 96 + 8u * RING + 8u * s; }
  // of items, two in turn: the notes of a second pass are complete; handed over;
  // taken by the MMA issuer and the softmax warps
  NT_BARRIER item_clean(int s) const { return ctrl + 96 + 16u * RING + 8u * s; }
  // after a wait gave up: the MMAs in flight are done
  NT_BARRIER settled() const { return ctrl + 112 + 16u * RING; }
  NT_BARRIER item_full(int s) const { return ctrl + 248 + 8u * s; }
  NT_BARRIER item_empty(int s) const { return ctrl + 264 + 8u * s; }
#undef NT_BARRIER
  // The CTA's i-th item; queries 0 is the end of a pass.
  __device__ __forceinline__ void hand_over(int i, const Entry &e, int item) const {
    volatile int4 *to = item_slots + 2 * (i & 1);
    to[0].x = e.q0; to[0].y = e.queries; to[0].z = e.k0; to[0].w = e.keys;
    to[1].x = e.limit0; to[1].y = item; to[1].w = e.head;
    ptx::mbar_arrive(item_full(i & 1));
  }
  // Takes it once it was handed over; false where the wait gave up.  The caller
  // then lets go of it.
  __device__ __forceinline__ bool take_item(int i, Entry &e) const {
    if (!ptx::mbar_wait(item_full(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag)) return false;
    const volatile int4 *at = item_slots + 2 * (i & 1);
    e.q0 = at[0].x; e.queries = at[0].y; e.k0 = at[0].z; e.keys = at[0].w;
    e.limit0 = at[1].x; e.first = at[1].y; e.head = at[1].w;
    return true;
  }
};

// Where a role stands.
struct Standing {
  int i;                    // items so far
  int r;                    // ring position of the item's K_0
  int blocks[TILES];        // key blocks of tile t in earlier items
  int used[TILES];          // earlier items that had tile t
  uint32_t s_turn, o_turn;  // phases of s_full and o_done
};
// Items' places in the chain of second passes, before and at its end.
constexpr int kUnchained = -2, kEnd = -1;

// ---------------------------------------------------------------- producer
// One thread: hands over the items and loads their tiles and blocks.  In the first
// pass the next item is fetched in three steps, each waiting for the one before only
// when it comes to its turn among this item's loads; the second goes along the chain.
template <int DP, bool AGAIN>
__device__ __forceinline__ void produce(const Control<DP> &c, const Params &prm, const CUtensorMap *tmap_q,
                                        const CUtensorMap *tmap_k, const CUtensorMap *tmap_v, Standing &at) {
  using L = Layout<DP>;
  const Problem &p = prm.p;
  const int per_tile = prm.per_tile;
  const uint32_t q_bytes = (uint32_t)(per_tile * p.group * 128 * L::ATOMS);
  // Items count along the list by a sequence's entries of one class, among them
  // head by head, in it entry by entry.
  Plan *plan = static_cast<Plan *>(p.workspace);
  const Entry *list = prm.list();
  const int64_t num_items = (int64_t)plan->count * p.kv_heads;
  int next = 0;
  Entry any{}, ahead{};
  auto fetch = [&](int step) {
    if (step == 0) {
      next = AGAIN ? prm.chain()[next] : atomicAdd(&plan->next, 1);
    } else if (step == 1) {
      any = Entry{};
      if (next >= 0 && next < num_items) any = list[next / p.kv_heads];  // of the same sequence and class
    } else {
      ahead = Entry{};
      if (next >= 0 && next < num_items) {
        const int r = (int)(next - (int64_t)any.first * p.kv_heads), h = r / any.total;
        ahead = list[any.first + r - h * any.total];
        ahead.head = h;
      }
    }
  };
  if (AGAIN) next = *c.again;
  else fetch(0);
  fetch(1);
  fetch(2);
  for (;; ++at.i) {
    const Entry e = ahead;
    if (!ptx::mbar_wait(c.item_empty(at.i & 1), ((uint32_t)(at.i >> 1) & 1u) ^ 1u, c.abort_flag)) return;
    if (!AGAIN && e.queries != 0) prm.chain()[next] = kUnchained;
    c.hand_over(at.i, e, next);
    if (e.queries == 0) break;
    fetch(0);
    const int h = e.head;
    const int n[TILES] = {blocks_of(e, 0, per_tile, p.causal), blocks_of(e, 1, per_tile, p.causal)};
    const int n_max = max(n[0], n[1]);
    for (int t = 0; t < TILES; ++t) {
      if (n[t] == 0) continue;
      if (at.used[t] > 0 && !ptx::mbar_wait(c.q_free(t), (uint32_t)(at.used[t] - 1) & 1u, c.abort_flag)) return;
      ++at.used[t];
      ptx::mbar_arrive_expect_tx(c.q_full(t), q_bytes);
      for (int x = 0; x < L::ATOMS; ++x)
        ptx::tma_load_3d(c.base + t * L::Q_BYTES + x * (BM * 128), tmap_q, c.q_full(t), 64 * x, h * p.group,
                         e.q0 + t * per_tile);
    }
    for (int j = 0; j < 2 * n_max; ++j, ++at.r) {  // K_0, V_0, K_1, V_1, ...
      const int slot = at.r % RING;
      if (!ptx::mbar_wait(c.slot_empty(slot), ((uint32_t)(at.r / RING) & 1u) ^ 1u, c.abort_flag)) return;
      ptx::mbar_arrive_expect_tx(c.slot_full(slot), L::KV_BYTES);
      const CUtensorMap *map = (j & 1) ? tmap_v : tmap_k;
      for (int x = 0; x < L::ATOMS; ++x)
        ptx::tma_load_3d(c.base + L::RING_OFF + slot * L::KV_BYTES + x * (BN * 128), map, c.slot_full(slot), 64 * x, h,
                         e.k0 + (j >> 1) * BN);
      if (j == 4) fetch(1);
      if (j == 8) fetch(2);
    }
    if (2 * n_max <= 4) fetch(1);
    if (2 * n_max <= 8) fetch(2);
  }
  ++at.i;
}

// ---------------------------------------------------------------- MMA issuer
// An item's MMAs; false where a wait gave up.  The first pass: one thread.  The
// second (AGAIN): a full warp, which takes out values on the way; lane 0 issues.
template <typename T, int DP, bool AGAIN>
__device__ __forceinline__ bool issue_item(const Control<DP> &c, uint32_t tmem_base, const Problem &p, int per_tile,
                                           const Entry &e, Standing &at) {
  using L = Layout<DP>;
  constexpr uint32_t fmt = tc::umma_format<T>();
  constexpr uint32_t idesc_qk = ptx::f16_idesc(fmt, 0, 0, BM, BN);  // B = keys, K-major
  constexpr uint32_t idesc_pv = ptx::f16_idesc(fmt, 0, 1, BM, DP);  // B = values, MN-major
  const bool issues = !AGAIN || (threadIdx.x & 31) == 0;
  auto tmem_s = [&](int t) { return tmem_base + (uint32_t)(t * BN); };
  auto tmem_o = [&](int t) { return tmem_base + (uint32_t)(TILES * BN + t * 128); };
  auto slot_addr = [&](int r) { return c.base + L::RING_OFF + (r % RING) * L::KV_BYTES; };
  auto wait = [&](uint32_t bar, uint32_t parity) {
    return AGAIN ? ptx::mbar_wait_warp(bar, parity, c.abort_flag) : ptx::mbar_wait(bar, parity, c.abort_flag);
  };
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
  const int n[TILES] = {blocks_of(e, 0, per_tile, p.causal), blocks_of(e, 1, per_tile, p.causal)};
  const int n_max = max(n[0], n[1]);
  bool any = false;
  if (!wait_slot(at.r)) return false;  // K_0
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    if (n[t] == 0) continue;
    if (!wait(c.q_full(t), (uint32_t)at.used[t] & 1u)) return false;
    ptx::tc_fence_after();
    issue_qk(t, at.r);
    if (n[t] == 1) commit(c.q_free(t));
  }
  commit(c.slot_empty(at.r % RING));
  for (int j = 0; j < n_max; ++j) {
    const int rv = at.r + 2 * j + 1, rk = at.r + 2 * j + 2;
    if (!wait_slot(rv)) return false;
    if constexpr (AGAIN) {
      const int lo = first_unseen(e, p.causal) - j * BN, hi = first_seen_by_none(e, p.causal) - j * BN;
      if (lo < BN) {
        any = take_out<T, DP>(slot_addr(rv), max(lo, 0), min(max(hi, 0), BN), max(-lo, 0), c.notes + (at.i & 1) * 128, any);
        ptx::fence_proxy_async_smem();  // the MMA reads what was written here
        __syncwarp();
      }
    }
    bool next_keys = false;
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
        if (!next_keys) {
          if (!wait_slot(rk)) return false;
          next_keys = true;
          ptx::tc_fence_after();
        }
        issue_qk(t, rk);
        if (j + 2 == n[t]) commit(c.q_free(t));
      }
    }
    commit(c.slot_empty(rv % RING));
    if (next_keys) commit(c.slot_empty(rk % RING));
  }
  at.r += 2 * n_max;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    at.blocks[t] += n[t];
    at.used[t] += n[t] > 0;
  }
  if (AGAIN && issues) {
    c.notes_taken[at.i & 1] = any;
    ptx::mbar_arrive(c.item_clean(at.i & 1));
  }
  return true;
}

template <typename T, int DP, bool AGAIN>
__device__ __forceinline__ void issue(const Control<DP> &c, uint32_t tmem_base, const Params &prm, Standing &at) {
  Entry e;
  for (bool more = true; more; ++at.i) {
    const bool taken = c.take_item(at.i, e);
    if (AGAIN ? !__all_sync(0xffffffffu, taken) : !taken) return;
    if (!AGAIN || (threadIdx.x & 31) == 0) ptx::mbar_arrive(c.item_empty(at.i & 1));
    more = e.queries != 0;
    if (more && !issue_item<T, DP, AGAIN>(c, tmem_base, prm.p, prm.per_tile, e, at)) return;
  }
}

// ---------------------------------------------------------------- softmax, rescaling, output
// What was taken out of a second pass, to a row that sees the keys before `seen`,
// counted from the first that was searched.
template <typename T>
__device__ __noinline__ void give_back(T *out, int64_t stride, int head_dim, const uint32_t *notes, int seen) {
  for (int d = 0; d < head_dim; ++d) {
    const float back = noted(notes[d], seen);
    if (!(back == 0.f)) out[d * stride] = from_f<T>(to_f(out[d * stride]) + back);
  }
}

// A row's maximum moves only when a block passes it by 2^kLead, so that O is
// rescaled rarely, and P is kept 2^kRise above it.  P is rounded to the operands'
// type for the MMA, 8 bits (bfloat16) or 11 (float16).  float16: its largest, 2^15,
// stays in range, and what a long tail adds out of the subnormals: of 131072 keys
// with 2^-25.5 of the largest weight all was lost at (14, 0); values of up to 65504
// cannot bring O out of fp32's range.  bfloat16: values can, so the lead that adds
// to them is kept small (2^24 took as long), and its range needs no rise.
template <typename T> constexpr float kLead = Elem<T>::is_f16 ? 6.f : 8.f;
template <typename T> constexpr float kRise = Elem<T>::is_f16 ? 9.f : 0.f;
template <typename T> constexpr float kFall = Elem<T>::is_f16 ? 1.f / 512.f : 1.f;  // 2^-kRise

template <typename T, int DP, bool AGAIN>
__device__ __forceinline__ void attend(const Control<DP> &c, uint32_t tmem_base, const Params &prm, const ushort2 *rows,
                                       Standing &at) {
  const Problem &p = prm.p;
  const int per_tile = prm.per_tile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto tmem_s = [&](int t) { return tmem_base + (uint32_t)(t * BN); };
  auto tmem_o = [&](int t) { return tmem_base + (uint32_t)(TILES * BN + t * 128); };
  const int t = (warp - 2) / 4, quarter = warp & 3;
  const int row = quarter * 32 + lane;  // row of the tile = lane of tensor memory
  const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
  auto arrive_warp = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(bar);
  };
  const float scale = p.scale;
  const int first = at.i;
  // A block's scores fill a thread's registers: what an item's end needs is read
  // again there, and the item let go only then.
  for (;; ++at.i) {
    int n_t, limit, sure;  // key blocks; keys that the row sees; keys that all rows see
    {
      Entry e;
      if (!__all_sync(0xffffffffu, c.take_item(at.i, e))) return;
      if (e.queries == 0) break;
      n_t = blocks_of(e, t, per_tile, p.causal);
      limit = p.causal ? min(e.limit0 + t * per_tile + rows[row].x, e.keys) : e.keys;
      sure = p.causal ? min(e.limit0 + t * per_tile, e.keys) : e.keys;
    }
    if (n_t == 0) {
      arrive_warp(c.item_empty(at.i & 1));
      continue;
    }

    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n_t; ++j) {
      if (!ptx::mbar_wait_warp(c.s_full(t), at.s_turn, c.abort_flag)) return;
      at.s_turn ^= 1;
      ptx::tc_fence_after();
      uint32_t sr[BN];
#pragma unroll
      for (int x = 0; x < BN / 32; ++x)
        ptx::tmem_ld_32x32b_x32(tmem_s(t) + lane_base + (uint32_t)(x * 32), *reinterpret_cast<uint32_t(*)[32]>(&sr[x * 32]));
      ptx::tmem_ld_wait();
      float *s = reinterpret_cast<float *>(sr);
      if ((j + 1) * BN > sure) {
        const int seen = limit - j * BN;
#pragma unroll
        for (int x = 0; x < BN; ++x) s[x] = x < seen ? s[x] : -INFINITY;
      }
      float top[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) top[u] = s[u];
#pragma unroll
      for (int x = 8; x < BN; ++x) top[x & 7] = fmaxf(top[x & 7], s[x]);
#pragma unroll
      for (int u = 4; u > 0; u >>= 1)
#pragma unroll
        for (int v = 0; v < u; ++v) top[v] = fmaxf(top[v], top[v + u]);
      const float block_top = top[0] * scale;
      const bool move = block_top > m + kLead<T>;
      const float m_new = move ? block_top : m;
      const float alpha = move ? exp2_fast(m - m_new) : 1.f;
      const float ref = reference(m_new) - kRise<T>;
      float sum[8] = {};
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t packed[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          const int k = half * 64 + 2 * x;
          const float p0 = exp2_fast(fmaf(s[k], scale, -ref)), p1 = exp2_fast(fmaf(s[k + 1], scale, -ref));
          sum[(2 * x) & 7] += p0;
          sum[(2 * x + 1) & 7] += p1;
          packed[x] = tc::attn::pack2<T>(p0, p1);
        }
        ptx::tmem_st_32x32b_x32(tmem_s(t) + lane_base + (uint32_t)(half * 32), packed);
      }
#pragma unroll
      for (int u = 4; u > 0; u >>= 1)
#pragma unroll
        for (int v = 0; v < u; ++v) sum[v] += sum[v + u];
      if (j > 0 && __any_sync(0xffffffffu, move)) {
        // O_t holds P(j-1) V(j-1): the commit of S_t(j) covers it
        uint32_t o[DP];
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
          ptx::tmem_ld_32x32b_x32(tmem_o(t) + lane_base + (uint32_t)(x * 32), *reinterpret_cast<uint32_t(*)[32]>(&o[x * 32]));
        ptx::tmem_ld_wait();
#pragma unroll
        for (int y = 0; y < DP; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * alpha);
#pragma unroll
        for (int x = 0; x < DP / 32; ++x)
          ptx::tmem_st_32x32b_x32(tmem_o(t) + lane_base + (uint32_t)(x * 32), *reinterpret_cast<uint32_t(*)[32]>(&o[x * 32]));
      }
      m = m_new;
      l = l * alpha + sum[0];
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      arrive_warp(c.p_full(t));
    }
    if (!ptx::mbar_wait_warp(c.o_done(t), at.o_turn, c.abort_flag)) return;
    at.o_turn ^= 1;
    ptx::tc_fence_after();
    uint32_t o[DP];
#pragma unroll
    for (int x = 0; x < DP / 32; ++x)
      ptx::tmem_ld_32x32b_x32(tmem_o(t) + lane_base + (uint32_t)(x * 32), *reinterpret_cast<uint32_t(*)[32]>(&o[x * 32]));
    ptx::tmem_ld_wait();
    ptx::tc_fence_before();
    arrive_warp(c.o_free(t));
    Entry e;
    c.take_item(at.i, e);
    if (!AGAIN) arrive_warp(c.item_empty(at.i & 1));
    const int query = t * per_tile + rows[row].x;
    if (query < e.queries && rows[row].x < per_tile) {
      const int64_t token = e.q0 + query;
      const int head = e.head * p.group + rows[row].y;
      const float f = l == 0.f ? 0.f : 1.f / l;
      T *out = static_cast<T *>(p.o) + token * p.o_token + (int64_t)head * p.o_head;
      if (p.head_dim == DP && p.o_dim == 1 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
#pragma unroll
        for (int x = 0; x < DP / 8; ++x) {
          const float *v = reinterpret_cast<const float *>(o + x * 8);
          *reinterpret_cast<int4 *>(out + x * 8) =
              make_int4((int)tc::attn::pack2<T>(v[0] * f, v[1] * f), (int)tc::attn::pack2<T>(v[2] * f, v[3] * f),
                        (int)tc::attn::pack2<T>(v[4] * f, v[5] * f), (int)tc::attn::pack2<T>(v[6] * f, v[7] * f));
        }
      } else {
#pragma unroll
        for (int x = 0; x < DP; ++x)
          if (x < p.head_dim) out[x * p.o_dim] = from_f<T>(__uint_as_float(o[x]) * f);
      }
      if (p.lse)
        p.lse[token * p.l_token + (int64_t)head * p.l_head] = l == 0.f ? -INFINITY : (m + log2_fast(l * kFall<T>)) * kLn2;
      if (!AGAIN) {
        float worst[8] = {};  // a sum is NaN if any element is NaN or infinite
#pragma unroll
        for (int x = 0; x < DP; ++x) worst[x & 7] = fmaf(__uint_as_float(o[x]), 0.f, worst[x & 7]);
#pragma unroll
        for (int u = 4; u > 0; u >>= 1)
#pragma unroll
          for (int v = 0; v < u; ++v) worst[v] += worst[v + u];
        if (!(worst[0] == 0.f) && atomicCAS(prm.chain() + e.first, kUnchained, kEnd) == kUnchained)
          prm.chain()[e.first] = atomicExch(c.again, e.first);
      } else if (ptx::mbar_wait(c.item_clean(at.i & 1), (uint32_t)(at.i - first) >> 1 & 1u, c.abort_flag) &&
                 c.notes_taken[at.i & 1]) {
        give_back(out, p.o_dim, p.head_dim, c.notes + (at.i & 1) * 128, limit - first_unseen(e, p.causal));
      }
    }
    if (AGAIN) arrive_warp(c.item_empty(at.i & 1));
  }
  arrive_warp(c.item_empty(at.i & 1));
  ++at.i;
}

// The second pass, from where a thread stands.  Out of line: in the kernel's own
// code it took registers and time from the first (packed prompts of up to 2048
// tokens: 147 us beside 139).
template <typename T, int DP>
__device__ __noinline__ Standing second_pass(uint8_t *smem, uint32_t tmem_base, const Params &prm, const CUtensorMap *tmap_q,
                                         const CUtensorMap *tmap_k, const CUtensorMap *tmap_v, Standing at) {
  const Control<DP> c(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    if (lane == 0) produce<DP, true>(c, prm, tmap_q, tmap_k, tmap_v, at);
  } else if (warp == 1) {
    at.i = __shfl_sync(0xffffffffu, at.i, 0);
    at.r = __shfl_sync(0xffffffffu, at.r, 0);
    for (int t = 0; t < TILES; ++t) {
      at.blocks[t] = __shfl_sync(0xffffffffu, at.blocks[t], 0);
      at.used[t] = __shfl_sync(0xffffffffu, at.used[t], 0);
    }
    issue<T, DP, true>(c, tmem_base, prm, at);
  } else {
    attend<T, DP, true>(c, tmem_base, prm, reinterpret_cast<const ushort2 *>(smem + Layout<DP>::ROWS_OFF), at);
  }
  return at;
}

// After a wait gave up: the copies and MMAs that a thread has in flight, so that the
// CTA's shared and tensor memory are at rest when it ends.
template <int DP> __device__ __noinline__ void settle(uint8_t *smem, Standing at) {
  constexpr uint64_t limit_ns = 1000000000ull;
  const Control<DP> c(smem);
  volatile int over = 0;
  if (threadIdx.x == 0) {
    for (int r = max(at.r - RING, 0); r < at.r; ++r)
      ptx::mbar_wait(c.slot_full(r % RING), (uint32_t)(r / RING) & 1u, &over, limit_ns);
    for (int t = 0; t < TILES; ++t)
      if (at.used[t] > 0) ptx::mbar_wait(c.q_full(t), (uint32_t)(at.used[t] - 1) & 1u, &over, limit_ns);
  } else if (threadIdx.x == 32) {
    ptx::mma_commit(c.settled());
    ptx::mbar_wait(c.settled(), 0, &over, limit_ns);
  }
}

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Params prm) {
  using L = Layout<DP>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  if ((base & 1023u) != 0) {  // the swizzle needs it; there is no room to align by hand
    record_error(NT_B200_ERR_INVALID_ARGUMENT);
    return;
  }
  const Control<DP> c(smem);
  const Problem &p = prm.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_tile = prm.per_tile;

  if (threadIdx.x == 0) {
    for (int t = 0; t < TILES; ++t) {
      ptx::mbar_init(c.q_full(t), 1);
      ptx::mbar_init(c.q_free(t), 1);
      ptx::mbar_init(c.s_full(t), 1);
      ptx::mbar_init(c.p_full(t), 4);  // a warp's lanes arrive as one
      ptx::mbar_init(c.o_done(t), 1);
      ptx::mbar_init(c.o_free(t), 4);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(c.item_full(s), 1);
      ptx::mbar_init(c.item_empty(s), 1 + SOFTMAX_WARPS);
      ptx::mbar_init(c.item_clean(s), 1);
    }
    for (int s = 0; s < RING; ++s) {
      ptx::mbar_init(c.slot_full(s), 1);
      ptx::mbar_init(c.slot_empty(s), 1);
    }
    ptx::mbar_init(c.settled(), 1);
    *c.abort_flag = 0;
    *c.again = kEnd;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_q);
    ptx::prefetch_tmap(&tmap_k);
    ptx::prefetch_tmap(&tmap_v);
  }
  ushort2 *rows = reinterpret_cast<ushort2 *>(smem + L::ROWS_OFF);
  if (threadIdx.x < BM)
    rows[threadIdx.x] = make_ushort2((unsigned short)(threadIdx.x / p.group), (unsigned short)(threadIdx.x % p.group));
  // rows past per_tile * group are never loaded: zeros
  if (per_tile * p.group < BM) {
    for (int i = threadIdx.x; i < TILES * L::Q_BYTES / 16; i += THREADS)
      reinterpret_cast<int4 *>(smem)[i] = make_int4(0, 0, 0, 0);
    ptx::fence_proxy_async_smem();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t *>(c.tmem_base)), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  wait_prior_grid();
  const uint32_t tmem_base = *c.tmem_base;

  Standing at{};
  if (warp == 0) {
    if (lane == 0) produce<DP, false>(c, prm, &tmap_q, &tmap_k, &tmap_v, at);
  } else if (warp == 1) {
    if (lane == 0) issue<T, DP, false>(c, tmem_base, prm, at);
  } else {
    attend<T, DP, false>(c, tmem_base, prm, rows, at);
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (*c.again != kEnd && !*c.abort_flag) {
    ptx::tc_fence_after();
    at = second_pass<T, DP>(smem, tmem_base, prm, &tmap_q, &tmap_k, &tmap_v, at);
    ptx::tc_fence_before();
    __syncthreads();
  }
  if (*c.abort_flag) {
    settle<DP>(smem, at);
    __syncthreads();
  }
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// Tensor map over [tokens, heads, head_dim]: box of 64 elements, `box_heads`
// heads and `box_tokens` tokens, 128-byte swizzle, zeros outside.
inline bool make_map(CUtensorMap *map, const void *data, CUtensorMapDataType type, int64_t dim, int64_t heads,
                     int64_t tokens, int64_t head_stride, int64_t token_stride, int box_heads, int box_tokens) {
  tc::EncodeTiledFn fn = tc::encode_tiled_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  const cuuint32_t ones[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void *>(data), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline int64_t candidates_of(int64_t tokens, int64_t batch, int pair) { return tokens / pair + batch; }
inline int64_t plan_bytes(int64_t candidates, int64_t batch, int64_t kv_heads) {
  return (int64_t)sizeof(Plan) + candidates * ((int64_t)sizeof(Entry) + 4 * kv_heads) + batch * 4 * CLASSES;
}

template <typename T, int DP>
int launch_tiles(const Params &prm, const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, int64_t candidates,
                 cudaStream_t stream) {
  cudaError_t e = smem_optin<attention_kernel<T, DP>>(Layout<DP>::SMEM_BYTES);
  if (e != cudaSuccess) return (int)e;
  const int rc = launch_overlapped(plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, prm.p, candidates, prm.per_tile);
  if (rc != 0) return rc;
  const int64_t items = candidates * prm.p.kv_heads;
  const unsigned grid = (unsigned)(items < sm_count() ? items : sm_count());
  return launch_overlapped(attention_kernel<T, DP>, dim3(grid), dim3(THREADS), Layout<DP>::SMEM_BYTES, stream, tq, tk, tv,
                           prm);
}

// tc::kNotEligible where the operands do not meet the tensor-core kernel's layout.
template <typename T> int try_tiles(const Problem &p, int64_t workspace_bytes, cudaStream_t stream) {
  if constexpr (sizeof(T) != 2) {
    return tc::kNotEligible;
  } else {
    if (p.head_dim > 128 || p.group > BM || !(p.scale > 0.f) || p.k_tokens == 0) return tc::kNotEligible;
    if (p.q_dim != 1 || p.k_dim != 1 || p.v_dim != 1) return tc::kNotEligible;
    if (!rotary::aligned16(p.q) || !rotary::aligned16(p.k) || !rotary::aligned16(p.v)) return tc::kNotEligible;
    for (int64_t s : {p.q_token, p.q_head, p.k_token, p.k_head, p.v_token, p.v_head})
      if (s <= 0 || s % 8 != 0) return tc::kNotEligible;
    if (p.q_tokens > (1 << 30) || p.k_tokens > (1 << 30) || p.batch > (1 << 30)) return tc::kNotEligible;
    Params prm;
    prm.p = p;
    prm.per_tile = BM / p.group;
    const int64_t candidates = prm.candidates = candidates_of(p.q_tokens, p.batch, 2 * prm.per_tile);
    if (candidates * p.kv_heads > (1 << 30) || plan_bytes(candidates, p.batch, p.kv_heads) > workspace_bytes) return NT_B200_ERR_INVALID_ARGUMENT;
    CUtensorMap tq, tk, tv;
    const CUtensorMapDataType type = tc::tmap_dtype<T>();
    if (!make_map(&tq, p.q, type, p.head_dim, p.heads, p.q_tokens, p.q_head, p.q_token, p.group, prm.per_tile) ||
        !make_map(&tk, p.k, type, p.head_dim, p.kv_heads, p.k_tokens, p.k_head, p.k_token, 1, BN) ||
        !make_map(&tv, p.v, type, p.head_dim, p.kv_heads, p.k_tokens, p.v_head, p.v_token, 1, BN))
      return tc::kNotEligible;
    if (p.head_dim <= 64) return launch_tiles<T, 64>(prm, tq, tk, tv, candidates, stream);
    return launch_tiles<T, 128>(prm, tq, tk, tv, candidates, stream);
  }
}

}  // namespace prompt
}  // namespace nt

extern "C" int64_t nt_b200_prompt_attention_workspace_size(int64_t query_tokens, int64_t batch, int64_t heads,
                                                           int64_t kv_heads) {
  using namespace nt::prompt;
  if (query_tokens < 0 || batch < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0) return 0;
  const int64_t group = heads / kv_heads;
  const int pair = group > BM ? 2 : 2 * (int)(BM / group);
  return plan_bytes(candidates_of(query_tokens, batch, pair), batch, kv_heads);
}

extern "C" int nt_b200_prompt_attention(const NtB200PromptAttentionArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->query_tokens < 0 || a->key_tokens < 0 || a->batch < 0 || a->heads < 0 || a->kv_heads < 0 || a->head_dim < 0)
    return NT_B200_ERR_INVALID_ARGUMENT;
  if (!is_float_dtype((int)a->dtype) || !is_index_dtype(a->index_dtype)) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->query_tokens == 0 || a->batch == 0 || a->heads == 0 || a->head_dim == 0) return 0;
  if (a->kv_heads == 0 || a->heads % a->kv_heads != 0 || a->head_dim > prompt::kMostDim) return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->query || !a->output || !a->query_offsets || !a->key_offsets || (a->key_tokens > 0 && (!a->key || !a->value)) ||
      !a->workspace || (reinterpret_cast<uintptr_t>(a->workspace) & 31u) != 0 || a->heads > (1 << 30) ||
      !(a->scale == a->scale) ||
      a->workspace_bytes < nt_b200_prompt_attention_workspace_size(a->query_tokens, a->batch, a->heads, a->kv_heads))
    return NT_B200_ERR_INVALID_ARGUMENT;
  const int wide = a->index_dtype == NT_B200_INT64;
  prompt::Problem p{};
  p.q = a->query; p.k = a->key; p.v = a->value; p.o = a->output; p.lse = a->lse;
  p.q_offsets = {a->query_offsets, a->query_offsets_stride, wide};
  p.k_offsets = {a->key_offsets, a->key_offsets_stride, wide};
  p.q_tokens = a->query_tokens; p.k_tokens = a->key_tokens; p.batch = a->batch;
  p.q_token = a->query_strides[0]; p.q_head = a->query_strides[1]; p.q_dim = a->query_strides[2];
  p.k_token = a->key_strides[0]; p.k_head = a->key_strides[1]; p.k_dim = a->key_strides[2];
  p.v_token = a->value_strides[0]; p.v_head = a->value_strides[1]; p.v_dim = a->value_strides[2];
  p.o_token = a->output_strides[0]; p.o_head = a->output_strides[1]; p.o_dim = a->output_strides[2];
  p.l_token = a->lse_strides[0]; p.l_head = a->lse_strides[1];
  p.heads = (int)a->heads; p.kv_heads = (int)a->kv_heads; p.group = (int)(a->heads / a->kv_heads);
  p.head_dim = (int)a->head_dim;
  p.causal = a->is_causal != 0;
  p.scale = (float)(a->scale * 1.4426950408889634);
  p.workspace = a->workspace;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    const int rc = prompt::try_tiles<scalar_t>(p, a->workspace_bytes, s);
    if (rc != tc::kNotEligible) return rc;
    const int64_t blocks = (p.q_tokens * p.heads + 3) / 4;
    if (blocks > (1LL << 31) - 1) return NT_B200_ERR_INVALID_ARGUMENT;
    prompt::rows_kernel<scalar_t><<<(unsigned)blocks, 128, 0, s>>>(p);
    return launch_status();
  });
}
