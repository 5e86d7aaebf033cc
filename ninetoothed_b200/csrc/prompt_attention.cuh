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
// bfloat16 elements: 600-640 us, 860-915 TFLOP/s.
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
  float qv[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < p.head_dim ? to_f(q[d * p.q_dim]) : 0.f;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int64_t t = 0; t < limit; ++t) {
    const T *k = static_cast<const T *>(p.k) + (k0 + t) * p.k_token + g * p.k_head;
    const T *v = static_cast<const T *>(p.v) + (k0 + t) * p.v_token + g * p.v_head;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.head_dim) dot = fmaf(qv[e], to_f(k[(lane + 32 * e) * p.k_dim]), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = dot * p.scale, m_new = fmaxf(m, s);
    const float alpha = exp2f(m - reference(m_new)), w = exp2f(s - reference(m_new));
    l = l * alpha + w;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < p.head_dim) acc[e] = fmaf(w, to_f(v[(lane + 32 * e) * p.v_dim]), acc[e] * alpha);
    m = m_new;
  }
  T *out = static_cast<T *>(p.o) + token * p.o_token + h * p.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    if (d < p.head_dim) out[d * p.o_dim] = from_f<T>(limit > 0 ? acc[e] / l : 0.f);
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
  int32_t first, total;
  int32_t head;         // of an item; unused in the list
};
// The workspace: Plan, the entries, then an int32 for each sequence and class.
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
  static constexpr int SMEM_BYTES = ROWS_OFF + BM * 4;
  static_assert(96 + 16 * RING <= 240, "barrier slots");
  static_assert(SMEM_BYTES <= 232448, "shared memory of a CTA");
};

struct Params {
  Problem p;
  int per_tile;  // queries of a tile
};

// A row again, key by key on the CUDA cores, from its final maximum.  An
// infinity or NaN in the value of a key that the row does not see makes the
// row's MMA sums NaN (0 * inf): such rows come here.
template <typename T>
__device__ __noinline__ void row_again(const Problem &p, int k0, int64_t token, int head, int limit, float m, float f,
                                       T *out) {
  const T *q = static_cast<const T *>(p.q) + token * p.q_token + head * p.q_head;
  const int g = head / p.group;
  for (int c = 0; c < p.head_dim; c += 16) {
    float acc[16] = {};
    for (int t = 0; t < limit; ++t) {
      const T *k = static_cast<const T *>(p.k) + (int64_t)(k0 + t) * p.k_token + g * p.k_head;
      const T *v = static_cast<const T *>(p.v) + (int64_t)(k0 + t) * p.v_token + g * p.v_head;
      float dot = 0.f;
      for (int d = 0; d < p.head_dim; ++d) dot = fmaf(to_f(q[d]), to_f(k[d]), dot);
      const float w = exp2f(dot * p.scale - m);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < p.head_dim) acc[i] = fmaf(w, to_f(v[c + i]), acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c + i < p.head_dim) out[(c + i) * p.o_dim] = from_f<T>(acc[i] * f);
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
  const uint32_t ctrl = base + L::CTRL_OFF;
  // barriers (8 bytes each), per tile t unless noted
  auto q_full = [&](int t) { return ctrl + 8u * t; };        // Q_t landed
  auto q_free = [&](int t) { return ctrl + 16 + 8u * t; };   // the item's last Q_t K^T done
  auto s_full = [&](int t) { return ctrl + 32 + 8u * t; };   // S_t of a key block in tensor memory
  auto p_full = [&](int t) { return ctrl + 48 + 8u * t; };   // P_t written, O_t rescaled
  auto o_done = [&](int t) { return ctrl + 64 + 8u * t; };   // the item's last P_t V done
  auto o_free = [&](int t) { return ctrl + 80 + 8u * t; };   // O_t read out
  auto slot_full = [&](int s) { return ctrl + 96 + 8u * s; };
  auto slot_empty = [&](int s) { return ctrl + 96 + 8u * RING + 8u * s; };
  // items, two in turn: handed over, taken by the MMA issuer and the softmax warps
  auto item_full = [&](int s) { return ctrl + 248 + 8u * s; };
  auto item_empty = [&](int s) { return ctrl + 264 + 8u * s; };
  volatile int4 *item_slots = reinterpret_cast<volatile int4 *>(smem + L::CTRL_OFF + 288);
  volatile uint32_t *tmem_base_ptr = reinterpret_cast<volatile uint32_t *>(smem + L::CTRL_OFF + 240);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + L::CTRL_OFF + 244);

  const Problem &p = prm.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_tile = prm.per_tile;

  if (threadIdx.x == 0) {
    for (int t = 0; t < TILES; ++t) {
      ptx::mbar_init(q_full(t), 1);
      ptx::mbar_init(q_free(t), 1);
      ptx::mbar_init(s_full(t), 1);
      ptx::mbar_init(p_full(t), 4);  // a warp's lanes arrive as one
      ptx::mbar_init(o_done(t), 1);
      ptx::mbar_init(o_free(t), 4);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(item_full(s), 1);
      ptx::mbar_init(item_empty(s), 1 + SOFTMAX_WARPS);
    }
    for (int s = 0; s < RING; ++s) {
      ptx::mbar_init(slot_full(s), 1);
      ptx::mbar_init(slot_empty(s), 1);
    }
    *abort_flag = 0;
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
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t *>(tmem_base_ptr)), TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  wait_prior_grid();
  const uint32_t tmem_base = *tmem_base_ptr;
  auto tmem_s = [&](int t) { return tmem_base + (uint32_t)(t * BN); };
  auto tmem_o = [&](int t) { return tmem_base + (uint32_t)(TILES * BN + t * 128); };

  // The CTA's i-th item (queries 0: no more), once it was handed over; false
  // where the wait gave up.  The caller then lets go of it.
  auto take_item = [&](int i, Entry &e) {
    if (!ptx::mbar_wait(item_full(i & 1), (uint32_t)(i >> 1) & 1u, abort_flag)) return false;
    const volatile int4 *at = item_slots + 2 * (i & 1);
    e.q0 = at[0].x; e.queries = at[0].y; e.k0 = at[0].z; e.keys = at[0].w;
    e.limit0 = at[1].x; e.head = at[1].w;
    return true;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      bool ok = true;
      int r = 0;             // ring items so far
      int used[TILES] = {};  // items so far that had tile t
      const uint32_t q_bytes = (uint32_t)(per_tile * p.group * 128 * L::ATOMS);
      // Items count along the list by a sequence's entries of one class, among
      // them head by head, in it entry by entry.
      Plan *plan = static_cast<Plan *>(p.workspace);
      const Entry *list = reinterpret_cast<const Entry *>(plan + 1);
      const int64_t num_items = (int64_t)plan->count * p.kv_heads;
      // The next item is fetched in three steps, each waiting for the one before
      // only when it comes to its turn among this item's loads.
      int64_t next = 0;
      Entry any{}, ahead{};
      auto fetch = [&](int step) {
        if (step == 0) {
          next = atomicAdd(&plan->next, 1);
        } else if (step == 1) {
          any = Entry{};
          if (next < num_items) any = list[next / p.kv_heads];  // of the same sequence and class
        } else {
          ahead = Entry{};
          if (next < num_items) {
            const int r = (int)(next - (int64_t)any.first * p.kv_heads), h = r / any.total;
            ahead = list[any.first + r - h * any.total];
            ahead.head = h;
          }
        }
      };
      for (int x = 0; x < 3; ++x) fetch(x);
      for (int i = 0; ok; ++i) {
        const Entry e = ahead;
        if (!ptx::mbar_wait(item_empty(i & 1), ((uint32_t)(i >> 1) & 1u) ^ 1u, abort_flag)) break;
        volatile int4 *to = item_slots + 2 * (i & 1);
        to[0].x = e.q0; to[0].y = e.queries; to[0].z = e.k0; to[0].w = e.keys;
        to[1].x = e.limit0; to[1].w = e.head;
        ptx::mbar_arrive(item_full(i & 1));
        if (e.queries == 0) break;
        fetch(0);
        const int h = e.head;
        const int n[TILES] = {blocks_of(e, 0, per_tile, p.causal), blocks_of(e, 1, per_tile, p.causal)};
        const int n_max = max(n[0], n[1]);
        for (int t = 0; t < TILES && ok; ++t) {
          if (n[t] == 0) continue;
          if (used[t] > 0 && !ptx::mbar_wait(q_free(t), (uint32_t)(used[t] - 1) & 1u, abort_flag)) { ok = false; break; }
          ++used[t];
          ptx::mbar_arrive_expect_tx(q_full(t), q_bytes);
          for (int x = 0; x < L::ATOMS; ++x)
            ptx::tma_load_3d(base + t * L::Q_BYTES + x * (BM * 128), &tmap_q, q_full(t), 64 * x, h * p.group,
                             e.q0 + t * per_tile);
        }
        for (int j = 0; j < 2 * n_max && ok; ++j, ++r) {  // K_0, V_0, K_1, V_1, ...
          const int slot = r % RING;
          if (!ptx::mbar_wait(slot_empty(slot), ((uint32_t)(r / RING) & 1u) ^ 1u, abort_flag)) { ok = false; break; }
          ptx::mbar_arrive_expect_tx(slot_full(slot), L::KV_BYTES);
          const CUtensorMap *map = (j & 1) ? &tmap_v : &tmap_k;
          for (int x = 0; x < L::ATOMS; ++x)
            ptx::tma_load_3d(base + L::RING_OFF + slot * L::KV_BYTES + x * (BN * 128), map, slot_full(slot), 64 * x, h,
                             e.k0 + (j >> 1) * BN);
          if (j == 4) fetch(1);
          if (j == 8) fetch(2);
        }
        if (2 * n_max <= 4) fetch(1);
        if (2 * n_max <= 8) fetch(2);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t fmt = tc::umma_format<T>();
      constexpr uint32_t idesc_qk = ptx::f16_idesc(fmt, 0, 0, BM, BN);  // B = keys, K-major
      constexpr uint32_t idesc_pv = ptx::f16_idesc(fmt, 0, 1, BM, DP);  // B = values, MN-major
      auto slot_addr = [&](int r) { return base + L::RING_OFF + (r % RING) * L::KV_BYTES; };
      auto wait_slot = [&](int r) { return ptx::mbar_wait(slot_full(r % RING), (uint32_t)(r / RING) & 1u, abort_flag); };
      auto issue_qk = [&](int t, int r) {
        const uint32_t kb = slot_addr(r);
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          const uint32_t qoff = (kk / 4) * (BM * 128) + (kk % 4) * 32, koff = (kk / 4) * (BN * 128) + (kk % 4) * 32;
          ptx::mma_f16_ss(tmem_s(t), ptx::sw128_desc(base + t * L::Q_BYTES + qoff, 16, 1024),
                          ptx::sw128_desc(kb + koff, 16, 1024), idesc_qk, kk > 0 ? 1u : 0u);
        }
        ptx::mma_commit(s_full(t));
      };
      auto issue_pv = [&](int t, int r, bool first) {
        const uint32_t vb = slot_addr(r);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk)
          ptx::mma_f16_ts(tmem_o(t), tmem_s(t) + (uint32_t)(kk * 8), ptx::sw128_desc(vb + kk * 16 * 128, BN * 128, 1024),
                          idesc_pv, (!first || kk > 0) ? 1u : 0u);
      };
      bool ok = true;
      int r = 0;             // ring position of the item's K_0
      int blk[TILES] = {};   // key blocks of tile t in earlier items
      int used[TILES] = {};  // earlier items that had tile t
      for (int i = 0; ok; ++i) {
        Entry e;
        if (!take_item(i, e) || e.queries == 0) break;
        ptx::mbar_arrive(item_empty(i & 1));
        const int n[TILES] = {blocks_of(e, 0, per_tile, p.causal), blocks_of(e, 1, per_tile, p.causal)};
        const int n_max = max(n[0], n[1]);
        ok = wait_slot(r);  // K_0
        for (int t = 0; t < TILES && ok; ++t) {
          if (n[t] == 0) continue;
          if (!ptx::mbar_wait(q_full(t), (uint32_t)used[t] & 1u, abort_flag)) { ok = false; break; }
          ptx::tc_fence_after();
          issue_qk(t, r);
          if (n[t] == 1) ptx::mma_commit(q_free(t));
        }
        if (!ok) break;
        ptx::mma_commit(slot_empty(r % RING));
        for (int j = 0; j < n_max && ok; ++j) {
          const int rv = r + 2 * j + 1, rk = r + 2 * j + 2;
          if (!wait_slot(rv)) { ok = false; break; }
          bool next_keys = false;
          for (int t = 0; t < TILES && ok; ++t) {
            if (j >= n[t]) continue;
            // P_t written also means that S_t was read: Q K^T may overwrite it
            if (!ptx::mbar_wait(p_full(t), (uint32_t)(blk[t] + j) & 1u, abort_flag)) { ok = false; break; }
            if (j == 0 && used[t] > 0 && !ptx::mbar_wait(o_free(t), (uint32_t)(used[t] - 1) & 1u, abort_flag)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after();
            issue_pv(t, rv, j == 0);
            if (j == n[t] - 1) ptx::mma_commit(o_done(t));
            if (j + 1 < n[t]) {
              if (!next_keys) {
                if (!wait_slot(rk)) { ok = false; break; }
                next_keys = true;
                ptx::tc_fence_after();
              }
              issue_qk(t, rk);
              if (j + 2 == n[t]) ptx::mma_commit(q_free(t));
            }
          }
          if (!ok) break;
          ptx::mma_commit(slot_empty(rv % RING));
          if (next_keys) ptx::mma_commit(slot_empty(rk % RING));
        }
        r += 2 * n_max;
        for (int t = 0; t < TILES; ++t) {
          blk[t] += n[t];
          used[t] += n[t] > 0;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax, rescaling, output
    const int t = (warp - 2) / 4, quarter = warp & 3;
    const int row = quarter * 32 + lane;  // row of the tile = lane of tensor memory
    const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
    bool ok = true;
    auto arrive_warp = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(bar);
    };
    const float c = p.scale;
    uint32_t s_turn = 0, o_turn = 0;
    // A block's scores fill a thread's registers: what an item's end needs is
    // read again there, and the item let go only then.
    for (int i = 0; ok; ++i) {
      int n_t, limit, sure;  // key blocks; keys that the row sees; keys that all rows see
      {
        Entry e;
        if (!__all_sync(0xffffffffu, take_item(i, e)) || e.queries == 0) break;
        n_t = blocks_of(e, t, per_tile, p.causal);
        limit = p.causal ? min(e.limit0 + t * per_tile + rows[row].x, e.keys) : e.keys;
        sure = p.causal ? min(e.limit0 + t * per_tile, e.keys) : e.keys;
      }
      if (n_t == 0) {
        arrive_warp(item_empty(i & 1));
        continue;
      }

      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_t; ++j) {
        if (!ptx::mbar_wait_warp(s_full(t), s_turn, abort_flag)) { ok = false; break; }
        s_turn ^= 1;
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
        const float block_top = top[0] * c;
        // the maximum moves only when a block passes it by 2^14 (bf16: 2^24):
        // P stays in its type's range and O is rescaled rarely
        const bool move = block_top > m + tc::attn::RescaleLog2<T>::value;
        const float m_new = move ? block_top : m;
        const float alpha = move ? exp2_fast(m - m_new) : 1.f;
        const float ref = reference(m_new);
        float sum[8] = {};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t packed[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const int k = half * 64 + 2 * x;
            const float p0 = exp2_fast(fmaf(s[k], c, -ref)), p1 = exp2_fast(fmaf(s[k + 1], c, -ref));
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
        arrive_warp(p_full(t));
      }
      if (!ok || !ptx::mbar_wait_warp(o_done(t), o_turn, abort_flag)) break;
      o_turn ^= 1;
      ptx::tc_fence_after();
      uint32_t o[DP];
#pragma unroll
      for (int x = 0; x < DP / 32; ++x)
        ptx::tmem_ld_32x32b_x32(tmem_o(t) + lane_base + (uint32_t)(x * 32), *reinterpret_cast<uint32_t(*)[32]>(&o[x * 32]));
      ptx::tmem_ld_wait();
      ptx::tc_fence_before();
      arrive_warp(o_free(t));
      Entry e;
      take_item(i, e);
      arrive_warp(item_empty(i & 1));
      const int query = t * per_tile + rows[row].x;
      if (query < e.queries && rows[row].x < per_tile) {
        const int64_t token = e.q0 + query;
        const int head = e.head * p.group + rows[row].y;
        const float f = l == 0.f ? 0.f : 1.f / l;
        T *out = static_cast<T *>(p.o) + token * p.o_token + (int64_t)head * p.o_head;
        float worst = 0.f;  // NaN or infinite if any element is
#pragma unroll
        for (int x = 0; x < DP; ++x) worst = fmaf(__uint_as_float(o[x]), 0.f, worst);
        if (!(worst == 0.f)) {
          row_again<T>(p, e.k0, token, head, limit, reference(m), f, out);
        } else if (p.head_dim == DP && p.o_dim == 1 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
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
          p.lse[token * p.l_token + (int64_t)head * p.l_head] = l == 0.f ? -INFINITY : (m + log2_fast(l)) * kLn2;
      }
    }
  }

  ptx::tc_fence_before();
  __syncthreads();
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
inline int64_t plan_bytes(int64_t candidates, int64_t batch) {
  return (int64_t)sizeof(Plan) + candidates * (int64_t)sizeof(Entry) + batch * 4 * CLASSES;
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
    const int64_t candidates = candidates_of(p.q_tokens, p.batch, 2 * prm.per_tile);
    if (candidates * p.kv_heads > (1 << 30) || plan_bytes(candidates, p.batch) > workspace_bytes) return NT_B200_ERR_INVALID_ARGUMENT;
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
  return plan_bytes(candidates_of(query_tokens, batch, pair), batch);
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
