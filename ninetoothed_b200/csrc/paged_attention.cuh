// Attention of a few new tokens of each sequence over a paged 8-bit cache:
//     s = (q . k_code) * (scale * key_scale[page])      for the keys a query sees
//     o = sum_j softmax(s)_j * value_scale[page_j] * v_code_j
//     lse = ln sum_j exp(s_j)
// Query i of `queries` sees the first length - queries + 1 + i cached tokens; one
// that sees none gets o = 0 and lse = -inf.  All math is base 2 in fp32.
//
// Bound by memory: each cached byte is read once (grouped query heads share
// it), 2 * length * kv_heads * head_dim bytes a sequence, for 4 heads_per_group
// flops a byte.
//
// The work is one line of 32-token steps: sequence by sequence, within it
// (kv head, row tile) unit by unit.  The line is cut into equal pieces, one a
// CTA, and a piece into equal shares, one a warp, so that any mix of lengths
// keeps every SM busy to the end and no warp waits for another; a unit that
// lies in one share is finished there.  Of the others, a CTA joins at its end
// what neighbouring warps hold of one unit, and leaves its parts (o, m, l) in a
// workspace; the CTA that brings a unit's last part joins them, always in the
// line's order.  A second kernel for that cost 3 us of the device's time and 6 us
// of the host's a call.  Warps that took the steps of a unit in turn and joined
// at the end of every unit took 108 us where this takes 27 us for 256 units of up
// to 2047 tokens: short units cost a CTA as much as long ones.
//
// Measured (32 query heads on 8 key/value heads of 128 e4m3 elements, 64-token
// pages): 6 x 131072 tokens 285-290 us, 5.6 TB/s of the cache; 64 sequences of 1
// to 8192 tokens 121 us, 4.7 TB/s; one of 1023 tokens 14 us.  Loads alone, without
// the arithmetic, take 266 us for the first.
//
// A warp's step, S^T = K Q^T and O^T += V^T P^T on 16x8x16 tensor-core
// instructions with the cached tokens (head elements) as the 16 rows and 8
// query rows as the columns: with the 4 to 8 query heads of a group that wastes
// nothing, where queries as the 16 rows would.  Any order of the contracted
// elements is as good as another, so each lane takes 16 neighbouring bytes of a
// key as its share of the head, and 16 neighbouring elements of four tokens'
// values: loads are whole 16-byte words and bytes are paired with one permute.
// Each warp copies for itself (cp.async) through a ring of its own, so nothing
// waits for another warp.
//
// Codes become fp16 (exact for both types).  A query row is scaled by a power
// of two to a largest element in [2^14, 2^15): bfloat16 rows fit, and elements
// down to 2^-28 of the largest keep all their bits (scaled to [1, 2), elements
// beside an outlier of 60000 lost theirs).  P is rounded to fp16 (11 bits; the
// MMA takes its two operands in one type, and the codes are in fp16) relative to
// the largest weight value_scale * p of its row, so neither scales far apart nor a
// long tail lose bits that count.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "paged_append.cuh"
#include "ptx.cuh"

namespace nt {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_fast(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x where it is finite or +inf; 0 for the -inf of a row that has seen no key.
__device__ __forceinline__ float reference(float m) { return m == -INFINITY ? 0.f : m; }

struct Attention {
  const void *query;
  void *out;
  float *lse;  // or null
  const uint8_t *key, *value;
  const float *key_scale, *value_scale;
  IndexArray lengths, block_table;
  int64_t table_row_stride;
  int64_t q_batch, q_token, q_head, q_dim, o_batch, o_token, o_head, o_dim, l_batch, l_token, l_head;
  int64_t k_page, k_head, k_token, v_page, v_head, v_token, ks_page, ks_head, vs_page, vs_head;
  int64_t pages;
  int capacity;  // tokens a block table row can hold
  int batch, queries, heads, kv_heads, group, head_dim, page;
  int page_groups;          // page / 16
  uint64_t page_reciprocal; // ceil(2^36 / page_groups)
  int rows, row_tiles;      // queries * group; tiles of them
  int q_vector;             // queries can be read 16 bytes at a time
  int bf16;                 // query and output elements: bfloat16, else fp16
  float scale;              // softmax scale * log2 e
  unsigned long long *counters; // workspace: one a warp, then
  float *parts;                 // two parts a warp
  unsigned long long tag;       // of this call, 48 bits
};

// The cached length of a sequence, in its block table's capacity.
__device__ __forceinline__ int cached_length(const Attention &a, int64_t b) {
  const int64_t n = a.lengths[b];
  if (n < 0 || n > a.capacity) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return n < 0 ? 0 : a.capacity;
  }
  return (int)n;
}

// The page of column `column` of sequence b's block table, or -1.
__device__ __forceinline__ int page_of(const Attention &a, int64_t b, int64_t column) {
  const int64_t at = b * a.table_row_stride + column * a.block_table.stride;
  const int64_t id = a.block_table.wide ? static_cast<const int64_t *>(a.block_table.data)[at]
                                        : (int64_t) static_cast<const int32_t *>(a.block_table.data)[at];
  return id >= 0 && id < a.pages ? (int)id : -1;
}

// ---------------------------------------------------------------- any type
// A warp a query row: head elements dealt over the lanes, one key at a time.  64
// sequences of 1 to 8192 tokens, 32 query heads on 8: 26 ms at 256 elements, 23 ms
// at 192, where the tensor-core kernel takes 121 us at 128.
// Every FAR_KEYS keys the sums go over to others: beside a weight of 1, what weights
// of 2^-25 and less add one by one is lost.
constexpr int kMostDim = 256, FAR_KEYS = 256;
template <typename T, typename C>
__global__ void __launch_bounds__(128) attention_rows_kernel(Attention a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)a.batch * a.queries * a.heads) return;
  const int h = (int)(row % a.heads), i = (int)(row / a.heads % a.queries);
  const int64_t b = row / a.heads / a.queries;
  const int64_t limit = cached_length(a, b) - a.queries + 1 + i;
  const T *q = static_cast<const T *>(a.query) + b * a.q_batch + i * a.q_token + h * a.q_head;
  constexpr int E = kMostDim / 32;
  float qv[E], acc[E], far[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < a.head_dim ? to_f(q[d * a.q_dim]) : 0.f;
    acc[e] = far[e] = 0.f;
  }
  const int g = h / a.group;
  float m = -INFINITY, l = 0.f, l_far = 0.f;
  for (int64_t t = 0; t < limit; ++t) {
    const int id = page_of(a, b, t / a.page);
    if (id < 0) {
      record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
      continue;
    }
    const uint8_t *k = a.key + id * a.k_page + g * a.k_head + (t % a.page) * a.k_token;
    const uint8_t *v = a.value + id * a.v_page + g * a.v_head + (t % a.page) * a.v_token;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < a.head_dim) dot = fmaf(qv[e], decode<C>(k[lane + 32 * e]), dot);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float s = dot * (a.scale * a.key_scale[id * a.ks_page + g * a.ks_head]);
    const float vs = a.value_scale[id * a.vs_page + g * a.vs_head];
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
    const float p = exp2f(s - reference(m));
    l += p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < a.head_dim) acc[e] = fmaf(p, decode<C>(v[lane + 32 * e]) * vs, acc[e]);
    if (t % FAR_KEYS == FAR_KEYS - 1) {
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
  T *out = static_cast<T *>(a.out) + b * a.o_batch + i * a.o_token + h * a.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    if (d < a.head_dim) out[d * a.o_dim] = from_f<T>(l == 0.f ? 0.f : (acc[e] + far[e]) / l);
  }
  if (a.lse && lane == 0) a.lse[b * a.l_batch + i * a.l_token + h * a.l_head] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// ---------------------------------------------------------------- tensor cores
constexpr int STEP = 32;
constexpr int Q_TOP = 14;  // a query row's largest element, as a power of two
// Steps of a CTA at least: fewer would be parts to join rather than work.  One
// sequence of 1023 e4m3 tokens, 8 key/value heads of 128: 14.6 us at 2, 13.9 at 4,
// 15.4 at 6.
constexpr int LEAST_STEPS = 4;
// A unit's start and end (its queries, its output) take a warp about three steps'
// time, and count as that in the line where a warp's share is BUSY_STEPS or more:
// a share of nine short units took 113 us beside 80 of long ones.  With 4 queries
// each of 16 sequences of up to 2047 tokens, 16 heads of 64, at (UNIT_STEPS,
// BUSY_STEPS) of (2, 8) 31.2 us, (2, 2) 29.6, (3, 2) 26.9.  Shares below that are
// bound by latency and are cut by what there is to read.
constexpr int UNIT_STEPS = 3, BUSY_STEPS = 2;
// A block table row's tokens that are looked at; a page's size.  With them the
// block table column of a 16-token group is one multiplication: for g < 2^27
// groups and d = page / 16 <= 2^8, floor(g ceil(2^36 / d) / 2^36) = floor(g / d).
constexpr int64_t MOST_TOKENS = (1LL << 31) - 64;
constexpr int MOST_PAGE = 4096;

__device__ __forceinline__ void copy_async16(uint32_t to, const void *from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async4(uint32_t to, const void *from, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 load_shared16(uint32_t from) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
  return v;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t from) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(from) : "memory");
  return v;
}
__device__ __forceinline__ void store_shared4(uint32_t to, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(v) : "memory");
}

// D[16 x 8] += A[16 x 16] B[16 x 8], fp16 in, fp32 accumulator.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of 16-bit elements held two a lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// Four codes (bytes 0-3 of w) as two pairs of fp16.
template <typename C> __device__ __forceinline__ void to_halves(uint32_t w, uint32_t &lo, uint32_t &hi);
template <> __device__ __forceinline__ void to_halves<__nv_fp8_e4m3>(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)w));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(w >> 16)));
}
template <> __device__ __forceinline__ void to_halves<int8_t>(uint32_t w, uint32_t &lo, uint32_t &hi) {
  // 0x64xx is the fp16 1024 + xx, so with the sign bit flipped (xx = code +
  // 128) a subtraction of 1152 leaves the code, exactly.
  const uint32_t u = w ^ 0x80808080u;
  uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
  const uint32_t bias = 0x64806480u;  // 1152, twice
  __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<const __half2 *>(&bias));
  __half2 y = __hsub2(*reinterpret_cast<__half2 *>(&b), *reinterpret_cast<const __half2 *>(&bias));
  lo = *reinterpret_cast<uint32_t *>(&x);
  hi = *reinterpret_cast<uint32_t *>(&y);
}

// Stands for the key scale of a page outside the pool (a NaN that no scale is):
// nobody sees its tokens.
constexpr uint32_t kNoPage = 0xffffffffu;

// Tokens of a 16-token group in the order of the MMAs' rows: row r holds token
// r / 2 (even r) or 4 + r / 2 (odd r), and so on from 8.  A lane's four values
// (rows 2 c4, 2 c4 + 1, 2 c4 + 8, 2 c4 + 9) are then those of the tokens c4, 4 +
// c4, 8 + c4 and 12 + c4: four neighbouring rows of shared memory a load.
__device__ __forceinline__ int token_of(int row) { return (row >> 1 & 3) + 4 * (row & 1) + (row & 8); }
__device__ __forceinline__ int row_at(int token) { return 2 * (token & 3) + (token >> 2 & 1) + (token & 8); }
// Where a row's 16-byte word w lies in shared memory: moved so that a quarter
// warp's (8-byte words: half a warp's) loads meet every bank once.  Keys are
// kept in MMA order and read 8 rows by 4 words, values in token order and read
// 4 rows by 2 words.
template <int DP> __device__ __forceinline__ int key_place(int row, int w) { return DP == 128 ? w ^ ((row & 1) << 2) : w; }
template <int DP> __device__ __forceinline__ int value_place(int token, int w) {
  return DP == 128 ? w ^ ((token & 3) << 1) : w ^ (token & 2);
}

template <int DP, int NT> struct Layout {
  static constexpr int ROWS = 8 * NT;
  // One column tile: 12 warps of up to 168 registers, three a scheduler, to cover
  // each other's latencies, each with two steps in flight (8 warps reach 0.8 of
  // their rate; 16 warps of 128 registers spill and have room for a step and a
  // half each: 0.88).  Two column tiles hold twice the accumulators: 8 warps.
  static constexpr int WARPS = NT == 1 ? 12 : 8;
  static constexpr int V_WORD = DP / 8;           // bytes of a token's value a lane takes
  static constexpr int SLOTS = 4;                 // of a warp's ring: keys, values of a step, of the next
  static constexpr int CODES = STEP * DP;
  static constexpr int SLOT = CODES + 16;         // + the step's scales (two of keys, two of values), with the keys
  static constexpr int RING = SLOTS * SLOT;
  static constexpr int SMEM = WARPS * RING;
  // a part in the workspace: o [ROWS][DP], then m, l, mo [ROWS]
  static constexpr int PART = ROWS * (DP + 3);
  static_assert(SMEM + 3072 <= 232448, "shared memory of a CTA");
  static_assert(PART * 4 <= RING, "a warp's part fits its ring");
};

// A value's NaN reaches only the rows that see its token, but 0 * NaN in an MMA
// would reach every row.  In steps where rows differ in what they see, NaN
// codes are taken out of a 16-token group's value words (token 4 i + c4 in v[i],
// as loaded) and set into the rows' O here.
template <int DP, int NT>
__device__ __forceinline__ void separate_nans(uint32_t (&v)[4][DP / 32], float (&o)[NT][DP / 16][4],
                                              const int (&limit)[NT][2], int token0) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int w = 0; w < DP / 32; ++w) any |= (v[i][w] & 0x7f7f7f7fu) + 0x01010101u;
  if (!__any_sync(0xffffffffu, (any & 0x80808080u) != 0)) return;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t mask = 0;  // bit d: element d of the lane's share is NaN
#pragma unroll
    for (int w = 0; w < DP / 32; ++w) {
      const uint32_t nan = ((v[i][w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
      v[i][w] &= ~((nan >> 7) * 0xffu);
#pragma unroll
      for (int e = 0; e < 4; ++e) mask |= (nan >> (8 * e + 7) & 1u) << (4 * w + e);
    }
    for (int c = 0; c < 4; ++c) {
      const uint32_t other = __shfl_sync(0xffffffffu, mask, (lane & ~3) | c);
      const int token = token0 + 4 * i + c;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int t = 0; t < DP / 16; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (token < limit[nt][e & 1] && (other >> (2 * t + (e >> 1)) & 1u)) o[nt][t][e] = NAN;
    }
  }
}

// The cut of a line of `total` steps: `cta` steps a CTA, `warp` a warp; `extra`
// steps of each unit stand for its start and end.  (The host has seen to it that
// the line's steps fit 31 bits.)
struct Cut {
  int total, cta, warp, extra;
};
// Where a walk along the line stands: before step s of a unit of sequence b (n
// steps a unit, `extra` among them), `left` steps to go in the share.
struct Walk {
  int left, b, length, n, unit, s;
};
// Steps [s0, s1) of one unit; those from `real` on are extra.
struct Segment {
  int length, b, head, tile, s0, s1, n, real;
};

__host__ __device__ __forceinline__ int steps_of(int64_t length) { return (int)((length + STEP - 1) / STEP); }
__device__ __forceinline__ int line_steps(int length, int extra) { return length > 0 ? steps_of(length) + extra : 0; }

__device__ __forceinline__ bool next_segment(const Attention &a, int extra, Walk &w, Segment &g) {
  if (w.left <= 0) return false;
  while (w.n == 0 || w.unit >= a.kv_heads * a.row_tiles) {
    if (++w.b >= a.batch) return false;
    w.length = cached_length(a, w.b);
    w.n = line_steps(w.length, extra);
    w.unit = w.s = 0;
  }
  g.b = w.b;
  g.length = w.length;
  g.n = w.n;
  g.head = w.unit / a.row_tiles;
  g.tile = w.unit % a.row_tiles;
  g.s0 = w.s;
  const int take = min(w.left, w.n - w.s);
  g.s1 = g.s0 + take;
  g.real = min(g.s1, g.n - extra);
  w.left -= take;
  w.s += take;
  if (w.s == w.n) {
    w.s = 0;
    ++w.unit;
  }
  return true;
}

// Steps of one unit of sequence b; 0 past the last sequence.
__device__ __forceinline__ int unit_steps(const Attention &a, int b, int extra) {
  const int64_t n = b < a.batch ? a.lengths[b] : 0;
  return n <= 0 ? 0 : line_steps((int)(n < a.capacity ? n : a.capacity), extra);
}

__device__ __forceinline__ Cut cut_line(const Attention &a, int ctas, int warps) {
  Cut c{0, 0, 0, 0};
  int some = 0;  // sequences with keys
  for (int b = threadIdx.x & 31; b < a.batch; b += 32) {
    const int n = unit_steps(a, b, 0);
    c.total += n;
    some += n > 0;
  }
  const int units = a.kv_heads * a.row_tiles;
  c.total = __reduce_add_sync(0xffffffffu, c.total) * units;
  if (c.total / (ctas * warps) >= BUSY_STEPS) {
    c.extra = UNIT_STEPS;
    c.total += UNIT_STEPS * units * (int)__reduce_add_sync(0xffffffffu, some);
  }
  c.cta = max((int)(((unsigned)c.total + ctas - 1) / ctas), LEAST_STEPS);
  c.warp = (c.cta + warps - 1) / warps;
  return c;
}

// Query and output elements are fp16 or, with `bf16`, bfloat16: a run-time flag,
// as only the ends of a unit depend on it.
__device__ __forceinline__ float element(uint16_t bits, int bf16) {
  return bf16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
}
__device__ __forceinline__ uint16_t element_bits(float x, int bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}

// The maxima that P is taken against move only when a score passes them by LEAD
// (base 2): a step's scores are compared in their own threads, and the reduction
// over the threads of a row and the rescaling of O happen rarely.  P is kept RISE
// above them, so that its largest, 2^(LEAD + RISE), stays in fp16's range and what
// a long tail adds does not fall among fp16's subnormals: tokens with 2^-25.5 of
// the largest weight were lost in the share that holds it at (8, 0), 15 % of what
// 65536 of them give.
constexpr float LEAD = 6.f, RISE = 9.f;
// A lane's sum of weights goes over to a second one every FAR_STEPS steps: beside
// a weight of 1, weights of 2^-25 and less added one by one are lost.
constexpr int FAR_STEPS = 64;

// N neighbouring elements of a finished row: o = acc * 2^(mo - RISE - m) / l, and the
// row's lse.
template <int N>
__device__ __forceinline__ void write_row(const Attention &a, int64_t b, int h, int row, int d, const float (&acc)[N],
                                          float m, float l, float mo) {
  if (row >= a.rows || d >= a.head_dim) return;
  const int i = row / a.group, hq = h * a.group + row % a.group;
  const float f = l == 0.f ? 0.f : exp2_fast(reference(mo) - RISE - reference(m)) / l;
  uint16_t *out = static_cast<uint16_t *>(a.out) + b * a.o_batch + i * a.o_token + (int64_t)hq * a.o_head + d * a.o_dim;
  if (a.o_dim == 1 && (reinterpret_cast<uintptr_t>(out) & (2 * N - 1)) == 0) {
    struct alignas(2 * N < 16 ? 2 * N : 16) Pack { uint16_t v[N]; } pack;
#pragma unroll
    for (int e = 0; e < N; ++e) pack.v[e] = element_bits(acc[e] * f, a.bf16);
    *reinterpret_cast<Pack *>(out) = pack;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e * a.o_dim] = element_bits(acc[e] * f, a.bf16);
  }
  if (a.lse && d == 0)
    a.lse[b * a.l_batch + i * a.l_token + (int64_t)hq * a.l_head] = l == 0.f ? -INFINITY : (m + log2_fast(l)) * kLn2;
}

// A lane's elements of one of its rows, in order.
template <int DP, int NT>
__device__ __forceinline__ void row_of(const float (&o)[NT][DP / 16][4], int nt, int u, float (&acc)[DP / 8]) {
#pragma unroll
  for (int t = 0; t < DP / 16; ++t) {
    acc[2 * t] = o[nt][t][u];
    acc[2 * t + 1] = o[nt][t][u + 2];
  }
}

// A warp's part of a unit: o [ROWS][DP], then m, l, mo of each row.
template <int DP, int NT>
__device__ __forceinline__ void write_part(float *part, const float (&o)[NT][DP / 16][4], const float (&m)[NT][2],
                                           const float (&l)[NT][2], const float (&mo)[NT][2]) {
  const int lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int row = nt * 8 + 2 * c4 + u;
      float acc[DP / 8];
      row_of<DP, NT>(o, nt, u, acc);
#pragma unroll
      for (int e = 0; e < DP / 8; e += 4)
        *reinterpret_cast<float4 *>(part + row * DP + n8 * (DP / 8) + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
      if (n8 == 0) {
        float *st = part + 8 * NT * DP + row * 3;
        st[0] = m[nt][u];
        st[1] = l[nt][u];
        st[2] = mo[nt][u];
      }
    }
}

// A unit that several shares hold: n steps (0: none) from step `first` of the
// line; `only`: it is all that the warp's share has.
struct Shared {
  int first, b, head, tile, n;
  bool only;
};

// Where the CTAs' parts of a unit are: the first CTA's run at `head` (the run
// begins with the warp that holds the unit's first step, in that warp's second
// place, unless its share begins with the unit), the runs of the CTAs k0 + 1 ..
// k1 in their first warps' first places, and, if the unit ends inside a later
// warp's share of CTA k1, that warp's first place (`tail`, else < 0).
struct Parts {
  int counter, k0, k1, head, tail;
  __device__ int count() const { return k1 - k0 + 1 + (tail >= 0); }
  __device__ int place(int j, int warps) const { return j == 0 ? head : j <= k1 - k0 ? 2 * (k0 + j) * warps : tail; }
};
__device__ __forceinline__ Parts parts_of(const Shared &u, const Cut &c, int warps) {
  Parts p;
  p.k0 = (unsigned)u.first / (unsigned)c.cta;
  const int lo = u.first - p.k0 * c.cta, w0 = (unsigned)lo / (unsigned)c.warp, last = u.first + u.n - 1;
  p.counter = p.k0 * warps + w0;
  p.head = 2 * p.counter + (lo == w0 * c.warp ? 0 : 1);
  p.k1 = (unsigned)last / (unsigned)c.cta;
  const int hi = last - p.k1 * c.cta, w1 = (unsigned)hi / (unsigned)c.warp;
  const int share_end = min(min((w1 + 1) * c.warp, c.cta), c.total - p.k1 * c.cta);
  const bool later = w1 > (p.k1 == p.k0 ? w0 : 0);
  p.tail = later && hi + 1 < share_end ? 2 * (p.k1 * warps + w1) : -1;
  return p;
}

// Counts one more of a unit's parts as written; true for the last.  A counter is
// the call's 48-bit tag and a count; one without the tag, whatever the workspace
// held, is first set to the tag and zero (once: whoever else tries finds it
// changed).  The last to come leaves it without the tag, for a graph that
// replays the call with the same tag.
__device__ __forceinline__ bool arrive(unsigned long long *counter, unsigned long long tag, int expected) {
  const unsigned long long now = *reinterpret_cast<volatile unsigned long long *>(counter);
  if ((now >> 16) != tag) atomicCAS(counter, now, tag << 16);
  if ((int)(atomicAdd(counter, 1ull) & 0xffffu) + 1 != expected) return false;
  *reinterpret_cast<volatile unsigned long long *>(counter) = 0;
  return true;
}

// Joins a unit's parts and writes its rows; a warp of the block takes a row.
// (This runs once a call, mostly from a cold instruction cache: small code.)
template <int DP, int NT>
__device__ __forceinline__ void join_unit(const Attention &a, const Shared &u, const Parts &where) {
  using L = Layout<DP, NT>;
  const int lane = threadIdx.x & 31, parts = where.count();
  constexpr int LANES = DP / 4, AT_ONCE = 32 / LANES;  // lanes of a part's row; parts read side by side
#pragma unroll 1
  for (int r = threadIdx.x >> 5; r < L::ROWS; r += L::WARPS) {
    float top = -INFINITY, top_o = -INFINITY, sum = 0.f, acc[4] = {};
    // 32 parts at a time, each chunk's maxima joined to those before
#pragma unroll 1
    for (int j0 = 0; j0 < parts; j0 += 32) {
      float m = -INFINITY, l = 0.f, mo = -INFINITY;
      const float *p = nullptr;
      if (j0 + lane < parts) {
        p = a.parts + (int64_t)where.place(j0 + lane, L::WARPS) * L::PART;
        m = __ldcg(p + L::ROWS * DP + r * 3);
        l = __ldcg(p + L::ROWS * DP + r * 3 + 1);
        mo = __ldcg(p + L::ROWS * DP + r * 3 + 2);
        p += r * DP;
      }
      float m_new = m, mo_new = mo;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) {
        m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, x));
        mo_new = fmaxf(mo_new, __shfl_xor_sync(0xffffffffu, mo_new, x));
      }
      m_new = fmaxf(m_new, top);
      mo_new = fmaxf(mo_new, top_o);
      sum = sum * exp2_fast(top - reference(m_new)) + l * exp2_fast(m - reference(m_new));
      const float alpha = exp2_fast(top_o - reference(mo_new)), f = exp2_fast(mo - reference(mo_new));
      top = m_new;
      top_o = mo_new;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= alpha;
      const int count = min(parts - j0, 32);
#pragma unroll 8
      for (int j = 0; j < count; j += AT_ONCE) {
        const int from = j + lane / LANES;
        const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(p), from);
        const float g = __shfl_sync(0xffffffffu, f, from);
        if (at != 0) {
          const float4 v = __ldcg(reinterpret_cast<const float4 *>(at) + lane % LANES);
          acc[0] = fmaf(v.x, g, acc[0]); acc[1] = fmaf(v.y, g, acc[1]);
          acc[2] = fmaf(v.z, g, acc[2]); acc[3] = fmaf(v.w, g, acc[3]);
        }
      }
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (AT_ONCE == 2) {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
    }
    if (lane < LANES) write_row(a, u.b, u.head, u.tile * L::ROWS + r, lane * 4, acc, top, sum, top_o);
  }
}

// SPLIT: pages of an odd number of 16-token groups, so that a step may lie in
// two pages with a scale each.
template <typename C, int DP, int NT, bool SPLIT>
__global__ void __launch_bounds__(Layout<DP, NT>::WARPS * 32, 1) attention_kernel(const __grid_constant__ Attention a) {
  using L = Layout<DP, NT>;
  constexpr int WARPS = L::WARPS;
  constexpr int KS = DP / 16, OT = DP / 16;  // contraction steps of QK; 16-element tiles of O
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ Shared runs[WARPS], joins[2 * WARPS];
  __shared__ Parts places[2 * WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * L::RING;
  wait_prior_grid();
  allow_dependent_launch();

  // this warp's share of the line
  const Cut cut = cut_line(a, gridDim.x, WARPS);
  int first = min((int64_t)blockIdx.x * cut.cta + warp * cut.warp, (int64_t)cut.total);
  const int end = min((int64_t)cut.total, min((int64_t)first + cut.warp, (int64_t)(blockIdx.x + 1) * cut.cta));
  Walk start{};
  start.left = max(end - first, 0);
  if (start.left > 0) {
    // the sequence that holds step `first`, 32 sequences at a time
    const int units = a.kv_heads * a.row_tiles;
    for (int b0 = 0;; b0 += 32) {
      const int n = unit_steps(a, b0 + lane, cut.extra) * units;
      int up = n;  // inclusive sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += x;
      }
      const int which = __popc(__ballot_sync(0xffffffffu, up <= first));  // sums are nondecreasing
      if (which == 32) {
        first -= __shfl_sync(0xffffffffu, up, 31);
        continue;
      }
      first -= __shfl_sync(0xffffffffu, up - n, which);
      start.b = b0 + which;
      break;
    }
    start.length = cached_length(a, start.b);
    start.n = line_steps(start.length, cut.extra);
    start.unit = (unsigned)first / (unsigned)start.n;
    start.s = first - start.unit * start.n;
  }

  // ------------------------------------------------------------ loads ahead
  // A ring of four slots, keys and values of two steps; each is loaded again,
  // two steps on, as soon as it has been read.
  Walk ahead = start;
  Segment lseg{};
  bool lmore = true;
  int lstep = 0;           // the step to load
  int id0 = -1, id1 = -1;  // pages of its two 16-token groups
  int group0 = 0;          // the first group's place in its page
  // This lane's share of a 16-token group: whole rows, neighbouring words by
  // neighbouring lanes, four (head_dim up to 64: eight) tokens an instruction.
  // (Copied as the lanes read them, by lanes of four tokens in turn, values came
  // from memory in 32-byte pieces: 318 us where this takes 283 us for 6 x 131072
  // tokens.)
  constexpr int ROW_WORDS = DP / 16, COPIES = 16 * ROW_WORDS / 32;
  const int k_row = lane / ROW_WORDS, k_word = lane % ROW_WORDS;  // of the first copy
  const uint32_t k_token = (uint32_t)a.k_token, v_token = (uint32_t)a.v_token;
  auto k_place = [&](int i) {
    const int row = row_at(k_row + i * (32 / ROW_WORDS));
    return ring + (uint32_t)(row * DP + key_place<DP>(row, k_word) * 16);
  };
  const uint32_t k_even = k_place(0), k_odd = k_place(1);  // places of copies 0 and 1; two copies on, eight rows on
  const uint32_t v_place = ring + (uint32_t)(k_row * DP + value_place<DP>(k_row, k_word) * 16);
  const uint8_t *key_head = nullptr, *value_head = nullptr;  // of the load segment
  const float *scale_head = nullptr;                         // even lanes: key scales, odd: value scales
  const uint32_t scale_page = (uint32_t)(lane & 1 ? a.vs_page : a.ks_page);
  auto find_pages = [&]() {
    const int g = lstep * (STEP / 16);
    const int col = (int)(((uint64_t)(uint32_t)g * a.page_reciprocal) >> 36);
    group0 = g - col * a.page_groups;
    id0 = page_of(a, lseg.b, col);
    if (SPLIT) {
      id1 = id0;
      if (group0 + 1 == a.page_groups) id1 = (g + 1) * 16 < lseg.length ? page_of(a, lseg.b, col + 1) : -1;
    }
  };
  auto enter = [&]() {  // the next segment with something to load
    do {
      lmore = next_segment(a, cut.extra, ahead, lseg);
      if (!lmore) return;
      lstep = lseg.s0;
    } while (lstep >= lseg.real);
    key_head = a.key + lseg.head * a.k_head + k_row * k_token + k_word * 16;
    value_head = a.value + lseg.head * a.v_head + k_row * v_token + k_word * 16;
    scale_head = lane & 1 ? a.value_scale + lseg.head * a.vs_head : a.key_scale + lseg.head * a.ks_head;
    find_pages();
  };
  auto next_step = [&]() {
    if (!lmore) return;
    if (++lstep < lseg.real) find_pages();
    else enter();
  };
  auto page_known = [&](int g) { return (SPLIT && g == 1 ? id1 : id0) >= 0; };
  // the live tokens of a group, its page (0 where it has none) and slot in it
  auto group_of = [&](int g, int &live, uint32_t &id, uint32_t &slot) {
    live = lseg.length - (lstep * STEP + 16 * g);
    const int page = SPLIT && g == 1 ? id1 : id0;
    if (page < 0) {
      if (live > 0) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
      live = 0;
    }
    id = page < 0 ? 0 : page;
    slot = (g == 0 ? group0 : SPLIT && group0 + 1 == a.page_groups ? 0 : group0 + 1) * 16;
  };
  auto load_keys = [&](int at) {
    if (lmore) {
      constexpr int EIGHT = DP == 128 ? 2 : 1;  // copies for eight tokens
      auto to = [&](int g, int i) {
        return (EIGHT == 2 && (i & 1) ? k_odd : k_even) + at * L::SLOT + g * 16 * DP + i / EIGHT * 8 * DP;
      };
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        int live;
        uint32_t id, slot;
        group_of(g, live, id, slot);
        const uint8_t *k = key_head + (uint64_t)id * (uint32_t)a.k_page + (uint64_t)slot * k_token;
        if (live >= 16 && a.head_dim == DP) {
#pragma unroll
          for (int i = 0; i < COPIES; ++i)
            copy_async16(to(g, i), k + i * (uint64_t)(32 / ROW_WORDS * k_token), true);
        } else {  // zeros for what is not there; its address stays inside
#pragma unroll
          for (int i = 0; i < COPIES; ++i) {
            const bool valid = k_word * 16 < a.head_dim && k_row + i * (32 / ROW_WORDS) < live;
            copy_async16(to(g, i), valid ? k + i * (uint64_t)(32 / ROW_WORDS * k_token) : a.key, valid);
          }
        }
        if ((SPLIT || g == 0) && lane < 2) {
          const uint32_t place = ring + at * L::SLOT + L::CODES + (lane * 2 + g) * 4;
          if (lane == 0 && !page_known(g)) store_shared4(place, kNoPage);
          else copy_async4(place, scale_head + (uint64_t)id * scale_page, live > 0);
        }
      }
    }
    copy_commit();
  };
  auto load_values = [&](int at) {
    if (lmore) {
      const uint32_t to = v_place + at * L::SLOT;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        int live;
        uint32_t id, slot;
        group_of(g, live, id, slot);
        const uint8_t *v = value_head + (uint64_t)id * (uint32_t)a.v_page + (uint64_t)slot * v_token;
        const bool all = live >= 16 && a.head_dim == DP;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) {
          const uint8_t *src = v + i * (uint64_t)(32 / ROW_WORDS * v_token);
          const bool valid = all || (k_word * 16 < a.head_dim && k_row + i * (32 / ROW_WORDS) < live);
          copy_async16(to + g * 16 * DP + i * 512, valid ? src : a.value, valid);
        }
      }
    }
    copy_commit();
  };

  enter();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    load_keys(2 * i);
    load_values(2 * i + 1);
    next_step();
  }
  int at = 0;  // slot of the step's keys; its values are in the next
  // this lane's elements (V_WORD from n8 V_WORD on) of token c4
  const uint32_t v_read =
      ring + (uint32_t)(c4 * DP + value_place<DP>(c4, n8 * L::V_WORD / 16) * 16 + n8 * L::V_WORD % 16);

  // rows of sequences without keys
  for (int64_t b = (int64_t)blockIdx.x * WARPS + warp; b < a.batch; b += (int64_t)gridDim.x * WARPS) {
    if (cached_length(a, b) > 0) continue;
    const float zero[1] = {0.f};
    for (int64_t x = lane; x < (int64_t)a.kv_heads * a.rows * a.head_dim; x += 32) {
      const int64_t r = x / a.head_dim;
      write_row(a, b, (int)(r / a.rows), (int)(r % a.rows), (int)(x % a.head_dim), zero, -INFINITY, 0.f, -INFINITY);
    }
  }

  Walk here = start;
  Segment seg;
  Shared before{}, held{};  // parts of the unit from the share before, and of the last
  while (next_segment(a, cut.extra, here, seg)) {
    const int row0 = seg.tile * L::ROWS;

    // Q: lane (n8, c4) holds row n8's elements 16 c4 .. + 15 of each 64, as
    // the B operand of contraction step 4 x + w: bytes 4w .. 4w + 3 of a key's
    // 16-byte word x
    uint32_t qf[NT][KS][2];
    float q_unit[NT];  // the power of two a row was divided by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + n8;
      const bool valid = row < a.rows;
      const int i = valid ? row / a.group : 0, hq = seg.head * a.group + (valid ? row % a.group : 0);
      const uint16_t *q = static_cast<const uint16_t *>(a.query) + seg.b * a.q_batch + i * a.q_token + hq * a.q_head;
      float x[DP / 4], top = 0.f;
      if (a.q_vector) {
#pragma unroll
        for (int e = 0; e < DP / 4; e += 8) {
          const int d = (e / 16) * 64 + 16 * c4 + e % 16;
          uint4 chunk = make_uint4(0, 0, 0, 0);
          if (valid && d < a.head_dim) chunk = *reinterpret_cast<const uint4 *>(q + d);
          const uint32_t w[4] = {chunk.x, chunk.y, chunk.z, chunk.w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            x[e + 2 * y] = element((uint16_t)w[y], a.bf16);
            x[e + 2 * y + 1] = element((uint16_t)(w[y] >> 16), a.bf16);
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < DP / 4; ++e) {
          const int d = (e / 16) * 64 + 16 * c4 + e % 16;
          x[e] = valid && d < a.head_dim ? element(q[d * a.q_dim], a.bf16) : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < DP / 4; ++e) top = fmaxf(top, fabsf(x[e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int exponent = (int)(__float_as_uint(top) >> 23) - Q_TOP;  // biased, of the power
      exponent = exponent < 1 ? 1 : exponent > 253 ? 253 : exponent;
      q_unit[nt] = __uint_as_float((uint32_t)exponent << 23);
      // with the softmax scale's sign, so that a larger score is a larger weight
      const float inv = copysignf(__uint_as_float((uint32_t)(254 - exponent) << 23), a.scale);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int e = (s / 4) * 16 + (s % 4) * 4;
        qf[nt][s][0] = half2_bits(x[e] * inv, x[e + 1] * inv);
        qf[nt][s][1] = half2_bits(x[e + 2] * inv, x[e + 3] * inv);
      }
    }
    // of the rows 2 c4 and 2 c4 + 1 of each tile: score factor, maxima, sum,
    // keys seen
    float factor[NT][2], m[NT][2], mo[NT][2], l[NT][2], l_far[NT][2];
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        factor[nt][u] = fabsf(a.scale) * __shfl_sync(0xffffffffu, q_unit[nt], (2 * c4 + u) * 4);
        limit[nt][u] = seg.length - a.queries + 1 + (row0 + nt * 8 + 2 * c4 + u) / a.group;
        m[nt][u] = mo[nt][u] = -INFINITY;
        l[nt][u] = l_far[nt][u] = 0.f;
      }
    const int sure = seg.length - a.queries + 1 + row0 / a.group;  // keys that every row sees
    float o[NT][OT][4] = {};

    for (int step = seg.s0; step < seg.real; ++step) {
      copy_wait<3>();  // all but this step's values and the next step
      __syncwarp();    // other lanes' copies
      const uint32_t from = ring + at * L::SLOT, from_v = v_read + (at + 1) * L::SLOT;

      float s[2][NT][4] = {};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int x = 0; x < DP / 64; ++x) {
          const uint32_t word = from + (g * 16 + n8) * DP + key_place<DP>(n8, 4 * x + c4) * 16;
          const uint4 k0 = load_shared16(word), k1 = load_shared16(word + 8 * DP);
          const uint32_t lo[4] = {k0.x, k0.y, k0.z, k0.w}, hi[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            uint32_t a0, a1, a2, a3;
            to_halves<C>(lo[w], a0, a2);
            to_halves<C>(hi[w], a1, a3);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(s[g][nt], a0, a1, a2, a3, qf[nt][x * 4 + w][0], qf[nt][x * 4 + w][1]);
          }
        }
      }
      // scales: two of the keys, two of the values
      const uint4 scales = load_shared16(from + L::CODES);
      const float ks[2] = {__uint_as_float(scales.x), __uint_as_float(SPLIT ? scales.y : scales.x)};
      float lv[2];
      lv[0] = log2_fast(__uint_as_float(scales.z));
      lv[1] = SPLIT ? log2_fast(__uint_as_float(scales.w)) : lv[0];
      const int t0 = step * STEP;
      const bool masked = t0 + STEP > sure;
      const bool gone[2] = {scales.x == kNoPage, (SPLIT ? scales.y : scales.x) == kNoPage};
      // scores in base 2 are s * unit; where some are masked they are multiplied
      // out first
      float unit[2][NT][2];
      bool passed = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int u = 0; u < 2; ++u) unit[g][nt][u] = factor[nt][u] * ks[g];
        if (masked) {
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[g][nt][e] = t0 + 16 * g + token_of(n8) + 8 * (e >> 1) < limit[nt][e & 1] ? s[g][nt][e] * unit[g][nt][e & 1] : -INFINITY;
#pragma unroll
          for (int g = 0; g < 2; ++g) unit[g][nt][0] = unit[g][nt][1] = 1.f;
        }
        if (gone[0] || gone[1]) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!gone[g]) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[g][nt][e] = -INFINITY;
            unit[g][nt][0] = unit[g][nt][1] = 1.f;
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float b0 = fmaxf(s[0][nt][u], s[0][nt][u + 2]) * unit[0][nt][u];
          const float b1 = fmaxf(s[1][nt][u], s[1][nt][u + 2]) * unit[1][nt][u];
          passed |= fmaxf(b0, b1) > m[nt][u] + LEAD || fmaxf(b0 + lv[0], b1 + lv[1]) > mo[nt][u] + LEAD;
        }
      }
      const bool move = __any_sync(0xffffffffu, passed);
      load_keys(at);  // every lane has read this step's keys and scales
      if (move) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float b0 = fmaxf(s[0][nt][u], s[0][nt][u + 2]) * unit[0][nt][u];
            const float b1 = fmaxf(s[1][nt][u], s[1][nt][u + 2]) * unit[1][nt][u];
            float top = fmaxf(b0, b1), top_o = fmaxf(b0 + lv[0], b1 + lv[1]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
              top_o = fmaxf(top_o, __shfl_xor_sync(0xffffffffu, top_o, x));
            }
            const float m_new = fmaxf(m[nt][u], top), mo_new = fmaxf(mo[nt][u], top_o);
            const float fade = exp2_fast(m[nt][u] - reference(m_new));
            l[nt][u] *= fade;
            l_far[nt][u] *= fade;
            const float alpha = exp2_fast(mo[nt][u] - reference(mo_new));
            m[nt][u] = m_new;
            mo[nt][u] = mo_new;
#pragma unroll
            for (int t = 0; t < OT; ++t) {
              o[nt][t][u] *= alpha;
              o[nt][t][u + 2] *= alpha;
            }
          }
      }
      uint32_t pf[2][NT][2];  // P^T: MMA rows 2 c4, 2 c4 + 1 (and + 8) of query row n8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = reference(m[nt][0]), r1 = reference(m[nt][1]);
        const float w0 = reference(mo[nt][0]) - RISE, w1 = reference(mo[nt][1]) - RISE;
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float x0 = s[g][nt][2 * r], x1 = s[g][nt][2 * r + 1], u0 = unit[g][nt][0], u1 = unit[g][nt][1];
            l[nt][0] += exp2_fast(fmaf(x0, u0, -r0));
            l[nt][1] += exp2_fast(fmaf(x1, u1, -r1));
            pf[g][nt][r] = transpose8x8(half2_bits(exp2_fast(fmaf(x0, u0, lv[g] - w0)), exp2_fast(fmaf(x1, u1, lv[g] - w1))));
          }
      }
      copy_wait<3>();  // all but the next step and the keys after it
      __syncwarp();
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t v[4][L::V_WORD / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t word = from_v + (g * 4 + i) * 4 * DP;
          if constexpr (DP == 128) {
            const uint4 x = load_shared16(word);
            v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
          } else {
            const uint2 x = load_shared8(word);
            v[i][0] = x.x; v[i][1] = x.y;
          }
        }
        if (std::is_same<C, __nv_fp8_e4m3>::value && masked && a.queries > 1)
          separate_nans<DP, NT>(v, o, limit, t0 + 16 * g);
#pragma unroll
        for (int t = 0; t < OT; ++t) {
          const uint32_t select = t & 1 ? 0x7362 : 0x5140;
          uint32_t a0, a1, a2, a3;
          to_halves<C>(__byte_perm(v[0][t / 2], v[1][t / 2], select), a0, a1);
          to_halves<C>(__byte_perm(v[2][t / 2], v[3][t / 2], select), a2, a3);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][t], a0, a1, a2, a3, pf[g][nt][0], pf[g][nt][1]);
        }
      }
      __syncwarp();  // every lane has read this step's values
      load_values(at + 1);
      next_step();
      at ^= 2;
      if (step % FAR_STEPS == FAR_STEPS - 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            l_far[nt][u] += l[nt][u];
            l[nt][u] = 0.f;
          }
      }
    }

#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        l[nt][u] += l_far[nt][u];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][u] += __shfl_xor_sync(0xffffffffu, l[nt][u], x);
      }
    if (seg.s0 == 0 && seg.s1 == seg.n) {  // a whole unit
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float acc[L::V_WORD];
          row_of<DP, NT>(o, nt, u, acc);
          write_row(a, seg.b, seg.head, row0 + nt * 8 + 2 * c4 + u, n8 * L::V_WORD, acc, m[nt][u], l[nt][u], mo[nt][u]);
        }
      continue;
    }
    const Shared unit{end - here.left - seg.s1, seg.b, seg.head, seg.tile, seg.n, here.left + (seg.s1 - seg.s0) == start.left};
    if (here.left > 0) {
      before = unit;
      write_part<DP, NT>(a.parts + 2 * ((int64_t)blockIdx.x * WARPS + warp) * L::PART, o, m, l, mo);
    } else {  // kept for the CTA's join
      held = unit;
      write_part<DP, NT>(reinterpret_cast<float *>(smem + warp * L::RING), o, m, l, mo);
    }
  }

  // ------------------------------------------------------------ the CTA's join
  // A run: a warp's last segment and the warps after it that have nothing but
  // the same unit.  Its first warp adds up the others'.
  if (lane == 0) {
    runs[warp] = held;
    joins[2 * warp].n = joins[2 * warp + 1].n = 0;
  }
  __syncthreads();
  const bool leads = held.n > 0 && !(warp > 0 && held.only && runs[warp - 1].n > 0 && runs[warp - 1].first == held.first);
  if (leads) {
    int last = warp;
    while (last + 1 < WARPS && runs[last + 1].n > 0 && runs[last + 1].only && runs[last + 1].first == held.first) ++last;
    const int row = lane / (32 / L::ROWS);  // ROWS divides 32: lanes of a row share its elements
    float *part = a.parts + (2 * ((int64_t)blockIdx.x * WARPS + warp) + (held.only ? 0 : 1)) * L::PART;
    const float *in = reinterpret_cast<const float *>(smem + warp * L::RING);
    constexpr int NEXT = L::RING / 4, STATS = L::ROWS * DP;
    float top = -INFINITY, top_o = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int w = 0; w <= last - warp; ++w) {
      const float *st = in + w * NEXT + STATS + row * 3;
      const float m_new = fmaxf(top, st[0]);
      sum = sum * exp2_fast(top - reference(m_new)) + st[1] * exp2_fast(st[0] - reference(m_new));
      top = m_new;
      top_o = fmaxf(top_o, st[2]);
    }
#pragma unroll 1
    for (int d = lane % (32 / L::ROWS) * 4; d < DP; d += 128 / L::ROWS) {
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int w = 0; w <= last - warp; ++w) {
        const float f = exp2_fast(in[w * NEXT + STATS + row * 3 + 2] - reference(top_o));
        const float4 v = *reinterpret_cast<const float4 *>(in + w * NEXT + row * DP + d);
        acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
      }
      *reinterpret_cast<float4 *>(part + row * DP + d) = acc;
    }
    if (lane % (32 / L::ROWS) == 0) {
      part[STATS + row * 3] = top;
      part[STATS + row * 3 + 1] = sum;
      part[STATS + row * 3 + 2] = top_o;
    }
  }

  // ------------------------------------------------------------ the units' join
  // lanes 0 and 1: the run, the part of the unit from the share before
  __threadfence();
  __syncwarp();
  const Shared mine = lane == 0 ? held : before;
  if (lane < 2 && mine.n > 0 && (leads || lane == 1)) {
    const Parts where = parts_of(mine, cut, WARPS);
    if (arrive(a.counters + where.counter, a.tag, where.count())) {
      joins[2 * warp + lane] = mine;
      places[2 * warp + lane] = where;
      __threadfence();
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2 * WARPS; ++i)
    if (joins[i].n > 0) join_unit<DP, NT>(a, joins[i], places[i]);
}

template <typename C, int DP, int NT, bool SPLIT>
int launch_split(Attention a, cudaStream_t stream) {
  using L = Layout<DP, NT>;
  cudaError_t e = smem_optin<attention_kernel<C, DP, NT, SPLIT>>(L::SMEM);
  if (e != cudaSuccess) return (int)e;
  a.row_tiles = (a.rows + L::ROWS - 1) / L::ROWS;
  return launch_overlapped(attention_kernel<C, DP, NT, SPLIT>, dim3((unsigned)sm_count()), dim3(L::WARPS * 32), L::SMEM, stream,
                           a);
}
template <typename C, int DP, int NT>
int launch_tiles(const Attention &a, cudaStream_t stream) {
  return a.page_groups % 2 ? launch_split<C, DP, NT, true>(a, stream) : launch_split<C, DP, NT, false>(a, stream);
}

// Counters of a workspace: one for each warp of up to 512 SMs.
constexpr int64_t COUNTERS = 512 * 12;

// A tag that no other call of the process has: a counter through an invertible
// mix, so that it looks like nothing that a workspace may have held before.
inline unsigned long long call_tag() {
  static std::atomic<unsigned long long> calls{0};
  constexpr unsigned long long mask = (1ull << 48) - 1;
  unsigned long long x = calls.fetch_add(1, std::memory_order_relaxed) + 1;
  x = (x * 0x9e3779b97f4a7c15ull) & mask;
  x ^= x >> 25;
  return (x * 0xbf58476d1ce4e5b9ull) & mask;
}

template <typename T, typename C>
int launch_attention(const Attention &a, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    // 32-bit strides within a pool of pages
    bool small = true;
    for (int64_t x : {a.k_page, a.v_page, a.k_token * 32, a.v_token * 32, a.ks_page, a.vs_page})
      small = small && x >= 0 && x < (1LL << 32);
    small = small && a.k_token * a.page < (1LL << 32) && a.v_token * a.page < (1LL << 32);
    // and a line of steps that 31 bits count
    small = small && (double)a.batch * a.kv_heads * ((a.rows + 7) / 8) * (a.capacity / STEP + 1 + UNIT_STEPS) < 2e9;
    if (a.head_dim <= 128 && small && sm_count() <= 512) {
      const bool one = a.rows <= 8;
      if (a.head_dim <= 64)
        return one ? launch_tiles<C, 64, 1>(a, stream) : launch_tiles<C, 64, 2>(a, stream);
      return one ? launch_tiles<C, 128, 1>(a, stream) : launch_tiles<C, 128, 2>(a, stream);
    }
  }
  const int64_t blocks = ((int64_t)a.batch * a.queries * a.heads + 3) / 4;
  if (blocks > (1LL << 31) - 1) return NT_B200_ERR_INVALID_ARGUMENT;
  attention_rows_kernel<T, C><<<(unsigned)blocks, 128, 0, stream>>>(a);
  return launch_status();
}

}  // namespace paged
}  // namespace nt

extern "C" int64_t nt_b200_paged_attention_workspace_size(void) {
  using namespace nt::paged;
  // two parts a warp of the largest layout; the CTAs of a launch are the SMs
  constexpr int64_t one = (int64_t)Layout<128, 1>::WARPS * Layout<128, 1>::PART;
  constexpr int64_t two = (int64_t)Layout<128, 2>::WARPS * Layout<128, 2>::PART;
  return COUNTERS * 8 + 2 * (int64_t)nt::sm_count() * (one > two ? one : two) * (int64_t)sizeof(float);
}

extern "C" int nt_b200_paged_attention(const NtB200PagedAttentionArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->batch < 0 || a->queries < 0 || a->heads < 0 || a->table_columns < 0) return NT_B200_ERR_INVALID_ARGUMENT;
  if (!is_float_dtype((int)a->dtype) || !is_index_dtype(a->index_dtype)) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->batch == 0 || a->queries == 0 || a->heads == 0) return 0;
  const NtB200PagedCache &c = a->cache;
  const int rc = paged::check_cache(c);
  if (rc != 0) return rc;
  if (c.kv_heads == 0 || a->heads % c.kv_heads != 0 || c.head_dim > paged::kMostDim) return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->query || !a->output || !a->lengths || (a->table_columns > 0 && !a->block_table) || !a->workspace ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 15u) != 0 ||
      a->workspace_bytes < nt_b200_paged_attention_workspace_size() || a->batch > (1 << 30) ||
      a->queries > (1 << 30) || a->queries * a->heads > (1 << 30) || a->table_columns > (1LL << 40) || !(a->scale == a->scale))
    return NT_B200_ERR_INVALID_ARGUMENT;
  const int wide = a->index_dtype == NT_B200_INT64;
  paged::Attention p{};
  p.query = a->query;
  p.out = a->output;
  p.lse = a->lse;
  p.key = static_cast<const uint8_t *>(c.key);
  p.value = static_cast<const uint8_t *>(c.value);
  p.key_scale = c.key_scale;
  p.value_scale = c.value_scale;
  p.lengths = {a->lengths, a->lengths_stride, wide};
  p.block_table = {a->block_table, a->block_table_strides[1], wide};
  p.table_row_stride = a->block_table_strides[0];
  p.q_batch = a->query_strides[0]; p.q_token = a->query_strides[1]; p.q_head = a->query_strides[2]; p.q_dim = a->query_strides[3];
  p.o_batch = a->output_strides[0]; p.o_token = a->output_strides[1]; p.o_head = a->output_strides[2]; p.o_dim = a->output_strides[3];
  p.l_batch = a->lse_strides[0]; p.l_token = a->lse_strides[1]; p.l_head = a->lse_strides[2];
  p.k_page = c.key_strides[0]; p.k_head = c.key_strides[1]; p.k_token = c.key_strides[2];
  p.v_page = c.value_strides[0]; p.v_head = c.value_strides[1]; p.v_token = c.value_strides[2];
  p.ks_page = c.key_scale_strides[0]; p.ks_head = c.key_scale_strides[1];
  p.vs_page = c.value_scale_strides[0]; p.vs_head = c.value_scale_strides[1];
  p.pages = c.pages;
  const int64_t capacity = a->table_columns * c.page;
  p.capacity = (int)(capacity < paged::MOST_TOKENS ? capacity : paged::MOST_TOKENS);
  p.page_groups = (int)(c.page / 16);
  p.page_reciprocal = ((1ull << 36) + p.page_groups - 1) / p.page_groups;
  p.batch = (int)a->batch; p.queries = (int)a->queries; p.heads = (int)a->heads; p.kv_heads = (int)c.kv_heads;
  p.group = (int)(a->heads / c.kv_heads);
  p.head_dim = (int)c.head_dim;
  p.page = (int)c.page;
  p.rows = (int)(a->queries * p.group);
  p.bf16 = a->dtype == NT_B200_BFLOAT16;
  p.q_vector = p.q_dim == 1 && p.q_batch % 8 == 0 && p.q_token % 8 == 0 && p.q_head % 8 == 0 && rotary::aligned16(p.query);
  p.scale = (float)(a->scale * 1.4426950408889634);
  p.counters = static_cast<unsigned long long *>(a->workspace);
  p.parts = reinterpret_cast<float *>(p.counters + paged::COUNTERS);
  p.tag = paged::call_tag();
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    if (c.code_dtype == NT_B200_INT8) return paged::launch_attention<scalar_t, int8_t>(p, s);
    return paged::launch_attention<scalar_t, __nv_fp8_e4m3>(p, s);
  });
}
