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
// CTA, so that any mix of lengths keeps every SM busy to the end; a unit that
// lies in one piece is finished there, the others leave their parts (o, m, l)
// in a workspace and a second kernel joins them.  Warps of a CTA take the steps
// of a unit in turn and are joined through shared memory at its end.
//
// A warp's step, S^T = K Q^T and O^T += V^T P^T on 16x8x16 tensor-core
// instructions with the cached tokens (head elements) as the 16 rows and 8
// query rows as the columns: with the 4 to 8 query heads of a group that wastes
// nothing, where queries as the 16 rows would.  Any order of the contracted
// elements is as good as another, so each lane takes 16 neighbouring bytes of a
// key as its share of the head, and 16 neighbouring elements of four tokens'
// values: loads are whole 16-byte words and bytes are paired with one permute.
// A lane reads from shared memory just what it copied there itself
// (cp.async), so the ring of stages needs no barrier.
//
// Codes become fp16 (exact for both types).  A query row is scaled by a power
// of two to a largest element in [1, 2), so that bfloat16 rows fit too; P is
// rounded to fp16 relative to the largest weight value_scale * p of its row, so
// neither scales far apart nor a long tail lose bits that count.
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
  int64_t pages, capacity;  // tokens a block table row can hold
  int batch, queries, heads, kv_heads, group, head_dim, page;
  int rows, row_tiles;      // queries * group; tiles of them
  float scale;              // softmax scale * log2 e
  float *parts;             // workspace: two parts a CTA
  int64_t least;            // fewest steps of a piece
  int whole;                // one CTA a unit, nothing to join
};

// The cached length of a sequence, in its block table's capacity.
__device__ __forceinline__ int64_t cached_length(const Attention &a, int64_t b) {
  const int64_t n = a.lengths[b];
  if (n < 0 || n > a.capacity) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return n < 0 ? 0 : a.capacity;
  }
  return n;
}

// The page of column `column` of sequence b's block table, or -1.
__device__ __forceinline__ int64_t page_of(const Attention &a, int64_t b, int64_t column) {
  const int64_t at = b * a.table_row_stride + column * a.block_table.stride;
  const int64_t id = a.block_table.wide ? static_cast<const int64_t *>(a.block_table.data)[at]
                                        : (int64_t) static_cast<const int32_t *>(a.block_table.data)[at];
  return id >= 0 && id < a.pages ? id : -1;
}

// ---------------------------------------------------------------- any type
// A warp a query row: head elements dealt over the lanes, one key at a time.
constexpr int kMostDim = 256;
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
  float qv[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    qv[e] = d < a.head_dim ? to_f(q[d * a.q_dim]) : 0.f;
    acc[e] = 0.f;
  }
  const int g = h / a.group;
  float m = -INFINITY, l = 0.f;
  for (int64_t t = 0; t < limit; ++t) {
    const int64_t id = page_of(a, b, t / a.page);
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
    const float m_new = fmaxf(m, s);
    const float alpha = exp2f(m - reference(m_new)), p = exp2f(s - reference(m_new));
    l = l * alpha + p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (lane + 32 * e < a.head_dim) acc[e] = fmaf(p, decode<C>(v[lane + 32 * e]) * vs, acc[e] * alpha);
    m = m_new;
  }
  T *out = static_cast<T *>(a.out) + b * a.o_batch + i * a.o_token + h * a.o_head;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane + 32 * e;
    if (d < a.head_dim) out[d * a.o_dim] = from_f<T>(limit > 0 ? acc[e] / l : 0.f);
  }
  if (a.lse && lane == 0) a.lse[b * a.l_batch + i * a.l_token + h * a.l_head] = limit > 0 ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// ---------------------------------------------------------------- tensor cores
constexpr int WARPS = 8, STEP = 32;

__device__ __forceinline__ void copy_async16(uint32_t to, const void *from, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t to, const void *from, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(valid ? 8 : 0) : "memory");
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
__device__ __forceinline__ float load_shared4(uint32_t from) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(from) : "memory");
  return v;
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

template <int DP, int NT> struct Layout {
  static constexpr int ROWS = 8 * NT;
  static constexpr int STAGES = NT == 1 ? 3 : 2;
  static constexpr int K_COPIES = DP / 64 * 4;              // 16-byte words a lane and step
  static constexpr int V_WORD = DP / 8;                     // bytes of a token's value a lane takes
  static constexpr int K_BYTES = STEP * DP, V_BYTES = STEP * DP;
  static constexpr int STAGE = K_BYTES + V_BYTES + 32;      // + 2 key scales, 2 value scales
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int PITCH = DP + 4;                      // of a row's partial output, in floats
  static constexpr int JOIN = WARPS * ROWS * PITCH * 4;
  static constexpr int STATS = WARPS * ROWS * 3 * 4;
  static constexpr int SMEM = RING + JOIN + STATS + 64;
  // a part in the workspace: o [ROWS][DP], then m, l, mo [ROWS]
  static constexpr int PART = ROWS * (DP + 3);
  static_assert(SMEM <= 232448, "shared memory of a CTA");
};

// A value's NaN reaches only the rows that see its token, but 0 * NaN in an MMA
// would reach every row.  In steps where rows differ in what they see, NaN
// codes are taken out of a 16-token group's value words (token 2 c4 + i % 2 +
// 8 (i / 2) in v[i], as loaded) and set into the rows' O here.
template <int DP, int NT>
__device__ __forceinline__ void separate_nans(uint32_t (&v)[4][DP / 32], float (&o)[NT][DP / 16][4],
                                              const int64_t (&limit)[NT][2], int64_t token0) {
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
      const int64_t token = token0 + 2 * c + (i & 1) + 8 * (i >> 1);
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

// Where a walk along the line of steps stands: sequence b, `at` steps into its
// units * n, `left` steps to go in the piece.
struct Walk {
  int64_t at, left, length;
  int b, n;  // n: steps of one unit of the sequence
};
struct Segment {  // steps [s0, s1) of one unit
  int64_t length;
  int b, unit, s0, s1, n;
};

__device__ __forceinline__ int steps_of(int64_t length) { return (int)((length + STEP - 1) / STEP); }

__device__ __forceinline__ bool next_segment(const Attention &a, Walk &w, Segment &g) {
  if (w.left <= 0) return false;
  const int units = a.kv_heads * a.row_tiles;
  while (w.at >= (int64_t)w.n * units) {
    w.at -= (int64_t)w.n * units;
    if (++w.b >= a.batch) return false;
    w.length = cached_length(a, w.b);
    w.n = steps_of(w.length);
  }
  g.b = w.b;
  g.length = w.length;
  g.n = w.n;
  g.unit = (int)(w.at / w.n);
  g.s0 = (int)(w.at - (int64_t)g.unit * w.n);
  const int64_t take = w.left < g.n - g.s0 ? w.left : g.n - g.s0;
  g.s1 = g.s0 + (int)take;
  w.at += take;
  w.left -= take;
  return true;
}

// Steps of all sequences below `end`, by a whole block (shared: one int64 a warp).
template <int THREADS>
__device__ __forceinline__ int64_t steps_below(const Attention &a, int64_t end, int64_t *shared) {
  int64_t sum = 0;
  for (int64_t b = threadIdx.x; b < end; b += THREADS) {
    const int64_t n = a.lengths[b];
    sum += n <= 0 ? 0 : steps_of(n < a.capacity ? n : a.capacity);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) sum += shared[i];
  return sum * a.kv_heads * a.row_tiles;
}

// Steps of a piece: total / pieces, at least `least`.
__device__ __forceinline__ int64_t piece_of(int64_t total, int64_t pieces, int64_t least) {
  const int64_t q = (total + pieces - 1) / pieces;
  return q > least ? q : least;
}

// Four elements of a finished row: o = acc * 2^(mo - m) / l, and its lse.
template <typename T>
__device__ __forceinline__ void write_row(const Attention &a, int64_t b, int h, int row, int d, const float (&acc)[4],
                                          float m, float l, float mo) {
  if (row >= a.rows || d >= a.head_dim) return;
  const int i = row / a.group, hq = h * a.group + row % a.group;
  const float f = l == 0.f ? 0.f : exp2_fast(reference(mo) - reference(m)) / l;
  T *out = static_cast<T *>(a.out) + b * a.o_batch + i * a.o_token + (int64_t)hq * a.o_head;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[(d + e) * a.o_dim] = from_f<T>(acc[e] * f);
  if (a.lse && d == 0)
    a.lse[b * a.l_batch + i * a.l_token + (int64_t)hq * a.l_head] = l == 0.f ? -INFINITY : (m + log2_fast(l)) * kLn2;
}

template <typename T, typename C, int DP, int NT>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_kernel(const __grid_constant__ Attention a) {
  using L = Layout<DP, NT>;
  constexpr int KS = DP / 16, OT = DP / 16;  // contraction steps of QK; 16-element tiles of O
  extern __shared__ __align__(16) uint8_t smem[];
  float *join = reinterpret_cast<float *>(smem + L::RING);
  float *stats = reinterpret_cast<float *>(smem + L::RING + L::JOIN);
  int64_t *reduce = reinterpret_cast<int64_t *>(smem + L::RING + L::JOIN + L::STATS);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n8 = lane >> 2, c4 = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * L::STAGES * L::STAGE;
  wait_prior_grid();
  allow_dependent_launch();

  // this CTA's piece of the line
  Walk start{};
  if (a.whole) {
    const int units = a.kv_heads * a.row_tiles;
    start.b = blockIdx.x / units;
    start.length = cached_length(a, start.b);
    start.n = steps_of(start.length);
    start.at = (int64_t)(blockIdx.x % units) * start.n;
    start.left = start.n;
  } else {
    const int64_t total = steps_below<WARPS * 32>(a, a.batch, reduce);
    const int64_t piece = piece_of(total, gridDim.x, a.least);
    int64_t first = blockIdx.x * piece;
    if (first >= total) return;
    start.left = total - first < piece ? total - first : piece;
    // the sequence that holds step `first`: 256 sequences at a time, each
    // warp's 32 summed, then the lanes of the warp that holds it
    const int units = a.kv_heads * a.row_tiles;
    for (int64_t b0 = 0;; b0 += WARPS * 32) {
      const int64_t b = b0 + threadIdx.x;
      int64_t n = b < a.batch ? a.lengths[b] : 0;
      n = n <= 0 ? 0 : (int64_t)steps_of(n < a.capacity ? n : a.capacity) * units;
      int64_t up = n;  // inclusive sum over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += x;
      }
      __syncthreads();
      if (lane == 31) reduce[warp] = up;
      __syncthreads();
      int64_t base = 0;
      int found = -1;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        if (found < 0) {
          if (first < base + reduce[i]) found = i;
          else base += reduce[i];
        }
      }
      if (found < 0) {
        first -= base;
        continue;
      }
      __syncthreads();
      if (warp == found) {
        const unsigned past = __ballot_sync(0xffffffffu, base + up <= first);
        const int which = __popc(past);  // sums are nondecreasing
        const int64_t before = __shfl_sync(0xffffffffu, up - n, which);
        if (lane == 0) {
          reduce[0] = b0 + warp * 32 + which;
          reduce[1] = first - base - before;
        }
      }
      __syncthreads();
      start.b = (int)reduce[0];
      start.at = reduce[1];
      break;
    }
    start.length = cached_length(a, start.b);
    start.n = steps_of(start.length);
  }

  // ------------------------------------------------------------ loads ahead
  Walk ahead = start;
  Segment lseg{};
  int lstep = 0;
  bool lmore = next_segment(a, ahead, lseg);
  lstep = lseg.s0 + warp;
  int64_t id0 = -1, id1 = -1;  // pages of the next step to load
  auto find_pages = [&]() {
    while (lmore && lstep >= lseg.s1) {
      lmore = next_segment(a, ahead, lseg);
      lstep = lseg.s0 + warp;
    }
    if (!lmore) return;
    const int64_t t = (int64_t)lstep * STEP;
    const int64_t col = t / a.page;
    id0 = page_of(a, lseg.b, col);
    const int64_t col1 = t % a.page + 16 == a.page ? col + 1 : col;
    id1 = t + 16 < lseg.length ? (col1 == col ? id0 : page_of(a, lseg.b, col1)) : -1;
  };
  auto issue = [&](int stage) {
    if (lmore) {
      const int64_t t0 = (int64_t)lstep * STEP;
      const int h = lseg.unit / a.row_tiles;
      const uint32_t to = ring + stage * L::STAGE;
      const int slot = (int)(t0 % a.page);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int64_t base = t0 + 16 * g;
        int64_t id = g == 0 ? id0 : id1;
        const int64_t live64 = lseg.length - base;
        int live = live64 > 16 ? 16 : (int)live64;  // tokens of the group in the cache
        if (live > 0 && id < 0) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
        if (id < 0) { live = 0; id = 0; }
        const int in_page = g == 0 ? slot : (slot + 16 == a.page ? 0 : slot + 16);
        const uint8_t *k = a.key + id * a.k_page + (int64_t)h * a.k_head + (int64_t)in_page * a.k_token;
        const uint8_t *v = a.value + id * a.v_page + (int64_t)h * a.v_head + (int64_t)in_page * a.v_token;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int x = 0; x < DP / 64; ++x) {
            const int token = n8 + 8 * r, d = x * 64 + 16 * c4;
            const bool valid = token < live && d < a.head_dim;
            copy_async16(to + (((g * 2 + r) * (DP / 64) + x) * 32 + lane) * 16, valid ? k + token * a.k_token + d : k, valid);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int token = 2 * c4 + (i & 1) + 8 * (i >> 1), d = n8 * L::V_WORD;
          const bool valid = token < live && d < a.head_dim;
          const uint32_t dst = to + L::K_BYTES + ((g * 4 + i) * 32 + lane) * L::V_WORD;
          const uint8_t *src = valid ? v + token * a.v_token + d : v;
          if constexpr (DP == 128) copy_async16(dst, src, valid);
          else copy_async8(dst, src, valid);
        }
        if (lane < 2) {
          const float *src = lane == 0 ? a.key_scale + id * a.ks_page + h * a.ks_head
                                       : a.value_scale + id * a.vs_page + h * a.vs_head;
          copy_async4(to + L::K_BYTES + L::V_BYTES + (lane * 2 + g) * 4, src, live > 0);
        }
      }
      lstep += WARPS;
    }
    copy_commit();
  };

  find_pages();
#pragma unroll
  for (int i = 0; i < L::STAGES - 1; ++i) {
    issue(i);
    find_pages();
  }
  int stage = 0;

  Walk here = start;
  Segment seg;
  bool empty = a.whole && start.n == 0;  // a unit without keys, to be written all the same
  while (true) {
    if (empty) {
      seg = Segment{0, start.b, (int)(blockIdx.x % (a.kv_heads * a.row_tiles)), 0, 0, 0};
    } else if (!next_segment(a, here, seg)) {
      break;
    }
    const int h = seg.unit / a.row_tiles, row0 = seg.unit % a.row_tiles * L::ROWS;
    const bool at_start = seg.s0 == 0, at_end = seg.s1 == seg.n;

    // Q: lane (n8, c4) holds row n8's elements 16 c4 .. + 15 of each 64, as
    // the B operand of contraction step 4 x + w: bytes 4w .. 4w + 3 of a key's
    // 16-byte word x
    uint32_t qf[NT][KS][2];
    float q_unit[NT];  // the power of two a row was divided by
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + nt * 8 + n8;
      const bool valid = row < a.rows;
      const int i = valid ? row / a.group : 0, hq = h * a.group + (valid ? row % a.group : 0);
      const T *q = static_cast<const T *>(a.query) + seg.b * a.q_batch + i * a.q_token + hq * a.q_head;
      float x[DP / 4], top = 0.f;
#pragma unroll
      for (int e = 0; e < DP / 4; ++e) {
        const int d = (e / 16) * 64 + 16 * c4 + e % 16;
        x[e] = valid && d < a.head_dim ? to_f(q[d * a.q_dim]) : 0.f;
        top = fmaxf(top, fabsf(x[e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      int exponent = (int)(__float_as_uint(top) >> 23);  // biased; subnormal and zero rows as 2^-126
      exponent = exponent < 1 ? 1 : exponent > 253 ? 253 : exponent;
      q_unit[nt] = __uint_as_float((uint32_t)exponent << 23);
      const float inv = __uint_as_float((uint32_t)(254 - exponent) << 23);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int e = (s / 4) * 16 + (s % 4) * 4;
        qf[nt][s][0] = half2_bits(x[e] * inv, x[e + 1] * inv);
        qf[nt][s][1] = half2_bits(x[e + 2] * inv, x[e + 3] * inv);
      }
    }
    // of the rows 2 c4 and 2 c4 + 1 of each tile: score factor, keys seen
    float factor[NT][2], m[NT][2], mo[NT][2], l[NT][2];
    int64_t limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        factor[nt][u] = a.scale * __shfl_sync(0xffffffffu, q_unit[nt], (2 * c4 + u) * 4);
        limit[nt][u] = seg.length - a.queries + 1 + (row0 + nt * 8 + 2 * c4 + u) / a.group;
        m[nt][u] = mo[nt][u] = -INFINITY;
        l[nt][u] = 0.f;
      }
    const int64_t sure = seg.length - a.queries + 1 + row0 / a.group;  // keys that every row sees
    float o[NT][OT][4] = {};

    for (int step = seg.s0 + warp; step < seg.s1; step += WARPS) {
      issue(stage == 0 ? L::STAGES - 1 : stage - 1);  // the stage read one step ago
      find_pages();
      copy_wait<L::STAGES - 1>();
      __syncwarp();  // the scales were copied by two lanes
      const uint32_t from = ring + stage * L::STAGE;
      stage = stage + 1 == L::STAGES ? 0 : stage + 1;

      float s[2][NT][4] = {};
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint4 k[2][DP / 64];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int x = 0; x < DP / 64; ++x) k[r][x] = load_shared16(from + (((g * 2 + r) * (DP / 64) + x) * 32 + lane) * 16);
#pragma unroll
        for (int x = 0; x < DP / 64; ++x) {
          const uint32_t lo[4] = {k[0][x].x, k[0][x].y, k[0][x].z, k[0][x].w};
          const uint32_t hi[4] = {k[1][x].x, k[1][x].y, k[1][x].z, k[1][x].w};
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
      float ks[2], lv[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        ks[g] = load_shared4(from + L::K_BYTES + L::V_BYTES + g * 4);
        lv[g] = log2_fast(load_shared4(from + L::K_BYTES + L::V_BYTES + 8 + g * 4));
      }
      const int64_t t0 = (int64_t)step * STEP;
      const bool masked = t0 + STEP > sure;
      bool grew = false;
      float alpha[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[g][nt][e] *= factor[nt][e & 1] * ks[g];
            if (masked && t0 + 16 * g + n8 + 8 * (e >> 1) >= limit[nt][e & 1]) s[g][nt][e] = -INFINITY;
          }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float b0 = fmaxf(s[0][nt][u], s[0][nt][u + 2]), b1 = fmaxf(s[1][nt][u], s[1][nt][u + 2]);
          float top = fmaxf(b0, b1), top_o = fmaxf(b0 + lv[0], b1 + lv[1]);
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            top_o = fmaxf(top_o, __shfl_xor_sync(0xffffffffu, top_o, x));
          }
          const float m_new = fmaxf(m[nt][u], top), mo_new = fmaxf(mo[nt][u], top_o);
          l[nt][u] *= exp2_fast(m[nt][u] - reference(m_new));
          alpha[nt][u] = exp2_fast(mo[nt][u] - reference(mo_new));
          grew |= mo_new > mo[nt][u];
          m[nt][u] = m_new;
          mo[nt][u] = mo_new;
        }
      }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int t = 0; t < OT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[nt][t][e] *= alpha[nt][e & 1];
      }
      uint32_t pf[2][NT][2];  // P^T: keys 2 c4, 2 c4 + 1 (and + 8) of row n8
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float r0 = reference(m[nt][0]), r1 = reference(m[nt][1]);
        const float w0 = reference(mo[nt][0]), w1 = reference(mo[nt][1]);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float x0 = s[g][nt][2 * r], x1 = s[g][nt][2 * r + 1];
            l[nt][0] += exp2_fast(x0 - r0);
            l[nt][1] += exp2_fast(x1 - r1);
            pf[g][nt][r] = transpose8x8(half2_bits(exp2_fast(x0 + lv[g] - w0), exp2_fast(x1 + lv[g] - w1)));
          }
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t v[4][L::V_WORD / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t at = from + L::K_BYTES + ((g * 4 + i) * 32 + lane) * L::V_WORD;
          if constexpr (DP == 128) {
            const uint4 x = load_shared16(at);
            v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
          } else {
            const uint2 x = load_shared8(at);
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
    }

    // ---------------------------------------------------------- join the warps
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float sum = l[nt][u];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int row = nt * 8 + 2 * c4 + u;
        if (n8 == 0) {
          stats[(warp * L::ROWS + row) * 3] = m[nt][u];
          stats[(warp * L::ROWS + row) * 3 + 1] = sum;
          stats[(warp * L::ROWS + row) * 3 + 2] = mo[nt][u];
        }
        float *to = join + (warp * L::ROWS + row) * L::PITCH + n8 * L::V_WORD;
#pragma unroll
        for (int t = 0; t < OT; t += 2)
          *reinterpret_cast<float4 *>(to + 2 * t) =
              make_float4(o[nt][t][u], o[nt][t][u + 2], o[nt][t + 1][u], o[nt][t + 1][u + 2]);
      }
    __syncthreads();
    const bool complete = at_start && at_end;
    float *part = a.parts;
    if (!complete) part += (2 * (int64_t)blockIdx.x + (here.left + (seg.s1 - seg.s0) == start.left ? 0 : 1)) * L::PART;
    for (int i = threadIdx.x; i < L::ROWS * (DP / 4); i += WARPS * 32) {
      const int r = i / (DP / 4), d = i % (DP / 4) * 4;
      float top = -INFINITY, top_o = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        top = fmaxf(top, stats[(w * L::ROWS + r) * 3]);
        top_o = fmaxf(top_o, stats[(w * L::ROWS + r) * 3 + 2]);
      }
      float sum = 0.f, acc[4] = {};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float *st = stats + (w * L::ROWS + r) * 3;
        sum += st[1] * exp2_fast(st[0] - reference(top));
        const float f = exp2_fast(st[2] - reference(top_o));
        const float4 x = *reinterpret_cast<const float4 *>(join + (w * L::ROWS + r) * L::PITCH + d);
        acc[0] = fmaf(x.x, f, acc[0]); acc[1] = fmaf(x.y, f, acc[1]);
        acc[2] = fmaf(x.z, f, acc[2]); acc[3] = fmaf(x.w, f, acc[3]);
      }
      if (complete) {
        write_row<T>(a, seg.b, h, row0 + r, d, acc, top, sum, top_o);
      } else {
        *reinterpret_cast<float4 *>(part + r * DP + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) {
          part[L::ROWS * DP + r * 3] = top;
          part[L::ROWS * DP + r * 3 + 1] = sum;
          part[L::ROWS * DP + r * 3 + 2] = top_o;
        }
      }
    }
    __syncthreads();
    if (empty) break;
  }
}

// Joins the parts of the units that several CTAs shared, one block a unit, and
// writes the rows of sequences without keys.
constexpr int JOIN_THREADS = 128;
template <typename T, int DP, int NT>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Attention a, int64_t pieces) {
  using L = Layout<DP, NT>;
  __shared__ int64_t reduce[JOIN_THREADS / 32];
  wait_prior_grid();
  const int units = a.kv_heads * a.row_tiles;
  const int64_t b = blockIdx.x / units;
  const int unit = (int)(blockIdx.x % units), h = unit / a.row_tiles, row0 = unit % a.row_tiles * L::ROWS;
  const int64_t n = steps_of(cached_length(a, b));
  const int64_t piece = piece_of(steps_below<JOIN_THREADS>(a, a.batch, reduce), pieces, a.least);
  const int64_t first = steps_below<JOIN_THREADS>(a, b, reduce) + unit * n;
  const int64_t c0 = n > 0 ? first / piece : 0, c1 = n > 0 ? (first + n - 1) / piece : 0;
  if (n > 0 && c0 == c1) return;
  // the first CTA's part is its first segment only if the unit starts its piece
  auto part_of = [&](int64_t c) {
    return a.parts + (2 * c + (c == c0 && first != c0 * piece ? 1 : 0)) * L::PART;
  };
  for (int i = threadIdx.x; i < L::ROWS * (DP / 4); i += JOIN_THREADS) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    float top = -INFINITY, top_o = -INFINITY, sum = 0.f, acc[4] = {};
    if (n > 0) {
      for (int64_t c = c0; c <= c1; ++c) {
        const float *st = part_of(c) + L::ROWS * DP + r * 3;
        top = fmaxf(top, st[0]);
        top_o = fmaxf(top_o, st[2]);
      }
      for (int64_t c = c0; c <= c1; ++c) {
        const float *p = part_of(c), *st = p + L::ROWS * DP + r * 3;
        sum += st[1] * exp2_fast(st[0] - reference(top));
        const float f = exp2_fast(st[2] - reference(top_o));
        const float4 x = *reinterpret_cast<const float4 *>(p + r * DP + d);
        acc[0] = fmaf(x.x, f, acc[0]); acc[1] = fmaf(x.y, f, acc[1]);
        acc[2] = fmaf(x.z, f, acc[2]); acc[3] = fmaf(x.w, f, acc[3]);
      }
    }
    write_row<T>(a, b, h, row0 + r, d, acc, top, sum, top_o);
  }
}

// Contexts of at most this many tokens (eight warps' single steps) go one CTA a
// unit, without a second kernel.
constexpr int64_t WHOLE_TOKENS = WARPS * STEP;

template <typename T, typename C, int DP, int NT>
int launch_tiles(Attention a, cudaStream_t stream) {
  using L = Layout<DP, NT>;
  cudaError_t e = smem_optin<attention_kernel<T, C, DP, NT>>(L::SMEM);
  if (e != cudaSuccess) return (int)e;
  a.row_tiles = (a.rows + L::ROWS - 1) / L::ROWS;
  const int64_t units = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  if (units > (1LL << 31) - 1) return NT_B200_ERR_INVALID_ARGUMENT;
  a.whole = a.capacity <= WHOLE_TOKENS;
  a.least = WARPS;
  const int64_t grid = a.whole ? units : sm_count();
  const int rc = launch_overlapped(attention_kernel<T, C, DP, NT>, dim3((unsigned)grid), dim3(WARPS * 32), L::SMEM, stream, a);
  if (rc != 0 || a.whole) return rc;
  return launch_overlapped(join_kernel<T, DP, NT>, dim3((unsigned)units), dim3(JOIN_THREADS), 0, stream, a, grid);
}

template <typename T, typename C>
int launch_attention(const Attention &a, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2) {
    if (a.head_dim <= 128) {
      const bool one = a.rows <= 8;
      if (a.head_dim <= 64)
        return one ? launch_tiles<T, C, 64, 1>(a, stream) : launch_tiles<T, C, 64, 2>(a, stream);
      return one ? launch_tiles<T, C, 128, 1>(a, stream) : launch_tiles<T, C, 128, 2>(a, stream);
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
  // two parts a CTA of the largest layout; the CTAs of a launch are the SMs
  return 2 * (int64_t)nt::sm_count() * Layout<128, 2>::PART * (int64_t)sizeof(float);
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
      a->queries * a->heads > (1 << 30) || !(a->scale == a->scale))
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
  p.capacity = a->table_columns * c.page;
  p.batch = (int)a->batch; p.queries = (int)a->queries; p.heads = (int)a->heads; p.kv_heads = (int)c.kv_heads;
  p.group = (int)(a->heads / c.kv_heads);
  p.head_dim = (int)c.head_dim;
  p.page = (int)c.page;
  p.rows = (int)(a->queries * p.group);
  p.scale = (float)(a->scale * 1.4426950408889634);
  p.parts = static_cast<float *>(a->workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    if (c.code_dtype == NT_B200_INT8) return paged::launch_attention<scalar_t, int8_t>(p, s);
    return paged::launch_attention<scalar_t, __nv_fp8_e4m3>(p, s);
  });
}
