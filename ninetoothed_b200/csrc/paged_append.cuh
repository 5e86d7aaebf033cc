// Appending keys and values to a paged 8-bit cache, rotated on the way.
//
// A unit of work is one touched page of one sequence, one key/value head, and
// one of key or value: the new tokens that fall into the page share its scale,
// so a unit first takes the largest magnitude among them (after the rotation),
// then settles the scale, rounds the codes the page already held again if the
// scale grew, and writes the new codes.  No two units share a page and a head,
// so nothing is atomic and the result does not depend on the order.
//
// Bound by memory: key and value are read once and written as a byte each.  A
// unit's elements stay on the SM between the two passes: a team of warps takes
// two chunk pairs (32 16-bit elements) a thread, 16-token pages of 128-element
// heads two warps, 64-token pages eight; what a larger page has beyond that is
// read a second time.  What a block does before its first load of elements is
// one round of loads of offsets and past lengths; the page and its scale come
// while the elements are on their way.
#pragma once

#include "common.cuh"
#include "rotary.cuh"

namespace nt {
namespace paged {

// The scale of a block of elements whose largest finite magnitude is `amax`.
// E4M3 takes a power of two: multiplying and dividing by it is exact, so a
// block's codes survive a later growth of its scale; a step of INT8 is even,
// and its scale spends none of the 127 steps.
constexpr float kLeastScale = 1.1754943508222875e-38f;  // 2^-126
template <typename C> __device__ __forceinline__ float block_scale(float amax);
template <> __device__ __forceinline__ float block_scale<int8_t>(float amax) {
  return fmaxf(__fmul_rn(amax, 1.f / 127.f), kLeastScale);
}
template <> __device__ __forceinline__ float block_scale<__nv_fp8_e4m3>(float amax) {
  // 448 = 1.75 * 2^8: the least k with amax <= 448 * 2^k from amax's exponent
  // and whether its significand passes 1.75.  Magnitudes under 2^-118 take
  // the least scale.
  const uint32_t bits = __float_as_uint(amax);
  int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  if (k < -126) k = -126;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

template <typename C> __device__ __forceinline__ uint8_t encode(float x);
template <> __device__ __forceinline__ uint8_t encode<__nv_fp8_e4m3>(float x) {
  return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
template <> __device__ __forceinline__ uint8_t encode<int8_t>(float x) {
  const int v = __float2int_rn(x);  // NaN converts to 0
  return (uint8_t)(int8_t)max(-127, min(127, v));
}
template <typename C> __device__ __forceinline__ float decode(uint8_t code);
template <> __device__ __forceinline__ float decode<__nv_fp8_e4m3>(uint8_t code) {
  __nv_fp8_e4m3 v;
  v.__x = code;
  return static_cast<float>(v);
}
template <> __device__ __forceinline__ float decode<int8_t>(uint8_t code) { return (float)(int8_t)code; }

// The codes of four values, the first in the low byte.
template <typename C> __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d);
template <> __device__ __forceinline__ uint32_t encode4<__nv_fp8_e4m3>(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
template <> __device__ __forceinline__ uint32_t encode4<int8_t>(float a, float b, float c, float d) {
  return encode<int8_t>(a) | (uint32_t)encode<int8_t>(b) << 8 | (uint32_t)encode<int8_t>(c) << 16 | (uint32_t)encode<int8_t>(d) << 24;
}

// Codes of eight or four values, in memory order.
template <typename C, int N> __device__ __forceinline__ void store_codes(uint8_t *to, const float (&x)[N], float inv) {
  uint32_t w[N / 4];
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    w[i] = encode4<C>(__fmul_rn(x[4 * i], inv), __fmul_rn(x[4 * i + 1], inv), __fmul_rn(x[4 * i + 2], inv),
                      __fmul_rn(x[4 * i + 3], inv));
  if constexpr (N == 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t *>(to) = w[0];
}

// |x| where it is finite, else 0.
__device__ __forceinline__ float finite_magnitude(float x) {
  const float m = fabsf(x);
  return m < INFINITY ? m : 0.f;  // NaN compares false
}

// The largest i in [0, n) with f(i) <= x, for a nondecreasing f with
// f(0) <= x; all 32 lanes call it and narrow the range 32-fold a step.
template <typename F> __device__ __forceinline__ int64_t warp_search(int64_t n, int64_t x, F f) {
  const int lane = threadIdx.x & 31;
  int64_t low = 0, length = n;
  while (length > 1) {
    const int64_t step = (length + 31) / 32, i = lane * step;
    const bool le = i < length && f(low + i) <= x;
    const int count = __popc(__ballot_sync(0xffffffffu, le));
    const int64_t skip = (count > 0 ? count - 1 : 0) * step;
    low += skip;
    length = length - skip < step ? length - skip : step;
  }
  return low;
}

struct Side {  // key or value
  const void *in;
  uint8_t *codes;
  float *scales;
  void *out;  // rotated copy in the input type, or null
  int64_t in_token, in_head, in_dim, page_stride, head_stride, token_stride, scale_page, scale_head;
  int64_t out_token, out_head, out_dim;
};

struct Params {
  Side side[2];
  rotary::Params query;  // input null: no queries
  rotary::Tables tables;
  IndexArray offsets, past, block_table;
  int64_t table_row_stride;
  int64_t tokens, batch, pages, table_columns;
  int64_t units;  // candidates a head and side: tokens / page + 2 * batch
  int page, kv_heads, head_dim, chunk_pairs;
  uint32_t unit_blocks;  // blockIdx.x below this: pages; the rest: queries
  uint32_t groups;       // blocks of one page: heads and sides / teams
  int team_warps;
  uint32_t chunk_reciprocal;  // ceil(2^32 / chunk_pairs): exact for a page's items
  int interleaved;
};

// Where offsets are out of order the search can miss sequences, and with them
// tokens.  The grid's last block looks for that and does nothing else (in the
// others it took a step of 32 sequences from 3.9 to 4.2 us).
__device__ __forceinline__ bool checks_order(const Params &p) {
  if (blockIdx.x != gridDim.x - 1) return false;
  for (int64_t i = threadIdx.x; i < p.batch; i += blockDim.x)
    if (p.offsets[i + 1] < p.offsets[i]) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
  return true;
}

struct Unit {
  int64_t token0;    // packed index of the first new token in the page
  int64_t position0; // its position in the sequence
  int64_t entry;     // of the page in the block table
  int count, slot0;  // new tokens, first new slot
};

// An offset as a 32-bit number of tokens, for the search (offsets that leave
// the tensors are found out after it).
__device__ __forceinline__ uint32_t bounded(int64_t offset, int64_t tokens) {
  return offset < 0 ? 0u : offset > tokens ? (uint32_t)tokens : (uint32_t)offset;
}

// A sequence: its packed tokens o0 .. o1 - 1 and how many it had.
struct Sequence {
  int64_t index, o0, o1, past;
};
// The last sequence s with key(bounded(offsets[s]), s) <= x; the key does not
// decrease.  All lanes of a warp ask for the same; up to 32 sequences take one
// round of loads.
template <typename F>
__device__ __forceinline__ Sequence find_sequence(const Params &p, uint32_t x, F key) {
  Sequence q;
  if (p.batch <= 32) {
    const int lane = threadIdx.x & 31, i = lane < (int)p.batch ? lane : (int)p.batch - 1;
    const int64_t o0 = p.offsets[i], o1 = p.offsets[i + 1], past = p.past[i];
    const unsigned le = __ballot_sync(0xffffffffu, lane < (int)p.batch && key(bounded(o0, p.tokens), (uint32_t)i) <= x);
    const int s = le ? 31 - __clz(le) : 0;
    q.index = s;
    q.o0 = __shfl_sync(0xffffffffu, o0, s);
    q.o1 = __shfl_sync(0xffffffffu, o1, s);
    q.past = __shfl_sync(0xffffffffu, past, s);
  } else {
    q.index = warp_search(p.batch, x, [&](int64_t i) { return (int64_t)key(bounded(p.offsets[i], p.tokens), (uint32_t)i); });
    q.o0 = p.offsets[q.index];
    q.o1 = p.offsets[q.index + 1];
    q.past = p.past[q.index];
  }
  return q;
}

// The u-th candidate.  Sequence s owns the candidates from offsets[s] / page +
// 2 s on, at least one for each page it can touch; those past its last page
// are empty.  All lanes of a warp ask for the same unit.
__device__ __forceinline__ bool find_unit(const Params &p, uint32_t u, Unit &w) {
  const uint32_t page = (uint32_t)p.page;
  const Sequence q = find_sequence(p, u, [&](uint32_t o, uint32_t s) { return o / page + 2 * s; });
  if (q.o1 <= q.o0) return false;
  if (q.o0 < 0 || q.o1 > p.tokens || q.past < 0 || q.past > INT32_MAX - p.tokens) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return false;
  }
  const uint32_t past = (uint32_t)q.past, column = past / page + (u - ((uint32_t)q.o0 / page + 2 * (uint32_t)q.index));
  const uint32_t low = max(past, column * page), high = min(past + (uint32_t)(q.o1 - q.o0), (column + 1) * page);
  if (low >= high) return false;
  if ((int64_t)column >= p.table_columns || (p.tables.pairs > 0 && (int64_t)high > p.tables.rows)) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return false;
  }
  w.entry = q.index * p.table_row_stride + column * p.block_table.stride;
  w.token0 = q.o0 + (low - past);
  w.position0 = low;
  w.count = (int)(high - low);
  w.slot0 = (int)(low - column * page);
  return true;
}

// The unit's page in the pool, or -1.
__device__ __forceinline__ int64_t find_page(const Params &p, const Unit &w) {
  const int64_t block = p.block_table.wide ? static_cast<const int64_t *>(p.block_table.data)[w.entry]
                                           : (int64_t) static_cast<const int32_t *>(p.block_table.data)[w.entry];
  return block >= 0 && block < p.pages ? block : -1;
}

constexpr int THREADS = 128;

// The largest v of a team of `warps` neighbouring warps; the whole block calls it.
__device__ __forceinline__ float team_max(float v, int warps, float *shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  const int first = (threadIdx.x >> 5) / warps * warps;
  for (int i = 0; i < warps; ++i) v = fmaxf(v, shared[first + i]);
  return v;
}

// Settles a page's scale and rounds its held codes again where it grew.  Every
// thread of the team has read `held` before the team's barrier; `me` of `threads`
// is its place in the team.
template <typename C>
__device__ __forceinline__ float settle_scale(const Params &p, const Side &side, const Unit &w, int64_t block, int h,
                                              float amax, float held, int me, int threads) {
  const float scale = block_scale<C>(amax);
  if (w.slot0 > 0 && held >= scale) return held;
  if (w.slot0 > 0) {
    const float ratio = __fdiv_rn(held, scale);
    uint8_t *base = side.codes + block * side.page_stride + (int64_t)h * side.head_stride;
    const int words = p.head_dim / 4;
    for (int i = me; i < w.slot0 * words; i += threads) {
      uint32_t *at = reinterpret_cast<uint32_t *>(base + (int64_t)(i / words) * side.token_stride) + i % words;
      const uint32_t old = *at;
      *at = encode4<C>(__fmul_rn(decode<C>((uint8_t)old), ratio), __fmul_rn(decode<C>((uint8_t)(old >> 8)), ratio),
                       __fmul_rn(decode<C>((uint8_t)(old >> 16)), ratio), __fmul_rn(decode<C>((uint8_t)(old >> 24)), ratio));
    }
  }
  if (me == 0) side.scales[block * side.scale_page + (int64_t)h * side.scale_head] = scale;
  return scale;
}

// Rotates a block's share of the queries.  Tokens of a block are near one
// another: a warp searches for its first one's sequence and each thread goes on
// from there.
template <typename T, bool VEC>
__device__ __forceinline__ void rotate_queries(const Params &p, uint32_t block) {
  const rotary::Params &q = p.query;
  const uint32_t per_token = VEC ? (uint32_t)(q.chunk_pairs * q.head_groups) : (uint32_t)q.heads;
  const uint32_t i = block * THREADS + threadIdx.x, token = i / per_token, r = i % per_token;
  const bool valid = token < (uint32_t)p.tokens;
  auto position_of = [&]() -> int64_t {
    Sequence s = find_sequence(p, (i & ~31u) / per_token, [](uint32_t o, uint32_t) { return o; });
    while (token >= s.o1 && s.index + 1 < p.batch) {
      ++s.index;
      s.o0 = s.o1;
      s.o1 = p.offsets[s.index + 1];
      s.past = p.past[s.index];
    }
    return token >= s.o0 && token < s.o1 ? s.past + (token - s.o0) : INT64_MIN;
  };
  if constexpr (VEC) {
    rotary::rotate_heads<T>(q, token, valid, (int)(r / q.chunk_pairs) * rotary::HEADS, (int)(r % q.chunk_pairs), position_of);
  } else {
    const int64_t position = position_of();
    if (!valid || position < rotary::kNone) return;
    const bool known = p.tables.pairs == 0 || (position >= 0 && position < p.tables.rows);
    if (!known) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    const T *in = static_cast<const T *>(q.input) + token * q.in_token + (int64_t)r * q.in_head;
    T *out = static_cast<T *>(q.output) + token * q.out_token + (int64_t)r * q.out_head;
    for (int e = 0; e < p.tables.pairs; ++e) {
      const int64_t d0 = q.interleaved ? 2 * e : e, d1 = q.interleaved ? 2 * e + 1 : e + p.tables.pairs;
      float a = to_f(in[d0 * q.in_dim]), b = to_f(in[d1 * q.in_dim]);
      rotary::turn(a, b, known ? p.tables.cos[position * p.tables.cos_stride + e] : NAN,
                   known ? p.tables.sin[position * p.tables.sin_stride + e] : NAN);
      out[d0 * q.out_dim] = from_f<T>(a);
      out[d1 * q.out_dim] = from_f<T>(b);
    }
    for (int64_t d = 2 * p.tables.pairs; d < q.head_dim; ++d) out[d * q.out_dim] = in[d * q.in_dim];
  }
}

// A block takes a candidate page and as many heads and sides of it as it has
// teams of `team_warps` warps.  KEPT chunk pairs a thread stay between the passes
// in shared memory, rotated, as fp32.  Four prompts of 4096 tokens (32 + 8 heads of
// 128, 64-token pages), queries among them: 93 us, 4.0 TB/s; with the values kept
// in registers (139 of them, 12 warps an SM) 182 us, read and rotated again for
// the second pass 125 us, in blocks of 256 threads 101 us.
constexpr int KEPT = 2;
template <typename T> constexpr int kept_bytes() { return KEPT * THREADS * 2 * rotary::Chunk<T>::N * 4; }

template <typename T, typename C>
__global__ void __launch_bounds__(THREADS, 8) append_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) float4 kept[];  // [KEPT][chunk pair / 4][THREADS]
  __shared__ float shared[THREADS / 32];
  if (checks_order(p)) return;
  if (blockIdx.x >= p.unit_blocks) {
    rotate_queries<T, true>(p, blockIdx.x - p.unit_blocks);
    return;
  }
  using Chunk = rotary::Chunk<T>;
  constexpr int N = Chunk::N;
  Unit w;
  if (!find_unit(p, blockIdx.x / p.groups, w)) return;
  const uint32_t threads = 32 * p.team_warps, team = threadIdx.x / threads, me = threadIdx.x % threads;
  const uint32_t which = blockIdx.x % p.groups * (THREADS / threads) + team;  // head and side
  const bool active = which < (uint32_t)(2 * p.kv_heads);
  const int h = active ? (int)(which >> 1) : 0;
  const Side &side = p.side[which & 1];
  const int pairs = (which & 1) == 0 ? p.tables.pairs : 0;
  const uint32_t items = active ? w.count * p.chunk_pairs : 0;
  const T *in = static_cast<const T *>(side.in) + (int64_t)h * side.in_head + w.token0 * side.in_token;

  struct Item {
    uint32_t j;  // token of the unit
    rotary::Place<T> at;
  };
  auto item = [&](uint32_t i) {
    const uint32_t j = p.chunk_pairs == 1 ? i : __umulhi(i, p.chunk_reciprocal);
    return Item{j, rotary::place<T>(i - j * p.chunk_pairs, p.head_dim, pairs, p.interleaved != 0)};
  };
  auto load = [&](const Item &t, Chunk &a, Chunk &b) {
    const T *row = in + (int64_t)t.j * side.in_token;
    a = *reinterpret_cast<const Chunk *>(row + t.at.first);
    if (t.at.second >= 0) b = *reinterpret_cast<const Chunk *>(row + t.at.second);
  };
  // a chunk pair's values, rotated
  auto values = [&](const Item &t, const Chunk &a, const Chunk &b, float(&x)[N], float(&y)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) { x[e] = to_f(a.v[e]); y[e] = to_f(b.v[e]); }
    if (t.at.pair >= 0) {
      float c[N], s[N];
      rotary::load_angles<T>(p.tables, w.position0 + t.j, t.at.pair, c, s);
      rotary::turn_chunks<N>(x, y, c, s, p.interleaved != 0, pairs - t.at.pair);
    }
  };
  float amax = 0.f;
  auto measure = [&](const float(&x)[N], const float(&y)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) amax = fmaxf(amax, fmaxf(fabsf(x[e]), fabsf(y[e])));
  };

  Chunk a[KEPT] = {}, b[KEPT] = {};
#pragma unroll
  for (int k = 0; k < KEPT; ++k)
    if (me + k * threads < items) load(item(me + k * threads), a[k], b[k]);
  const int64_t block = find_page(p, w);
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    if (me + k * threads < items) {
      float x[N], y[N];
      values(item(me + k * threads), a[k], b[k], x, y);
      measure(x, y);
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        kept[(2 * q + k * (N / 2)) * THREADS + threadIdx.x] = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        kept[(2 * q + 1 + k * (N / 2)) * THREADS + threadIdx.x] =
            make_float4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
      }
    }
  }
  for (uint32_t i = me + KEPT * threads; i < items; i += threads) {
    Chunk c = {}, d = {};
    float x[N], y[N];
    load(item(i), c, d);
    values(item(i), c, d, x, y);
    measure(x, y);
  }
  if (block < 0) {  // for the whole thread block
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return;
  }
  const float held = w.slot0 > 0 && active ? side.scales[block * side.scale_page + (int64_t)h * side.scale_head] : 0.f;
  amax = team_max(amax, p.team_warps, shared);
  if (__syncthreads_or(amax == INFINITY)) {  // rarely: the largest finite magnitudes
    float finite = 0.f;
    for (uint32_t i = me; i < items; i += threads) {
      Chunk c = {}, d = {};
      float x[N], y[N];
      load(item(i), c, d);
      values(item(i), c, d, x, y);
#pragma unroll
      for (int e = 0; e < N; ++e) finite = fmaxf(finite, fmaxf(finite_magnitude(x[e]), finite_magnitude(y[e])));
    }
    amax = team_max(finite, p.team_warps, shared);
  }
  if (!active) return;
  const float scale = settle_scale<C>(p, side, w, block, h, amax, held, me, threads);
  const float inv = __fdiv_rn(1.f, scale);
  uint8_t *page = side.codes + block * side.page_stride + (int64_t)h * side.head_stride;

  auto store = [&](const Item &t, const float(&x)[N], const float(&y)[N]) {
    uint8_t *codes = page + (int64_t)(w.slot0 + t.j) * side.token_stride;
    store_codes<C, N>(codes + t.at.first, x, inv);
    if (t.at.second >= 0) store_codes<C, N>(codes + t.at.second, y, inv);
    if (side.out) {
      T *out = static_cast<T *>(side.out) + (w.token0 + t.j) * side.out_token + (int64_t)h * side.out_head;
      *reinterpret_cast<Chunk *>(out + t.at.first) = rotary::to_chunk<T>(x);
      if (t.at.second >= 0) *reinterpret_cast<Chunk *>(out + t.at.second) = rotary::to_chunk<T>(y);
    }
  };
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    if (me + k * threads < items) {
      float x[N], y[N];
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        const float4 u = kept[(2 * q + k * (N / 2)) * THREADS + threadIdx.x];
        const float4 v = kept[(2 * q + 1 + k * (N / 2)) * THREADS + threadIdx.x];
        x[4 * q] = u.x; x[4 * q + 1] = u.y; x[4 * q + 2] = u.z; x[4 * q + 3] = u.w;
        y[4 * q] = v.x; y[4 * q + 1] = v.y; y[4 * q + 2] = v.z; y[4 * q + 3] = v.w;
      }
      store(item(me + k * threads), x, y);
    }
  }
  for (uint32_t i = me + KEPT * threads; i < items; i += threads) {
    Chunk c = {}, d = {};
    float x[N], y[N];
    load(item(i), c, d);
    values(item(i), c, d, x, y);
    store(item(i), x, y);
  }
}

// Any strides of the new tokens and any rotary extent: an element or a pair a
// thread.  Four prompts of 4096 tokens, 32 + 8 heads of 96 bfloat16 elements: 628 us
// with 24 of them rotated (the halves are no whole chunks) where the kernel above
// takes 75 us with 96.
template <typename T, typename C>
__global__ void __launch_bounds__(THREADS) append_scalar_kernel(const __grid_constant__ Params p) {
  __shared__ float shared[THREADS / 32];
  if (checks_order(p)) return;
  if (blockIdx.x >= p.unit_blocks) {
    rotate_queries<T, false>(p, blockIdx.x - p.unit_blocks);
    return;
  }
  const uint32_t which = blockIdx.x % p.groups;  // head and side
  Unit w;
  if (!find_unit(p, blockIdx.x / p.groups, w)) return;
  const int64_t block = find_page(p, w);
  if (block < 0) {
    record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    return;
  }
  const int h = (int)which >> 1;
  const Side &side = p.side[which & 1];
  const int pairs = (which & 1) == 0 ? p.tables.pairs : 0;
  const int per_token = p.head_dim - pairs;  // pairs, then single elements
  const int items = w.count * per_token;
  const float held = side.scales[block * side.scale_page + (int64_t)h * side.scale_head];
  const T *in = static_cast<const T *>(side.in) + (int64_t)h * side.in_head;

  auto load = [&](int i, int &d0, int &d1, float &a, float &b) {
    const int j = i / per_token, e = i % per_token;
    const T *row = in + (w.token0 + j) * side.in_token;
    if (e < pairs) {
      d0 = p.interleaved ? 2 * e : e;
      d1 = p.interleaved ? 2 * e + 1 : e + pairs;
      a = to_f(row[d0 * side.in_dim]);
      b = to_f(row[d1 * side.in_dim]);
      const int64_t position = w.position0 + j;
      rotary::turn(a, b, p.tables.cos[position * p.tables.cos_stride + e], p.tables.sin[position * p.tables.sin_stride + e]);
    } else {
      d0 = e + pairs;
      d1 = -1;
      a = to_f(row[d0 * side.in_dim]);
      b = 0.f;
    }
  };

  float amax = 0.f;
  for (int i = threadIdx.x; i < items; i += THREADS) {
    int d0, d1;
    float a, b;
    load(i, d0, d1, a, b);
    amax = fmaxf(amax, fmaxf(finite_magnitude(a), finite_magnitude(b)));
  }
  const float scale = settle_scale<C>(p, side, w, block, h, team_max(amax, THREADS / 32, shared), held, threadIdx.x, THREADS);
  const float inv = __fdiv_rn(1.f, scale);
  for (int i = threadIdx.x; i < items; i += THREADS) {
    int d0, d1;
    float a, b;
    load(i, d0, d1, a, b);
    const int j = i / per_token;
    uint8_t *codes = side.codes + block * side.page_stride + (int64_t)h * side.head_stride +
                     (int64_t)(w.slot0 + j) * side.token_stride;
    codes[d0] = encode<C>(__fmul_rn(a, inv));
    if (d1 >= 0) codes[d1] = encode<C>(__fmul_rn(b, inv));
    if (side.out) {
      T *out = static_cast<T *>(side.out) + (w.token0 + j) * side.out_token + (int64_t)h * side.out_head;
      out[d0 * side.out_dim] = from_f<T>(a);
      if (d1 >= 0) out[d1 * side.out_dim] = from_f<T>(b);
    }
  }
}

template <typename T, typename C>
int launch_append(Params p, cudaStream_t stream) {
  constexpr int N = rotary::Chunk<T>::N;
  const int64_t pairs = p.tables.pairs;
  bool vec = pairs == 0 || rotary::vector_tables(p.tables);
  for (int i = 0; i < 2; ++i) {
    const Side &s = p.side[i];
    const int64_t turned = i == 0 ? pairs : 0;
    vec = vec && rotary::vector_heads<T>(s.in, s.in_token, s.in_head, s.in_dim, p.head_dim, turned, p.interleaved);
    if (s.out)
      vec = vec && rotary::vector_heads<T>(s.out, s.out_token, s.out_head, s.out_dim, p.head_dim, turned, p.interleaved);
  }
  rotary::Params &q = p.query;
  if (q.input)
    vec = vec && rotary::vector_heads<T>(q.input, q.in_token, q.in_head, q.in_dim, p.head_dim, pairs, p.interleaved) &&
          rotary::vector_heads<T>(q.output, q.out_token, q.out_head, q.out_dim, p.head_dim, pairs, p.interleaved);
  p.chunk_pairs = q.chunk_pairs = (p.head_dim + 2 * N - 1) / (2 * N);
  q.head_groups = (q.heads + rotary::HEADS - 1) / rotary::HEADS;
  const int64_t threads = q.input ? p.tokens * (vec ? (int64_t)q.chunk_pairs * q.head_groups : (int64_t)q.heads) : 0;
  // a team's threads hold a page of new tokens, up to a block's
  p.team_warps = 1;
  while (p.team_warps < THREADS / 32 && p.team_warps * 32 * KEPT < p.page * p.chunk_pairs) p.team_warps *= 2;
  const int teams = vec ? THREADS / 32 / p.team_warps : 1;
  p.groups = (uint32_t)((2 * p.kv_heads + teams - 1) / teams);
  const int64_t units = p.units * p.groups, blocks = units + (threads + THREADS - 1) / THREADS + 1;
  if (blocks > (1LL << 31) - 1 || threads >= (1LL << 32)) return NT_B200_ERR_INVALID_ARGUMENT;
  p.unit_blocks = (uint32_t)units;
  const dim3 grid((unsigned)blocks);
  p.chunk_reciprocal = (uint32_t)(((1ull << 32) + p.chunk_pairs - 1) / p.chunk_pairs);
  if (vec) append_kernel<T, C><<<grid, THREADS, kept_bytes<T>(), stream>>>(p);
  else append_scalar_kernel<T, C><<<grid, THREADS, 0, stream>>>(p);
  return launch_status();
}

// Host-side checks of a cache (no launch): 0 or an error code.
inline int check_cache(const NtB200PagedCache &c) {
  if (c.pages < 0 || c.pages >= (1LL << 31) || c.kv_heads < 0 || c.page <= 0 || c.head_dim <= 0) return NT_B200_ERR_INVALID_ARGUMENT;
  if (c.code_dtype != NT_B200_FLOAT8_E4M3FN && c.code_dtype != NT_B200_INT8) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (c.page % 16 != 0 || c.page > 4096 || c.head_dim % 16 != 0 || c.head_dim > (1 << 12))
    return NT_B200_ERR_SHAPE_MISMATCH;
  if (!c.key || !c.value || !c.key_scale || !c.value_scale || !rotary::aligned16(c.key) || !rotary::aligned16(c.value))
    return NT_B200_ERR_INVALID_ARGUMENT;
  for (int i = 0; i < 3; ++i)
    if (c.key_strides[i] % 16 != 0 || c.value_strides[i] % 16 != 0) return NT_B200_ERR_INVALID_ARGUMENT;
  return 0;
}

}  // namespace paged
}  // namespace nt

extern "C" int nt_b200_paged_append(const NtB200PagedAppendArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->tokens < 0 || a->batch < 0 || a->heads < 0 || a->rotary_dim < 0 || a->rotary_dim % 2 != 0 ||
      a->table_rows < 0 || a->table_columns < 0)
    return NT_B200_ERR_INVALID_ARGUMENT;
  if (!is_float_dtype((int)a->dtype) || !is_index_dtype(a->index_dtype)) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->tokens == 0 || a->batch == 0) return 0;
  const NtB200PagedCache &c = a->cache;
  const int rc = paged::check_cache(c);
  if (rc != 0) return rc;
  const bool turns = a->cos != nullptr;
  if (turns && (!a->sin || a->rotary_dim > c.head_dim)) return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->key || !a->value || !a->offsets || !a->past || !a->block_table ||
      (a->query && ((!turns && a->rotary_dim > 0) || !a->query_out)) || a->tokens > (1 << 30) || a->batch > (1 << 28) || a->heads > (1 << 20) || a->table_columns > (1LL << 31))
    return NT_B200_ERR_INVALID_ARGUMENT;
  if (c.kv_heads == 0 && !a->query) return 0;
  paged::Params p{};
  p.side[0] = {a->key, static_cast<uint8_t *>(c.key), c.key_scale, a->key_out,
               a->key_strides[0], a->key_strides[1], a->key_strides[2],
               c.key_strides[0], c.key_strides[1], c.key_strides[2], c.key_scale_strides[0], c.key_scale_strides[1],
               a->key_out_strides[0], a->key_out_strides[1], a->key_out_strides[2]};
  p.side[1] = {a->value, static_cast<uint8_t *>(c.value), c.value_scale, nullptr,
               a->value_strides[0], a->value_strides[1], a->value_strides[2],
               c.value_strides[0], c.value_strides[1], c.value_strides[2], c.value_scale_strides[0],
               c.value_scale_strides[1], 0, 0, 0};
  const int wide = a->index_dtype == NT_B200_INT64;
  p.tables = {a->cos, a->sin, a->cos_stride, a->sin_stride, a->table_rows, turns ? (int)(a->rotary_dim / 2) : 0, 1.f};
  p.offsets = {a->offsets, a->offsets_stride, wide};
  p.past = {a->past, a->past_stride, wide};
  p.block_table = {a->block_table, a->block_table_strides[1], wide};
  p.table_row_stride = a->block_table_strides[0];
  p.tokens = a->tokens;
  p.batch = a->batch;
  p.pages = c.pages;
  p.table_columns = a->table_columns;
  p.units = c.kv_heads > 0 ? a->tokens / c.page + 2 * a->batch : 0;
  p.page = (int)c.page;
  p.kv_heads = (int)c.kv_heads;
  p.head_dim = (int)c.head_dim;
  p.interleaved = a->interleaved != 0;
  if (a->query && a->heads > 0) {
    p.query.input = a->query;
    p.query.output = a->query_out;
    p.query.tables = p.tables;
    p.query.in_token = a->query_strides[0]; p.query.in_head = a->query_strides[1]; p.query.in_dim = a->query_strides[2];
    p.query.out_token = a->query_out_strides[0]; p.query.out_head = a->query_out_strides[1];
    p.query.out_dim = a->query_out_strides[2];
    p.query.heads = (int)a->heads;
    p.query.head_dim = (int)c.head_dim;
    p.query.interleaved = p.interleaved;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    if (c.code_dtype == NT_B200_INT8) return paged::launch_append<scalar_t, int8_t>(p, s);
    return paged::launch_append<scalar_t, __nv_fp8_e4m3>(p, s);
  });
}
