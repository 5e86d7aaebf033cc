// Rotary positions.  The first `rotary_dim` elements of every head are pairs
// (a, b); a token at position p turns pair i by the angle whose cosine and sine
// are row p, column i of two fp32 tables:
//     u = a cos - b sin,   v = b cos + a sin        (adjoint: sin -> -sin)
// Half layout: a = x[i], b = x[i + rotary_dim / 2]; interleaved: a = x[2i],
// b = x[2i + 1].  The remaining elements are copied.  Each product is rounded
// to fp32 before the sum (no fused multiply-add), so that a value's 8-bit code
// (paged_append.cuh) follows from the formula alone, and the result is rounded
// once to the element type.
//
// Bound by memory: every element is read and written once, a table row serves
// all heads of its token.
#pragma once

#include "common.cuh"

namespace nt {

// A device array of indices, int32 or int64.
struct IndexArray {
  const void *data;
  int64_t stride;
  int wide;
  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t *>(data)[i * stride] : (int64_t)static_cast<const int32_t *>(data)[i * stride];
  }
};

inline bool is_index_dtype(int64_t dtype) { return dtype == NT_B200_INT32 || dtype == NT_B200_INT64; }

namespace rotary {

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
  const float u = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
  b = __fadd_rn(__fmul_rn(b, c), __fmul_rn(a, s));
  a = u;
}

// 16 bytes of elements.
template <typename T> struct alignas(16) Chunk {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// Elements of a chunk from fp32 values, two a conversion.
template <typename T> __device__ __forceinline__ Chunk<T> to_chunk(const float (&x)[Chunk<T>::N]) {
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < Chunk<T>::N; i += 2) {
    if constexpr (sizeof(T) == 4) {
      c.v[i] = x[i];
      c.v[i + 1] = x[i + 1];
    } else if constexpr (Elem<T>::is_f16) {
      const __half2 h = __floats2half2_rn(x[i], x[i + 1]);
      c.v[i] = h.x;
      c.v[i + 1] = h.y;
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[i], x[i + 1]);
      c.v[i] = h.x;
      c.v[i + 1] = h.y;
    }
  }
  return c;
}

struct Tables {
  const float *cos, *sin;
  int64_t cos_stride, sin_stride, rows;
  int pairs;  // rotary_dim / 2
  float sign; // -1: adjoint
};

// Head data of a thread: two chunks that hold whole pairs.  Chunk pair c of a
// head: half layout, c < pairs / N: chunks at c N and pairs + c N (the two
// sides of N pairs); interleaved: the two neighbouring chunks 2c and 2c + 1.
// Past the rotated part both layouts take neighbouring chunks.
template <typename T> struct Place {
  int first, second;  // element offsets in the head; second < 0: none
  int pair;           // first pair's table column, < 0: copied
};
template <typename T>
__device__ __forceinline__ Place<T> place(int c, int head_dim, int pairs, bool interleaved) {
  constexpr int N = Chunk<T>::N;
  Place<T> p;
  if (!interleaved && c * N < pairs) {
    p.first = c * N;
    p.second = pairs + c * N;
    p.pair = c * N;
  } else {
    p.first = 2 * c * N;
    p.second = p.first + N < head_dim ? p.first + N : -1;
    p.pair = interleaved && p.first < 2 * pairs ? c * N : -1;
  }
  return p;
}

// The table entries of a chunk pair: N pairs, fewer where the rotated part of
// the interleaved layout ends with the first chunk.
template <typename T>
__device__ __forceinline__ void load_angles(const Tables &t, int64_t position, int pair, float (&c)[Chunk<T>::N],
                                            float (&s)[Chunk<T>::N]) {
  constexpr int N = Chunk<T>::N;
  const float *cr = t.cos + position * t.cos_stride + pair, *sr = t.sin + position * t.sin_stride + pair;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    float4 cv = make_float4(1.f, 1.f, 1.f, 1.f), sv = make_float4(0.f, 0.f, 0.f, 0.f);
    if (pair + i < t.pairs) {
      cv = __ldg(reinterpret_cast<const float4 *>(cr + i));
      sv = __ldg(reinterpret_cast<const float4 *>(sr + i));
    }
    c[i] = cv.x; c[i + 1] = cv.y; c[i + 2] = cv.z; c[i + 3] = cv.w;
    s[i] = sv.x; s[i + 1] = sv.y; s[i + 2] = sv.z; s[i + 3] = sv.w;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] *= t.sign;
}

// Turns the 2 N values of a chunk pair in registers.  `pairs`: how many of its
// N pairs are in the rotated part (a copied chunk is left alone, not turned by
// the angle 0: infinities would not survive that).
template <int N>
__device__ __forceinline__ void turn_chunks(float (&x)[N], float (&y)[N], const float (&c)[N], const float (&s)[N],
                                            bool interleaved, int pairs) {
  if (!interleaved) {
#pragma unroll
    for (int i = 0; i < N; ++i) turn(x[i], y[i], c[i], s[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) turn(x[2 * i], x[2 * i + 1], c[i], s[i]);
    if (pairs > N / 2) {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) turn(y[2 * i], y[2 * i + 1], c[N / 2 + i], s[N / 2 + i]);
    }
  }
}

struct Params {
  const void *input;
  void *output;
  Tables tables;
  IndexArray positions;
  int64_t in_token, in_head, in_dim, out_token, out_head, out_dim;
  int heads, head_dim, chunk_pairs, head_groups;
  int interleaved;
};

// A thread takes one chunk pair of HEADS heads of a token, so a table entry is
// read once for all of them and 2 HEADS 16-byte loads are in flight.  Two heads
// (64 registers, 32 warps an SM) take 69 us for 16384 tokens of 40 heads of 128
// bfloat16 elements, four (96 registers, 20 warps) 82 us, one 76 us.
constexpr int HEADS = 2, THREADS = 128;

// Rotates chunk pair `cpair` of the heads h0 .. h0 + HEADS - 1 of a token.
// `position_of` gives its position (or says with a value below kNone that the
// token is not to be written) and is asked only after the loads: a wait for it
// before them would put its latency in front of theirs.
constexpr int64_t kNone = INT64_MIN / 2;
template <typename T, typename F>
__device__ __forceinline__ void rotate_heads(const Params &p, int64_t token, bool valid, int h0, int cpair, F position_of) {
  constexpr int N = Chunk<T>::N;
  const Place<T> at = place<T>(cpair, p.head_dim, p.tables.pairs, p.interleaved != 0);
  const T *in = static_cast<const T *>(p.input) + token * p.in_token;
  Chunk<T> a[HEADS] = {}, b[HEADS] = {};
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (!valid || h0 + i >= p.heads) break;
    const T *row = in + (int64_t)(h0 + i) * p.in_head;
    a[i] = *reinterpret_cast<const Chunk<T> *>(row + at.first);
    if (at.second >= 0) b[i] = *reinterpret_cast<const Chunk<T> *>(row + at.second);
  }
  const int64_t position = position_of();
  if (!valid || position < kNone) return;
  if (at.pair >= 0) {
    const bool known = position >= 0 && position < p.tables.rows;
    if (!known) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
    float c[N], s[N];
    if (known) {
      load_angles<T>(p.tables, position, at.pair, c, s);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] = s[i] = NAN;
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
      float x[N], y[N];
#pragma unroll
      for (int j = 0; j < N; ++j) { x[j] = to_f(a[i].v[j]); y[j] = to_f(b[i].v[j]); }
      turn_chunks<N>(x, y, c, s, p.interleaved != 0, p.tables.pairs - at.pair);
      a[i] = to_chunk<T>(x);
      b[i] = to_chunk<T>(y);
    }
  }
  T *out = static_cast<T *>(p.output) + token * p.out_token;
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    if (h0 + i >= p.heads) break;
    T *row = out + (int64_t)(h0 + i) * p.out_head;
    *reinterpret_cast<Chunk<T> *>(row + at.first) = a[i];
    if (at.second >= 0) *reinterpret_cast<Chunk<T> *>(row + at.second) = b[i];
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) chunk_kernel(Params p, uint32_t total) {
  const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
  if (i >= total) return;
  const uint32_t c = i % (uint32_t)p.chunk_pairs, r = i / (uint32_t)p.chunk_pairs;
  const uint32_t g = r % (uint32_t)p.head_groups, token = r / (uint32_t)p.head_groups;
  const int64_t position = p.positions[token];  // on its way with the loads of elements
  rotate_heads<T>(p, token, true, (int)g * HEADS, (int)c, [&] { return position; });
}

// Any strides, any head and rotary extents: a thread per pair or copied element.
// 16384 tokens of 40 heads of 96 bfloat16 elements: 295 us with 24 of them rotated
// where chunk_kernel takes 61 us with 48.
template <typename T>
__global__ void __launch_bounds__(THREADS) scalar_kernel(Params p, uint32_t total) {
  const uint32_t i = blockIdx.x * THREADS + threadIdx.x;
  if (i >= total) return;
  const int per_head = p.head_dim - p.tables.pairs;  // pairs, then copied elements
  const int e = (int)(i % (uint32_t)per_head);
  const uint32_t r = i / (uint32_t)per_head;
  const int h = (int)(r % (uint32_t)p.heads);
  const int64_t token = r / (uint32_t)p.heads;
  const T *in = static_cast<const T *>(p.input) + token * p.in_token + (int64_t)h * p.in_head;
  T *out = static_cast<T *>(p.output) + token * p.out_token + (int64_t)h * p.out_head;
  if (e >= p.tables.pairs) {
    const int64_t d = e + p.tables.pairs;
    out[d * p.out_dim] = in[d * p.in_dim];
    return;
  }
  const int64_t position = p.positions[token];
  const bool known = position >= 0 && position < p.tables.rows;
  if (!known) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
  const int64_t d0 = p.interleaved ? 2 * e : e, d1 = p.interleaved ? 2 * e + 1 : e + p.tables.pairs;
  float a = to_f(in[d0 * p.in_dim]), b = to_f(in[d1 * p.in_dim]);
  const float c = known ? p.tables.cos[position * p.tables.cos_stride + e] : NAN;
  const float s = known ? p.tables.sin[position * p.tables.sin_stride + e] * p.tables.sign : NAN;
  turn(a, b, c, s);
  out[d0 * p.out_dim] = from_f<T>(a);
  out[d1 * p.out_dim] = from_f<T>(b);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Whether tables can be read four columns at a time.
inline bool vector_tables(const Tables &t) {
  return aligned16(t.cos) && aligned16(t.sin) && t.cos_stride % 4 == 0 && t.sin_stride % 4 == 0 && t.pairs % 4 == 0;
}

// Whether heads of `head_dim` elements at this base and these strides are whole
// 16-byte chunks, and the rotated part whole chunk pairs (half layout) or whole
// chunks (interleaved).
template <typename T>
inline bool vector_heads(const void *base, int64_t token, int64_t head, int64_t dim, int64_t head_dim, int64_t pairs,
                         bool interleaved) {
  constexpr int N = Chunk<T>::N;
  return aligned16(base) && dim == 1 && token % N == 0 && head % N == 0 && head_dim % N == 0 &&
         (interleaved ? 2 * pairs : pairs) % N == 0;
}

template <typename T>
int launch(Params p, int64_t tokens, cudaStream_t stream) {
  const int64_t pairs = p.tables.pairs;
  const bool vec = vector_tables(p.tables) &&
                   vector_heads<T>(p.input, p.in_token, p.in_head, p.in_dim, p.head_dim, pairs, p.interleaved) &&
                   vector_heads<T>(p.output, p.out_token, p.out_head, p.out_dim, p.head_dim, pairs, p.interleaved);
  constexpr int N = Chunk<T>::N;
  p.chunk_pairs = (p.head_dim + 2 * N - 1) / (2 * N);
  p.head_groups = (p.heads + HEADS - 1) / HEADS;
  const int64_t per_token = vec ? (int64_t)p.chunk_pairs * p.head_groups : (int64_t)p.heads * (p.head_dim - pairs);
  // 32-bit thread indices: more work than that goes in several launches
  const int64_t slab = ((1LL << 31) - THREADS) / per_token;
  if (slab <= 0) return NT_B200_ERR_INVALID_ARGUMENT;
  const int64_t index_size = p.positions.wide ? 8 : 4;
  for (int64_t t0 = 0; t0 < tokens; t0 += slab) {
    const int64_t n = tokens - t0 < slab ? tokens - t0 : slab;
    Params q = p;
    q.input = static_cast<const T *>(p.input) + t0 * p.in_token;
    q.output = static_cast<T *>(p.output) + t0 * p.out_token;
    q.positions.data = static_cast<const char *>(p.positions.data) + t0 * p.positions.stride * index_size;
    const uint32_t total = (uint32_t)(n * per_token);
    const unsigned grid = (total + THREADS - 1) / THREADS;
    if (vec) chunk_kernel<T><<<grid, THREADS, 0, stream>>>(q, total);
    else scalar_kernel<T><<<grid, THREADS, 0, stream>>>(q, total);
    const int rc = launch_status();
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace rotary
}  // namespace nt

extern "C" int nt_b200_rotary(const NtB200RotaryArgs *a, void *stream) {
  if (!a || a->tokens < 0 || a->heads < 0 || a->head_dim < 0 || a->rotary_dim < 0 || a->rotary_dim % 2 != 0 ||
      a->table_rows < 0)
    return NT_B200_ERR_INVALID_ARGUMENT;
  if (!nt::is_float_dtype((int)a->dtype) || !nt::is_index_dtype(a->index_dtype)) return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->rotary_dim > a->head_dim) return NT_B200_ERR_SHAPE_MISMATCH;
  if (a->tokens == 0 || a->heads == 0 || a->head_dim == 0) return 0;
  if (!a->input || !a->output || !a->positions || (a->rotary_dim > 0 && (!a->cos || !a->sin)) ||
      a->heads > (1 << 30) || a->head_dim > (1 << 20))
    return NT_B200_ERR_INVALID_ARGUMENT;
  nt::rotary::Params p{};
  p.input = a->input;
  p.output = a->output;
  p.tables = {a->cos, a->sin, a->cos_stride, a->sin_stride, a->table_rows, (int)(a->rotary_dim / 2),
              a->adjoint ? -1.f : 1.f};
  p.positions = {a->positions, a->positions_stride, a->index_dtype == NT_B200_INT64};
  p.in_token = a->input_strides[0]; p.in_head = a->input_strides[1]; p.in_dim = a->input_strides[2];
  p.out_token = a->output_strides[0]; p.out_head = a->output_strides[1]; p.out_dim = a->output_strides[2];
  p.heads = (int)a->heads;
  p.head_dim = (int)a->head_dim;
  p.interleaved = a->interleaved != 0;
  return NT_DISPATCH_FLOAT((int)a->dtype,
                           [&] { return nt::rotary::launch<scalar_t>(p, a->tokens, static_cast<cudaStream_t>(stream)); });
}
