// Root-mean-square norm of rows, after the residual's addition, with an output
// in the rows' type or in 8 bits:
//     t = round(x + residual)                     (t = x without a residual)
//     y = (t * r) * w,   r = 1 / sqrt(mean(t^2) + eps)
//     output = round(y), or codes round(y * (1 / s)) with a scale s for each group
// What is normed is the sum as it is stored, so that a later pass over the stored
// residual gives the same row.  Squares are summed in 64 bits (16-bit elements'
// squares exactly) and r is rounded once: a code then follows from the formula and
// does not hang on the order of a sum.  At 4 elements a clock and SM of memory
// bandwidth that costs a quarter of the 64-bit units' rate and no time.
//
// Bound by memory: a row is read once, stays in registers and is written once.
// Measured: 16384 x 4096 bfloat16 with a residual to e4m3 88 us, 5.3 TB/s (issue at 0.69 of
// its limit, DRAM 0.82 of the copy rate), to bfloat16 without one 58 us, 4.6 TB/s; 3001 x
// 5120 float16 to int8 in groups of 128 18-19 us; 32 x 4096 2.4 us, the launch; rows off the
// 16-byte grid, 12000 x 5003 bfloat16 with a residual, 129 us, 3.7 TB/s, 212 to e4m3.
#pragma once

#include <type_traits>

#include "attention_tc.cuh"
#include "common.cuh"
#include "paged_append.cuh"

namespace nt {
namespace norm {

struct Params {
  const void *input, *residual, *weight;  // residual may be null
  void *output, *total;                   // total: with a residual
  float *scale;                           // with codes
  int64_t rows, in_row, in_col, res_row, res_col, w_col, out_row, out_col, tot_row, tot_col, s_row, s_col;
  int width, group, groups;   // group: elements that share a scale
  uint32_t group_reciprocal;  // ceil(2^28 / group)
  double eps;
};

constexpr int UNIT = 8;  // elements a thread takes at a time
constexpr int MOST_THREADS = 512;
template <typename T> struct alignas(sizeof(T) * UNIT >= 16 ? 16 : 8) Unit { T v[UNIT]; };

template <typename T> __device__ __forceinline__ Unit<T> load_unit(const T *at) {
  return *reinterpret_cast<const Unit<T> *>(at);
}

// The sum (largest) over the threads that share a row: a warp, or the block.
template <typename V, typename F>
__device__ __forceinline__ V reduce(V v, V *warps, bool block, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (!block) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, count = blockDim.x >> 5;
  if (lane == 0) warps[warp] = v;
  __syncthreads();
  v = warps[lane < count ? lane : 0];
  const V none = V(0);
  if (lane >= count) v = none;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float inverse_rms(double sum, int width, double eps) {
  return (float)(1.0 / sqrt(sum / width + eps));
}

__device__ __forceinline__ void raise(int *slot, float magnitude) {  // magnitudes order as their bits do
  atomicMax(slot, __float_as_int(magnitude));
}

template <typename C> struct IsCode { static constexpr bool value = false; };
template <> struct IsCode<int8_t> { static constexpr bool value = true; };
template <> struct IsCode<__nv_fp8_e4m3> { static constexpr bool value = true; };

// Two elements from fp32, in one conversion.
template <typename T> __device__ __forceinline__ void to_pair(T *to, float a, float b) {
  if constexpr (sizeof(T) == 4) {
    to[0] = a;
    to[1] = b;
  } else {
    *reinterpret_cast<uint32_t *>(to) = tc::attn::pack2<T>(a, b);
  }
}

// The larger of m and |x|, or NaN where either is.
__device__ __forceinline__ float most_or_nan(float m, float x) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(m), "f"(fabsf(x)));
  return y;
}

// Eight codes of values that the scale covers: none leaves the range.  1.5 * 2^23 + x
// holds x, rounded to a whole number, in its low bits.
template <typename C> __device__ __forceinline__ void store_covered(uint8_t *to, const float (&x)[UNIT], float inv) {
  if constexpr (std::is_same<C, int8_t>::value) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = __float_as_uint(__fadd_rn(__fmul_rn(x[4 * i + k], inv), 12582912.f));
      w[i] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
    *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
  } else {
    paged::store_codes<C, UNIT>(to, x, inv);
  }
}

// Rows in registers: blockDim.x threads a row, blockDim.y rows a block (more than
// one only where a warp takes a row).  O: the output's element type.
template <typename T, typename W, typename O, int PER>
__global__ void __launch_bounds__(MOST_THREADS) rows_kernel(const __grid_constant__ Params p) {
  constexpr bool CODES = IsCode<O>::value;
  __shared__ double sums[32];
  __shared__ float tops[32];
  extern __shared__ int slots[];  // with groups that a warp's shuffles do not cover: one a group
  const bool block = blockDim.x > 32;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  wait_prior_grid();
  allow_dependent_launch();
  if (row >= p.rows) return;  // a whole warp
  const T *x = static_cast<const T *>(p.input) + row * p.in_row;
  const T *res = static_cast<const T *>(p.residual) + row * p.res_row;
  const W *w = static_cast<const W *>(p.weight);
  const int units = p.width / UNIT;
  constexpr int BATCH = PER < 4 ? PER : 4;
  Unit<T> t[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int u = threadIdx.x + i * blockDim.x;
    if (u < units) t[i] = load_unit(x + u * UNIT);
  }
  if (p.residual) {
#pragma unroll
    for (int b = 0; b < PER; b += BATCH) {
      Unit<T> r[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int u = threadIdx.x + (b + i) * blockDim.x;
        if (u < units) r[i] = load_unit(res + u * UNIT);
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        const int u = threadIdx.x + (b + i) * blockDim.x;
        if (u >= units) continue;
#pragma unroll
        for (int e = 0; e < UNIT; e += 2)
          to_pair(&t[b + i].v[e], to_f(t[b + i].v[e]) + to_f(r[i].v[e]), to_f(t[b + i].v[e + 1]) + to_f(r[i].v[e + 1]));
        *reinterpret_cast<Unit<T> *>(static_cast<T *>(p.total) + row * p.tot_row + u * UNIT) = t[b + i];
      }
    }
  }
  // the weight waits in registers where there is room, else it comes when used
  constexpr bool AHEAD = PER <= 4;
  Unit<W> weight[AHEAD ? PER : 1];
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * blockDim.x;
      if (u < units) weight[i] = load_unit(w + u * UNIT);
    }
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (threadIdx.x + i * blockDim.x >= units) continue;
#pragma unroll
    for (int e = 0; e < UNIT; ++e) {
      const double d = (double)to_f(t[i].v[e]);
      sum = fma(d, d, sum);
    }
  }
  sum = reduce(sum, sums, block, [](double a, double b) { return a + b; });
  const float r = inverse_rms(sum, p.width, p.eps);
  // y, once where there is room for it
  const auto product = [&](int i, const Unit<W> &v, float (&y)[UNIT]) {
#pragma unroll
    for (int e = 0; e < UNIT; ++e) y[e] = __fmul_rn(__fmul_rn(to_f(t[i].v[e]), r), to_f(v.v[e]));
  };
  float kept[AHEAD ? PER : 1][UNIT];
  if constexpr (AHEAD) {
#pragma unroll
    for (int i = 0; i < PER; ++i) product(i, weight[i], kept[i]);
  }
  const auto values = [&](int i, float (&y)[UNIT]) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int e = 0; e < UNIT; ++e) y[e] = kept[i][e];
    } else {
      product(i, load_unit(w + (threadIdx.x + i * blockDim.x) * UNIT), y);
    }
  };

  O *out = static_cast<O *>(p.output) + row * p.out_row;
  if constexpr (!CODES) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * blockDim.x;
      if (u >= units) continue;
      float y[UNIT];
      values(i, y);
      Unit<O> o;
#pragma unroll
      for (int e = 0; e < UNIT; e += 2) to_pair(&o.v[e], y[e], y[e + 1]);
      *reinterpret_cast<Unit<O> *>(out + u * UNIT) = o;
    }
  } else {
    float top[PER];
    uint32_t odd = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      top[i] = 0.f;
      if (threadIdx.x + i * blockDim.x >= units) continue;
      float y[UNIT];
      values(i, y);
#pragma unroll
      for (int e = 0; e < UNIT; ++e) top[i] = most_or_nan(top[i], y[e]);
      if (!(top[i] < INFINITY)) {  // (rare) what is not finite does not count
        odd |= 1u << i;
        top[i] = 0.f;
#pragma unroll
        for (int e = 0; e < UNIT; ++e) top[i] = fmaxf(top[i], paged::finite_magnitude(y[e]));
      }
    }
    const auto most = [](float a, float b) { return fmaxf(a, b); };
    const int share = p.group / UNIT;  // threads of a group
    const bool lanes = p.groups > 1 && share <= 32 && (share & (share - 1)) == 0;
    if (p.groups == 1) {
      float m = top[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) m = fmaxf(m, top[i]);
      m = reduce(m, tops, block, most);
#pragma unroll
      for (int i = 0; i < PER; ++i) top[i] = m;
    } else if (lanes) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        for (int o = share >> 1; o > 0; o >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
    } else {
      int *mine = slots + threadIdx.y * p.groups;
      for (int g = threadIdx.x; g < p.groups; g += blockDim.x) mine[g] = 0;
      if (block) __syncthreads();
      else __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int u = threadIdx.x + i * blockDim.x;
        if (u < units) raise(mine + u * UNIT / p.group, top[i]);
      }
      if (block) __syncthreads();
      else __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int u = threadIdx.x + i * blockDim.x;
        if (u < units) top[i] = __int_as_float(mine[u * UNIT / p.group]);
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int u = threadIdx.x + i * blockDim.x;
      if (u >= units) continue;
      float y[UNIT];
      values(i, y);
      const float s = paged::block_scale<O>(top[i]);
      uint8_t *to = reinterpret_cast<uint8_t *>(out) + u * UNIT;
      if (odd >> i & 1) paged::store_codes<O, UNIT>(to, y, __frcp_rn(s));
      else store_covered<O>(to, y, __frcp_rn(s));
      if (p.groups == 1) {
        if (u == 0) p.scale[row * p.s_row] = s;
      } else if (lanes) {
        if ((u & (share - 1)) == 0) p.scale[row * p.s_row + (u >> (__ffs(share) - 1)) * p.s_col] = s;
      } else if (u * UNIT % p.group == 0) {
        p.scale[row * p.s_row + u * UNIT / p.group * p.s_col] = s;
      }
    }
  }
}

// Rows off the 16-byte grid: a block a row, its elements dealt out one by one and kept in
// registers.  Of 12000 x 5003 bfloat16 with a residual, 64-bit places and runtime strides
// took 430 us.
template <typename T, typename W, typename O, int PER, int THREADS>
__global__ void __launch_bounds__(THREADS) elements_kernel(const __grid_constant__ Params p) {
  constexpr bool CODES = IsCode<O>::value;
  __shared__ double sums[32];
  __shared__ float tops[32];
  extern __shared__ int slots[];
  wait_prior_grid();
  allow_dependent_launch();
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.input) + row * p.in_row;
  const T *res = static_cast<const T *>(p.residual) + row * p.res_row;
  const W *w = static_cast<const W *>(p.weight);
  T *total = static_cast<T *>(p.total) + row * p.tot_row;
  float y[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (int)threadIdx.x + i * THREADS;
    y[i] = c < p.width ? to_f(x[c]) : 0.f;
  }
  if (p.residual) {
    float r[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (int)threadIdx.x + i * THREADS;
      r[i] = c < p.width ? to_f(res[c]) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (int)threadIdx.x + i * THREADS;
      const T t = from_f<T>(y[i] + r[i]);
      y[i] = to_f(t);
      if (c < p.width) total[c] = t;
    }
  }
  double sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum = fma((double)y[i], (double)y[i], sum);
  if (CODES && p.groups > 1)
    for (int g = threadIdx.x; g < p.groups; g += THREADS) slots[g] = 0;
  sum = reduce(sum, sums, true, [](double a, double b) { return a + b; });
  const float r = inverse_rms(sum, p.width, p.eps);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int c = (int)threadIdx.x + i * THREADS;
    y[i] = c < p.width ? __fmul_rn(__fmul_rn(y[i], r), to_f(w[c])) : 0.f;
  }
  O *out = static_cast<O *>(p.output) + row * p.out_row;
  if constexpr (!CODES) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (int)threadIdx.x + i * THREADS;
      if (c < p.width) out[c] = from_f<O>(y[i]);
    }
  } else {
    float inverse = 0.f;
    // c / group, exactly: c and the group are less than 2^14 here
    const auto group_of = [&](int c) { return (int)__umulhi((uint32_t)c << 4, p.group_reciprocal); };
    if (p.groups == 1) {
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) top = fmaxf(top, paged::finite_magnitude(y[i]));
      top = reduce(top, tops, true, [](float a, float b) { return fmaxf(a, b); });
      const float s = paged::block_scale<O>(top);
      inverse = __frcp_rn(s);
      if (threadIdx.x == 0) p.scale[row * p.s_row] = s;
    } else {
      // 16 neighbouring lanes have elements of one group
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int c = (int)threadIdx.x + i * THREADS;
        float m = paged::finite_magnitude(y[i]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 15) == 0 && c < p.width) raise(slots + group_of(c), m);
      }
      __syncthreads();
      for (int g = threadIdx.x; g < p.groups; g += THREADS) {
        const float s = paged::block_scale<O>(__int_as_float(slots[g]));
        p.scale[row * p.s_row + g * p.s_col] = s;
        slots[g] = __float_as_int(__frcp_rn(s));
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int c = (int)threadIdx.x + i * THREADS;
      if (c >= p.width) continue;
      const float by = p.groups == 1 ? inverse : __int_as_float(slots[group_of(c)]);
      reinterpret_cast<uint8_t *>(out)[c] = paged::encode<O>(__fmul_rn(y[i], by));
    }
  }
}

// Any layout and width: a block a row, an element at a time, the row read again
// (from the caches) for each pass.  2048 x 20003 bfloat16 115 us, 1.4 TB/s, 359 to e4m3 in
// groups of 128; 4096 x 4096, every second column of a wider tensor, 63 us.
template <typename T, typename W, typename O>
__global__ void __launch_bounds__(MOST_THREADS) any_kernel(const __grid_constant__ Params p) {
  constexpr bool CODES = IsCode<O>::value;
  __shared__ double sums[32];
  extern __shared__ int slots[];
  wait_prior_grid();
  allow_dependent_launch();
  const int64_t row = blockIdx.x;
  const T *x = static_cast<const T *>(p.input) + row * p.in_row;
  const T *res = static_cast<const T *>(p.residual) + row * p.res_row;
  const W *w = static_cast<const W *>(p.weight);
  T *total = static_cast<T *>(p.total) + row * p.tot_row;
  double sum = 0;
  for (int64_t c = threadIdx.x; c < p.width; c += blockDim.x) {
    T t = x[c * p.in_col];
    if (p.residual) {
      t = from_f<T>(to_f(t) + to_f(res[c * p.res_col]));
      total[c * p.tot_col] = t;
    }
    const double d = (double)to_f(t);
    sum = fma(d, d, sum);
  }
  if (CODES)
    for (int g = threadIdx.x; g < p.groups; g += blockDim.x) slots[g] = 0;
  sum = reduce(sum, sums, true, [](double a, double b) { return a + b; });
  const float r = inverse_rms(sum, p.width, p.eps);
  // a thread reads back what it wrote itself
  const auto value = [&](int64_t c) {
    const float t = to_f(p.residual ? total[c * p.tot_col] : x[c * p.in_col]);
    return __fmul_rn(__fmul_rn(t, r), to_f(w[c * p.w_col]));
  };
  O *out = static_cast<O *>(p.output) + row * p.out_row;
  if constexpr (!CODES) {
    for (int64_t c = threadIdx.x; c < p.width; c += blockDim.x) out[c * p.out_col] = from_f<O>(value(c));
  } else {
    for (int64_t c = threadIdx.x; c < p.width; c += blockDim.x)
      raise(slots + c / p.group, paged::finite_magnitude(value(c)));
    __syncthreads();
    for (int64_t c = threadIdx.x; c < p.width; c += blockDim.x) {
      const float s = paged::block_scale<O>(__int_as_float(slots[c / p.group]));
      reinterpret_cast<uint8_t *>(out)[c * p.out_col] = paged::encode<O>(__fmul_rn(value(c), __frcp_rn(s)));
      if (c % p.group == 0) p.scale[row * p.s_row + c / p.group * p.s_col] = s;
    }
  }
}

constexpr int MOST_WIDTH = 131072;  // with it, a scale for each 16 elements fits shared memory

template <typename T> bool vector_rows(const void *base, int64_t row, int64_t col) {
  constexpr int64_t bytes = sizeof(T) * UNIT < 16 ? sizeof(T) * UNIT : 16;
  return (reinterpret_cast<uintptr_t>(base) % bytes) == 0 && col == 1 && row * (int64_t)sizeof(T) % bytes == 0;
}

template <typename T, typename W, typename O> int launch(const Params &p, cudaStream_t stream) {
  constexpr bool CODES = IsCode<O>::value;
  const int units = p.width / UNIT;
  const bool vec = p.width % UNIT == 0 && units <= 8 * MOST_THREADS && (p.groups == 1 || p.group % UNIT == 0) &&
                   vector_rows<T>(p.input, p.in_row, p.in_col) && vector_rows<W>(p.weight, 0, p.w_col) &&
                   vector_rows<O>(p.output, p.out_row, p.out_col) &&
                   (!p.residual || (vector_rows<T>(p.residual, p.res_row, p.res_col) &&
                                    vector_rows<T>(p.total, p.tot_row, p.tot_col)));
  if (p.rows > (1LL << 31) - 1) return NT_B200_ERR_INVALID_ARGUMENT;
  const size_t slots = CODES ? (size_t)p.groups * sizeof(int) : 0;
  const bool dense = p.in_col == 1 && p.w_col == 1 && p.out_col == 1 && (!p.residual || (p.res_col == 1 && p.tot_col == 1));
  if (!vec && dense && p.width <= 32 * MOST_THREADS) {
    const auto go = [&](auto per, auto count) {
      constexpr int PER = decltype(per)::value, THREADS = decltype(count)::value;
      return launch_overlapped(elements_kernel<T, W, O, PER, THREADS>, dim3((unsigned)p.rows), dim3(THREADS), slots, stream, p);
    };
    if (p.width <= 4 * 256) return go(std::integral_constant<int, 4>{}, std::integral_constant<int, 256>{});
    if (p.width <= 24 * 256) return go(std::integral_constant<int, 24>{}, std::integral_constant<int, 256>{});
    return go(std::integral_constant<int, 32>{}, std::integral_constant<int, MOST_THREADS>{});
  }
  if (!vec) {
    const unsigned threads = p.width < MOST_THREADS ? (unsigned)(p.width + 31) / 32 * 32 : MOST_THREADS;
    return launch_overlapped(any_kernel<T, W, O>, dim3((unsigned)p.rows), dim3(threads), slots, stream, p);
  }
  const auto go = [&](auto per) {
    constexpr int PER = decltype(per)::value;
    const unsigned threads = (unsigned)((units + PER - 1) / PER + 31) / 32 * 32;
    const unsigned rows = threads == 32 ? 4 : 1;
    const unsigned grid = (unsigned)((p.rows + rows - 1) / rows);
    return launch_overlapped(rows_kernel<T, W, O, PER>, dim3(grid), dim3(threads, rows), slots * rows, stream, p);
  };
  // Units a thread.  16384 x 4096 bfloat16 to e4m3 take 88 us at 4 and 100 at 2; 32 rows,
  // which are latency, 2.8 and 2.6.
  if (units <= 64 || (units <= 1024 && p.rows <= 2 * sm_count())) return go(std::integral_constant<int, 2>{});
  if (units <= 2048) return go(std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 8>{});
}

template <typename T, typename W> int dispatch_output(const Params &p, int64_t output_dtype, int64_t dtype, cudaStream_t s) {
  if (output_dtype == dtype) return launch<T, W, T>(p, s);
  if (output_dtype == NT_B200_INT8) return launch<T, W, int8_t>(p, s);
  if (output_dtype == NT_B200_FLOAT8_E4M3FN) return launch<T, W, __nv_fp8_e4m3>(p, s);
  return NT_B200_ERR_UNSUPPORTED_DTYPE;
}

}  // namespace norm
}  // namespace nt

extern "C" int nt_b200_rms_norm(const NtB200RmsNormArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->rows < 0 || a->width < 0 || a->group < 0) return NT_B200_ERR_INVALID_ARGUMENT;
  if (!is_float_dtype((int)a->dtype) || (a->weight_dtype != a->dtype && a->weight_dtype != NT_B200_FLOAT32))
    return NT_B200_ERR_UNSUPPORTED_DTYPE;
  const bool codes = a->output_dtype != a->dtype;
  if (codes && a->output_dtype != NT_B200_INT8 && a->output_dtype != NT_B200_FLOAT8_E4M3FN)
    return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->rows == 0 || a->width == 0) return 0;
  if (a->width > norm::MOST_WIDTH || (codes && (a->group == 0 || (a->group < a->width && a->group % 16 != 0))))
    return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->input || !a->weight || !a->output || (codes && !a->scale) || (a->residual && !a->total) || !(a->eps >= 0))
    return NT_B200_ERR_INVALID_ARGUMENT;
  norm::Params p{};
  p.input = a->input; p.residual = a->residual; p.weight = a->weight;
  p.output = a->output; p.total = a->total; p.scale = a->scale;
  p.rows = a->rows; p.width = (int)a->width;
  p.group = codes ? (int)(a->group < a->width ? a->group : a->width) : p.width;
  p.groups = (p.width + p.group - 1) / p.group;
  p.group_reciprocal = (uint32_t)((0xfffffffLL + p.group) / p.group);
  p.in_row = a->input_strides[0]; p.in_col = a->input_strides[1];
  p.res_row = a->residual_strides[0]; p.res_col = a->residual_strides[1];
  p.w_col = a->weight_stride;
  p.out_row = a->output_strides[0]; p.out_col = a->output_strides[1];
  p.tot_row = a->total_strides[0]; p.tot_col = a->total_strides[1];
  p.s_row = a->scale_strides[0]; p.s_col = a->scale_strides[1];
  p.eps = a->eps;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return NT_DISPATCH_FLOAT((int)a->dtype, [&] {
    if (a->weight_dtype == a->dtype) return norm::dispatch_output<scalar_t, scalar_t>(p, a->output_dtype, a->dtype, s);
    return norm::dispatch_output<scalar_t, float>(p, a->output_dtype, a->dtype, s);
  });
}
