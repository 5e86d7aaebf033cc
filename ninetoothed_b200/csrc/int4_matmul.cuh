// Product of a few rows with a matrix of 4-bit weights:
//     y[m, n] = input_scale[m] * sum_k x[m, k] * (code[n, k] - zero[n, k / G]) * scale[n, k / G]
// with two codes a byte, the even element in the low half, and a zero point of 8
// where none are given.
//
// Bound by memory: a weight is half a byte and serves every row of x, 4 flops a
// byte and row.  The weights go through shared memory once; x comes from L2.
//
// Codes become 16-bit floats without rounding (their bits set into the mantissa
// of 1024, or of 128 in bfloat16, and the zero point taken off, which leaves a
// whole number), x keeps its type (8-bit x becomes fp16, exactly), and tensor
// cores sum a group's products in fp32.  The scale then multiplies the group's
// sum in fp32, so that nothing is rounded but the fp32 sums and the result.
//
// 16x8x16 steps take 16 weight rows as their rows and 8 rows of x as their
// columns.  Any order of the contracted elements is as good as another, so a lane
// takes eight neighbouring weights, one 32-bit word, whose halves' equal places
// make the pairs (0, 4), (1, 5), (2, 6), (3, 7): a shift, a mask and a
// subtraction for two weights, and one permute for two elements of x.
//
// A block has 8 warps and 32 * WR weight rows; a stage of its ring holds KS = 1024
// / WR columns of them, 16 KB at any WR, and x's columns beside it.  A warp takes
// 32 rows and 128 columns of a stage.  More rows of x take more weight rows a
// block, so that x is never more than the weights.  Where the weight rows are too
// few for the SMs, a cluster's blocks share the columns and join their sums
// through distributed shared memory, always in the same order.
#pragma once

#include "common.cuh"
#include "paged_attention.cuh"
#include "ptx.cuh"

namespace nt {
namespace four_bit {

struct Params {
  const void *x;
  const uint8_t *codes, *scales, *zeros;  // zeros may be null
  const float *x_scale;                   // or null
  void *y;
  int64_t x_row, x_col, c_row, c_col, s_row, s_col, z_row, z_col, xs_stride, y_row, y_col;
  int64_t rows, inner, outer;
  int groups, group;  // of a weight row; weights of a group
  int scale_dtype, y_dtype;
  int parts;          // of the columns: blocks of a cluster
  int stages;         // of the columns, all parts together
  uint32_t group32;   // 32-column steps of a group
  int scale_words, zero_words;           // 4-byte words of a weight row in a stage
  int x_bytes, stage_bytes;              // x's part of a stage; the whole
};

__device__ __forceinline__ float any_float(const uint8_t *at, int dtype) {
  if (dtype == NT_B200_FLOAT32) return *reinterpret_cast<const float *>(at);
  if (dtype == NT_B200_FLOAT16) return __half2float(*reinterpret_cast<const __half *>(at));
  return __bfloat162float(*reinterpret_cast<const __nv_bfloat16 *>(at));
}
__device__ __forceinline__ void store_any(void *y, int64_t at, int dtype, float v) {
  if (dtype == NT_B200_FLOAT32) static_cast<float *>(y)[at] = v;
  else if (dtype == NT_B200_FLOAT16) static_cast<__half *>(y)[at] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
}
__host__ __device__ constexpr int float_size(int dtype) { return dtype == NT_B200_FLOAT32 ? 4 : 2; }

// ---------------------------------------------------------------- any layout
// A warp a weight row and 8 rows of x: 32-bit floats, strides off the 16-byte grid.
template <typename X>
__global__ void __launch_bounds__(128) rows_kernel(const __grid_constant__ Params p) {
  constexpr int M = 8;
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), m0 = (int64_t)blockIdx.y * M;
  if (n >= p.outer) return;
  const X *x = static_cast<const X *>(p.x) + m0 * p.x_row;
  const int count = (int)(p.rows - m0 < M ? p.rows - m0 : M);
  float sum[M] = {};
  for (int64_t b = lane; b < p.inner / 2; b += 32) {
    const int64_t g = 2 * b / p.group;
    const uint8_t code = p.codes[n * p.c_row + b * p.c_col];
    const float s = any_float(p.scales + (n * p.s_row + g * p.s_col) * float_size(p.scale_dtype), p.scale_dtype);
    const float z = p.zeros ? (float)(p.zeros[n * p.z_row + g * p.z_col] & 15) : 8.f;
    const float w0 = ((float)(code & 15) - z) * s, w1 = ((float)(code >> 4) - z) * s;
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (m < count) {
        const X *at = x + m * p.x_row + 2 * b * p.x_col;
        sum[m] = fmaf(to_f(at[0]), w0, fmaf(to_f(at[p.x_col]), w1, sum[m]));
      }
  }
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], o);
    if (lane == 0 && m < count) {
      const float f = p.x_scale ? p.x_scale[(m0 + m) * p.xs_stride] : 1.f;
      store_any(p.y, (m0 + m) * p.y_row + n * p.y_col, p.y_dtype, p.x_scale ? sum[m] * f : sum[m]);
    }
  }
}

// ---------------------------------------------------------------- tensor cores
constexpr int WARPS = 8, THREADS = WARPS * 32, RING = 4;

// Two 16-bit floats from the low four bits of w's halves, less the zero point.
template <typename F> struct Codes;
template <> struct Codes<__half> {
  static constexpr uint32_t ONE = 0x64006400u;  // 1024, twice
  static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t zero) {
    const uint32_t bits = (w & 0x000f000fu) | ONE;
    const __half2 v = __hsub2(*reinterpret_cast<const __half2 *>(&bits), *reinterpret_cast<const __half2 *>(&zero));
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    paged::mma16816(d, a[0], a[1], a[2], a[3], b0, b1);
  }
};
template <> struct Codes<__nv_bfloat16> {
  static constexpr uint32_t ONE = 0x43004300u;  // 128, twice
  static __device__ __forceinline__ uint32_t pair(uint32_t w, uint32_t zero) {
    const uint32_t bits = (w & 0x000f000fu) | ONE;
    const __nv_bfloat162 v =
        __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&bits), *reinterpret_cast<const __nv_bfloat162 *>(&zero));
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <typename X> struct Operand { using type = __half; };  // 8-bit x
template <> struct Operand<__nv_bfloat16> { using type = __nv_bfloat16; };

__device__ __forceinline__ uint32_t load_shared4(uint32_t from) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
  return v;
}
__device__ __forceinline__ void copy_async4(uint32_t to, const void *from, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <typename X, int NT> struct Layout {
  static constexpr int WR = NT, WK = WARPS / WR;
  static constexpr int R = 32 * WR, KS = 128 * WK;  // weight rows; columns of a stage
  static constexpr int M = 8 * NT;                  // rows of x
  static constexpr int CODES = R * KS / 2;
  // x's rows in a stage, moved so that the rows a quarter (8-bit x: half) of a warp
  // loads at once start in different banks
  static constexpr int X_PITCH = KS * (int)sizeof(X) + 32 * (int)sizeof(X);
  static constexpr int JOIN = WARPS * 32 * M * 4;  // the warps' sums, at the end
  static_assert(CODES == 16384, "a stage's codes");
};

template <typename X, int NT>
__global__ void __launch_bounds__(THREADS, 2) tiles_kernel(const __grid_constant__ Params p) {
  using L = Layout<X, NT>;
  using F = typename Operand<X>::type;
  constexpr int XS = sizeof(X);
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wr = warp % L::WR, wk = warp / L::WR, g = lane >> 2, c = lane & 3;
  const int part = (int)(blockIdx.x % (unsigned)p.parts);
  const int64_t n0 = (int64_t)(blockIdx.x / (unsigned)p.parts) * L::R, m0 = (int64_t)blockIdx.y * L::M;
  const int m_count = (int)(p.rows - m0 < L::M ? p.rows - m0 : L::M);
  const int first = (int)((int64_t)p.stages * part / p.parts), last = (int)((int64_t)p.stages * (part + 1) / p.parts);
  const int scale_size = float_size(p.scale_dtype);
  wait_prior_grid();

  // ---- copies of a stage
  const auto copy = [&](int stage) {
    const uint32_t slot = base + (uint32_t)((stage - first) % RING) * (uint32_t)p.stage_bytes;
    const int64_t k0 = (int64_t)stage * L::KS;
    constexpr int CHUNKS = L::KS / 32;  // 16-byte chunks of a weight row
#pragma unroll
    for (int i = 0; i < L::CODES / 16 / THREADS; ++i) {
      const int at = threadIdx.x + i * THREADS, row = at / CHUNKS, q = at % CHUNKS;
      const bool valid = n0 + row < p.outer && k0 + q * 32 < p.inner;
      const uint8_t *from = valid ? p.codes + (n0 + row) * p.c_row + k0 / 2 + q * 16 : p.codes;
      paged::copy_async16(slot + row * (L::KS / 2) + ((q & ~7) | ((q ^ row) & 7)) * 16, from, valid);
    }
    constexpr int X_CHUNKS = L::KS * XS / 16;  // of a row of x
    for (int at = threadIdx.x; at < m_count * X_CHUNKS; at += THREADS) {
      const int m = at / X_CHUNKS, q = at % X_CHUNKS;
      const int64_t k = k0 + q * (16 / XS);
      const bool valid = k < p.inner;
      const uint8_t *from = static_cast<const uint8_t *>(p.x) + ((m0 + m) * p.x_row + (valid ? k : 0)) * XS;
      paged::copy_async16(slot + L::CODES + m * L::X_PITCH + q * 16, from, valid);
    }
    // scales and zero points: the words that hold a row's part, read no further
    // than the row
    const int row = threadIdx.x % L::R;
    if (n0 + row < p.outer) {
      const int g0 = (int)((uint32_t)k0 / (uint32_t)p.group);
      const int g1 = min(p.groups, (int)((uint32_t)(k0 + L::KS + p.group - 1) / (uint32_t)p.group));
      const auto words = [&](const uint8_t *array, int64_t row_stride, int size, int most, uint32_t to) {
        const int64_t from = ((n0 + row) * row_stride + g0) * size, until = ((n0 + row) * row_stride + g1) * size;
        const int64_t word0 = from & ~(int64_t)3;
        for (int w = threadIdx.x / L::R; w < most; w += THREADS / L::R) {
          const int64_t at = word0 + 4 * w;
          if (at < until) copy_async4(to + 4 * w, array + at, (int)min((int64_t)4, until - at));
        }
      };
      const uint32_t s_slot = slot + L::CODES + p.x_bytes;
      words(p.scales, p.s_row, scale_size, p.scale_words, s_slot + 4 * row * p.scale_words);
      if (p.zeros) words(p.zeros, p.z_row, 1, p.zero_words, s_slot + 4 * (L::R * p.scale_words + row * p.zero_words));
    }
  };

  float acc[2][NT][4] = {};
  // ---- a warp's share of a stage
  const auto consume = [&](int stage) {
    const uint32_t slot_at = (uint32_t)((stage - first) % RING) * (uint32_t)p.stage_bytes;
    const uint32_t slot = base + slot_at;
    const int64_t k0 = (int64_t)stage * L::KS;
    const uint32_t step0 = (uint32_t)(k0 / 32) + wk * 4;
    uint32_t gi = step0 / p.group32, left = p.group32 - (step0 - gi * p.group32);  // steps to the group's end
    const uint32_t g0 = (uint32_t)k0 / (uint32_t)p.group;
    const uint8_t *s_slot = smem + slot_at + L::CODES + p.x_bytes;
    const uint8_t *scale_at[4], *zero_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = wr * 32 + g + 8 * i;
      const uint32_t s_mis = (uint32_t)(((n0 + row) * p.s_row + g0) * scale_size) & 3u;
      scale_at[i] = s_slot + 4 * row * p.scale_words + s_mis;
      const uint32_t z_mis = (uint32_t)((n0 + row) * p.z_row + g0) & 3u;
      zero_at[i] = s_slot + 4 * (L::R * p.scale_words + row * p.zero_words) + z_mis;
    }
    uint32_t zero[4];
    const auto load_zeros = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        zero[i] = Codes<F>::ONE | (p.zeros ? (uint32_t)zero_at[i][gi - g0] & 15u : 8u) * 0x10001u;
    };
    float sum[2][NT][4] = {};
    load_zeros();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = wk * 4 + j;
      // x: eight elements a lane, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
      uint32_t b[NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int m = min(t * 8 + g, m_count - 1);  // columns past the last are not written
        const uint32_t at = slot + L::CODES + m * L::X_PITCH + (q * 32 + c * 8) * XS;
        uint4 v;
        if constexpr (XS == 2) {
          v = paged::load_shared16(at);
        } else {
          const uint2 w = paged::load_shared8(at);
          paged::to_halves<X>(w.x, v.x, v.y);
          paged::to_halves<X>(w.y, v.z, v.w);
        }
        b[t][0] = __byte_perm(v.x, v.z, 0x5410);
        b[t][1] = __byte_perm(v.x, v.z, 0x7632);
        b[t][2] = __byte_perm(v.y, v.w, 0x5410);
        b[t][3] = __byte_perm(v.y, v.w, 0x7632);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = wr * 32 + r * 16 + g;
        const uint32_t at = slot + row * (L::KS / 2) + ((q & ~7) | ((q ^ row) & 7)) * 16 + c * 4;
        const uint32_t lo = load_shared4(at), hi = load_shared4(at + 8 * (L::KS / 2));
        const uint32_t zl = zero[2 * r], zh = zero[2 * r + 1];
        const uint32_t a0[4] = {Codes<F>::pair(lo, zl), Codes<F>::pair(hi, zh), Codes<F>::pair(lo >> 4, zl),
                                Codes<F>::pair(hi >> 4, zh)};
        const uint32_t a1[4] = {Codes<F>::pair(lo >> 8, zl), Codes<F>::pair(hi >> 8, zh), Codes<F>::pair(lo >> 12, zl),
                                Codes<F>::pair(hi >> 12, zh)};
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          Codes<F>::mma(sum[r][t], a0, b[t][0], b[t][1]);
          Codes<F>::mma(sum[r][t], a1, b[t][2], b[t][3]);
        }
      }
      if (--left == 0 || j == 3) {
        // (past the last column there are no scales, and all x are 0)
        const bool some = gi < (uint32_t)p.groups;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float lo = some ? any_float(scale_at[2 * r] + (gi - g0) * scale_size, p.scale_dtype) : 0.f;
          const float hi = some ? any_float(scale_at[2 * r + 1] + (gi - g0) * scale_size, p.scale_dtype) : 0.f;
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            acc[r][t][0] = fmaf(lo, sum[r][t][0], acc[r][t][0]);
            acc[r][t][1] = fmaf(lo, sum[r][t][1], acc[r][t][1]);
            acc[r][t][2] = fmaf(hi, sum[r][t][2], acc[r][t][2]);
            acc[r][t][3] = fmaf(hi, sum[r][t][3], acc[r][t][3]);
            sum[r][t][0] = sum[r][t][1] = sum[r][t][2] = sum[r][t][3] = 0.f;
          }
        }
        if (left == 0) {
          left = p.group32;
          ++gi;
          if (j < 3) load_zeros();
        }
      }
    }
  };

  for (int s = first; s < first + RING - 1; ++s) {
    if (s < last) copy(s);
    paged::copy_commit();
  }
  for (int s = first; s < last; ++s) {
    paged::copy_wait<RING - 2>();
    __syncthreads();
    if (s + RING - 1 < last) copy(s + RING - 1);
    paged::copy_commit();
    consume(s);
  }
  allow_dependent_launch();
  paged::copy_wait<0>();
  __syncthreads();

  // ---- the warps' sums, [WK][M][R], then the cluster's
  float *joined = reinterpret_cast<float *>(smem);
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int m = t * 8 + 2 * c + (e & 1), row = wr * 32 + r * 16 + g + (e >> 1) * 8;
        joined[(wk * L::M + m) * L::R + row] = acc[r][t][e];
      }
  __syncthreads();
  for (int at = threadIdx.x; at < L::M * L::R; at += THREADS) {
    float v = joined[at];
#pragma unroll
    for (int w = 1; w < L::WK; ++w) v += joined[w * L::M * L::R + at];
    joined[at] = v;
  }
  if (p.parts > 1) ptx::cluster_sync();
  else __syncthreads();
  for (int at = threadIdx.x + part * THREADS; at < L::M * L::R; at += THREADS * p.parts) {
    const int m = at / L::R;
    const int64_t n = n0 + at % L::R;
    float v;
    if (p.parts == 1) {
      v = joined[at];
    } else {
      v = 0.f;
      for (int r = 0; r < p.parts; ++r) {
        float other;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(other) : "r"(ptx::mapa(base + 4 * at, r)) : "memory");
        v += other;
      }
    }
    if (m < m_count && n < p.outer)
      store_any(p.y, (m0 + m) * p.y_row + n * p.y_col, p.y_dtype, p.x_scale ? v * p.x_scale[(m0 + m) * p.xs_stride] : v);
  }
  if (p.parts > 1) ptx::cluster_sync();  // no block ends while another reads its sums
}

template <typename X, int NT> int launch_tiles(Params p, cudaStream_t stream) {
  using L = Layout<X, NT>;
  const int size = float_size(p.scale_dtype);
  const int in_stage = (L::KS + p.group - 1) / p.group + 1;  // groups that a stage can touch
  p.scale_words = ((in_stage * size + 3) / 4 + 1) | 1;       // odd: rows in different banks
  p.zero_words = p.zeros ? ((in_stage + 3) / 4 + 1) | 1 : 0;
  const int64_t most = p.rows < L::M ? p.rows : L::M;
  p.x_bytes = (int)most * L::X_PITCH;
  p.stage_bytes = (L::CODES + p.x_bytes + 4 * L::R * (p.scale_words + p.zero_words) + 127) / 128 * 128;
  p.stages = (int)((p.inner + L::KS - 1) / L::KS);
  const int ring = RING * p.stage_bytes, bytes = ring > L::JOIN ? ring : L::JOIN;
  constexpr int most_bytes = 232448;
  if (bytes > most_bytes) return tc::kNotEligible;
  cudaError_t e = smem_optin<tiles_kernel<X, NT>>(most_bytes);
  if (e != cudaSuccess) return (int)e;
  const int64_t row_blocks = (p.outer + L::R - 1) / L::R, m_blocks = (p.rows + L::M - 1) / L::M;
  // Parts of the columns: as many as bring the grid to two blocks an SM, of two
  // stages at least.
  int parts = 1;
  while (parts < 8 && row_blocks * m_blocks * parts < 2 * sm_count() && p.stages >= 4 * parts) parts *= 2;
  p.parts = parts;
  if (row_blocks * parts > (1LL << 31) - 1 || m_blocks > 65535) return NT_B200_ERR_INVALID_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(row_blocks * parts), (unsigned)m_blocks);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim = {(unsigned)parts, 1, 1};
  cfg.attrs = attrs;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, tiles_kernel<X, NT>, p);
}

template <typename X> int launch(const Params &p, cudaStream_t stream) {
  if constexpr (sizeof(X) <= 2) {
    const bool aligned = rotary::aligned16(p.x) && rotary::aligned16(p.codes) && p.x_col == 1 && p.c_col == 1 &&
                         p.s_col == 1 && (!p.zeros || p.z_col == 1) && (p.x_row * (int64_t)sizeof(X)) % 16 == 0 &&
                         p.c_row % 16 == 0 && p.c_row >= 0 && p.s_row >= 0 && p.z_row >= 0 &&
                         reinterpret_cast<uintptr_t>(p.scales) % 4 == 0 && reinterpret_cast<uintptr_t>(p.zeros) % 4 == 0;
    if (aligned && p.inner <= (1LL << 30) && (p.rows + 31) / 32 <= 65535) {
      const int rc = p.rows <= 8    ? launch_tiles<X, 1>(p, stream)
                     : p.rows <= 16 ? launch_tiles<X, 2>(p, stream)
                                    : launch_tiles<X, 4>(p, stream);
      if (rc != tc::kNotEligible) return rc;
    }
  }
  const int64_t blocks = (p.outer + 3) / 4, m_blocks = (p.rows + 7) / 8;
  if (blocks > (1LL << 31) - 1 || m_blocks > 65535) return NT_B200_ERR_INVALID_ARGUMENT;
  rows_kernel<X><<<dim3((unsigned)blocks, (unsigned)m_blocks), 128, 0, stream>>>(p);
  return launch_status();
}

}  // namespace four_bit
}  // namespace nt

extern "C" int nt_b200_int4_matmul(const NtB200Int4MatmulArgs *a, void *stream) {
  using namespace nt;
  if (!a || a->rows < 0 || a->inner < 0 || a->outer < 0 || a->group < 0) return NT_B200_ERR_INVALID_ARGUMENT;
  const bool codes = a->dtype == NT_B200_INT8 || a->dtype == NT_B200_FLOAT8_E4M3FN;
  if ((!codes && !is_float_dtype((int)a->dtype)) || !is_float_dtype((int)a->scales_dtype) ||
      !is_float_dtype((int)a->output_dtype))
    return NT_B200_ERR_UNSUPPORTED_DTYPE;
  if (a->rows == 0 || a->outer == 0) return 0;
  if (a->inner == 0 || a->group == 0 || a->group % 32 != 0 || a->inner % a->group != 0 || a->inner > (1LL << 31) - 1)
    return NT_B200_ERR_SHAPE_MISMATCH;
  if (!a->input || !a->codes || !a->scales || !a->output) return NT_B200_ERR_INVALID_ARGUMENT;
  four_bit::Params p{};
  p.x = a->input; p.y = a->output;
  p.codes = static_cast<const uint8_t *>(a->codes);
  p.scales = static_cast<const uint8_t *>(a->scales);
  p.zeros = static_cast<const uint8_t *>(a->zeros);
  p.x_scale = a->input_scale;
  p.x_row = a->input_strides[0]; p.x_col = a->input_strides[1];
  p.c_row = a->codes_strides[0]; p.c_col = a->codes_strides[1];
  p.s_row = a->scales_strides[0]; p.s_col = a->scales_strides[1];
  p.z_row = a->zeros ? a->zeros_strides[0] : 0; p.z_col = a->zeros ? a->zeros_strides[1] : 1;
  p.xs_stride = a->input_scale_stride;
  p.y_row = a->output_strides[0]; p.y_col = a->output_strides[1];
  p.rows = a->rows; p.inner = a->inner; p.outer = a->outer;
  p.group = (int)a->group; p.groups = (int)(a->inner / a->group);
  p.group32 = (uint32_t)(a->group / 32);
  p.scale_dtype = (int)a->scales_dtype; p.y_dtype = (int)a->output_dtype;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case NT_B200_FLOAT16: return four_bit::launch<__half>(p, s);
    case NT_B200_BFLOAT16: return four_bit::launch<__nv_bfloat16>(p, s);
    case NT_B200_FLOAT32: return four_bit::launch<float>(p, s);
    case NT_B200_FLOAT8_E4M3FN: return four_bit::launch<__nv_fp8_e4m3>(p, s);
    default: return four_bit::launch<int8_t>(p, s);
  }
}
