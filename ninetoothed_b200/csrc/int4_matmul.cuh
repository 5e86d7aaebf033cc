// Product of a few rows with a matrix of 4-bit weights:
//     y[m, n] = input_scale[m] * sum_k x[m, k] * (code[n, k] - zero[n, k / G]) * scale[n, k / G]
// with two codes a byte, the even element in the low half, and a zero point of 8
// where none are given.
//
// A weight is half a byte and serves every row of x, 4 flops a byte and row: reading the
// weights is the floor.  They go through shared memory once for every 8, 16 or 32 rows of
// x; x comes from L2.
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
// A block has 8 warps and 32, 64 or 128 weight rows; a stage of its ring holds 1024, 512
// or 256 columns of them, 16 KB, and x's columns beside it, of which a warp takes 32 rows
// by 128 columns.  More rows of x take more weight rows a block, so that x is never more
// than the weights.  Blocks go on from one set of rows to the next with the copies
// running ahead.  Where the weight rows are too few for the SMs, a cluster's blocks share
// the columns and join their sums through distributed shared memory, always in the same
// order.
//
// Measured (codes' bytes a second): 4096 x 4096 with one bfloat16 row 7.0 us, launch,
// first copies and join for the most part; 10240 -> 4099 with 5 float16 rows, groups of 64
// with zero points 14.0 us; 8192 x 8192 with 32 bfloat16 rows 24.7 us (weights in tensor
// memory, see tall_kernel; in groups of 64 or of 8-bit rows, with these steps, 35); 8192 ->
// 65536 with 16 E4M3 rows, groups of 32 with zero points 166 us, 1.6 TB/s.  Bound by issue,
// not by the floor: a warp takes about 600 instructions for 4096 codes, half of them to unpack, and
// the copies alone take 71 us of the last.  (With a warp of its own for the copies the
// register file holds 96 a thread and the products spill: 47 us for the third against 36.)
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
  // scales and zero points of a weight row in a stage: bytes of a copy, of all, from row to row
  int s_copy, z_copy, s_span, z_span, s_pitch, z_pitch;
  int copiers;                             // threads that copy them
  int x_rows, x_bytes, stage_bytes, ring, join, control;  // x's part of a stage; the whole; stages in shared memory; what follows them
  int64_t row_blocks;
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

// Zero points are whole numbers up to 63, which both unpackings take off without rounding
// (formats that store them less one hold 16); larger ones are an error.  `seen`: a thread's,
// joined by or.
constexpr uint32_t MOST_ZERO = 63;
__device__ __forceinline__ void check_zeros(uint32_t seen) {
  if (seen > MOST_ZERO) record_error(NT_B200_ERR_INDEX_OUT_OF_RANGE);
}

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
  uint32_t seen = 0;
  for (int64_t b = lane; b < p.inner / 2; b += 32) {
    const int64_t g = 2 * b / p.group;
    const uint8_t code = p.codes[n * p.c_row + b * p.c_col];
    const float s = any_float(p.scales + (n * p.s_row + g * p.s_col) * float_size(p.scale_dtype), p.scale_dtype);
    const uint32_t zero = p.zeros ? p.zeros[n * p.z_row + g * p.z_col] : 8u;
    seen |= zero;
    const float z = (float)zero;
    const float w0 = ((float)(code & 15) - z) * s, w1 = ((float)(code >> 4) - z) * s;
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (m < count) {
        const X *at = x + m * p.x_row + 2 * b * p.x_col;
        sum[m] = fmaf(to_f(at[0]), w0, fmaf(to_f(at[p.x_col]), w1, sum[m]));
      }
  }
  check_zeros(seen);
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
constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int MOST_RING = 8, CONTROL_BYTES = 16 * MOST_RING + 16;  // the stages' barriers and the abort flag

// Two 16-bit floats from four bits of w's halves, less the zero point: `low` takes
// bits 0-3, `high` bits 4-7 of each half.  The zero point comes as prepared.
template <typename F> struct Codes;
template <> struct Codes<__half> {
  // the zero point as `low` and `high` take it: 1024 + zero, -(64 + zero), twice each
  static __device__ __forceinline__ uint32_t zero_low(uint32_t zero) { return 0x64006400u + zero * 0x10001u; }
  static __device__ __forceinline__ uint32_t zero_high(uint32_t zero) { return 0xd400d400u + zero * 0x100010u; }
  static __device__ __forceinline__ __half2 as(uint32_t v) { return *reinterpret_cast<const __half2 *>(&v); }
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t z) {
    const __half2 v = __hsub2(as((w & 0x000f000fu) | 0x64006400u), as(z));
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  // (1024 + 16 code) / 16 - (64 + zero): nothing to round
  static __device__ __forceinline__ uint32_t high(uint32_t w, uint32_t z) {
    const __half2 v = __hfma2(as((w & 0x00f000f0u) | 0x64006400u), as(0x2c002c00u), as(z));
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <> struct Codes<__nv_bfloat16> {
  // 128 + zero, twice
  static __device__ __forceinline__ uint32_t zero_low(uint32_t zero) { return 0x43004300u + zero * 0x10001u; }
  static __device__ __forceinline__ uint32_t zero_high(uint32_t zero) { return zero_low(zero); }
  static __device__ __forceinline__ __nv_bfloat162 as(uint32_t v) { return *reinterpret_cast<const __nv_bfloat162 *>(&v); }
  static __device__ __forceinline__ uint32_t low(uint32_t w, uint32_t z) {
    const __nv_bfloat162 v = __hsub2(as((w & 0x000f000fu) | 0x43004300u), as(z));
    return *reinterpret_cast<const uint32_t *>(&v);
  }
  static __device__ __forceinline__ uint32_t high(uint32_t w, uint32_t z) { return low(w >> 4, z); }
  static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
};
template <typename X> struct Operand { using type = __half; };  // 8-bit x
template <> struct Operand<__nv_bfloat16> { using type = __nv_bfloat16; };

// Copies `span` bytes of a row's scales or zero points from `from` on, BYTES a thread
// and time.  Four at a time start with the word that holds the first.  What is past
// the row, `until`, is not read: zeros.
template <int BYTES>
__device__ __forceinline__ void copy_row(uint32_t to, const uint8_t *array, int64_t from, int64_t until, int span, int first,
                                         int step) {
  if (BYTES == 4) from &= ~(int64_t)3;
  for (int at = first * BYTES; at < span; at += step * BYTES) {
    const int64_t left = until - from - at;
    const int bytes = left >= BYTES ? BYTES : left > 0 ? (int)left : 0;
    const uint8_t *source = left > 0 ? array + from + at : array;
    if constexpr (BYTES == 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + at), "l"(source), "r"(bytes) : "memory");
    else
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to + at), "l"(source), "n"(BYTES), "r"(bytes) : "memory");
  }
}
// Arrives on the barrier once this thread's copies so far are done.
__device__ __forceinline__ void arrive_after_copies(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

template <typename X, int NT> struct Layout {
  // Row tiles of a warp and steps of its slice of a stage.  (4 and 2, so that a step of x
  // serves 64 rows, spilled: the head of 16 rows took 183 us, 166 at 2 and 4.)
  static constexpr int RT = 2, WSTEPS = 4;
  static constexpr int WR = NT, WK = WARPS / WR;
  static constexpr int R = 16 * RT * WR, KS = 32 * WSTEPS * WK;  // weight rows; columns of a stage
  static constexpr int STEPS = KS / 32;                          // of 32 columns
  static constexpr int M = 8 * NT;                               // rows of x
  static constexpr int CODES = R * KS / 2, BOX = R * 128, BOXES = CODES / BOX;  // 128-byte columns of all rows
  static constexpr int PITCH = R + 4, JOIN = WK * M * PITCH * 4;  // the warps' sums: lanes' stores in different banks
  static constexpr int FACTORS = 16 * RT * WSTEPS * 16;           // a warp's scales and zero points, see Factor
  static_assert(CODES == 16384, "a stage's codes");
};

// What a row's group needs at its products: the scale, and the zero point as Codes takes it.
struct alignas(16) Factor {
  float scale;
  uint32_t zero_low, zero_high, unused;
};

// Where the steps of a warp (or a stage) stand among the groups.
struct Group {
  uint32_t index, into;  // the group; steps into it
  __device__ __forceinline__ Group(uint32_t step, uint32_t group32) : index(step / group32), into(step % group32) {}
  __device__ __forceinline__ void advance(uint32_t quotient, uint32_t rest, uint32_t group32) {
    index += quotient;
    into += rest;
    if (into >= group32) {
      into -= group32;
      ++index;
    }
  }
};

// After a wait gave up: the copies in flight, so that the block's shared memory is at
// rest when it ends.  Nothing tells how far each stage's barrier went: both phases are
// waited for, the later one until the limit.
__device__ __noinline__ void settle(uint32_t full0, int ring) {
  constexpr uint64_t limit_ns = 100000000ull;
  if (threadIdx.x < (unsigned)ring) {
    volatile int over = 0;
    ptx::mbar_wait(full0 + 8u * threadIdx.x, 0, &over, limit_ns);
    over = 0;
    ptx::mbar_wait(full0 + 8u * threadIdx.x, 1, &over, limit_ns);
  }
  __syncthreads();
}

// The eight warps that compute.
__device__ __forceinline__ void sync_warps() { asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory"); }
__device__ __forceinline__ bool any_of_warps(int flag) {
  int any;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.s32 p, %1, 0;\n"
      "barrier.cta.red.or.pred p, 1, %2, p;\n"
      "selp.s32 %0, 1, 0, p;\n"
      "}"
      : "=r"(any)
      : "r"(flag), "n"(WARPS * 32)
      : "memory");
  return any != 0;
}
__device__ __forceinline__ void add(float4 &a, const float4 &b) {
  a.x += b.x;
  a.y += b.y;
  a.z += b.z;
  a.w += b.w;
}

// The sums of the warps that share columns, [WK][M][PITCH] in shared memory at `joined`,
// and of a cluster's blocks, into y; for the eight warps that have them.
template <typename L>
__device__ __forceinline__ void join_sums(const Params &p, float *joined, uint32_t address, int64_t n0, int64_t m0, int m_count,
                                          int part) {
  constexpr int COUNT = WARPS * 32, QUADS = L::R / 4;
  sync_warps();
  const auto sum_of = [&](int at) {
    float4 v = *reinterpret_cast<const float4 *>(joined + at);
#pragma unroll
    for (int k = 1; k < L::WK; ++k) add(v, *reinterpret_cast<const float4 *>(joined + k * L::M * L::PITCH + at));
    return v;
  };
  const auto store = [&](int m, int row, const float4 &v) {
    const float f[4] = {v.x, v.y, v.z, v.w};
    const float by = p.x_scale ? p.x_scale[(m0 + m) * p.xs_stride] : 1.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n0 + row + e < p.outer)
        store_any(p.y, (m0 + m) * p.y_row + (n0 + row + e) * p.y_col, p.y_dtype, p.x_scale ? f[e] * by : f[e]);
  };
  if (p.parts == 1) {
    for (int i = threadIdx.x; i < m_count * QUADS; i += COUNT)
      store(i / QUADS, i % QUADS * 4, sum_of(i / QUADS * L::PITCH + i % QUADS * 4));
    sync_warps();  // the sums are read: the next unit's may come
    return;
  }
  // (a grid with parts has one unit a cluster)
  for (int i = threadIdx.x; i < m_count * QUADS; i += COUNT) {
    const int at = i / QUADS * L::PITCH + i % QUADS * 4;
    *reinterpret_cast<float4 *>(joined + at) = sum_of(at);
  }
  ptx::cluster_sync();
  for (int i = threadIdx.x + part * COUNT; i < m_count * QUADS; i += COUNT * p.parts) {
    const uint32_t from = address + 4 * (i / QUADS * L::PITCH + i % QUADS * 4);
    float4 v[8];
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < p.parts)
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w)
                     : "r"(ptx::mapa(from, r)));
#pragma unroll
    for (int r = 1; r < 8; ++r)
      if (r < p.parts) add(v[0], v[r]);
    store(i / QUADS, i % QUADS * 4, v[0]);
  }
  ptx::cluster_sync();  // no block ends while another reads its sums
}

// GS: steps between two applications of a scale, a divisor of a group's and of a slice's
template <typename X, int NT, int GS>
__global__ void __launch_bounds__(THREADS, NT == 4 ? 1 : 2)
tiles_kernel(const __grid_constant__ CUtensorMap tmap_codes, const __grid_constant__ CUtensorMap tmap_x,
             const __grid_constant__ Params p) {
  using L = Layout<X, NT>;
  using F = typename Operand<X>::type;
  constexpr int XS = sizeof(X), RT = L::RT, SCALES = L::WSTEPS / GS;  // bytes of an element of x; scales of a row in a warp's slice
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem), bar0 = base + p.control;
  if ((base & 1023u) != 0) {  // the swizzle needs it
    record_error(NT_B200_ERR_INVALID_ARGUMENT);
    return;
  }
  const auto full = [&](int slot) { return bar0 + 8u * slot; };
  const auto empty = [&](int slot) { return bar0 + 8u * (MOST_RING + slot); };
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + p.control + CONTROL_BYTES - 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int wr = warp % L::WR, wk = warp / L::WR, g = lane >> 2, c = lane & 3;
  const int part = (int)(blockIdx.x % (unsigned)p.parts);
  const uint32_t unit0 = blockIdx.x / (unsigned)p.parts;  // of weight rows; the next are the grid's clusters further on
  const uint32_t units = (uint32_t)p.row_blocks, unit_step = gridDim.x / (uint32_t)p.parts;
  const int64_t m0 = (int64_t)blockIdx.y * L::M;
  const int m_count = (int)(p.rows - m0 < L::M ? p.rows - m0 : L::M);
  const int first = p.stages / p.parts * part + min(part, p.stages % p.parts);
  const int last = first + p.stages / p.parts + (part < p.stages % p.parts ? 1 : 0);
  const int scale_size = float_size(p.scale_dtype);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) {
      ptx::mbar_init(full(s), 1 + p.copiers);
      ptx::mbar_init(empty(s), WARPS);
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_codes);
    ptx::prefetch_tmap(&tmap_x);
  }
  __syncthreads();
  wait_prior_grid();

  // ---- copies of a stage: codes and x by TMA, scales and zero points by the first threads
  const uint32_t stage_quotient = L::STEPS / p.group32, stage_rest = L::STEPS % p.group32;
  const Group stage0((uint32_t)first * L::STEPS, p.group32), slice0((uint32_t)first * L::STEPS + wk * L::WSTEPS, p.group32);
  uint32_t fill_unit = unit0, fill_phase = 1;
  int fill_stage = first, fill_slot = 0;
  Group fill_at = stage0;
  const auto fill = [&]() {
    if (fill_unit >= units || !ptx::mbar_wait(empty(fill_slot), fill_phase, abort_flag)) return;
    const uint32_t to = base + (uint32_t)fill_slot * (uint32_t)p.stage_bytes, bar = full(fill_slot);
    if (threadIdx.x == 0) {
      ptx::mbar_arrive_expect_tx(bar, (uint32_t)(L::CODES + p.x_bytes));
#pragma unroll
      for (int b = 0; b < L::BOXES; ++b)
        ptx::tma_load_2d(to + b * L::BOX, &tmap_codes, bar, fill_stage * (L::KS / 2) + b * 128, (int32_t)(fill_unit * L::R));
      ptx::tma_load_3d(to + L::CODES, &tmap_x, bar, 0, (int32_t)m0, fill_stage * L::STEPS);
    }
    const int g0 = (int)fill_at.index;
    fill_at.advance(stage_quotient, stage_rest, p.group32);
    const int r = threadIdx.x % L::R, copier = threadIdx.x / L::R;
    const int64_t row = (int64_t)fill_unit * L::R + r;
    if (row < p.outer) {
      const uint32_t s_to = to + L::CODES + p.x_bytes + r * p.s_pitch;
      const int64_t s_from = (row * p.s_row + g0) * scale_size, s_until = (row * p.s_row + p.groups) * scale_size;
      constexpr int STEP = THREADS / L::R;
      if (p.s_copy == 16) copy_row<16>(s_to, p.scales, s_from, s_until, p.s_span, copier, STEP);
      else if (p.s_copy == 8) copy_row<8>(s_to, p.scales, s_from, s_until, p.s_span, copier, STEP);
      else copy_row<4>(s_to, p.scales, s_from, s_until, p.s_span, copier, STEP);
      if (p.zeros) {
        const uint32_t z_to = to + L::CODES + p.x_bytes + L::R * p.s_pitch + r * p.z_pitch;
        const int64_t z_from = row * p.z_row + g0, z_until = row * p.z_row + p.groups;
        if (p.z_copy == 16) copy_row<16>(z_to, p.zeros, z_from, z_until, p.z_span, copier, STEP);
        else if (p.z_copy == 8) copy_row<8>(z_to, p.zeros, z_from, z_until, p.z_span, copier, STEP);
        else copy_row<4>(z_to, p.zeros, z_from, z_until, p.z_span, copier, STEP);
      }
    }
    arrive_after_copies(bar);
    if (++fill_slot == p.ring) {
      fill_slot = 0;
      fill_phase ^= 1u;
    }
    if (++fill_stage == last) {
      fill_stage = first;
      fill_unit += unit_step;
      fill_at = stage0;
    }
  };
  const bool copies = threadIdx.x < (unsigned)p.copiers;
  if (copies)
    for (int i = 0; i < p.ring - 1; ++i) fill();

  const uint32_t q0 = wk * L::WSTEPS;
  const uint32_t code_row = (wr * 16 * RT + g) * 128 + (q0 / 8) * L::BOX + c * 4;
  const uint32_t x_step = 32 * XS * p.x_rows, x_at = L::CODES + q0 * x_step + c * 8 * XS;
  uint32_t x_row[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x_row[t] = min(t * 8 + g, p.x_rows - 1) * (32 * XS);  // (columns past the last are not written)
  Factor *factors = reinterpret_cast<Factor *>(smem + p.join + L::JOIN + warp * L::FACTORS);  // [SCALES][16 * RT]
  int slot = 0;
  uint32_t phase = 0;
  for (uint32_t unit = unit0; unit < units; unit += unit_step) {
    const int64_t n0 = (int64_t)unit * L::R;
    Group stage_at = stage0, slice_at = slice0;
    float acc[RT][NT][4] = {};
    uint32_t seen = 0;
    // ---- a warp's slice of each stage: 16 RT rows, WSTEPS steps of 32 columns
    for (int s = first; s < last; ++s) {
      if (copies) fill();
      if (!ptx::mbar_wait_warp(full(slot), phase, abort_flag)) break;
      const uint8_t *stage = smem + (uint32_t)slot * (uint32_t)p.stage_bytes;
      // a lane readies the factors of a row
      {
        static_assert(RT == 2, "a lane a row");
        const auto ready = [&](auto value) {
          const int r = wr * 16 * RT + lane;
          const uint8_t *from = stage + L::CODES + p.x_bytes + r * p.s_pitch;
          const uint8_t *zeros = stage + L::CODES + p.x_bytes + L::R * p.s_pitch + r * p.z_pitch;
          // where a row's part starts in the first word of its copy
          if (p.s_copy == 4) from += ((uint32_t)((n0 + r) * p.s_row) + stage_at.index) * (uint32_t)scale_size & 3u;
          if (p.z_copy == 4) zeros += ((uint32_t)((n0 + r) * p.z_row) + stage_at.index) & 3u;
          Group now = slice_at;
#pragma unroll
          for (int k = 0; k < SCALES; ++k) {
            const uint32_t nth = now.index - stage_at.index;
            uint32_t zero = 8;
            if (p.zeros) seen |= zero = zeros[nth];
            factors[k * 16 * RT + lane] =
                Factor{value(from + nth * scale_size), Codes<F>::zero_low(zero), Codes<F>::zero_high(zero), 0u};
            now.advance(0, GS, p.group32);
          }
        };
        if (p.scale_dtype == NT_B200_BFLOAT16)
          ready([](const uint8_t *v) { return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(v) << 16); });
        else if (p.scale_dtype == NT_B200_FLOAT16)
          ready([](const uint8_t *v) { return __half2float(*reinterpret_cast<const __half *>(v)); });
        else ready([](const uint8_t *v) { return *reinterpret_cast<const float *>(v); });
        __syncwarp();
      }
      float sum[RT][NT][4];
      const float none[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < L::WSTEPS; ++j) {
        // x: eight elements a lane, as the pairs (0, 4), (1, 5), (2, 6), (3, 7)
        uint32_t b[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint8_t *from = stage + x_at + j * x_step + x_row[t];
          if constexpr (XS == 2) {
            const uint4 x = *reinterpret_cast<const uint4 *>(from);
            b[t][0] = __byte_perm(x.x, x.z, 0x5410);
            b[t][1] = __byte_perm(x.x, x.z, 0x7632);
            b[t][2] = __byte_perm(x.y, x.w, 0x5410);
            b[t][3] = __byte_perm(x.y, x.w, 0x7632);
          } else {
            const uint2 x = *reinterpret_cast<const uint2 *>(from);
            paged::to_halves<X>(__byte_perm(x.x, x.y, 0x5140), b[t][0], b[t][1]);
            paged::to_halves<X>(__byte_perm(x.x, x.y, 0x7362), b[t][2], b[t][3]);
          }
        }
        const uint8_t *codes = stage + code_row + (((q0 + j) ^ g) & 7) * 16;  // TMA's 128-byte swizzle of a row's 16-byte words
        const Factor *factor = factors + (j / GS) * 16 * RT + g;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t lo = *reinterpret_cast<const uint32_t *>(codes + r * 2048);
          const uint32_t hi = *reinterpret_cast<const uint32_t *>(codes + r * 2048 + 1024);
          const uint32_t lo8 = lo >> 8, hi8 = hi >> 8;
          const Factor fl = factor[r * 16], fh = factor[r * 16 + 8];
          const uint32_t a0[4] = {Codes<F>::low(lo, fl.zero_low), Codes<F>::low(hi, fh.zero_low),
                                  Codes<F>::high(lo, fl.zero_high), Codes<F>::high(hi, fh.zero_high)};
          const uint32_t a1[4] = {Codes<F>::low(lo8, fl.zero_low), Codes<F>::low(hi8, fh.zero_low),
                                  Codes<F>::high(lo8, fl.zero_high), Codes<F>::high(hi8, fh.zero_high)};
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if (j % GS == 0) Codes<F>::mma(sum[r][t], none, a0, b[t][0], b[t][1]);
            else Codes<F>::mma(sum[r][t], sum[r][t], a0, b[t][0], b[t][1]);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) Codes<F>::mma(sum[r][t], sum[r][t], a1, b[t][2], b[t][3]);
          if (j % GS == GS - 1) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[r][t][e] = fmaf(e < 2 ? fl.scale : fh.scale, sum[r][t][e], acc[r][t][e]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(empty(slot));
      stage_at.advance(stage_quotient, stage_rest, p.group32);
      slice_at.advance(stage_quotient, stage_rest, p.group32);
      if (++slot == p.ring) {
        slot = 0;
        phase ^= 1u;
      }
    }
    if (n0 + wr * 16 * RT + lane < p.outer) check_zeros(seen);  // (nothing was copied for other rows)
    if (unit + unit_step >= units) allow_dependent_launch();

    // ---- the warps' sums, [WK][M][R + 4], then the cluster's
    float *joined = reinterpret_cast<float *>(smem + p.join);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int m = t * 8 + 2 * c + (e & 1), row = wr * 16 * RT + r * 16 + g + (e >> 1) * 8;
          joined[(wk * L::M + m) * L::PITCH + row] = acc[r][t][e];
        }
    join_sums<L>(p, joined, base + p.join, n0, m0, m_count, part);
    if (any_of_warps(*abort_flag)) break;  // (a warp ahead may set it at any time: one answer for all)
  }
  __syncthreads();
  if (*abort_flag) settle(bar0, p.ring);
}

// ---------------------------------------------------------------- weights through tensor memory
// The same products for more rows of x, with the weights as tcgen05's 128 rows and x's as
// its columns: a thread unpacks the codes of its row of 128 into tensor memory, where the
// MMAs read them (x from shared memory), and takes a group's sums out of tensor memory.
// Scale and zero point are then its own row's, x needs no permutes and the MMAs no
// registers, so that two blocks an SM fit.  A block's two warpgroups take the halves of a
// stage's 256 columns, which share a scale each: groups of 128 columns and their multiples.
//
// 8192 x 8192 with 32 bfloat16 rows: 24.7 us (36 with fragments), bound by latency: a
// warpgroup's unpacking, MMAs and sums follow one another.  Without the unpacking 19 us,
// without the scales' loads 23.  Tried: 64 columns at a time in two buffers each, the sums
// taken while the next MMAs run, 29 us (twice the stores and loads of tensor memory, and
// their waits).  Sums of two groups a half, for groups of 64, spill: 30 us, 34 with fragments.
struct Tall {
  static constexpr int N = 32, R = 128, KS = 256, HALF = 128;
  static constexpr int CODES = R * KS / 2, X_BOX = N * 128, X = 4 * X_BOX;  // x: 64 columns a box
  static constexpr int STAGE = CODES + X;
  static constexpr int M = N, WK = 1, PITCH = R + 4, JOIN = WK * M * PITCH * 4;
  static constexpr int A_COLS = HALF / 2, D_COLS = 64, TMEM_COLS = 2 * (A_COLS + D_COLS);  // a warpgroup's weights, its sums
};
constexpr int TALL_WARPS = 10, TALL_THREADS = TALL_WARPS * 32;  // 8 that unpack, one that copies, one that issues
constexpr int TALL_CONTROL = 16 * MOST_RING + 48;               // the stages' and warpgroups' barriers, and two words

template <typename F>
__global__ void __launch_bounds__(TALL_THREADS, 2)
tall_kernel(const __grid_constant__ CUtensorMap tmap_codes, const __grid_constant__ CUtensorMap tmap_x,
            const __grid_constant__ Params p) {
  using L = Tall;
  constexpr int N = L::N;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = ptx::smem_u32(smem), bar0 = base + p.control;
  if ((base & 1023u) != 0) {  // the swizzle needs it
    record_error(NT_B200_ERR_INVALID_ARGUMENT);
    return;
  }
  const auto full = [&](int slot) { return bar0 + 8u * slot; };
  const auto empty = [&](int slot) { return bar0 + 8u * (MOST_RING + slot); };
  const auto a_full = [&](int wg) { return bar0 + 16u * MOST_RING + 8u * wg; };       // weights in tensor memory, sums read
  const auto d_full = [&](int wg) { return bar0 + 16u * MOST_RING + 16u + 8u * wg; }; // sums in tensor memory
  const uint32_t settled = bar0 + 16u * MOST_RING + 32u;
  volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + p.control + 16 * MOST_RING + 40);
  volatile uint32_t *tmem_at = reinterpret_cast<volatile uint32_t *>(smem + p.control + 16 * MOST_RING + 44);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = (int)(blockIdx.x % (unsigned)p.parts);
  const uint32_t unit0 = blockIdx.x / (unsigned)p.parts, units = (uint32_t)p.row_blocks, unit_step = gridDim.x / (uint32_t)p.parts;
  const int64_t m0 = (int64_t)blockIdx.y * N;
  const int m_count = (int)(p.rows - m0 < N ? p.rows - m0 : N);
  const int first = p.stages / p.parts * part + min(part, p.stages % p.parts);
  const int last = first + p.stages / p.parts + (part < p.stages % p.parts ? 1 : 0);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.ring; ++s) {
      ptx::mbar_init(full(s), 1);
      ptx::mbar_init(empty(s), 8 + 1);
    }
    for (int wg = 0; wg < 2; ++wg) {
      ptx::mbar_init(a_full(wg), 4);
      ptx::mbar_init(d_full(wg), 1);
    }
    ptx::mbar_init(settled, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmap_codes);
    ptx::prefetch_tmap(&tmap_x);
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t *>(tmem_at)), L::TMEM_COLS);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_at;
  wait_prior_grid();

  int slot = 0;
  uint32_t phase = 0;
  const auto next_slot = [&]() {
    if (++slot == p.ring) {
      slot = 0;
      phase ^= 1u;
    }
  };
  if (warp == 8) {
    // ---- copies
    if (lane == 0) {
      for (uint32_t unit = unit0; unit < units && !*abort_flag; unit += unit_step)
        for (int s = first; s < last; ++s) {
          if (!ptx::mbar_wait(empty(slot), phase ^ 1u, abort_flag)) break;
          const uint32_t to = base + (uint32_t)slot * L::STAGE;
          ptx::mbar_arrive_expect_tx(full(slot), L::STAGE);
          ptx::tma_load_2d(to, &tmap_codes, full(slot), s * (L::KS / 2), (int32_t)(unit * L::R));
#pragma unroll
          for (int b = 0; b < 4; ++b)
            ptx::tma_load_2d(to + L::CODES + b * L::X_BOX, &tmap_x, full(slot), s * L::KS + 64 * b, (int32_t)m0);
          next_slot();
        }
    }
  } else if (warp == 9) {
    // ---- MMAs
    constexpr uint32_t idesc = ptx::f16_idesc(tc::umma_format<F>(), 0, 0, L::R, N);
    if (lane == 0) {
      uint32_t turn = 0;
      for (uint32_t unit = unit0; unit < units && !*abort_flag; unit += unit_step)
        for (int s = first; s < last; ++s, ++turn) {
          if (!ptx::mbar_wait(full(slot), phase, abort_flag)) break;
          const uint32_t x = base + (uint32_t)slot * L::STAGE + L::CODES;
          bool good = true;
          for (int wg = 0; wg < 2 && good; ++wg) {
            good = ptx::mbar_wait(a_full(wg), turn & 1u, abort_flag);
            if (!good) break;
            ptx::tc_fence_after();
            const uint32_t a = tmem + (uint32_t)(wg * (L::A_COLS + L::D_COLS)), d = a + L::A_COLS;
#pragma unroll
            for (int kk = 0; kk < L::HALF / 16; ++kk)
              ptx::mma_f16_ts(d, a + (uint32_t)(kk * 8), ptx::sw128_desc(x + (2 * wg + kk / 4) * L::X_BOX + (kk % 4) * 32, 16, 1024), idesc,
                              kk > 0 ? 1u : 0u);
            ptx::mma_commit(d_full(wg));
          }
          if (!good) break;
          ptx::mma_commit(empty(slot));
          next_slot();
        }
    }
  } else {
    // ---- a thread's row, half a stage at a time
    const int wg = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t a_cols = tmem + (uint32_t)(wg * (L::A_COLS + L::D_COLS)) + ((uint32_t)(quarter * 32) << 16);
    const uint32_t d_cols = a_cols + L::A_COLS;
    const int scale_size = float_size(p.scale_dtype);
    uint32_t turn = 0;
    for (uint32_t unit = unit0; unit < units; unit += unit_step) {
      const int64_t n = (int64_t)unit * L::R + row;
      const bool some_row = n < p.outer;
      float acc[N] = {};
      // raw scale and zero point of the next half stage: on their way while this one is worked on
      uint32_t raw, zero;
      const auto fetch = [&](int s) {
        const uint32_t group = (uint32_t)(s * (L::KS / 32) + wg * (L::HALF / 32)) / p.group32;
        raw = 0;  // (past the last column x is 0)
        zero = 8;
        if (!some_row || s >= last || group >= (uint32_t)p.groups) return;
        const uint8_t *at = p.scales + (n * p.s_row + group * p.s_col) * scale_size;
        raw = scale_size == 4 ? *reinterpret_cast<const uint32_t *>(at) : *reinterpret_cast<const uint16_t *>(at);
        if (p.zeros) zero = p.zeros[n * p.z_row + group * p.z_col];
      };
      const auto value = [&](uint32_t v) {
        if (p.scale_dtype == NT_B200_FLOAT32) return __uint_as_float(v);
        return p.scale_dtype == NT_B200_BFLOAT16 ? __uint_as_float(v << 16) : __half2float(__ushort_as_half((uint16_t)v));
      };
      float scale = 0.f;  // of the sums that the MMAs are at
      const auto take_sums = [&]() {
#pragma unroll
        for (int m = 0; m < N; m += 16) {
          uint32_t d[16];
          ptx::tmem_ld_32x32b_x16(d_cols + (uint32_t)m, d);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[m + e] = fmaf(scale, __uint_as_float(d[e]), acc[m + e]);
        }
      };
      fetch(first);
      bool good = true;
      for (int s = first; s < last; ++s, ++turn) {
        good = ptx::mbar_wait_warp(full(slot), phase, abort_flag);
        if (!good) break;
        const float next_scale = value(raw);
        const uint32_t z0 = Codes<F>::zero_low(zero), z1 = Codes<F>::zero_high(zero);
        check_zeros(zero);
        fetch(s + 1);
        if (s > first) {  // the weights before were read, and their sums are there
          good = ptx::mbar_wait_warp(d_full(wg), (turn - 1) & 1u, abort_flag);
          if (!good) break;
          ptx::tc_fence_after();
          take_sums();
        }
        const uint8_t *codes = smem + (uint32_t)slot * L::STAGE + row * 128;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // (at its place in TMA's 128-byte swizzle)
          const uint4 w = *reinterpret_cast<const uint4 *>(codes + (((wg * 4 + i) ^ row) & 7) * 16);
          const uint32_t word[4] = {w.x, w.y, w.z, w.w};
          uint32_t a[16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t v = word[k], v8 = v >> 8;
            const uint32_t e04 = Codes<F>::low(v, z0), e15 = Codes<F>::high(v, z1);
            const uint32_t e26 = Codes<F>::low(v8, z0), e37 = Codes<F>::high(v8, z1);
            a[4 * k] = __byte_perm(e04, e15, 0x5410);
            a[4 * k + 1] = __byte_perm(e26, e37, 0x5410);
            a[4 * k + 2] = __byte_perm(e04, e15, 0x7632);
            a[4 * k + 3] = __byte_perm(e26, e37, 0x7632);
          }
          ptx::tmem_st_32x32b_x16(a_cols + (uint32_t)(i * 16), a);
        }
        ptx::tmem_st_wait();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(a_full(wg));
          ptx::mbar_arrive(empty(slot));
        }
        scale = next_scale;
        next_slot();
      }
      if (good && ptx::mbar_wait_warp(d_full(wg), (turn - 1) & 1u, abort_flag)) {
        ptx::tc_fence_after();
        take_sums();
        ptx::tc_fence_before();
      }
      if (unit + unit_step >= units) allow_dependent_launch();
      // the warpgroups' sums, [N][PITCH]
      float *joined = reinterpret_cast<float *>(smem + p.join);
      if (wg == 1) {
#pragma unroll
        for (int m = 0; m < N; ++m) joined[m * L::PITCH + row] = acc[m];
      }
      sync_warps();
      if (wg == 0) {
#pragma unroll
        for (int m = 0; m < N; ++m) joined[m * L::PITCH + row] += acc[m];
      }
      join_sums<L>(p, joined, base + p.join, (int64_t)unit * L::R, m0, m_count, part);
      if (any_of_warps(*abort_flag)) break;  // (the other warps may set it at any time: one answer for all)
    }
  }
  if (warp >= 8 && p.parts > 1) {  // the join's barriers are the whole cluster's
    __syncwarp();
    ptx::cluster_sync();
    ptx::cluster_sync();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    // after a wait gave up: the MMAs in flight
    if (threadIdx.x == 9 * 32) {
      volatile int over = 0;
      ptx::mma_commit(settled);
      ptx::mbar_wait(settled, 0, &over, 100000000ull);
    }
    settle(bar0, p.ring);
  }
  if (warp == 9) {
    __syncwarp();
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

// Launches a kernel over the row blocks, x's blocks of rows and parts of the columns.
template <typename L, typename K>
int launch_blocks(K kernel, Params &p, int threads, int bytes, const CUtensorMap &tmap_codes, const CUtensorMap &tmap_x,
                  cudaStream_t stream) {
  const int64_t row_blocks = (p.outer + L::R - 1) / L::R, m_blocks = (p.rows + L::M - 1) / L::M;
  // Parts of the columns: as many as leave the grid in two blocks an SM.  (tiles_kernel with
  // 32 rows of x fits once: it goes through such a grid in two turns.)
  const int64_t room = 2 * (int64_t)sm_count();
  int parts = 1;
  while (parts < 8 && row_blocks * m_blocks * parts * 2 <= room && p.stages >= 2 * parts) parts *= 2;
  p.parts = parts;
  p.row_blocks = row_blocks;
  int64_t grid = row_blocks;
  if (grid * m_blocks > room) grid = (room + m_blocks - 1) / m_blocks < grid ? (room + m_blocks - 1) / m_blocks : grid;
  if (m_blocks > 65535) return NT_B200_ERR_INVALID_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(grid * parts), (unsigned)m_blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)parts;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = parts > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, tmap_codes, tmap_x, p);
}

template <typename F> int launch_tall(Params p, cudaStream_t stream) {
  using L = Tall;
  tc::EncodeTiledFn encode = tc::encode_tiled_fn();
  if (!encode) return tc::kNotEligible;
  p.stage_bytes = L::STAGE;
  p.stages = (int)((p.inner + L::KS - 1) / L::KS);
  constexpr int half_bytes = 113 * 1024 - TALL_CONTROL - L::JOIN;
  p.ring = half_bytes / L::STAGE < MOST_RING ? half_bytes / L::STAGE : MOST_RING;
  static_assert(half_bytes / L::STAGE >= 2, "a ring");
  p.join = p.ring * L::STAGE;
  p.control = p.join + L::JOIN;
  const int bytes = p.control + TALL_CONTROL;
  cudaError_t e = smem_optin<tall_kernel<F>>(bytes);
  if (e != cudaSuccess) return (int)e;
  CUtensorMap tmap_codes, tmap_x;
  const cuuint32_t ones[2] = {1, 1}, code_box[2] = {128, (cuuint32_t)L::R}, x_box[2] = {64, (cuuint32_t)L::N};
  const cuuint64_t code_dims[2] = {(cuuint64_t)(p.inner / 2), (cuuint64_t)p.outer}, code_strides[1] = {(cuuint64_t)p.c_row};
  const cuuint64_t x_dims[2] = {(cuuint64_t)p.inner, (cuuint64_t)p.rows}, x_strides[1] = {(cuuint64_t)p.x_row * 2};
  if (encode(&tmap_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(p.codes), code_dims, code_strides, code_box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      encode(&tmap_x, tc::tmap_dtype<F>(), 2, const_cast<void *>(p.x), x_dims, x_strides, x_box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return tc::kNotEligible;
  return launch_blocks<L>(tall_kernel<F>, p, TALL_THREADS, bytes, tmap_codes, tmap_x, stream);
}

template <typename X, int NT, int GS> int launch_tiles(Params p, cudaStream_t stream) {
  using L = Layout<X, NT>;
  constexpr int XS = sizeof(X);
  tc::EncodeTiledFn encode = tc::encode_tiled_fn();
  if (!encode) return tc::kNotEligible;
  p.x_rows = (int)(p.rows < L::M ? p.rows : L::M);
  p.x_bytes = p.x_rows * L::KS * XS;
  // A row's scales in a stage: as wide a copy as every row and stage starts on; an odd
  // number of 16 bytes apart, so that the rows that a warp reads lie in different banks.
  const auto part = [&](const uint8_t *array, int64_t row_bytes, int size, int &copy, int &span, int &pitch) {
    const int whole = L::KS % p.group == 0 ? L::KS / p.group * size : 0;  // 0: stages start within groups
    copy = 16;
    while (copy > 4 && (whole == 0 || whole % copy || row_bytes % copy || reinterpret_cast<uintptr_t>(array) % copy)) copy /= 2;
    span = copy > 4 ? whole : ((L::KS + p.group - 1) / p.group + 1) * size + 3;
    pitch = ((span + 18) / 16 | 1) * 16;
    const int copies = (span + copy - 1) / copy;
    return (copies < THREADS / L::R ? copies : THREADS / L::R) * L::R;
  };
  p.copiers = part(p.scales, p.s_row * float_size(p.scale_dtype), float_size(p.scale_dtype), p.s_copy, p.s_span, p.s_pitch);
  if (p.zeros) {
    const int more = part(p.zeros, p.z_row, 1, p.z_copy, p.z_span, p.z_pitch);
    if (more > p.copiers) p.copiers = more;
  }
  p.stage_bytes = (L::CODES + p.x_bytes + L::R * (p.s_pitch + p.z_pitch) + 1023) / 1024 * 1024;
  p.stages = (int)((p.inner + L::KS - 1) / L::KS);
  // Stages on their way: what half of an SM's shared memory holds.
  constexpr int half_bytes = 113 * 1024 - CONTROL_BYTES - L::JOIN - WARPS * L::FACTORS;
  p.ring = half_bytes / p.stage_bytes;
  if (p.ring > MOST_RING) p.ring = MOST_RING;
  if (p.ring < 2) p.ring = 2;
  p.join = p.ring * p.stage_bytes;
  p.control = p.join + L::JOIN + WARPS * L::FACTORS;
  const int bytes = p.control + CONTROL_BYTES;
  constexpr int most_bytes = 220 * 1024;
  if (bytes > most_bytes) return tc::kNotEligible;
  cudaError_t e = smem_optin<tiles_kernel<X, NT, GS>>(most_bytes);
  if (e != cudaSuccess) return (int)e;

  CUtensorMap tmap_codes, tmap_x;
  const cuuint32_t ones[3] = {1, 1, 1};
  const cuuint64_t code_dims[2] = {(cuuint64_t)(p.inner / 2), (cuuint64_t)p.outer}, code_strides[1] = {(cuuint64_t)p.c_row};
  const cuuint32_t code_box[2] = {128, (cuuint32_t)L::R};
  // x as [steps][rows][32 columns]: a warp then reads its rows of a step side by side
  const cuuint64_t x_dims[3] = {32, (cuuint64_t)p.rows, (cuuint64_t)(p.inner / 32)};
  const cuuint64_t x_strides[2] = {(cuuint64_t)p.x_row * XS, 32 * XS};
  const cuuint32_t x_box[3] = {32, (cuuint32_t)p.x_rows, (cuuint32_t)L::STEPS};
  if (encode(&tmap_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(p.codes), code_dims, code_strides, code_box,
             ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      encode(&tmap_x, XS == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(p.x),
             x_dims, x_strides, x_box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return tc::kNotEligible;

  return launch_blocks<L>(tiles_kernel<X, NT, GS>, p, THREADS, bytes, tmap_codes, tmap_x, stream);
}
template <typename X, int NT> int launch_groups(const Params &p, cudaStream_t stream) {
  if (p.group32 % 4 == 0) return launch_tiles<X, NT, 4>(p, stream);
  if (p.group32 % 2 == 0) return launch_tiles<X, NT, 2>(p, stream);
  return launch_tiles<X, NT, 1>(p, stream);
}

template <typename X> int launch(Params p, cudaStream_t stream) {
  if constexpr (sizeof(X) <= 2) {
    // (a single row's stride is never used)
    if (p.rows == 1) p.x_row = p.inner;
    if (p.outer == 1) p.c_row = p.inner / 2;
    const bool aligned = rotary::aligned16(p.x) && rotary::aligned16(p.codes) && p.x_col == 1 && p.c_col == 1 &&
                         p.s_col == 1 && (!p.zeros || p.z_col == 1) && (p.x_row * (int64_t)sizeof(X)) % 16 == 0 &&
                         p.c_row % 16 == 0 && p.c_row > 0 && p.x_row > 0 && p.s_row >= 0 && p.z_row >= 0 &&
                         reinterpret_cast<uintptr_t>(p.scales) % 4 == 0 && reinterpret_cast<uintptr_t>(p.zeros) % 4 == 0;
    if (aligned && p.inner <= (1LL << 30) && p.outer <= (1LL << 30) && (p.rows + 31) / 32 <= 65535) {
      // Through tensor memory from 17 rows on, in groups of whole 128 columns: 24 us to 36 at
      // 32 x 8192 -> 8192, 10.5 to 21 at 17 x 4096 -> 4096, equal at 32 x 1024 -> 4096 (below,
      // the fragments' shorter start wins: 4.3 us to 6.0 at 256 columns); at 16 rows 23.9 to
      // 22.8 and 144 to 148 (8192 -> 8192, 8192 -> 65536), at 9 x 4096 -> 4096 10.5 to 8.3.
      if constexpr (sizeof(X) == 2)
        if (p.rows > 16 && p.group32 % 4 == 0 && p.inner >= 1024) {
          const int rc = launch_tall<X>(p, stream);
          if (rc != tc::kNotEligible) return rc;
        }
      const int rc = p.rows <= 8    ? launch_groups<X, 1>(p, stream)
                     : p.rows <= 16 ? launch_groups<X, 2>(p, stream)
                                    : launch_groups<X, 4>(p, stream);
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
