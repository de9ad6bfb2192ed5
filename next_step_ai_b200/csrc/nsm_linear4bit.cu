// nsm_linear4bit.cu -- y = x W^T (+ bias) for 1..32 rows of x and a weight W
// [N, K] in 4 bits with a scale for each group of columns of a row:
//
//   y[r][n] = b[n] + sum_g s[n][g] * sum_{k in g} x[r][k] * (T[q[n][k]] - z[n][g])
//
// T is a 16-entry codebook (z = 0: NF4 and the like) or the identity (integer
// weights, z = 8 or a zero point per group).
//
// Layout (written once by nsm_linear4bit_pack): tiles of 128 rows x 128 columns, 8 KB
// each, row tile by row tile, as [4 column chunks][128 rows][16 bytes]: a thread owns a
// row, and a warp's 16-byte loads are 512 contiguous bytes.  Scales and zero points lie
// as [row tile][tile][128 rows][granules], a granule being the group or 128 columns.
//
// One to three launches, linked by programmatic dependent launch:
//  1. for more than 8 columns of x, lin4_prep_kernel: per row of x a power-of-two scale that
//     brings the largest finite |x| to [2^14, 2^15), and x as fp16: exact for fp16, for bf16 exact
//     down to 2^-31 of the row's largest value (below that off by at most 2^-39 of it); an
//     fp32 x becomes two fp16 columns, value and remainder: 22 bits.  x is written as the 8 x
//     16-byte core matrices of a K-major tensor-core operand.  For up to 8 columns lin4_kernel
//     does this itself, with a scale for each 128 columns of a row, that brings their largest to
//     [2^13, 2^15): one launch and 5 us less at 16384 columns;
//  2. lin4_kernel: one CTA per SM, four warpgroups of 128 rows each.  A unit is 512 rows x
//     128 columns; the units, row block by row block, are cut into equal contiguous runs,
//     one per CTA, so no CTA finishes late.  Bulk copies bring each warpgroup's tile and
//     scales into its own ring, and x into a ring that all share.  A warpgroup turns its
//     tile into fp16 (a byte -> half2 table for codebooks, and a second one for what fp16
//     leaves of a value; mask and subtract for integers, exact) and stores it to tensor
//     memory; a warp of its own multiplies it with x (tcgen05.mma, M = 128 rows, N = the
//     columns of x, fp32 accumulation), and then the warpgroup adds scale * product to its
//     fp32 sums in registers, after it has converted what comes next.  With weights as the M
//     operand in tensor memory x never passes through registers: one row of x or 32 cost the
//     threads the same but for the sums.  Each CTA leaves one fp32 partial per row block that it
//     touched;
//  3. lin4_finalize_kernel: the partials of a row block in a fixed order (the same
//     bits every time), times the scale of x, + bias, in the output's type.  Small weights
//     go without it: there a cluster of CTAs has a row block, and its sums join in shared memory.
//
// Measured, 16384 x 16384 with weights larger than L2: NF4, one row of x in bf16, 48 us; integers
// with groups of 128, 30 us for one row and 41 us for 32.  The codebook's 22 bits take two table
// reads per byte, and shared memory bounds a unit at 1.64 us.  With the codebook rounded to
// fp16 (32 us) a unit takes 0.94 us, one of integers 0.88 us with 32 rows: 90% and 91% of the copy
// bandwidth.  The rest is a start of 3 us, the last CTAs' tail with the partials (3 us), and prep.
#include <algorithm>

#include "nsm_common.cuh"
#include "nsm_internal.h"

namespace nsm {
namespace {

constexpr int kL4Groups = 4;                          // warpgroups of a CTA
constexpr int kL4XStages = 4;                         // x tiles in flight, and warps that bring them
constexpr int kL4Threads = kL4Groups * 160 + kL4XStages * 32;  // each group with a warp that issues its copies and MMAs
constexpr int kL4TileRows = 128;
constexpr int kL4TileCols = 128;
constexpr int kL4TileBytes = kL4TileRows * kL4TileCols / 2;
constexpr int kL4BlockRows = kL4TileRows * kL4Groups;  // rows of a unit
constexpr int kL4MaxCols = 32;                        // fp16 columns of x in one call
constexpr int kL4MaxSegs = 32;                        // CTAs that share one row block
constexpr uint32_t kL4TmemGroup = 128;                // columns of tensor memory per warpgroup
constexpr int kL4BarBytes = 640;                      // of Lin4Bars

// Kinds of weights: codebook rounded to fp16 (where the caller asks for it); codebook as
// fp16 value + remainder (22 bits, two table reads and two MMAs); integers with the zero
// point 8; integers with a zero point per group.
enum { kCode = 0, kCodeExact = 1, kInt = 2, kIntZeros = 3 };

struct Lin4Shape {
  int N, K, group;
  int row_tiles, steps, row_blocks, kp;  // kp = steps * 128
  int npg;                               // scale granules per tile: 4, 2 or 1
  int div;                               // tiles per scale when npg == 1
  int scale_steps;                       // scale entries per row tile
};

Lin4Shape lin4_shape(int N, int K, int group) {
  Lin4Shape s;
  s.N = N;
  s.K = K;
  s.group = group;
  s.row_tiles = (N + kL4TileRows - 1) / kL4TileRows;
  s.steps = (K + kL4TileCols - 1) / kL4TileCols;
  s.row_blocks = (s.row_tiles + kL4Groups - 1) / kL4Groups;
  s.kp = s.steps * kL4TileCols;
  s.npg = group % 128 == 0 ? 1 : (group % 64 == 0 ? 2 : 4);
  s.div = s.npg == 1 ? group / 128 : 1;
  s.scale_steps = (s.steps + s.div - 1) / s.div;
  return s;
}

// ---- packing ------------------------------------------------------------------
// One thread per 32-bit word of the tiled weight: columns 8w .. of a row.  Codebook
// words keep the byte order (byte i = columns 2i, 2i+1: an index into the byte
// table).  Integer words put columns c and c + 1 of a pair 16 bits apart, so one mask
// leaves a half2: nibbles 0..7 = columns 0, 2, 4, 6, 1, 3, 5, 7.
__global__ void lin4_pack_kernel(const uint8_t* __restrict__ src, int64_t row_bytes, Lin4Shape sh, int is_code,
                                 uint32_t* __restrict__ dst) {
  constexpr int kWords = kL4TileBytes / 4;
  const int64_t words = (int64_t)sh.row_tiles * sh.steps * kWords;
  const int kb = sh.K / 2;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x) {
    const int in_tile = (int)(i % kWords);  // [4 chunks][128 rows][4 words]
    const int64_t tile = i / kWords;
    const int j = in_tile & 3, chunk = in_tile / (4 * kL4TileRows);
    const int64_t row = tile / sh.steps * kL4TileRows + (in_tile / 4) % kL4TileRows;
    const int col_byte = (int)(tile % sh.steps) * (kL4TileCols / 2) + 16 * chunk + 4 * j;
    uint32_t v = 0;
    if (row < sh.N) {
      const uint8_t* r = src + row * row_bytes;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint32_t byte = col_byte + b < kb ? r[col_byte + b] : 0u;  // high nibble = even column
        if (is_code)
          v |= byte << (8 * b);
        else
          v |= ((byte >> 4) << (4 * b)) | ((byte & 15u) << (16 + 4 * b));
      }
    }
    dst[i] = v;
  }
}

// Scales (and zero points) as [row tile][scale step][128 rows][npg]; rows and columns
// past the end get scale 0 and zero point 0.
__global__ void lin4_pack_scales_kernel(const void* __restrict__ scales, int dt, const uint8_t* __restrict__ zeros,
                                        Lin4Shape sh, int groups, float* __restrict__ ds, uint8_t* __restrict__ dz) {
  const int per = kL4TileRows * sh.npg;
  const int64_t n = (int64_t)sh.row_tiles * sh.scale_steps * per;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int e = (int)(i % per);
    const int64_t ts = i / per;
    const int pg = e % sh.npg;
    const int64_t row = ts / sh.scale_steps * kL4TileRows + e / sh.npg;
    const int64_t col = (ts % sh.scale_steps) * sh.div * kL4TileCols + pg * (kL4TileCols / sh.npg);
    const int64_t grp = col / sh.group;
    const bool in = row < sh.N && grp < groups && col < sh.K;
    ds[i] = in ? load_as_f32(scales, dt, row * groups + grp) : 0.f;
    if (dz) dz[i] = in ? zeros[row * groups + grp] : 0;
  }
}

// ---- activations ----------------------------------------------------------------
// An even power of two (see x_scale_root) that brings the largest |code| (m) to [64, 256): the
// remainders of the exact codebook then stay normal fp16 numbers.
__device__ __forceinline__ float code_scale_of(float m) {
  if (!(m > 0.f)) return 1.f;
  const int e = 6 - ilogbf(m);
  return ldexpf(1.f, max(-120, min(120, e + (e & 1))));
}
__device__ __forceinline__ float code_scale(const float* code) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fabsf(__ldg(code + i));
    if (a <= 3.4e38f) m = fmaxf(m, a);
  }
  return code_scale_of(m);
}

// The power of two (and its reciprocal) that brings m, the largest of some values, to [2^14,
// 2^15), from its exponent bits; m below 2^-111 (0 too) is left smaller.  m is finite.
__device__ __forceinline__ float x_scale_for(float m, float& inv) {
  const int e = max(16, (int)(__float_as_uint(m) >> 23));
  inv = __uint_as_float((uint32_t)(268 - e) << 23);
  return __uint_as_float((uint32_t)(e - 14) << 23);
}

// Of a tile of x: what its products are multiplied by is 2^(2 j), and half of it, 2^j, goes to the
// product and half to the weights' scale.  As one factor it would make that scale subnormal for a
// tiny x, and the product infinite for a large one.  Scales s and inv of x (powers of two) are
// moved so that the exponent is even; icode, what the codebook's scale takes back, has one.
__device__ __forceinline__ float x_scale_root(float& s, float& inv, float icode) {
  const int e = (int)(__float_as_uint(s) >> 23) - 127;
  if (e & 1) {
    s *= 2.f;
    inv *= 0.5f;
  }
  const int j = ((int)(__float_as_uint(s) >> 23) - 127 + (int)(__float_as_uint(icode) >> 23) - 127) / 2;
  return __uint_as_float((uint32_t)(127 + j) << 23);
}

// A codebook entry (scaled) as two fp16, value and remainder (in the upper half), 22 bits.  The
// value is cut towards zero and the remainder is never 0 beside a value that is not, so that both
// have one sign: an infinite x times the two is infinite, not NaN.  That costs a value at most
// 2^-24, 2^-30 of the largest (one below 2^-24 itself, 2^-29 of it).
__device__ __forceinline__ uint32_t split_code(float c) {
  const uint32_t sign = __float_as_uint(c) >> 31 << 15;
  uint32_t h = __half_as_ushort(__float2half_rz(c)), r = 0;
  if (c != 0.f) {
    if ((h & 0x7fffu) == 0) h = sign | 1u;
    const float rem = c - __half2float(__ushort_as_half((unsigned short)h));  // NaN beside an infinity
    r = __half_as_ushort(__float2half_rn(rem));
    if (!(fabsf(rem) > 0.f) || (r & 0x7fffu) == 0 || (r & 0x8000u) != sign) r = sign | 1u;
  }
  return h | r << 16;
}
// The entry as one fp16; what is not 0 stays so, for infinite x.
__device__ __forceinline__ uint32_t round_code(float c) {
  const uint32_t h = __half_as_ushort(__float2half_rn(c));
  return c != 0.f && (h & 0x7fffu) == 0 ? h | 1u : h;
}
// The sums of an fp32 x's values and of its remainders.  Infinite weights make the first infinite
// or NaN, which it then is; the second's sign says nothing.
__device__ __forceinline__ float join_remainder(float value, float rem) {
  return fabsf(value) <= 3.4028234e38f ? value + rem : value;
}

// Eight columns of a row of x on their way to an operand tile.
struct XRun {
  uint32_t r[8];  // fp32 values, or four words of 16-bit pairs
  __device__ __forceinline__ void load(const void* x, int dtype, int64_t stride, int rows, int K, int row, int col) {
    const int es = dtype == NSM_F32 ? 4 : 2;
    const char* at = static_cast<const char*>(x) + ((int64_t)row * stride + col) * es;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = 0;
    if (row >= rows || col >= K) return;
    if (((uintptr_t)at & 15) == 0 && col + 8 <= K) {
      const uint4 a = *reinterpret_cast<const uint4*>(at);
      r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w;
      if (es == 4) {
        const uint4 b = *reinterpret_cast<const uint4*>(at + 16);
        r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (col + i < K) {
          if (es == 4) {
            r[i] = reinterpret_cast<const uint32_t*>(at)[i];
          } else {
            r[i / 2] |= (uint32_t) reinterpret_cast<const unsigned short*>(at)[i] << (16 * (i % 2));
          }
        }
      }
    }
  }
  __device__ __forceinline__ float value(int dtype, int i) const {  // fp32 or bf16
    return dtype == NSM_F32 ? __uint_as_float(r[i]) : __uint_as_float(i % 2 ? r[i / 2] & 0xffff0000u : r[i / 2] << 16);
  }
  __device__ __forceinline__ float largest(int dtype) const {  // infinities and NaN stay what they are
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(value(dtype, i));
      m = fmaxf(m, a <= 3.4028234e38f ? a : 0.f);
    }
    return m;
  }
  // As fp16 (and, for fp32, the remainders), times inv, a power of two.
  __device__ __forceinline__ void to_half(int dtype, float inv, uint4& hi, uint4& lo) const {
    if (dtype == NSM_F16) {
      hi = make_uint4(r[0], r[1], r[2], r[3]);
      return;
    }
    __half h[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = value(dtype, i) * inv;
      h[i] = __float2half_rn(x);
      const float rem = x - __half2float(h[i]);
      l[i] = __float2half_rn(fabsf(rem) <= 3.4028234e38f ? rem : 0.f);
    }
    auto pair = [](const __half* q, int i) {
      return (uint32_t)__half_as_ushort(q[2 * i]) | ((uint32_t)__half_as_ushort(q[2 * i + 1]) << 16);
    };
    hi = make_uint4(pair(h, 0), pair(h, 1), pair(h, 2), pair(h, 3));
    if (dtype == NSM_F32) lo = make_uint4(pair(l, 0), pair(l, 1), pair(l, 2), pair(l, 3));
  }
};

// Halves of column c of x, column k of the weight: [tile][k / 8][c / 8][c % 8][k % 8].
__device__ __forceinline__ int64_t x_index(int c, int k, int groups) {
  const int step = k / kL4TileCols, kk = k % kL4TileCols;
  return (((int64_t)step * (kL4TileCols / 8) + kk / 8) * groups + c / 8) * 64 + (c % 8) * 8 + kk % 8;
}

// CTA (slice, row): the row's largest value (each slice reads the whole row, from
// L2, rather than wait for the others), then its slice as fp16.  kp / 8 runs of eight columns.
__global__ void __launch_bounds__(256) lin4_prep_kernel(const void* x, int dt, int64_t stride, int K, int kp, int rows,
                                                        int groups, const float* code, __half* xh, float* scale) {
  pdl_trigger();
  __shared__ float wmax[8];
  const int r = blockIdx.y, runs = kp / 8;
  float s = 1.f, inv = 1.f;
  if (dt != NSM_F16) {
    float m = 0.f;
#pragma unroll 4
    for (int q = threadIdx.x; q < runs; q += 256) {
      XRun v;
      v.load(x, dt, stride, rows, K, r, 8 * q);
      m = fmaxf(m, v.largest(dt));
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
    __syncthreads();
    s = x_scale_for(warp_max(wmax[threadIdx.x & 7]), inv);
  }
  for (int q = blockIdx.x * 256 + threadIdx.x; q < runs; q += gridDim.x * 256) {
    XRun v;
    v.load(x, dt, stride, rows, K, r, 8 * q);
    uint4 hi, lo;
    v.to_half(dt, inv, hi, lo);
    *reinterpret_cast<uint4*>(xh + x_index(r, 8 * q, groups)) = hi;
    if (dt == NSM_F32) *reinterpret_cast<uint4*>(xh + x_index(rows + r, 8 * q, groups)) = lo;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) scale[r] = code ? s / code_scale(code) : s;
}

// ---- products -------------------------------------------------------------------
__device__ int g_lin4_error;  // a wait ran out: NSM_ERR_TIMEOUT until nsm_linear4bit_error reads it
__device__ __forceinline__ void lin4_failed() { atomicCAS(&g_lin4_error, 0, NSM_ERR_TIMEOUT); }

struct Lin4Params {
  const uint8_t* w;
  const float* s;
  const uint8_t* z;
  const float* code;
  const void* x;     // [rows][K], read by the kernel itself (NC <= 8)
  const __half* xh;  // or its tiles from lin4_prep_kernel
  int64_t x_stride;
  int x_dtype, rows, K;
  float* part;  // [row block][segment][column of x][512]
  int row_tiles, steps, scale_steps, div, cols;
  int units, ctas, max_segs, wait_limit;
  // One launch, a cluster of CTAs per row block (0: partials and lin4_finalize_kernel)
  int cluster, N;
  const float* scale;  // of x's rows, from lin4_prep_kernel
  const void* bias;
  void* out;
  int64_t out_stride;
  int bias_dt, out_dt;
};

__device__ __forceinline__ uint32_t hsub2_u32(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2_u32(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                            *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Nibbles k and k + 4 (k = kPair) of an integer word as half2 {q - z, q' - z}:
// 0x6400 | q is 1024 + q in fp16; the odd pairs are taken 4 bits higher (1024 +
// 16 q) and brought down by 1/16.  za = 1024 + z, zb = -(64 + z): all exact.
template <uint32_t kMask>
__device__ __forceinline__ uint32_t masked_1024(uint32_t v) {  // (v & kMask) | 0x64006400 in one instruction
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "n"(kMask), "r"(0x64006400u));
  return r;
}
template <int kPair>
__device__ __forceinline__ uint32_t int_pair(uint32_t w, uint32_t za, uint32_t zb) {
  const uint32_t v = kPair >= 2 ? w >> 8 : w;
  if (kPair % 2 == 0) return hsub2_u32(masked_1024<0x000f000fu>(v), za);
  return hfma2_u32(masked_1024<0x00f000f0u>(v), 0x2c002c00u, zb);
}

// ---- tensor memory and the 5th-generation tensor core ----
// Volatile, so that they keep their order; no memory clobber, so that the compiler may
// move table reads over them (tensor memory is nothing that C++ code reads or writes).
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;"); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// 16 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;"); }
// The loaded registers pass through the wait, so that nothing uses them before it.
template <int N>
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]));
#pragma unroll
  for (int i = 1; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
  if constexpr (N == 1) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r[0]) : "r"(addr));
  } else if constexpr (N == 2) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr));
  } else if constexpr (N == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
  } else if constexpr (N == 16) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
  } else {
    static_assert(N == 8, "columns at a time");
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
  }
}
// D[128 lanes][N] (+)= A (tensor memory, fp16 pairs along K) x B (shared memory, K-major)
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b_desc), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// One lane of a converged warp; the compiler keeps the operands of what it guards in uniform
// registers, which tcgen05 instructions take.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
// The barrier is arrived at when the MMAs issued so far by this thread are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// What a kernel variant holds, for device and host.  NPG: scale granules per tile of 128
// columns.  NC: columns of x that the sums hold.
template <int MODE, int NPG, int NC>
struct Lin4Config {
  static constexpr bool kIsCode = MODE == kCode || MODE == kCodeExact;
  static constexpr int kXGroups = NC <= 8 ? 1 : NC / 8;                    // groups of eight columns of x
  static constexpr int kXBytes = kXGroups * 8 * kL4TileCols * 2;           // of a tile
  static constexpr bool kOwnX = NC <= 8;                                   // the kernel makes x's tiles itself
  static constexpr int kN = NC <= 16 ? 16 : 32;                            // of the MMA
  // A whole tile as one slot (64 columns of tensor memory) whose MMAs the other warpgroups' work
  // hides, where the products fit beside it; else slots of 32 columns, two or three of them.
  static constexpr bool kWhole = MODE != kCodeExact && NPG * kN <= 64;
  static constexpr int kSlotCols = kWhole ? 128 : MODE == kCodeExact ? 32 : 64;  // weight columns of a slot
  static constexpr int kSlots = kL4TileCols / kSlotCols;                   // per tile
  static constexpr int kScalesPerSlot = NPG >= kSlots ? NPG / kSlots : 1;
  static constexpr int kSlotsPerScale = NPG >= kSlots ? 1 : kSlots / NPG;
  // Rounds of MMAs under way while the warpgroup fills the next slot
  static constexpr int kDCols = kScalesPerSlot * kN;
  static constexpr int kLag = !kWhole && 3 * 32 + 2 * kDCols <= (int)kL4TmemGroup ? 2 : 1;
  static constexpr int kASlots = kWhole ? 1 : kLag + 1;
  static constexpr uint32_t kD = kWhole ? 64 : kASlots * 32;  // where the products begin
  static_assert((int)kD + kLag * kDCols <= (int)kL4TmemGroup, "tensor memory");
  static constexpr int kScaleBytes = kL4TileRows * NPG * 4;
  static constexpr int kStageBytes = kL4TileBytes + kScaleBytes + (MODE == kIntZeros ? kL4TileRows * NPG : 0);
  static constexpr int kStages = kIsCode ? 3 : 4;                          // weight tiles in flight per warpgroup
  static constexpr int kLut = kIsCode ? kLutBytes : 0;
  static constexpr int kRing = kLut, kX = kRing + kL4Groups * kStages * kStageBytes;
  static constexpr int kBars = kX + kL4XStages * kXBytes + 1024;  // the last tile of x is read 128 bytes over
  static constexpr int kSmem = kBars + kL4BarBytes;
  static_assert(kSmem <= 227 * 1024, "shared memory of an SM");
  static_assert(kX - kRing >= kL4BlockRows * NC * 4, "a cluster's sums fit the rings");
};

struct Lin4Bars {
  unsigned long long w_full[kL4Groups][4];  // a tile of weights and its scales are in shared memory
  unsigned long long full[kL4Groups][2];    // a slot of weights is in tensor memory (rounds in turn)
  unsigned long long done[kL4Groups][2];    // its MMAs are done
  unsigned long long x_full[kL4XStages];    // a tile of x is in shared memory
  unsigned long long x_free[kL4XStages];    // all warpgroups' MMAs that read it are done
  unsigned long long drained[kL4Groups];    // all of the warpgroup's MMAs are done
  unsigned long long dead[2];               // where a warp arrives instead of at `full` after a failure
  float x_scale[kL4XStages][8];             // kOwnX: of a tile's columns of x (x_scale_root)
  uint32_t tmem;
  int asked[kL4XStages];   // by the warps that bring tiles, at their end: the last unit whose weights each asked for
  int failed[kL4XStages];  // and whether a wait of theirs ran out
};
static_assert(sizeof(Lin4Bars) <= kL4BarBytes, "barriers");

template <int MODE, int NPG, int NC, bool kCluster>
__global__ void __launch_bounds__(kL4Threads, 1) lin4_kernel(const __grid_constant__ Lin4Params p) {
  extern __shared__ __align__(1024) uint32_t l4_smem[];
  using C = Lin4Config<MODE, NPG, NC>;
  constexpr int kSlotCols = C::kSlotCols, kSlots = C::kSlots;
  constexpr int kScalesPerSlot = C::kScalesPerSlot, kSlotsPerScale = C::kSlotsPerScale, kLag = C::kLag;
  constexpr int kScaleCols = kSlotCols / kScalesPerSlot;  // columns of one product
  constexpr int kLd = NC < 32 ? NC : 16;                  // products read at a time
  // fp32 accumulators, fp16 operands, both K-major, N / 8 and M / 16 in bits 17 and 24
  constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(C::kN / 8) << 17) | ((128u / 16) << 24);

  unsigned char* smem = reinterpret_cast<unsigned char*>(l4_smem);
  Lin4Bars& bars = *reinterpret_cast<Lin4Bars*>(smem + C::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = threadIdx.x & 127;
  int u0, u1;
  if constexpr (kCluster) {  // (no trigger: what comes next reads what this kernel writes)
    const int block = blockIdx.x / p.cluster, rank = blockIdx.x - block * p.cluster;
    u0 = block * p.steps + p.steps * rank / p.cluster;
    u1 = block * p.steps + p.steps * (rank + 1) / p.cluster;
  } else {
    u0 = stream_begin(p.units, p.ctas, blockIdx.x);
    u1 = stream_begin(p.units, p.ctas, blockIdx.x + 1);
    pdl_trigger();
  }

  // warps 0-15: the warpgroups; 16-19: one that issues MMAs for each; 20-23: bring the tiles
  const int my_warp = __shfl_sync(0xffffffffu, warp, 0);
  const bool issuing = my_warp >= 4 * kL4Groups && my_warp < 5 * kL4Groups, bringing = my_warp >= 5 * kL4Groups;
  const int wg = issuing ? my_warp - 4 * kL4Groups : my_warp >> 2;
  const uint64_t once = l2_evict_first_policy();
  auto copy_weights = [&](int i, int g) {  // a lane's: tile, scales and zero points of unit u0 + i, warpgroup g
    const int at_rb = (u0 + i) / p.steps, at = u0 + i - at_rb * p.steps;
    const int64_t rt = (int64_t)at_rb * kL4Groups + g;
    if (rt < p.row_tiles) {
      const uint32_t bar = smem_u32(&bars.w_full[g][i % C::kStages]);
      const uint32_t dst = smem_u32(smem + C::kRing + (g * C::kStages + i % C::kStages) * C::kStageBytes);
      const int64_t e = (rt * p.scale_steps + ((NPG == 1 && p.div > 1) ? at / p.div : at)) * (kL4TileRows * NPG);
      mbar_arrive_expect_tx(bar, C::kStageBytes);
      bulk_g2s(dst, p.w + (rt * p.steps + at) * kL4TileBytes, kL4TileBytes, bar, once);
      bulk_g2s(dst + kL4TileBytes, p.s + e, C::kScaleBytes, bar, once);
      if (MODE == kIntZeros) bulk_g2s(dst + kL4TileBytes + C::kScaleBytes, p.z + e, kL4TileRows * NPG, bar, once);
    }
  };
  constexpr int kRuns = C::kOwnX ? (NC + 1) / 2 : 1;
  XRun v[kRuns];  // of a warp that brings x: lanes 0-15 8 columns each of row 2q, lanes 16-31 of row 2q + 1
  auto load_x = [&](int i) {
    const int col = (u0 + i) % p.steps * kL4TileCols + 8 * (lane & 15);
#pragma unroll
    for (int q = 0; q < kRuns; ++q) v[q].load(p.x, p.x_dtype, p.x_stride, p.rows, p.K, 2 * q + (lane >> 4), col);
  };

  // Without lin4_prep_kernel in front, nothing in global memory is read or written before the
  // kernel before this one is done; with it, only x waits (the weights are not its work).
  if (C::kOwnX) pdl_wait();
  if (my_warp == 5 * kL4Groups) {  // the first copies are under way while the rest is set up
    // the barriers in the order of Lin4Bars, and what they count
    constexpr int kFull = kL4Groups * 4, kDone = kFull + kL4Groups * 2, kXFree = kDone + kL4Groups * 2 + kL4XStages;
    constexpr int kDrained = kXFree + kL4XStages;
    for (int i = lane; i < kDrained + kL4Groups + 2; i += 32)
      mbar_init(smem_u32(&bars) + 8 * i, i >= kXFree && i < kDrained ? kL4Groups : i >= kFull && i < kDone ? 4 : 1);
    mbar_init_fence();
    __syncwarp();
    if (lane < kL4Groups * C::kStages && lane / kL4Groups < u1 - u0) copy_weights(lane / kL4Groups, lane % kL4Groups);
    __syncwarp();
  }
  if (C::kOwnX && bringing && my_warp - 5 * kL4Groups < u1 - u0) load_x(my_warp - 5 * kL4Groups);
  if (my_warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)),
                 "r"(kL4Groups * kL4TmemGroup)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  int rb = u0 / p.steps, step = u0 - rb * p.steps;

  if (C::kIsCode && !bringing) {  // byte -> half2 table, one copy per lane (conflict-free); the second holds the remainders
    const float code = __ldg(p.code + (lane & 15));
    const float mine = fabsf(code) <= 3.4e38f ? fabsf(code) : 0.f;
    const float scaled = code * code_scale_of(warp_max(mine));
    const uint32_t halves = MODE == kCodeExact ? split_code(scaled) : round_code(scaled);
    uint4* lut4 = reinterpret_cast<uint4*>(smem);
    for (int e = my_warp; e < 256; e += kL4Groups * 5) {  // a warp per byte: 8 lanes fill a table's 32 words
      const uint32_t c0 = __shfl_sync(0xffffffffu, halves, e >> 4), c1 = __shfl_sync(0xffffffffu, halves, e & 15);
      const uint32_t v = __byte_perm(c0, c1, lane & 8 ? 0x7632 : 0x5410);
      if (lane < (MODE == kCodeExact ? 16 : 8)) lut4[e * 16 + lane] = make_uint4(v, v, v, v);
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars.tmem, 0);

  // Every wait is bounded.  After one that ran out nothing more is copied, multiplied or handed
  // on, so the waits that depend on it run out too, and the warpgroups that saw one leave NaN in
  // their partials and record NSM_ERR_TIMEOUT.  Copies and MMAs under way are waited for before
  // the CTA ends.
  if (bringing) {
    // ---- tiles: each of these warps fills one place of x's ring, and when all MMAs that read it
    // are done, so that all warpgroups have read their weights of that unit too, the place of those
    const int st = my_warp - 5 * kL4Groups, count = u1 - u0;
    const uint32_t full = smem_u32(&bars.x_full[st]), free = smem_u32(&bars.x_free[st]);
    unsigned char* dst = smem + C::kX + st * C::kXBytes;
    const uint64_t keep = l2_evict_last_policy();
    const float icode = C::kOwnX && C::kIsCode ? 1.f / code_scale(p.code) : 1.f;  // a power of two
    bool ok = true;
    int w_last = st < min(C::kStages, count) ? st : -1;  // the last unit of this place whose weights were asked for
    int x_last = -1;                                     // and the last round of x
    if (!C::kOwnX) {
      pdl_wait();
      fence_proxy_async_global();
    }
    for (int i = st; i < count + kL4XStages - C::kStages; i += kL4XStages) {
      if (i >= kL4XStages) {
        ok = mbar_wait(free, (i / kL4XStages - 1) & 1, p.wait_limit);
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        const int j = i - kL4XStages + C::kStages;
        if (j < count) {
          fence_proxy_async_smem();
          if (lane < kL4Groups) copy_weights(j, lane);
          w_last = j;
          __syncwarp();
        }
      }
      if (i >= count) break;
      x_last = i / kL4XStages;
      if constexpr (C::kOwnX) {
#pragma unroll
        for (int q = 0; q < kRuns; ++q) {
          const int r = 2 * q + (lane >> 4);
          uint4 hi, lo;
          float s = 1.f, inv = 1.f;
          if (p.x_dtype != NSM_F16) {  // a scale for the row's 128 columns: the half-warp's
            float m = v[q].largest(p.x_dtype);
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            s = x_scale_for(m, inv);
          }
          const float root = x_scale_root(s, inv, icode);
          v[q].to_half(p.x_dtype, inv, hi, lo);
          if (r < p.rows) {
            // core matrices of 8 columns of x by 8 of the weight: [k / 8][c][k % 8]
            *reinterpret_cast<uint4*>(dst + ((lane & 15) * 8 + r) * 16) = hi;
            if ((lane & 15) == 0) bars.x_scale[st][r] = root;
            if (p.x_dtype == NSM_F32) {
              *reinterpret_cast<uint4*>(dst + ((lane & 15) * 8 + p.rows + r) * 16) = lo;
              if ((lane & 15) == 0) bars.x_scale[st][p.rows + r] = root;
            }
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
        if (i + kL4XStages < count) load_x(i + kL4XStages);
      } else if (lane == 0) {
        mbar_arrive_expect_tx(full, C::kXBytes);
        bulk_g2s(smem_u32(dst), reinterpret_cast<const unsigned char*>(p.xh) + (int64_t)((u0 + i) % p.steps) * C::kXBytes, C::kXBytes, full,
                 keep);
      }
    }
    // Nothing may arrive in shared memory that is gone: the last commits (they come after the
    // copies they waited for), and after a failure the copies under way.  The units that use a
    // warp's last copies may be another's to wait for, so a failure of one is a failure of all;
    // and where another has filled the same place of the ring since, these were waited for.
    if (lane == 0 && x_last >= 0 && ok) ok = mbar_wait(free, x_last & 1, p.wait_limit);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    if (lane == 0) {
      bars.asked[st] = w_last;
      bars.failed[st] = !ok;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kL4XStages * 32) : "memory");
    bool failed = false, newest = w_last >= 0;
#pragma unroll
    for (int o = 0; o < kL4XStages; ++o) {
      failed |= bars.failed[o] != 0;
      newest &= !(bars.asked[o] > w_last && bars.asked[o] % C::kStages == w_last % C::kStages);
    }
    if (failed) {
      if (lane == 0) lin4_failed();
      if (lane < kL4Groups && newest && (u0 + w_last) / p.steps * kL4Groups + lane < p.row_tiles)
        mbar_wait(smem_u32(&bars.w_full[lane][w_last % C::kStages]), (w_last / C::kStages) & 1);
      if (!C::kOwnX && lane == 0 && x_last >= 0) mbar_wait(full, x_last & 1);
    }
    __syncwarp();
  } else if (issuing) {
    // ---- the warpgroup's MMAs
    const uint32_t a0 = tmem + wg * kL4TmemGroup;
    const uint32_t full_bar = smem_u32(&bars.full[wg][0]), done_bar = smem_u32(&bars.done[wg][0]);
    bool ok = true;
    int slots = 0, xst = 0, x_phase = 0;  // rounds so far, ring position of x
    uint32_t a_col = 0, d_col = C::kD;    // of this round
    for (int u = u0; u < u1; ++u) {
      const uint32_t xfree = smem_u32(&bars.x_free[xst]);
      ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bars.x_full[xst]), x_phase, p.wait_limit));
      if (!ok) break;
      if (rb * kL4Groups + wg < p.row_tiles) {
        const uint32_t x0 = smem_u32(smem + C::kX + xst * C::kXBytes);
        // K-major without swizzle: 8 columns of the weight are kXGroups x 128 bytes on, 8 columns of
        // x 128 bytes (with one group the upper eight of N = 16 are never read back)
        const uint64_t desc0 = (uint64_t)((x0 >> 4) & 0x3fff) | ((uint64_t)(C::kXGroups * 128 / 16) << 16) |
                               ((uint64_t)(128 / 16) << 32) | (1ull << 46);
#pragma unroll
        for (int t = 0; t < kSlots; ++t) {
          ok = mbar_wait(full_bar + 8 * (slots & 1), (slots >> 1) & 1, p.wait_limit);
          __syncwarp();
          tmem_fence_after();
          const uint32_t a = a0 + a_col;
          if (elect_one() && ok) {
#pragma unroll
            for (int k = 0; k < kSlotCols / 16; ++k) {
              const uint32_t d = a0 + d_col + (16 * k / kScaleCols) * C::kN;
#pragma unroll
              for (int half = 0; half < (MODE == kCodeExact ? 2 : 1); ++half)
                mma_f16_ts(d, a + half * (kSlotCols / 2) + k * 8,
                           desc0 + (uint64_t)((t * (kSlotCols / 8) + 2 * k) * C::kXGroups * 128 / 16), kIdesc,
                           !(t % kSlotsPerScale == 0 && half == 0 && 16 * k % kScaleCols == 0));
            }
            mma_commit(done_bar + 8 * (slots & 1));
            if (t == kSlots - 1) mma_commit(xfree);
          }
          ++slots;
          ok = __all_sync(0xffffffffu, ok);  // after the MMAs: they wait for no vote
          if (!ok) break;
          a_col = a_col == (C::kASlots - 1) * 32 ? 0 : a_col + 32;
          if (kLag == 2 && t % kSlotsPerScale == kSlotsPerScale - 1) d_col ^= C::kD ^ (C::kD + C::kDCols);
        }
        if (!ok) break;
      } else if (lane == 0) {  // no rows here (in the last row block): only x goes by
        mbar_arrive(xfree);
      }
      if (++xst == kL4XStages) {
        xst = 0;
        x_phase ^= 1;
      }
      if (++step == p.steps) {
        step = 0;
        ++rb;
      }
    }
    // tensor memory and the tiles of x outlive the MMAs: a barrier of their own, as after a failure
    // the warpgroup has not waited for them
    __syncwarp();
    if (slots > 0) {
      if (elect_one()) mma_commit(smem_u32(&bars.drained[wg]));
      __syncwarp();
      mbar_wait(smem_u32(&bars.drained[wg]), 0);
    }
    __syncwarp();
  } else {
    // ---- the warpgroup: 4 bits -> fp16 -> tensor memory, and the sums
    const uint32_t mine = tmem + wg * kL4TmemGroup + ((uint32_t)(my_warp & 3) << 21);  // this warp's 32 lanes
    const uint32_t lanebase = (uint32_t)lane * 4u;
    uint32_t full_bar = smem_u32(&bars.full[wg][0]);
    const uint32_t done_bar = smem_u32(&bars.done[wg][0]);
    // sums of two columns each (16 columns 41.5 -> 40.0 us, 32 44.4 -> 43.4), or of one
    unsigned long long acc[(NC + 1) / 2] = {};
    float acc1 = 0.f;
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (ok && !mbar_wait(bar, parity, p.wait_limit)) {
        ok = false;
        full_bar = smem_u32(&bars.dead[0]);  // (testing ok at each arrival took 2% more with 32 columns)
      }
    };
    int slots = 0;                         // rounds so far
    uint32_t a_col = 0, d_col = C::kD;     // of this round; of the products to add next
    constexpr int kXs = C::kOwnX ? NC : 1;
    float ps[NPG], pxs[kXs];               // the scales of the tile before, its weights' and x's
    int open = -1;                         // its row block: that of the sums
    // waits for round i; its products, scaled, join the sums if they are whole
    auto add_round = [&](int i, bool whole, const float* s, const float* xs) {
      wait(done_bar + 8 * (i & 1), (i >> 1) & 1);
      __syncwarp();
      tmem_fence_after();
      if (whole) {
#pragma unroll
        for (int g = 0; g < kScalesPerSlot; ++g) {
#pragma unroll
          for (int c0 = 0; c0 < NC; c0 += kLd) {
            uint32_t r[kLd];
            tmem_ld<kLd>(mine + d_col + g * C::kN + c0, r);
            tmem_wait_ld<kLd>(r);
            if constexpr (NC == 1) {
              acc1 = fmaf(s[g] * xs[0], __uint_as_float(r[0]) * xs[0], acc1);
            } else {
#pragma unroll
              for (int c = 0; c < kLd; c += 2) {
                unsigned long long sc = pair2(s[g], s[g]), d = pair2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
                if constexpr (C::kOwnX) {  // (powers of two: exact)
                  const unsigned long long root = pair2(xs[c0 + c], xs[c0 + c + 1]);
                  sc = mul2(sc, root);
                  d = mul2(d, root);
                }
                acc[(c0 + c) / 2] = fma2(sc, d, acc[(c0 + c) / 2]);
              }
            }
          }
        }
        if (kLag == 2) d_col ^= C::kD ^ (C::kD + C::kDCols);
      }
    };
    auto flush = [&]() {
      const int seg = (int)blockIdx.x - stream_owner(p.units, p.ctas, open * p.steps);
      float* dst = p.part + ((int64_t)(open * p.max_segs + seg) * p.cols) * kL4BlockRows + wg * kL4TileRows + row;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float2 v = NC == 1 ? make_float2(acc1, 0.f) : unpair2(acc[c / 2]);
        if (c < p.cols) dst[(int64_t)c * kL4BlockRows] = !ok ? __int_as_float(0x7fc00000) : c % 2 ? v.y : v.x;
        if (c % 2 == 1) acc[c / 2] = 0;
      }
      acc1 = 0.f;
    };
    int st = 0, w_phase = 0, xst = 0, x_phase = 0;  // ring positions
    for (int u = u0; u < u1; ++u) {
      if (rb * kL4Groups + wg >= p.row_tiles) break;  // no rows here, nor later
      const uint32_t stage = smem_u32(smem + C::kRing + (wg * C::kStages + st) * C::kStageBytes);
      wait(smem_u32(&bars.w_full[wg][st]), w_phase);
      float s[NPG], xs[kXs];
      if constexpr (C::kOwnX) {
        wait(smem_u32(&bars.x_full[xst]), x_phase);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(xs[c]) : "r"(smem_u32(&bars.x_scale[xst][c])));
        if (++xst == kL4XStages) {
          xst = 0;
          x_phase ^= 1;
        }
      }
      uint32_t z = 0;
      {
        const uint32_t sa = stage + kL4TileBytes + row * NPG * 4, za = stage + kL4TileBytes + C::kScaleBytes + row * NPG;
        if constexpr (NPG == 1) {
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s[0]) : "r"(sa));
          if (MODE == kIntZeros) asm volatile("ld.shared.u8 %0, [%1];" : "=r"(z) : "r"(za));
        } else if constexpr (NPG == 2) {
          asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(s[0]), "=f"(s[1]) : "r"(sa));
          if (MODE == kIntZeros) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(z) : "r"(za));
        } else {
          const float4 v = lds_f4(sa);
          s[0] = v.x;
          s[1] = v.y;
          s[2] = v.z;
          s[3] = v.w;
          if (MODE == kIntZeros) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(z) : "r"(za));
        }
      }
      auto add_earlier = [&](int t) {  // the round kLag before slot t's, which went on meanwhile
        const int was = (t + kSlots - kLag) % kSlots;  // its slot: of this tile, or of the one before
        constexpr int kLast = kSlotsPerScale - 1;
        if (t >= kLag) {
          add_round(slots - kLag, was % kSlotsPerScale == kLast, s + was * NPG / kSlots, xs);
        } else if (open >= 0) {
          add_round(slots - kLag, was % kSlotsPerScale == kLast, ps + was * NPG / kSlots, pxs);
          if (!kCluster && was == kSlots - 1 && open != rb) flush();  // (a cluster's CTA has one row block)
        }
      };
#pragma unroll
      for (int t = 0; t < kSlots; ++t) {
#pragma unroll
        for (int c = 0; c < kSlotCols / 32; ++c) {
          const uint4 q = lds_u4(stage + ((t * (kSlotCols / 32) + c) * kL4TileRows + row) * 16);
          const uint32_t word[4] = {q.x, q.y, q.z, q.w};
          uint32_t za = 0x64086408u, zb = 0xd480d480u;  // 1024 + 8, -(64 + 8)
          if constexpr (MODE == kIntZeros) {
            za = (0x6400u | ((z >> (8 * ((t * kSlotCols + c * 32) * NPG / kL4TileCols))) & 255u)) * 0x10001u;
            zb = hsub2_u32(0x63806380u, za);  // 960 - (1024 + z)
          }
#pragma unroll
          for (int half = 0; half < (MODE == kCodeExact ? 2 : 1); ++half) {
            uint32_t r[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if constexpr (C::kIsCode) {
#pragma unroll
                for (int b = 0; b < 4; ++b) r[4 * j + b] = lut_lookup_rt(l4_smem, word[j], lanebase, b, half);
              } else {
                r[4 * j] = int_pair<0>(word[j], za, zb);
                r[4 * j + 1] = int_pair<1>(word[j], za, zb);
                r[4 * j + 2] = int_pair<2>(word[j], za, zb);
                r[4 * j + 3] = int_pair<3>(word[j], za, zb);
              }
            }
            if (C::kWhole && c == 0) add_earlier(t);  // the slot is free
            tmem_st16(mine + a_col + half * (kSlotCols / 2) + c * 16, r);
          }
        }
        if (!C::kWhole) add_earlier(t);
        tmem_wait_st();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar + 8 * (slots & 1));
        ++slots;
        a_col = a_col == (C::kASlots - 1) * 32 ? 0 : a_col + 32;
      }
      open = rb;
#pragma unroll
      for (int g = 0; g < NPG; ++g) ps[g] = s[g];
#pragma unroll
      for (int c = 0; c < kXs; ++c) pxs[c] = xs[c];
      if (++st == C::kStages) {
        st = 0;
        w_phase ^= 1;
      }
      if (++step == p.steps) {
        step = 0;
        ++rb;
      }
    }
    if (open >= 0) {
#pragma unroll
      for (int t = kSlots - kLag; t < kSlots; ++t)
        add_round(slots - kSlots + t, t % kSlotsPerScale == kSlotsPerScale - 1, ps + t * NPG / kSlots, pxs);
      if (!kCluster) flush();
    }
    if (!ok) lin4_failed();
    __syncwarp();
    tmem_fence_before();
    if constexpr (kCluster) {
      // The cluster's CTAs share the row block's outputs: each gets the sums of its slice of rows
      // into its weight rings, which nobody reads any more, and adds them in the CTAs' order.
      const int slice = kL4BlockRows / p.cluster, block = blockIdx.x / p.cluster, rank = blockIdx.x - block * p.cluster;
      const int mine_at = wg * kL4TileRows + row, to = mine_at / slice;
      float* const sums = reinterpret_cast<float*>(smem + C::kRing);  // [CTA][column of x][row of the slice]
      cluster_arrive();
      cluster_wait();
      const uint32_t dst = in_cluster_cta(smem_u32(sums + rank * p.cols * slice + mine_at % slice), to);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float2 v = NC == 1 ? make_float2(acc1, 0.f) : unpair2(acc[c / 2]);
        const float e = !ok ? __int_as_float(0x7fc00000) : c % 2 ? v.y : v.x;
        if (c < p.cols) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + c * slice * 4), "f"(e) : "memory");
      }
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      for (int o = threadIdx.x; o < slice * p.rows; o += kL4Groups * 128) {
        const int r = o / slice, i = o - r * slice, n = block * kL4BlockRows + rank * slice + i;
        if (n >= p.N) continue;
        float v = 0.f;
        for (int k = 0; k < p.cluster; ++k) {
          const float* at = sums + (k * p.cols + r) * slice + i;
          v += p.cols > p.rows ? join_remainder(at[0], at[p.rows * slice]) : at[0];
        }
        if (!C::kOwnX) v *= __ldcg(p.scale + r);
        if (p.bias) v += load_as_f32(p.bias, p.bias_dt, n);
        store_from_f32(p.out, p.out_dt, (int64_t)r * p.out_stride + n, v);
      }
    }
  }
  if (kCluster && my_warp >= 4 * kL4Groups) {
    cluster_arrive();
    cluster_wait();
    cluster_arrive();
    cluster_wait();
  }
  __syncthreads();
  tmem_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kL4Groups * kL4TmemGroup) : "memory");
}

// An output's segments are added as four sums, of every fourth each, and these in order: the same
// bits every time, and whether one thread or four (kShare) do it, so whatever the number of rows.
// Four threads where an output has more than four segments and the threads of all outputs fit the
// GPU at once (4096 outputs of one row: 3.7 -> 1.5 us), else one (16384 outputs of 32 rows would
// take 10 us more with four).  kMany: more than four segments; with four at most each is a sum of
// its own, and the loop is short (104 us -> 111 with the other at 53248 outputs of 32 rows).
template <int kShare, bool kMany>
__global__ void __launch_bounds__(kL4BlockRows) lin4_finalize_kernel(const float* part, const float* scale, int units,
                                                                       int ctas, int steps, int max_segs, int cols,
                                                                       int rows, int N, const void* bias, int bias_dt,
                                                                       void* out, int out_dt, int64_t out_stride) {
  constexpr int kRows = kL4BlockRows / kShare;
  __shared__ float sums[kShare][kRows];
  const int i = threadIdx.x % kRows, q = threadIdx.x / kRows;
  const int n = blockIdx.x * kRows + i, rb = n / kL4BlockRows, r = blockIdx.y;
  __shared__ int owner[2];  // the first and last CTA of the row block (64-bit divisions: by two threads)
  if (threadIdx.x < 2) owner[threadIdx.x] = stream_owner(units, ctas, rb * steps + (threadIdx.x ? steps - 1 : 0));
  __syncthreads();
  const int segs = owner[1] - owner[0] + 1;
  pdl_wait();
  const float* src = part + ((int64_t)rb * max_segs * cols + r) * kL4BlockRows + n % kL4BlockRows;
  auto load = [&](int k) {
    const float* at = src + (int64_t)k * cols * kL4BlockRows;
    return cols > rows ? join_remainder(__ldcg(at), __ldcg(at + (int64_t)rows * kL4BlockRows)) : __ldcg(at);
  };
  float v = 0.f;
  if (kShare > 1) {
#pragma unroll 8
    for (int k = q; k < segs; k += kShare) v += load(k);
    sums[q][i] = v;
    __syncthreads();
#pragma unroll
    for (int j = 1; j < kShare; ++j) v += sums[j][i];
  } else if (!kMany) {
#pragma unroll 4
    for (int k = 0; k < segs; ++k) v += load(k);
  } else {
    float u[4] = {};
    for (int k0 = 0; k0 < segs; k0 += 8) {  // eight loads under way
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = k0 + j < segs ? load(k0 + j) : 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j % 4] += e[j];
    }
    v = ((u[0] + u[1]) + u[2]) + u[3];
  }
  if (q != 0 || n >= N) return;
  if (scale) v *= __ldcg(scale + r);
  if (bias) v += load_as_f32(bias, bias_dt, n);
  store_from_f32(out, out_dt, (int64_t)r * out_stride + n, v);
}

// Tries of a wait: 0 = copy_wait_spins(), -1 = none.
std::atomic<int> g_lin4_wait{0};
int lin4_wait_limit() {
  const int tries = g_lin4_wait.load(std::memory_order_relaxed);
  return tries == 0 ? copy_wait_spins() : std::max(tries, 0);
}

struct Lin4Plan {
  bool own_x = false;  // few columns: the kernel reads x itself
  int cluster = 0;     // CTAs of a row block in one launch, 0: partials and lin4_finalize_kernel
  int cols = 0, col_groups = 1, units = 0, ctas = 0, max_segs = 0;
  size_t scale_off = 0, part_off = 0, bytes = 0;
};

bool lin4_size_ok(int N, int K, int group) {
  return N > 0 && K > 0 && K % 2 == 0 && group > 0 && group % 32 == 0 && N <= (1 << 24) && K <= (1 << 20) &&
         (int64_t)((N + 255) / 256) * ((K + 127) / 128) < (1 << 30);
}

int lin4_max_rows(int x_dtype) { return x_dtype == NSM_F32 ? kL4MaxCols / 2 : kL4MaxCols; }

struct Lin4Fn {
  void (*fn)(Lin4Params);
  int smem;
};

// Columns of x that the sums hold: the next of 1, 2, 4, 8, 16, 32.
int lin4_col_case(int cols) { return cols <= 1 ? 0 : cols <= 2 ? 1 : cols <= 4 ? 2 : cols <= 8 ? 3 : cols <= 16 ? 4 : 5; }

template <int MODE, int NPG, int NC, bool kCluster>
constexpr Lin4Fn lin4_fn() {
  return {lin4_kernel<MODE, NPG, NC, kCluster>, Lin4Config<MODE, NPG, NC>::kSmem};
}
template <int MODE, int NPG, bool kCluster>
Lin4Fn lin4_pick_cols(int c) {
  constexpr Lin4Fn fns[6] = {lin4_fn<MODE, NPG, 1, kCluster>(), lin4_fn<MODE, NPG, 2, kCluster>(),
                             lin4_fn<MODE, NPG, 4, kCluster>(), lin4_fn<MODE, NPG, 8, kCluster>(),
                             lin4_fn<MODE, NPG, 16, kCluster>(), lin4_fn<MODE, NPG, 32, kCluster>()};
  return fns[c];
}
template <int MODE, bool kCluster>
Lin4Fn lin4_pick_npg(int npg, int c) {
  return npg == 1   ? lin4_pick_cols<MODE, 1, kCluster>(c)
         : npg == 2 ? lin4_pick_cols<MODE, 2, kCluster>(c)
                    : lin4_pick_cols<MODE, 4, kCluster>(c);
}
template <bool kCluster>
Lin4Fn lin4_pick(int mode, int npg, int c) {
  return mode == kCode        ? lin4_pick_npg<kCode, kCluster>(npg, c)
         : mode == kCodeExact ? lin4_pick_npg<kCodeExact, kCluster>(npg, c)
         : mode == kInt       ? lin4_pick_npg<kInt, kCluster>(npg, c)
                              : lin4_pick_npg<kIntZeros, kCluster>(npg, c);
}

ClusterOnce lin4_once[2][4][3][6];  // of lin4_kernel's variants

int lin4_clusters_at_once(int ctas, const DeviceInfo& di) {
  static ClustersAtOnce known;
  const Lin4Fn f = lin4_fn<kCode, 1, 1, true>();  // as all of them: one CTA per SM
  if (lin4_once[1][kCode][0][0].set(f.fn, f.smem, di.device) != cudaSuccess) return -1;
  return known.get(f.fn, kL4Threads, f.smem, ctas, di);
}

// In one launch, a row block is a cluster's, cut evenly over its CTAs, and the sums join in shared
// memory: no finalize kernel and no workspace of partials.  The host then takes 8.5 us per call
// instead of 12, the GPU 0.4 to 0.7 us more (4096 x 4096 with the codebook in fp16 10.0 in a graph
// instead of 9.3), so it is taken where calls one after another wait for the host: runs of at most
// four units (0.94 us each; 1.64 with the codebook to 22 bits, where calls take 12.3 us), two longer
// than an even cut's, of clusters that fit the GPU at once (14336 x 4096, eight units instead of
// seven: 17.8 us instead of 17.2).  The choice depends on the weight's sizes alone, so a row's bits do
// not depend on the number of rows, nor the workspace on the codebook.
Lin4Plan lin4_plan(const Lin4Shape& sh, int rows, int x_dtype, const DeviceInfo& di) {
  Lin4Plan pl;
  pl.cols = x_dtype == NSM_F32 ? 2 * rows : rows;
  pl.units = sh.row_blocks * sh.steps;
  pl.ctas = std::max(1, std::min({di.sm_count, pl.units, sh.row_blocks * (kL4MaxSegs - 2)}));
  const int least = pl.units / pl.ctas;  // units of the shortest run
  pl.max_segs = (sh.steps - 1 + least - 1) / least + 1;
  pl.col_groups = pl.cols <= 8 ? 1 : pl.cols <= 16 ? 2 : 4;
  pl.own_x = pl.cols <= 8;
  pl.scale_off = pl.own_x ? 0 : align_up((size_t)pl.col_groups * 8 * sh.kp * 2, 256);
  pl.part_off = pl.scale_off + (pl.own_x ? 0 : align_up((size_t)rows * 4, 256));
  const int longest = (pl.units + pl.ctas - 1) / pl.ctas;
  int best = std::min(longest + 2, 4);
  for (int c = 1; c <= 16; c *= 2) {
    const int mine = (sh.steps + c - 1) / c;
    if (c > sh.steps || c * sh.row_blocks > di.sm_count) break;
    if (mine < best + (pl.cluster == 0) && lin4_clusters_at_once(c, di) >= sh.row_blocks) {
      best = mine;
      pl.cluster = c;
    }
  }
  pl.bytes = std::max<size_t>(
      256, pl.part_off + (pl.cluster > 0 ? 0 : (size_t)sh.row_blocks * pl.max_segs * pl.cols * kL4BlockRows * 4));
  return pl;
}

}  // namespace
}  // namespace nsm

using namespace nsm;

extern "C" {

size_t nsm_linear4bit_packed_bytes(int32_t out_features, int32_t in_features) {
  if (!lin4_size_ok(out_features, in_features, 32)) return 0;
  const Lin4Shape sh = lin4_shape(out_features, in_features, 32);
  return (size_t)sh.row_tiles * sh.steps * kL4TileBytes;
}

size_t nsm_linear4bit_scale_count(int32_t out_features, int32_t in_features, int32_t group_size) {
  if (!lin4_size_ok(out_features, in_features, group_size)) return 0;
  const Lin4Shape sh = lin4_shape(out_features, in_features, group_size);
  return (size_t)sh.row_tiles * sh.scale_steps * kL4TileRows * sh.npg;
}

int nsm_linear4bit_max_rows(int32_t x_dtype) { return lin4_max_rows(x_dtype); }

int nsm_linear4bit_error(int32_t* code_out, nsm_stream_t stream) {
  NSM_REQUIRE(code_out != nullptr, NSM_ERR_INVALID_ARG, "nsm_linear4bit_error: code_out is NULL");
  void* word = nullptr;
  NSM_CHECK_CUDA(cudaGetSymbolAddress(&word, g_lin4_error));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int32_t v = 0;
  NSM_CHECK_CUDA(cudaMemcpyAsync(&v, word, sizeof(int32_t), cudaMemcpyDeviceToHost, s));
  NSM_CHECK_CUDA(cudaMemsetAsync(word, 0, sizeof(int32_t), s));
  NSM_CHECK_CUDA(cudaStreamSynchronize(s));
  *code_out = v;
  return NSM_OK;
}

int nsm_linear4bit_set_wait_limit(int32_t tries) {
  NSM_REQUIRE(tries >= -1, NSM_ERR_INVALID_ARG, "nsm_linear4bit_set_wait_limit: tries must be >= -1");
  g_lin4_wait.store(tries, std::memory_order_relaxed);
  return NSM_OK;
}

int nsm_linear4bit_pack(const uint8_t* packed, int64_t packed_row_bytes, const void* scales, int32_t scale_dtype,
                        const uint8_t* zeros, int32_t out_features, int32_t in_features, int32_t group_size,
                        int32_t codebook, uint8_t* packed_out, float* scales_out, uint8_t* zeros_out,
                        nsm_stream_t stream) {
  NSM_REQUIRE(lin4_size_ok(out_features, in_features, group_size), NSM_ERR_UNSUPPORTED,
              "nsm_linear4bit_pack: in_features must be even, group_size a multiple of 32");
  NSM_REQUIRE(packed && scales && packed_out && scales_out && (zeros == nullptr) == (zeros_out == nullptr),
              NSM_ERR_INVALID_ARG, "nsm_linear4bit_pack: NULL pointer");
  NSM_REQUIRE(!(codebook && zeros), NSM_ERR_INVALID_ARG, "nsm_linear4bit_pack: a codebook has no zero points");
  NSM_REQUIRE(scale_dtype == NSM_F32 || scale_dtype == NSM_F16 || scale_dtype == NSM_BF16, NSM_ERR_INVALID_ARG,
              "nsm_linear4bit_pack: bad scale dtype");
  NSM_REQUIRE(packed_row_bytes >= in_features / 2, NSM_ERR_INVALID_ARG,
              "nsm_linear4bit_pack: packed_row_bytes is smaller than a row");
  NSM_REQUIRE(((uintptr_t)packed_out & 15) == 0 && ((uintptr_t)scales_out & 15) == 0 && ((uintptr_t)zeros_out & 15) == 0,
              NSM_ERR_INVALID_ARG, "nsm_linear4bit_pack: outputs must be 16-byte aligned");
  DeviceInfo di;
  const int rc = current_device(&di);
  if (rc != NSM_OK) return rc;
  const Lin4Shape sh = lin4_shape(out_features, in_features, group_size);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int groups = (in_features + group_size - 1) / group_size;
  const int64_t words = (int64_t)sh.row_tiles * sh.steps * (kL4TileBytes / 4);
  const int64_t ns = (int64_t)sh.row_tiles * sh.scale_steps * kL4TileRows * sh.npg;
  lin4_pack_kernel<<<(int)std::min<int64_t>((words + 255) / 256, 64L * di.sm_count), 256, 0, s>>>(
      packed, packed_row_bytes, sh, codebook != 0, reinterpret_cast<uint32_t*>(packed_out));
  NSM_CHECK_CUDA(cudaGetLastError());
  lin4_pack_scales_kernel<<<(int)std::min<int64_t>((ns + 255) / 256, 64L * di.sm_count), 256, 0, s>>>(
      scales, scale_dtype, zeros, sh, groups, scales_out, zeros_out);
  NSM_CHECK_CUDA(cudaGetLastError());
  return NSM_OK;
}

size_t nsm_linear4bit_workspace_bytes(int32_t rows, int32_t x_dtype, int32_t out_features, int32_t in_features) {
  if (!lin4_size_ok(out_features, in_features, 32) || rows <= 0 || rows > lin4_max_rows(x_dtype)) return 0;
  DeviceInfo di;
  if (current_device(&di) != NSM_OK) return 0;
  return lin4_plan(lin4_shape(out_features, in_features, 32), rows, x_dtype, di).bytes;
}

}  // extern "C"

namespace nsm {
namespace {

int lin4_run(const void* x, int32_t x_dtype, int32_t rows, int64_t x_row_stride, const nsm_linear4bit_weights* w,
             bool code16, void* out, int32_t out_dtype, int64_t out_row_stride, void* workspace,
             size_t workspace_bytes, nsm_stream_t stream) {
  auto dtype_ok = [](int d) { return d == NSM_F32 || d == NSM_F16 || d == NSM_BF16; };
  NSM_REQUIRE(w != nullptr, NSM_ERR_INVALID_ARG, "nsm_linear4bit: NULL weights");
  NSM_REQUIRE(dtype_ok(x_dtype) && dtype_ok(out_dtype) && (w->bias == nullptr || dtype_ok(w->bias_dtype)),
              NSM_ERR_INVALID_ARG, "nsm_linear4bit: bad dtype");
  NSM_REQUIRE(rows >= 0, NSM_ERR_INVALID_ARG, "nsm_linear4bit: negative rows");
  if (rows == 0) return NSM_OK;
  NSM_REQUIRE(lin4_size_ok(w->out_features, w->in_features, w->group_size), NSM_ERR_UNSUPPORTED,
              "nsm_linear4bit: in_features must be even, group_size a multiple of 32");
  NSM_REQUIRE(rows <= lin4_max_rows(x_dtype), NSM_ERR_UNSUPPORTED,
              "nsm_linear4bit: too many rows for one call (see nsm_linear4bit_max_rows)");
  NSM_REQUIRE(x && out && w->packed && w->scales && workspace, NSM_ERR_INVALID_ARG, "nsm_linear4bit: NULL pointer");
  NSM_REQUIRE(!(w->code && w->zeros), NSM_ERR_INVALID_ARG, "nsm_linear4bit: a codebook has no zero points");
  NSM_REQUIRE(rows == 1 || (x_row_stride >= w->in_features && out_row_stride >= w->out_features), NSM_ERR_INVALID_ARG,
              "nsm_linear4bit: rows overlap");
  NSM_REQUIRE(((uintptr_t)w->packed & 15) == 0 && ((uintptr_t)w->scales & 15) == 0 && ((uintptr_t)w->zeros & 15) == 0,
              NSM_ERR_INVALID_ARG, "nsm_linear4bit: packed weights, scales and zero points must be 16-byte aligned");
  const uintptr_t xa = x_dtype == NSM_F32 ? 3 : 1, oa = out_dtype == NSM_F32 ? 3 : 1;
  NSM_REQUIRE(((uintptr_t)x & xa) == 0 && ((uintptr_t)out & oa) == 0, NSM_ERR_INVALID_ARG,
              "nsm_linear4bit: x and out must be aligned to their type");
  DeviceInfo di;
  const int rc = current_device(&di);
  if (rc != NSM_OK) return rc;
  const Lin4Shape sh = lin4_shape(w->out_features, w->in_features, w->group_size);
  const Lin4Plan pl = lin4_plan(sh, rows, x_dtype, di);
  NSM_REQUIRE(((uintptr_t)workspace & 255) == 0 && workspace_bytes >= pl.bytes, NSM_ERR_WORKSPACE,
              "nsm_linear4bit: workspace misaligned or too small (nsm_linear4bit_workspace_bytes)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  __half* xh = reinterpret_cast<__half*>(ws);
  float* scale = reinterpret_cast<float*>(ws + pl.scale_off);
  float* part = reinterpret_cast<float*>(ws + pl.part_off);

  // The codebook's values keep 22 bits.  Rounded to fp16 (2^-11 of a value at most, random over
  // the columns: about 1e-4 of the output) they take half the table reads, which bound the
  // kernel: that is the caller's choice (nsm_linear4bit_code16).
  const int mode = w->code ? (code16 ? kCode : kCodeExact) : (w->zeros ? kIntZeros : kInt);
  const int cc = lin4_col_case(pl.cols);
  const bool cluster = pl.cluster > 0;
  const Lin4Fn f = cluster ? lin4_pick<true>(mode, sh.npg, cc) : lin4_pick<false>(mode, sh.npg, cc);
  NSM_CHECK_CUDA(lin4_once[cluster][mode][sh.npg / 2][cc].set(f.fn, f.smem, di.device));
  if (!pl.own_x) {
    const int slices = std::max(1, std::min(8, sh.kp / 2048));
    lin4_prep_kernel<<<dim3(slices, rows), 256, 0, s>>>(x, x_dtype, x_row_stride, sh.K, sh.kp, rows, pl.col_groups,
                                                        w->code, xh, scale);
    NSM_CHECK_CUDA(cudaGetLastError());
  }
  Lin4Params p;
  p.w = w->packed;
  p.s = w->scales;
  p.z = w->zeros;
  p.code = w->code;
  p.x = x;
  p.xh = xh;
  p.x_stride = x_row_stride;
  p.x_dtype = x_dtype;
  p.rows = rows;
  p.K = sh.K;
  p.part = part;
  p.row_tiles = sh.row_tiles;
  p.steps = sh.steps;
  p.scale_steps = sh.scale_steps;
  p.div = sh.div;
  p.cols = pl.cols;
  p.units = pl.units;
  p.ctas = pl.ctas;
  p.max_segs = pl.max_segs;
  p.wait_limit = lin4_wait_limit();
  p.cluster = pl.cluster;
  p.N = sh.N;
  p.scale = scale;
  p.bias = w->bias;
  p.bias_dt = w->bias_dtype;
  p.out = out;
  p.out_dt = out_dtype;
  p.out_stride = out_row_stride;
  if (cluster) {
    NSM_CHECK_CUDA(launch_pdl_cluster(f.fn, dim3(sh.row_blocks * pl.cluster), dim3(kL4Threads), (size_t)f.smem, s,
                                      pl.cluster, p));
    return NSM_OK;
  }
  NSM_CHECK_CUDA(launch_pdl(f.fn, dim3(pl.ctas), dim3(kL4Threads), (size_t)f.smem, s, p));
  const bool many = pl.max_segs > 4;
  const int share = many && 4LL * sh.N * rows <= 2048LL * di.sm_count ? 4 : 1;
  const int fin_rows = kL4BlockRows / share;
  NSM_CHECK_CUDA(launch_pdl(share == 4 ? lin4_finalize_kernel<4, true> : many ? lin4_finalize_kernel<1, true> : lin4_finalize_kernel<1, false>,
                            dim3((sh.N + fin_rows - 1) / fin_rows, rows), dim3(kL4BlockRows), 0, s, (const float*)part,
                            (const float*)(pl.own_x ? nullptr : scale), pl.units, pl.ctas, sh.steps, pl.max_segs, pl.cols,
                            (int)rows, sh.N, w->bias, (int)w->bias_dtype, out, (int)out_dtype, out_row_stride));
  return NSM_OK;
}

}  // namespace
}  // namespace nsm

extern "C" {

int nsm_linear4bit(const void* x, int32_t x_dtype, int32_t rows, int64_t x_row_stride,
                   const nsm_linear4bit_weights* w, void* out, int32_t out_dtype, int64_t out_row_stride,
                   void* workspace, size_t workspace_bytes, nsm_stream_t stream) {
  return lin4_run(x, x_dtype, rows, x_row_stride, w, false, out, out_dtype, out_row_stride, workspace, workspace_bytes,
                  stream);
}

int nsm_linear4bit_code16(const void* x, int32_t x_dtype, int32_t rows, int64_t x_row_stride,
                          const nsm_linear4bit_weights* w, void* out, int32_t out_dtype, int64_t out_row_stride,
                          void* workspace, size_t workspace_bytes, nsm_stream_t stream) {
  return lin4_run(x, x_dtype, rows, x_row_stride, w, true, out, out_dtype, out_row_stride, workspace, workspace_bytes,
                  stream);
}

}  // extern "C"
