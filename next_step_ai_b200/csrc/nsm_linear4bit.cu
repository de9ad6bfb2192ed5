// nsm_linear4bit.cu -- y = x W^T (+ bias) for 1..32 rows of x and a weight W
// [N, K] in 4 bits with a scale for each group of columns of a row:
//
//   y[r][n] = b[n] + sum_g s[n][g] * sum_{k in g} x[r][k] * (T[q[n][k]] - z[n][g])
//
// T is a 16-entry codebook (z = 0: NF4 and the like) or the identity (integer
// weights, z = 8 or a zero point per group).
//
// Layout (written once by nsm_linear4bit_pack): tiles of 16 rows x 128 columns,
// 1 KB each, row tile by row tile, so a warp streams contiguous memory with two
// 16-byte loads per lane and tile.  Lane (g = lane / 4, t = lane % 4) holds, of
// row g (first load) and row g + 8 (second), one 32-bit word for each of the
// tile's four 32-column blocks: columns 32j + 8t .. + 8.  A block's two
// mma.sync m16n8k16 therefore stay inside one scale group of 32 or more, and
// their B fragments are 16 contiguous bytes of x in natural order.
//
// Three launches, linked by programmatic dependent launch:
//  1. lin4_prep_kernel: per row of x a power-of-two scale that brings the
//     largest finite |x| to [2^14, 2^15) and x as fp16 (exact for fp16, and for bf16
//     down to 2^-38 of the row's largest); an fp32 x becomes two fp16 columns
//     (value and remainder, 22 bits);
//  2. lin4_kernel: one CTA of 16 warps per SM.  A unit is 256 rows (one tile per
//     warp) x 128 columns; the units, row block by row block, are cut into equal
//     contiguous runs, one per CTA, so no CTA finishes late, and the 16 warps
//     read the same piece of x at the same time (it stays in L1).  fp16 weights x
//     fp16 x on the tensor pipe with fp32 accumulation -- every product is exact
//     -- and the group's scale is applied in fp32.  Each CTA leaves one
//     fp32 partial per row block that it touched;
//  3. lin4_finalize_kernel: the partials of a row block in CTA order (the same
//     bits every time), times the scale of x, + bias, in the output's type.
#include <algorithm>
#include <mutex>

#include "nsm_common.cuh"
#include "nsm_internal.h"

namespace nsm {
namespace {

constexpr int kL4Warps = 16;
constexpr int kL4Threads = 32 * kL4Warps;
constexpr int kL4TileRows = 16;
constexpr int kL4TileCols = 128;
constexpr int kL4TileBytes = kL4TileRows * kL4TileCols / 2;
constexpr int kL4BlockRows = kL4TileRows * kL4Warps;  // rows of a unit
constexpr int kL4MaxCols = 32;                        // fp16 columns of x in one call
constexpr int kL4MaxSegs = 32;                        // CTAs that share one row block
constexpr int kL4Depth = 3;                           // tiles in flight per warp

// Kinds of weights: codebook rounded to fp16; codebook as fp16 value +
// remainder (22 bits, two table reads and two MMAs: outputs in fp32); integers
// with the zero point 8; integers with a zero point per group.
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
  s.row_blocks = (s.row_tiles + kL4Warps - 1) / kL4Warps;
  s.kp = s.steps * kL4TileCols;
  s.npg = group % 128 == 0 ? 1 : (group % 64 == 0 ? 2 : 4);
  s.div = s.npg == 1 ? group / 128 : 1;
  s.scale_steps = (s.steps + s.div - 1) / s.div;
  return s;
}

// ---- packing ------------------------------------------------------------------
// One thread per 32-bit word of the tiled weight.  Codebook words keep the byte
// order (byte i = columns 2i, 2i+1: an index into the byte table).  Integer
// words put columns c and c + 1 of a pair 16 bits apart, so one mask leaves a
// half2: nibbles 0..7 = columns 0, 2, 4, 6, 1, 3, 5, 7.
__global__ void lin4_pack_kernel(const uint8_t* __restrict__ src, int64_t row_bytes, Lin4Shape sh, int is_code,
                                 uint32_t* __restrict__ dst) {
  const int64_t words = (int64_t)sh.row_tiles * sh.steps * (kL4TileBytes / 4);
  const int kb = sh.K / 2;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x) {
    const int in_tile = (int)(i & 255);  // [2 halves][32 lanes][4 words]
    const int64_t tile = i >> 8;
    const int j = in_tile & 3, lane = (in_tile >> 2) & 31, h = in_tile >> 7;
    const int64_t row = tile / sh.steps * kL4TileRows + (lane >> 2) + 8 * h;
    const int col_byte = (int)(tile % sh.steps) * (kL4TileCols / 2) + 16 * j + 4 * (lane & 3);
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

// Scales (and zero points) as [row tile][scale step][8 g][npg][2 rows g, g + 8];
// rows and columns past the end get scale 0 and zero point 0.
__global__ void lin4_pack_scales_kernel(const void* __restrict__ scales, int dt, const uint8_t* __restrict__ zeros,
                                        Lin4Shape sh, int groups, float* __restrict__ ds, uint8_t* __restrict__ dz) {
  const int per = 16 * sh.npg;
  const int64_t n = (int64_t)sh.row_tiles * sh.scale_steps * per;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int e = (int)(i % per);
    const int64_t ts = i / per;
    const int h = e & 1, pg = (e >> 1) % sh.npg, g = (e >> 1) / sh.npg;
    const int64_t row = ts / sh.scale_steps * kL4TileRows + g + 8 * h;
    const int64_t col = (ts % sh.scale_steps) * sh.div * kL4TileCols + pg * (kL4TileCols / sh.npg);
    const int64_t grp = col / sh.group;
    const bool in = row < sh.N && grp < groups && col < sh.K;
    ds[i] = in ? load_as_f32(scales, dt, row * groups + grp) : 0.f;
    if (dz) dz[i] = in ? zeros[row * groups + grp] : 0;
  }
}

// ---- activations ----------------------------------------------------------------
// Power of two that brings the largest |code| to [64, 128): the remainders of the
// exact codebook then stay normal fp16 numbers.
__device__ __forceinline__ float code_scale(const float* code) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float a = fabsf(__ldg(code + i));
    if (a <= 3.4e38f) m = fmaxf(m, a);
  }
  if (!(m > 0.f)) return 1.f;
  return ldexpf(1.f, max(-120, min(120, 6 - ilogbf(m))));
}

__global__ void __launch_bounds__(1024) lin4_prep_kernel(const void* x, int dt, int64_t stride, int K, int kp, int rows,
                                                         int split, const float* code, __half* xh, float* scale) {
  pdl_trigger();
  __shared__ float wmax[32];
  const int r = blockIdx.x;
  const int64_t base = (int64_t)r * stride;
  float s = 1.f;
  if (dt != NSM_F16) {
    float m = 0.f;
    for (int k = threadIdx.x; k < K; k += blockDim.x) {
      const float a = fabsf(load_as_f32(x, dt, base + k));
      if (a <= 3.4028234e38f) m = fmaxf(m, a);  // infinities and NaN stay what they are
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = m;
    __syncthreads();
    m = warp_max(wmax[threadIdx.x & 31]);
    if (m > 0.f) s = ldexpf(1.f, max(-120, min(120, ilogbf(m) - 14)));
  }
  const float inv = 1.f / s;  // a power of two: exact
  __half* hi = xh + (int64_t)r * kp;
  __half* lo = xh + (int64_t)(rows + r) * kp;
  for (int k = threadIdx.x; k < kp; k += blockDim.x) {
    const float v = k < K ? load_as_f32(x, dt, base + k) * inv : 0.f;
    const __half h = __float2half_rn(v);
    hi[k] = h;
    if (split) {
      const float rem = v - __half2float(h);
      lo[k] = __float2half_rn(fabsf(rem) <= 3.4028234e38f ? rem : 0.f);
    }
  }
  if (threadIdx.x == 0) scale[r] = code ? s / code_scale(code) : s;
}

// ---- products -------------------------------------------------------------------
struct Lin4Params {
  const uint8_t* w;
  const float* s;
  const uint8_t* z;
  const float* code;
  const __half* xh;
  float* part;  // [row block][segment][column of x][256]
  int row_tiles, steps, scale_steps, div, kp, cols;
  int units, ctas, max_segs;
};

// x written by the kernel before: volatile, so it is never moved over the wait
__device__ __forceinline__ uint4 ld_x(const void* p) {
  uint4 r;
  asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
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
template <int kPair>
__device__ __forceinline__ uint32_t int_pair(uint32_t w, uint32_t za, uint32_t zb) {
  const uint32_t v = kPair >= 2 ? w >> 8 : w;
  if (kPair % 2 == 0) return hsub2_u32((v & 0x000f000fu) | 0x64006400u, za);
  return hfma2_u32((v & 0x00f000f0u) | 0x64006400u, 0x2c002c00u, zb);
}

template <int NPG>
struct Lin4Stage {
  uint4 a, b;
  float s[2 * NPG];
  uint32_t z[(NPG + 1) / 2];  // zero points, two bytes per granule
};

template <int MODE, int NPG, int NT>
__global__ void __launch_bounds__(kL4Threads, 1) lin4_kernel(Lin4Params p) {
  extern __shared__ __align__(1024) uint32_t l4_lut[];
  constexpr bool kIsCode = MODE == kCode || MODE == kCodeExact;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t lanebase = (uint32_t)lane * 4u;
  const int u0 = stream_begin(p.units, p.ctas, blockIdx.x), u1 = stream_begin(p.units, p.ctas, blockIdx.x + 1);
  pdl_trigger();

  Lin4Stage<NPG> st[kL4Depth];
  auto load = [&](Lin4Stage<NPG>& q, int rb, int step) {
    const int rt = rb * kL4Warps + warp;
    if (rt >= p.row_tiles) return;
    const uint8_t* w = p.w + ((int64_t)rt * p.steps + step) * kL4TileBytes + lane * 16;
    q.a = ldg_stream_u4(w);
    q.b = ldg_stream_u4(w + 512);
    const int ss = (NPG == 1 && p.div > 1) ? step / p.div : step;
    const int64_t e = (((int64_t)rt * p.scale_steps + ss) * 8 + g) * (2 * NPG);
    if constexpr (NPG == 1) {
      const float2 v = __ldg(reinterpret_cast<const float2*>(p.s + e));
      q.s[0] = v.x;
      q.s[1] = v.y;
      if (MODE == kIntZeros) q.z[0] = __ldg(reinterpret_cast<const unsigned short*>(p.z + e));
    } else {
#pragma unroll
      for (int i = 0; i < NPG / 2; ++i) {
        const float4 v = ldg_f4(p.s + e + 4 * i);
        q.s[4 * i] = v.x;
        q.s[4 * i + 1] = v.y;
        q.s[4 * i + 2] = v.z;
        q.s[4 * i + 3] = v.w;
        if (MODE == kIntZeros) q.z[i] = __ldg(reinterpret_cast<const uint32_t*>(p.z + e + 4 * i));
      }
    }
  };
  int prb = u0 / p.steps, pstep = u0 - prb * p.steps;  // the next unit to load
  auto advance = [&](int& rb, int& step) {
    if (++step == p.steps) {
      step = 0;
      ++rb;
    }
  };
  int rb = prb, step = pstep;  // the next unit to multiply
#pragma unroll
  for (int d = 0; d < kL4Depth; ++d) {
    if (u0 + d < u1) {
      load(st[d], prb, pstep);
      advance(prb, pstep);
    }
  }

  if constexpr (kIsCode) {  // byte -> half2 table, one copy per lane (conflict-free); the second holds the remainders
    const float cs = code_scale(p.code);
    uint4* lut4 = reinterpret_cast<uint4*>(l4_lut);
    for (int i = threadIdx.x; i < 256 * 16; i += kL4Threads) {
      const int e = i >> 4;
      if (MODE == kCode && (i & 8)) continue;
      const float c0 = __ldg(p.code + (e >> 4)) * cs, c1 = __ldg(p.code + (e & 15)) * cs;
      __half h0 = __float2half_rn(c0), h1 = __float2half_rn(c1);
      if (i & 8) {
        h0 = __float2half_rn(c0 - __half2float(h0));
        h1 = __float2half_rn(c1 - __half2float(h1));
      }
      const uint32_t v = (uint32_t)__half_as_ushort(h0) | ((uint32_t)__half_as_ushort(h1) << 16);
      lut4[i] = make_uint4(v, v, v, v);
    }
    __syncthreads();
  }
  pdl_wait();

  const __half* xlane = p.xh + (int64_t)g * p.kp + 8 * t;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  auto flush = [&](int at) {  // this warp's partial of row block `at`
    if (at * kL4Warps + warp < p.row_tiles) {
      const int seg = (int)blockIdx.x - stream_owner(p.units, p.ctas, at * p.steps);
      float* dst = p.part + ((int64_t)(at * p.max_segs + seg) * p.cols) * kL4BlockRows + warp * kL4TileRows + g;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = 8 * n + 2 * t + (i & 1);
          if (c < p.cols) dst[(int64_t)c * kL4BlockRows + (i >> 1) * 8] = acc[n][i];
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  };

  auto multiply = [&](const Lin4Stage<NPG>& q, int at, int stp) {
    if (at * kL4Warps + warp >= p.row_tiles) return;
    float d[NT][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      constexpr int kPer = 4 / NPG;  // 32-column blocks per scale
      if (j % kPer == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[n][i] = 0.f;
      }
      uint4 xf[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        xf[n] = make_uint4(0, 0, 0, 0);
        if (8 * n + g < p.cols) xf[n] = ld_x(xlane + (int64_t)(8 * n) * p.kp + stp * kL4TileCols + 32 * j);
      }
      const uint32_t wa = j == 0 ? q.a.x : j == 1 ? q.a.y : j == 2 ? q.a.z : q.a.w;
      const uint32_t wb = j == 0 ? q.b.x : j == 1 ? q.b.y : j == 2 ? q.b.z : q.b.w;
      uint32_t f[8];  // A fragments of the block's two MMAs
      if constexpr (kIsCode) {
#pragma unroll
        for (int tab = 0; tab < (MODE == kCodeExact ? 2 : 1); ++tab) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            f[4 * (b >> 1) + 2 * (b & 1)] = lut_lookup_rt(l4_lut, wa, lanebase, b, tab);
            f[4 * (b >> 1) + 2 * (b & 1) + 1] = lut_lookup_rt(l4_lut, wb, lanebase, b, tab);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(d[n], f[0], f[1], f[2], f[3], xf[n].x, xf[n].y);
            mma_16816(d[n], f[4], f[5], f[6], f[7], xf[n].z, xf[n].w);
          }
        }
      } else {
        uint32_t za = 0x64086408u, zb = 0xd480d480u;  // 1032, -72
        uint32_t za8 = za, zb8 = zb;
        if constexpr (MODE == kIntZeros) {
          const int gr = j / kPer;
          const uint32_t zz = q.z[gr / 2] >> (16 * (gr % 2));
          const uint32_t z0 = zz & 255u, z1 = (zz >> 8) & 255u;
          za = (0x6400u | z0) * 0x10001u;
          za8 = (0x6400u | z1) * 0x10001u;
          zb = hsub2_u32(0x63806380u, za);   // 960 - (1024 + z)
          zb8 = hsub2_u32(0x63806380u, za8);
        }
        f[0] = int_pair<0>(wa, za, zb);
        f[1] = int_pair<0>(wb, za8, zb8);
        f[2] = int_pair<1>(wa, za, zb);
        f[3] = int_pair<1>(wb, za8, zb8);
        f[4] = int_pair<2>(wa, za, zb);
        f[5] = int_pair<2>(wb, za8, zb8);
        f[6] = int_pair<3>(wa, za, zb);
        f[7] = int_pair<3>(wb, za8, zb8);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_16816(d[n], f[0], f[1], f[2], f[3], xf[n].x, xf[n].y);
          mma_16816(d[n], f[4], f[5], f[6], f[7], xf[n].z, xf[n].w);
        }
      }
      if (j % kPer == kPer - 1) {
        const float s0 = q.s[2 * (j / kPer)], s1 = q.s[2 * (j / kPer) + 1];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          acc[n][0] = fmaf(s0, d[n][0], acc[n][0]);
          acc[n][1] = fmaf(s0, d[n][1], acc[n][1]);
          acc[n][2] = fmaf(s1, d[n][2], acc[n][2]);
          acc[n][3] = fmaf(s1, d[n][3], acc[n][3]);
        }
      }
    }
  };

  for (int u = u0; u < u1; u += kL4Depth) {
#pragma unroll
    for (int d = 0; d < kL4Depth; ++d) {
      if (u + d < u1) {
        multiply(st[d], rb, step);
        if (u + d + kL4Depth < u1) {
          load(st[d], prb, pstep);
          advance(prb, pstep);
        }
        const int done = rb;
        advance(rb, step);
        if (rb != done || u + d + 1 == u1) flush(done);
      }
    }
  }
}

__global__ void __launch_bounds__(kL4BlockRows) lin4_finalize_kernel(const float* part, const float* scale, int units,
                                                                     int ctas, int steps, int max_segs, int cols,
                                                                     int rows, int N, const void* bias, int bias_dt,
                                                                     void* out, int out_dt, int64_t out_stride) {
  pdl_wait();
  const int rb = blockIdx.x, r = blockIdx.y, n = rb * kL4BlockRows + threadIdx.x;
  if (n >= N) return;
  const int first = stream_owner(units, ctas, rb * steps);
  const int segs = stream_owner(units, ctas, (rb + 1) * steps - 1) - first + 1;
  const float* src = part + ((int64_t)rb * max_segs * cols + r) * kL4BlockRows + threadIdx.x;
  float v = 0.f;
#pragma unroll 4
  for (int k = 0; k < segs; ++k) {
    const float* q = src + (int64_t)k * cols * kL4BlockRows;
    float e = __ldcg(q);
    if (cols > rows) e += __ldcg(q + (int64_t)rows * kL4BlockRows);  // the remainders of an fp32 x
    v += e;
  }
  v *= __ldcg(scale + r);
  if (bias) v += load_as_f32(bias, bias_dt, n);
  store_from_f32(out, out_dt, (int64_t)r * out_stride + n, v);
}

struct Lin4Plan {
  int cols = 0, units = 0, ctas = 0, max_segs = 0;
  size_t scale_off = 0, part_off = 0, bytes = 0;
};

Lin4Plan lin4_plan(const Lin4Shape& sh, int rows, int x_dtype, int sm_count) {
  Lin4Plan pl;
  pl.cols = x_dtype == NSM_F32 ? 2 * rows : rows;
  pl.units = sh.row_blocks * sh.steps;
  pl.ctas = std::max(1, std::min({sm_count, pl.units, sh.row_blocks * (kL4MaxSegs - 2)}));
  const int least = pl.units / pl.ctas;  // units of the shortest run
  pl.max_segs = (sh.steps - 1 + least - 1) / least + 1;
  pl.scale_off = align_up((size_t)pl.cols * sh.kp * 2, 256);
  pl.part_off = pl.scale_off + align_up((size_t)rows * 4, 256);
  pl.bytes = pl.part_off + (size_t)sh.row_blocks * pl.max_segs * pl.cols * kL4BlockRows * 4;
  return pl;
}

bool lin4_size_ok(int N, int K, int group) {
  return N > 0 && K > 0 && K % 2 == 0 && group > 0 && group % 32 == 0 && N <= (1 << 24) && K <= (1 << 20) &&
         (int64_t)((N + 255) / 256) * ((K + 127) / 128) < (1 << 30);
}

int lin4_max_rows(int x_dtype) { return x_dtype == NSM_F32 ? kL4MaxCols / 2 : kL4MaxCols; }

using Lin4Fn = void (*)(Lin4Params);

template <int MODE, int NPG>
Lin4Fn lin4_pick_nt(int cols) {
  return cols <= 8 ? lin4_kernel<MODE, NPG, 1> : cols <= 16 ? lin4_kernel<MODE, NPG, 2> : lin4_kernel<MODE, NPG, 4>;
}
template <int MODE>
Lin4Fn lin4_pick_npg(int npg, int cols) {
  return npg == 1 ? lin4_pick_nt<MODE, 1>(cols) : npg == 2 ? lin4_pick_nt<MODE, 2>(cols) : lin4_pick_nt<MODE, 4>(cols);
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
  return (size_t)sh.row_tiles * sh.scale_steps * 16 * sh.npg;
}

int nsm_linear4bit_max_rows(int32_t x_dtype) { return lin4_max_rows(x_dtype); }

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
  const int64_t ns = (int64_t)sh.row_tiles * sh.scale_steps * 16 * sh.npg;
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
  return lin4_plan(lin4_shape(out_features, in_features, 32), rows, x_dtype, di.sm_count).bytes;
}

int nsm_linear4bit(const void* x, int32_t x_dtype, int32_t rows, int64_t x_row_stride,
                   const nsm_linear4bit_weights* w, void* out, int32_t out_dtype, int64_t out_row_stride,
                   void* workspace, size_t workspace_bytes, nsm_stream_t stream) {
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
  const Lin4Plan pl = lin4_plan(sh, rows, x_dtype, di.sm_count);
  NSM_REQUIRE(((uintptr_t)workspace & 255) == 0 && workspace_bytes >= pl.bytes, NSM_ERR_WORKSPACE,
              "nsm_linear4bit: workspace misaligned or too small (nsm_linear4bit_workspace_bytes)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  __half* xh = reinterpret_cast<__half*>(ws);
  float* scale = reinterpret_cast<float*>(ws + pl.scale_off);
  float* part = reinterpret_cast<float*>(ws + pl.part_off);

  // fp32 outputs keep the codebook's values to 22 bits; fp16 and bf16 ones round
  // it to fp16 (2^-12 of a value at most, random over the columns: about 1e-4 of the output,
  // half an fp16 rounding), which halves the table reads that bound the kernel
  const int mode = w->code ? (out_dtype == NSM_F32 ? kCodeExact : kCode) : (w->zeros ? kIntZeros : kInt);
  Lin4Fn fn = mode == kCode        ? lin4_pick_npg<kCode>(sh.npg, pl.cols)
              : mode == kCodeExact ? lin4_pick_npg<kCodeExact>(sh.npg, pl.cols)
              : mode == kInt       ? lin4_pick_npg<kInt>(sh.npg, pl.cols)
                                   : lin4_pick_npg<kIntZeros>(sh.npg, pl.cols);
  const size_t smem = w->code ? (size_t)kLutBytes : 0;
  static SmemOnce once[2][3][3];
  if (smem > 0)
    NSM_CHECK_CUDA(once[mode][sh.npg / 2][pl.cols <= 8 ? 0 : pl.cols <= 16 ? 1 : 2].set(fn, (int)smem, di.device));
  lin4_prep_kernel<<<rows, 1024, 0, s>>>(x, x_dtype, x_row_stride, sh.K, sh.kp, rows, x_dtype == NSM_F32, w->code, xh,
                                         scale);
  NSM_CHECK_CUDA(cudaGetLastError());
  Lin4Params p;
  p.w = w->packed;
  p.s = w->scales;
  p.z = w->zeros;
  p.code = w->code;
  p.xh = xh;
  p.part = part;
  p.row_tiles = sh.row_tiles;
  p.steps = sh.steps;
  p.scale_steps = sh.scale_steps;
  p.div = sh.div;
  p.kp = sh.kp;
  p.cols = pl.cols;
  p.units = pl.units;
  p.ctas = pl.ctas;
  p.max_segs = pl.max_segs;
  NSM_CHECK_CUDA(launch_pdl(fn, dim3(pl.ctas), dim3(kL4Threads), smem, s, p));
  NSM_CHECK_CUDA(launch_pdl(lin4_finalize_kernel, dim3(sh.row_blocks, rows), dim3(kL4BlockRows), 0, s,
                            (const float*)part, (const float*)scale, pl.units, pl.ctas, sh.steps, pl.max_segs, pl.cols,
                            (int)rows, sh.N, w->bias, (int)w->bias_dtype, out, (int)out_dtype, out_row_stride));
  return NSM_OK;
}

}  // extern "C"
