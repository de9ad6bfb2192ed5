// nsm_beam.cu -- beam search after the logits: the best continuations over
// beams and vocabulary, and the reordering of the beams' states.
//
// Selection.  A candidate (beam w, token v) of a batch item has the score
//
//   score[w] + logit[w][v] - logsumexp(logit[w][:])
//
// and the k best are wanted, equal scores in the order of w, then v.  Inside one
// beam the order of the scores is the order of the logits, so the logits are
// read once (beam_scan_kernel): a CTA takes a contiguous piece of a row, keeps
// a running maximum and sum of exponentials per thread (fp32), and collects its
// piece's k best as 64-bit keys (value in ordered bits, then the complement of
// the index: every key differs, so "the k best" is one set whatever the order
// in which threads find them).  A value enters the list only at or above a
// threshold, the smallest of 16 to 64 group maxima so far (at least k values are that
// large); what the last threshold leaves is ranked by counting.
// beam_merge_kernel, one CTA per batch item, joins the pieces: the sums in 64
// bits, the scores of at most W * pieces * k + W candidates in 64 bits, and the
// k best of them.
//
// Reordering.  beam_reorder_kernel moves the states in place: a thread owns
// one 1- to 16-byte column of all beams of a batch item, loads the beams that
// others go on with, then stores them where they moved.  A beam that stays
// is not written, and one that nobody else takes is not read.
#include <algorithm>
#include <climits>

#include "nsm_common.cuh"
#include "nsm_internal.h"

namespace nsm {
namespace {

using u64 = unsigned long long;

constexpr int kBsThreads = 512;
constexpr int kBsWarps = kBsThreads / 32;
constexpr int kBsPer = 16;                       // values per thread and tile
constexpr int kBsTile = kBsThreads * kBsPer;
constexpr int kBsCap = 1024;                     // keys of the candidate list
constexpr int kBsMaxK = 64;
constexpr int kBsMaxBeams = 32;
constexpr int kBsMaxMerge = 12288;               // candidates of one merge (12 bytes each in shared memory)
constexpr float kFltMax = 3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f;

// Larger float <-> larger unsigned.
__device__ __forceinline__ uint32_t order_f32(float v) {
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unorder_f32(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 order_f64(double v) {
  const u64 b = (u64)__double_as_longlong(v);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double unorder_f64(u64 o) {
  return __longlong_as_double((long long)(o >> 63 ? o ^ (1ull << 63) : ~o));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// NaN counts as -infinity, +infinity as the largest finite value: tokens at
// +infinity then share the whole probability.
__device__ __forceinline__ float clean(float v) { return fminf(fmaxf(v, -INFINITY), kFltMax); }
// 0 = no candidate (-infinity); -0 counts as 0
__device__ __forceinline__ u64 make_key(float v, uint32_t idx) {
  return v == -INFINITY ? 0ull : ((u64)order_f32(v + 0.f) << 32) | (0xffffffffu - idx);
}

struct ScanParams {
  const void* logits;
  int64_t batch_stride, beam_stride;  // elements
  const float* scores;                // [B][W]
  const uint8_t* finished;            // [B][W] or NULL
  int W, V, k, pieces, piece;         // piece = elements per CTA, a multiple of the tile
  float* piece_max;                   // [rows][pieces]
  float* piece_sum;
  int* piece_count;
  u64* piece_keys;                    // [rows][pieces][k]
};

// The 16 values of a thread as they are loaded: 16-byte pieces, or one value each.
template <typename T, bool kVec>
struct RawTile {
  uint32_t r[kVec ? 4 * (int)sizeof(T) : kBsPer];
};
// Position in the tile of value i of a thread.  A full tile with kVec: runs of 16
// bytes, so that 16-byte loads of neighbouring lanes touch neighbouring memory; otherwise
// one value per lane, so that a short tile reaches all threads.  The mapping is the same
// for every row of a call: equal rows give equal sums, bit for bit.
template <typename T, bool kVec>
__device__ __forceinline__ int tile_pos(int i, bool full) {
  constexpr int n = 16 / sizeof(T);
  if (kVec && full) return (i / n) * (kBsThreads * n) + threadIdx.x * n + i % n;
  return i * kBsThreads + threadIdx.x;
}

template <typename T>
__device__ __forceinline__ uint32_t raw_bits(T v);
template <>
__device__ __forceinline__ uint32_t raw_bits<float>(float v) { return __float_as_uint(v); }
template <>
__device__ __forceinline__ uint32_t raw_bits<__half>(__half v) { return __half_as_ushort(v); }
template <>
__device__ __forceinline__ uint32_t raw_bits<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

template <typename T>
constexpr uint32_t kMinusInf = sizeof(T) == 4 ? 0xff800000u : 0xff80u;  // fp32, bf16
template <>
constexpr uint32_t kMinusInf<__half> = 0xfc00u;

template <typename T, bool kVec>
__device__ __forceinline__ void load_tile(const T* row, int64_t at, int left, RawTile<T, kVec>& q) {
  if constexpr (kVec) {
    if (left >= kBsTile) {
      const uint4* src = reinterpret_cast<const uint4*>(row + at) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) {
        const uint4 u = ldg_stream_u4(src + i * kBsThreads);
        q.r[4 * i] = u.x;
        q.r[4 * i + 1] = u.y;
        q.r[4 * i + 2] = u.z;
        q.r[4 * i + 3] = u.w;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kBsPer; ++i) {
    const int pos = tile_pos<T, kVec>(i, false);
    const uint32_t b = pos < left ? raw_bits<T>(row[at + pos]) : kMinusInf<T>;
    if constexpr (kVec && sizeof(T) == 2) {
      q.r[i / 2] = i % 2 ? q.r[i / 2] | b << 16 : b;
    } else {
      q.r[i] = b;
    }
  }
}

template <typename T, bool kVec>
__device__ __forceinline__ void unpack_tile(const RawTile<T, kVec>& q, float* v) {
#pragma unroll
  for (int i = 0; i < kBsPer; ++i) {
    if constexpr (sizeof(T) == 4) {
      v[i] = __uint_as_float(q.r[i]);
    } else {
      const uint32_t h = kVec ? (i % 2 ? q.r[i / 2] >> 16 : q.r[i / 2] & 0xffffu) : q.r[i];
      v[i] = to_f32<T>(*reinterpret_cast<const T*>(&h));
    }
  }
}

struct ScanShared {
  u64 list[kBsCap];
  uint32_t group[64];     // running maxima of the groups, in ordered bits
  float wmax[kBsWarps], wsum[kBsWarps];
  int wcnt[kBsWarps];
  int count, kept;
};

__device__ __forceinline__ int block_sum(int v, ScanShared& sh) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.wcnt[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < kBsWarps; ++w) s += sh.wcnt[w];
  return s;
}

// 16, 32 or 64 groups of threads, at least k of them.  If every group has a value >= x,
// at least k values are >= x: the smallest of the groups' maxima is a threshold.
__device__ __forceinline__ int group_count(int k) { return k <= 16 ? 16 : k <= 32 ? 32 : 64; }
__device__ __forceinline__ void st_relaxed(uint32_t* p, uint32_t v) {
  asm volatile("st.relaxed.cta.shared.u32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_relaxed(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.relaxed.cta.shared.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
__device__ __forceinline__ void put_group_max(uint32_t v, int groups, uint32_t* group) {
  if (groups == 16) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) st_relaxed(group + (threadIdx.x >> 5), v);
  } else {
    const int span = kBsThreads / groups;
    for (int o = span / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (threadIdx.x % span == 0) st_relaxed(group + threadIdx.x / span, v);
  }
}
__device__ __forceinline__ uint32_t min_group_max(int groups, const uint32_t* group) {
  const int lane = threadIdx.x & 31;
  uint32_t v = ld_relaxed(group + (lane & (groups - 1)));
  if (groups == 64) v = min(v, ld_relaxed(group + lane + 32));
  return __reduce_min_sync(0xffffffffu, v);
}

// The k best keys of a piece whose list ran over (it takes very many equal
// values): tile by tile, a search of the k-th largest key bit by bit over the list so far and
// the tile.  The values are read again, so that the scan keeps no registers for
// this.  Leaves the keys in sh.list and their number in sh.kept.
template <typename T>
__device__ __noinline__ void list_again(ScanShared& sh, int k, const T* row, int64_t begin, int64_t end) {
  __syncthreads();
  if (threadIdx.x == 0) sh.kept = 0;
  __syncthreads();
  uint32_t enter = 1;  // once k keys are listed, an equal value at a later index loses
  for (int64_t at = begin; at < end; at += kBsTile) {
    const int n = sh.kept;  // at most k
    const u64 mine = (int)threadIdx.x < n ? sh.list[threadIdx.x] : 0ull;
    u64 tile[kBsPer];
    bool any = false;
#pragma unroll
    for (int i = 0; i < kBsPer; ++i) {
      const int64_t pos = at + i * kBsThreads + threadIdx.x;
      tile[i] = pos < end ? make_key(clean(to_f32<T>(row[pos])), (uint32_t)pos) : 0ull;
      if ((uint32_t)(tile[i] >> 32) < enter) tile[i] = 0;
      any |= tile[i] != 0;
    }
    if (!__syncthreads_or(any)) continue;
    u64 cut = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const u64 tr = cut | (1ull << bit);
      int c = mine >= tr;
#pragma unroll
      for (int i = 0; i < kBsPer; ++i) c += tile[i] >= tr;
      c = block_sum(c, sh);
      if (c >= k) cut = tr;
      if (c == k) break;
    }
    // the keys are unique, so exactly k are >= cut, or all are (cut stays 0)
    if (threadIdx.x == 0) sh.kept = 0;
    __syncthreads();
    auto keep = [&](u64 key) {
      if (key != 0 && key >= cut) sh.list[atomicAdd(&sh.kept, 1)] = key;
    };
    keep(mine);
#pragma unroll
    for (int i = 0; i < kBsPer; ++i) keep(tile[i]);
    __syncthreads();
    if (cut) enter = (uint32_t)(cut >> 32) + 1;
  }
  __syncthreads();
}

// Rank of each of the n keys among all: eight threads count for one key.
__device__ __forceinline__ int count_above(const u64* list, int n, u64 key, int part) {
  int rank = 0;
#pragma unroll 4
  for (int j = part; j < n; j += 8) rank += list[j] > key;
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  rank += __shfl_xor_sync(0xffffffffu, rank, 2);
  rank += __shfl_xor_sync(0xffffffffu, rank, 4);
  return rank;
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kBsThreads, 2) beam_scan_kernel(ScanParams p) {
  __shared__ ScanShared sh;
  pdl_trigger();
  const int row = blockIdx.x / p.pieces, pc = blockIdx.x - row * p.pieces;
  const int b = row / p.W, w = row - b * p.W;
  const int64_t slot = (int64_t)row * p.pieces + pc;
  // a beam that is out (no score above -infinity) or finished is not read
  if (!(p.scores[row] > -INFINITY) || (p.finished && p.finished[row])) {
    if (threadIdx.x == 0) {
      p.piece_max[slot] = -INFINITY;
      p.piece_sum[slot] = 0.f;
      p.piece_count[slot] = 0;
    }
    return;
  }
  const T* src = reinterpret_cast<const T*>(p.logits) + b * p.batch_stride + w * p.beam_stride;
  const int64_t begin = (int64_t)pc * p.piece, end = min((int64_t)p.V, begin + p.piece);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = group_count(p.k);
  if (threadIdx.x == 0) sh.count = sh.kept = 0;

  float m = -INFINITY, s = 0.f;
  bool over = false;
  RawTile<T, kVec> next;
  load_tile<T, kVec>(src, begin, (int)min((int64_t)kBsTile, end - begin), next);
  for (int64_t at = begin; at < end; at += kBsTile) {
    float v[kBsPer];
    unpack_tile<T, kVec>(next, v);
    if (at + kBsTile < end)
      load_tile<T, kVec>(src, at + kBsTile, (int)min((int64_t)kBsTile, end - at - kBsTile), next);
    // fmaxf passes over NaN, so a tile with NaN or +infinity shows in its sum (NaN)
    // or its maximum; such a tile is cleaned and summed again
    float tm;
    for (int again = 0;; ++again) {
      tm = v[0];
#pragma unroll
      for (int i = 1; i < kBsPer; ++i) tm = fmaxf(tm, v[i]);
      if (!(tm > -INFINITY)) break;  // nothing but -infinity (and NaN)
      const float nm = fmaxf(m, tm);
      float e0 = 0.f, e1 = 0.f;
#pragma unroll
      for (int i = 0; i < kBsPer; i += 2) {
        e0 += exp2_fast((v[i] - nm) * kLog2e);
        e1 += exp2_fast((v[i + 1] - nm) * kLog2e);
      }
      const float e = e0 + e1;
      if (again || (tm <= kFltMax && e == e)) {
        s = s * exp2_fast((m - nm) * kLog2e) + e;  // m = -infinity: s is 0
        m = nm;
        break;
      }
#pragma unroll
      for (int i = 0; i < kBsPer; ++i) v[i] = clean(v[i]);
    }
    // The threshold of the running maxima.  All groups have to be in it once; after
    // that a maximum that is not up to date is only a lower threshold.
    put_group_max(m > -INFINITY ? order_f32(m + 0.f) : 0u, groups, sh.group);
    if (at == begin) __syncthreads();
    const uint32_t cut = min_group_max(groups, sh.group);
    const float thr = cut ? unorder_f32(cut) : -kFltMax;
    if (tm >= thr) {
      const bool full = end - at >= kBsTile;
#pragma unroll
      for (int i = 0; i < kBsPer; ++i) {
        if (v[i] >= thr) {
          const int e = atomicAdd(&sh.count, 1);
          if (e < kBsCap)
            sh.list[e] = make_key(v[i], (uint32_t)(at + tile_pos<T, kVec>(i, full)));
          else
            over = true;
        }
      }
    }
  }

  // the piece's maximum and sum; of the list, what the last threshold leaves
  const float wm = warp_max(m);
  if (lane == 0) sh.wmax[warp] = wm;
  over = __syncthreads_or(over);
  float pm = sh.wmax[0];
#pragma unroll
  for (int i = 1; i < kBsWarps; ++i) pm = fmaxf(pm, sh.wmax[i]);
  const float ws = warp_sum(m > -INFINITY ? s * exp2_fast((m - pm) * kLog2e) : 0.f);
  if (lane == 0) sh.wsum[warp] = ws;
  if (over) {
    list_again<T>(sh, p.k, src, begin, end);
  } else {
    u64 mine[kBsCap / kBsThreads];
    const int listed = sh.count;
    const uint32_t cut = min_group_max(groups, sh.group);
#pragma unroll
    for (int i = 0; i < kBsCap / kBsThreads; ++i) {
      const int e = i * kBsThreads + threadIdx.x;
      mine[i] = e < listed ? sh.list[e] : 0ull;
      if ((uint32_t)(mine[i] >> 32) < cut) mine[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBsCap / kBsThreads; ++i)
      if (mine[i]) sh.list[atomicAdd(&sh.kept, 1)] = mine[i];
    __syncthreads();
  }
  const int n = sh.kept;
  if (threadIdx.x == 0) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kBsWarps; ++i) t += sh.wsum[i];
    p.piece_max[slot] = pm;
    p.piece_sum[slot] = t;
    p.piece_count[slot] = min(n, p.k);
  }
  for (int i0 = 0; i0 < n; i0 += kBsThreads / 8) {  // uniform: the shuffles need whole warps
    const int i = i0 + (threadIdx.x >> 3);
    const u64 key = i < n ? sh.list[i] : 0ull;
    const int rank = count_above(sh.list, n, key, threadIdx.x & 7);
    if (i < n && rank < p.k && (threadIdx.x & 7) == 0) p.piece_keys[slot * p.k + rank] = key;
  }
}

struct MergeParams {
  const float* scores;
  const uint8_t* finished;
  int W, V, k, pieces, pad;
  const float* piece_max;
  const float* piece_sum;
  const int* piece_count;
  const u64* piece_keys;
  float* out_scores;  // [B][k]
  int64_t* out_tokens;
  int64_t* out_parents;
};

__global__ void __launch_bounds__(kBsThreads) beam_merge_kernel(MergeParams p) {
  extern __shared__ __align__(16) unsigned char bm_smem[];
  __shared__ ScanShared sh;
  __shared__ u64 at_flat[kBsCap];  // the flat indices of sh.list's candidates
  __shared__ double lse[kBsMaxBeams];
  const int per = p.pieces * p.k, M = p.W * per + p.W;
  u64* key = reinterpret_cast<u64*>(bm_smem);            // [M] scores in ordered bits, 0 = none
  uint32_t* tok = reinterpret_cast<uint32_t*>(key + M);  // [M]
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) sh.count = 0;
  pdl_wait();
  const int64_t lists = (int64_t)b * p.W * p.pieces;
  // a candidate's key and token, as the scan left them; the first ones are on their way while
  // the sums are joined
  auto fetch = [&](int i) -> u64 {
    if (i >= p.W * per) return 0ull;
    const int list = i / p.k, e = i - list * p.k;
    const int have = __ldcg(p.piece_count + lists + list);
    const u64 x = __ldcg(p.piece_keys + (lists + list) * p.k + e);  // (stale beyond the count)
    return e < have ? x : 0ull;
  };
  u64 first = fetch(threadIdx.x);
  for (int w = warp; w < p.W; w += kBsWarps) {
    const int64_t base = lists + (int64_t)w * p.pieces;
    float m = -INFINITY, q = -INFINITY, u = 0.f;  // the warp's pieces one by one per lane
    for (int i = lane; i < p.pieces; i += 32) m = fmaxf(m, __ldcg(p.piece_max + base + i));
    m = warp_max(m);
    double s = 0.0;
    for (int i = lane; i < p.pieces; i += 32) {
      q = __ldcg(p.piece_max + base + i);
      u = __ldcg(p.piece_sum + base + i);
      if (q > -INFINITY) s += (double)u * exp((double)q - (double)m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) lse[w] = m > -INFINITY ? (double)m + log(s) : 0.0;
  }
  __syncthreads();
  u64 best = 0;
  for (int i = threadIdx.x; i < M; i += kBsThreads) {
    const u64 x = i == (int)threadIdx.x ? first : fetch(i);
    u64 q = 0;
    uint32_t t = 0;
    if (x) {
      const int w = i / per;
      t = 0xffffffffu - (uint32_t)x;
      const double sc = (double)p.scores[b * p.W + w] + ((double)unorder_f32((uint32_t)(x >> 32)) - lse[w]);
      q = sc > -INFINITY ? order_f64(sc) : 0ull;
    } else if (i >= p.W * per) {
      const int w = i - p.W * per;  // a finished beam goes on as it is
      const float sc = p.scores[b * p.W + w];
      if (p.finished && p.finished[b * p.W + w] && sc > -INFINITY) {
        q = order_f64((double)sc);
        t = (uint32_t)p.pad;
      }
    }
    key[i] = q;
    tok[i] = t;
    best = q > best ? q : best;
  }
  auto beam_of = [&](int i) { return i < p.W * per ? i / per : i - p.W * per; };
  auto flat = [&](int i) { return (u64)beam_of(i) * (u64)p.V + tok[i]; };
  // a threshold as in the scan, on the upper half of the scores
  const int groups = group_count(p.k);
  put_group_max((uint32_t)(best >> 32), groups, sh.group);
  __syncthreads();
  const uint32_t cut = min_group_max(groups, sh.group);
  for (int i = threadIdx.x; i < M; i += kBsThreads) {
    const u64 q = key[i];
    if (q != 0 && (uint32_t)(q >> 32) >= cut) {
      const int e = atomicAdd(&sh.count, 1);
      if (e < kBsCap) {
        sh.list[e] = q;
        at_flat[e] = flat(i);
      }
    }
  }
  __syncthreads();
  int n = sh.count;
  if (n > kBsCap) {
    // many equal scores: the k-th best (score, flat index) bit by bit
    u64 ck = 0, cf = 0;  // candidates with (key, ~flat) >= (ck, cf) stay
    bool done = false;
    for (int bit = 63; bit >= 0 && !done; --bit) {
      const u64 tr = ck | (1ull << bit);
      int c = 0;
      for (int i = threadIdx.x; i < M; i += kBsThreads) c += key[i] >= tr;
      c = block_sum(c, sh);
      if (c >= p.k) ck = tr;
      done = c == p.k;
    }
    for (int bit = 63; bit >= 0 && !done; --bit) {
      const u64 tr = cf | (1ull << bit);
      int c = 0;
      for (int i = threadIdx.x; i < M; i += kBsThreads) c += key[i] > ck || (key[i] == ck && ~flat(i) >= tr);
      c = block_sum(c, sh);
      if (c >= p.k) cf = tr;
      done = c == p.k;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < M; i += kBsThreads) {
      if (key[i] != 0 && (key[i] > ck || (key[i] == ck && ~flat(i) >= cf))) {
        const int e = atomicAdd(&sh.count, 1);
        if (e < kBsCap) {
          sh.list[e] = key[i];
          at_flat[e] = flat(i);
        }
      }
    }
    __syncthreads();
    n = min(sh.count, kBsCap);
  }
  const int64_t out = (int64_t)b * p.k;
  for (int i0 = 0; i0 < n; i0 += kBsThreads / 8) {  // eight threads count for one candidate
    const int i = i0 + (threadIdx.x >> 3);
    const u64 ki = i < n ? sh.list[i] : ~0ull, fi = i < n ? at_flat[i] : 0ull;
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 7; j < n; j += 8) {
      const u64 kj = sh.list[j], fj = at_flat[j];
      rank += kj > ki || (kj == ki && fj < fi);
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    rank += __shfl_xor_sync(0xffffffffu, rank, 4);
    if (i < n && rank < p.k && (threadIdx.x & 7) == 0) {
      const u64 w = fi / (u64)p.V;
      p.out_scores[out + rank] = (float)unorder_f64(ki);
      p.out_tokens[out + rank] = (int64_t)(fi - w * (u64)p.V);
      p.out_parents[out + rank] = (int64_t)w;
    }
  }
  for (int r = n + threadIdx.x; r < p.k; r += kBsThreads) {  // too few candidates
    p.out_scores[out + r] = -INFINITY;
    p.out_tokens[out + r] = -1;
    p.out_parents[out + r] = 0;
  }
}

struct BeamPlan {
  int pieces = 1, piece = kBsTile;
  size_t max_off = 0, sum_off = 0, count_off = 0, key_off = 0, bytes = 0, merge_smem = 0;
};

// Pieces per row: the split that takes the fewest rounds of tiles when two CTAs fit
// an SM; a piece costs about 1.5 tiles beside its tiles (threshold, final ranks).
BeamPlan beam_plan(int rows, int W, int V, int k, int sm_count) {
  BeamPlan pl;
  const int tiles = (int)(((int64_t)V + kBsTile - 1) / kBsTile);
  const int most = std::max(1, std::min({tiles, (kBsMaxMerge - W) / (W * k), 1024, INT_MAX / rows}));
  double best = 1e30;
  for (int s = 1; s <= most; ++s) {
    const int t = (tiles + s - 1) / s;
    if ((t - 1) * s >= tiles && s > 1) continue;
    const int64_t rounds = ((int64_t)rows * s + 2 * sm_count - 1) / (2 * sm_count);
    const double cost = (double)rounds * (t + 1.5);
    if (cost < best) {
      best = cost;
      pl.piece = t * kBsTile;
      pl.pieces = (tiles + t - 1) / t;
    }
  }
  const size_t n = (size_t)rows * pl.pieces;
  pl.max_off = 0;
  pl.sum_off = align_up(n * 4, 256);
  pl.count_off = pl.sum_off + align_up(n * 4, 256);
  pl.key_off = pl.count_off + align_up(n * 4, 256);
  pl.bytes = pl.key_off + n * k * 8;
  pl.merge_smem = ((size_t)W * pl.pieces * k + W) * 12;
  return pl;
}

bool beam_size_ok(int batch, int beams, int vocab, int k) {
  return batch > 0 && beams > 0 && beams <= kBsMaxBeams && vocab > 0 && vocab <= (1 << 30) && k > 0 && k <= kBsMaxK &&
         (int64_t)batch * beams <= (1 << 20);
}

using ScanFn = void (*)(ScanParams);

// ---- reordering -------------------------------------------------------------------
constexpr int kBrThreads = 256;

struct ReorderParams {
  const nsm_beam_state* states;
  const int64_t* parents;  // [B][W]
  int W;
  int64_t length;          // < 0: whole states
};

// Bytes of a run of `st` that move, and the largest power of two that divides its
// addresses and that number.
__host__ __device__ __forceinline__ int64_t run_bytes(const nsm_beam_state& st, int64_t length) {
  return st.position_bytes > 0 && length >= 0 ? (length < st.positions ? length : st.positions) * st.position_bytes
                                              : st.run_bytes;
}
__host__ __device__ __forceinline__ int state_unit(const nsm_beam_state& st) {
  const u64 a = (u64)(uintptr_t)st.data | (u64)st.row_stride | (st.outer0 > 1 ? (u64)st.outer0_stride : 0) |
                (st.outer1 > 1 ? (u64)st.outer1_stride : 0) |
                (u64)(st.position_bytes > 0 ? st.position_bytes : st.run_bytes) | 16u;
  return (int)(a & (~a + 1));
}

template <int kMaxW, typename U>
__device__ __forceinline__ void move_columns(const nsm_beam_state& st, int64_t run, int W, int b, uint32_t need,
                                             const uint32_t* to) {
  const int64_t per = run / (int64_t)sizeof(U);
  const int64_t total = per * st.outer0 * st.outer1;
  char* base = reinterpret_cast<char*>(st.data) + (int64_t)b * W * st.row_stride;
  for (int64_t i = blockIdx.x * (int64_t)kBrThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kBrThreads) {
    const int64_t o = i / per, in = i - o * per, o0 = o / st.outer1, o1 = o - o0 * st.outer1;
    char* col = base + o0 * st.outer0_stride + o1 * st.outer1_stride + in * (int64_t)sizeof(U);
    U v[kMaxW];
#pragma unroll
    for (int w = 0; w < kMaxW; ++w)
      if (need >> w & 1) v[w] = *reinterpret_cast<const U*>(col + w * st.row_stride);
#pragma unroll
    for (int w = 0; w < kMaxW; ++w) {
      if (need >> w & 1) {
        uint32_t m = to[w];
        while (m) {
          const int j = __ffs(m) - 1;
          m &= m - 1;
          *reinterpret_cast<U*>(col + j * st.row_stride) = v[w];
        }
      }
    }
  }
}

template <int kMaxW>
__global__ void __launch_bounds__(kBrThreads) beam_reorder_kernel(ReorderParams p) {
  __shared__ uint32_t to[kBsMaxBeams];  // beams that go on with beam w's state, w itself not among them
  __shared__ uint32_t need_sh;
  const int b = blockIdx.z;
  if (threadIdx.x < 32) {
    const int j = threadIdx.x;
    int64_t src = j < p.W ? p.parents[(int64_t)b * p.W + j] : j;
    if (src < 0 || src >= p.W) src = j;  // no such beam: the row stays
    uint32_t need = 0;
    for (int w = 0; w < p.W; ++w) {
      const uint32_t m = __ballot_sync(0xffffffffu, j < p.W && src == w && j != w);
      if (m) need |= 1u << w;
      if (j == 0) to[w] = m;
    }
    if (j == 0) need_sh = need;
  }
  __syncthreads();
  const uint32_t need = need_sh;
  if (need == 0) return;
  const nsm_beam_state st = p.states[blockIdx.y];
  const int64_t run = run_bytes(st, p.length);
  if (run <= 0) return;
  switch (state_unit(st)) {
    case 16: move_columns<kMaxW, uint4>(st, run, p.W, b, need, to); break;
    case 8: move_columns<kMaxW, uint2>(st, run, p.W, b, need, to); break;
    case 4: move_columns<kMaxW, uint32_t>(st, run, p.W, b, need, to); break;
    case 2: move_columns<kMaxW, unsigned short>(st, run, p.W, b, need, to); break;
    default: move_columns<kMaxW, unsigned char>(st, run, p.W, b, need, to); break;
  }
}

int check_state(const nsm_beam_state& st) {
  if (st.data == nullptr || st.outer0 < 1 || st.outer1 < 1 || st.run_bytes < 1 || st.position_bytes < 0)
    return fail(NSM_ERR_INVALID_ARG, "beam state: NULL data or a size below 1");
  if (st.row_stride < 0 || st.outer0_stride < 0 || st.outer1_stride < 0)
    return fail(NSM_ERR_INVALID_ARG, "beam state: negative stride");
  if (st.position_bytes > 0 && st.positions * st.position_bytes != st.run_bytes)
    return fail(NSM_ERR_INVALID_ARG, "beam state: run_bytes is not positions * position_bytes");
  return NSM_OK;
}

}  // namespace
}  // namespace nsm

using namespace nsm;

extern "C" {

size_t nsm_beam_select_workspace_bytes(int32_t batch, int32_t beams, int32_t vocab, int32_t candidates) {
  if (!beam_size_ok(batch, beams, vocab, candidates)) return 0;
  DeviceInfo di;
  if (current_device(&di) != NSM_OK) return 0;
  return beam_plan(batch * beams, beams, vocab, candidates, di.sm_count).bytes;
}

int nsm_beam_select(const void* logits, int32_t logits_dtype, int64_t batch_stride, int64_t beam_stride,
                    const float* scores, const uint8_t* finished, int32_t batch, int32_t beams, int32_t vocab,
                    int32_t candidates, int32_t pad_token, float* out_scores, int64_t* out_tokens,
                    int64_t* out_parents, void* workspace, size_t workspace_bytes, nsm_stream_t stream) {
  NSM_REQUIRE(logits_dtype == NSM_F32 || logits_dtype == NSM_F16 || logits_dtype == NSM_BF16, NSM_ERR_INVALID_ARG,
              "nsm_beam_select: bad dtype");
  NSM_REQUIRE(batch >= 0, NSM_ERR_INVALID_ARG, "nsm_beam_select: negative batch");
  if (batch == 0) return NSM_OK;
  NSM_REQUIRE(beam_size_ok(batch, beams, vocab, candidates), NSM_ERR_UNSUPPORTED,
              "nsm_beam_select: needs 1..32 beams, 1..64 candidates, 1..2^30 tokens and at most 2^20 rows");
  NSM_REQUIRE(logits && scores && out_scores && out_tokens && out_parents && workspace, NSM_ERR_INVALID_ARG,
              "nsm_beam_select: NULL pointer");
  NSM_REQUIRE(pad_token >= 0 && pad_token < vocab, NSM_ERR_INVALID_ARG, "nsm_beam_select: pad_token outside the vocabulary");
  NSM_REQUIRE(batch_stride >= 0 && beam_stride >= 0, NSM_ERR_INVALID_ARG, "nsm_beam_select: negative stride");
  const int es = logits_dtype == NSM_F32 ? 4 : 2;
  NSM_REQUIRE(((uintptr_t)logits & (es - 1)) == 0, NSM_ERR_INVALID_ARG, "nsm_beam_select: logits misaligned");
  DeviceInfo di;
  const int rc = current_device(&di);
  if (rc != NSM_OK) return rc;
  const int rows = batch * beams;
  const BeamPlan pl = beam_plan(rows, beams, vocab, candidates, di.sm_count);
  NSM_REQUIRE(((uintptr_t)workspace & 255) == 0 && workspace_bytes >= pl.bytes, NSM_ERR_WORKSPACE,
              "nsm_beam_select: workspace misaligned or too small (nsm_beam_select_workspace_bytes)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  ScanParams sp;
  sp.logits = logits;
  sp.batch_stride = batch_stride;
  sp.beam_stride = beam_stride;
  sp.scores = scores;
  sp.finished = finished;
  sp.W = beams;
  sp.V = vocab;
  sp.k = candidates;
  sp.pieces = pl.pieces;
  sp.piece = pl.piece;
  sp.piece_max = reinterpret_cast<float*>(ws + pl.max_off);
  sp.piece_sum = reinterpret_cast<float*>(ws + pl.sum_off);
  sp.piece_count = reinterpret_cast<int*>(ws + pl.count_off);
  sp.piece_keys = reinterpret_cast<u64*>(ws + pl.key_off);
  // 16-byte loads when every row starts on 16 bytes, else one value per lane
  const bool vec = (((uintptr_t)logits | (uintptr_t)(batch_stride * es) | (uintptr_t)(beam_stride * es)) & 15) == 0;
  const ScanFn fn = logits_dtype == NSM_F32   ? (vec ? beam_scan_kernel<float, true> : beam_scan_kernel<float, false>)
                    : logits_dtype == NSM_F16 ? (vec ? beam_scan_kernel<__half, true> : beam_scan_kernel<__half, false>)
                                              : (vec ? beam_scan_kernel<__nv_bfloat16, true>
                                                     : beam_scan_kernel<__nv_bfloat16, false>);
  fn<<<(unsigned)(rows * pl.pieces), kBsThreads, 0, s>>>(sp);
  NSM_CHECK_CUDA(cudaGetLastError());
  MergeParams mp;
  mp.scores = scores;
  mp.finished = finished;
  mp.W = beams;
  mp.V = vocab;
  mp.k = candidates;
  mp.pieces = pl.pieces;
  mp.pad = pad_token;
  mp.piece_max = sp.piece_max;
  mp.piece_sum = sp.piece_sum;
  mp.piece_count = sp.piece_count;
  mp.piece_keys = sp.piece_keys;
  mp.out_scores = out_scores;
  mp.out_tokens = out_tokens;
  mp.out_parents = out_parents;
  NSM_CHECK_CUDA(cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBsMaxMerge * 12));
  NSM_CHECK_CUDA(launch_pdl(beam_merge_kernel, dim3(batch), dim3(kBsThreads), pl.merge_smem, s, mp));
  return NSM_OK;
}

size_t nsm_beam_states_bytes(int32_t count) { return count > 0 ? (size_t)count * sizeof(nsm_beam_state) : 0; }

int nsm_beam_states_set(const nsm_beam_state* states, int32_t count, void* table, size_t table_bytes,
                        nsm_stream_t stream) {
  NSM_REQUIRE(states && table && count > 0 && count <= 65535, NSM_ERR_INVALID_ARG,
              "nsm_beam_states_set: NULL pointer or a count outside 1..65535");
  NSM_REQUIRE(((uintptr_t)table & 15) == 0 && table_bytes >= nsm_beam_states_bytes(count), NSM_ERR_WORKSPACE,
              "nsm_beam_states_set: table misaligned or too small (nsm_beam_states_bytes)");
  for (int i = 0; i < count; ++i) {
    const int rc = check_state(states[i]);
    if (rc != NSM_OK) return rc;
  }
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  NSM_CHECK_CUDA(cudaMemcpyAsync(table, states, nsm_beam_states_bytes(count), cudaMemcpyHostToDevice, s));
  NSM_CHECK_CUDA(cudaStreamSynchronize(s));
  return NSM_OK;
}

int nsm_beam_reorder(const nsm_beam_state* states, const void* table, int32_t count, int32_t batch, int32_t beams,
                     const int64_t* parents, int64_t length, nsm_stream_t stream) {
  NSM_REQUIRE(batch >= 0, NSM_ERR_INVALID_ARG, "nsm_beam_reorder: negative batch");
  if (batch == 0 || count == 0) return NSM_OK;
  NSM_REQUIRE(states && table && parents && count > 0 && count <= 65535, NSM_ERR_INVALID_ARG,
              "nsm_beam_reorder: NULL pointer or a count outside 1..65535");
  NSM_REQUIRE(batch <= 65535 && beams > 0 && beams <= kBsMaxBeams, NSM_ERR_UNSUPPORTED,
              "nsm_beam_reorder: needs 1..32 beams and at most 65535 batch items");
  DeviceInfo di;
  const int rc = current_device(&di);
  if (rc != NSM_OK) return rc;
  if (beams == 1) return NSM_OK;  // the only beam's state is its own
  int64_t most = 0;
  for (int i = 0; i < count; ++i) {
    const int bad = check_state(states[i]);
    if (bad != NSM_OK) return bad;
    most = std::max(most, run_bytes(states[i], length) / state_unit(states[i]) * states[i].outer0 * states[i].outer1);
  }
  if (most == 0) return NSM_OK;
  ReorderParams p;
  p.states = reinterpret_cast<const nsm_beam_state*>(table);
  p.parents = parents;
  p.W = beams;
  p.length = length;
  // enough CTAs for 16 per SM over all states, and no more than there are columns
  const int64_t want = std::max<int64_t>(1, (16LL * di.sm_count + (int64_t)count * batch - 1) / ((int64_t)count * batch));
  const dim3 grid((unsigned)std::min<int64_t>((most + kBrThreads - 1) / kBrThreads, want), (unsigned)count,
                  (unsigned)batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (beams <= 4)
    beam_reorder_kernel<4><<<grid, kBrThreads, 0, s>>>(p);
  else if (beams <= 8)
    beam_reorder_kernel<8><<<grid, kBrThreads, 0, s>>>(p);
  else if (beams <= 16)
    beam_reorder_kernel<16><<<grid, kBrThreads, 0, s>>>(p);
  else
    beam_reorder_kernel<32><<<grid, kBrThreads, 0, s>>>(p);
  NSM_CHECK_CUDA(cudaGetLastError());
  return NSM_OK;
}

}  // extern "C"
