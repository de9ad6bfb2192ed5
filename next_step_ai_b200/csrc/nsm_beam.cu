// nsm_beam.cu -- beam search after the logits: the best continuations over
// beams and vocabulary, and the reordering of the beams' states.
//
// Selection.  A candidate (beam w, token v) of a batch item has the score
//
//   score[w] + logit[w][v] - logsumexp(logit[w][:])
//
// and the k best are wanted, equal scores in the order of w, then v.  Inside one
// beam the order of the scores is the order of the logits.  beam_scan_kernel reads
// the logits once and selects nothing: a warp takes a contiguous piece of a row,
// 1024 values at a time in registers, keeps a running maximum and sum of exponentials per
// lane (fp32), and notes the largest value of each block of 1024.
// beam_merge_kernel, one CTA per batch item, joins the sums (in 64 bits) and picks
// the k best blocks by (largest score, position).  The k best candidates are in
// them: any candidate of another block is beaten by the largest of each of these k,
// equal scores included, since blocks are contiguous and in the order of the
// candidates.  Their values are read again (from L2), scored in 64 bits, and those
// that reach the k-th block's largest, hardly more than k, are ranked by counting.
// beam_select_kernel is both in one launch, for inputs that a cluster of CTAs per batch item
// goes through as quickly: a call then costs the host 12.5 us instead of 16.5 (one launch and no
// workspace), and the GPU 1.3 us more in a graph (9.8 and 11.7 us instead of 8.6 and 10.3 for
// 1 x 4 x 128256 in fp32 and 24 x 5 x 50257 in fp16).
//
// Measured in a graph: 32 x 16 x 128256 in fp32, 32 candidates 41 us (the scan 33: 200 MB, 94% of
// the copy bandwidth); 16 x 8 x 128256 in bf16 16 us, 9.7 of them the scan, four blocks per warp
// one wait for memory after the other (1.1 instructions per cycle, DRAM 31%).  The merge is a chain of short
// steps of one CTA, 5 to 6 us: loads from L2, a double-precision logarithm, ranks.
//
// Reordering.  beam_reorder_kernel moves the states in place: a thread owns
// one 1- to 16-byte column of all beams of a batch item, loads the beams that
// others go on with, then stores them where they moved.  A beam that stays
// is not written, and one that nobody else takes is not read.
#include <algorithm>

#include "nsm_common.cuh"
#include "nsm_internal.h"

namespace nsm {
namespace {

using u64 = unsigned long long;

constexpr int kBsThreads = 256;
constexpr int kBsWarps = kBsThreads / 32;
constexpr int kBsPer = 32;                       // values per lane
constexpr int kBsBlock = 32 * kBsPer;            // values of a block: one warp's registers
constexpr int kBsMaxEntries = 384;               // noted maxima of a row
constexpr int kBmThreads = 1024;                 // of the merge: a warp per beam, 8 threads per ranked candidate
constexpr int kBmGroups = 128;                   // groups of blocks for the first threshold
constexpr int kBmWarps = kBmThreads / 32;
constexpr int kBmCap = 2048;                     // candidates ranked by counting
constexpr int kBsMaxK = 64;
constexpr int kBsMaxBeams = 32;
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
__device__ __forceinline__ uint32_t order_clean(float v) {
  v = clean(v);
  return v == -INFINITY ? 0u : order_f32(v + 0.f);
}

struct ScanParams {
  const void* logits;
  int64_t batch_stride, beam_stride;  // elements
  const float* scores;                // [B][W]
  const uint8_t* finished;            // [B][W] or NULL
  int rows, W, V;
  int segs, seg_blocks;               // warps per row, blocks of 1024 per warp (a multiple of run)
  int entries, run;                   // noted maxima per row, blocks of each
  float2* seg;                        // [rows][segs] maximum, sum of exp(value - maximum)
  uint32_t* top;                      // [rows][entries] largest value in ordered bits
};

// The values of a thread as they are loaded; 16-bit types two to a word.
template <typename T>
struct RawTile {
  uint32_t r[kBsPer * (int)sizeof(T) / 4];
};
template <typename T>
__device__ __forceinline__ float raw_value(uint32_t word, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(word);
  } else if constexpr (sizeof(T) == 2 && __is_same(T, __nv_bfloat16)) {
    return __uint_as_float(i % 2 ? word & 0xffff0000u : word << 16);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&word));
    return i % 2 ? f.y : f.x;
  }
}
template <typename T>
__device__ __forceinline__ float raw_value(const RawTile<T>& q, int i) {
  return raw_value<T>(q.r[i * (int)sizeof(T) / 4], i);
}
// The largest value (NaN is passed over); 16-bit types two at a time.
template <typename T>
__device__ __forceinline__ float raw_max(const RawTile<T>& q) {
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(q.r[0]);
#pragma unroll
    for (int i = 1; i < kBsPer; ++i) m = fmaxf(m, __uint_as_float(q.r[i]));
    return m;
  } else if constexpr (__is_same(T, __nv_bfloat16)) {
    __nv_bfloat162 m = *reinterpret_cast<const __nv_bfloat162*>(&q.r[0]);
#pragma unroll
    for (int i = 1; i < kBsPer / 2; ++i) m = __hmax2(m, *reinterpret_cast<const __nv_bfloat162*>(&q.r[i]));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    __half2 m = *reinterpret_cast<const __half2*>(&q.r[0]);
#pragma unroll
    for (int i = 1; i < kBsPer / 2; ++i) m = __hmax2(m, *reinterpret_cast<const __half2*>(&q.r[i]));
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// sum of exp(value - top) over the thread's values
template <typename T, bool kClean>
__device__ __forceinline__ float raw_exp_sum(const RawTile<T>& q, float top) {
  const u64 off = pair2(-top, -top), l2e = pair2(kLog2e, kLog2e);
  u64 sum[2] = {0, 0};  // two chains of two sums
#pragma unroll
  for (int i = 0; i < kBsPer; i += 2) {
    float a = raw_value<T>(q, i), b = raw_value<T>(q, i + 1);
    if (kClean) {
      a = clean(a);
      b = clean(b);
    }
    const float2 x = unpair2(mul2(add2(pair2(a, b), off), l2e));
    sum[(i / 2) % 2] = add2(sum[(i / 2) % 2], pair2(exp2_fast(x.x), exp2_fast(x.y)));
  }
  const float2 t = unpair2(add2(sum[0], sum[1]));
  return t.x + t.y;
}

// Position in the block of value i of a lane.  A full block with kVec: runs of 16
// bytes, so that 16-byte loads of neighbouring lanes touch neighbouring memory; otherwise
// one value per lane.  The mapping is the same for every row of a call: equal rows give
// equal sums, bit for bit.
template <typename T, bool kVec>
__device__ __forceinline__ int block_pos(int i, bool full) {
  constexpr int n = 16 / sizeof(T);
  const int lane = threadIdx.x & 31;
  if (kVec && full) return (i / n) * (32 * n) + lane * n + i % n;
  return i * 32 + lane;
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

// Block values [at, at + left) of a row (left > 0); beyond it -infinity.
template <typename T, bool kVec>
__device__ __forceinline__ void load_block(const T* row, int64_t at, int left, RawTile<T>& q) {
  if constexpr (kVec) {
    if (left >= kBsBlock) {
      const uint4* src = reinterpret_cast<const uint4*>(row + at) + (threadIdx.x & 31);
#pragma unroll
      for (int i = 0; i < kBsPer * (int)sizeof(T) / 16; ++i) {
        const uint4 u = ldg_stream_u4(src + i * 32);
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
    const int pos = block_pos<T, kVec>(i, false);
    const uint32_t b = pos < left ? raw_bits<T>(row[at + pos]) : kMinusInf<T>;
    if constexpr (sizeof(T) == 2) {
      q.r[i / 2] = i % 2 ? q.r[i / 2] | b << 16 : b;
    } else {
      q.r[i] = b;
    }
  }
}

// Piece sg of a row, by one warp: put_top(e, largest value in ordered bits) for each of its
// entries, put_seg(maximum, sum of exp(value - maximum)).
template <typename T, bool kVec, typename PutTop, typename PutSeg>
__device__ __forceinline__ void scan_piece(const ScanParams& p, int row, int sg, PutTop put_top, PutSeg put_seg) {
  // a beam that is out (no score above -infinity) or finished is not read, here or later
  if (!(p.scores[row] > -INFINITY) || (p.finished && p.finished[row])) return;
  const int b = row / p.W, w = row - b * p.W;
  const T* src = reinterpret_cast<const T*>(p.logits) + b * p.batch_stride + w * p.beam_stride;
  const int64_t begin = (int64_t)sg * p.seg_blocks * kBsBlock;
  const int64_t end = min((int64_t)p.V, begin + (int64_t)p.seg_blocks * kBsBlock);
  float m = -INFINITY, s = 0.f, run_top = -INFINITY;
  int in_run = 0, entry = sg * (p.seg_blocks / p.run);
  for (int64_t at = begin; at < end; at += kBsBlock) {  // the SM's other warps cover the wait for a block
    RawTile<T> q;
    load_block<T, kVec>(src, at, (int)min((int64_t)kBsBlock, end - at), q);
    const float rm = raw_max<T>(q);
    if (rm > -INFINITY) {  // else nothing but -infinity and NaN
      const float tm = fminf(rm, kFltMax), nm = fmaxf(m, tm);
      float e = raw_exp_sum<T, false>(q, nm);
      // the maximum passes over NaN and infinities make NaN: such a block is summed again
      if (!(e <= kFltMax)) e = raw_exp_sum<T, true>(q, nm);
      s = s * exp2_fast((m - nm) * kLog2e) + e;  // m = -infinity: s is 0
      m = nm;
      run_top = fmaxf(run_top, tm);
    }
    if (++in_run == p.run || at + kBsBlock >= end) {
      put_top(entry++, __reduce_max_sync(0xffffffffu, order_clean(run_top)));
      run_top = -INFINITY;
      in_run = 0;
    }
  }
  const float wm = warp_max(m);
  put_seg(wm, warp_sum(m > -INFINITY ? s * exp2_fast((m - wm) * kLog2e) : 0.f));
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kBsThreads, 4) beam_scan_kernel(ScanParams p) {
  pdl_wait();
  pdl_trigger();  // not before: the merge reads the scores before it waits
  const int lane = threadIdx.x & 31;
  const int64_t unit = (int64_t)blockIdx.x * kBsWarps + (threadIdx.x >> 5);
  const int row = (int)(unit / p.segs), sg = (int)(unit - (int64_t)row * p.segs);
  if (row >= p.rows) return;
  scan_piece<T, kVec>(
      p, row, sg,
      [&](int e, uint32_t o) {
        if (lane == 0) p.top[(int64_t)row * p.entries + e] = o;
      },
      [&](float m, float s) {
        if (lane == 0) p.seg[(int64_t)row * p.segs + sg] = make_float2(m, s);
      });
}

struct MergeParams {
  ScanParams scan;
  int k, pad;
  float* out_scores;  // [B][k]
  int64_t* out_tokens;
  int64_t* out_parents;
};

// A candidate is (beam * V + token), a block (its index among [W][entries + 1]): smaller
// comes first among equal scores.  A finished beam has one block, of one candidate.
struct MergeShared {
  u64 key[kBmCap];  // scores in ordered bits, larger is better
  u64 id[kBmCap];
  double lse[kBsMaxBeams], score[kBsMaxBeams];
  int alive[kBsMaxBeams];  // 0: out, 1: read, 2: finished
  uint32_t group[kBmGroups], cut;
  u64 best_key[kBsMaxK];   // the k best blocks
  int best_id[kBsMaxK];
  int entries_listed, values_listed, hits;
};

// The k-th largest of the values in [lo, hi] that `each` runs over (it calls its argument with
// every value), where none is above hi and lo > 0.  need: how many of those equal to it are among
// the k; 0 when all that are at least the result are, which are k, or fewer if there are fewer.
// Every round counts the values in up to 2048 equal parts of the range and goes on with the part
// that holds the k-th.  kNarrow: the range is cut to the values seen too, so that equal values end
// it after one or two rounds.  Uses the candidates' list.
constexpr int kBmBins = 2048;
template <bool kNarrow, typename Each>
__device__ __forceinline__ u64 kth_value(MergeShared& sh, int k, u64 lo, u64 hi, Each each, int& need) {
  static_assert(kBmBins * 4 <= (int)sizeof(sh.key) && kBmBins == 2 * kBmThreads, "two parts per thread");
  int* const count = reinterpret_cast<int*>(sh.key);
  u64* const seen = sh.id;  // the least and largest value, then what the next round goes on with
  int* const warp_count = reinterpret_cast<int*>(sh.id + 8);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, mine = 2 * threadIdx.x;
  int above = 0;
  for (;;) {
    const u64 span = hi - lo;
    const int shift = max(0, 64 - 11 - __clzll((long long)span));
    __syncthreads();
    count[mine] = count[mine + 1] = 0;
    if (threadIdx.x == 0) {
      seen[0] = ~0ull;
      seen[1] = 0;
      seen[2] = seen[3] = 0;  // unless a part has the k-th: all there are
      seen[4] = 1;
    }
    __syncthreads();
    u64 least = ~0ull, most = 0, last = lo - 1;
    int part = 0, run = 0, in = 0;  // a thread's values are often equal, or lie in one part: added up first
    each([&](u64 v) {
      if (v != last) {
        last = v;
        in = v - lo <= span;
        if (!in) return;
        const int at = (int)((v - lo) >> shift);
        if (at != part) {
          if (run > 0) atomicAdd(&count[part], run);
          part = at;
          run = 0;
        }
        if (kNarrow) {
          least = min(least, v);
          most = max(most, v);
        }
      }
      run += in;
    });
    if (run > 0) atomicAdd(&count[part], run);
    __syncwarp();
    if (kNarrow) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      if (lane == 0 && least <= most) {
        atomicMin(&seen[0], least);
        atomicMax(&seen[1], most);
      }
    }
    __syncthreads();
    const int c[2] = {count[mine], count[mine + 1]};
    int n = c[0] + c[1];  // of this thread's parts and all above, in the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int from = __shfl_down_sync(0xffffffffu, n, o);
      if (lane + o < 32) n += from;
    }
    if (lane == 0) warp_count[warp] = n;
    __syncthreads();
    static_assert(kBmWarps == 32, "a lane per warp");
    n += above + __reduce_add_sync(0xffffffffu, lane > warp ? warp_count[lane] : 0) - c[0] - c[1];
#pragma unroll
    for (int i = 1; i >= 0; --i) {
      if (n < k && n + c[i] >= k) {
        const u64 at = lo + ((u64)(mine + i) << shift), last_of = at + ((1ull << shift) - 1);
        seen[2] = kNarrow ? max(at, seen[0]) : at;
        seen[3] = (hi - at) >> shift ? last_of : hi;
        if (kNarrow) seen[3] = min(seen[3], seen[1]);
        seen[4] = (u64)n << 1 | (u64)(n + c[i] == k);
      }
      n += c[i];
    }
    __syncthreads();
    lo = seen[2];
    hi = seen[3];
    above = (int)(seen[4] >> 1);
    const bool all = seen[4] & 1;
    if (all || lo == hi) {
      need = all ? 0 : k - above;
      __syncthreads();
      return lo;
    }
  }
}

// The k-th best (key, id) of what `each` runs over (it calls its argument with every key in
// [lo, hi] and its id, below id_end): exactly k are at least that good if there are k.
template <typename Each>
__device__ __forceinline__ void kth_best(MergeShared& sh, int k, u64 lo, u64 hi, u64 id_end, Each each, u64& ck, u64& cf) {
  int need;
  ck = kth_value<true>(sh, k, lo, hi, [&](auto use) { each([&](u64 key, u64) { use(key); }); }, need);
  cf = ~0ull;
  if (need == 0) return;
  const u64 key_k = ck;  // ids are different: the need-th smallest has need at least as small
  cf = ~kth_value<false>(sh, need, ~id_end, ~0ull, [&](auto use) {
    each([&](u64 key, u64 id) {
      if (key == key_k) use(~id);
    });
  }, need);
}

// Calls found(rank, key, id) for the k best of the n in sh.key / sh.id; eight
// threads count for one.
template <typename Found>
__device__ __forceinline__ void rank_list(const MergeShared& sh, int n, int k, Found found) {
  for (int i0 = 0; i0 < n; i0 += kBmThreads / 8) {
    const int i = i0 + (threadIdx.x >> 3);
    const u64 ki = i < n ? sh.key[i] : ~0ull, di = i < n ? sh.id[i] : 0ull;
    int rank = 0;
#pragma unroll 4
    for (int j = threadIdx.x & 7; j < n; j += 8) {
      const u64 kj = sh.key[j], dj = sh.id[j];
      rank += kj > ki || (kj == ki && dj < di);
    }
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    rank += __shfl_xor_sync(0xffffffffu, rank, 4);
    if (i < n && rank < k && (threadIdx.x & 7) == 0) found(rank, ki, di);
  }
}

// Group maxima: a hash spreads what is put in over the groups.  The k-th largest of the
// maxima is a threshold that k of them reach, and hardly more than k / (1 - k / 256) of all
// (0 when fewer than k groups have any).
__device__ __forceinline__ void put_group(MergeShared& sh, int i, u64 key) {
  static_assert(kBmGroups == 128, "the upper 7 bits of the hash");
  if (key) atomicMax(&sh.group[((uint32_t)i * 2654435769u) >> 25], (uint32_t)(key >> 32));
}
__device__ __forceinline__ uint32_t group_threshold(MergeShared& sh, int k) {
  static_assert(kBmGroups * 8 == kBmThreads && kBmGroups >= kBsMaxK, "eight threads per group");
  const int g = threadIdx.x >> 3;
  const uint32_t mine = sh.group[g];
  int rank = 0;
#pragma unroll 4
  for (int o = threadIdx.x & 7; o < kBmGroups; o += 8) {
    const uint32_t other = sh.group[o];
    rank += other > mine || (other == mine && o < g);
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  rank += __shfl_xor_sync(0xffffffffu, rank, 2);
  rank += __shfl_xor_sync(0xffffffffu, rank, 4);
  if (rank == k - 1 && (threadIdx.x & 7) == 0) sh.cut = mine;
  __syncthreads();
  return sh.cut;
}

// What the steps of the merge share.  The functions that are not inlined copy it: through a
// reference every use in their loops would be a load.
struct MergeView {
  const MergeParams& mp;
  MergeShared& sh;
  u64* entry;  // [W][entries + 1] the blocks' largest scores, 0 = none
  int b;

  __device__ __forceinline__ u64 score_key(int w, float v) const {
    return order_f64(sh.score[w] + ((double)v - sh.lse[w]));
  }
  __device__ __forceinline__ u64 candidate(int w, int64_t token) const { return (u64)w * (unsigned)mp.scan.V + (u64)token; }
  // Above every candidate and block.
  __device__ __forceinline__ u64 id_end() const { return (u64)mp.scan.W * (unsigned)max(mp.scan.V, mp.scan.entries + 1); }
  __device__ __forceinline__ void append(int* count, u64 key, u64 id) const {
    const int e = atomicAdd(count, 1);
    if (e < kBmCap) {
      sh.key[e] = key;
      sh.id[e] = id;
    }
  }
  // More than the list holds: it is made again, and nothing more need be put in.
  __device__ __forceinline__ bool over(const int* count) const {
    return *reinterpret_cast<const volatile int*>(count) > kBmCap;
  }
  template <typename T>
  __device__ __forceinline__ const T* row(int w) const {
    return reinterpret_cast<const T*>(mp.scan.logits) + b * mp.scan.batch_stride + w * mp.scan.beam_stride;
  }
};

// Cuts a list of more than kBmRank candidates down before they are ranked by counting (which
// costs their number squared): by the groups' threshold, and if very many scores are equal
// exactly.
constexpr int kBmRank = 256;
constexpr int kBmMany = kBsBlock - 1;  // candidates listed (one value after the other): no block of equal values
static_assert(kBmMany + kBsMaxBeams <= kBmCap, "the list, with the finished beams' candidates");
__device__ __noinline__ void shrink_list(const MergeView& view, int* count) {
  const MergeParams mp = view.mp;
  const MergeView v{mp, view.sh, view.entry, view.b};
  MergeShared& sh = v.sh;
  constexpr int kMine = kBmCap / kBmThreads;
  u64 key[kMine], id[kMine];
  const int n = *count;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int e = i * kBmThreads + threadIdx.x;
    key[i] = e < n ? sh.key[e] : 0ull;
    id[i] = e < n ? sh.id[e] : 0ull;
  }
  if (threadIdx.x < kBmGroups) sh.group[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; ++i) put_group(sh, i * kBmThreads + threadIdx.x, key[i]);
  __syncthreads();
  u64 ck = (u64)group_threshold(sh, v.mp.k) << 32, cf = ~0ull;
  for (int exact = 0; exact < 2; ++exact) {
    if (exact) {
      kth_best(sh, v.mp.k, max(ck, 1ull), ~0ull, v.id_end(), [&](auto use) {
#pragma unroll
        for (int i = 0; i < kMine; ++i)
          if (key[i]) use(key[i], id[i]);
      }, ck, cf);
    }
    __syncthreads();
    if (threadIdx.x == 0) *count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (key[i] && (key[i] > ck || (key[i] == ck && id[i] <= cf))) v.append(count, key[i], id[i]);
    __syncthreads();
    if (*count <= kBmRank) break;
  }
}

// The k best blocks when very many have equal maxima.
__device__ __noinline__ void entries_again(const MergeView& view) {
  const MergeParams mp = view.mp;
  const MergeView v{mp, view.sh, view.entry, view.b};
  const int n = v.mp.scan.W * (v.mp.scan.entries + 1);
  u64 ck, cf;
  kth_best(v.sh, v.mp.k, 1ull, ~0ull, v.id_end(), [&](auto use) {
    for (int i = threadIdx.x; i < n; i += kBmThreads)
      if (v.entry[i]) use(v.entry[i], (u64)i);
  }, ck, cf);
  if (threadIdx.x == 0) v.sh.entries_listed = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kBmThreads) {
    const u64 q = v.entry[i];
    if (q && (q > ck || (q == ck && (u64)i <= cf))) v.append(&v.sh.entries_listed, q, i);
  }
  __syncthreads();
}

// Block i % run of the chosen entry i / run: its beam w and where it begins; false where there
// are no values (a finished beam, the last entry's end).
__device__ __forceinline__ bool find_chosen(const MergeView& v, int i, int& w, int64_t& at) {
  const ScanParams& p = v.mp.scan;
  const int j = p.run == 1 ? i : i / p.run, per_beam = p.entries + 1;
  const int id = v.sh.best_id[j];
  w = id / per_beam;
  at = ((int64_t)(id - w * per_beam) * p.run + (i - j * p.run)) * kBsBlock;
  return v.sh.alive[w] != 2 && at < p.V;
}

// Eight values per lane of a block of `left`: block_pos's 8 part .. 8 part + 7.
constexpr int kBmPer = 8, kBmParts = kBsPer / kBmPer;
template <typename T, bool kVec>
__device__ __forceinline__ void load_part(const T* block, int left, int part, uint32_t* r) {
  constexpr int n = 16 / sizeof(T);
  if (kVec && left >= kBsBlock) {
#pragma unroll
    for (int c = 0; c < kBmPer / n; ++c) {
      const uint4 u = *(reinterpret_cast<const uint4*>(block) + (part * (kBmPer / n) + c) * 32 + (threadIdx.x & 31));
      r[4 * c] = u.x;
      r[4 * c + 1] = u.y;
      r[4 * c + 2] = u.z;
      r[4 * c + 3] = u.w;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < kBmPer; ++e) {
    const int pos = block_pos<T, kVec>(part * kBmPer + e, false);
    const uint32_t b = pos < left ? raw_bits<T>(block[pos]) : kMinusInf<T>;
    uint32_t& word = r[e * (int)sizeof(T) / 4];
    word = sizeof(T) == 2 && e % 2 ? word | b << 16 : b;
  }
}

// The k best of the blocks' values when very many reach `least`: equal scores, or large values
// next to each other.  Every pass reads the blocks again, from L2, a warp per quarter of a block and
// the next quarter under way.  With every word of 1 x 4 x 128256 masked by the lowest value but one,
// 8 candidates, the call takes 41 us (ordinary logits 12.5; five passes over 8192 values); of
// 1 x 32 x 128256, 64 candidates, 125 us (20.6; over 65536 values, by the issue of some 50
// instructions each).
template <typename T, bool kVec>
__device__ __noinline__ void values_again(const MergeView& view, int blocks, u64 least) {
  const MergeParams mp = view.mp;
  const MergeView v{mp, view.sh, view.entry, view.b};
  const ScanParams& p = mp.scan;
  const int lane = threadIdx.x & 31;
  struct Part {
    uint32_t r[kBmPer * sizeof(T) / 4];
    int64_t at;
    int w, left;  // left: 0 = no values, -1 = a finished beam's candidate
  };
  auto load = [&](int i, Part& q) {
    q.left = 0;
    if (i >= blocks * p.run * kBmParts) return;
    if (!find_chosen(v, i / kBmParts, q.w, q.at)) {
      if (v.sh.alive[q.w] == 2 && i % (p.run * kBmParts) == 0) q.left = -1;
      q.at = i / (p.run * kBmParts);
      return;
    }
    q.left = (int)min((int64_t)kBsBlock, p.V - q.at);
    load_part<T, kVec>(v.row<T>(q.w) + q.at, q.left, i % kBmParts, q.r);
  };
  auto each = [&](auto use) {
    Part next;
    load(threadIdx.x >> 5, next);
    for (int i = threadIdx.x >> 5; i < blocks * p.run * kBmParts; i += kBmWarps) {
      const Part q = next;
      load(i + kBmWarps, next);
      if (q.left < 0 && lane == 0) use(v.sh.best_key[q.at], v.candidate(q.w, v.mp.pad));
      if (q.left <= 0) continue;
      float last = -INFINITY;
      u64 key = 0;
#pragma unroll
      for (int e = 0; e < kBmPer; ++e) {
        const float x = clean(raw_value<T>(q.r[e * (int)sizeof(T) / 4], e));
        if (x != last) {  // equal values follow each other where there are very many
          key = x > -INFINITY ? v.score_key(q.w, x) : 0ull;
          last = x;
        }
        if (key >= least)
          use(key, v.candidate(q.w, q.at + block_pos<T, kVec>(i % kBmParts * kBmPer + e, q.left >= kBsBlock)));
      }
    }
  };
  u64 ck, cf;
  kth_best(v.sh, v.mp.k, least, v.sh.best_key[0], v.id_end(), each, ck, cf);
  if (threadIdx.x == 0) v.sh.values_listed = 0;
  __syncthreads();
  each([&](u64 key, u64 id) {
    if (key > ck || (key == ck && id <= cf)) v.append(&v.sh.values_listed, key, id);
  });
  __syncthreads();
}

// What the scan noted: in global memory, by the kernel before (pdl_wait first), or in shared
// memory.
template <bool kShared>
struct Notes {
  const float2* seg;
  const uint32_t* top;
  __device__ __forceinline__ float2 load(const float2* at) const { return kShared ? *at : __ldcg(at); }
  __device__ __forceinline__ uint32_t load(const uint32_t* at) const { return kShared ? *at : __ldcg(at); }
};

// The k best of batch item b by a CTA.
template <typename T, bool kVec, bool kShared>
__device__ __forceinline__ void merge_item(const MergeParams& mp, MergeShared& sh, u64* entries, const Notes<kShared> notes,
                                           const int b) {
  const ScanParams& p = mp.scan;
  const MergeView view{mp, sh, entries, b};
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, W = p.W;
  const int per_beam = p.entries + 1;
  if (threadIdx.x == 0) sh.entries_listed = sh.values_listed = sh.hits = 0;
  if (threadIdx.x < kBmGroups) sh.group[threadIdx.x] = 0;
  __syncthreads();

  // 1. a warp per beam: the sums joined, the scores of its blocks' maxima
  bool waited = kShared;
  for (int w = warp; w < W; w += kBmWarps) {
    const float sc = p.scores[b * W + w];
    const int alive = !(sc > -INFINITY) ? 0 : p.finished && p.finished[b * W + w] ? 2 : 1;
    if (!waited) pdl_wait();
    waited = true;
    u64* entry = view.entry + w * per_beam;
    double lse = 0.0;
    if (alive == 1) {
      const float2* seg = notes.seg + w * p.segs;
      const uint32_t* top = notes.top + w * p.entries;
      const float2 none = make_float2(-INFINITY, 0.f);
      const float2 q0 = lane < p.segs ? notes.load(seg + lane) : none;
      uint32_t o[4];  // on their way while the sums are joined
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = lane + 32 * i < p.entries ? notes.load(top + lane + 32 * i) : 0u;
      float m = q0.x;
      for (int i = lane + 32; i < p.segs; i += 32) m = fmaxf(m, notes.load(seg + i).x);
      m = warp_max(m);
      if (m > -INFINITY) {
        float s = q0.y * exp2_fast((q0.x - m) * kLog2e);
        for (int i = lane + 32; i < p.segs; i += 32) {
          const float2 q = notes.load(seg + i);
          s += q.y * exp2_fast((q.x - m) * kLog2e);
        }
        s = warp_sum(s);
        lse = (double)m + log((double)s);
      }
      for (int e0 = 0; e0 < p.entries; e0 += 128) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int e = e0 + lane + 32 * i;
          if (e < p.entries) {
            const u64 q = o[i] ? order_f64((double)sc + ((double)unorder_f32(o[i]) - lse)) : 0ull;
            entry[e] = q;
            put_group(sh, w * per_beam + e, q);
          }
          if (e + 128 < p.entries) o[i] = notes.load(top + e + 128);
        }
      }
    } else {
      for (int e = lane; e < p.entries; e += 32) entry[e] = 0;
    }
    if (lane == 0) {
      sh.score[w] = (double)sc;
      sh.alive[w] = alive;
      sh.lse[w] = lse;
      const u64 q = alive == 2 ? order_f64((double)sc) : 0ull;
      entry[p.entries] = q;
      put_group(sh, w * per_beam + p.entries, q);
    }
  }
  if (!waited) pdl_wait();
  __syncthreads();

  // 2. the k best blocks
  const uint32_t cut = group_threshold(sh, mp.k);
  for (int i = threadIdx.x; i < W * per_beam; i += kBmThreads) {
    const u64 q = view.entry[i];
    if (q && (uint32_t)(q >> 32) >= cut && !view.over(&sh.entries_listed)) view.append(&sh.entries_listed, q, i);
  }
  __syncthreads();
  if (sh.entries_listed > kBmCap) entries_again(view);
  if (sh.entries_listed > kBmRank) shrink_list(view, &sh.entries_listed);
  const int listed = sh.entries_listed, blocks = min(listed, mp.k);
  rank_list(sh, listed, mp.k, [&](int rank, u64 key, u64 id) {
    sh.best_key[rank] = key;
    sh.best_id[rank] = (int)id;
  });
  __syncthreads();

  // 3. their values that reach the k-th block's largest score
  u64 least = blocks == mp.k ? sh.best_key[blocks - 1] : 1ull;
  auto load_chosen = [&](int i, RawTile<T>& q, int& w, int64_t& at) {
    const bool has = find_chosen(view, i, w, at);
    if (has) load_block<T, kVec>(view.row<T>(w), at, (int)min((int64_t)kBsBlock, p.V - at), q);
    return has;
  };
  // Where there are fewer blocks than candidates (a small vocabulary, a heavy mask), or too many values
  // reach that score (few blocks, large values next to each other), a threshold from the lanes'
  // maxima: at 28 x 11 x 1429 with 15 candidates 1379 -> 18 us.
  for (bool refine = blocks < mp.k;; refine = true) {
    if (refine) {
      __syncthreads();
      if (threadIdx.x < kBmGroups) sh.group[threadIdx.x] = 0;
      if (threadIdx.x == 0) sh.values_listed = sh.hits = 0;
      __syncthreads();
      for (int i = warp; i < blocks * p.run; i += kBmWarps) {
        RawTile<T> q;
        int w;
        int64_t at;
        if (!load_chosen(i, q, w, at)) {
          if (sh.alive[w] == 2 && lane == 0 && i % p.run == 0) put_group(sh, i * 32, sh.best_key[i / p.run]);
          continue;
        }
        const uint32_t o = order_clean(raw_max<T>(q));
        put_group(sh, i * 32 + lane, o ? view.score_key(w, unorder_f32(o)) : 0ull);
      }
      __syncthreads();
      least = max(least, (u64)group_threshold(sh, mp.k) << 32);
    }
    for (int i = warp; i < blocks * p.run; i += kBmWarps) {
      RawTile<T> q;
      int w;
      int64_t at;
      if (!load_chosen(i, q, w, at)) {
        if (sh.alive[w] == 2 && lane == 0 && i % p.run == 0)
          view.append(&sh.values_listed, sh.best_key[i / p.run], view.candidate(w, mp.pad));
        continue;
      }
      const int left = (int)min((int64_t)kBsBlock, p.V - at);
      // the lowest logit of this beam that can reach `least`, with room for rounding
      const double lo = unorder_f64(least) - sh.score[w] + sh.lse[w];
      const float thr = least > 1ull && isfinite(lo)
                            ? (float)(lo - 1e-6 * (fabs(lo) + fabs(sh.score[w]) + fabs(sh.lse[w]) + 1.0))
                            : -kFltMax;
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < kBsPer; ++e)
        if (clean(raw_value<T>(q, e)) >= thr) hits |= 1u << e;
      const int n = __reduce_add_sync(0xffffffffu, __popc(hits));
      int before = 0;
      if (lane == 0 && n > 0) before = atomicAdd(&sh.hits, n);
      // too many: another threshold, or, where that was it, the search that needs no list
      if (__shfl_sync(0xffffffffu, before, 0) + n > (refine ? kBmMany : kBmRank)) continue;
      while (hits) {  // few
        const int at_e = __ffs(hits) - 1;
        hits &= hits - 1;
        uint32_t word = q.r[0];
#pragma unroll
        for (int e = 1; e < kBsPer * (int)sizeof(T) / 4; ++e)
          if (e == at_e * (int)sizeof(T) / 4) word = q.r[e];
        const u64 key = view.score_key(w, clean(raw_value<T>(word, at_e)));
        if (key >= least)
          view.append(&sh.values_listed, key, view.candidate(w, at + block_pos<T, kVec>(at_e, left >= kBsBlock)));
      }
    }
    __syncthreads();
    if (refine || sh.hits <= kBmRank) break;
  }
  if (sh.hits > kBmMany) values_again<T, kVec>(view, blocks, least);
  if (sh.values_listed > kBmRank) shrink_list(view, &sh.values_listed);
  const int n = sh.values_listed;
  const int64_t out = (int64_t)b * mp.k;
  rank_list(sh, n, mp.k, [&](int rank, u64 key, u64 id) {
    mp.out_scores[out + rank] = (float)unorder_f64(key);
    const u64 w = id / (unsigned)p.V;
    mp.out_tokens[out + rank] = (int64_t)(id - w * (unsigned)p.V);
    mp.out_parents[out + rank] = (int64_t)w;
  });
  for (int r = n + threadIdx.x; r < mp.k; r += kBmThreads) {  // too few candidates
    mp.out_scores[out + r] = -INFINITY;
    mp.out_tokens[out + r] = -1;
    mp.out_parents[out + r] = 0;
  }
}

template <typename T, bool kVec>
__global__ void __launch_bounds__(kBmThreads, 1) beam_merge_kernel(const __grid_constant__ MergeParams mp) {
  extern __shared__ __align__(16) unsigned char bm_smem[];
  const ScanParams& p = mp.scan;
  const int64_t row = (int64_t)blockIdx.x * p.W;
  merge_item<T, kVec, false>(mp, *reinterpret_cast<MergeShared*>(bm_smem),
                             reinterpret_cast<u64*>(bm_smem + sizeof(MergeShared)),
                             Notes<false>{p.seg + row * p.segs, p.top + row * p.entries}, blockIdx.x);
}

// Both in one launch: a cluster of CTAs scans a batch item, its first CTA, in whose shared
// memory all leave their notes, merges.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kBmThreads, 1) beam_select_kernel(const __grid_constant__ MergeParams mp, int ctas) {
  extern __shared__ __align__(16) unsigned char bm_smem[];
  const ScanParams& p = mp.scan;
  const int b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas, lane = threadIdx.x & 31;
  u64* entries = reinterpret_cast<u64*>(bm_smem + sizeof(MergeShared));
  float2* seg = reinterpret_cast<float2*>(entries + p.W * (p.entries + 1));
  uint32_t* top = reinterpret_cast<uint32_t*>(seg + p.W * p.segs);
  cluster_arrive();
  pdl_wait();
  const uint32_t seg_at = in_cluster_cta(smem_u32(seg), 0), top_at = in_cluster_cta(smem_u32(top), 0);
  cluster_wait();  // the first CTA is there
  for (int u = rank * kBmWarps + (threadIdx.x >> 5); u < p.W * p.segs; u += ctas * kBmWarps) {
    const int w = u / p.segs;
    scan_piece<T, kVec>(
        p, b * p.W + w, u - w * p.segs,
        [&](int e, uint32_t o) {
          if (lane == 0) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(top_at + (w * p.entries + e) * 4), "r"(o) : "memory");
        },
        [&](float m, float s) {
          if (lane == 0)
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(seg_at + u * 8), "f"(m), "f"(s) : "memory");
        });
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank == 0) merge_item<T, kVec, true>(mp, *reinterpret_cast<MergeShared*>(bm_smem), entries, Notes<true>{seg, top}, b);
}

constexpr int kSelectMaxSmem = 96 * 1024;
ClusterOnce select_once[6];  // of beam_select_kernel's variants: dtype * 2 + kVec

struct BeamPlan {
  int segs = 1, seg_blocks = 1, entries = 1, run = 1;
  int cluster = 0;  // CTAs of a batch item in one launch; 0: two launches
  double cost = 0;  // blocks that the slowest warp goes through
  size_t top_off = 0, bytes = 0, merge_smem = 0;
};

constexpr int kMergeMaxSmem = (int)sizeof(MergeShared) + (kBsMaxBeams * kBsMaxEntries + kBsMaxBeams) * 8;

// Blocks per warp: the split that takes the fewest rounds of blocks for so many warps; a
// warp costs about half a block beside its blocks.
BeamPlan beam_split(int rows, int W, int V, int64_t warps) {
  BeamPlan pl;
  const int blocks = (int)(((int64_t)V + kBsBlock - 1) / kBsBlock);
  pl.run = (blocks + kBsMaxEntries - 1) / kBsMaxEntries;
  pl.entries = (blocks + pl.run - 1) / pl.run;
  pl.cost = 1e30;
  for (int e = 1; e <= pl.entries; ++e) {  // entries per warp
    const int segs = (pl.entries + e - 1) / e;
    const int64_t rounds = ((int64_t)rows * segs + warps - 1) / warps;
    const double cost = (double)rounds * (e * pl.run + 0.5);
    if (cost < pl.cost) {
      pl.cost = cost;
      pl.seg_blocks = e * pl.run;
      pl.segs = segs;
    }
    if (rounds == 1) break;  // longer pieces take no fewer rounds
  }
  pl.merge_smem = sizeof(MergeShared) + ((size_t)W * pl.entries + W) * 8;
  return pl;
}

int clusters_at_once(int ctas, const DeviceInfo& di) {
  static ClustersAtOnce known;
  constexpr auto kern = beam_select_kernel<float, true>;
  if (select_once[2 * NSM_F32 + 1].set(kern, kSelectMaxSmem, di.device) != cudaSuccess) return -1;
  return known.get(kern, kBmThreads, kSelectMaxSmem, ctas, di);
}

// One launch where clusters of up to 16 CTAs with 32 warps each fit the GPU at once and take
// at most a block more per warp than all SMs would.
BeamPlan beam_plan(int batch, int W, int V, const DeviceInfo& di) {
  BeamPlan pl = beam_split(batch * W, W, V, 32LL * di.sm_count), best;
  for (int ctas = 16; ctas >= 1; ctas /= 2) {
    if (ctas * batch > di.sm_count || clusters_at_once(ctas, di) < batch) continue;
    BeamPlan one = beam_split(W, W, V, (int64_t)ctas * kBmWarps);
    one.merge_smem += (size_t)W * one.segs * sizeof(float2) + (size_t)W * one.entries * 4;
    if (one.cost <= pl.cost + 1.0 && one.merge_smem <= kSelectMaxSmem && (best.cluster == 0 || one.cost <= best.cost)) {
      best = one;
      best.cluster = ctas;
    }
  }
  if (best.cluster > 0) return best;
  pl.top_off = align_up((size_t)batch * W * pl.segs * sizeof(float2), 256);
  pl.bytes = pl.top_off + (size_t)batch * W * pl.entries * 4;
  return pl;
}

bool beam_size_ok(int batch, int beams, int vocab, int k) {
  return batch > 0 && beams > 0 && beams <= kBsMaxBeams && vocab > 0 && vocab <= (1 << 30) && k > 0 && k <= kBsMaxK &&
         (int64_t)batch * beams <= (1 << 20);
}

struct BeamFns {
  void (*scan)(ScanParams);
  void (*merge)(MergeParams);
  void (*both)(MergeParams, int);
};

template <typename T>
BeamFns beam_pick(bool vec) {
  if (vec) return {beam_scan_kernel<T, true>, beam_merge_kernel<T, true>, beam_select_kernel<T, true>};
  return {beam_scan_kernel<T, false>, beam_merge_kernel<T, false>, beam_select_kernel<T, false>};
}

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
  return beam_plan(batch, beams, vocab, di).bytes;
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
  const BeamPlan pl = beam_plan(batch, beams, vocab, di);
  NSM_REQUIRE(pl.bytes == 0 || (((uintptr_t)workspace & 255) == 0 && workspace_bytes >= pl.bytes), NSM_ERR_WORKSPACE,
              "nsm_beam_select: workspace misaligned or too small (nsm_beam_select_workspace_bytes)");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto* ws = static_cast<unsigned char*>(workspace);
  MergeParams mp;
  ScanParams& sp = mp.scan;
  sp.logits = logits;
  sp.batch_stride = batch_stride;
  sp.beam_stride = beam_stride;
  sp.scores = scores;
  sp.finished = finished;
  sp.rows = rows;
  sp.W = beams;
  sp.V = vocab;
  sp.segs = pl.segs;
  sp.seg_blocks = pl.seg_blocks;
  sp.entries = pl.entries;
  sp.run = pl.run;
  sp.seg = reinterpret_cast<float2*>(ws);
  sp.top = reinterpret_cast<uint32_t*>(ws + pl.top_off);
  mp.k = candidates;
  mp.pad = pad_token;
  mp.out_scores = out_scores;
  mp.out_tokens = out_tokens;
  mp.out_parents = out_parents;
  // 16-byte loads when every row starts on 16 bytes, else one value per lane
  const bool vec = (((uintptr_t)logits | (uintptr_t)(batch_stride * es) | (uintptr_t)(beam_stride * es)) & 15) == 0;
  const BeamFns f = logits_dtype == NSM_F32   ? beam_pick<float>(vec)
                    : logits_dtype == NSM_F16 ? beam_pick<__half>(vec)
                                              : beam_pick<__nv_bfloat16>(vec);
  if (pl.cluster > 0) {
    NSM_CHECK_CUDA(select_once[logits_dtype * 2 + vec].set(f.both, kSelectMaxSmem, di.device));
    NSM_CHECK_CUDA(launch_pdl_cluster(f.both, dim3(batch * pl.cluster), dim3(kBmThreads), pl.merge_smem, s, pl.cluster, mp,
                                      pl.cluster));
    return NSM_OK;
  }
  const int64_t warps = (int64_t)rows * pl.segs;
  NSM_CHECK_CUDA(launch_pdl(f.scan, dim3((unsigned)((warps + kBsWarps - 1) / kBsWarps)), dim3(kBsThreads), 0, s, sp));
  static SmemOnce once[6];
  NSM_CHECK_CUDA(once[logits_dtype * 2 + vec].set(f.merge, kMergeMaxSmem, di.device));
  NSM_CHECK_CUDA(launch_pdl(f.merge, dim3(batch), dim3(kBmThreads), pl.merge_smem, s, mp));
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
