// sampling.cu — the next token of every request from its logits: temperature, top-k, top-p,
// min-p and a given uniform number, each request with its own settings, in one launch.
//
// Order of a row: value descending, index ascending. With m = max l,
//   w_i = exp((l_i - m) / T) in fp32,   W_i = floor(w_i 2^40) in int64,
// so every sum below is a whole number: it does not depend on the order of summation, on the
// split of the row over CTAs or on the other rows of the batch, and a token is the same
// wherever it is drawn.
//   top-k   the first k of the order;
//   top-p   of those, the shortest prefix whose sum reaches ceil(p * sum of those);
//   min-p   w_i >= min_p;
//   token   the first index whose running sum over the kept (in index order) exceeds
//           floor(u * sum of the kept);  logprob = (l - m) / T - log(sum 2^-40).
// What is kept is a prefix of the order, i.e. one bound (value, index), found without sorting
// the row:
//   top-k   a histogram of the threads' largest logits, in 1024 linear buckets of (m - l) / T (1/32
//           wide), names a bucket that k of them reach: all values up to it, few more than k, are sorted;
//   top-p   the weights replace the logits in shared memory; a sample of them (an eighth, and all
//           heavy ones), in 16 buckets an octave, names a window around the border; the sum above it is exact, and
//           counts in up to 1024 parts of it name three parts, which are sorted, after the exact sum above
//           them (or, where they hold more than kList, are the next window). Slices of up to kWhole
//           values take one exact histogram instead.
// Few values go through the histograms: an addition to shared memory costs a warp more than all
// arithmetic of a pass.
// Where more than kList values are left (many equal ones), or the border is not in the window,
// find_bound refines exact histograms over the row's bits, read again from memory.
//
// Measured on a B200: 200 x 128000 fp32 greedy 40 us, unfiltered 66, top-k 50 91, top-p 0.9 196 to 204 (the logits'
// bytes at the copy rate: 15.6); 3 x 50000 bf16 4.4 / 11 / 16 / 26 to 40; 16 x 256 3.0 / 5.6 / 10.3 / 10.3. Bound by
// the chain of cluster barriers and of the first CTA's steps (barriers are the first stall, 43 % of the issue slots are
// used, DRAM is busy for 6 to 18 %), not by bytes or arithmetic. A grid that walks over the rows was slower
// (unfiltered 99): a cluster then waits for its last token before the next row.
//
// A row is split over a cluster of C CTAs that keep their slice of it in shared memory (the
// logits are read from memory once) and merge maxima, histograms and sums through
// distributed shared memory.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <torch/extension.h>

#include <cfloat>

#include "launches.h"

namespace bd {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 256;
constexpr int kWarpsS = kThreads / 32;
constexpr int kBuckets = 1024;
constexpr int kList = 1024;  // values that are sorted
constexpr int kEach = kBuckets / kThreads;  // buckets, and values of the list, of a thread
static_assert(kBuckets == kList, "one count for both");
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 32768;  // logits a CTA can hold
constexpr int kWhole = 8192;      // a slice whose weights all go through one exact histogram
constexpr float kMinusInf = -INFINITY;

struct SampleArgs {
  const void* logits;
  long long row_stride;
  int rows, V, slice;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t* tokens;
  float* logprobs;
};

// With a slice of 64,000 bytes (128,000 tokens over 8 CTAs) three CTAs share an SM.
struct __align__(16) Shared {
  union {
    struct {
      unsigned count[kBuckets];
      unsigned lo[kBuckets], hi[kBuckets];  // a bucket's weight as two words
    };
    u64 list[kList];  // order bits : index, ascending = the order of the row
  };
  float4 warp_estimate[kWarpsS];
  u64 warp_sum[kWarpsS];
  unsigned warp_count[kWarpsS];
  u64 slot[3][kMaxCluster];  // one value per CTA of the cluster; the next exchange uses another row
  float slot_max[kMaxCluster];
  u64 before_count, before_weight, bound;
  unsigned list_n, digit_count;
  int digit, window[2];
};

__device__ __forceinline__ unsigned order_bits(float l) {  // ascending in descending l
  const unsigned b = __float_as_uint(l);
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}
__device__ __forceinline__ float order_value(unsigned o) {
  return __uint_as_float((o & 0x80000000u) ? o : (~o & 0x7fffffffu));
}
__device__ __forceinline__ u64 order_of(float l, int index) { return (u64)order_bits(l) << 32 | (unsigned)index; }

__device__ __forceinline__ u64 fixed40(float w) {  // floor(w 2^40) for 0 <= w <= 1
  const unsigned b = __float_as_uint(w);
  const int s = (int)(b >> 23) - (127 + 23 - 40);
  const u64 m = (b & 0x7fffffu) | 0x800000u;
  return s >= 0 ? (s <= 17 ? m << s : 0ull) : (s > -24 ? m >> -s : 0ull);
}

// Sums of fixed40(w) in 32-bit halves: w is split at 2^-17 by adding and taking away 1.5 * 2^6, the rest is
// floored at 2^-40 by adding 1.5 * 2^-17 rounded down; both sums leave their bits in the low mantissa. Six
// single-rate instructions a value against about twenty for 64-bit shifts and adds.
struct WeightSum {
  // At most 511 values: each puts a signed rest of up to 2^22 units into the 32 bits of `low`.
  unsigned high = 0, low = 0, n = 0;
  __device__ __forceinline__ void add(float w) {
    const float t = __fadd_rn(w, 96.f);
    const float rest = __fsub_rn(w, __fsub_rn(t, 96.f));
    high += __float_as_uint(t);
    low += __float_as_uint(__fadd_rd(rest, 1.1444091796875e-05f));
  }
  __device__ __forceinline__ u64 total() const {
    return ((u64)(high - n * 0x42c00000u) << 23) + (u64)(long long)(int)(low - n * 0x37400000u);
  }
};

// A thread sums its share of a slice (a warp's run is a whole number of 256 values), twice where values equal the border.
static_assert(2 * (kMaxSlice / kThreads) < 512, "WeightSum holds a thread's values");

struct Row {
  float top, inv_t, per_bucket;
  __device__ __forceinline__ float z(float l) const { return l == top ? 0.f : __fmul_rn(__fsub_rn(l, top), inv_t); }
  __device__ __forceinline__ float w(float l) const { return expf(z(l)); }
  __device__ __forceinline__ u64 weight(float l) const { return l == kMinusInf ? 0ull : fixed40(w(l)); }
  // linear in (top - l) / T; a NaN product (0 * inf: l is the top) is bucket 0
  __device__ __forceinline__ int bucket(float l) const { return min(kBuckets - 1, (int)((top - l) * per_bucket)); }
};

// 16 buckets an octave of a weight in (2^-40, 1]
__device__ __forceinline__ int weight_bucket(float w) { return (int)((0x3f800000u - __float_as_uint(w)) >> 19); }
constexpr float kOne40 = 9.094947017729282e-13f;  // 2^-40

__device__ __forceinline__ float logit(float x) { return fmaxf(x, kMinusInf) + 0.f; }  // NaN counts as -inf, -0 as 0
__device__ __forceinline__ float logit(__nv_bfloat16 x) { return logit(__bfloat162float(x)); }

__device__ __forceinline__ u64 warp_total(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ u64 warp_inclusive(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

struct Sums {
  u64 count, weight;
};

// Exclusive running sums over the block's threads; `all` gets the totals.
__device__ __forceinline__ Sums block_exclusive(Shared& s, Sums mine, bool weigh, Sums& all) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const u64 ic = warp_inclusive(mine.count, lane), iw = weigh ? warp_inclusive(mine.weight, lane) : 0;
  __syncthreads();
  if (lane == 31) s.warp_count[warp] = (unsigned)ic, s.warp_sum[warp] = iw;
  __syncthreads();
  Sums e{ic - mine.count, iw - mine.weight};
  all = Sums{0, 0};
#pragma unroll
  for (int q = 0; q < kWarpsS; ++q) {
    if (q < warp) e.count += s.warp_count[q], e.weight += s.warp_sum[q];
    all.count += s.warp_count[q], all.weight += s.warp_sum[q];
  }
  return e;
}

// A barrier of the cluster.
__device__ __forceinline__ void sync_all(cg::cluster_group& cluster) {
  if (cluster.num_blocks() == 1)
    __syncthreads();
  else
    cluster.sync();
}

// The sum of one value per thread over the cluster; also a barrier of the cluster. `row`: of slot, another
// one than the last exchange's unless a barrier lies between.
__device__ __forceinline__ u64 cluster_total(Shared& s, int row, u64 mine, u64* before = nullptr) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int lane = threadIdx.x % 32;
  const u64 w = warp_total(mine);
  __syncthreads();
  if (lane == 0) s.warp_sum[threadIdx.x / 32] = w;
  __syncthreads();
  if (threadIdx.x < 32) {
    const u64 block = warp_total(lane < kWarpsS ? s.warp_sum[lane] : 0ull);
    if (lane < C) cluster.map_shared_rank(&s, lane)->slot[row][rank] = block;
  }
  sync_all(cluster);
  u64 total = 0;
  for (int q = 0; q < C; ++q) {
    if (before && q < rank) *before += s.slot[row][q];
    total += s.slot[row][q];
  }
  return total;
}

__device__ __forceinline__ void add_weight(Shared& s, int d, u64 w) {
  const unsigned lo = (unsigned)w, old = atomicAdd(&s.lo[d], lo);
  const unsigned hi = (unsigned)(w >> 32) + (old + lo < old ? 1u : 0u);
  if (hi) atomicAdd(&s.hi[d], hi);
}

__device__ __forceinline__ void clear_histogram(Shared& s, bool weigh) {
  for (int b = threadIdx.x; b < kBuckets; b += kThreads) {
    s.count[b] = 0;
    if (weigh) s.lo[b] = s.hi[b] = 0;
  }
  __syncthreads();
}

// In the first CTA (the others go on to the next barrier): this thread's buckets of the cluster's
// histogram, and their sum.
__device__ __forceinline__ Sums merged(Shared& s, bool weigh, Sums (&b)[kEach]) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks();
  const int at = kEach * threadIdx.x;
#pragma unroll
  for (int k = 0; k < kEach; ++k) b[k] = Sums{0, 0};
#pragma unroll
  for (int q = 0; q < kMaxCluster; ++q) {  // unrolled: the loads of all CTAs are in flight together
    if (q >= C) break;
    const Shared* o = cluster.map_shared_rank(&s, q);
    const uint4 c = *reinterpret_cast<const uint4*>(&o->count[at]);
    b[0].count += c.x, b[1].count += c.y, b[2].count += c.z, b[3].count += c.w;
    if (weigh) {
      const uint4 lo = *reinterpret_cast<const uint4*>(&o->lo[at]), hi = *reinterpret_cast<const uint4*>(&o->hi[at]);
      b[0].weight += (u64)hi.x << 32 | lo.x, b[1].weight += (u64)hi.y << 32 | lo.y;
      b[2].weight += (u64)hi.z << 32 | lo.z, b[3].weight += (u64)hi.w << 32 | lo.w;
    }
  }
  Sums all{0, 0};
#pragma unroll
  for (int k = 0; k < kEach; ++k) all.count += b[k].count, all.weight += b[k].weight;
  return all;
}
static_assert(kEach == 4, "merged reads four buckets a thread");

// In the first CTA: the first bucket after which `most` values or `reach` weight is there, from running
// sums `at`. Told to every CTA by the one thread that has it; digit stays as it was if there is none.
__device__ __forceinline__ void pick(Shared& s, const Sums (&b)[kEach], Sums at, u64 most, u64 reach) {
  cg::cluster_group cluster = cg::this_cluster();
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    if (b[k].count > 0 && at.count < most && at.weight < reach &&
        (at.count + b[k].count >= most || at.weight + b[k].weight >= reach)) {
      for (int q = 0; q < (int)cluster.num_blocks(); ++q) {
        Shared* o = cluster.map_shared_rank(&s, q);
        o->digit = kEach * threadIdx.x + k;
        o->digit_count = (unsigned)min(b[k].count, 0xffffffffull);
        o->before_count = at.count;
        o->before_weight = at.weight;
      }
    }
    at.count += b[k].count;
    at.weight += b[k].weight;
  }
}

__device__ __forceinline__ void push(Shared* first, u64 order) {
  const unsigned at = atomicAdd(&first->list_n, 1u);
  if (at < kList) first->list[at] = order;
}

// Ascending order of up to 256 values of the first CTA's list, a value a thread: each counts the ones before it.
// One broadcast read and four instructions a value, all independent, where a step of a sorting
// network is a chain of shuffles (16 rows of 256 with top-k: 10.1 against 13.4 us).
__device__ void rank_list(Shared& s, int n) {
  const int t = threadIdx.x;
  const u64 mine = t < n ? s.list[t] : ~0ull;
  int before = 0;
  if (t < (n + 31) / 32 * 32) {
#pragma unroll 8
    for (int j = 0; j < n; ++j) before += s.list[j] < mine ? 1 : 0;
  }
  __syncthreads();
  if (t < n) s.list[before] = mine;
  __syncthreads();
}

// Ascending bitonic sort of the first CTA's list, value t + 256 e in register e of thread t: partners in one
// thread and in one warp exchange without shared memory.
__device__ void sort_list(Shared& s, int n) {
  const int t = threadIdx.x;
  int size = 32;
  while (size < n) size <<= 1;
  u64 v[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) v[e] = t + e * kThreads < n ? s.list[t + e * kThreads] : ~0ull;
  auto keep = [&](int e, u64 o, int j, int k) {
    const int i = t + e * kThreads;
    const bool low = ((i & j) == 0) == ((i & k) == 0);  // this place gets the smaller one
    if ((v[e] > o) == low) v[e] = o;
  };
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64 o[kEach];
      if (j >= kThreads) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) o[e] = j == kThreads ? v[e ^ 1] : v[e ^ 2];
#pragma unroll
        for (int e = 0; e < kEach; ++e) keep(e, o[e], j, k);
      } else if (j >= 32) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (e * kThreads < size) s.list[t + e * kThreads] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (e * kThreads < size) keep(e, s.list[(t + e * kThreads) ^ j], j, k);
      } else if (t < size) {  // whole warps
#pragma unroll
        for (int e = 0; e < kEach; ++e)
          if (e * kThreads < size) keep(e, __shfl_xor_sync(0xffffffffu, v[e], j), j, k);
      }
    }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < kEach; ++e)
    if (e * kThreads < size) s.list[t + e * kThreads] = v[e];
  __syncthreads();
}

// After the gather's barrier: the first CTA sorts the list and finds the last value that is kept: fewer
// than `most` values and less than `reach` weight before it, counted from `before`. Where `share` is
// given, reach is that share of the first `most` values' weight. Every CTA gets the bound.
__device__ u64 list_bound(Shared& s, const Row& r, Sums before, u64 most, u64 reach, const float* share) {
  cg::cluster_group cluster = cg::this_cluster();
  if (cluster.block_rank() == 0) {
    const int n = (int)min(s.list_n, (unsigned)kList);
    if (n <= kThreads)
      rank_list(s, n);
    else
      sort_list(s, n);
    Sums v[kEach], all, own{0, 0};
    u64 order[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int i = kEach * threadIdx.x + k;
      order[k] = i < n ? s.list[i] : ~0ull;
      v[k] = Sums{i < n ? 1ull : 0ull, 0};
      if (i < n && (share || reach != ~0ull) && before.count + i < most) v[k].weight = r.weight(order_value((unsigned)(order[k] >> 32)));
      own.count += v[k].count, own.weight += v[k].weight;
    }
    Sums at = block_exclusive(s, own, true, all);
    if (share) {
      const double want = ceil(__dmul_rn(__ull2double_rn(all.weight), (double)*share));
      reach = want > 1.0 ? (u64)want : 1ull;
    }
    at.count += before.count;
    at.weight += before.weight;
    // without a reach the last value is the bound; with one it has to be reached
    const u64 end = reach == ~0ull ? min(most, before.count + n) : most;
    if (threadIdx.x == 0)
      for (int q = 0; q < (int)cluster.num_blocks(); ++q) cluster.map_shared_rank(&s, q)->bound = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      if (v[k].count && at.count < most && at.weight < reach &&
          (at.count + 1 >= end || at.weight + v[k].weight >= reach)) {
        for (int q = 0; q < (int)cluster.num_blocks(); ++q) cluster.map_shared_rank(&s, q)->bound = order[k];
      }
      at.count += v[k].count;
      at.weight += v[k].weight;
    }
  }
  sync_all(cluster);
  return s.bound;
}

// Digits of a value after its linear bucket: ten bits of its order thrice, the last two, its index's ten and ten.
constexpr int kLevels = 7;
__device__ __forceinline__ int digit_of(int level, const Row& r, float l, int index) {
  switch (level) {
    case 0: return r.bucket(l);
    case 1: return (int)(order_bits(l) >> 22);
    case 2: return (int)(order_bits(l) >> 12) & 1023;
    case 3: return (int)(order_bits(l) >> 2) & 1023;
    case 4: return (int)order_bits(l) & 3;
    case 5: return index >> 10;
    default: return index & 1023;
  }
}

// The same bound for any row: exact histograms digit by digit, until at most kList values share all of
// them. Reads the logits from memory. Values after `bound` and of weight zero are not there. Returns
// `bound` if all are kept; `kept_weight` gets the weight of the kept.
template <typename T>
__device__ __noinline__ u64 find_bound(Shared& s, const T* src, int base, int n, const Row& r, u64 bound, u64 most,
                                       u64 reach, u64& kept_weight) {
  cg::cluster_group cluster = cg::this_cluster();
  int path[kLevels];
  Sums before{0, 0};
  int level = 0;
  for (;; ++level) {
    sync_all(cluster);  // what the shared memory held is read
    clear_histogram(s, true);
    if (threadIdx.x == 0) s.list_n = 0, s.digit = -1;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const float l = logit(src[i]);
      bool on = order_of(l, base + i) <= bound;
      for (int q = 0; q < level; ++q) on = on && digit_of(q, r, l, base + i) == path[q];
      const u64 w = on ? r.weight(l) : 0ull;
      if (w) {
        const int d = digit_of(level, r, l, base + i);
        atomicAdd(&s.count[d], 1u);
        add_weight(s, d, w);
      }
    }
    sync_all(cluster);
    if (cluster.block_rank() == 0) {
      Sums b[kEach], all;
      const Sums at = block_exclusive(s, merged(s, true, b), true, all);
      pick(s, b, Sums{at.count + before.count, at.weight + before.weight}, most, reach);
    }
    sync_all(cluster);
    if (s.digit < 0) {  // neither is reached: all are kept
      u64 mine = 0;
      for (int i = threadIdx.x; i < n; i += kThreads)
        if (order_of(logit(src[i]), base + i) <= bound) mine += r.weight(logit(src[i]));
      kept_weight = cluster_total(s, 1, mine);
      return bound;
    }
    path[level] = s.digit;
    before = Sums{s.before_count, s.before_weight};
    if (s.digit_count <= kList || level + 1 == kLevels) break;
  }
  Shared* first = cluster.map_shared_rank(&s, 0);
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float l = logit(src[i]);
    bool on = order_of(l, base + i) <= bound;
    for (int q = 0; q <= level; ++q) on = on && digit_of(q, r, l, base + i) == path[q];
    if (on && r.weight(l)) push(first, order_of(l, base + i));
  }
  sync_all(cluster);
  bound = list_bound(s, r, before, most, reach, nullptr);
  // the weight of the kept: of what lies before the bound and of itself
  u64 mine = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const float l = logit(src[i]);
    if (order_of(l, base + i) <= bound) mine += r.weight(l);
  }
  kept_weight = cluster_total(s, 1, mine);
  return bound;
}

__device__ __forceinline__ u64 share_of(u64 total, float p) {
  const double want = ceil(__dmul_rn(__ull2double_rn(total), (double)p));
  return want > 1.0 ? (u64)want : 1ull;
}

// top-k (and, inside it, top-p). `own`: the largest logit this thread has read.
template <typename T>
__device__ __forceinline__ u64 bound_of_k(Shared& s, const float* x, const T* src, int base, int n, const Row& r, int k,
                                          const float* p, float own) {
  cg::cluster_group cluster = cg::this_cluster();
  clear_histogram(s, false);
  if (threadIdx.x == 0) s.list_n = 0, s.digit = -1;
  // the last bucket holds weights of zero only: 2^-40 is (top - l) / T = 27.7 of 32
  const int b0 = r.bucket(own);
  if (b0 < kBuckets - 1) atomicAdd(&s.count[b0], 1u);
  sync_all(cluster);
  if (cluster.block_rank() == 0) {
    Sums b[kEach], all;
    const Sums at = block_exclusive(s, merged(s, false, b), false, all);
    pick(s, b, at, (u64)k, ~0ull);
  }
  sync_all(cluster);
  const int last = s.digit;
  bool listed = last >= 0;  // else fewer than k threads have a value
  if (listed) {
    Shared* first = cluster.map_shared_rank(&s, 0);
    const float4* x4 = reinterpret_cast<const float4*>(x);
    const int n4 = (n + 3) / 4;
#pragma unroll 2
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const float4 l = x4[i];
      if (r.bucket(fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w))) > last) continue;
      const float v[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (r.bucket(v[q]) <= last) push(first, order_of(v[q], base + 4 * i + q));
    }
    sync_all(cluster);
    listed = first->list_n <= kList;
  }
  if (listed) return list_bound(s, r, Sums{0, 0}, (u64)k, ~0ull, p);
  u64 kept = 0;
  u64 bound = find_bound(s, src, base, n, r, ~0ull, (u64)k, ~0ull, kept);
  if (p) {
    const u64 reach = share_of(kept, *p);
    if (reach < kept) bound = find_bound(s, src, base, n, r, bound, ~0ull, reach, kept);
  }
  return bound;
}

// top-p alone; replaces the logits in x by their weights w
template <typename T>
__device__ __forceinline__ u64 bound_of_p(Shared& s, float* x, const T* src, int base, int n, int slice, const Row& r,
                                          float p) {
  cg::cluster_group cluster = cg::this_cluster();
  const bool whole = slice <= kWhole;
  clear_histogram(s, whole);
  if (threadIdx.x == 0) s.list_n = 0, s.digit = -1;
  float4* x4 = reinterpret_cast<float4*>(x);
  const int n4 = (n + 3) / 4;
  WeightSum sum;
#pragma unroll 2
  for (int i = threadIdx.x; i < n4; i += kThreads) {
    const float4 l = x4[i];
    const float4 w = make_float4(r.w(l.x), r.w(l.y), r.w(l.z), r.w(l.w));
    x4[i] = w;
    sum.n += 4;
    const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      sum.add(v[q]);
      if (whole && v[q] >= kOne40) {
        atomicAdd(&s.count[weight_bucket(v[q])], 1u);
        add_weight(s, weight_bucket(v[q]), fixed40(v[q]));
      }
    }
  }
  const u64 total = cluster_total(s, 1, sum.total());
  const u64 reach = share_of(total, p);
  if (reach >= total) return ~0ull;
  Shared* first = cluster.map_shared_rank(&s, 0);
  int w0 = 0, wide = 1;  // the window: its first bucket, and their number
  if (whole) {
    if (cluster.block_rank() == 0) {
      Sums b[kEach], all;
      const Sums at = block_exclusive(s, merged(s, true, b), true, all);
      pick(s, b, at, ~0ull, reach);
    }
    sync_all(cluster);
    w0 = s.digit;
    if (s.digit_count <= kList) {
      const Sums before{0, s.before_weight};
      for (int i = threadIdx.x; i < n4; i += kThreads) {
        const float4 w = x4[i];
        const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (weight_bucket(v[q]) == w0 && v[q] >= kOne40) push(first, order_of(logit(src[4 * i + q]), base + 4 * i + q));
      }
      sync_all(cluster);
      return list_bound(s, r, before, ~0ull, reach, nullptr);
    }
  } else {
    // the window from a sample: every weight above total / 16384, and each thread's first eight for the rest
    const float heavy = __fmul_rn(__ull2float_rn(total), kOne40 / 16384.f);
    const unsigned share = 16u * (unsigned)n4 / (unsigned)max(1, min(n4, 2 * kThreads));
    if (threadIdx.x == 0) s.window[0] = 0, s.window[1] = weight_bucket(kOne40);
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const float4 w = x4[i];
      if (i >= 2 * kThreads && fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) < heavy) continue;
      const float v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (v[q] >= kOne40 && (i < 2 * kThreads || v[q] >= heavy))
          atomicAdd(&s.count[weight_bucket(v[q])], v[q] >= heavy ? 16u : share);
    }
    sync_all(cluster);
    if (cluster.block_rank() == 0) {
      // A bucket's weight is near its count times its middle. The window: 3.5 deviations of the sampled part (a
      // sampled weight w stands for share / 16 like it: share / 16 w^2 each), half a bucket's width for
      // the heavy ones, and 0.2 %. fp32: a window that misses the border is found out.
      Sums b[kEach];
      merged(s, false, b);
      float w[kEach], sum = 0.f, spread = 0.f, big = 0.f;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const unsigned below = ((unsigned)(kEach * threadIdx.x + k) << 19) + (1u << 18);
        const float mid = below < 0x3f800000u ? __uint_as_float(0x3f800000u - below) : 0.f;
        w[k] = mid * (float)(unsigned)b[k].count * 0.0625f;
        sum += w[k];
        spread += mid < heavy ? w[k] * mid * (float)share * 0.0625f : 0.f;
        big += mid < heavy ? 0.f : w[k];
      }
      const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
      float run = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float t = __shfl_up_sync(0xffffffffu, run, o);
        run += lane >= o ? t : 0.f;
        spread += __shfl_xor_sync(0xffffffffu, spread, o);
        big += __shfl_xor_sync(0xffffffffu, big, o);
      }
      if (lane == 31) s.warp_estimate[warp] = make_float4(run, spread, big, 0.f);
      __syncthreads();
      float at = run - sum, all = 0.f;
      spread = 0.0625f, big = 0.f;
#pragma unroll
      for (int q = 0; q < kWarpsS; ++q) {
        const float4 e = s.warp_estimate[q];
        at += q < warp ? e.x : 0.f;
        all += e.x, spread += e.y, big += e.z;
      }
      const float near = __ull2float_rn(reach) / __ull2float_rn(total) * all;
      const float margin = (share > 16u ? 3.5f * sqrtf(spread) : 0.f) + big * 0.03125f + all * 0.002f;
      const float lo = fmaxf(near - margin, 0.f), hi = fminf(near + margin, all * 0.99999f);
      // the first bucket that reaches lo, and the first that reaches hi
      int opens = -1, ends = -1;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        if (b[k].count > 0) {
          if (at <= lo && at + w[k] > lo) opens = kEach * threadIdx.x + k;
          if (at < hi && at + w[k] >= hi) ends = kEach * threadIdx.x + k;
        }
        at += w[k];
      }
      for (int q = 0; q < (int)cluster.num_blocks(); ++q) {
        if (opens >= 0) cluster.map_shared_rank(&s, q)->window[0] = opens;
        if (ends >= 0) cluster.map_shared_rank(&s, q)->window[1] = ends;
      }
    }
    sync_all(cluster);
    w0 = s.window[0], wide = max(1, s.window[1] - w0 + 1);
  }
  __syncthreads();
  unsigned head = 0x3f800000u - ((unsigned)w0 << 19);  // bits of the largest weight in the window
  unsigned span = (unsigned)wide << 19;
  int shift = 9 + (wide > 1 ? 32 - __clz(wide - 1) : 0);  // of a part's width: 1024 parts at most
  for (;;) {
    clear_histogram(s, false);
    if (threadIdx.x == 0) s.list_n = 0, s.digit = -1;
    sum = WeightSum();
#pragma unroll 2
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const float4 w = x4[i];
      const float v[4] = {w.x, w.y, w.z, w.w};
      sum.n += 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned under = head - __float_as_uint(v[q]);  // wraps for what is above
        sum.add((int)under < 0 ? v[q] : 0.f);
        if (under < span && v[q] >= kOne40) atomicAdd(&s.count[under >> shift], 1u);
      }
    }
    const u64 above = cluster_total(s, 2, sum.total());
    if (above >= reach) break;
    // counts times the parts' middles miss the border by one part at most
    if (cluster.block_rank() == 0) {
      Sums b[kEach], all, own{0, 0};
      merged(s, false, b);
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const unsigned below = ((unsigned)(kEach * threadIdx.x + k) << shift) + (1u << shift) / 2;
        b[k].weight = below < head ? b[k].count * fixed40(__uint_as_float(head - below)) : 0ull;
        own.count += b[k].count, own.weight += b[k].weight;
      }
      const Sums at = block_exclusive(s, own, true, all);
      pick(s, b, Sums{at.count, at.weight + above}, ~0ull, min(reach, above + all.weight));
    }
    sync_all(cluster);
    const int part = max(s.digit, 1) - 1;  // the first of three parts that are sorted
    sum = WeightSum();
#pragma unroll 2
    for (int i = threadIdx.x; i < n4; i += kThreads) {
      const float4 w = x4[i];
      const float v[4] = {w.x, w.y, w.z, w.w};
      sum.n += 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int at = (int)(head - __float_as_uint(v[q])) >> shift;  // its part; negative for what is above
        sum.add(at < part ? v[q] : 0.f);
        if (at >= part && at < part + 3 && v[q] >= kOne40) push(first, order_of(logit(src[4 * i + q]), base + 4 * i + q));
      }
    }
    const u64 before = cluster_total(s, 1, sum.total());
    if (s.digit < 0 || before >= reach) break;
    const unsigned listed = first->list_n;
    if (listed <= kList) {
      const u64 bound = list_bound(s, r, Sums{0, before}, ~0ull, reach, nullptr);
      if (bound) return bound;
      break;  // the border is not in the list
    }
    if (shift == 0) break;  // equal weights
    head -= (unsigned)part << shift;  // too many: the three parts are the next window
    span = 3u << shift;
    shift = max(shift - 8, 0);
    sync_all(cluster);  // list_n is read
  }
  u64 kept;
  return find_bound(s, src, base, n, r, ~0ull, ~0ull, reach, kept);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) float x[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int base = min(rank * a.slice, a.V), n = min(a.slice, a.V - base);
  cluster.barrier_arrive();  // waited for before the first access to another CTA's memory
  const int row = blockIdx.x / C;
  const T* src = static_cast<const T*>(a.logits) + (long long)row * a.row_stride + base;
  const float temperature = a.temperature ? a.temperature[row] : a.temperature0;
  const int k = a.top_k ? a.top_k[row] : a.top_k0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0;
  const float least = fminf(a.min_p ? a.min_p[row] : a.min_p0, 1.f);
  const float u = a.u[row];

  // ---- the slice, and the row's maximum
  float top = kMinusInf;
  constexpr int VEC = 16 / sizeof(T);
  const int nv = reinterpret_cast<uintptr_t>(src) % 16 == 0 ? n / VEC : 0;
  const uint4* src4 = reinterpret_cast<const uint4*>(src);
  auto take = [&](const uint4& raw, int v) {
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 l = make_float4(logit(t[e]), logit(t[e + 1]), logit(t[e + 2]), logit(t[e + 3]));
      top = fmaxf(fmaxf(top, fmaxf(l.x, l.y)), fmaxf(l.z, l.w));
      *reinterpret_cast<float4*>(x + v * VEC + e) = l;
    }
  };
  int v = tid;
  for (; v + 7 * kThreads < nv; v += 8 * kThreads) {
    uint4 raw[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) raw[q] = __ldcs(src4 + v + q * kThreads);
#pragma unroll
    for (int q = 0; q < 8; ++q) take(raw[q], v + q * kThreads);
  }
#pragma unroll 3
  for (; v < nv; v += kThreads) take(__ldcs(src4 + v), v);
#pragma unroll 4
  for (int i = nv * VEC + tid; i < n; i += kThreads) {
    const float l = logit(src[i]);
    x[i] = l;
    top = fmaxf(top, l);
  }
  if (tid < 3 && n + tid < (n + 3) / 4 * 4) x[n + tid] = kMinusInf;  // the passes read whole float4
  const float own = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.warp_sum[warp] = __float_as_uint(top);
  __syncthreads();
  cluster.barrier_wait();
  if (tid < C) {
    top = kMinusInf;
    for (int q = 0; q < kWarpsS; ++q) top = fmaxf(top, __uint_as_float((unsigned)s.warp_sum[q]));
    cluster.map_shared_rank(&s, tid)->slot_max[rank] = top;
  }
  sync_all(cluster);
  top = s.slot_max[0];
  for (int q = 1; q < C; ++q) top = fmaxf(top, s.slot_max[q]);

  if (top == kMinusInf) {  // nothing to draw from
    if (rank == 0 && tid == 0) a.tokens[row] = -1, a.logprobs[row] = kMinusInf;
    return;
  }
  if (!(temperature > 0.f)) {  // the first maximum
    int first = 0x7fffffff;
    const float4* x4 = reinterpret_cast<const float4*>(x);
    for (int i = tid; i < (n + 3) / 4; i += kThreads) {
      const float4 l = x4[i];
      if (fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)) == top) {
        first = min(first, base + 4 * i + (l.x == top ? 0 : l.y == top ? 1 : l.z == top ? 2 : 3));
        break;
      }
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.warp_count[warp] = (unsigned)first;
    __syncthreads();
    if (tid == 0) {
      for (int q = 0; q < kWarpsS; ++q) first = min(first, (int)s.warp_count[q]);
      cluster.map_shared_rank(&s, 0)->slot[2][rank] = (unsigned)first;
    }
    sync_all(cluster);
    if (rank == 0 && tid == 0) {
      for (int q = 0; q < C; ++q) first = min(first, (int)s.slot[2][q]);
      a.tokens[row] = first;
      a.logprobs[row] = 0.f;
    }
    return;
  }
  Row r;
  r.top = top;
  r.inv_t = __fdiv_rn(1.f, fminf(temperature, FLT_MAX));  // never 0, which would make a weight of -inf * 0
  r.per_bucket = r.inv_t * 32.f;
  const bool use_k = k > 0 && k < a.V, use_p = p < 1.f;

  u64 bound = ~0ull;
  if (a.V <= kList && (use_k || use_p)) {  // a short row (in one CTA) is the list
    for (int i = tid; i < n; i += kThreads) s.list[i] = order_of(x[i], i);
    if (tid == 0) s.list_n = n;
    __syncthreads();
    bound = list_bound(s, r, Sums{0, 0}, use_k ? (u64)k : ~0ull, ~0ull, use_p ? &p : nullptr);
  } else if (use_k)
    bound = bound_of_k(s, x, src, base, n, r, k, use_p ? &p : nullptr, own);
  else if (use_p)
    bound = bound_of_p(s, x, src, base, n, a.slice, r, p);
  const bool weights = !use_k && use_p && a.V > kList;  // x holds weights

  // ---- sums of the kept weights: warp w owns a run of the slice
  const float last = bound == ~0ull ? kMinusInf : order_value((unsigned)(bound >> 32));  // the border's logit
  const float border = weights ? (bound == ~0ull ? 0.f : r.w(last)) : last;            // and as x holds it
  auto kept = [&](int i, float v) -> float {  // the weight of x[i] = v, 0 where it is not kept
    if (v < border) return 0.f;
    if (v == border && bound != ~0ull) {  // equal values are kept in order; equal weights may be of other logits
      if (order_of(weights ? logit(src[i]) : v, base + i) > bound) return 0.f;
    }
    const float w = weights ? v : r.w(v);
    return w >= least ? w : 0.f;
  };
  const int per_warp = ((n + kWarpsS * 256 - 1) / (kWarpsS * 256)) * 256;
  const int w0 = min(warp * per_warp, n), w1 = min(w0 + per_warp, n);
  WeightSum run;
  const float4* x4 = reinterpret_cast<const float4*>(x);
  if (bound == ~0ull && !weights) {  // every value counts
#pragma unroll 2
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
      const float4 l = x4[i / 4];
      const float w[4] = {r.w(l.x), r.w(l.y), r.w(l.z), r.w(l.w)};
      run.n += 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) run.add(w[q] >= least ? w[q] : 0.f);
    }
  } else if (weights) {
#pragma unroll 2
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
      const float4 l = x4[i / 4];
      const float v[4] = {l.x, l.y, l.z, l.w};
      run.n += 4;
      bool equal = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        run.add(v[q] > border && v[q] >= least ? v[q] : 0.f);
        equal |= v[q] == border;
      }
      if (equal && border > 0.f) {
        run.n += 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) run.add(v[q] == border ? kept(i + q, v[q]) : 0.f);
      }
    }
  } else {
#pragma unroll 2
    for (int i = w0 + 4 * lane; i < w1; i += 128) {
      const float4 l = x4[i / 4];
      if (fmaxf(fmaxf(l.x, l.y), fmaxf(l.z, l.w)) < border) continue;
      const float v[4] = {l.x, l.y, l.z, l.w};
      run.n += 4;
#pragma unroll
      for (int q = 0; q < 4; ++q) run.add(kept(i + q, v[q]));
    }
  }
  u64 before = 0;
  const u64 total = cluster_total(s, 0, run.total(), &before);
  u64 target = (u64)__dmul_rn((double)u, __ull2double_rn(total));
  target = min(target, total - 1);
  const u64 sum = s.warp_sum[warp];
  u64 at = before;
  for (int q = 0; q < warp; ++q) at += s.warp_sum[q];
  // ---- the warp whose run crosses the target: steps of 256 values, 8 a lane
  if (target < at || target >= at + sum) return;
  for (int j0 = w0; j0 < w1; j0 += 256) {
    u64 part[8], mine = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int i = j0 + 8 * lane + q;
      part[q] = i < w1 ? fixed40(kept(i, x[i])) : 0ull;
      mine += part[q];
    }
    const u64 end = at + warp_inclusive(mine, lane);
    const u64 next = __shfl_sync(0xffffffffu, end, 31);
    if (target >= next) {
      at = next;
      continue;
    }
    if (target < end && target >= end - mine) {
      u64 here = end - mine;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (target >= here && target < here + part[q]) {
          const int i = j0 + 8 * lane + q;
          a.tokens[row] = base + i;
          a.logprobs[row] = r.z(logit(src[i])) - logf(__fmul_rn(__ull2float_rn(total), kOne40));
        }
        here += part[q];
      }
    }
    return;
  }
}

template <typename T>
void launch(const SampleArgs& a, int C, cudaStream_t st, int dev) {
  auto kern = sample_kernel<T>;
  const size_t bytes = (size_t)a.slice * sizeof(float);
  static bool attr_set[64] = {false};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice * (int)sizeof(float)));
    attr_set[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(a.rows * C));
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a));
  ++counted_launches;
}

template <typename S>
const S* setting(const c10::optional<at::Tensor>& t, int64_t rows, at::ScalarType type, int dev, const char* what) {
  if (!t) return nullptr;
  TORCH_CHECK(t->scalar_type() == type && t->dim() == 1 && t->size(0) == rows && t->is_contiguous() && t->is_cuda() &&
                  t->get_device() == dev,
              "sample_tokens: ", what, " must be one value per row on the logits' device");
  return t->data_ptr<S>();
}

}  // namespace

// logits [B, V] fp32 or bf16 (rows may be strided); u [B] fp32 in [0, 1). A setting is a tensor
// of one value per row, or the number beside it. tokens [B] int64, logprobs [B] fp32.
void sample_tokens(const at::Tensor& logits, const at::Tensor& u, const c10::optional<at::Tensor>& temperature,
                   double temperature0, const c10::optional<at::Tensor>& top_k, int64_t top_k0,
                   const c10::optional<at::Tensor>& top_p, double top_p0, const c10::optional<at::Tensor>& min_p,
                   double min_p0, const at::Tensor& tokens, const at::Tensor& logprobs) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) == 1 || logits.stride(1) == 1),
              "sample_tokens: logits must be [rows, vocabulary] on the GPU, each row contiguous");
  const bool bf16 = logits.scalar_type() == at::kBFloat16;
  TORCH_CHECK(bf16 || logits.scalar_type() == at::kFloat, "sample_tokens: fp32 or bf16 logits");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= (int64_t)kMaxCluster * kMaxSlice, "sample_tokens: vocabulary of 1 to 262144 tokens");
  const int dev = logits.get_device();
  c10::cuda::CUDAGuard guard(dev);
  if (B == 0) return;
  TORCH_CHECK(B <= (1 << 24), "sample_tokens: too many rows");
  SampleArgs a;
  a.logits = logits.data_ptr();
  a.row_stride = logits.stride(0);
  a.rows = (int)B, a.V = (int)V;
  a.u = setting<float>(u, B, at::kFloat, dev, "u (fp32)");
  a.temperature = setting<float>(temperature, B, at::kFloat, dev, "temperature (fp32)");
  a.top_k = setting<int>(top_k, B, at::kInt, dev, "top_k (int32)");
  a.top_p = setting<float>(top_p, B, at::kFloat, dev, "top_p (fp32)");
  a.min_p = setting<float>(min_p, B, at::kFloat, dev, "min_p (fp32)");
  a.temperature0 = (float)temperature0, a.top_p0 = (float)top_p0, a.min_p0 = (float)min_p0;
  a.top_k0 = (int)std::min<int64_t>(std::max<int64_t>(top_k0, 0), 1 << 30);
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.numel() == B && tokens.is_contiguous() &&
                  logprobs.scalar_type() == at::kFloat && logprobs.numel() == B && logprobs.is_contiguous(),
              "sample_tokens: outputs");
  a.tokens = tokens.data_ptr<int64_t>();
  a.logprobs = logprobs.data_ptr<float>();
  int C = 1;
  while (C < kMaxCluster && (V > (int64_t)C * 16384 || (B * C < 148 && V > (int64_t)C * 2048))) C *= 2;
  a.slice = (int)(((V + C - 1) / C + 7) / 8 * 8);
  auto st = at::cuda::getCurrentCUDAStream(dev).stream();
  if (bf16)
    launch<__nv_bfloat16>(a, C, st, dev);
  else
    launch<float>(a, C, st, dev);
}

}  // namespace bd
