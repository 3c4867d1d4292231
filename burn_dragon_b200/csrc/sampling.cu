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
// What is kept is a prefix of the order, i.e. one bound (value, index). It is found by
// histograms of counts and weights, not by sorting: 1024 linear buckets of (m - l) / T first
// (1/32 wide; a weight below 2^-40 is zero and needs no bucket), then, among the bucket
// that holds the bound, the bits of the value and of the index, until at most kList
// candidates are left, which are ranked against each other.
//
// A row is split over a cluster of C CTAs that keep their slice of it in shared memory (the
// logits are read from memory once) and merge maxima, histograms and sums through
// distributed shared memory.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <torch/extension.h>

namespace bd {
namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarpsS = kThreads / 32;
constexpr int kBuckets = 1024;
constexpr int kList = 512;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 40960;  // logits a CTA can hold

struct SampleArgs {
  const void* logits;
  long long row_stride;
  int V, slice;
  const float *u, *temperature, *top_p, *min_p;
  const int* top_k;
  float temperature0, top_p0, min_p0;
  int top_k0;
  int64_t* tokens;
  float* logprobs;
};

struct Shared {
  unsigned count[kBuckets];
  unsigned lo[kBuckets], hi[kBuckets];  // a bucket's weight as two words
  u64 list_order[kList];                // ~value bits : index, ascending = the order of the row
  u64 list_weight[kList];
  u64 warp_sum[kWarpsS];
  u64 warp_count[kWarpsS];
  u64 slot[kMaxCluster];  // one value per CTA of the cluster
  float slot_max[kMaxCluster];
  int slot_first[kMaxCluster];
  unsigned list_n;
  // result of a bucket search / of a ranking
  int digit;
  unsigned digit_count;
  u64 before_count, before_weight;
  u64 bound, list_kept_weight;
};

__device__ __forceinline__ unsigned order_bits(float l) {  // ascending in descending l
  const unsigned b = __float_as_uint(l);
  return (b & 0x80000000u) ? b : ~(b | 0x80000000u);
}

__device__ __forceinline__ u64 fixed40(float w) {  // floor(w 2^40) for 0 <= w <= 1
  const unsigned b = __float_as_uint(w);
  const int s = (int)(b >> 23) - (127 + 23 - 40);
  const u64 m = (b & 0x7fffffu) | 0x800000u;
  return s >= 0 ? m << s : (s > -24 ? m >> -s : 0ull);
}

struct Row {
  float top, inv_t;
  __device__ __forceinline__ float z(float l) const { return l == top ? 0.f : __fmul_rn(__fsub_rn(l, top), inv_t); }
  __device__ __forceinline__ float w(float l) const { return expf(z(l)); }
  __device__ __forceinline__ int bucket(float l) const {
    return l == top ? 0 : min(kBuckets - 1, (int)(__fmul_rn(__fsub_rn(top, l), inv_t) * 32.f));
  }
};

template <typename T>
__device__ __forceinline__ float logit(T x);
template <>
__device__ __forceinline__ float logit<float>(float x) {
  return isnan(x) ? -INFINITY : x + 0.f;  // -0 counts as 0
}
template <>
__device__ __forceinline__ float logit<__nv_bfloat16>(__nv_bfloat16 x) {
  return logit<float>(__bfloat162float(x));
}

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

// Candidate digits after the linear bucket: three digits of the value's order bits, its
// last two bits, two digits of the index.
constexpr int kLevels = 7;
__device__ __forceinline__ int digit_of(int level, const Row& r, float l, unsigned ob, int index) {
  switch (level) {
    case 0: return r.bucket(l);
    case 1: return (int)(ob >> 22);
    case 2: return (int)(ob >> 12) & 1023;
    case 3: return (int)(ob >> 2) & 1023;
    case 4: return (int)ob & 3;
    case 5: return index >> 10;
    default: return index & 1023;
  }
}

struct Path {  // digits chosen so far
  int n;
  int digit[kLevels];
};

__device__ __forceinline__ bool on_path(const Path& p, const Row& r, float l, int index) {
  const unsigned ob = order_bits(l);
  for (int i = 0; i < p.n; ++i)
    if (digit_of(i, r, l, ob, index) != p.digit[i]) return false;
  return true;
}

// Finds the last kept candidate of the row's order, where a candidate is kept while its count of
// predecessors is below `most` and the weight of its predecessors below `reach`, or 2^64-1 if every
// candidate is kept. Candidates: weight above zero and order <= `bound`. Also the weight of all kept.
// Every CTA of the cluster calls it with the same arguments and gets the same answer.
__device__ u64 find_bound(Shared& s, const float* x, int base, int n, const Row& r, u64 bound, u64 most, u64 reach,
                          bool weigh, u64& kept_weight) {
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  Path path;
  path.n = 0;
  u64 count0 = 0, weight0 = 0;  // before the candidates on the path
  for (int level = 0; level < kLevels; ++level) {
    for (int b = tid; b < kBuckets; b += kThreads) s.count[b] = s.lo[b] = s.hi[b] = 0;
    if (tid == 0) s.list_n = 0, s.digit = -1;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const float l = x[i];
      if (l == -INFINITY || !on_path(path, r, l, base + i)) continue;
      const unsigned ob = order_bits(l);
      if (((u64)ob << 32 | (unsigned)(base + i)) > bound) continue;
      const u64 w = fixed40(r.w(l));
      if (w == 0) continue;
      const int d = digit_of(level, r, l, ob, base + i);
      atomicAdd(&s.count[d], 1u);
      if (weigh) {
        const unsigned lo = (unsigned)w, old = atomicAdd(&s.lo[d], lo);
        const unsigned hi = (unsigned)(w >> 32) + (old + lo < old ? 1u : 0u);
        if (hi) atomicAdd(&s.hi[d], hi);
      }
    }
    cluster.sync();
    // merged histogram: two buckets a thread, then the block's running sums
    u64 c[2], w[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      c[k] = w[k] = 0;
      const int b = 2 * tid + k;
      for (int q = 0; q < C; ++q) {
        const Shared* o = cluster.map_shared_rank(&s, q);
        c[k] += o->count[b];
        if (weigh) w[k] += (u64)o->hi[b] << 32 | o->lo[b];
      }
    }
    u64 ic = warp_inclusive(c[0] + c[1], lane), iw = weigh ? warp_inclusive(w[0] + w[1], lane) : 0;
    if (lane == 31) s.warp_count[warp] = ic, s.warp_sum[warp] = iw;
    __syncthreads();
    u64 bc = count0 + ic - c[0] - c[1], bw = weight0 + iw - w[0] - w[1];
    u64 all_c = count0, all_w = weight0;
    for (int q = 0; q < kWarpsS; ++q) {
      if (q < warp) bc += s.warp_count[q], bw += s.warp_sum[q];
      all_c += s.warp_count[q], all_w += s.warp_sum[q];
    }
    // the bound lies in the first bucket after which the count or the weight is reached
    if (level == 0 && all_c <= most && all_w <= reach) {
      kept_weight = all_w;
      cluster.sync();  // the histograms are read
      return bound;
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (c[k] > 0 && bc < most && bw < reach && (bc + c[k] >= most || bw + w[k] >= reach)) {
        s.digit = 2 * tid + k;
        s.digit_count = (unsigned)c[k];
        s.before_count = bc;
        s.before_weight = bw;
      }
      bc += c[k];
      bw += w[k];
    }
    cluster.sync();  // the search is written, the histograms are read
    if (s.digit < 0) {  // neither is reached: everything is kept
      kept_weight = all_w;
      return bound;
    }
    path.digit[path.n++] = s.digit;
    count0 = s.before_count;
    weight0 = s.before_weight;
    if (s.digit_count <= kList || level == kLevels - 1) break;
    __syncthreads();
  }
  // gather the candidates in the first CTA, rank them there
  Shared* first = cluster.map_shared_rank(&s, 0);
  for (int i = tid; i < n; i += kThreads) {
    const float l = x[i];
    if (l == -INFINITY || !on_path(path, r, l, base + i)) continue;
    const u64 order = (u64)order_bits(l) << 32 | (unsigned)(base + i);
    if (order > bound) continue;
    const u64 w = fixed40(r.w(l));
    if (w == 0) continue;
    const unsigned at = atomicAdd(&first->list_n, 1u);
    if (at < kList) {
      first->list_order[at] = order;
      first->list_weight[at] = w;
    }
  }
  cluster.sync();
  if (cluster.block_rank() == 0) {
    const int m = (int)min(s.list_n, (unsigned)kList);
    for (int i = tid; i < m; i += kThreads) {
      const u64 me = s.list_order[i];
      u64 bc = count0, bw = weight0;
      for (int j = 0; j < m; ++j) {
        const bool before = s.list_order[j] < me;
        bc += before ? 1 : 0;
        bw += before ? s.list_weight[j] : 0;
      }
      const u64 ac = bc + 1, aw = bw + s.list_weight[i];
      // exactly one candidate is kept and its successor is not
      if (bc < most && bw < reach && (ac >= most || aw >= reach)) {
        for (int q = 0; q < C; ++q) {
          Shared* o = cluster.map_shared_rank(&s, q);
          o->bound = me;
          o->list_kept_weight = aw;
        }
      }
    }
  }
  cluster.sync();
  kept_weight = s.list_kept_weight;
  return s.bound;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ float x[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();  // waited for before the first access to another CTA's memory
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int base = min(rank * a.slice, a.V), n = min(a.slice, a.V - base);
  const T* src = static_cast<const T*>(a.logits) + (long long)row * a.row_stride + base;

  // ---- the slice, and the row's maximum with its first index
  float top = -INFINITY;
  int first = 0x7fffffff;
  for (int i = tid; i < n; i += kThreads) {
    const float l = logit<T>(src[i]);
    x[i] = l;
    if (l > top) top = l, first = base + i;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float t = __shfl_xor_sync(0xffffffffu, top, o);
    const int f = __shfl_xor_sync(0xffffffffu, first, o);
    if (t > top || (t == top && f < first)) top = t, first = f;
  }
  if (lane == 0) {
    s.warp_sum[warp] = __float_as_uint(top);
    s.warp_count[warp] = (unsigned)first;
  }
  __syncthreads();
  cluster.barrier_wait();
  if (tid < C) {
    for (int q = 0; q < kWarpsS; ++q) {
      const float t = __uint_as_float((unsigned)s.warp_sum[q]);
      const int f = (int)s.warp_count[q];
      if (q == 0 || t > top || (t == top && f < first)) top = t, first = f;
    }
    Shared* o = cluster.map_shared_rank(&s, tid);
    o->slot_max[rank] = top;
    o->slot_first[rank] = first;
  }
  cluster.sync();
  top = s.slot_max[0];
  first = s.slot_first[0];
  for (int q = 1; q < C; ++q)
    if (s.slot_max[q] > top) top = s.slot_max[q], first = s.slot_first[q];

  const float temperature = a.temperature ? a.temperature[row] : a.temperature0;
  if (top == -INFINITY || !(temperature > 0.f)) {  // nothing to draw from, or the first maximum
    if (rank == 0 && tid == 0) {
      a.tokens[row] = top == -INFINITY ? -1 : first;
      a.logprobs[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    cluster.sync();
    return;
  }
  Row r;
  r.top = top;
  r.inv_t = __fdiv_rn(1.f, temperature);
  const int k = a.top_k ? a.top_k[row] : a.top_k0;
  const float p = a.top_p ? a.top_p[row] : a.top_p0;
  const float least = fminf(a.min_p ? a.min_p[row] : a.min_p0, 1.f);
  const bool use_k = k > 0 && k < a.V, use_p = p < 1.f;

  // ---- the bound of the kept prefix
  u64 bound = ~0ull, kept = 0;
  if (use_k || use_p) {
    bound = find_bound(s, x, base, n, r, bound, use_k ? (u64)k : ~0ull, ~0ull, use_p, kept);
    if (use_p) {
      const double want = ceil(__dmul_rn(__ull2double_rn(kept), (double)p));
      const u64 reach = want > 1.0 ? (u64)want : 1ull;
      if (reach < kept) bound = find_bound(s, x, base, n, r, bound, ~0ull, reach, true, kept);
    }
  }

  // ---- sums of the kept weights: warp w owns a run of 32-value steps of the slice
  const int per_warp = ((n + kWarpsS * 32 - 1) / (kWarpsS * 32)) * 32;
  const int w0 = min(warp * per_warp, n), w1 = min(w0 + per_warp, n);
  auto weight = [&](int i) -> u64 {
    const float l = x[i];
    if (l == -INFINITY || ((u64)order_bits(l) << 32 | (unsigned)(base + i)) > bound) return 0ull;
    const float w = r.w(l);
    return w >= least ? fixed40(w) : 0ull;
  };
  u64 sum = 0;
  for (int i = w0 + lane; i < w1; i += 32) sum += weight(i);
  sum = warp_total(sum);
  if (lane == 0) s.warp_sum[warp] = sum;
  __syncthreads();
  u64 mine = 0;
  for (int q = 0; q < kWarpsS; ++q) mine += s.warp_sum[q];
  if (tid < C) cluster.map_shared_rank(&s, tid)->slot[rank] = mine;
  cluster.sync();
  u64 total = 0, before = 0;
  for (int q = 0; q < C; ++q) {
    if (q < rank) before += s.slot[q];
    total += s.slot[q];
  }
  u64 target = (u64)__dmul_rn((double)a.u[row], __ull2double_rn(total));
  target = min(target, total - 1);
  if (target < before || target >= before + mine) return;
  // ---- this CTA holds the token: the warp whose run crosses the target walks it
  u64 at = before;
  for (int q = 0; q < warp; ++q) at += s.warp_sum[q];
  if (target < at || target >= at + sum) return;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const int i = i0 + lane;
    const u64 w = i < w1 ? weight(i) : 0ull;
    const u64 run = at + warp_inclusive(w, lane);
    const unsigned hit = __ballot_sync(0xffffffffu, run > target);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.tokens[row] = base + i;
        a.logprobs[row] = r.z(x[i]) - logf(__fmul_rn(__ull2float_rn(total), 9.094947017729282e-13f));
      }
      return;
    }
    at = __shfl_sync(0xffffffffu, run, 31);
  }
}

template <typename T>
void launch(const SampleArgs& a, int rows, int C, cudaStream_t st) {
  auto kern = sample_kernel<T>;
  const size_t bytes = (size_t)a.slice * sizeof(float);
  C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice * (int)sizeof(float)));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a));
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
  TORCH_CHECK(V >= 1 && V <= (int64_t)kMaxCluster * 32768, "sample_tokens: vocabulary of 1 to 262144 tokens");
  const int dev = logits.get_device();
  c10::cuda::CUDAGuard guard(dev);
  if (B == 0) return;
  TORCH_CHECK(B <= (1 << 24), "sample_tokens: too many rows");
  SampleArgs a;
  a.logits = logits.data_ptr();
  a.row_stride = logits.stride(0);
  a.V = (int)V;
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
    launch<__nv_bfloat16>(a, (int)B, C, st);
  else
    launch<float>(a, (int)B, C, st);
}

}  // namespace bd
