// adamw_many.cu — one AdamW step over many tensors, states in fp32 or in 8 bits.
//
//   g' = g c;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps);  shadow = bf16(p)
//
// t counts the tensor's own steps: one without a gradient keeps its moments, and its count.
// The states of all tensors lie in one buffer, each tensor padded to blocks of 256 values;
// one warp owns one block and `owner[block]` names its tensor. The tensors' addresses are
// kernel arguments (up to 32 KB of them), so a step is one launch and copies no table.
//
// 8-bit states: a block keeps scale = absmax / 256 and 256 e4m3 codes of value / scale. One
// step moves v by about (1 - b2) of itself, far below half an e4m3 step (6 to 12 %), so
// rounding to nearest would freeze it; the codes are rounded stochastically instead, with 16
// bits for m and 16 for v from a hash of (seed, step, index): the stored average is the
// true one, and a step can be repeated bit for bit. A v above zero keeps at least the lowest
// code, since a denominator rounded to zero would blow its update up. m and v are
// computed with separately rounded products and sums, so any implementation of the formulas
// gives the same codes.
//
// Measured on a B200: 25.2 M values, fp32 states and gradients, 28 B each: 109 us = 6.5 TB/s, the copy rate. 26 M
// values with e4m3 states, bf16 gradients and working copies, 16 B each: 93 us = 4.5 TB/s; there the
// instructions bound it (about 84 a value: 71 % of the issue slots, with DRAM busy for half of the time).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <torch/extension.h>

#include <cmath>
#include <vector>

#include "launches.h"

namespace bd {
namespace {

constexpr int kBlock = 256;   // values per state block: 8 a lane
constexpr int kWarps = 8;     // blocks per CTA
constexpr float kTiny = 7.703719777548943e-34f;  // 2^-110: below it a block is stored as zero

enum : int { kParamBf16 = 1, kGradBf16 = 2, kWide = 4 };

struct ManyTensor {
  void* p;
  const void* g;  // null: no gradient, the tensor keeps its state
  __nv_bfloat16* shadow;
  long long n;
  int block0;  // first state block
  int flags;
  float step, inv_bc2;  // lr / (1 - b1^t), 1 / (1 - b2^t)
};

template <int CAP>
struct ManyTable {
  ManyTensor t[CAP];
};

struct ManyHyper {
  float decay, b1, nb1, b2, nb2, eps;
  unsigned key;
  const float* gscale;
};

template <bool WIDE>
__device__ __forceinline__ int elem(int lane, int j) {  // value j (0..7) of a lane inside its block
  return WIDE ? (j >> 2) * 128 + lane * 4 + (j & 3) : j * 32 + lane;
}

template <bool WIDE>
__device__ __forceinline__ void load8(const void* base, bool bf16, long long at, int lane, int n, float (&v)[8]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (bf16) {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + at + h * 128 + lane * 4);
        const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
        const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
        v[4 * h] = a.x, v[4 * h + 1] = a.y, v[4 * h + 2] = b.x, v[4 * h + 3] = b.y;
      } else {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + h * 128 + lane * 4);
        v[4 * h] = f.x, v[4 * h + 1] = f.y, v[4 * h + 2] = f.z, v[4 * h + 3] = f.w;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = elem<false>(lane, j);
      v[j] = e >= n ? 0.f
             : bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[at + e])
                    : static_cast<const float*>(base)[at + e];
    }
  }
}

template <bool WIDE>
__device__ __forceinline__ void store8(void* base, bool bf16, long long at, int lane, int n, const float (&v)[8]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (bf16) {
        __nv_bfloat162 a = __floats2bfloat162_rn(v[4 * h], v[4 * h + 1]), b = __floats2bfloat162_rn(v[4 * h + 2], v[4 * h + 3]);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(base) + at + h * 128 + lane * 4) =
            make_uint2(*reinterpret_cast<unsigned*>(&a), *reinterpret_cast<unsigned*>(&b));
      } else {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + at + h * 128 + lane * 4) =
            make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int e = elem<false>(lane, j);
      if (e >= n) continue;
      if (bf16)
        static_cast<__nv_bfloat16*>(base)[at + e] = __float2bfloat16_rn(v[j]);
      else
        static_cast<float*>(base)[at + e] = v[j];
    }
  }
}

// Four e4m3 codes, two a conversion.
__device__ __forceinline__ void e4m3_values(unsigned u, float* v) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(u >> (16 * k)), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[2 * k] = f.x, v[2 * k + 1] = f.y;
  }
}

template <bool WIDE>
__device__ __forceinline__ void load_codes(const unsigned char* s, int lane, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unsigned u = 0;
    if constexpr (WIDE) {
      u = *reinterpret_cast<const unsigned*>(s + h * 128 + lane * 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) u |= (unsigned)s[elem<false>(lane, 4 * h + k)] << (8 * k);
    }
    e4m3_values(u, v + 4 * h);
  }
}

template <bool WIDE>
__device__ __forceinline__ void store_codes(unsigned char* s, int lane, const unsigned (&c)[8]) {
  if constexpr (WIDE) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<unsigned*>(s + h * 128 + lane * 4) = __byte_perm(
          __byte_perm(c[4 * h], c[4 * h + 1], 0x0040), __byte_perm(c[4 * h + 2], c[4 * h + 3], 0x0040), 0x5410);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) s[elem<false>(lane, j)] = (unsigned char)c[j];
  }
}

// m / (sqrt(v) + eps). Beside 8-bit states, whose own rounding is 2^-4 and which the instructions bound (102 us
// with the correctly rounded forms when 90 without), root and quotient are good to 2^-22 of the step; the states do not use
// them. With 32-bit states the bytes bound the step, and both are rounded correctly.
template <bool EIGHT>
__device__ __forceinline__ float ratio(float m, float v, float eps) {
  if constexpr (!EIGHT) return __fdiv_rn(m, __fadd_rn(__fsqrt_rn(v), eps));
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return __fdividef(m, r + eps);
}

// absmax over the warp's block as bits: NaN and infinity win, as they have to
__device__ __forceinline__ unsigned block_amax(const float (&x)[8]) {
  unsigned a = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) a = max(a, __float_as_uint(x[j]) & 0x7fffffffu);
  return __reduce_max_sync(0xffffffffu, a);
}

// {scale to store, factor to multiply by}; a block below 2^-110 is zero, one that is not finite decodes to NaN
__device__ __forceinline__ float2 block_scale(unsigned amax_bits) {
  const float amax = __uint_as_float(amax_bits);
  if (amax >= kTiny && amax < INFINITY) return make_float2(amax * 0.00390625f, __fdiv_rn(256.f, amax));
  return make_float2(amax < kTiny ? 0.f : amax, 0.f);
}

// |x| / scale on the e4m3 grid: scaled so that the grid is bits 20 and up of the (denormal
// included) fp32 pattern; the random fraction carries into it.
__device__ __forceinline__ unsigned e4m3_stochastic(float x, float inverse, unsigned bits16) {
  const float y = __fmul_rn(__fmul_rn(fabsf(x), inverse), 7.52316384526264e-37f);  // 2^-120
  return (__float_as_uint(y) + (bits16 << 4)) >> 20;
}

template <int CAP, bool EIGHT, bool WIDE>
__device__ __forceinline__ void update_block(const ManyTensor& t, const ManyHyper& h, long long block, int lane, int n,
                                             void* M, void* V, float* MS, float* VS) {
  const long long at = (block - t.block0) * (long long)kBlock;
  const long long st = block * (long long)kBlock;
  float p[8], g[8], m[8], v[8];
  load8<WIDE>(t.g, t.flags & kGradBf16, at, lane, n, g);
  load8<WIDE>(t.p, t.flags & kParamBf16, at, lane, n, p);
  if constexpr (EIGHT) {
    load_codes<WIDE>(static_cast<unsigned char*>(M) + st, lane, m);
    load_codes<WIDE>(static_cast<unsigned char*>(V) + st, lane, v);
    const float sm = MS[block], sv = VS[block];
#pragma unroll
    for (int j = 0; j < 8; ++j) m[j] = __fmul_rn(m[j], sm), v[j] = __fmul_rn(v[j], sv);
  } else {
    load8<WIDE>(M, false, st, lane, kBlock, m);
    load8<WIDE>(V, false, st, lane, kBlock, v);
  }
  const float gs = h.gscale ? *h.gscale : 1.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float gi = __fmul_rn(g[j], gs);
    m[j] = __fadd_rn(__fmul_rn(m[j], h.b1), __fmul_rn(gi, h.nb1));
    v[j] = __fadd_rn(__fmul_rn(v[j], h.b2), __fmul_rn(__fmul_rn(gi, gi), h.nb2));
    p[j] = p[j] * h.decay - ratio<EIGHT>(m[j] * t.step, v[j] * t.inv_bc2, h.eps);
  }
  store8<WIDE>(t.p, t.flags & kParamBf16, at, lane, n, p);
  if (t.shadow) store8<WIDE>(t.shadow, true, at, lane, n, p);
  if constexpr (EIGHT) {
    const float2 fm = block_scale(block_amax(m)), fv = block_scale(block_amax(v));
    unsigned cm[8], cv[8];
    const unsigned first = (unsigned)st * 0x9E3779B1u + h.key;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      unsigned x = first + (unsigned)elem<WIDE>(lane, j) * 0x9E3779B1u;
      x = (x ^ (x >> 16)) * 0x85EBCA6Bu;
      x = (x ^ (x >> 13)) * 0xC2B2AE35u;
      x ^= x >> 16;
      cm[j] = e4m3_stochastic(m[j], fm.y, x & 0xffffu) | (m[j] < 0.f ? 0x80u : 0u);
      cv[j] = max(e4m3_stochastic(v[j], fv.y, x >> 16), v[j] > 0.f ? 1u : 0u);
    }
    if (fm.y == 0.f || fv.y == 0.f) {  // a block of zeros, or one that is not finite (of the whole warp)
#pragma unroll
      for (int j = 0; j < 8; ++j) cm[j] = fm.y == 0.f ? 0u : cm[j], cv[j] = fv.y == 0.f ? 0u : cv[j];
    }
    store_codes<WIDE>(static_cast<unsigned char*>(M) + st, lane, cm);
    store_codes<WIDE>(static_cast<unsigned char*>(V) + st, lane, cv);
    if (lane == 0) MS[block] = fm.x, VS[block] = fv.x;
  } else {
    store8<WIDE>(M, false, st, lane, kBlock, m);
    store8<WIDE>(V, false, st, lane, kBlock, v);
  }
}

template <int CAP, bool EIGHT>
__global__ void __launch_bounds__(32 * kWarps, EIGHT ? 5 : 4) adamw_many_kernel(const __grid_constant__ ManyTable<CAP> table,
                                                                 const __grid_constant__ ManyHyper h,
                                                                 const int* __restrict__ owner, int first,
                                                                 long long block0, long long block1, void* M, void* V,
                                                                 float* MS, float* VS) {
  const int lane = threadIdx.x % 32;
  const long long block = block0 + (long long)blockIdx.x * kWarps + threadIdx.x / 32;
  if (block >= block1) return;
  const ManyTensor& t = table.t[owner[block] - first];
  if (t.g == nullptr) return;
  const long long left = t.n - (block - t.block0) * (long long)kBlock;
  const int n = (int)min(left, (long long)kBlock);
  if (n == kBlock && (t.flags & kWide))
    update_block<CAP, EIGHT, true>(t, h, block, lane, n, M, V, MS, VS);
  else
    update_block<CAP, EIGHT, false>(t, h, block, lane, n, M, V, MS, VS);
}

int dtype_of(const at::Tensor& t, int bf16_flag) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, "adamw_many: fp32 or bf16 tensors");
  return t.scalar_type() == at::kBFloat16 ? bf16_flag : 0;
}

bool wide(const void* p, bool bf16) { return reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16) == 0; }

template <int CAP>
void launch(const std::vector<ManyTensor>& all, size_t first, size_t count, const ManyHyper& h, const at::Tensor& owner,
            long long block0, long long block1, const at::Tensor& m, const at::Tensor& v, float* ms, float* vs,
            cudaStream_t st) {
  ManyTable<CAP> table;
  std::copy(all.begin() + first, all.begin() + first + count, table.t);
  const unsigned grid = (unsigned)((block1 - block0 + kWarps - 1) / kWarps);
  if (ms)
    adamw_many_kernel<CAP, true><<<grid, 32 * kWarps, 0, st>>>(table, h, owner.data_ptr<int>(), (int)first, block0,
                                                               block1, m.data_ptr(), v.data_ptr(), ms, vs);
  else
    adamw_many_kernel<CAP, false><<<grid, 32 * kWarps, 0, st>>>(table, h, owner.data_ptr<int>(), (int)first, block0,
                                                                block1, m.data_ptr(), v.data_ptr(), ms, vs);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
}

constexpr int kFew = 64, kMany = 640;  // tensors a launch names: 3 KB or 30 KB of arguments
static_assert(sizeof(ManyTable<kMany>) + sizeof(ManyHyper) + 128 <= 32764, "arguments of a launch");

}  // namespace

// params / grads / shadows: one entry per tensor (a gradient may be None, shadows may be
// empty); block0[i]: the first 256-value state block of tensor i, with the total last;
// owner [total] int32: the tensor of each block. m, v: [total * 256] fp32, or e4m3 with
// m_scale, v_scale [total] fp32. steps [n] int64 on the host: each tensor's own steps so far; those of the
// tensors with a gradient are advanced.
void adamw_many(const std::vector<at::Tensor>& params, const std::vector<c10::optional<at::Tensor>>& grads,
                const std::vector<at::Tensor>& shadows, const std::vector<int64_t>& block0, const at::Tensor& owner,
                const at::Tensor& m, const at::Tensor& v, const c10::optional<at::Tensor>& m_scale,
                const c10::optional<at::Tensor>& v_scale, double lr, double b1, double b2, double eps, double wd,
                const at::Tensor& steps, int64_t key, const c10::optional<at::Tensor>& gscale) {
  const size_t n = params.size();
  TORCH_CHECK(n > 0 && grads.size() == n && block0.size() == n + 1, "adamw_many: one gradient and state range per tensor");
  TORCH_CHECK(steps.device().is_cpu() && steps.scalar_type() == at::kLong && steps.is_contiguous() && steps.numel() == (int64_t)n,
              "adamw_many: one step count per tensor, on the host");
  int64_t* had = steps.data_ptr<int64_t>();
  TORCH_CHECK(shadows.empty() || shadows.size() == n, "adamw_many: no shadows or one per tensor");
  const int dev = m.get_device();
  c10::cuda::CUDAGuard guard(dev);
  const long long total = block0[n];
  TORCH_CHECK(owner.numel() == total && m.numel() == total * kBlock && v.numel() == total * kBlock,
              "adamw_many: state sizes");
  const bool eight = m_scale.has_value();
  TORCH_CHECK(m.scalar_type() == v.scalar_type() && m.scalar_type() == (eight ? at::kFloat8_e4m3fn : at::kFloat),
              "adamw_many: fp32 states, or e4m3 states with scales");
  if (eight) TORCH_CHECK(v_scale && m_scale->numel() == total && v_scale->numel() == total, "adamw_many: scale sizes");
  if (gscale) TORCH_CHECK(gscale->scalar_type() == at::kFloat && gscale->get_device() == dev, "adamw_many: gradient scale");
  ManyHyper h;
  h.decay = (float)(1.0 - lr * wd);
  h.b1 = (float)b1, h.nb1 = (float)(1.0 - b1), h.b2 = (float)b2, h.nb2 = (float)(1.0 - b2);
  h.eps = (float)eps;
  h.key = (unsigned)key;
  h.gscale = gscale ? gscale->data_ptr<float>() : nullptr;
  std::vector<ManyTensor> all(n);
  int64_t last = 0;  // of most tensors the same
  float step = 0.f, inv_bc2 = 0.f;
  for (size_t i = 0; i < n; ++i) {
    ManyTensor& t = all[i];
    const at::Tensor& p = params[i];
    TORCH_CHECK(p.get_device() == dev && p.is_contiguous(), "adamw_many: contiguous tensors on one device");
    t.p = p.data_ptr();
    t.n = p.numel();
    t.block0 = (int)block0[i];
    TORCH_CHECK((t.n + kBlock - 1) / kBlock == block0[i + 1] - block0[i], "adamw_many: a tensor's size has changed");
    t.flags = dtype_of(p, kParamBf16);
    bool w = wide(t.p, t.flags & kParamBf16);
    t.g = nullptr;
    t.step = t.inv_bc2 = 0.f;
    if (grads[i]) {
      TORCH_CHECK(had[i] >= 0, "adamw_many: step counts below 0");
      if (had[i] + 1 != last) {
        last = had[i] + 1;
        step = (float)(lr / (1.0 - std::pow(b1, (double)last)));
        inv_bc2 = (float)(1.0 / (1.0 - std::pow(b2, (double)last)));
      }
      t.step = step, t.inv_bc2 = inv_bc2;
      const at::Tensor& g = *grads[i];
      TORCH_CHECK(g.get_device() == dev && g.is_contiguous() && g.numel() == t.n, "adamw_many: a gradient like its tensor");
      t.flags |= dtype_of(g, kGradBf16);
      t.g = g.data_ptr();
      w = w && wide(t.g, t.flags & kGradBf16);
    }
    t.shadow = nullptr;
    if (!shadows.empty()) {
      const at::Tensor& s = shadows[i];
      TORCH_CHECK(s.get_device() == dev && s.is_contiguous() && s.numel() == t.n && s.scalar_type() == at::kBFloat16,
                  "adamw_many: bf16 shadows like their tensors");
      t.shadow = reinterpret_cast<__nv_bfloat16*>(s.data_ptr());
      w = w && wide(t.shadow, true);
    }
    if (w) t.flags |= kWide;
  }
  auto st = at::cuda::getCurrentCUDAStream(dev).stream();
  float* ms = eight ? m_scale->data_ptr<float>() : nullptr;
  float* vs = eight ? v_scale->data_ptr<float>() : nullptr;
  for (size_t i = 0; i < n;) {
    const size_t count = std::min<size_t>(n - i, n - i <= kFew ? kFew : kMany);
    if (block0[i + count] > block0[i]) {
      if (count <= kFew)
        launch<kFew>(all, i, count, h, owner, block0[i], block0[i + count], m, v, ms, vs, st);
      else
        launch<kMany>(all, i, count, h, owner, block0[i], block0[i + count], m, v, ms, vs, st);
    }
    i += count;
  }
  for (size_t i = 0; i < n; ++i) had[i] += grads[i].has_value();
}

}  // namespace bd
