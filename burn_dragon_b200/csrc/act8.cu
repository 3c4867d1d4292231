// act8.cu — pack and unpack of activations in 8 bits (act8.cuh): rows of N values, blocks of 32 along a row (the last
// one of a row may be shorter), codes [R, N] and exponents [R, ceil(N / 32)].
//
// Bound by bytes: a value is read once (2 or 4 bytes) and leaves as 33/32 bytes, and back.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <torch/extension.h>

#include "act8.cuh"
#include "launches.h"

namespace bd {
namespace {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <typename T>
constexpr float limit_of() {
  return sizeof(T) == 4 ? kAct8LimitF32 : std::is_same<T, __half>::value ? kAct8LimitF16 : kAct8LimitBF16;
}

// 8 values of a row a thread and step, four threads a block; kUnits steps are read before the first is coded.
// FLAT: rows are whole blocks, so that the tensor is one row. Else N is a multiple of 8.
constexpr int kUnits = 4;

template <typename T>
struct Eight {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ void get(float* f) const {
    const T* t = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = as_float(t[i]);
  }
  __device__ __forceinline__ void put(const float* f) {
    T* t = reinterpret_cast<T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_float<T>(f[i]);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, v[i]);
  }
};

// Where unit u (4 a block) lies: its first value, its block, and whether it has values.
template <bool FLAT>
__device__ __forceinline__ bool unit_at(long long u, long long units, int N, int nb, long long& at, long long& block) {
  block = u / 4;
  if constexpr (FLAT) {
    at = u * 8;
    return u < units;
  } else {
    const long long r = block / nb;
    const int c = (int)(u - r * 4 * nb) * 8;
    at = r * N + c;
    return u < units && c < N;
  }
}

template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) act8_pack8_kernel(const T* __restrict__ x, long long units, int N, int nb,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const long long first = (long long)blockIdx.x * (256 * kUnits) + threadIdx.x;
  Eight<T> raw[kUnits];
  long long at[kUnits], block[kUnits];
  bool in[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    in[k] = unit_at<FLAT>(first + 256 * k, units, N, nb, at[k], block[k]);
    if (in[k]) raw[k].load(x + at[k]);
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    float f[8], largest = 0.f;
    if (in[k]) {
      raw[k].get(f);
#pragma unroll
      for (int i = 0; i < 8; ++i) largest = fmaxf(largest, act8_size(f[i]));
    }
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    if (!in[k]) continue;
    const int e = act8_exponent(largest);
    const float inverse = act8_power(-e);
    __stcs(reinterpret_cast<uint2*>(codes + at[k]), make_uint2(act8_code4(f, inverse), act8_code4(f + 4, inverse)));
    if (threadIdx.x % 4 == 0) scales[block[k]] = (uint8_t)(e + 127);
  }
}

template <typename T, bool FLAT>
__global__ void __launch_bounds__(256) act8_unpack8_kernel(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, long long units, int N,
                                                           int nb, T* __restrict__ y) {
  const long long first = (long long)blockIdx.x * (256 * kUnits) + threadIdx.x;
  uint2 raw[kUnits];
  uint8_t scale[kUnits];
  long long at[kUnits], block[kUnits];
  bool in[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    in[k] = unit_at<FLAT>(first + 256 * k, units, N, nb, at[k], block[k]);
    if (in[k]) {
      raw[k] = __ldcs(reinterpret_cast<const uint2*>(codes + at[k]));
      scale[k] = scales[block[k]];
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (!in[k]) continue;
    const float power = act8_power((int)scale[k] - 127);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = act8_value2(((i < 2 ? raw[k].x : raw[k].y) >> (16 * (i & 1))) & 0xFFFFu, power, limit_of<T>());
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
    Eight<T> out;
    out.put(f);
    out.store(y + at[k]);
  }
}

// A block of 32 a warp, a value a lane: any N.
template <typename T>
__global__ void __launch_bounds__(256) act8_pack_kernel(const T* __restrict__ x, long long R, int N, int nb,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int lane = threadIdx.x % 32;
  const long long blocks = R * nb;
  for (long long b = (long long)blockIdx.x * 8 + threadIdx.x / 32; b < blocks; b += (long long)gridDim.x * 8) {
    const long long r = b / nb;
    const int c = (int)(b - r * nb) * 32 + lane;
    const float v = c < N ? as_float(x[r * N + c]) : 0.f;
    float largest = act8_size(v);
#pragma unroll
    for (int o = 16; o > 0; o /= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const int e = act8_exponent(largest);
    if (c < N) codes[r * N + c] = (uint8_t)act8_code2(v, 0.f, act8_power(-e));
    if (lane == 0) scales[b] = (uint8_t)(e + 127);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) act8_unpack_kernel(const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, long long R, int N, int nb,
                                                          T* __restrict__ y) {
  const int lane = threadIdx.x % 32;
  const long long blocks = R * nb;
  for (long long b = (long long)blockIdx.x * 8 + threadIdx.x / 32; b < blocks; b += (long long)gridDim.x * 8) {
    const long long r = b / nb;
    const int c = (int)(b - r * nb) * 32 + lane;
    if (c < N) y[r * N + c] = from_float<T>(act8_value2(codes[r * N + c], act8_power((int)scales[b] - 127), limit_of<T>()).x);
  }
}

template <typename F>
void for_type(at::ScalarType t, F&& f) {
  if (t == at::kFloat)
    f((float*)nullptr);
  else if (t == at::kBFloat16)
    f((__nv_bfloat16*)nullptr);
  else if (t == at::kHalf)
    f((__half*)nullptr);
  else
    TORCH_CHECK(false, "act8: fp32, bf16 or fp16 values");
}

unsigned grid_of(long long blocks) { return (unsigned)std::max<long long>(1, std::min<long long>((blocks + 7) / 8, 148 * 32)); }

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned unit_grid(long long units) {
  const long long grid = (units + 256 * kUnits - 1) / (256 * kUnits);
  TORCH_CHECK(grid < (1ll << 31), "act8: too many values");
  return (unsigned)grid;
}

}  // namespace

// x, of any shape: codes [R, N] and exponents [R, ceil(N / 32)], uint8, N its last dimension (of at least one value).
std::vector<at::Tensor> act8_pack(const at::Tensor& given) {
  TORCH_CHECK(given.is_cuda(), "act8_pack: values on a GPU");
  c10::cuda::CUDAGuard guard(given.get_device());
  const at::Tensor x = given.contiguous();
  const int64_t N = x.numel() == 0 || x.dim() == 0 ? 1 : x.size(-1), R = x.numel() / N, nb = (N + 31) / 32;
  TORCH_CHECK(N < (1ll << 31) - 32, "act8_pack: rows of less than 2^31 - 32 values");
  auto st = at::cuda::getCurrentCUDAStream(x.get_device()).stream();
  const auto bytes = x.options().dtype(at::kByte).requires_grad(false);
  at::Tensor codes = at::empty({R, N}, bytes), scales = at::empty({R, nb}, bytes);
  if (x.numel() == 0) return {codes, scales};
  for_type(x.scalar_type(), [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    const T* v = reinterpret_cast<const T*>(x.data_ptr());
    uint8_t *c = codes.data_ptr<uint8_t>(), *s = scales.data_ptr<uint8_t>();
    const long long units = R * nb * 4;
    if (N % 32 == 0 && aligned(v))
      act8_pack8_kernel<T, true><<<unit_grid(units), 256, 0, st>>>(v, units, (int)N, (int)nb, c, s);
    else if (N % 8 == 0 && aligned(v))
      act8_pack8_kernel<T, false><<<unit_grid(units), 256, 0, st>>>(v, units, (int)N, (int)nb, c, s);
    else
      act8_pack_kernel<T><<<grid_of(R * nb), 256, 0, st>>>(v, R, (int)N, (int)nb, c, s);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return {codes, scales};
}

// The values that codes and exponents stand for, in `shape` (R N values) and type 0 fp32, 1 bf16 or 2 fp16.
at::Tensor act8_unpack(const at::Tensor& codes, const at::Tensor& scales, const std::vector<int64_t>& shape, int64_t type) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.is_contiguous() && codes.scalar_type() == at::kByte,
              "act8_unpack: contiguous codes [R, N]");
  const int64_t R = codes.size(0), N = codes.size(1), nb = (N + 31) / 32;
  TORCH_CHECK(scales.is_cuda() && scales.get_device() == codes.get_device() && scales.scalar_type() == at::kByte &&
                  scales.is_contiguous() && scales.dim() == 2 && scales.size(0) == R && scales.size(1) == nb,
              "act8_unpack: exponents [R, ceil(N / 32)]");
  c10::cuda::CUDAGuard guard(codes.get_device());
  auto st = at::cuda::getCurrentCUDAStream(codes.get_device()).stream();
  const at::ScalarType t = type == 0 ? at::kFloat : type == 1 ? at::kBFloat16 : at::kHalf;
  at::Tensor y = at::empty(shape, codes.options().dtype(t));
  TORCH_CHECK(y.numel() == codes.numel(), "act8_unpack: the shape has another number of values");
  if (y.numel() == 0) return y;
  for_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    T* v = reinterpret_cast<T*>(y.data_ptr());
    const uint8_t *c = codes.data_ptr<uint8_t>(), *s = scales.data_ptr<uint8_t>();
    const long long units = R * nb * 4;
    if (N % 32 == 0 && aligned(c))
      act8_unpack8_kernel<T, true><<<unit_grid(units), 256, 0, st>>>(c, s, units, (int)N, (int)nb, v);
    else if (N % 8 == 0 && aligned(c))
      act8_unpack8_kernel<T, false><<<unit_grid(units), 256, 0, st>>>(c, s, units, (int)N, (int)nb, v);
    else
      act8_unpack_kernel<T><<<grid_of(R * nb), 256, 0, st>>>(c, s, R, (int)N, (int)nb, v);
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return y;
}

}  // namespace bd
