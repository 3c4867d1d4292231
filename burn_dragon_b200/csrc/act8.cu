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

}  // namespace

// x [R, N] contiguous -> codes [R, N] and exponents [R, ceil(N / 32)], uint8.
std::vector<at::Tensor> act8_pack(const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "act8_pack: contiguous rows [R, N] on a GPU");
  const int64_t R = x.size(0), N = x.size(1), nb = (N + 31) / 32;
  TORCH_CHECK(N < (1ll << 31) - 32, "act8_pack: rows of less than 2^31 - 32 values");
  c10::cuda::CUDAGuard guard(x.get_device());
  auto st = at::cuda::getCurrentCUDAStream(x.get_device()).stream();
  at::Tensor codes = at::empty({R, N}, x.options().dtype(at::kByte)), scales = at::empty({R, nb}, codes.options());
  if (x.numel() == 0) return {codes, scales};
  for_type(x.scalar_type(), [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    act8_pack_kernel<T><<<grid_of(R * nb), 256, 0, st>>>(reinterpret_cast<const T*>(x.data_ptr()), R, (int)N, (int)nb,
                                                         codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>());
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return {codes, scales};
}

// The values [R, N] that codes and exponents stand for, as `like`'s type.
at::Tensor act8_unpack(const at::Tensor& codes, const at::Tensor& scales, int64_t type) {
  TORCH_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.is_contiguous() && codes.scalar_type() == at::kByte,
              "act8_unpack: contiguous codes [R, N]");
  const int64_t R = codes.size(0), N = codes.size(1), nb = (N + 31) / 32;
  TORCH_CHECK(scales.is_cuda() && scales.get_device() == codes.get_device() && scales.scalar_type() == at::kByte &&
                  scales.is_contiguous() && scales.dim() == 2 && scales.size(0) == R && scales.size(1) == nb,
              "act8_unpack: exponents [R, ceil(N / 32)]");
  c10::cuda::CUDAGuard guard(codes.get_device());
  auto st = at::cuda::getCurrentCUDAStream(codes.get_device()).stream();
  const at::ScalarType t = type == 0 ? at::kFloat : type == 1 ? at::kBFloat16 : at::kHalf;
  at::Tensor y = at::empty({R, N}, codes.options().dtype(t));
  if (y.numel() == 0) return y;
  for_type(t, [&](auto* p) {
    using T = std::remove_pointer_t<decltype(p)>;
    act8_unpack_kernel<T><<<grid_of(R * nb), 256, 0, st>>>(codes.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(), R, (int)N,
                                                           (int)nb, reinterpret_cast<T*>(y.data_ptr()));
  });
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return y;
}

}  // namespace bd
