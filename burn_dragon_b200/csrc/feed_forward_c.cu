// feed_forward_c.cu — ff_few_kernel, the products of up to 128 rows.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>

#include "feed_forward_launch.cuh"

namespace bd {
namespace {

template <int EPI, int MP>
void launch(const FfGemm& p, cudaStream_t st, int dev) {
  using Cfg = FfFewCfg<ff_products(EPI), MP>;
  auto kern = ff_few_kernel<EPI, MP>;
  static bool attr_set[64] = {false};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    attr_set[dev] = true;
  }
  const long long total = (long long)p.tiles_m * p.splits * p.e.heads;
  kern<<<(unsigned)std::min<long long>(total, num_sms_of(dev)), Cfg::THREADS, Cfg::SMEM, st>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
}

template <int EPI>
void go(int rows, const FfGemm& p, cudaStream_t st, int dev) {
  if (rows == 16)
    launch<EPI, 16>(p, st, dev);
  else if (rows == 64)
    launch<EPI, 64>(p, st, dev);
  else
    launch<EPI, 128>(p, st, dev);
}

}  // namespace

void ff_launch_few(int epi, int rows, const FfGemm& p, cudaStream_t st, int dev) {
  switch (epi) {
    case FF_STORE: return go<FF_STORE>(rows, p, st, dev);
    case FF_ACT: return go<FF_ACT>(rows, p, st, dev);
    case FF_ACT_BWD: return go<FF_ACT_BWD>(rows, p, st, dev);
    case FF_GATED: return go<FF_GATED>(rows, p, st, dev);
    default: return go<FF_GATED_BWD>(rows, p, st, dev);
  }
}

}  // namespace bd
