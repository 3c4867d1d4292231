// feed_forward_launch.cuh — one launch of ff_gemm_kernel, shared by its instantiation units.
#pragma once
#include <c10/cuda/CUDAException.h>

#include "feed_forward.cuh"
#include "gemm_table.h"
#include "launches.h"

namespace bd {

template <int EPI, int BN, bool PAIR>
void ff_launch(const FfGemm& p, cudaStream_t st, int dev) {
  using Cfg = FfCfg<EPI, BN, PAIR>;
  auto kern = ff_gemm_kernel<EPI, BN, PAIR>;
  static bool attr_set[64] = {false};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    attr_set[dev] = true;
  }
  const long long total = (long long)p.tiles_m * p.tiles_n * p.splits * p.e.heads * p.out_sets;
  const long long workers = ff_workers(total, FfTile{PAIR, BN}, num_sms_of(dev));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(workers * Cfg::CTAS));
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = Cfg::CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  ++counted_launches;
}

}  // namespace bd
