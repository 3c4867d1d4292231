// feed_forward_b.cu — ff_gemm_kernel with the two products of the gated form.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>

#include "feed_forward_launch.cuh"

namespace bd {

void ff_launch_gated(int epi, FfTile t, const FfGemm& p, cudaStream_t st, int dev) {
  if (epi == FF_GATED)
    t.pair ? ff_launch<FF_GATED, 128, true>(p, st, dev) : ff_launch<FF_GATED, 64, false>(p, st, dev);
  else
    t.pair ? ff_launch<FF_GATED_BWD, 128, true>(p, st, dev) : ff_launch<FF_GATED_BWD, 64, false>(p, st, dev);
}

}  // namespace bd
