// feed_forward_b.cu — ff_gemm_kernel with the two products of the gated form.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>

#include "feed_forward_launch.cuh"

namespace bd {

namespace {
template <int EPI>
void go(FfTile t, const FfGemm& p, cudaStream_t st, int dev) {
  if (t.pair)
    ff_launch<EPI, 128, true>(p, st, dev);
  else
    ff_launch<EPI, 64, false>(p, st, dev);
}
}  // namespace

void ff_launch_gated(int epi, FfTile t, const FfGemm& p, cudaStream_t st, int dev) {
  if (epi == FF_GATED)
    go<FF_GATED>(t, p, st, dev);
  else
    go<FF_GATED_BWD>(t, p, st, dev);
}

}  // namespace bd
