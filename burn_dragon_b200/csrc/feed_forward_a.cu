// feed_forward_a.cu — ff_gemm_kernel with one product.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include <algorithm>

#include "feed_forward_launch.cuh"

namespace bd {

namespace {
template <int EPI>
void go(FfTile t, const FfGemm& p, cudaStream_t st, int dev) {
  if (t.pair && t.bn == 256)
    ff_launch<EPI, 256, true>(p, st, dev);
  else if (t.pair)
    ff_launch<EPI, 128, true>(p, st, dev);
  else if (t.bn == 128)
    ff_launch<EPI, 128, false>(p, st, dev);
  else
    ff_launch<EPI, 64, false>(p, st, dev);
}
}  // namespace

void ff_launch_one(int epi, FfTile t, const FfGemm& p, cudaStream_t st, int dev) {
  if (epi == FF_STORE)
    go<FF_STORE>(t, p, st, dev);
  else if (epi == FF_ACT)
    go<FF_ACT>(t, p, st, dev);
  else
    go<FF_ACT_BWD>(t, p, st, dev);
}

}  // namespace bd
