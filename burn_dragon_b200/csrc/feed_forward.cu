// feed_forward.cu — host side of the feed-forward products (feed_forward.cuh), the sums of split reductions, and the
// backward pass from held pre-activations.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "feed_forward.cuh"
#include "feed_forward_host.h"
#include "gemm_table.h"
#include "launches.h"
#include "tensor_map.h"

namespace bd {
namespace {

// ------------------------------------------------------------------------------- sums of a split reduction

// The parts [splits, NB, sets, heads, M, N] summed in a fixed order, then the epilogue of the unsplit form. A lane takes 4
// columns, eight lanes a block of 32; `ways` of the eight warps (2, 4 or 8) share the parts, so that few columns of many
// parts do not wait for one another. Launched while the products run (programmatic launch): it waits for them itself.
template <int EPI>
__global__ void __launch_bounds__(256) ff_join_kernel(const __grid_constant__ FfOut e, const float* __restrict__ partial,
                                                      int splits, int sets, int ways) {
  constexpr int NB = ff_products(EPI);
  __shared__ float4 red[8][NB][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, way = warp % ways;
  const int groups = (e.N + 31) / 32 * 8;
  const long long at = ((long long)blockIdx.x * (8 / ways) + warp / ways) * 32 + lane;
  const int col = (int)(at % groups) * 4;
  const long long row_of_all = at / groups, rows = (long long)sets * e.heads * e.M;
  const bool in = row_of_all < rows && col < e.N;
  const long long part = rows * e.N;  // of one product
  float v[2][4] = {};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (in) {
#pragma unroll 4
    for (int q = way; q < splits; q += ways)
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        const float4 f = *reinterpret_cast<const float4*>(partial + ((long long)q * NB + s) * part + row_of_all * e.N + col);
        v[s][0] += f.x, v[s][1] += f.y, v[s][2] += f.z, v[s][3] += f.w;
      }
  }
#pragma unroll
  for (int s = 0; s < NB; ++s) red[warp][s][lane] = make_float4(v[s][0], v[s][1], v[s][2], v[s][3]);
  __syncthreads();
  if (way > 0) return;
  for (int q = 1; q < ways; ++q)
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      const float4 f = red[warp + q][s][lane];
      v[s][0] += f.x, v[s][1] += f.y, v[s][2] += f.z, v[s][3] += f.w;
    }
  const int m = (int)(row_of_all % e.M);
  const int head = (int)(row_of_all / e.M % e.heads), set = (int)(row_of_all / e.M / e.heads);
  const long long to = (long long)m * e.ld + (long long)head * e.head + col;
  auto put = [&](void* out, long long where, const float* f) {
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(out) + where) =
        make_uint2(ff_pack2(f[0], f[1], e.half), ff_pack2(f[2], f[3], e.half));
  };
  if constexpr (EPI == FF_STORE) {
    if (in) put(e.out[set], to, v[0]);
  } else {
    if (in) {
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        if (!ff_has_bias(e, s)) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const long long hn = (long long)head * e.N + col + i;
          v[s][i] += !e.bias[s]   ? e.bias0[s]
                     : e.bias_f32 ? reinterpret_cast<const float*>(e.bias[s])[hn]
                                  : ff_as_float(reinterpret_cast<const uint16_t*>(e.bias[s])[hn], e.half);
        }
      }
    }
    const long long rh = (long long)m * e.heads + head;
    if (!ff_backward(EPI) && e.keep != FF_KEEP_NOTHING) {
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        if (e.keep == FF_KEEP_16) {
          if (in) put(e.held[s], rh * e.N + col, v[s]);
        } else {
          float largest = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) largest = fmaxf(largest, in ? act8_size(v[s][i]) : 0.f);
#pragma unroll
          for (int o = 1; o < 8; o *= 2) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
          const int ex = act8_exponent(largest);
          if (in) {
            *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(e.held[s]) + rh * e.N + col) = act8_code4(v[s], act8_power(-ex));
            if (lane % 8 == 0) e.exponents[s][rh * (groups / 8) + col / 32] = (uint8_t)(ex + 127);
          }
        }
      }
    }
    if (!in) return;
    float a[4];
    if (e.aux) {
      const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(e.aux) + (long long)m * e.aux_ld +
                                                      (long long)head * e.aux_head + col);
      put_pair(a, 0, ff_unpack2(r.x, e.half)), put_pair(a, 1, ff_unpack2(r.y, e.half));
    }
    if constexpr (ff_backward(EPI)) {
      ff_with_act(e.act, [&](auto k) {
        ff_backward_values<EPI, 4, decltype(k)::value>(e.up_relu, v[0], v[1], [&](int i) { return pair_of(a, i); });
      });
    } else {
      ff_forward_values<EPI, 4>(e, v[0], v[1]);
      if (EPI == FF_ACT && e.aux) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[0][i] += a[i];
      }
    }
    put(e.out[0], to, v[0]);
    if constexpr (EPI == FF_GATED_BWD) put(e.out[1], to, v[1]);
  }
}

template <int EPI>
void launch_join(const FfOut& e, const float* partial, int splits, int sets, cudaStream_t st) {
  const long long n = (long long)(e.N + 31) / 32 * 8 * sets * e.heads * e.M;
  const int ways = splits >= 8 ? 8 : splits >= 4 ? 4 : 2;
  const long long a_cta = 32 * (8 / ways), grid = (n + a_cta - 1) / a_cta;
  TORCH_CHECK(grid < (1ll << 31), "feed_forward: too many outputs of a split reduction");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, ff_join_kernel<EPI>, e, partial, splits, sets, ways));
  ++counted_launches;
}

// ------------------------------------------------------------------------------- backward from held pre-activations

// dp (or dg, du) from dy and what the forward pass held: 32 rows x 256 columns of a head a CTA, 8 columns a lane. KEEP
// nothing: only the column sums of dy. Bound by bytes.
template <int EPI, int KEEP>
__global__ void __launch_bounds__(256) ff_held_kernel(const __grid_constant__ FfOut e) {
  constexpr int NB = ff_products(EPI);
  __shared__ float red[8][8 * NB][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int head = blockIdx.y, col = ((int)blockIdx.x * 32 + lane) * 8, nb = (e.N + 31) / 32;
  const bool in = col < e.N;
  float sum[NB][8];
#pragma unroll
  for (int s = 0; s < NB; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[s][i] = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int m = (int)blockIdx.z * 32 + j * 8 + warp;
    if (!in || m >= e.M) continue;
    const long long rh = (long long)m * e.heads + head;
    float a[8], v[2][8];
    ff_unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(e.aux) + (long long)m * e.aux_ld +
                                               (long long)head * e.aux_head + col),
               e.half, a);
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      if constexpr (KEEP == FF_KEEP_16) {
        ff_unpack8(*reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(e.held[s]) + rh * e.N + col), e.half, v[s]);
      } else if constexpr (KEEP == FF_KEEP_8) {
        const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(e.held[s]) + rh * e.N + col);
        const float scale = act8_power((int)e.exponents[s][rh * nb + col / 32] - 127);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = act8_value2(((i < 2 ? c.x : c.y) >> (16 * (i & 1))) & 0xFFFFu, scale, kAct8LimitF32);
          v[s][2 * i] = f.x, v[s][2 * i + 1] = f.y;
        }
      }
    }
    if constexpr (KEEP != FF_KEEP_NOTHING) {
      ff_with_act(e.act, [&](auto k) {
        ff_backward_values<EPI, 8, decltype(k)::value>(e.up_relu, v[0], v[1], [&](int i) { return pair_of(a, i); });
      });
      const long long to = (long long)m * e.ld + (long long)head * e.head + col;
#pragma unroll
      for (int s = 0; s < NB; ++s)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(e.out[s]) + to) = ff_pack8(v[s], e.half);
#pragma unroll
      for (int s = 0; s < NB; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[s][i] += v[s][i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[0][i] += a[i];
    }
  }
  if (!e.colsum[0] && !e.colsum[1]) return;
#pragma unroll
  for (int s = 0; s < NB; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i) red[warp][8 * s + i][lane] = sum[s][i];
  __syncthreads();
  if (warp >= NB || !in || !e.colsum[warp]) return;
  float* o = e.colsum[warp] + ((long long)blockIdx.z * e.heads + head) * e.N + col;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float f = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) f += red[q][8 * warp + i][lane];
    o[i] = f;
  }
}

// [B, R, C] of any strides (the last 1) to [B, R8, C8], zeros behind: 8 values a thread. Rows of odd lengths cannot be read
// by TMA; torch's constant padding took 150 us for a weight of 32 MB.
__global__ void __launch_bounds__(256) ff_pad_kernel(const uint16_t* __restrict__ in, long long in_batch, long long in_row,
                                                     int R, int C, uint4* __restrict__ out, int R8, int C8, long long units) {
  const int per_row = C8 / 8;
  for (long long u = (long long)blockIdx.x * 256 + threadIdx.x; u < units; u += (long long)gridDim.x * 256) {
    const long long row = u / per_row;
    const int c = (int)(u - row * per_row) * 8, b = (int)(row / R8), r = (int)(row - (long long)b * R8);
    uint32_t v[4] = {0, 0, 0, 0};
    if (r < R) {
      const uint16_t* src = in + b * in_batch + r * in_row + c;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < C) v[i / 2] |= (uint32_t)src[i] << (16 * (i & 1));
    }
    out[u] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

// out [C] = the sum over R rows of part [R, C], in a fixed order: a column a lane, every eighth row a warp.
template <typename T>
__global__ void __launch_bounds__(256) ff_colsum_kernel(const float* __restrict__ part, int R, long long C, T* __restrict__ out) {
  __shared__ float red[8][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long c = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int r = warp; r < R; r += 8) s += part[r * C + c];
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp > 0 || c >= C) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) s += red[q][lane];
  if constexpr (sizeof(T) == 4)
    out[c] = s;
  else if constexpr (std::is_same<T, __half>::value)
    out[c] = __float2half_rn(s);
  else
    out[c] = __float2bfloat16_rn(s);
}

// ------------------------------------------------------------------------------- host

// A matrix of 16-bit values, or one a head: [heads, rows, cols] with the contiguous dimension found.
struct Mat {
  const void* p;
  int64_t inner, outer, heads;  // extents: contiguous, other
  int64_t ld, head;             // strides in values
  bool per_head;
  CUtensorMap map(uint32_t box_outer) const {
    return tensor_map_bf16(p, {inner, outer, per_head ? heads : 1}, {ld, per_head ? head : ld * outer}, 64, box_outer);
  }
};

// Rows [M, C] or [M, H, C] as an operand.
Mat rows_of(const at::Tensor& t) {
  const bool per = t.dim() == 3;
  return Mat{t.data_ptr(), t.size(-1), t.size(0), per ? t.size(1) : 1, t.stride(0), per ? t.stride(1) : 0, per};
}

// A weight [H, K, N]; `turned`: K is contiguous.
Mat weight_of(const at::Tensor& w, bool& turned) {
  turned = w.stride(2) != 1;
  return Mat{w.data_ptr(), w.size(turned ? 1 : 2), w.size(turned ? 2 : 1), w.size(0), w.stride(turned ? 2 : 1), w.stride(0), true};
}

// Clocks of one launch, by a model of the busiest CTA, from measured loops: a 64-wide block takes at least 800 (its way
// through the ring where few CTAs run), 60 % of the tensor core's rate, or what its operands take into shared memory (40 bytes a
// clock); a tile 1500 of its own; a split reduction writes and reads its parts and starts another kernel.
struct Choice {
  FfTile tile;
  int splits;
};

Choice choose(int64_t rows, int64_t cols, int64_t batch, int64_t blocks, int nb, int a_count, int sms, bool may_split) {
  struct Option {
    bool pair;
    int bn;
  };
  const Option one[] = {{true, 256}, {true, 128}, {false, 128}, {false, 64}}, two[] = {{true, 128}, {false, 64}};
  const Option* options = nb == 1 ? one : two;
  Choice best{{false, 64}, 1};
  double least = 1e300;
  for (int i = 0; i < (nb == 1 ? 4 : 2); ++i) {
    const Option o = options[i];
    if (o.pair && rows <= 128) continue;
    const int ctas = o.pair ? 2 : 1;
    const int64_t tiles = (rows + 128 * ctas - 1) / (128 * ctas) * ((cols + o.bn - 1) / o.bn) * batch;
    const int64_t workers = sms / ctas;
    const double block = std::max({800.0, 3.3 * nb * o.bn, (a_count * 16384.0 + nb * (o.bn / ctas) * 128.0) / 40.0});
    for (int64_t parts = 1; parts == 1 || (may_split && parts <= blocks / 2); ++parts) {
      if (parts > 1 && tiles * parts > workers) break;
      const double waves = (double)((tiles * parts + workers - 1) / workers);
      double cost = waves * ((double)((blocks + parts - 1) / parts) * block + 1500.0);
      if (parts > 1) cost += 5000.0 + 8.0 * parts * rows * cols * batch * nb / 3000.0;
      if (cost < least) least = cost, best = Choice{{o.pair, o.bn}, (int)parts};
    }
  }
  return best;
}

// The same for few rows: a block is the weights' bytes at an SM's share of the memory's (23 a clock).
constexpr int kFewRows = 128;

Choice choose_few(int64_t rows, int64_t cols, int64_t batch, int64_t blocks, int nb, int sms, bool may_split) {
  const int64_t tiles = (cols + 127) / 128 * batch;
  Choice best{{false, rows <= 16 ? 16 : rows <= 64 ? 64 : 128}, 1};
  double least = 1e300;
  for (int64_t parts = 1; parts == 1 || (may_split && parts <= blocks / 2 && tiles * parts <= sms); ++parts) {
    const double waves = (double)((tiles * parts + sms - 1) / sms);
    double cost = waves * ((double)((blocks + parts - 1) / parts) * nb * 712.0 + 1200.0);
    if (parts > 1) cost += 4000.0 + 8.0 * parts * rows * cols * batch * nb / 3000.0;
    if (cost < least) least = cost, best.splits = (int)parts;
  }
  return best;
}

struct Launch {
  cudaStream_t st;
  int dev;
  int* err;
  at::TensorOptions options;
};

uint32_t idesc_of(bool pair, int bn, bool half, bool a_mn) {
  uint32_t d = make_idesc_bf16(pair ? 256 : 128, bn, a_mn, false);
  if (half) d &= ~((1u << 7) | (1u << 10));  // f16 operands
  return d;
}

// The walk's constants, room for the parts of a split reduction, the launch, and their sum.
void split_and_launch(const Launch& l, int epi, const FfOut& e, FfGemm& p, const Choice& c, int64_t batch, int out_sets, int nb,
                      int ctas, bool few) {
  const int64_t total = (int64_t)p.tiles_m * p.tiles_n * p.splits * batch;
  TORCH_CHECK(total < (1ll << 31), "feed_forward: too many tiles");
  const unsigned sizes[4] = {(unsigned)p.tiles_n, (unsigned)p.tiles_m, (unsigned)p.splits, (unsigned)e.heads};
  unsigned step = (unsigned)std::min<int64_t>(total, num_sms_of(l.dev) / ctas);
  for (int i = 0; i < 4; ++i) {
    p.size[i] = sizes[i];
    p.step[i] = step % sizes[i];
    step /= sizes[i];
  }
  p.step[4] = step;
  at::Tensor partial;
  if (p.splits > 1) {
    partial = at::empty({(int64_t)p.splits * nb * batch * e.M * e.N}, l.options.dtype(at::kFloat));
    p.partial = partial.data_ptr<float>();
  }
  p.e = e;
  if (few)
    ff_launch_few(epi, c.tile.bn, p, l.st, l.dev);
  else if (nb == 1)
    ff_launch_one(epi, c.tile, p, l.st, l.dev);
  else
    ff_launch_gated(epi, c.tile, p, l.st, l.dev);
  if (p.splits > 1) {
    switch (epi) {
      case FF_STORE: launch_join<FF_STORE>(e, p.partial, p.splits, out_sets, l.st); break;
      case FF_ACT: launch_join<FF_ACT>(e, p.partial, p.splits, out_sets, l.st); break;
      case FF_ACT_BWD: launch_join<FF_ACT_BWD>(e, p.partial, p.splits, out_sets, l.st); break;
      case FF_GATED: launch_join<FF_GATED>(e, p.partial, p.splits, out_sets, l.st); break;
      default: launch_join<FF_GATED_BWD>(e, p.partial, p.splits, out_sets, l.st);
    }
  }
}

// One launch (two where the reduction is split): rows x cols outputs of e, the reduction `depth` long in each of
// `segments` pairs of operands. a, b: one or two sets.
void product(const Launch& l, int epi, FfOut e, const Mat* a, const Mat* b, int sets, int64_t depth, int segments,
             int sum_heads, int out_sets, bool a_mn, const bool* b_mn, bool two_a, bool may_split) {
  const int nb = ff_products(epi);
  FfGemm p;
  memset(&p, 0, sizeof(p));
  p.KB = (int)((depth + 63) / 64);
  p.segments = segments, p.sum_heads = sum_heads, p.out_sets = out_sets;
  p.two_a = two_a;
  p.err = l.err;
  const int64_t blocks = (int64_t)p.KB * segments, batch = (int64_t)e.heads * out_sets;
  const bool few = e.M <= kFewRows && !a_mn && out_sets == 1;
  const Choice c = few ? choose_few(e.M, e.N, batch, blocks, nb, num_sms_of(l.dev), may_split) : choose(e.M, e.N, batch, blocks, nb, nb == 2 && two_a ? 2 : 1, num_sms_of(l.dev), may_split);
  p.splits = c.splits;
  TORCH_CHECK(blocks * (c.splits + 1) < (1ll << 32), "feed_forward: the reduction is too long");
  if (few) {
    p.tiles_m = (e.N + 127) / 128, p.tiles_n = 1;
    p.idesc = idesc_of(false, c.tile.bn, e.half, false);
    for (int s = 0; s < 2; ++s) {
      const int q = s < sets ? s : 0;
      p.ta[s] = b[q].map(b_mn[q] ? 64 : 128);
      p.tb[s] = a[q].map((uint32_t)c.tile.bn);
      if (b[q].per_head) p.a_heads |= 1 << s;
      if (a[q].per_head) p.b_heads |= 1 << s;
      p.a_mn |= b_mn[q] ? (nb == 2 ? 1 << s : 1) : 0;
    }
    split_and_launch(l, epi, e, p, c, batch, out_sets, nb, 1, true);
    return;
  }
  const int rows = c.tile.pair ? 256 : 128, b_rows = c.tile.pair ? c.tile.bn / 2 : c.tile.bn;
  p.tiles_m = (e.M + rows - 1) / rows, p.tiles_n = (e.N + c.tile.bn - 1) / c.tile.bn;
  p.a_mn = a_mn;
  for (int s = 0; s < 2; ++s) {
    const int q = s < sets ? s : 0;
    if (s > 0 && q == 0) {
      p.ta[1] = p.ta[0], p.tb[1] = p.tb[0];
      p.a_heads |= (p.a_heads & 1) << 1, p.b_heads |= (p.b_heads & 1) << 1;
      break;
    }
    p.ta[s] = a[q].map(a_mn ? 64 : 128);
    p.tb[s] = b[q].map(b_mn[q] ? 64 : (uint32_t)b_rows);
    if (a[q].per_head) p.a_heads |= 1 << s;
    if (b[q].per_head) p.b_heads |= 1 << s;
    if (b_mn[q]) p.b_mn |= nb == 2 ? 1 << s : 1;
  }
  p.idesc = idesc_of(c.tile.pair, c.tile.bn, e.half, a_mn);
  split_and_launch(l, epi, e, p, c, batch, out_sets, nb, c.tile.pair ? 2 : 1, false);
}

void check_rows(const at::Tensor& t, int dev, at::ScalarType type, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == dev && t.scalar_type() == type, "feed_forward: ", what,
              " must lie on the operands' GPU and have their type");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "feed_forward: ", what, " must be 16-byte aligned");
  TORCH_CHECK(t.stride(-1) == 1, "feed_forward: ", what, " must be contiguous in its last dimension");
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    TORCH_CHECK(t.stride(i) % 8 == 0 && t.stride(i) > 0, "feed_forward: ", what, ": strides must be multiples of 8 values");
}

void check_weight(const at::Tensor& w, int dev, at::ScalarType type) {
  TORCH_CHECK(w.is_cuda() && w.get_device() == dev && w.scalar_type() == type && w.dim() == 3,
              "feed_forward: weights [H, K, N] of the operands' type on one GPU");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 && (w.stride(1) == 1 || w.stride(2) == 1),
              "feed_forward: weights must be 16-byte aligned and contiguous along K or N");
  const int64_t other = w.stride(2) == 1 ? w.stride(1) : w.stride(2);
  TORCH_CHECK(other % 8 == 0 && other > 0 && w.stride(0) % 8 == 0 && w.stride(0) > 0,
              "feed_forward: weight strides must be multiples of 8 values");
}

// What a call is about, checked.
struct Layer {
  int nb, dev, act;
  int64_t M, H, K, N;
  bool two_a, half;
  at::ScalarType type;
  Mat x[2], w[2];
  bool turned[2];
  FfOut e;  // with biases, activation, sizes
  Launch l;
};

Layer layer_of(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu, const OptTensor& bg,
               const OptTensor& bu, double bg0, double bu0, int64_t act, bool up_relu, const at::Tensor& err) {
  Layer c;
  c.dev = wg.get_device(), c.type = wg.scalar_type();
  TORCH_CHECK(c.type == at::kBFloat16 || c.type == at::kHalf, "feed_forward: bf16 or fp16 operands");
  c.half = c.type == at::kHalf;
  c.nb = wu ? 2 : 1, c.two_a = z.has_value(), c.act = (int)act;
  TORCH_CHECK(act >= 0 && act <= 3 && (c.nb == 2 || !c.two_a), "feed_forward: bad call");
  check_weight(wg, c.dev, c.type);
  c.H = wg.size(0), c.K = wg.size(1), c.N = wg.size(2), c.M = x.size(0);
  const int64_t big = 1ll << 30;
  TORCH_CHECK(c.K > 0 && c.N > 0 && c.K % 8 == 0 && c.N % 8 == 0 && c.M > 0 && c.H > 0 && c.M < big && c.K < big && c.N < big &&
                  c.H <= 65535,
              "feed_forward: K and N must be multiples of 8, at most 2^30 rows, 65535 heads");
  auto rows = [&](const at::Tensor& t, const char* what) {
    check_rows(t, c.dev, c.type, what);
    TORCH_CHECK((t.dim() == 2 || (t.dim() == 3 && t.size(1) == c.H)) && t.size(0) == c.M && t.size(-1) == c.K, "feed_forward: ",
                what, " must be [M, K] or [M, H, K]");
    return rows_of(t);
  };
  c.x[0] = rows(x, "x");
  c.x[1] = z ? rows(*z, "z") : c.x[0];
  c.w[0] = weight_of(wg, c.turned[0]);
  if (wu) {
    check_weight(*wu, c.dev, c.type);
    TORCH_CHECK(wu->sizes() == wg.sizes(), "feed_forward: both weights must have one shape");
    c.w[1] = weight_of(*wu, c.turned[1]);
  } else {
    c.w[1] = c.w[0], c.turned[1] = c.turned[0];
  }
  memset(&c.e, 0, sizeof(c.e));
  FfOut& e = c.e;
  e.act = (int)act, e.up_relu = up_relu, e.half = c.half;
  e.M = (int)c.M, e.N = (int)c.N, e.heads = (int)c.H;
  e.ld = c.H * c.N, e.head = c.N;
  const OptTensor* biases[2] = {&bg, &bu};
  int kinds = 0;
  for (int s = 0; s < 2; ++s) {
    if (!biases[s]->has_value()) continue;
    const at::Tensor& b = **biases[s];
    TORCH_CHECK(b.is_cuda() && b.get_device() == c.dev && b.is_contiguous() && b.numel() == c.H * c.N &&
                    (b.scalar_type() == c.type || b.scalar_type() == at::kFloat) &&
                    reinterpret_cast<uintptr_t>(b.data_ptr()) % 16 == 0,
                "feed_forward: a bias [H, N], contiguous, fp32 or of the operands' type");
    e.bias[s] = b.data_ptr();
    e.bias_f32 = b.scalar_type() == at::kFloat;
    kinds |= e.bias_f32 ? 1 : 2;
  }
  TORCH_CHECK(kinds != 3, "feed_forward: both biases must have one type");
  e.bias0[0] = (float)bg0, e.bias0[1] = (float)bu0;
  TORCH_CHECK(err.is_cuda() && err.get_device() == c.dev && err.scalar_type() == at::kInt, "feed_forward: bad error word");
  c.l = Launch{at::cuda::getCurrentCUDAStream(c.dev).stream(), c.dev, err.data_ptr<int>(), wg.options()};
  return c;
}

// The layer's own products, with epilogue `epi`.
void forward_products(const Layer& c, int epi, const FfOut& e, bool may_split) {
  const bool b_mn[2] = {!c.turned[0], !c.turned[1]};
  product(c.l, epi, e, c.x, c.w, c.nb, c.K, 1, 1, 1, false, b_mn, c.two_a, may_split);
}

}  // namespace

std::vector<at::Tensor> ff_forward(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu,
                                   const OptTensor& bg, const OptTensor& bu, double bg0, double bu0, const OptTensor& residual,
                                   int64_t act, bool up_relu, int64_t keep, const at::Tensor& err) {
  Layer c = layer_of(x, z, wg, wu, bg, bu, bg0, bu0, act, up_relu, err);
  c10::cuda::CUDAGuard guard(c.dev);
  c.l.st = at::cuda::getCurrentCUDAStream(c.dev).stream();
  std::vector<at::Tensor> out{at::empty({c.M, c.H, c.N}, wg.options())};
  FfOut e = c.e;
  e.out[0] = out[0].data_ptr();
  e.keep = (int)keep;
  for (int s = 0; s < c.nb && keep != FF_KEEP_NOTHING; ++s) {
    const auto bytes = wg.options().dtype(at::kByte);
    out.push_back(at::empty({c.M, c.H, c.N}, keep == FF_KEEP_8 ? bytes : wg.options()));
    e.held[s] = out.back().data_ptr();
    if (keep == FF_KEEP_8) {
      out.push_back(at::empty({c.M, c.H, (c.N + 31) / 32}, bytes));
      e.exponents[s] = out.back().data_ptr<uint8_t>();
    }
  }
  if (residual) {
    check_rows(*residual, c.dev, c.type, "residual");
    TORCH_CHECK(c.nb == 1 && residual->dim() == 3 && residual->size(0) == c.M && residual->size(1) == c.H &&
                    residual->size(2) == c.N,
                "feed_forward: residual [M, H, N]");
    e.aux = residual->data_ptr(), e.aux_ld = residual->stride(0), e.aux_head = residual->stride(1);
  }
  forward_products(c, c.nb == 2 ? FF_GATED : FF_ACT, e, true);
  return out;
}

std::vector<at::Tensor> ff_backward(const at::Tensor& dy, const at::Tensor& x, const OptTensor& z, const at::Tensor& wg,
                                    const OptTensor& wu, const OptTensor& bg, const OptTensor& bu, double bg0, double bu0,
                                    const std::vector<at::Tensor>& held, int64_t act, bool up_relu, int64_t keep,
                                    int64_t want, const at::Tensor& err) {
  Layer c = layer_of(x, z, wg, wu, bg, bu, bg0, bu0, act, up_relu, err);
  c10::cuda::CUDAGuard guard(c.dev);
  c.l.st = at::cuda::getCurrentCUDAStream(c.dev).stream();
  check_rows(dy, c.dev, c.type, "dy");
  TORCH_CHECK(dy.dim() == 3 && dy.size(0) == c.M && dy.size(1) == c.H && dy.size(2) == c.N, "feed_forward: dy [M, H, N]");
  at::Tensor none = at::empty({0}, wg.options());
  std::vector<at::Tensor> out(6, none);
  const bool want_x = want & 1, want_z = want & 2, want_w[2] = {(want & 4) != 0, (want & 8) != 0},
             want_b[2] = {(want & 16) != 0, (want & 32) != 0};

  // ---- dp, and the biases' gradients
  FfOut e = c.e;
  e.aux = dy.data_ptr(), e.aux_ld = dy.stride(0), e.aux_head = dy.stride(1);
  at::Tensor dp[2], sums[2];
  const int64_t row_blocks = (c.M + 31) / 32;
  for (int s = 0; s < c.nb; ++s)
    if (want_b[s]) {
      sums[s] = at::empty({row_blocks, c.H * c.N}, wg.options().dtype(at::kFloat));
      e.colsum[s] = sums[s].data_ptr<float>();
    }
  const bool sums_wanted = want_b[0] || want_b[1];
  const bool plain = c.nb == 1 && c.act == FF_NONE;  // dp is dy
  const bool needs_dp = want_x || want_z || want_w[0] || want_w[1] || sums_wanted;
  if (!needs_dp) return out;
  const dim3 held_grid((unsigned)((c.N + 255) / 256), (unsigned)c.H, (unsigned)row_blocks);
  TORCH_CHECK(row_blocks <= 65535 || (keep == FF_KEEP_NOTHING && !plain), "feed_forward: at most 2097120 rows in a backward pass");
  if (plain) {
    dp[0] = dy;
    if (sums_wanted) {
      ff_held_kernel<FF_ACT_BWD, FF_KEEP_NOTHING><<<held_grid, 256, 0, c.l.st>>>(e);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++counted_launches;
    }
  } else {
    for (int s = 0; s < c.nb; ++s) {
      dp[s] = at::empty({c.M, c.H, c.N}, wg.options());
      e.out[s] = dp[s].data_ptr();
    }
    if (keep == FF_KEEP_NOTHING) {
      forward_products(c, c.nb == 2 ? FF_GATED_BWD : FF_ACT_BWD, e, !sums_wanted);
    } else {
      const size_t each = keep == FF_KEEP_8 ? 2 : 1;
      TORCH_CHECK(held.size() == each * c.nb, "feed_forward: bad held pre-activations");
      for (int s = 0; s < c.nb; ++s) {
        const at::Tensor& h = held[each * s];
        TORCH_CHECK(h.is_cuda() && h.get_device() == c.dev && h.is_contiguous() && h.numel() == c.M * c.H * c.N &&
                        h.scalar_type() == (keep == FF_KEEP_8 ? at::kByte : c.type),
                    "feed_forward: bad held pre-activations");
        e.held[s] = h.data_ptr();
        if (keep == FF_KEEP_8) {
          const at::Tensor& x8 = held[each * s + 1];
          TORCH_CHECK(x8.is_cuda() && x8.get_device() == c.dev && x8.is_contiguous() && x8.scalar_type() == at::kByte &&
                          x8.numel() == c.M * c.H * ((c.N + 31) / 32),
                      "feed_forward: bad exponents");
          e.exponents[s] = x8.data_ptr<uint8_t>();
        }
      }
      if (c.nb == 2) {
        if (keep == FF_KEEP_8)
          ff_held_kernel<FF_GATED_BWD, FF_KEEP_8><<<held_grid, 256, 0, c.l.st>>>(e);
        else
          ff_held_kernel<FF_GATED_BWD, FF_KEEP_16><<<held_grid, 256, 0, c.l.st>>>(e);
      } else {
        if (keep == FF_KEEP_8)
          ff_held_kernel<FF_ACT_BWD, FF_KEEP_8><<<held_grid, 256, 0, c.l.st>>>(e);
        else
          ff_held_kernel<FF_ACT_BWD, FF_KEEP_16><<<held_grid, 256, 0, c.l.st>>>(e);
      }
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++counted_launches;
    }
  }
  for (int s = 0; s < c.nb; ++s)
    if (want_b[s]) {
      const at::Tensor& b = s ? *bu : *bg;
      out[4 + s] = at::empty_like(b);
      const long long C = c.H * c.N;
      const unsigned grid = (unsigned)((C + 31) / 32);
      if (b.scalar_type() == at::kFloat)
        ff_colsum_kernel<float><<<grid, 256, 0, c.l.st>>>(sums[s].data_ptr<float>(), (int)row_blocks, C, out[4 + s].data_ptr<float>());
      else if (c.half)
        ff_colsum_kernel<__half><<<grid, 256, 0, c.l.st>>>(sums[s].data_ptr<float>(), (int)row_blocks, C,
                                                           reinterpret_cast<__half*>(out[4 + s].data_ptr()));
      else
        ff_colsum_kernel<__nv_bfloat16><<<grid, 256, 0, c.l.st>>>(sums[s].data_ptr<float>(), (int)row_blocks, C,
                                                                  reinterpret_cast<__nv_bfloat16*>(out[4 + s].data_ptr()));
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      ++counted_launches;
    }
  const Mat d[2] = {rows_of(dp[0]), rows_of(c.nb == 2 ? dp[1] : dp[0])};
  FfOut g;
  memset(&g, 0, sizeof(g));
  g.half = c.half;

  // ---- dx = dp W^T: the reduction is N long, over one or both projections, and over the heads where they share the input
  auto input_grad = [&](const at::Tensor& like, int first, int sets) {
    at::Tensor o = at::empty(like.sizes(), wg.options());
    const bool shared = like.dim() == 2;
    g.M = (int)c.M, g.N = (int)c.K, g.heads = shared ? 1 : (int)c.H;
    g.ld = o.stride(0), g.head = shared ? 0 : o.stride(1);
    g.out[0] = o.data_ptr(), g.out[1] = nullptr;
    const bool b_mn[2] = {c.turned[first], c.turned[first + sets - 1]};
    const int sum_heads = shared ? (int)c.H : 1;
    auto run = [&](int from, int n) {
      product(c.l, FF_STORE, g, d + from, c.w + from, n, c.N, n * sum_heads, sum_heads, 1, false, b_mn, false, true);
    };
    run(first, sets);
    return o;
  };
  if (c.nb == 2 && !c.two_a) {
    if (want_x) {
      TORCH_CHECK(c.turned[0] == c.turned[1], "feed_forward: one input of two projections wants their weights laid out alike");
      out[0] = input_grad(x, 0, 2);
    }
  } else {
    if (want_x) out[0] = input_grad(x, 0, 1);
    if (want_z && c.nb == 2) out[1] = input_grad(*z, 1, 1);
  }

  // ---- dW = x^T dp, laid out as the weight: the reduction is over the rows
  auto weight_grad = [&](int first, int sets) {
    const bool turned = c.turned[first];
    g.M = (int)(turned ? c.N : c.K), g.N = (int)(turned ? c.K : c.N), g.heads = (int)c.H;
    g.ld = g.N, g.head = (long long)g.M * g.N;
    for (int s = 0; s < sets; ++s) {
      at::Tensor o = at::empty({c.H, g.M, g.N}, wg.options());
      g.out[s] = o.data_ptr();
      out[2 + first + s] = turned ? o.transpose(1, 2) : o;
    }
    const bool mn[2] = {true, true};
    const Mat* a = turned ? d + first : c.x + first;
    const Mat* b = turned ? c.x + first : d + first;
    product(c.l, FF_STORE, g, a, b, sets, c.M, 1, 1, sets, true, mn, false, true);
  };
  if (c.nb == 2 && want_w[0] && want_w[1] && c.turned[0] == c.turned[1]) {
    weight_grad(0, 2);
  } else {
    if (want_w[0]) weight_grad(0, 1);
    if (want_w[1] && c.nb == 2) weight_grad(1, 1);
  }
  return out;
}

at::Tensor ff_pad(const at::Tensor& t, int64_t R8, int64_t C8) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3 && t.element_size() == 2 && (t.stride(2) == 1 || t.size(2) <= 1) && C8 % 8 == 0 &&
                  R8 >= t.size(1) && C8 >= t.size(2) && R8 < (1ll << 31) && C8 < (1ll << 31),
              "ff_pad: [B, R, C] of 16-bit values, contiguous in C");
  c10::cuda::CUDAGuard guard(t.get_device());
  at::Tensor out = at::empty({t.size(0), R8, C8}, t.options().requires_grad(false));
  const long long units = out.numel() / 8;
  if (units == 0) return out;
  ff_pad_kernel<<<(unsigned)std::min<long long>((units + 255) / 256, 148 * 16), 256, 0,
                  at::cuda::getCurrentCUDAStream(t.get_device()).stream()>>>(
      reinterpret_cast<const uint16_t*>(t.data_ptr()), t.stride(0), t.stride(1), (int)t.size(1), (int)t.size(2),
      reinterpret_cast<uint4*>(out.data_ptr()), (int)R8, (int)C8, units);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return out;
}

}  // namespace bd
