// feed_forward.cuh — the products of a feed-forward layer on tcgen05, with the layer's arithmetic in their epilogue.
//
//   linear:  p = x W + b,             y = act(p) + r
//   gated:   g = x Wg + bg, u = z Wu + bu,  y = act(g) up(u)        (z may be x; up is the identity or relu)
// and in the backward pass, from the same products or from held pre-activations,
//   dp = dy act'(p);   dg = dy up(u) act'(g), du = dy act(g) up'(u);
//   dx = dp W^T (a sum over both projections and over the heads that share x), dW = x^T dp, db = sum of dp's rows.
//
// ff_gemm is persistent and warp-specialised like the GEMM engine (TMA producer, one MMA issuer, eight epilogue
// warps; two TMEM accumulators, so an epilogue runs under the next tile's products). What is its own: a tile has NB
// accumulators side by side (the gated form's two projections are one pass over x, and their product never
// leaves the SM), a reduction may run over several pairs of operands (dx), any tile may hold several operand sets
// (both weight gradients in one launch), and the majorness of both operands is a run-time flag, for the two threads that
// read it are not what bounds the kernel. With PAIR two CTAs share a 256-row tile (cta_group::2): each stages its 128
// rows of A and half of B.
#pragma once
#include <cuda_fp16.h>

#include "act8.cuh"
#include "sm100_ptx.cuh"

namespace bd {

enum FfEpi : int { FF_STORE = 0, FF_ACT = 1, FF_ACT_BWD = 2, FF_GATED = 3, FF_GATED_BWD = 4 };
enum FfAct : int { FF_NONE = 0, FF_RELU = 1, FF_SILU = 2, FF_GELU = 3 };
enum FfKeep : int { FF_KEEP_NOTHING = 0, FF_KEEP_16 = 1, FF_KEEP_8 = 2 };

constexpr bool ff_backward(int epi) { return epi == FF_ACT_BWD || epi == FF_GATED_BWD; }
constexpr int ff_products(int epi) { return epi >= FF_GATED ? 2 : 1; }

// What the epilogue does with a tile's products. Rows are the batch's, columns those of one head.
struct FfOut {
  void* out[2];            // y, or dg and du, or the outputs of a product's operand sets
  long long ld, head;      // strides in values
  const void* aux;         // r (may be null) or dy
  long long aux_ld, aux_head;
  const void* bias[2];     // [heads, N] or null
  int bias_f32;
  float bias0[2];          // added to every column
  int act, up_relu, half;  // half: fp16 values, else bf16
  int keep;
  void* held[2];           // [M, heads, N] values, or codes
  uint8_t* exponents[2];   // [M, heads, ceil(N / 32)]
  float* colsum[2];        // [ceil(M / 32), heads, N]: sums over 32 rows of dp, or null
  int M, N, heads;
};

struct alignas(64) FfGemm {
  CUtensorMap ta[2], tb[2];
  int KB;                 // 64-wide blocks of one pair of operands
  int segments;           // pairs in a reduction: sets x heads that are summed
  int sum_heads;          // heads among them
  int out_sets;           // operand sets among the outputs
  int a_heads, b_heads;   // bit s: set s has a head coordinate
  int a_mn, b_mn;         // the reduction is not the contiguous dimension; b_mn of the gated form: a bit a projection
  int two_a;              // the second product has an A of its own
  int tiles_m, tiles_n, splits;
  uint32_t idesc;
  float* partial;         // [splits, NB, sets, heads, M, N] where the reduction is split
  int* err;
  FfOut e;
};

// ------------------------------------------------------------------------------- arithmetic

template <int ACT>
__device__ __forceinline__ float ff_act(float p) {
  if constexpr (ACT == FF_RELU) return p <= 0.f ? 0.f : p;
  if constexpr (ACT == FF_SILU) return __fdividef(p, 1.f + __expf(-p));
  if constexpr (ACT == FF_GELU) return 0.5f * p * (1.f + erff(p * 0.70710678118654752f));
  return p;
}

// act(p) and its derivative.
template <int ACT>
__device__ __forceinline__ void ff_act_both(float p, float& f, float& d) {
  if constexpr (ACT == FF_RELU) {
    f = p <= 0.f ? 0.f : p;
    d = p > 0.f ? 1.f : 0.f;
  } else if constexpr (ACT == FF_SILU) {
    const float s = __fdividef(1.f, 1.f + __expf(-p));
    f = p * s;
    d = s * (1.f + p * (1.f - s));
  } else if constexpr (ACT == FF_GELU) {
    const float cdf = 0.5f * (1.f + erff(p * 0.70710678118654752f));
    f = p * cdf;
    d = cdf + p * 0.3989422804014327f * __expf(-0.5f * p * p);
  } else {
    f = p, d = 1.f;
  }
}

template <typename F>
__device__ __forceinline__ void ff_with_act(int act, F&& f) {
  if (act == FF_RELU)
    f(std::integral_constant<int, FF_RELU>());
  else if (act == FF_SILU)
    f(std::integral_constant<int, FF_SILU>());
  else if (act == FF_GELU)
    f(std::integral_constant<int, FF_GELU>());
  else
    f(std::integral_constant<int, FF_NONE>());
}

// n values: y = act(p) (+ r is the caller's), or dp in place.
template <int EPI, int n>
__device__ __forceinline__ void ff_values(const FfOut& e, float* p, float* u, const float* dy) {
  ff_with_act(e.act, [&](auto a) {
    constexpr int A = decltype(a)::value;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      if constexpr (EPI == FF_ACT) {
        p[i] = ff_act<A>(p[i]);
      } else if constexpr (EPI == FF_ACT_BWD) {
        float f, d;
        ff_act_both<A>(p[i], f, d);
        p[i] = dy[i] * d;
      } else if constexpr (EPI == FF_GATED) {
        p[i] = ff_act<A>(p[i]) * (e.up_relu && u[i] <= 0.f ? 0.f : u[i]);
      } else if constexpr (EPI == FF_GATED_BWD) {
        float f, d;
        ff_act_both<A>(p[i], f, d);
        const bool off = e.up_relu && !(u[i] > 0.f);
        const float h = e.up_relu && u[i] <= 0.f ? 0.f : u[i];
        p[i] = dy[i] * h * d;
        u[i] = off ? 0.f : dy[i] * f;
      }
    }
  });
}

__device__ __forceinline__ uint32_t ff_pack2(float a, float b, int half) {
  if (half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 ff_unpack2(uint32_t v, int half) {
  if (half) return __half22float2(*reinterpret_cast<const __half2*>(&v));
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
}
__device__ __forceinline__ uint4 ff_pack8(const float* v, int half) {
  return make_uint4(ff_pack2(v[0], v[1], half), ff_pack2(v[2], v[3], half), ff_pack2(v[4], v[5], half),
                    ff_pack2(v[6], v[7], half));
}
__device__ __forceinline__ void ff_unpack8(uint4 q, int half, float* v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = ff_unpack2(w[i], half);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

// Adds the bias to 8 columns.
__device__ __forceinline__ void ff_bias8(const FfOut& e, int s, int head, int col, float* v) {
  float b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = e.bias0[s];
  if (e.bias[s]) {
    const long long at = (long long)head * e.N + col;
    if (e.bias_f32) {
      const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(e.bias[s]) + at);
      const float4 lo = __ldg(q), hi = __ldg(q + 1);
      b[0] += lo.x, b[1] += lo.y, b[2] += lo.z, b[3] += lo.w, b[4] += hi.x, b[5] += hi.y, b[6] += hi.z, b[7] += hi.w;
    } else {
      float f[8];
      ff_unpack8(__ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(e.bias[s]) + at)), e.half, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] += f[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += b[i];
}

// ------------------------------------------------------------------------------- epilogue of 32 x 32 values a warp

// A warp's 32 x 32 tile of 16-bit values in shared memory: rows of 64 bytes, their 16-byte pieces turned by the row, so
// that a lane's row and four lanes' row are both free of bank conflicts. Global rows then move 64 bytes at a time.
__device__ __forceinline__ uint32_t ff_piece(int row, int q) { return (uint32_t)(row * 64 + ((q ^ ((row >> 1) & 3)) << 4)); }

struct FfAux {
  uint4 v[4];
};

__device__ __forceinline__ FfAux ff_load_aux(const FfOut& e, int head, int row0, int col, int lane) {
  FfAux a;
  const int c = col + 8 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + 8 * i + lane / 4;
    a.v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (r < e.M && c < e.N)
      a.v[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(e.aux) + (long long)r * e.aux_ld +
                                               (long long)head * e.aux_head + c);
  }
  return a;
}

__device__ __forceinline__ void ff_put_aux(const FfAux& a, uint8_t* buf, int lane) {
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(buf + ff_piece(8 * i + lane / 4, lane & 3)) = a.v[i];
}

// Rows [row0, row0 + 32) x 32 columns from the lanes' rows.
__device__ __forceinline__ void ff_store_tile(const FfOut& e, void* out, long long ld, long long head_stride, int head,
                                              const float* v, int row0, int col, uint8_t* buf, int lane) {
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(buf + ff_piece(lane, q)) = ff_pack8(v + 8 * q, e.half);
  __syncwarp();
  const int c = col + 8 * (lane & 3);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + lane / 4;
    const uint4 w = *reinterpret_cast<const uint4*>(buf + ff_piece(r, lane & 3));
    if (row0 + r < e.M && c < e.N)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + (long long)(row0 + r) * ld + (long long)head * head_stride +
                                c) = w;
  }
}

// The lane's row of 32 pre-activations in 8 bits. Columns past N count as zeros.
__device__ __forceinline__ void ff_hold8(const FfOut& e, int s, int head, const float* v, int row, int col) {
  if (row >= e.M) return;
  float largest = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (col + (i & ~7) < e.N) largest = fmaxf(largest, act8_size(v[i]));
  const int ex = act8_exponent(largest);
  const float inverse = act8_power(-ex);
  const int nb = (e.N + 31) / 32;
  const long long rh = (long long)row * e.heads + head;
  uint8_t* o = reinterpret_cast<uint8_t*>(e.held[s]) + rh * e.N + col;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    if (col + 8 * q < e.N)
      *reinterpret_cast<uint2*>(o + 8 * q) = make_uint2(act8_code4(v + 8 * q, inverse), act8_code4(v + 8 * q + 4, inverse));
  e.exponents[s][rh * nb + col / 32] = (uint8_t)(ex + 127);
}

// Sum over the warp's 32 rows (a row a lane) of 32 columns: lane l gets column l's. v is used up. The order is fixed.
__device__ __forceinline__ float ff_column_sum(float* v, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    const bool hi = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = hi ? v[i] : v[i + o], mine = hi ? v[i + o] : v[i];
      v[i] = mine + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

__device__ __forceinline__ void ff_put_sums(const FfOut& e, int s, int head, float* v, int row0, int col, int lane) {
  const bool in = row0 + lane < e.M;
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = in ? v[i] : 0.f;
  const float sum = ff_column_sum(v, lane);
  if (col + lane < e.N) e.colsum[s][((long long)(row0 / 32) * e.heads + head) * e.N + col + lane] = sum;
}

// g, u: the lane's row of the products (u unused where there is one).
template <int EPI>
__device__ __forceinline__ void ff_epilogue(const FfOut& e, int set, int head, int row0, int col, float* g, float* u,
                                            uint8_t* buf, int lane) {
  constexpr int NB = ff_products(EPI);
  if constexpr (EPI == FF_STORE) {
    ff_store_tile(e, e.out[set], e.ld, e.head, head, g, row0, col, buf, lane);
    return;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (col + 8 * q < e.N) {
        ff_bias8(e, 0, head, col + 8 * q, g + 8 * q);
        if constexpr (NB == 2) ff_bias8(e, 1, head, col + 8 * q, u + 8 * q);
      }
    }
    const bool has_aux = ff_backward(EPI) || (EPI == FF_ACT && e.aux);
    FfAux aux;
    if (has_aux) aux = ff_load_aux(e, head, row0, col, lane);
    if constexpr (!ff_backward(EPI)) {
      const long long hl = (long long)e.heads * e.N;
      if (e.keep == FF_KEEP_16) {
        ff_store_tile(e, e.held[0], hl, e.N, head, g, row0, col, buf, lane);
        if constexpr (NB == 2) ff_store_tile(e, e.held[1], hl, e.N, head, u, row0, col, buf, lane);
      } else if (e.keep == FF_KEEP_8) {
        ff_hold8(e, 0, head, g, row0 + lane, col);
        if constexpr (NB == 2) ff_hold8(e, 1, head, u, row0 + lane, col);
      }
    }
    float a[32];
    if (has_aux) {
      ff_put_aux(aux, buf + 2048, lane);
      __syncwarp();
#pragma unroll
      for (int q = 0; q < 4; ++q)
        ff_unpack8(*reinterpret_cast<const uint4*>(buf + 2048 + ff_piece(lane, q)), e.half, a + 8 * q);
    }
    ff_values<EPI, 32>(e, g, u, a);
    if constexpr (EPI == FF_ACT) {
      if (has_aux) {
#pragma unroll
        for (int i = 0; i < 32; ++i) g[i] += a[i];
      }
    }
    ff_store_tile(e, e.out[0], e.ld, e.head, head, g, row0, col, buf, lane);
    if constexpr (EPI == FF_GATED_BWD) ff_store_tile(e, e.out[1], e.ld, e.head, head, u, row0, col, buf, lane);
    if constexpr (ff_backward(EPI)) {
      if (e.colsum[0]) ff_put_sums(e, 0, head, g, row0, col, lane);
      if constexpr (NB == 2)
        if (e.colsum[1]) ff_put_sums(e, 1, head, u, row0, col, lane);
    }
  }
}

// ------------------------------------------------------------------------------- products

constexpr int kFfEpiWarps = 8;
constexpr int kFfThreads = 64 + 32 * kFfEpiWarps;

template <int NB, int BN, bool PAIR>
struct FfCfg {
  static constexpr int CTAS = PAIR ? 2 : 1;
  static constexpr int B_ROWS = BN / CTAS;  // of one product, staged by this CTA
  static constexpr int A_BYTES = 128 * 64 * 2, B_BYTES = B_ROWS * 64 * 2;
  static constexpr int STAGE_BYTES = NB * (A_BYTES + B_BYTES);
  static constexpr int EPI_BYTES = kFfEpiWarps * 4096;
  static constexpr int STAGES = (192 * 1024) / STAGE_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * NB * BN;
  static_assert(B_ROWS % 64 == 0 && TMEM_COLS <= 512 && SMEM <= 227 * 1024, "tile");
};

// The tiles of a CTA (or pair), t, t + step, ...: columns fastest, then rows, parts, heads, sets. Divided once.
struct FfWalk {
  unsigned at[4], by[4], size[4], set, bset;

  __device__ __forceinline__ FfWalk(const FfGemm& p, unsigned t, unsigned step) {
    size[0] = p.tiles_n, size[1] = p.tiles_m, size[2] = p.splits, size[3] = p.e.heads;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] = t % size[i], by[i] = step % size[i];
      t /= size[i], step /= size[i];
    }
    set = t, bset = step;
  }
  __device__ __forceinline__ void next() {
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] += by[i] + carry;
      carry = at[i] >= size[i] ? 1 : 0;
      at[i] -= carry ? size[i] : 0;
    }
    set += bset + carry;
  }
  __device__ __forceinline__ int n() const { return (int)at[0]; }
  __device__ __forceinline__ int m() const { return (int)at[1]; }
  __device__ __forceinline__ int split() const { return (int)at[2]; }
  __device__ __forceinline__ int head() const { return (int)at[3]; }
};

// The blocks [b0, b1) of part `split`.
__device__ __forceinline__ void ff_part(const FfGemm& p, int split, int& b0, int& b1) {
  const unsigned blocks = (unsigned)(p.segments * p.KB);  // times the parts below 2^32: the host checks
  b0 = (int)(blocks * (unsigned)split / (unsigned)p.splits);
  b1 = (int)(blocks * (unsigned)(split + 1) / (unsigned)p.splits);
}

template <bool PAIR>
__device__ __forceinline__ void ff_tma(void* dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2) {
  if constexpr (PAIR)
    tma_load_4d_pair(dst, m, bar, c0, c1, c2, 0);
  else
    tma_load_4d(dst, m, bar, c0, c1, c2, 0);
}

// ROWS rows of an operand x 64 of its reduction into a 128B-swizzled tile.
template <bool PAIR, int ROWS>
__device__ __forceinline__ void ff_load(void* dst, const CUtensorMap* m, bool mn, uint64_t* bar, int row, int k, int head) {
  if (mn) {
#pragma unroll
    for (int i = 0; i < ROWS / 64; ++i)
      ff_tma<PAIR>(reinterpret_cast<uint8_t*>(dst) + i * 8192, m, bar, row + 64 * i, k, head);
  } else {
    ff_tma<PAIR>(dst, m, bar, k, row, head);
  }
}

template <int EPI, int BN, bool PAIR>
__global__ void __launch_bounds__(kFfThreads, 1) ff_gemm_kernel(const __grid_constant__ FfGemm p) {
  constexpr int NB = ff_products(EPI);
  using Cfg = FfCfg<NB, BN, PAIR>;
  constexpr int STAGES = Cfg::STAGES, ROWS = 128 * Cfg::CTAS;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ uint64_t tfull_bar[2], tempty_bar[2], drain_bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int crank = PAIR ? (int)cluster_ctarank() : 0;
  const bool leader = crank == 0;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sEpi = smem + STAGES * Cfg::STAGE_BYTES;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], Cfg::CTAS * kFfEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    for (int s = 0; s < 2; ++s) {
      tma_prefetch_desc(&p.ta[s]);
      tma_prefetch_desc(&p.tb[s]);
    }
  }
  if (warp == 1) {
    if constexpr (PAIR)
      tmem_alloc_pair(&tmem_base_s, Cfg::TMEM_COLS);
    else
      tmem_alloc(&tmem_base_s, Cfg::TMEM_COLS);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  const unsigned worker = blockIdx.x / Cfg::CTAS, workers = gridDim.x / Cfg::CTAS;
  const unsigned total = (unsigned)(p.tiles_m * p.tiles_n * p.splits * p.e.heads * p.out_sets);

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer (both CTAs of a pair)
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      const uint32_t bytes = (uint32_t)(Cfg::CTAS * ((NB == 2 && !p.two_a ? 1 : NB) * Cfg::A_BYTES + NB * Cfg::B_BYTES));
      FfWalk w(p, worker, workers);
      for (unsigned t = worker; t < total && ok; t += workers, w.next()) {
        int b0, b1;
        ff_part(p, w.split(), b0, b1);
        const int am = w.m() * ROWS + 128 * crank, bn = w.n() * BN + Cfg::B_ROWS * crank;
        int seg = b0 / p.KB, kb = b0 - seg * p.KB;
        for (int i = b0; i < b1; ++i) {
          // the pair of operands: its set and head
          const int sum_set = seg / p.sum_heads;
          const int set = p.out_sets > 1 ? (int)w.set : sum_set;
          const int head = p.sum_heads > 1 ? seg - sum_set * p.sum_heads : w.head();
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          uint64_t* bar = &full_bar[stage];
          if (leader) mbar_arrive_expect_tx(bar, bytes);
          uint8_t* dst = smem + stage * Cfg::STAGE_BYTES;
          const int k = kb * 64;
          if constexpr (NB == 1) {
            ff_load<PAIR, 128>(dst, &p.ta[set], p.a_mn, bar, am, k, (p.a_heads >> set) & 1 ? head : 0);
            ff_load<PAIR, Cfg::B_ROWS>(dst + Cfg::A_BYTES, &p.tb[set], p.b_mn, bar, bn, k, (p.b_heads >> set) & 1 ? head : 0);
          } else {
            ff_load<PAIR, 128>(dst, &p.ta[0], p.a_mn, bar, am, k, (p.a_heads & 1) ? head : 0);
            if (p.two_a) ff_load<PAIR, 128>(dst + Cfg::A_BYTES, &p.ta[1], p.a_mn, bar, am, k, (p.a_heads & 2) ? head : 0);
            ff_load<PAIR, Cfg::B_ROWS>(dst + 2 * Cfg::A_BYTES, &p.tb[0], (p.b_mn & 1) != 0, bar, bn, k, head);
            ff_load<PAIR, Cfg::B_ROWS>(dst + 2 * Cfg::A_BYTES + Cfg::B_BYTES, &p.tb[1], (p.b_mn & 2) != 0, bar, bn, k, head);
          }
          if (++kb == p.KB) kb = 0, ++seg;
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && leader) {
        // wait (bounded, ignoring the abort flag) for the loads still in flight
        int dummy_abort = 0;
        const long long inflight = issued < STAGES ? issued : STAGES;
        int s = stage;
        uint32_t ph = phase;
        for (long long i = 0; i < inflight; ++i) {
          if (--s < 0) {
            s = STAGES - 1;
            ph ^= 1;
          }
          mbar_wait_bounded(&full_bar[s], ph, (volatile int*)&dummy_abort, p.err, kErrTimeoutDrain);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------------------------ MMA issuer
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      FfWalk w(p, worker, workers);
      for (unsigned t = worker; t < total && ok; t += workers, w.next()) {
        int b0, b1;
        ff_part(p, w.split(), b0, b1);
        if (!mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1, &abort_flag, p.err, kErrTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int i = b0; i < b1; ++i) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, &abort_flag, p.err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(smem + stage * Cfg::STAGE_BYTES);
#pragma unroll
          for (int s = 0; s < NB; ++s) {
            const bool b_mn = NB == 1 ? p.b_mn != 0 : (p.b_mn & (1 << s)) != 0;
            const uint32_t a_base = base + (s == 1 && p.two_a ? Cfg::A_BYTES : 0);
            const uint32_t b_base = base + NB * Cfg::A_BYTES + s * Cfg::B_BYTES;
            const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = b_mn ? 2048 : 32;
            const uint32_t a_lbo = p.a_mn ? 8192 : 16, b_lbo = b_mn ? 8192 : 16;
            const uint32_t idesc = p.idesc | (b_mn ? 1u << 16 : 0u);
            const uint32_t d = tmem_base + (acc * NB + s) * BN;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const uint64_t ad = make_sdesc_sw128(a_base + kk * a_step, a_lbo, 1024);
              const uint64_t bd = make_sdesc_sw128(b_base + kk * b_step, b_lbo, 1024);
              if constexpr (PAIR)
                umma_bf16_pair(d, ad, bd, idesc, (i > b0 || kk > 0) ? 1u : 0u);
              else
                umma_bf16(d, ad, bd, idesc, (i > b0 || kk > 0) ? 1u : 0u);
            }
          }
          if constexpr (PAIR)
            umma_commit_pair(&empty_bar[stage]);
          else
            umma_commit(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if constexpr (PAIR)
          umma_commit_pair(&tfull_bar[acc]);
        else
          umma_commit(&tfull_bar[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // every MMA of this thread is done before TMEM is released
      if constexpr (PAIR)
        umma_commit_pair(&drain_bar);
      else
        umma_commit(&drain_bar);
      int dummy_abort = 0;
      mbar_wait_bounded(&drain_bar, 0, (volatile int*)&dummy_abort, p.err, kErrTimeoutDrain);
    }
  } else {
    // ------------------------------------------------ epilogue (each CTA its own 128 rows)
    const int quad = warp & 3;         // TMEM lane quadrant of this warp
    const int half = (warp - 2) >> 2;  // half of the tile's columns
    uint8_t* buf = sEpi + (warp - 2) * 4096;
    constexpr int COLS = BN / 2;
    const int col0 = half * COLS;
    uint32_t leader_tempty0 = 0, leader_tempty1 = 0;
    if constexpr (PAIR) leader_tempty0 = map_to_cta(&tempty_bar[0], 0), leader_tempty1 = map_to_cta(&tempty_bar[1], 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    FfWalk w(p, worker, workers);
    for (unsigned t = worker; t < total; t += workers, w.next()) {
      // the same answer for the whole warp: the loads from TMEM need all of its lanes, also where a wait has run out
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], acc_phase, &abort_flag, p.err, kErrTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int row0 = w.m() * ROWS + 128 * crank + quad * 32;
#pragma unroll 1
      for (int cc = 0; cc < COLS; cc += 32) {
        const int col = w.n() * BN + col0 + cc;
        if (row0 >= p.e.M || col >= p.e.N) continue;
        const uint32_t at = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * NB * BN + col0 + cc;
        float g[32], u[32];
        tmem_ld32(at, g);
        if constexpr (NB == 2) tmem_ld32(at + BN, u);
        if (p.splits == 1) {
          ff_epilogue<EPI>(p.e, (int)w.set, w.head(), row0, col, g, u, buf, lane);
        } else if (row0 + lane < p.e.M) {
#pragma unroll
          for (int s = 0; s < NB; ++s) {
            const float* v = s ? u : g;
            float* o = p.partial +
                       (((((long long)w.split() * NB + s) * p.out_sets + w.set) * p.e.heads + w.head()) * p.e.M + row0 + lane) * p.e.N + col;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (col + 4 * q < p.e.N)
                reinterpret_cast<float4*>(o)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(&tempty_bar[acc]);
        else
          mbar_arrive_cluster(acc ? leader_tempty1 : leader_tempty0);
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the leader's MMAs (into both CTAs' TMEM and shared memory) are done
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem_base, Cfg::TMEM_COLS);
    else
      tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

}  // namespace bd

namespace bd {
// The tile of a launch: PAIR and BN. feed_forward_{a,b}.cu hold the instantiations.
struct FfTile {
  bool pair;
  int bn;
};
void ff_launch_one(int epi, FfTile tile, const FfGemm& p, cudaStream_t st, int dev);    // one product
void ff_launch_gated(int epi, FfTile tile, const FfGemm& p, cudaStream_t st, int dev);  // two
}  // namespace bd
