// adapters.cu — low-rank adapters of many requests at once beside a shared, frozen projection.
//
//   t[m,h,:]  = x[m(,h),:] a[g(m),h]^T                     (a [G, H, r, K], g(m) the row's adapter)
//   y[m,h,:]  = x[m(,h),:] W[h] + s[g(m)] t[m,h,:] b[g(m),h]        (W [H, K, N], b [G, H, r, N])
// and its gradients, which are the same three operations with the roles of a and b exchanged:
//   u = dy b^T,  dx = dy W^T + s u a  (summed over the heads where they share x),
//   da[g] = s u_g^T x_g,  db[g] = s t_g^T dy_g            (the rows of adapter g)
//
// Three kernels:
//  * adapter_shrink: t (or u), one CTA per run of up to 32 rows of one adapter, per head and
//    per part of the reduction. Bound by the bytes of x and a; both are K-contiguous, so the
//    mma.sync operands are loaded straight from memory, 16 bytes a lane.
//  * adapter_gemm: the projection on tcgen05 (TMA, TMEM, warp roles as in the GEMM engine),
//    with the adapters as an extension of its reduction: after the K-blocks of x and W
//    come blocks of 64 / rp adapter slots. A 128-row tile lists the distinct adapters of its rows
//    ("slots"); four builder warps write t s into the columns of each row's slot, and TMA loads the
//    slots' b rows beside each other. A slot's product leaves the accumulator's rows of other slots as they
//    are: they are masked off (zeros in their columns would not do: 0 b is NaN where another adapter's b is not
//    finite). So one accumulator takes both products, rows of any adapters can share a tile, and W and every b are
//    read once per row tile. The projection's blocks need no t, so with programmatic launch they run
//    while adapter_shrink still does; only the builders wait for it.
//  * adapter_grad: da / db, one CTA per adapter, head and slab of columns; for db it gives u in the same pass over dy.
// Measured on a B200: 48 rows, 43 adapters of rank 16, 4 heads 256 -> 8192: 21 us for 66 MB;
// 4099 rows the same way: shrink 12, product 107 us (45 us for its 295 MB at the copy rate: the issuing
// thread and the operands' way into shared memory, 192 KB a tile, bound it; 85 without adapters); 4096^3 with 8
// adapters 123 us. Masking the rows costs nothing beside writing zeros (48 rows 21.0 against 21.9 us, 9 prompts 110
// against 111): the masks are read while a block's b is on its way. Keeping w in shared memory over the row tiles
// (192 columns) was slower: 113 against 98 us.
// t and u are kept in fp32 (partial sums over the parts of the reduction) and rounded to bf16
// once, as an operand of the next product, like every activation of the bf16 path: y is off by 0.0018 to 0.0024
// of itself, where its own rounding to bf16 is 0.0017. (Two bf16 halves of t gave 0.0017, and took training from 207
// to 223 us, eight prompts of rank 64 from 190 to 208 and 48 rows from 21.9 to 22.5.) All sums are fp32 and in a
// fixed order: no atomics.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "gemm_table.h"
#include "launches.h"
#include "sm100_ptx.cuh"
#include "tensor_map.h"

namespace bd {
namespace {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// umma_bf16 with accumulation into the rows (TMEM lanes) whose bit in `off` is clear; the others keep what they hold.
__device__ __forceinline__ void umma_bf16_rows(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint4 off) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %5, %6, %7}, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(off.x), "r"(off.y), "r"(off.z), "r"(off.w)
      : "memory");
}

__device__ __forceinline__ void grid_dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ------------------------------------------------------------------------------- shrink

constexpr int kShrinkThreads = 256;

struct ShrinkArgs {
  const bf16* x;
  long long x_row, x_head;
  const bf16* a;  // [G, H, r, K]
  float* t;       // [parts, H, M, rp]
  const int* order;
  const int* chunks;  // (start in order, rows, adapter) each
  int M, H, K, r, part_k;
};

// Rank rows are the m of the product, the run's x rows its n (MT 16-row and NT 8-row tiles).
// The k order inside 32 values is permuted alike for both operands so that a lane's 16-byte
// load holds the fragments of two products.
template <int MT, int NT>
__global__ void __launch_bounds__(kShrinkThreads) adapter_shrink_kernel(const __grid_constant__ ShrinkArgs p) {
  constexpr int RP = 16 * MT;
  __shared__ float red[4][RP][NT * 8];
  grid_dependents_launch();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int start = p.chunks[3 * blockIdx.x], rows = p.chunks[3 * blockIdx.x + 1], g = p.chunks[3 * blockIdx.x + 2];
  const int h = blockIdx.y;
  const int k1 = min((int)(blockIdx.z + 1) * p.part_k, p.K);
  const bf16* a = p.a + ((long long)g * p.H + h) * p.r * p.K;
  // Rows past the run or the rank repeat the last one: their sums are not kept (n), or meet rows of b that
  // read as zero (m), and no load needs a condition.
  const bf16* xr[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    xr[nt] = p.x + (long long)p.order[start + min(nt * 8 + lane / 4, rows - 1)] * p.x_row + (long long)h * p.x_head;
  const bf16* ar[MT][2];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 2; ++i) ar[mt][i] = a + (long long)min(mt * 16 + i * 8 + lane / 4, p.r - 1) * p.K;
  float acc[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[mt][nt][i] = 0.f;
  auto step = [&](int k, bool in) {
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 xv[NT], av[MT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) xv[nt] = in ? *reinterpret_cast<const uint4*>(xr[nt] + k) : zero;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 2; ++i) av[mt][i] = in ? *reinterpret_cast<const uint4*>(ar[mt][i] + k) : zero;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_bf16(acc[mt][nt], av[mt][0].x, av[mt][1].x, av[mt][0].y, av[mt][1].y, xv[nt].x, xv[nt].y);
        mma_bf16(acc[mt][nt], av[mt][0].z, av[mt][1].z, av[mt][0].w, av[mt][1].w, xv[nt].z, xv[nt].w);
      }
  };
  constexpr int SWEEP = 32 * (kShrinkThreads / 32);
  int k0 = (int)blockIdx.z * p.part_k + warp * 32;  // of this warp's 32 values; a lane reads 8 of them
  const int off = 8 * (lane % 4);
#pragma unroll(NT == 1 ? 4 : 2)
  for (; k0 + 32 <= k1; k0 += SWEEP) step(k0 + off, true);
  if (k0 < k1) step(k0 + off, k0 + off < k1);
  // the warps' sums, folded in halves (a fixed order)
#pragma unroll
  for (int half = 4; half > 0; half /= 2) {
    if (warp >= half && warp < 2 * half) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            red[warp - half][mt * 16 + lane / 4 + (i / 2) * 8][nt * 8 + 2 * (lane % 4) + i % 2] = acc[mt][nt][i];
    }
    __syncthreads();
    if (warp < half) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[mt][nt][i] += red[warp][mt * 16 + lane / 4 + (i / 2) * 8][nt * 8 + 2 * (lane % 4) + i % 2];
    }
    __syncthreads();
  }
  if (warp == 0) {
    float* t = p.t + ((long long)blockIdx.z * p.H + h) * p.M * RP;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = nt * 8 + 2 * (lane % 4) + i % 2;
        if (n >= rows) continue;
        float* o = t + (long long)p.order[start + n] * RP + lane / 4 + (i / 2) * 8;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt * 16] = acc[mt][nt][i];
      }
  }
}

// ------------------------------------------------------------------------------- projection

struct AdapterGemm {
  CUtensorMap tx, tw, tb;
  bf16* y;  // [M, Z, N]
  int M, N, KB;      // rows, output columns, 64-wide blocks of one head's reduction
  int HR, Z;         // heads summed in the reduction, heads of the output
  int x_heads;       // x has a head coordinate
  int H;             // heads of b and t
  int tiles_m, tiles_n, splits;
  int r, rp, per_block, block_shift;  // rank, padded rank, slots per 64-wide block and its logarithm
  int parts;          // partial sums of t
  long long t_part;
  const float* t;     // [parts, H, M, rp]; null without adapters
  const int* row_slot;
  const int* row_adapter;
  const int* tile_ptr;
  const int* slots;
  const float* scale;  // per adapter, or null
  float scale0;
  float* partial;     // [splits, Z, M, N] where the reduction is split
  int* err;
};

struct AdapterTile {
  int m0, n0, z, slot0, nslots, ext, kb0, kb1, e0, e1, split;
};

// The tiles of a CTA, t, t + step, ...: columns fastest, then rows, parts, heads. Divided once; a role is one thread
// here, and divisions for every tile (64-bit ones above all) made a chain of over 1 us (4096 x 256 -> 4 x
// 8192 without adapters: 98 us with them).
struct AdapterWalk {
  unsigned at[3], by[3], size[3], z, bz;

  __device__ __forceinline__ AdapterWalk(const AdapterGemm& p, unsigned t, unsigned step) {
    size[0] = p.tiles_n, size[1] = p.tiles_m, size[2] = p.splits;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      at[i] = t % size[i], by[i] = step % size[i];
      t /= size[i], step /= size[i];
    }
    z = t, bz = step;
  }
  __device__ __forceinline__ void next() {
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      at[i] += by[i] + carry;
      carry = at[i] >= size[i] ? 1 : 0;
      at[i] -= carry ? size[i] : 0;
    }
    z += bz + carry;
  }
};

__device__ __forceinline__ AdapterTile adapter_place(const AdapterWalk& w, int BN) {
  AdapterTile c;
  c.n0 = (int)w.at[0] * BN;
  c.m0 = (int)w.at[1] * 128;
  c.split = (int)w.at[2];
  c.z = (int)w.z;
  return c;
}

// With the tile's slots, which are read from memory: every role asks one tile ahead.
__device__ __forceinline__ AdapterTile adapter_tile(const AdapterGemm& p, const AdapterWalk& w, int BN) {
  AdapterTile c = adapter_place(w, BN);
  c.slot0 = p.t ? p.tile_ptr[w.at[1]] : 0;
  c.nslots = (p.t ? p.tile_ptr[w.at[1] + 1] : 0) - c.slot0;
  c.ext = (c.nslots + p.per_block - 1) >> p.block_shift;
  // Blocks of the projection, then adapter blocks. A part takes its share of both (of the projection's at least four):
  // the first product of a tile writes every row of the accumulator, which an adapter's does not.
  // Times splits below 2^32: the host checks.
  const unsigned blocks = (unsigned)(p.HR * p.KB), adapters = (unsigned)(p.HR * c.ext);
  c.kb0 = 0, c.kb1 = (int)blocks, c.e0 = 0, c.e1 = (int)adapters;
  if (p.splits > 1) {
    const unsigned i = (unsigned)c.split, parts = (unsigned)p.splits;
    c.kb0 = (int)(blocks * i / parts), c.kb1 = (int)(blocks * (i + 1) / parts);
    c.e0 = (int)(adapters * i / parts), c.e1 = (int)(adapters * (i + 1) / parts);
  }
  return c;
}

constexpr int kEpiWarps = 8, kBuildWarps = 4;
constexpr int kAdapterThreads = 32 * (2 + kEpiWarps + kBuildWarps);

// EXT: buffers of the built operand (16 KB each), apart from the ring of x and w, so that the builders work ahead of
// the products. A 256-wide tile has room for three stages and two buffers, which short reductions want
// (an adapter block every few blocks), or four and one, which long ones want.
template <int BN, int EXT>
struct AdapterCfg {
  static constexpr int A_BYTES = 128 * 64 * 2;
  static constexpr int B_BYTES = BN * 64 * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? (EXT == 1 ? 4 : 3) : BN == 128 ? 5 : 6;
  static constexpr int EPI_BYTES = kEpiWarps * 2048;  // a 32 x 32 bf16 tile per epilogue warp
  static constexpr int SMEM = STAGES * STAGE_BYTES + EXT * A_BYTES + EPI_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * BN;
};

// Byte offset of 16-byte chunk `chunk` of row `row` in a 128-byte-row, 128B-swizzled tile.
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }

__device__ __forceinline__ uint4 to_bf16x8(const float* v) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  return *reinterpret_cast<uint4*>(h);
}

// W_MN: W's rows are the reduction (y = x W); else its columns are (dx = dy W^T).
template <int BN, bool W_MN, int EXT>
__global__ void __launch_bounds__(kAdapterThreads, 1) adapter_gemm_kernel(const __grid_constant__ AdapterGemm p) {
  using Cfg = AdapterCfg<BN, EXT>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ uint64_t built_bar[EXT], used_bar[EXT];  // of the built operands
  __shared__ uint4 rows_off[EXT][4];  // of each slot of a built operand: the tile's rows that are not its own
  __shared__ uint64_t tfull_bar[2], tempty_bar[2], drain_bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * Cfg::A_BYTES;
  uint8_t* sExt = smem + STAGES * Cfg::STAGE_BYTES;
  uint8_t* sEpi = sExt + EXT * Cfg::A_BYTES;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int e = 0; e < EXT; ++e) {
      mbar_init(&built_bar[e], kBuildWarps);
      mbar_init(&used_bar[e], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], kEpiWarps);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
    tma_prefetch_desc(&p.tx);
    tma_prefetch_desc(&p.tw);
  }
  if (warp == 1) tmem_alloc(&tmem_base_s, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_s;
  const int total = p.tiles_m * p.tiles_n * p.splits * p.Z;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      AdapterWalk walk(p, blockIdx.x, gridDim.x);
      AdapterTile next = adapter_tile(p, walk, BN);
      int ids[4];  // adapters of the next adapter block, read while other blocks are on their way
      auto read_ids = [&](const AdapterTile& c, int e) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          ids[j] = e * p.per_block + j < c.nslots && j < p.per_block ? p.slots[c.slot0 + e * p.per_block + j] : 0;
      };
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const AdapterTile c = next;
        walk.next();
        if (t + (int)gridDim.x < total) next = adapter_tile(p, walk, BN);
        if (c.ext > 0) read_ids(c, c.e0 % c.ext);
        const int projection = c.kb1 - c.kb0, blocks = projection + c.e1 - c.e0;
        for (int i = 0; i < blocks; ++i) {
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          uint8_t* a_dst = sA + stage * Cfg::A_BYTES;
          uint8_t* b_dst = sB + stage * Cfg::B_BYTES;
          if (i < projection) {
            const int kb = c.kb0 + i;
            const int h = p.HR > 1 ? kb / p.KB : c.z;
            const int k0 = (p.HR > 1 ? kb % p.KB : kb) * 64;
            mbar_arrive_expect_tx(&full_bar[stage], Cfg::STAGE_BYTES);
            tma_load_4d(a_dst, &p.tx, &full_bar[stage], k0, c.m0, p.x_heads ? h : 0, 0);
            if constexpr (W_MN) {
#pragma unroll
              for (int q = 0; q < BN / 64; ++q)
                tma_load_4d(b_dst + q * 8192, &p.tw, &full_bar[stage], c.n0 + 64 * q, k0, h, 0);
            } else {
              tma_load_4d(b_dst, &p.tw, &full_bar[stage], k0, c.n0, h, 0);
            }
          } else {
            const int e = c.e0 + i - projection;
            const int h = p.HR > 1 ? e / c.ext : c.z;
            const int j0 = (p.HR > 1 ? e % c.ext : e) * p.per_block;
            const int n = min(p.per_block, c.nslots - j0);
            mbar_arrive_expect_tx(&full_bar[stage], n * p.rp * 2 * BN);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (j >= n) break;
              const int gh = ids[j] * p.H + h;
#pragma unroll
              for (int q = 0; q < BN / 64; ++q)
                tma_load_4d(b_dst + q * 8192 + j * p.rp * 128, &p.tb, &full_bar[stage], c.n0 + 64 * q, 0, gh, 0);
            }
            read_ids(c, p.HR > 1 ? (e + 1) % c.ext : min(e + 1, c.ext - 1));
          }
          ++issued;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
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
    if (lane == 0) {
      // ------------------------------------------------ MMA issuer
      constexpr uint32_t idesc_w = make_idesc_bf16(128, BN, false, W_MN);
      constexpr uint32_t idesc_b = make_idesc_bf16(128, BN, false, true);
      int stage = 0, acc = 0, buf = 0;  // buf: the next built operand
      uint32_t phase = 0, acc_phase = 0, buf_phase = 0;
      bool ok = true;
      AdapterWalk walk(p, blockIdx.x, gridDim.x);
      AdapterTile next = adapter_tile(p, walk, BN);
      for (int t = blockIdx.x; t < total && ok; t += gridDim.x) {
        const AdapterTile c = next;
        walk.next();
        if (t + (int)gridDim.x < total) next = adapter_tile(p, walk, BN);
        if (!mbar_wait_bounded(&tempty_bar[acc], acc_phase ^ 1, &abort_flag, p.err, kErrTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        const int projection = c.kb1 - c.kb0, blocks = projection + c.e1 - c.e0;
        for (int i = 0; i < blocks; ++i) {
          const bool ext = i >= projection;
          uint4 off[4];  // of each step: read while the block's b is still on its way
          if (ext) {
            ok = mbar_wait_bounded(&built_bar[buf], buf_phase, &abort_flag, p.err, kErrTimeoutMma);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) off[kk] = rows_off[buf][kk >> (2 - p.block_shift)];
          }
          if (!ok || !mbar_wait_bounded(&full_bar[stage], phase, &abort_flag, p.err, kErrTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_base = smem_u32(sA + stage * Cfg::A_BYTES);
          const uint32_t b_base = smem_u32(sB + stage * Cfg::B_BYTES);
          if (!ext) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(d_tmem, make_sdesc_sw128(a_base + kk * 32, 16, 1024),
                        W_MN ? make_sdesc_sw128(b_base + kk * 2048, 8192, 1024)
                             : make_sdesc_sw128(b_base + kk * 32, 16, 1024),
                        idesc_w, (i > 0 || kk > 0) ? 1u : 0u);
          } else {
            const uint32_t e_base = smem_u32(sExt + buf * Cfg::A_BYTES);
            const int e = c.e0 + i - projection;
            const int j0 = (p.HR > 1 ? e % c.ext : e) * p.per_block;
            const int steps = (min(p.per_block, c.nslots - j0) * p.rp) >> 4;  // 1, 2 or 4 a slot
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (kk < steps)
                umma_bf16_rows(d_tmem, make_sdesc_sw128(e_base + kk * 32, 16, 1024),
                               make_sdesc_sw128(b_base + kk * 2048, 8192, 1024), idesc_b, off[kk]);
            umma_commit(&used_bar[buf]);
            if (++buf == EXT) {
              buf = 0;
              buf_phase ^= 1;
            }
          }
          umma_commit(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        umma_commit(&tfull_bar[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // every MMA of this thread is done before TMEM is released
      umma_commit(&drain_bar);
      int dummy_abort = 0;
      mbar_wait_bounded(&drain_bar, 0, (volatile int*)&dummy_abort, p.err, kErrTimeoutDrain);
    }
  } else if (warp < 2 + kEpiWarps) {
    // ------------------------------------------------ epilogue: bf16 rows, or fp32 parts
    const int quad = warp & 3;         // TMEM lane quadrant of this warp
    const int half = (warp - 2) >> 2;  // half of the tile's columns
    uint8_t* buf = sEpi + (warp - 2) * 2048;
    constexpr int COLS = BN / 2;
    const int col0 = half * COLS;
    int acc = 0;
    uint32_t acc_phase = 0;
    AdapterWalk walk(p, blockIdx.x, gridDim.x);
    for (int t = blockIdx.x; t < total; t += gridDim.x, walk.next()) {
      const AdapterTile c = adapter_place(walk, BN);
      // the same answer for the whole warp: the loads from TMEM need all of its lanes, also where a wait has run out
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], acc_phase, &abort_flag, p.err, kErrTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int row0 = c.m0 + quad * 32;
#pragma unroll 1
      for (int cc = 0; cc < COLS; cc += 32) {
        const int col = c.n0 + col0 + cc;
        if (row0 >= p.M || col >= p.N) continue;
        float v[32];
        tmem_ld32(tmem_base + ((uint32_t)(quad * 32) << 16) + acc * BN + col0 + cc, v);
        if (p.splits == 1) {
          // a lane holds a row: turned over in shared memory so that four lanes store 64 bytes of one row
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<uint4*>(buf + lane * 64 + ((q ^ ((lane >> 1) & 3)) << 4)) = to_bf16x8(v + 8 * q);
          __syncwarp();
          const int q = lane & 3;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + lane / 4;
            const uint4 w = *reinterpret_cast<const uint4*>(buf + r * 64 + ((q ^ ((r >> 1) & 3)) << 4));
            if (row0 + r < p.M && col + 8 * q < p.N)
              *reinterpret_cast<uint4*>(p.y + (long long)(row0 + r) * p.Z * p.N + (long long)c.z * p.N + col + 8 * q) = w;
          }
        } else if (row0 + lane < p.M) {
          float* o = p.partial + (((long long)c.split * p.Z + c.z) * p.M + row0 + lane) * p.N + col;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (col + 4 * q < p.N)
              reinterpret_cast<float4*>(o)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty_bar[acc]);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  } else {
    // ------------------------------------------------ builders: one row of the tile per thread
    grid_dependency_wait();  // t is complete (and this grid does not end before the one that wrote it)
    const int r = threadIdx.x - 32 * (2 + kEpiWarps);
    // The t of one row and head, scaled and rounded; the next one's loads run while this one is built.
    struct Row {
      int slot;
      uint4 t[8];
    };
    auto fetch = [&](const AdapterTile& c, int hr, Row& row) {
      const int m = c.m0 + r;
      row.slot = c.ext > 0 && m < p.M ? p.row_slot[m] : -1;
      if (row.slot < 0) return;
      const float s = p.scale ? p.scale[p.row_adapter[m]] : p.scale0;
      const float* src = p.t + ((long long)(p.HR > 1 ? hr : c.z) * p.M + m) * p.rp;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (8 * i >= p.rp) break;
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 0.f;
#pragma unroll 4
        for (int part = 0; part < p.parts; ++part) {
          const float4 lo = *reinterpret_cast<const float4*>(src + part * p.t_part + 8 * i);
          const float4 hi = *reinterpret_cast<const float4*>(src + part * p.t_part + 8 * i + 4);
          f[0] += lo.x, f[1] += lo.y, f[2] += lo.z, f[3] += lo.w;
          f[4] += hi.x, f[5] += hi.y, f[6] += hi.z, f[7] += hi.w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = 8 * i + e < p.r ? f[e] * s : 0.f;  // b reads as zero past the rank
        row.t[i] = to_bf16x8(f);
      }
    };
    int buf = 0;
    uint32_t buf_phase = 0;
    bool ok = true;
    Row row, next;
    int t = blockIdx.x, hr = 0;
    AdapterWalk walk(p, blockIdx.x, gridDim.x);
    AdapterTile c = adapter_tile(p, walk, BN);
    fetch(c, 0, row);
    while (ok && t < total) {
      const int hr2 = hr + 1 < p.HR ? hr + 1 : 0;
      const int t2 = hr2 ? t : t + (int)gridDim.x;
      if (!hr2) walk.next();
      const AdapterTile c2 = hr2 || t2 >= total ? c : adapter_tile(p, walk, BN);
      if (t2 < total) fetch(c2, hr2, next);
      for (int e = 0; e < c.ext; ++e) {
        const int block = hr * c.ext + e;
        if (block < c.e0 || block >= c.e1) continue;
        // the same answer for the whole warp: its lanes go on together
        if (!__all_sync(0xffffffffu,
                        mbar_wait_bounded(&used_bar[buf], buf_phase ^ 1, &abort_flag, p.err, kErrTimeoutProducer))) {
          ok = false;
          break;
        }
        uint8_t* dst = sExt + buf * Cfg::A_BYTES;
        // The row's slot in this block. Its other columns hold what they held: those products are masked off.
        const int j = row.slot - e * p.per_block;
        const bool here = row.slot >= 0 && j >= 0 && j < p.per_block;
        if (here) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (8 * i < p.rp) *reinterpret_cast<uint4*>(dst + sw128(r, j * p.rp / 8 + i)) = row.t[i];
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t own = __ballot_sync(0xffffffffu, here && j == s);
          if (lane == 0) reinterpret_cast<uint32_t*>(&rows_off[buf][s])[r / 32] = ~own;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&built_bar[buf]);
        if (++buf == EXT) {
          buf = 0;
          buf_phase ^= 1;
        }
      }
      row = next;
      t = t2, hr = hr2;
      c = c2;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// y [M, Z, N] bf16 = the sum of the parts [splits, Z, M, N] in a fixed order: 32 lanes take 4 columns each, 8 warps
// every eighth part, so that few columns of many parts do not wait for one another.
__global__ void __launch_bounds__(256) adapter_sum_kernel(const float* __restrict__ partial, int splits, int Z, int M,
                                                          int N, bf16* __restrict__ y) {
  __shared__ float4 red[8][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long long n = (long long)Z * M * N, i = ((long long)blockIdx.x * 32 + lane) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < n) {
#pragma unroll 4
    for (int q = warp; q < splits; q += 8) {
      const float4 v = *reinterpret_cast<const float4*>(partial + q * n + i);
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
  }
  red[warp][lane] = s;
  __syncthreads();
  if (warp > 0 || i >= n) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) {
    const float4 v = red[q][lane];
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  const int col = (int)(i % N);
  const long long zm = i / N;
  __nv_bfloat162 lo = __floats2bfloat162_rn(s.x, s.y), hi = __floats2bfloat162_rn(s.z, s.w);
  *reinterpret_cast<uint2*>(y + ((zm % M) * Z + zm / M) * N + col) =
      make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
}

// t [n] = the sum of its parts [parts, n], n a multiple of 4.
__global__ void __launch_bounds__(256) adapter_fold_kernel(const float* __restrict__ in, int parts, long long n,
                                                           float* __restrict__ out) {
  const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int q = 0; q < parts; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(in + q * n + i);
    s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
  }
  *reinterpret_cast<float4*>(out + i) = s;
}

// ------------------------------------------------------------------------------- weight gradients

struct GradArgs {
  const bf16* x;  // x or dy: rows of C values
  long long x_row, x_head;
  const float* t;  // [H, M, rp]
  const int* order;
  const int* group;    // [G + 1]: the rows of adapter g in `order`
  const int* by_size;  // adapters, the ones with most rows first
  const float* scale;
  float scale0;
  bf16* out;      // [G, H, r, C] = s t_g^T x_g
  const bf16* w;  // [G, H, r, C]: with WITH_U also u[slab, h, m, :] = x[m] w[g]^T over the slab's columns
  float* u;
  int M, H, r, C;
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&v)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(addr));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0) : "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

constexpr int kGradRows = 32;

// Padded rows: ldmatrix (x, w) and the fragments of t are read without bank conflicts.
template <int MT, int SLAB, bool WITH_U>
struct GradCfg {
  static constexpr int RP = 16 * MT, XP = SLAB + 8, TP = RP + 4;
  static constexpr int STAGES = SLAB > 128 ? 2 : 3;  // wide: two CTAs an SM (MT = 1) hide more than a third stage
  static constexpr int X_BYTES = kGradRows * XP * 2, T_BYTES = kGradRows * TP * 4;
  static constexpr int W_BYTES = WITH_U ? RP * XP * 2 : 0, RED_BYTES = WITH_U ? 4 * kGradRows * TP * 4 : 0;
  static constexpr int SMEM = STAGES * (X_BYTES + T_BYTES) + W_BYTES + RED_BYTES;
};

// One adapter, head and SLAB columns a CTA; the adapter's rows in steps of 32, staged by cp.async. A warp
// holds SLAB / 8 columns of the gradient in registers. With WITH_U the same staged rows also give
// their products with the adapter's other matrix, so that dy is read once for u and db: bound by that read.
template <int MT, int SLAB, bool WITH_U>
__global__ void __launch_bounds__(256) adapter_grad_kernel(const __grid_constant__ GradArgs p) {
  using Cfg = GradCfg<MT, SLAB, WITH_U>;
  constexpr int RP = Cfg::RP, XP = Cfg::XP, TP = Cfg::TP, ST = Cfg::STAGES, NT = SLAB / 64;
  extern __shared__ __align__(16) uint8_t smem[];
  bf16* xs = reinterpret_cast<bf16*>(smem);
  float* ts = reinterpret_cast<float*>(smem + ST * Cfg::X_BYTES);
  bf16* ws = reinterpret_cast<bf16*>(smem + ST * (Cfg::X_BYTES + Cfg::T_BYTES));
  float* red = reinterpret_cast<float*>(smem + ST * (Cfg::X_BYTES + Cfg::T_BYTES) + Cfg::W_BYTES);
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int c0 = blockIdx.x * SLAB, h = blockIdx.y, g = p.by_size[blockIdx.z];
  const int r0 = p.group[g], rows = p.group[g + 1] - r0;
  const int steps = (rows + kGradRows - 1) / kGradRows;
  const long long gh = (long long)g * p.H + h;
  auto load = [&](int step, int buf) {
    if (step < steps) {
#pragma unroll 4
      for (int i = tid; i < kGradRows * (SLAB / 8); i += 256) {
        const int row = i / (SLAB / 8), c = (i % (SLAB / 8)) * 8;
        const int at = step * kGradRows + row;
        const bool in = at < rows && c0 + c < p.C;
        cp_async16(xs + (buf * kGradRows + row) * XP + c,
                   in ? p.x + (long long)p.order[r0 + at] * p.x_row + (long long)h * p.x_head + c0 + c : p.x, in);
      }
      for (int i = tid; i < kGradRows * (RP / 4); i += 256) {
        const int row = i / (RP / 4), c = (i % (RP / 4)) * 4;
        const int at = step * kGradRows + row;
        const bool in = at < rows;
        cp_async16(ts + (buf * kGradRows + row) * TP + c,
                   in ? p.t + ((long long)h * p.M + p.order[r0 + at]) * RP + c : p.t, in);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (WITH_U) {
    for (int i = tid; i < RP * (SLAB / 8); i += 256) {
      const int row = i / (SLAB / 8), c = (i % (SLAB / 8)) * 8;
      const bool in = row < p.r && c0 + c < p.C;
      cp_async16(ws + row * XP + c, in ? p.w + (gh * p.r + row) * p.C + c0 + c : p.w, in);
    }
  }
  float acc[MT][NT][4];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[mt][nt][i] = 0.f;
#pragma unroll
  for (int q = 0; q < ST - 1; ++q) load(q, q);
  for (int step = 0; step < steps; ++step) {
    const int buf = step % ST;
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncthreads();
    load(step + ST - 1, (step + ST - 1) % ST);
    const bf16* xb = xs + buf * kGradRows * XP;
    const float* tb = ts + buf * kGradRows * TP;
    // out += t^T x: rank rows, the warp's columns, a 16-row reduction each
#pragma unroll
    for (int kk = 0; kk < kGradRows / 16; ++kk) {
      uint32_t a[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float* q = tb + (kk * 16 + (i / 2) * 8 + 2 * (lane % 4)) * TP + mt * 16 + (i % 2) * 8 + lane / 4;
          a[mt][i] = pack_bf16(q[0], q[TP]);
        }
#pragma unroll
      for (int nt = 0; nt < NT; nt += 2) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, smem_u32(xb + (kk * 16 + (lane & 15)) * XP + warp * (SLAB / 8) + nt * 8 + (lane >> 4) * 8));
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma_bf16(acc[mt][nt], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[0], b[1]);
          mma_bf16(acc[mt][nt + 1], a[mt][0], a[mt][1], a[mt][2], a[mt][3], b[2], b[3]);
        }
      }
    }
    if constexpr (WITH_U) {
      // u = x w^T: 16 rows and a quarter of the columns a warp, folded over the quarters
      const int m0 = (warp & 1) * 16, q0 = (warp >> 1) * (SLAB / 4);
      float uacc[2 * MT][4];
#pragma unroll
      for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) uacc[j][i] = 0.f;
#pragma unroll 4
      for (int kk = 0; kk < SLAB / 64; ++kk) {
        uint32_t a[4];
        ldmatrix_x4(a, smem_u32(xb + (m0 + (lane & 15)) * XP + q0 + kk * 16 + (lane >> 4) * 8));
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          uint32_t b[4];
          ldmatrix_x4(b, smem_u32(ws + (j * 16 + (lane & 7) + (lane >> 4) * 8) * XP + q0 + kk * 16 + ((lane >> 3) & 1) * 8));
          mma_bf16(uacc[2 * j], a[0], a[1], a[2], a[3], b[0], b[1]);
          mma_bf16(uacc[2 * j + 1], a[0], a[1], a[2], a[3], b[2], b[3]);
        }
      }
#pragma unroll
      for (int j = 0; j < 2 * MT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[((warp >> 1) * kGradRows + m0 + lane / 4 + (i / 2) * 8) * TP + j * 8 + 2 * (lane % 4) + i % 2] = uacc[j][i];
      __syncthreads();
      for (int i = tid; i < kGradRows * RP; i += 256) {
        const int row = i / RP, c = i % RP, at = step * kGradRows + row;
        if (at < rows) {
          float f = 0.f;
#pragma unroll
          for (int q = 0; q < 4; ++q) f += red[(q * kGradRows + row) * TP + c];
          p.u[(((long long)blockIdx.x * p.H + h) * p.M + p.order[r0 + at]) * RP + c] = f;
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  const float s = rows == 0 ? 0.f : p.scale ? p.scale[g] : p.scale0;  // 0 even where the scale is not finite
  bf16* out = p.out + gh * p.r * p.C;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = mt * 16 + lane / 4 + 8 * i, col = c0 + warp * (SLAB / 8) + nt * 8 + 2 * (lane % 4);
        if (row < p.r && col < p.C)
          *reinterpret_cast<__nv_bfloat162*>(out + (long long)row * p.C + col) =
              __floats2bfloat162_rn(acc[mt][nt][2 * i] * s, acc[mt][nt][2 * i + 1] * s);
      }
}

// ------------------------------------------------------------------------------- host

// The batch's plan: one int32 buffer, and where its parts lie.
struct Plan {
  int M, G, tiles, chunks, rows_per_chunk, rows;  // rows: those with an adapter
  const int *row_adapter, *row_slot, *tile_ptr, *slots, *order, *chunk, *group, *by_size;
};

Plan read_plan(const at::Tensor& buf, const std::vector<int64_t>& d, int dev) {
  TORCH_CHECK(buf.is_cuda() && buf.get_device() == dev, "adapter_linear: the batch's plan must be on the operands' GPU");
  TORCH_CHECK(buf.scalar_type() == at::kInt && buf.is_contiguous() && d.size() == 7,
              "adapter_linear: bad batch plan");
  Plan p;
  p.M = (int)d[0], p.G = (int)d[1], p.tiles = (int)d[2], p.rows = (int)d[4], p.chunks = (int)d[5], p.rows_per_chunk = (int)d[6];
  const int* b = buf.data_ptr<int>();
  p.row_adapter = b, b += p.M;
  p.row_slot = b, b += p.M;
  p.tile_ptr = b, b += p.tiles + 1;
  p.slots = b, b += d[3];
  p.order = b, b += p.rows;
  p.chunk = b, b += 3 * p.chunks;
  p.group = b, b += p.G + 1;
  p.by_size = b;
  TORCH_CHECK(buf.numel() == 2 * d[0] + d[2] + 1 + d[3] + d[4] + 3 * d[5] + 2 * d[1] + 1, "adapter_linear: bad batch plan");
  return p;
}

int padded_rank(int64_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : 64; }

struct Rows {  // [M, C] shared by the heads, or [M, H, C]
  const bf16* p;
  long long row, head;
  int C;
};

Rows rows_of(const at::Tensor& t, bool per_head) {
  Rows r;
  r.p = reinterpret_cast<const bf16*>(t.data_ptr());
  r.row = t.stride(0);
  r.head = per_head ? t.stride(1) : 0;
  r.C = (int)t.size(-1);
  return r;
}

at::Tensor shrink(const Rows& x, const at::Tensor& a, const Plan& p, int H, int r, cudaStream_t st) {
  const int rp = padded_rank(r);
  const long long ctas = (long long)p.chunks * H;
  // parts of the reduction: enough CTAs for four a SM, at least 512 values each, 32 at most
  const int parts = (int)std::max<long long>(1, std::min<long long>({32, (x.C + 511) / 512, (592 + ctas - 1) / ctas}));
  const int part_k = ((x.C + parts - 1) / parts + 31) / 32 * 32;
  const int used = (x.C + part_k - 1) / part_k;
  at::Tensor t = at::empty({used, H, p.M, rp}, a.options().dtype(at::kFloat));
  ShrinkArgs s{x.p, x.row, x.head, reinterpret_cast<const bf16*>(a.data_ptr()), t.data_ptr<float>(), p.order, p.chunk,
               p.M, H, x.C, r, part_k};
  const dim3 grid((unsigned)p.chunks, (unsigned)H, (unsigned)used);
  auto go = [&](auto mt) {
    if (p.rows_per_chunk <= 8)
      adapter_shrink_kernel<decltype(mt)::value, 1><<<grid, kShrinkThreads, 0, st>>>(s);
    else
      adapter_shrink_kernel<decltype(mt)::value, 4><<<grid, kShrinkThreads, 0, st>>>(s);
  };
  if (rp == 16)
    go(std::integral_constant<int, 1>());
  else if (rp == 32)
    go(std::integral_constant<int, 2>());
  else
    go(std::integral_constant<int, 4>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return t;
}

template <int BN, bool W_MN, int EXT>
void launch_gemm(const AdapterGemm& p, cudaStream_t st, int dev, bool after_shrink) {
  using Cfg = AdapterCfg<BN, EXT>;
  static_assert(Cfg::SMEM <= 226 * 1024, "shared memory of the projection kernel");
  auto kern = adapter_gemm_kernel<BN, W_MN, EXT>;
  static bool attr_set[64] = {false};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM));
    attr_set[dev] = true;
  }
  const long long total = (long long)p.tiles_m * p.tiles_n * p.splits * p.Z;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<long long>(total, num_sms_of(dev)));
  cfg.blockDim = dim3(kAdapterThreads);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after_shrink ? 1 : 0;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, p));
  ++counted_launches;
}

// out [M, Z, N] = sum over the reduction's heads of x w (+ s t b).
at::Tensor project(const Rows& x, const at::Tensor& w, bool w_mn, bool sum_heads, const at::Tensor& b,
                   const at::Tensor& t, const Plan& plan, int r, const c10::optional<at::Tensor>& scale, double scale0,
                   const at::Tensor& err, cudaStream_t st, int dev) {
  const int H = (int)w.size(0), K = (int)w.size(w_mn ? 1 : 2), N = (int)w.size(w_mn ? 2 : 1), M = plan.M;
  AdapterGemm p;
  memset(&p, 0, sizeof(p));
  p.M = M, p.N = N, p.KB = (K + 63) / 64, p.H = H;
  p.HR = sum_heads ? H : 1;
  p.Z = sum_heads ? 1 : H;
  p.x_heads = x.head != 0;
  p.r = r, p.rp = padded_rank(r), p.per_block = 64 / p.rp;
  p.block_shift = p.per_block == 4 ? 2 : p.per_block == 2 ? 1 : 0;
  TORCH_CHECK(((long long)p.KB + 128) * p.HR < (1 << 22), "adapter_linear: the reduction is too long");
  const bool adapters = plan.rows > 0;
  if (adapters) {
    p.t = t.data_ptr<float>(), p.parts = (int)t.size(0), p.t_part = t.stride(0);
    p.row_slot = plan.row_slot, p.row_adapter = plan.row_adapter, p.tile_ptr = plan.tile_ptr, p.slots = plan.slots;
    p.scale = scale ? scale->data_ptr<float>() : nullptr, p.scale0 = (float)scale0;
  }
  p.err = err.data_ptr<int>();
  p.tiles_m = (M + 127) / 128;
  // The tile width and the number of parts of the reduction: what the busiest CTA stages (a 64-wide block is 16 KB
  // of x and 128 B a column of w, and the operands' way into shared memory bounds the loop), and the fp32 parts
  // that are written and read again, spread over the chip. Wide tiles stage less per column; few
  // tiles leave SMs idle unless the reduction is split.
  const int sms = num_sms_of(dev);
  const long long blocks = (long long)p.HR * p.KB;
  int bn = 64;
  double best = 1e30;
  p.splits = 1;
  for (int w_ : {256, 128, 64}) {
    const long long tiles = (long long)p.tiles_m * ((N + w_ - 1) / w_) * p.Z;
    for (long long parts = 1; parts <= blocks / 4 || parts == 1; ++parts) {
      if (parts > 1 && tiles * parts > sms) break;
      const double waves = (double)((tiles * parts + sms - 1) / sms);
      double cost = waves * ((double)((blocks + parts - 1) / parts) * (16384.0 + 128.0 * w_) + 65536.0);
      if (parts > 1) cost += 8.0 * parts * M * N * p.Z / sms + 150000.0;
      if (cost < best) best = cost, bn = w_, p.splits = (int)parts;
    }
  }
  p.tiles_n = (N + bn - 1) / bn;
  at::Tensor y = at::empty({M, p.Z, N}, w.options());
  at::Tensor partial;
  if (p.splits > 1) {
    partial = at::empty({p.splits, p.Z, M, N}, w.options().dtype(at::kFloat));
    p.partial = partial.data_ptr<float>();
  }
  const int64_t xh = p.x_heads ? H : 1;
  p.tx = tensor_map_bf16(x.p, {K, M, xh}, {x.row, p.x_heads ? x.head : (int64_t)M * x.row}, 64, 128);
  if (w_mn)
    p.tw = tensor_map_bf16(w.data_ptr(), {N, K, H}, {w.stride(1), w.stride(0)}, 64, 64);
  else
    p.tw = tensor_map_bf16(w.data_ptr(), {K, N, H}, {w.stride(1), w.stride(0)}, 64, (uint32_t)bn);
  if (adapters)
    p.tb = tensor_map_bf16(b.data_ptr(), {N, r, b.size(0) * H}, {N, (int64_t)r * N}, 64, (uint32_t)p.rp);
  p.y = reinterpret_cast<bf16*>(y.data_ptr());
  // short: at most 16 blocks of the reduction between two adapter blocks' tiles
  const bool brief = blocks / p.splits <= 16;
  auto go = [&](auto width, auto ext) {
    constexpr int W = decltype(width)::value, E = decltype(ext)::value;
    if (w_mn)
      launch_gemm<W, true, E>(p, st, dev, adapters);
    else
      launch_gemm<W, false, E>(p, st, dev, adapters);
  };
  if (bn == 256 && brief)
    go(std::integral_constant<int, 256>(), std::integral_constant<int, 2>());
  else if (bn == 256)
    go(std::integral_constant<int, 256>(), std::integral_constant<int, 1>());
  else if (bn == 128)
    go(std::integral_constant<int, 128>(), std::integral_constant<int, 3>());
  else
    go(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
  if (p.splits > 1) {
    const long long n = (long long)p.Z * M * N;
    adapter_sum_kernel<<<(unsigned)((n + 127) / 128), 256, 0, st>>>(
        p.partial, p.splits, p.Z, M, N, reinterpret_cast<bf16*>(y.data_ptr()));
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    ++counted_launches;
  }
  return y;
}

// t with its parts summed.
at::Tensor fold(const at::Tensor& t, cudaStream_t st) {
  if (t.size(0) == 1) return t;
  at::Tensor out = at::empty({1, t.size(1), t.size(2), t.size(3)}, t.options());
  const long long n = out.numel();
  adapter_fold_kernel<<<(unsigned)((n + 1023) / 1024), 256, 0, st>>>(t.data_ptr<float>(), (int)t.size(0), n,
                                                                     out.data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
  return out;
}

template <int MT, int SLAB, bool WITH_U>
void launch_grad(const GradArgs& a, int G, cudaStream_t st, int dev) {
  constexpr int bytes = GradCfg<MT, SLAB, WITH_U>::SMEM;
  static_assert(bytes <= 227 * 1024, "shared memory of the gradient kernel");
  auto kern = adapter_grad_kernel<MT, SLAB, WITH_U>;
  static bool attr_set[64] = {false};
  if (!attr_set[dev]) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    attr_set[dev] = true;
  }
  kern<<<dim3((unsigned)((a.C + SLAB - 1) / SLAB), (unsigned)a.H, (unsigned)G), 256, bytes, st>>>(a);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  ++counted_launches;
}

constexpr int kWideSlab = 512, kNarrowSlab = 128;

// The gradient s t_g^T x_g of `like`; with `w` also u = x w^T in parts of 512 columns.
at::Tensor gradient(const Rows& x, const at::Tensor& t, const Plan& p, const at::Tensor& like, int H, int r,
                    const c10::optional<at::Tensor>& scale, double scale0, const at::Tensor* w, at::Tensor* u,
                    cudaStream_t st, int dev) {
  at::Tensor out = at::empty_like(like);
  GradArgs a{x.p, x.row, x.head, t.data_ptr<float>(), p.order, p.group, p.by_size,
             scale ? scale->data_ptr<float>() : nullptr, (float)scale0, reinterpret_cast<bf16*>(out.data_ptr()), nullptr,
             nullptr, p.M, H, r, x.C};
  const int rp = padded_rank(r);
  if (w) {
    *u = at::empty({(x.C + kWideSlab - 1) / kWideSlab, H, p.M, rp}, t.options());
    a.w = reinterpret_cast<const bf16*>(w->data_ptr());
    a.u = u->data_ptr<float>();
  }
  // narrow slabs where wide ones leave SMs without one (and nothing else comes out of them)
  const bool narrow = !w && (long long)p.G * H * ((x.C + kWideSlab - 1) / kWideSlab) < 2 * num_sms_of(dev);
  auto go = [&](auto mt) {
    constexpr int MT = decltype(mt)::value;
    if (w)
      launch_grad<MT, kWideSlab, true>(a, p.G, st, dev);
    else if (narrow)
      launch_grad<MT, kNarrowSlab, false>(a, p.G, st, dev);
    else
      launch_grad<MT, kWideSlab, false>(a, p.G, st, dev);
  };
  if (rp == 16)
    go(std::integral_constant<int, 1>());
  else if (rp == 32)
    go(std::integral_constant<int, 2>());
  else
    go(std::integral_constant<int, 4>());
  return out;
}

void check_operand(const at::Tensor& t, int dev, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.get_device() == dev && t.scalar_type() == at::kBFloat16, "adapter_linear: ", what,
              " must be bf16 on one GPU");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "adapter_linear: ", what, " must be 16-byte aligned");
  TORCH_CHECK(t.stride(-1) == 1, "adapter_linear: ", what, " must be contiguous in its last dimension");
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    TORCH_CHECK(t.stride(i) % 8 == 0, "adapter_linear: ", what, ": strides must be multiples of 8 values");
}

struct Checked {
  int H, K, N, r, dev;
};

Checked check_all(const at::Tensor& x, const at::Tensor& w, const at::Tensor& a, const at::Tensor& b, const Plan& p,
                  const c10::optional<at::Tensor>& scale) {
  const int dev = w.get_device();
  check_operand(x, dev, "x");
  check_operand(w, dev, "weight");
  check_operand(a, dev, "a");
  check_operand(b, dev, "b");
  TORCH_CHECK(w.dim() == 3 && a.dim() == 4 && b.dim() == 4 && a.is_contiguous() && b.is_contiguous(),
              "adapter_linear: weight [H, K, N]; a [G, H, r, K] and b [G, H, r, N] contiguous");
  const int64_t H = w.size(0), K = w.size(1), N = w.size(2), G = a.size(0), r = a.size(2);
  TORCH_CHECK(K % 8 == 0 && N % 8 == 0 && K > 0 && N > 0, "adapter_linear: K and N must be multiples of 8");
  TORCH_CHECK(r >= 1 && r <= 64, "adapter_linear: rank of 1 to 64");
  TORCH_CHECK(H <= 65535 && G <= 65535, "adapter_linear: at most 65535 heads and adapters");
  TORCH_CHECK(a.size(1) == H && a.size(3) == K && b.size(0) == G && b.size(1) == H && b.size(2) == r && b.size(3) == N,
              "adapter_linear: a and b do not fit the weight");
  TORCH_CHECK(G == p.G, "adapter_linear: the batch was planned for ", p.G, " adapters, not ", G);
  TORCH_CHECK((x.dim() == 2 || (x.dim() == 3 && x.size(1) == H)) && x.size(0) == p.M && x.size(-1) == K,
              "adapter_linear: x must be [M, K] or [M, H, K] with the batch's ", p.M, " rows");
  if (scale)
    TORCH_CHECK(scale->is_cuda() && scale->get_device() == dev && scale->scalar_type() == at::kFloat && scale->dim() == 1 &&
                    scale->size(0) == G && scale->is_contiguous(),
                "adapter_linear: scale must be fp32 [adapters]");
  return Checked{(int)H, (int)K, (int)N, (int)r, dev};
}

}  // namespace

std::vector<at::Tensor> adapter_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& a, const at::Tensor& b,
                                        const at::Tensor& plan, const std::vector<int64_t>& dims,
                                        const c10::optional<at::Tensor>& scale, double scale0, const at::Tensor& err);

namespace {
bool direct(const at::Tensor& t, int dev, int64_t inner) {
  if (!t.is_cuda() || t.get_device() != dev || t.scalar_type() != at::kBFloat16 || t.requires_grad()) return false;
  if (t._fw_grad(0).defined()) return false;  // a forward-mode tangent: refused, not dropped
  if (t.stride(-1) != 1 || t.size(-1) != inner || inner % 8 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 || t.stride(i) <= 0) return false;
  return true;
}
}  // namespace

// The call without gradients and without copies, with or without heads: y, or nothing where an argument needs a
// look (a copy, a gradient, an error). One crossing from Python for a token's projection.
c10::optional<at::Tensor> adapter_direct(const at::Tensor& x, const at::Tensor& w, const at::Tensor& a, const at::Tensor& b,
                                         const at::Tensor& plan, const std::vector<int64_t>& dims,
                                         const c10::optional<at::Tensor>& scale, double scale0, const at::Tensor& err) {
  const bool heads = w.dim() == 3;
  if (!w.is_cuda() || !(heads || w.dim() == 2) || a.dim() != w.dim() + 1 || b.dim() != w.dim() + 1) return c10::nullopt;
  const int dev = w.get_device();
  if (!(x.dim() == 2 || (heads && x.dim() == 3)) || !plan.is_cuda() || plan.get_device() != dev) return c10::nullopt;
  const int64_t H = heads ? w.size(0) : 1, K = w.size(-2), N = w.size(-1), G = a.size(0), r = a.size(-2);
  if (!direct(x, dev, K) || !direct(w, dev, N) || !direct(a, dev, K) || !direct(b, dev, N)) return c10::nullopt;
  if (!a.is_contiguous() || !b.is_contiguous() || r < 1 || r > 64 || G != dims[1] || dims[0] == 0 || x.size(0) != dims[0])
    return c10::nullopt;
  if (b.size(0) != G || b.size(-2) != r || (heads && (a.size(1) != H || b.size(1) != H || (x.dim() == 3 && x.size(1) != H))))
    return c10::nullopt;
  if (scale && (!scale->is_cuda() || scale->get_device() != dev || scale->scalar_type() != at::kFloat || scale->dim() != 1 ||
                scale->size(0) != G || !scale->is_contiguous() || scale->requires_grad() || scale->_fw_grad(0).defined()))
    return c10::nullopt;
  if (heads) return adapter_forward(x, w, a, b, plan, dims, scale, scale0, err)[0];
  return adapter_forward(x, w.unsqueeze(0), a.unsqueeze(1), b.unsqueeze(1), plan, dims, scale, scale0, err)[0].view(
      {x.size(0), N});
}

// y [M, H, N], and t [parts, H, M, rp] fp32 (empty without adapters) for the backward pass.
std::vector<at::Tensor> adapter_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& a, const at::Tensor& b,
                                        const at::Tensor& plan, const std::vector<int64_t>& dims,
                                        const c10::optional<at::Tensor>& scale, double scale0, const at::Tensor& err) {
  const Plan p = read_plan(plan, dims, w.get_device());
  const Checked c = check_all(x, w, a, b, p, scale);
  c10::cuda::CUDAGuard guard(c.dev);
  auto st = at::cuda::getCurrentCUDAStream(c.dev).stream();
  const Rows rows = rows_of(x, x.dim() == 3);
  at::Tensor t;
  if (p.rows > 0)
    t = shrink(rows, a, p, c.H, c.r, st);
  else
    t = at::empty({0}, a.options().dtype(at::kFloat));
  return {project(rows, w, true, false, b, t, p, c.r, scale, scale0, err, st, c.dev), t};
}

// dx (like x), da, db from dy [M, H, N]; an output that is not asked for is an empty tensor.
std::vector<at::Tensor> adapter_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w,
                                         const at::Tensor& a, const at::Tensor& b, const at::Tensor& t,
                                         const at::Tensor& plan, const std::vector<int64_t>& dims,
                                         const c10::optional<at::Tensor>& scale, double scale0, const at::Tensor& err,
                                         bool want_dx, bool want_da, bool want_db) {
  const Plan p = read_plan(plan, dims, w.get_device());
  const Checked c = check_all(x, w, a, b, p, scale);
  check_operand(dy, c.dev, "dy");
  TORCH_CHECK(dy.dim() == 3 && dy.size(0) == p.M && dy.size(1) == c.H && dy.size(2) == c.N, "adapter_linear: dy [M, H, N]");
  c10::cuda::CUDAGuard guard(c.dev);
  auto st = at::cuda::getCurrentCUDAStream(c.dev).stream();
  const bool shared = x.dim() == 2;
  const Rows rx = rows_of(x, !shared), ry = rows_of(dy, true);
  at::Tensor none = at::empty({0}, w.options()), u, dx = none, da = none, db = none;
  const bool want_u = want_dx || want_da;
  if (p.rows == 0) {
    if (want_da) da = at::zeros_like(a);
    if (want_db) db = at::zeros_like(b);
  } else if (want_db) {
    db = gradient(ry, fold(t, st), p, b, c.H, c.r, scale, scale0, want_u ? &b : nullptr, &u, st, c.dev);
    if (want_u) u = fold(u, st);
  } else if (want_u) {
    u = shrink(ry, b, p, c.H, c.r, st);
  }
  if (want_dx) dx = project(ry, w, false, shared, a, u, p, c.r, scale, scale0, err, st, c.dev);
  if (want_da && p.rows > 0)
    da = gradient(rx, fold(u, st), p, a, c.H, c.r, scale, scale0, nullptr, nullptr, st, c.dev);
  return {dx, da, db};
}

}  // namespace bd
