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

#include <algorithm>

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
  unsigned size[4];       // tiles_n, tiles_m, splits, heads of the output
  unsigned step[5];       // how far a worker goes from tile to tile, in digits of these sizes
  uint32_t idesc;
  float* partial;         // [splits, NB, sets, heads, M, N] where the reduction is split
  int* err;
  FfOut e;
};

// ------------------------------------------------------------------------------- arithmetic

// Pairs of fp32 values in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float exp2_approx(float x) {
  float r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float relu_nan(float x) {  // NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
  return r;
}

// The normal distribution's cdf at p, and exp(-p^2 / 2) where it is wanted. The lower tail at x = |p| is
// exp(-x^2 / 2) 2^R(x), R a least-squares fit of degree 8 on [0, 5] and constant from there: the tail is off by 8e-6 of
// itself to x = 5, by 1.4e-7 anywhere, p cdf(p) by 2e-7. One exponential a value and no quotient: with two of the
// latter's kind (a Chebyshev form of erfc) the special-function unit bound the epilogue (67 M outputs: 115 us).
__device__ __forceinline__ float2 normal_cdf2(float2 p, float2* bell) {
  const float2 x = make_float2(fminf(fabsf(p.x), 5.f), fminf(fabsf(p.y), 5.f));
  float2 q = both(-6.862234727122996e-07f);
  q = fma2(q, x, both(1.1530738447618205e-05f));
  q = fma2(q, x, both(-4.327946589910425e-05f));
  q = fma2(q, x, both(-0.0005067124147899449f));
  q = fma2(q, x, both(0.007572786882519722f));
  q = fma2(q, x, both(-0.05285993218421936f));
  q = fma2(q, x, both(0.2622605562210083f));
  q = fma2(q, x, both(-1.1511198282241821f));
  q = fma2(q, x, both(-0.9999997019767761f));
  const float2 e = mul2(mul2(p, p), both(-0.72134752f));
  q = add2(q, e);
  const float2 c = make_float2(exp2_approx(q.x), exp2_approx(q.y)), u = fma2(c, both(-1.f), both(1.f));
  if (bell) *bell = make_float2(exp2_approx(e.x), exp2_approx(e.y));
  return make_float2(p.x < 0.f ? c.x : u.x, p.y < 0.f ? c.y : u.y);
}

__device__ __forceinline__ float2 sigmoid2(float2 p) {
  const float2 e = mul2(p, both(-1.44269504f));
  const float2 w = add2(make_float2(exp2_approx(e.x), exp2_approx(e.y)), both(1.f));
  return make_float2(rcp_approx(w.x), rcp_approx(w.y));
}

template <int ACT>
__device__ __forceinline__ float2 ff_act(float2 p) {
  if constexpr (ACT == FF_RELU) return make_float2(relu_nan(p.x), relu_nan(p.y));
  if constexpr (ACT == FF_SILU) return mul2(p, sigmoid2(p));
  if constexpr (ACT == FF_GELU) return mul2(p, normal_cdf2(p, nullptr));
  return p;
}

// act(p) and its derivative.
template <int ACT>
__device__ __forceinline__ void ff_act_both(float2 p, float2& f, float2& d) {
  if constexpr (ACT == FF_RELU) {
    f = make_float2(relu_nan(p.x), relu_nan(p.y));
    d = make_float2(p.x > 0.f ? 1.f : 0.f, p.y > 0.f ? 1.f : 0.f);
  } else if constexpr (ACT == FF_SILU) {
    const float2 s = sigmoid2(p);
    f = mul2(p, s);
    d = fma2(f, fma2(s, both(-1.f), both(1.f)), s);  // s + p s (1 - s)
  } else if constexpr (ACT == FF_GELU) {
    float2 bell;
    const float2 cdf = normal_cdf2(p, &bell);
    f = mul2(p, cdf);
    d = fma2(mul2(p, both(0.3989422804014327f)), bell, cdf);
  } else {
    f = p, d = both(1.f);
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

__device__ __forceinline__ float2 pair_of(const float* v, int i) { return make_float2(v[2 * i], v[2 * i + 1]); }
__device__ __forceinline__ void put_pair(float* v, int i, float2 x) { v[2 * i] = x.x, v[2 * i + 1] = x.y; }

// n values (even) of the forward pass, in place: p becomes act(p) or act(p) up(u).
template <int EPI, int n>
__device__ __forceinline__ void ff_forward_values(const FfOut& e, float* p, float* u) {
  if constexpr (EPI == FF_GATED) {
    if (e.up_relu) {
#pragma unroll
      for (int i = 0; i < n; ++i) u[i] = relu_nan(u[i]);
    }
  }
  ff_with_act(e.act, [&](auto a) {
#pragma unroll
    for (int i = 0; i < n / 2; ++i) {
      float2 f = ff_act<decltype(a)::value>(pair_of(p, i));
      if constexpr (EPI == FF_GATED) f = mul2(f, pair_of(u, i));
      put_pair(p, i, f);
    }
  });
}

// n values of the backward pass, in place: p becomes dp, or p and u become dg and du. dy(i) gives the pair i of dy.
template <int EPI, int n, int ACT, typename DY>
__device__ __forceinline__ void ff_backward_values(bool up_relu, float* p, float* u, DY&& dy) {
#pragma unroll
  for (int i = 0; i < n / 2; ++i) {
    const float2 y = dy(i);
    float2 f, d;
    ff_act_both<ACT>(pair_of(p, i), f, d);
    if constexpr (EPI == FF_ACT_BWD) {
      put_pair(p, i, mul2(y, d));
    } else {
      float2 h = pair_of(u, i), du = mul2(y, f);
      if (up_relu) {
        du = make_float2(h.x > 0.f ? du.x : 0.f, h.y > 0.f ? du.y : 0.f);
        h = make_float2(relu_nan(h.x), relu_nan(h.y));
      }
      put_pair(p, i, mul2(mul2(y, h), d));
      put_pair(u, i, du);
    }
  }
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
  if (half)
    return make_uint4(ff_pack2(v[0], v[1], 1), ff_pack2(v[2], v[3], 1), ff_pack2(v[4], v[5], 1), ff_pack2(v[6], v[7], 1));
  return make_uint4(ff_pack2(v[0], v[1], 0), ff_pack2(v[2], v[3], 0), ff_pack2(v[4], v[5], 0), ff_pack2(v[6], v[7], 0));
}
__device__ __forceinline__ void ff_unpack8(uint4 q, int half, float* v) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  if (half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) put_pair(v, i, ff_unpack2(w[i], 1));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) put_pair(v, i, ff_unpack2(w[i], 0));
  }
}

// Adds the bias to 8 columns.
__device__ __forceinline__ void ff_bias8(const FfOut& e, int s, int head, int col, float* v) {
  float b[8];
  const long long at = (long long)head * e.N + col;
  if (!e.bias[s]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = e.bias0[s];
  } else if (e.bias_f32) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(e.bias[s]) + at);
    const float4 lo = __ldg(q), hi = __ldg(q + 1);
    b[0] = lo.x, b[1] = lo.y, b[2] = lo.z, b[3] = lo.w, b[4] = hi.x, b[5] = hi.y, b[6] = hi.z, b[7] = hi.w;
  } else {
    ff_unpack8(__ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(e.bias[s]) + at)), e.half, b);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) put_pair(v, i, add2(pair_of(v, i), pair_of(b, i)));
}

__device__ __forceinline__ bool ff_has_bias(const FfOut& e, int s) { return e.bias[s] || e.bias0[s] != 0.f; }

// ------------------------------------------------------------------------------- epilogue of 32 x 32 values a warp

// A warp's 32 x 32 tile of 16-bit values in shared memory (2 KB): rows of 64 bytes, their 16-byte pieces turned by the
// row, so that a lane's row and four lanes' row are both free of bank conflicts. Global rows then move 64 bytes at a time.
__device__ __forceinline__ uint32_t ff_piece(int row, int q) { return (uint32_t)(row * 64 + ((q ^ ((row >> 1) & 3)) << 4)); }

struct FfAux {
  uint4 v[4];
};

__device__ __forceinline__ void ff_load_aux(FfAux& a, const FfOut& e, int head, int row0, int col, int lane) {
  const int c = col + 8 * (lane & 3), r = row0 + lane / 4;
  const uint16_t* src = reinterpret_cast<const uint16_t*>(e.aux) + (long long)r * e.aux_ld + (long long)head * e.aux_head + c;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a.v[i] = make_uint4(0u, 0u, 0u, 0u);
    if (r + 8 * i < e.M && c < e.N) a.v[i] = *reinterpret_cast<const uint4*>(src + 8 * i * e.aux_ld);
  }
}

__device__ __forceinline__ void ff_put_aux(const FfAux& a, uint8_t* buf, int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(buf + ff_piece(8 * i + lane / 4, lane & 3)) = a.v[i];
  __syncwarp();
}

// The warp's tile in shared memory to rows [row0, row0 + 32) x 32 columns.
__device__ __forceinline__ void ff_flush(const FfOut& e, void* out, long long ld, long long head_stride, int head, int row0,
                                         int col, const uint8_t* buf, int lane) {
  __syncwarp();
  const int c = col + 8 * (lane & 3), r = lane / 4;
  uint16_t* o = reinterpret_cast<uint16_t*>(out) + (long long)(row0 + r) * ld + (long long)head * head_stride + c;
  const int rows = c < e.N ? e.M - row0 - r : 0;  // 8 i below it
  uint4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint4*>(buf + ff_piece(8 * i + r, lane & 3));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (8 * i < rows) *reinterpret_cast<uint4*>(o + 8 * i * ld) = w[i];
}

// Rows [row0, row0 + 32) x 32 columns from the lanes' rows.
__device__ __forceinline__ void ff_store_tile(const FfOut& e, void* out, long long ld, long long head_stride, int head,
                                              const float* v, int row0, int col, uint8_t* buf, int lane) {
  __syncwarp();
  if (e.half) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(buf + ff_piece(lane, q)) = ff_pack8(v + 8 * q, 1);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint4*>(buf + ff_piece(lane, q)) = ff_pack8(v + 8 * q, 0);
  }
  ff_flush(e, out, ld, head_stride, head, row0, col, buf, lane);
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

// Sums over the warp's 32 rows (a row a lane) of n = 16 or 32 columns: lane l gets column l % n's. v is used up. The
// order is fixed.
template <int n>
__device__ __forceinline__ float ff_column_sum(float* v, int lane) {
  if constexpr (n == 16) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], 16);
  }
#pragma unroll
  for (int o = n / 2; o > 0; o /= 2) {
    const bool hi = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float send = hi ? v[i] : v[i + o], mine = hi ? v[i + o] : v[i];
      v[i] = mine + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

template <int n>
__device__ __forceinline__ void ff_put_sums(const FfOut& e, int s, int head, float* v, int row0, int col, int lane) {
  const bool in = row0 + lane < e.M;
#pragma unroll
  for (int i = 0; i < n; ++i) v[i] = in ? v[i] : 0.f;
  const float sum = ff_column_sum<n>(v, lane);
  if (lane < n && col + lane < e.N) e.colsum[s][((long long)(row0 / 32) * e.heads + head) * e.N + col + lane] = sum;
}

template <int EPI>
__device__ __forceinline__ bool ff_has_aux(const FfOut& e) {
  return ff_backward(EPI) || (EPI == FF_ACT && e.aux != nullptr);
}

// 16 columns of one or both accumulators, one wait.
__device__ __forceinline__ void tmem_ld16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
                 "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at));
}
template <int NB>
__device__ __forceinline__ void ff_read16(uint32_t g_at, float (&g)[16], uint32_t u_at, float (&u)[16]) {
  uint32_t a[16], b[16];
  tmem_ld16(g_at, a);
  if constexpr (NB == 2) tmem_ld16(u_at, b);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    g[i] = __uint_as_float(a[i]);
    if constexpr (NB == 2) u[i] = __uint_as_float(b[i]);
  }
}

template <int n>
__device__ __forceinline__ void ff_add_bias(const FfOut& e, int s, int head, int col, float* v) {
  if (!ff_has_bias(e, s)) return;
#pragma unroll
  for (int q = 0; q < n / 8; ++q)
    if (col + 8 * q < e.N) ff_bias8(e, s, head, col + 8 * q, v + 8 * q);
}

// A warp's 32 x 32 chunk. g_at, u_at: its accumulators (one or two); aux: r or dy, as ff_load_aux left it; release:
// called once the accumulators have been read. The arithmetic goes over 16 columns at a time, and each result takes the
// place in shared memory that r or dy had: sixteen warps leave a thread 96 registers, and with both products of 32
// columns in them spills wrote as many bytes as the results.
template <int EPI, typename R>
__device__ __forceinline__ void ff_epilogue(const FfOut& e, int set, int head, int row0, int col, uint32_t g_at,
                                            uint32_t u_at, const FfAux& aux, uint8_t* buf, int lane, R&& release) {
  constexpr int NB = ff_products(EPI);
  if constexpr (EPI == FF_STORE) {
    float g[32];
    tmem_ld32(g_at, g);
    release();
    ff_store_tile(e, e.out[set], e.ld, e.head, head, g, row0, col, buf, lane);
    return;
  } else {
    if constexpr (!ff_backward(EPI)) {
      if (e.keep != FF_KEEP_NOTHING) {
#pragma unroll
        for (int s = 0; s < NB; ++s) {
          float v[32];
          tmem_ld32(s ? u_at : g_at, v);
          ff_add_bias<32>(e, s, head, col, v);
          if (e.keep == FF_KEEP_16)
            ff_store_tile(e, e.held[s], (long long)e.heads * e.N, e.N, head, v, row0, col, buf, lane);
          else
            ff_hold8(e, s, head, v, row0 + lane, col);
        }
      }
    }
    const bool has_aux = ff_has_aux<EPI>(e);
    if (has_aux)
      ff_put_aux(aux, buf, lane);
    else
      __syncwarp();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float g[16], u[16];
      ff_read16<NB>(g_at + 16 * h, g, u_at + 16 * h, u);
      if (h == 1) release();
      const int c = col + 16 * h;
      ff_add_bias<16>(e, 0, head, c, g);
      if constexpr (NB == 2) ff_add_bias<16>(e, 1, head, c, u);
      if constexpr (ff_backward(EPI)) {
        ff_with_act(e.act, [&](auto a) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float y[8];
            ff_unpack8(*reinterpret_cast<const uint4*>(buf + ff_piece(lane, 2 * h + q)), e.half, y);
            ff_backward_values<EPI, 8, decltype(a)::value>(e.up_relu, g + 8 * q, u + 8 * q, [&](int i) { return pair_of(y, i); });
          }
        });
      } else {
        ff_forward_values<EPI, 16>(e, g, u);
        if (EPI == FF_ACT && has_aux) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float a[8];
            ff_unpack8(*reinterpret_cast<const uint4*>(buf + ff_piece(lane, 2 * h + q)), e.half, a);
#pragma unroll
            for (int i = 0; i < 4; ++i) put_pair(g + 8 * q, i, add2(pair_of(g + 8 * q, i), pair_of(a, i)));
          }
        }
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        *reinterpret_cast<uint4*>(buf + ff_piece(lane, 2 * h + q)) = ff_pack8(g + 8 * q, e.half);
        if constexpr (EPI == FF_GATED_BWD)
          *reinterpret_cast<uint4*>(buf + 2048 + ff_piece(lane, 2 * h + q)) = ff_pack8(u + 8 * q, e.half);
      }
      if constexpr (ff_backward(EPI)) {
        if (e.colsum[0]) ff_put_sums<16>(e, 0, head, g, row0, c, lane);
        if constexpr (NB == 2)
          if (e.colsum[1]) ff_put_sums<16>(e, 1, head, u, row0, c, lane);
      }
    }
    ff_flush(e, e.out[0], e.ld, e.head, head, row0, col, buf, lane);
    if constexpr (EPI == FF_GATED_BWD) ff_flush(e, e.out[1], e.ld, e.head, head, row0, col, buf + 2048, lane);
  }
}

// ------------------------------------------------------------------------------- products


template <int EPI, int BN, bool PAIR>
struct FfCfg {
  static constexpr int NB = ff_products(EPI);
  static constexpr int CTAS = PAIR ? 2 : 1;
  static constexpr int B_ROWS = BN / CTAS;  // of one product, staged by this CTA
  static constexpr int A_BYTES = 128 * 64 * 2, B_BYTES = B_ROWS * 64 * 2;
  static constexpr int STAGE_BYTES = NB * (A_BYTES + B_BYTES);
  // Sixteen epilogue warps, four a scheduler: with eight the epilogue of 2 x 128 columns was bound by its own latencies
  // (gated, 4099 rows, 4 x 256 -> 8192: 240 us).
  static constexpr int EPI_WARPS = BN >= 128 ? 16 : 8;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int EPI_TILE = EPI == FF_GATED_BWD ? 4096 : 2048;  // of a warp: one result, or two
  static constexpr int EPI_BYTES = EPI_WARPS * EPI_TILE;
  static constexpr int STAGES = (224 * 1024 - EPI_BYTES) / STAGE_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + EPI_BYTES + 1024;
  static constexpr int TMEM_COLS = 2 * NB * BN;
  static_assert(B_ROWS % 64 == 0 && TMEM_COLS <= 512 && SMEM <= 227 * 1024, "tile");
};

// The tiles of a CTA (or pair): columns fastest, then rows, parts, heads, sets. Worker w of W takes w, w + W, ....
// Divided once; the digits of the step are the host's.
struct FfWalk {
  unsigned at[4], set, count;

  __device__ __forceinline__ FfWalk(const FfGemm& p, unsigned worker, unsigned workers) {
    const unsigned total = (unsigned)(p.tiles_m * p.tiles_n * p.splits * p.e.heads * p.out_sets);
    unsigned t = worker;
    count = worker < total ? (total - worker + workers - 1) / workers : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] = t % p.size[i];
      t /= p.size[i];
    }
    set = t;
  }
  __device__ __forceinline__ void next(const FfGemm& p) {
    unsigned carry = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      at[i] += p.step[i] + carry;
      carry = at[i] >= p.size[i] ? 1 : 0;
      at[i] -= carry ? p.size[i] : 0;
    }
    set += p.step[4] + carry;
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

// Without release semantics, which would wait for this thread's global stores: what the other side waits for are loads
// from TMEM, and those are done.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
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
__global__ void __launch_bounds__(FfCfg<EPI, BN, PAIR>::THREADS, 1)
    ff_gemm_kernel(const __grid_constant__ FfGemm p) {
  constexpr int NB = ff_products(EPI);
  using Cfg = FfCfg<EPI, BN, PAIR>;
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
      mbar_init(&tempty_bar[a], Cfg::CTAS * Cfg::EPI_WARPS);
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

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer (both CTAs of a pair)
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      const int a_count = NB == 2 && !p.two_a ? 1 : NB;
      const uint32_t bytes = (uint32_t)(Cfg::CTAS * (a_count * Cfg::A_BYTES + NB * Cfg::B_BYTES));
      FfWalk w(p, worker, workers);
      for (unsigned t = 0; t < w.count && ok; ++t, w.next(p)) {
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
      for (unsigned t = 0; t < w.count && ok; ++t, w.next(p)) {
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
    const int part = (warp - 2) >> 2;  // its share of the tile's columns
    uint8_t* buf = sEpi + (warp - 2) * Cfg::EPI_TILE;
    constexpr int COLS = BN * 4 / Cfg::EPI_WARPS;
    static_assert(COLS % 32 == 0, "a chunk is 32 columns");
    const int col0 = part * COLS;
    uint32_t leader_tempty0 = 0, leader_tempty1 = 0;
    if constexpr (PAIR) leader_tempty0 = map_to_cta(&tempty_bar[0], 0), leader_tempty1 = map_to_cta(&tempty_bar[1], 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    FfWalk w(p, worker, workers);
    for (unsigned t = 0; t < w.count; ++t, w.next(p)) {
      const int row0 = w.m() * ROWS + 128 * crank + quad * 32, first = w.n() * BN + col0;
      const bool one = p.splits == 1;
      FfAux aux;  // of the first chunk: on its way while the products are
      if (one && ff_has_aux<EPI>(p.e)) ff_load_aux(aux, p.e, w.head(), row0, first, lane);
      // the same answer for the whole warp: the loads from TMEM need all of its lanes, also where a wait has run out
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], acc_phase, &abort_flag, p.err, kErrTimeoutEpilogue)))
        break;
      tc_fence_after();
      // The accumulators go back as soon as this warp has its values in registers.
      bool held = true;
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (leader)
            mbar_arrive(&tempty_bar[acc]);
          else
            mbar_arrive_cluster_relaxed(acc ? leader_tempty1 : leader_tempty0);
        }
        held = false;
      };
      const int cols = row0 < p.e.M ? min(COLS, p.e.N - first) : 0;
#pragma unroll 1
      for (int cc = 0; cc < cols; cc += 32) {
        const int col = first + cc;
        const bool last = cc + 32 >= cols;
        const uint32_t at = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * NB * BN + col0 + cc;
        if (cc > 0 && one && ff_has_aux<EPI>(p.e)) ff_load_aux(aux, p.e, w.head(), row0, col, lane);
        auto give_back = [&] {
          if (last) release();
        };
        if (one) {
          ff_epilogue<EPI>(p.e, (int)w.set, w.head(), row0, col, at, at + BN, aux, buf, lane, give_back);
          continue;
        }
        float g[32], u[32];
        tmem_ld32(at, g);
        if constexpr (NB == 2) tmem_ld32(at + BN, u);
        give_back();
        if (row0 + lane < p.e.M) {
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
      if (held) release();
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

// ------------------------------------------------------------------------------- few rows

// Up to MP rows: the weights take the place of A (128 columns of the output are the tensor core's rows) and the batch's
// rows that of B, so that what is staged is the weights and little else: bound by their bytes. (With the rows as A a stage
// held 16 KB of mostly padding for each operand: 64 rows, 4 x 256 -> 8192, 18 us; 5.2 at the copy rate.) A lane then holds a column
// of the output and its rows lie in its registers.
template <int NB, int MP>
struct FfFewCfg {
  static constexpr int W_BYTES = 128 * 64 * 2, X_BYTES = MP * 64 * 2;
  static constexpr int STAGE_BYTES = NB * (W_BYTES + X_BYTES);
  static constexpr int STAGES = (200 * 1024) / STAGE_BYTES;
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024;
  static constexpr int ROWS = MP < 32 ? MP : 32;  // of a chunk
  static constexpr int EPI_WARPS = MP > 32 ? 8 : 4;
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int TMEM_COLS = 2 * NB * MP < 32 ? 32 : 2 * NB * MP;
  static_assert(MP % 16 == 0 && X_BYTES % 1024 == 0 && TMEM_COLS <= 512 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "tile");
};

__device__ __forceinline__ float ff_as_float(uint16_t v, int half) {
  return half ? __half2float(*reinterpret_cast<const __half*>(&v)) : __uint_as_float((uint32_t)v << 16);
}
__device__ __forceinline__ uint16_t ff_as_16(float v, int half) {
  if (half) {
    const __half h = __float2half_rn(v);
    return *reinterpret_cast<const uint16_t*>(&h);
  }
  const __nv_bfloat16 h = __float2bfloat16_rn(v);
  return *reinterpret_cast<const uint16_t*>(&h);
}

template <int n>
__device__ __forceinline__ void ff_read_rows(uint32_t at, float* v) {
  if constexpr (n == 32) {
    float r[32];
    tmem_ld32(at, r);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = r[i];
  } else {
    uint32_t r[16];
    tmem_ld16(at, r);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
  }
}

// The lane's column `col` of n rows from row0 on. All lanes of the warp call it; in: the column is one of the output's.
template <int EPI, int n>
__device__ __forceinline__ void ff_few_epilogue(const FfOut& e, int head, int row0, int col, bool in, float* g, float* u, int lane) {
  constexpr int NB = ff_products(EPI);
  const int rows = min(n, e.M - row0);
  const long long hn = (long long)head * e.N + col;
  uint16_t* out[2] = {reinterpret_cast<uint16_t*>(e.out[0]) + row0 * e.ld + (long long)head * e.head + col,
                      reinterpret_cast<uint16_t*>(e.out[1]) + row0 * e.ld + (long long)head * e.head + col};
  if constexpr (EPI != FF_STORE) {
#pragma unroll
    for (int s = 0; s < NB; ++s) {
      if (!ff_has_bias(e, s) || !in) continue;
      const float b = !e.bias[s]     ? e.bias0[s]
                      : e.bias_f32   ? reinterpret_cast<const float*>(e.bias[s])[hn]
                                     : ff_as_float(reinterpret_cast<const uint16_t*>(e.bias[s])[hn], e.half);
#pragma unroll
      for (int i = 0; i < n; ++i) (s ? u : g)[i] += b;
    }
    if (!ff_backward(EPI) && e.keep != FF_KEEP_NOTHING) {
      const int nb = (e.N + 31) / 32;
#pragma unroll
      for (int s = 0; s < NB; ++s) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
          if (i >= rows) break;
          const float v = (s ? u : g)[i];
          const long long rh = (long long)(row0 + i) * e.heads + head;
          if (e.keep == FF_KEEP_16) {
            if (in) reinterpret_cast<uint16_t*>(e.held[s])[rh * e.N + col] = ff_as_16(v, e.half);
          } else {  // the warp's 32 columns are a block
            const uint32_t size = in ? __float_as_uint(act8_size(v)) : 0u;
            const int ex = act8_exponent(__uint_as_float(__reduce_max_sync(0xffffffffu, size)));
            if (in) reinterpret_cast<uint8_t*>(e.held[s])[rh * e.N + col] = (uint8_t)act8_code2(v, 0.f, act8_power(-ex));
            if (lane == 0) e.exponents[s][rh * nb + col / 32] = (uint8_t)(ex + 127);
          }
        }
      }
    }
    float a[n];
    const bool has_aux = ff_has_aux<EPI>(e);
    if (has_aux) {
      const uint16_t* src = reinterpret_cast<const uint16_t*>(e.aux) + row0 * e.aux_ld + (long long)head * e.aux_head + col;
#pragma unroll
      for (int i = 0; i < n; ++i) a[i] = in && i < rows ? ff_as_float(src[i * e.aux_ld], e.half) : 0.f;
    }
    if constexpr (ff_backward(EPI)) {
      ff_with_act(e.act, [&](auto k) {
        ff_backward_values<EPI, n, decltype(k)::value>(e.up_relu, g, u, [&](int i) { return pair_of(a, i); });
      });
#pragma unroll
      for (int s = 0; s < NB; ++s) {
        if (!e.colsum[s] || !in) continue;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < n; ++i)
          if (i < rows) sum += (s ? u : g)[i];
        e.colsum[s][(long long)(row0 / 32) * e.heads * e.N + hn] = sum;
      }
    } else {
      ff_forward_values<EPI, n>(e, g, u);
      if (EPI == FF_ACT && has_aux) {
#pragma unroll
        for (int i = 0; i < n; ++i) g[i] += a[i];
      }
    }
  }
  if (!in) return;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (i >= rows) break;
    out[0][i * e.ld] = ff_as_16(g[i], e.half);
    if constexpr (EPI == FF_GATED_BWD) out[1][i * e.ld] = ff_as_16(u[i], e.half);
  }
}

// ta, a_mn, a_heads: of the weights; tb, b_heads: of the rows; two_a: the second product has rows of its own. tiles_m
// counts 128 columns of the output.
template <int EPI, int MP>
__global__ void __launch_bounds__(FfFewCfg<ff_products(EPI), MP>::THREADS, 1) ff_few_kernel(const __grid_constant__ FfGemm p) {
  constexpr int NB = ff_products(EPI);
  using Cfg = FfFewCfg<NB, MP>;
  constexpr int STAGES = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_bar[STAGES], empty_bar[STAGES];
  __shared__ uint64_t tfull_bar[2], tempty_bar[2], drain_bar;
  __shared__ uint32_t tmem_base_s;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], Cfg::EPI_WARPS);
    }
    mbar_init(&drain_bar, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&tmem_base_s, Cfg::TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the sum of the parts may get ready
  const uint32_t tmem_base = tmem_base_s;

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------------------------ TMA producer
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      const int x_count = NB == 2 && !p.two_a ? 1 : NB;
      const uint32_t bytes = (uint32_t)(NB * Cfg::W_BYTES + x_count * Cfg::X_BYTES);
      FfWalk w(p, blockIdx.x, gridDim.x);
      for (unsigned t = 0; t < w.count && ok; ++t, w.next(p)) {
        int b0, b1;
        ff_part(p, w.split(), b0, b1);
        int seg = b0 / p.KB, kb = b0 - seg * p.KB;
        for (int i = b0; i < b1; ++i) {
          const int set = seg / p.sum_heads;
          const int head = p.sum_heads > 1 ? seg - set * p.sum_heads : w.head();
          if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1, &abort_flag, p.err, kErrTimeoutProducer)) {
            ok = false;
            break;
          }
          uint64_t* bar = &full_bar[stage];
          mbar_arrive_expect_tx(bar, bytes);
          uint8_t* dst = smem + stage * Cfg::STAGE_BYTES;
          const int k = kb * 64;
#pragma unroll
          for (int s = 0; s < NB; ++s) {
            const int q = NB == 1 ? set : s;
            ff_load<false, 128>(dst + s * Cfg::W_BYTES, &p.ta[q], NB == 1 ? p.a_mn != 0 : (p.a_mn >> s & 1) != 0, bar,
                                w.m() * 128, k, (p.a_heads >> q) & 1 ? head : 0);
            if (s < x_count)
              ff_tma<false>(dst + NB * Cfg::W_BYTES + s * Cfg::X_BYTES, &p.tb[q], bar, k, 0, (p.b_heads >> q) & 1 ? head : 0);
          }
          if (++kb == p.KB) kb = 0, ++seg;
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
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      FfWalk w(p, blockIdx.x, gridDim.x);
      for (unsigned t = 0; t < w.count && ok; ++t, w.next(p)) {
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
            const bool mn = NB == 1 ? p.a_mn != 0 : (p.a_mn >> s & 1) != 0;
            const uint32_t a_base = base + s * Cfg::W_BYTES;
            const uint32_t b_base = base + NB * Cfg::W_BYTES + (s == 1 && p.two_a ? Cfg::X_BYTES : 0);
            const uint32_t idesc = p.idesc | (mn ? 1u << 15 : 0u);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma_bf16(tmem_base + (acc * NB + s) * MP, make_sdesc_sw128(a_base + kk * (mn ? 2048 : 32), mn ? 8192 : 16, 1024),
                        make_sdesc_sw128(b_base + kk * 32, 16, 1024), idesc, (i > b0 || kk > 0) ? 1u : 0u);
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
  } else {
    // ------------------------------------------------ epilogue
    const int quad = warp & 3, part = (warp - 2) >> 2;
    constexpr int SHARE = MP * 4 / Cfg::EPI_WARPS, n = Cfg::ROWS;
    int acc = 0;
    uint32_t acc_phase = 0;
    FfWalk w(p, blockIdx.x, gridDim.x);
    for (unsigned t = 0; t < w.count; ++t, w.next(p)) {
      // the same answer for the whole warp: the loads from TMEM need all of its lanes, also where a wait has run out
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(&tfull_bar[acc], acc_phase, &abort_flag, p.err, kErrTimeoutEpilogue)))
        break;
      tc_fence_after();
      const int col = w.m() * 128 + quad * 32 + lane;
      const bool in = col < p.e.N;
#pragma unroll 1
      for (int r = part * SHARE; r < (part + 1) * SHARE && r < p.e.M && w.m() * 128 + quad * 32 < p.e.N; r += n) {
        float v[NB][n];
#pragma unroll
        for (int s = 0; s < NB; ++s) ff_read_rows<n>(tmem_base + ((uint32_t)(quad * 32) << 16) + (acc * NB + s) * MP + r, v[s]);
        if (p.splits == 1) {
          ff_few_epilogue<EPI, n>(p.e, w.head(), r, col, in, v[0], v[NB - 1], lane);
        } else if (in) {
#pragma unroll
          for (int s = 0; s < NB; ++s) {
            float* o = p.partial + ((((long long)w.split() * NB + s) * p.e.heads + w.head()) * p.e.M + r) * p.e.N + col;
#pragma unroll
            for (int i = 0; i < n; ++i)
              if (r + i < p.e.M) o[(long long)i * p.e.N] = v[s][i];
          }
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
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
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
inline int64_t ff_workers(int64_t tiles, FfTile t, int sms) { return std::min<int64_t>(tiles, sms / (t.pair ? 2 : 1)); }
void ff_launch_few(int epi, int rows, const FfGemm& p, cudaStream_t st, int dev);       // either, up to 128 rows
void ff_launch_one(int epi, FfTile tile, const FfGemm& p, cudaStream_t st, int dev);    // one product
void ff_launch_gated(int epi, FfTile tile, const FfGemm& p, cudaStream_t st, int dev);  // two
}  // namespace bd
