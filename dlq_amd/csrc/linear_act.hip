// linear_act.hip -- dlq_linear_act_s8 / _f8 and dlq_linear_grouped_s8 / _f8:
//   y[m][n] = act(fma(float(acc), xs[m] * ws[n], bias[n])) + res[m][n],
//   acc = sum_k x[m][k] * w[n][k]
// on int8 or e4m3 codes, rows and weights both K-contiguous; grouped: rows
// sorted by expert, w / ws / bias of the row's expert.
//
// The MFMA's A operand is the weights (its rows are output columns n), its B
// operand the rows of x: a lane's four accumulators are then four consecutive
// n of one row m, so scale, bias and residual come in and y goes out in
// 4-element vectors.
#include <climits>

#include "rowops_common.h"

namespace dlq {
namespace {

struct LinearArgs {
  const int8_t* x;
  const int8_t* w;
  const float* xs;    // [M] or nullptr
  const float* ws;    // [E][N]
  const float* bias;  // [E][N] or nullptr
  const void* res;    // [M][ldr] or nullptr
  void* y;
  int M, N, K;
  size_t ldx, ldw, ldy, ldr;
  int odd;             // some row of x or w does not start on a dword
  int act, bf16, vec;  // vec: y, res, ws and bias take aligned 4-element accesses
  int cut;             // e4m3: the fp8 matrix instructions may be taken
  int E;               // 0: one product over all rows
  const int* off;      // [E + 1], E > 0
};

// The activations on the hardware's exp2 and reciprocal (1 ulp each).
//  * GELU = v Phi(v), both parts least-maximum fits of their function, made for
//    this kernel: below 1.25 v (1/2 + v R(v^2)), R(v^2) = erf(v / sqrt 2) / 2v
//    to 1e-9; above, max(v, 0) - |v| 2^Q(|v|), 2^Q = erfc(|v| / sqrt 2) / 2 to
//    a third of 2^-24 of |v| and 1e-3 of itself (0 below 2^-126).  Off by at most
//    1.7 * 2^-24 |v| over [-15, 15] in all (v/2 (1 + erf) in fp32: 1.8), and
//    right to 1e-3 where it is next to nothing.
//  * GELU_TANH: 1 + tanh(u) = 2 / (1 + e^-2u).
template <int ACT>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == DLQ_ACT_RELU) return v < 0.f ? 0.f : v;  // a NaN stays
  if constexpr (ACT == DLQ_ACT_GELU) {
    const float a = __builtin_fminf(__builtin_fabsf(v), 14.2f);  // 2^Q(14.2) |v| is below 2^-145
    float q = 3.35875221e-08f;
    q = __builtin_fmaf(q, a, -2.08408983e-06f);
    q = __builtin_fmaf(q, a, 5.51391022e-05f);
    q = __builtin_fmaf(q, a, -0.000824186835f);
    q = __builtin_fmaf(q, a, 0.00785342138f);
    q = __builtin_fmaf(q, a, -0.0518820174f);
    q = __builtin_fmaf(q, a, -0.462068886f);
    q = __builtin_fmaf(q, a, -1.14802313f);
    q = __builtin_fmaf(q, a, -1.00115383f);
    const float far = __builtin_fmaf(-a, __builtin_amdgcn_exp2f(q), v < 0.f ? 0.f : v);  // a NaN stays
    const float w = v * v;
    float r = -6.64485924e-06f;
    r = __builtin_fmaf(r, w, 0.000110327455f);
    r = __builtin_fmaf(r, w, -0.00118270959f);
    r = __builtin_fmaf(r, w, 0.00997150037f);
    r = __builtin_fmaf(r, w, -0.0664899871f);
    r = __builtin_fmaf(r, w, 0.398942262f);
    return __builtin_fabsf(v) < 1.25f ? v * __builtin_fmaf(v, r, 0.5f) : far;
  }
  if constexpr (ACT == DLQ_ACT_GELU_TANH) {
    const float u = v * __builtin_fmaf(0.044715f * v, v, 1.f) * (1.5957691216057308f * 1.4426950408889634f);
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-u));
  }
  if constexpr (ACT == DLQ_ACT_SILU)
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(v * -1.4426950408889634f));
  return v;
}

// f(constant of the activation): one branch around a loop, not one per value
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case DLQ_ACT_RELU: f(std::integral_constant<int, DLQ_ACT_RELU>{}); break;
    case DLQ_ACT_GELU: f(std::integral_constant<int, DLQ_ACT_GELU>{}); break;
    case DLQ_ACT_GELU_TANH: f(std::integral_constant<int, DLQ_ACT_GELU_TANH>{}); break;
    case DLQ_ACT_SILU: f(std::integral_constant<int, DLQ_ACT_SILU>{}); break;
    default: f(std::integral_constant<int, DLQ_ACT_NONE>{}); break;
  }
}

// The residual's / the output's columns n..n+3 of row m, all of them below N
// and aligned (a.vec).
__device__ __forceinline__ v4i residual_raw(const LinearArgs& a, int m, int n) {
  const size_t at = (size_t)m * a.ldr + n;
  if (!a.bf16) return *(const v4i*)((const float*)a.res + at);
  const v2u r = *(const v2u*)((const uint16_t*)a.res + at);
  return v4i{(int)r[0], (int)r[1], 0, 0};
}
__device__ __forceinline__ v4f residual_value(const LinearArgs& a, v4i r) {
  if (!a.bf16) return v4f{__int_as_float(r[0]), __int_as_float(r[1]), __int_as_float(r[2]), __int_as_float(r[3])};
  return v4f{bf_lo((unsigned)r[0]), bf_hi((unsigned)r[0]), bf_lo((unsigned)r[1]), bf_hi((unsigned)r[1])};
}
__device__ __forceinline__ void put4(const LinearArgs& a, int m, int n, v4f v) {
  const size_t at = (size_t)m * a.ldy + n;
  if (a.bf16)
    *(v2u*)((uint16_t*)a.y + at) = v2u{bf_pack(v[0], v[1]), bf_pack(v[2], v[3])};
  else
    *(v4f*)((float*)a.y + at) = v;
}
// The same, residual and output, one column at a time and those past N left out.
__device__ __forceinline__ void put4_any(const LinearArgs& a, int m, int n, v4f v) {
  const size_t ym = (size_t)m * a.ldy + n, rm = (size_t)m * a.ldr + n;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) break;
    if (a.bf16) {
      if (a.res) v[i] += __uint_as_float((unsigned)((const uint16_t*)a.res)[rm + i] << 16);
      ((uint16_t*)a.y)[ym + i] = (uint16_t)bf_pack(v[i], 0.f);
    } else {
      if (a.res) v[i] += ((const float*)a.res)[rm + i];
      ((float*)a.y)[ym + i] = v[i];
    }
  }
}
// act(fma(acc, sx ws, b)) of four columns
template <int ACT>
__device__ __forceinline__ v4f scaled4(v4f acc, float sx, v4f ws, v4f b) {
  v4f v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = act_of<ACT>(__builtin_fmaf(acc[i], sx * ws[i], b[i]));
  return v;
}

// p[n..n+3] of N values; those past N (and all of a null p) are 0.
__device__ __forceinline__ v4f column4(const float* p, int n, int N, int vec) {
  v4f v = {0.f, 0.f, 0.f, 0.f};
  if (!p) return v;
  if (vec) return *(const v4f*)(p + n);  // N % 4 == 0
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n + i < N) v[i] = p[n + i];
  return v;
}

// The t-th tile of BM rows over all experts: its expert e and rows [m0, m1);
// false if there are fewer.  Every wave of the grid walks the E + 1 offsets,
// 64 experts at a time: a prefix sum of their tile counts over the lanes.
template <int BM>
__device__ __forceinline__ bool expert_tile(const LinearArgs& a, int t, int& e, int& m0, int& m1) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.E; base += 64) {
    const int i = base + lane;
    int lo = 0, hi = 0;
    if (i < a.E) {
      lo = a.off[i];
      hi = a.off[i + 1];
      lo = lo < 0 ? 0 : lo > a.M ? a.M : lo;
      hi = hi < lo ? lo : hi > a.M ? a.M : hi;
    }
    const int mine = (hi - lo + BM - 1) / BM;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(sum, o);
      if (lane >= o) sum += v;
    }
    const unsigned long long past = __ballot(sum > t);
    if (past) {
      const int l = __ffsll(past) - 1;
      const int k = t - (__shfl(sum, l) - __shfl(mine, l));  // tile within the expert
      e = base + l;
      m0 = __shfl(lo, l) + k * BM;
      m1 = __shfl(hi, l);
      m1 = m1 < m0 + BM ? m1 : m0 + BM;
      return true;
    }
    t -= __shfl(sum, 63);
  }
  return false;
}

// One 16 x 16 product over 64 of K; a lane's operand is 16 codes.
//
// e4m3: the fp8 forms of the matrix pipe bring the products of 8 consecutive K
// to the largest one's exponent and cut them 13 bits below it (measured: a
// product of 2^2 beside one of 2^16 is lost, 1.5 * 2^3 keeps 2^3), which is
// coarser than a 32-bit sum: 1.4e-5 of a result on normal data, all of it where
// a row's large products cancel.  The codes are bf16 values as well, so they
// are widened (one conversion per two codes) and multiplied as bf16, whose
// products are exact and sums fp32.  Here that is twice the matrix
// instructions in a kernel that waits for memory; for the tiles see below.
template <bool F8>
struct Mma {
  typedef v4i frag;
  typedef v4i acc_t;
  static __device__ __forceinline__ frag prep(v4i v) { return v; }
  static __device__ __forceinline__ acc_t go(frag a, frag b, acc_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<true> {
  struct frag {
    v8bf h[2];
  };
  typedef v4f acc_t;
  static __device__ __forceinline__ frag prep(v4i v) {
    frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[i], 1.f, false);
      const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[i], 1.f, true);
      const int o = 4 * (i & 1);
      f.h[i >> 1][o] = a[0];
      f.h[i >> 1][o + 1] = a[1];
      f.h[i >> 1][o + 2] = b[0];
      f.h[i >> 1][o + 3] = b[1];
    }
    return f;
  }
  static __device__ __forceinline__ acc_t go(frag a, frag b, acc_t c) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h[0], b.h[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.h[1], b.h[1], c, 0, 0, 0);
  }
};

// Fragments straight from memory: 16 MI rows of x by 16 NJ rows of w per
// workgroup, its WK waves each take a slice of K and join their sums in LDS
// (in wave order).  Lane l holds row l & 15, 16 bytes at 16 (l >> 4) of every
// 64: the order of K within a step is free as long as both operands agree.
//
// Bound by the weights' bytes, which a few rows read once, and below some
// 20 MB by the latency of the loads: so each wave has 2 U of them in flight
// (U steps ahead), what is left of a slice is loaded at once (8 x 1000 x 2000
// 3.4 us; step by step 4.5), so are the epilogue's operands, behind the first
// loads, and K is split over the waves of a workgroup, four of them (eight
// gained nothing from 1 x 1024 x 4096 to 16 x 4096 x 16384).  int8, bf16
// out: 1 x 4096 x 4096 5.8 us (16.8 MB), 64 rows over 64 experts of
// 1536 x 2048 24 us (about 40 of them have rows: 126 MB, 5.2 TB/s).
template <bool F8, bool ODD, int MI, int NJ, int WK, int U>
__global__ __launch_bounds__(WK * 64) void linear_direct_kernel(const LinearArgs a, int nbm) {
  typedef Mma<F8> MM;
  typedef typename MM::acc_t acc_t;
  constexpr int BM = 16 * MI, BN = 16 * NJ, KB = 64;
  __shared__ acc_t part[WK][MI * NJ][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  // each XCD takes a run of tiles, row tiles fastest: those that share weights
  // run side by side on one L2
  const int l = xcd_remap(blockIdx.x, gridDim.x);
  const int n0 = l / nbm * BN, mt = l % nbm;
  int e = 0, m0 = mt * BM, m1 = a.M;
  if (a.E && !expert_tile<BM>(a, mt, e, m0, m1)) return;

  const int8_t *xp[MI], *wp[NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + 16 * i + lr;  // rows past the end repeat the last one; they are not stored
    xp[i] = a.x + (size_t)(m < m1 ? m : m1 - 1) * a.ldx + 16 * lg;
  }
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int n = n0 + 16 * j + lr;
    wp[j] = a.w + ((size_t)e * a.N + (n < a.N ? n : a.N - 1)) * a.ldw + 16 * lg;
  }
  acc_t acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = acc_t{0, 0, 0, 0};

  const int steps = (a.K + KB - 1) / KB, full = a.K / KB;
  const int s0 = (int)((long)steps * wave / WK), s1 = (int)((long)steps * (wave + 1) / WK);
  // U steps' loads are on their way while U others are multiplied
  Raw16<ODD> rx[2][U][MI], rw[2][U][NJ];
  auto load_step = [&](int b, int u, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) rw[b][u][j].load(wp[j] + (size_t)s * KB);
#pragma unroll
    for (int i = 0; i < MI; ++i) rx[b][u][i].load(xp[i] + (size_t)s * KB);
  };
  auto load = [&](int b, int s) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_step(b, u, s + u);
  };
  auto product = [&](const v4i* vx, const v4i* vw) __attribute__((always_inline)) {
    typename MM::frag fx[MI], fw[NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) fx[i] = MM::prep(vx[i]);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fw[j] = MM::prep(vw[j]);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = MM::go(fw[j], fx[i], acc[i][j]);
  };
  auto multiply_step = [&](int b, int u) __attribute__((always_inline)) {
    v4i vx[MI], vw[NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) vx[i] = rx[b][u][i].get(xp[i]);  // a step is a multiple of a dword
#pragma unroll
    for (int j = 0; j < NJ; ++j) vw[j] = rw[b][u][j].get(wp[j]);
    product(vx, vw);
  };
  auto multiply = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) multiply_step(b, u);
  };
  // the epilogue's operands of one 16 x 16, on their way behind the first loads
  // where a wave has no more than one
  struct Ends {
    float sx;
    v4f ws, bias;
    v4i res;
  };
  const auto ends = [&](int t) __attribute__((always_inline)) {
    Ends o = {1.f, {0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}, {0, 0, 0, 0}};
    const int m = m0 + 16 * (t / NJ) + lr, n = n0 + 16 * (t % NJ) + 4 * lg;
    if (m < m1 && n < a.N) {
      if (a.xs) o.sx = a.xs[m];
      o.ws = column4(a.ws + (size_t)e * a.N, n, a.N, a.vec);
      o.bias = column4(a.bias ? a.bias + (size_t)e * a.N : nullptr, n, a.N, a.vec);
      if (a.vec && a.res) o.res = residual_raw(a, m, n);
    }
    return o;
  };
  constexpr bool AHEAD = MI * NJ <= WK;
  Ends ahead;
  const int sf = s1 < full ? s1 : full;
  int s = s0;
  if (s + U <= sf) load(0, s);
  if (AHEAD && wave < MI * NJ) ahead = ends(wave);
  for (; s + 3 * U <= sf; s += 2 * U) {
    load(1, s + U);
    multiply(0);
    load(0, s + 2 * U);
    multiply(1);
  }
  if (s + 2 * U <= sf) {
    load(1, s + U);
    multiply(0);
    multiply(1);
    s += 2 * U;
  } else if (s + U <= sf) {
    multiply(0);
    s += U;
  }
  // what is left: fewer than U whole steps, and the end of K with zeros past it
#pragma unroll
  for (int u = 0; u + 1 < U; ++u)
    if (s + u < sf) load_step(0, u, s + u);
  v4i ex[MI], ew[NJ];
  if (s1 > full) {
    const int k = full * KB + 16 * lg, avail = a.K - k;
#pragma unroll
    for (int i = 0; i < MI; ++i) ex[i] = load_tail16<ODD>(xp[i] + full * KB, avail, k);
#pragma unroll
    for (int j = 0; j < NJ; ++j) ew[j] = load_tail16<ODD>(wp[j] + full * KB, avail, k);
  }
#pragma unroll
  for (int u = 0; u + 1 < U; ++u)
    if (s + u < sf) multiply_step(0, u);
  if (s1 > full) product(ex, ew);
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) part[wave][i * NJ + j][lane] = acc[i][j];
  __syncthreads();
  for (int t = wave; t < MI * NJ; t += WK) {
    acc_t s = part[0][t][lane];
#pragma unroll
    for (int k = 1; k < WK; ++k) s += part[k][t][lane];
    const int m = m0 + 16 * (t / NJ) + lr, n = n0 + 16 * (t % NJ) + 4 * lg;
    if (!AHEAD) ahead = ends(t);
    if (m < m1 && n < a.N) {
      v4f v;
      with_act(a.act, [&](auto act) {
        v = scaled4<decltype(act)::value>(v4f{(float)s[0], (float)s[1], (float)s[2], (float)s[3]}, ahead.sx, ahead.ws,
                                          ahead.bias);
      });
      if (!a.vec)
        put4_any(a, m, n, v);
      else
        put4(a, m, n, a.res ? v + residual_value(a, ahead.res) : v);
    }
  }
}

// ---- large products: tiles through LDS ------------------------------------
// TN columns (rows of w) by TM rows of x per workgroup of WN x WM waves, each
// wave NI x MJ tiles of 32 x 32; RES: with a residual that vec allows.  Both operands stream by LDS-DMA, 128 bytes
// of K per stage into SLOTS slots; row r of a slot is 128 bytes, its 16-byte
// chunk c at 16 (c ^ ((r >> 1) & 7)), so the 16 rows a ds_read_b128 lane group
// reads fall on 16 distinct bank quads (the DMA lanes fetch in that order;
// conflicts: 0.1 % of the LDS cycles).
//
// The pipeline of a wave: while the matrix instructions of one K step run, the
// fragments of the next are read.  Before the last step of a stage one barrier
// says both that the next stage has landed everywhere and that nobody reads
// this stage's slot any more; behind it the next stage's first fragments are
// read and the DMA of the stage SLOTS further on is issued, one piece behind
// each matrix instruction.  So with two slots a stage has all but one of a
// stage's steps to land, and no matrix instruction waits for a fragment read
// issued right before it.
//
// Waves own 128 x 128 outputs where there are enough rows and columns: an LDS
// byte then feeds 64 multiply-adds, and reads and DMA writes take 192 KB of
// the 256 KB that LDS moves in a stage's 2048 matrix cycles (with 128 x 64
// per wave: 256 KB, the bound).  8192^3, bf16 out, calls back to back: int8 466
// us, 2.36 POPS, with GELU 490 to 530 by the card, the clock at 1.7 GHz by the
// power limit and the matrix unit busy 53 to 57 % of the cycles.  Waves of
// 64 x 64 (128 x 128 tiles) read LDS for as long as they multiply: 576 us.  The
// small tiles are bound by what a stage takes from DMA to barrier, so they have
// more slots and up to 128 bytes of K per fragment step.
//
// e4m3 is widened to bf16 here as well (see Mma), behind the LDS read and while
// matrix instructions run that do not need the fragment: twice the matrix
// cycles per code, so 8192^3 takes 760 to 780 us by the card, 1.4 PFLOP/s, what
// a bf16 product of this size reaches.  kF8Cut (the caller's DLQ_FP8_SUMS) takes
// the fp8 instructions, 420 to 440 us, and their cut products.
enum { kS8, kF8, kF8Cut };
template <int T, int NV>
struct TileMma {  // a fragment: NV 16-byte reads, 32 K bytes of a row each
  typedef v16i acc_t;
  typedef v4i sum4;
  static __device__ __forceinline__ v16i go(const v4i* a, const v4i* b, v16i c) {
#pragma unroll
    for (int v = 0; v < NV; ++v) c = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[v], b[v], c, 0, 0, 0);
    return c;
  }
};
template <int NV>
struct TileMma<kF8, NV> {
  typedef v16f acc_t;
  typedef v4f sum4;
  typedef Mma<true>::frag wide;  // 16 codes as bf16
  static __device__ __forceinline__ v16f go(const wide& a, const wide& b, v16f c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h[0], b.h[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h[1], b.h[1], c, 0, 0, 0);
  }
};
template <int NV>
struct TileMma<kF8Cut, NV> {
  static_assert(NV % 2 == 0, "64 K bytes per instruction");
  typedef v16f acc_t;
  typedef v4f sum4;
  static __device__ __forceinline__ v16f go(const v4i* a, const v4i* b, v16f c) {
#pragma unroll
    for (int v = 0; v < NV; v += 2)
      c = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(cat8(a[v], a[v + 1]), cat8(b[v], b[v + 1]), c, 0, 0, 0, 0, 0,
                                                          0);
    return c;
  }
};

__device__ __attribute__((aligned(64))) int8_t g_zero_linear[64];

// a pointer that is the same in every lane, told to the compiler
__device__ __forceinline__ const int8_t* uniform(const int8_t* p) {
  const unsigned long long v = (unsigned long long)p;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)v), hi = __builtin_amdgcn_readfirstlane((unsigned)(v >> 32));
  return (const int8_t*)((unsigned long long)hi << 32 | lo);
}

template <int WN, int WM, int NI, int MJ, int KB, int SLOTS, bool RES>
struct TileLds {
  static constexpr int NW = WN * WM, SLOT = 32 * (WN * NI + WM * MJ) * KB;
  static constexpr int PITCH = NI * 32 * 4 + 16;  // epilogue staging: 32 rows of a wave's columns
  // lanes per row, rows per instruction, instructions per 32 rows, in flight of the epilogue
  static constexpr int LPR = NI * 8, RPI = 64 / LPR, NP = 32 / RPI, U = 4;
  static_assert(NP % U == 0, "rows of a staging pass");
  static constexpr int EPILOGUE = NW * (32 * PITCH + (RES ? NP * 1024 : 0));  // staging, residual
  static constexpr int BYTES = SLOTS * SLOT > EPILOGUE ? SLOTS * SLOT : EPILOGUE;
};

// Columns from n0 on of rows [m0, m1) of expert e.
template <int T, bool REG, int WN, int WM, int NI, int MJ, int NV, int KB, int SLOTS, bool RES>
__device__ __forceinline__ void linear_tile(const LinearArgs& a, int e, int m0, int m1, int n0, int8_t* lds) {
  typedef TileMma<T, NV> MM;
  typedef typename MM::acc_t acc_t;
  typedef typename MM::sum4 sum4;
  constexpr int NW = WN * WM, TN = 32 * WN * NI, TM = 32 * WM * MJ;
  constexpr int SPS = KB / 32 / NV;                        // K steps of a stage
  constexpr int CPR = KB / 16, RPP = 64 / CPR;             // chunks of a row, rows of a 1 KiB piece
  constexpr int SLOT = (TN + TM) * KB;
  constexpr int PW = TN / RPP / NW, PX = TM / RPP / NW, PP = PW + PX;  // pieces of a stage per wave
  constexpr int NM = NI * MJ, NR = (NI + MJ) * NV;
  static_assert(KB == 128 || KB == 64, "chunk swizzle");
  static_assert(NW % 2 == 0 && TN % (RPP * NW) == 0 && TM % (RPP * NW) == 0, "pieces per wave");
  static_assert(PP * (SLOTS - 1) <= 63, "counted waits");
  typedef TileLds<WN, WM, NI, MJ, KB, SLOTS, RES> L;
  constexpr int PITCH = L::PITCH, LPR = L::LPR, RPI = L::RPI, NP = L::NP, U = L::U;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, lh = lane >> 5, wn = wave % WN, wm = wave / WN;
  const int8_t* wbase = uniform(a.w + ((size_t)e * a.N + n0) * a.ldw);
  const int8_t* xbase = uniform(a.x + (size_t)m0 * a.ldx);

  // piece r of this wave: rows RPP (wave + NW r) ..; rows past the end repeat
  // the last one (they are not stored).  The swizzle is the same for all r.
  const auto swizzle = [](int row) { return KB == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  const int prow = RPP * wave + lane / CPR, chunk = (lane % CPR) ^ swizzle(prow);
  unsigned vw[PW], vx[PX];
#pragma unroll
  for (int r = 0; r < PW; ++r) {
    const int n = prow + RPP * NW * r, last = a.N - 1 - n0;
    vw[r] = (unsigned)(n < last ? n : last) * (unsigned)a.ldw + 16 * chunk;
  }
#pragma unroll
  for (int r = 0; r < PX; ++r) {
    const int m = prow + RPP * NW * r, last = m1 - 1 - m0;
    vx[r] = (unsigned)(m < last ? m : last) * (unsigned)a.ldx + 16 * chunk;
  }
  const unsigned lds32 = lds_addr32(lds);
  const int nst = (a.K + KB - 1) / KB, full = a.K / KB;
  const int8_t* zsrc = g_zero_linear;
  asm volatile("" : "+s"(zsrc));
  const auto slot_at = [&](int slot, int r) __attribute__((always_inline)) {
    return slot * SLOT + (r < PW ? 0 : TN * KB) + (wave + NW * (r < PW ? r : r - PW)) * 1024;
  };
  // piece r of stage st into a slot; whole: all of the stage lies within K.
  // REG (rows that are not 16-byte aligned, which the DMA cannot take): the
  // stage goes from registers into the slot, and the stage after the next into
  // the registers; hb: which of the two sets.
  Raw16<true> held[REG ? 2 : 1][REG ? PP : 1];  // pieces at the end of K: in place already
  auto fetch = [&](int st, int hb, int r, bool whole) __attribute__((always_inline)) {
    const int8_t* base = (r < PW ? wbase : xbase) + (size_t)st * KB;
    const unsigned v = r < PW ? vw[r < PW ? r : 0] : vx[r < PW ? 0 : r - PW];
    if (whole || st < full)
      held[hb][r].load(base + v);
    else
      held[hb][r].d = load_tail16<true>(base + v, a.K - st * KB - 16 * chunk, st * KB + 16 * chunk);  // zeros past K
  };
  auto stash = [&](int st, int hb, int slot, int r, bool whole) __attribute__((always_inline)) {
    const int8_t* p = (r < PW ? wbase : xbase) + (r < PW ? vw[r < PW ? r : 0] : vx[r < PW ? 0 : r - PW]);
    *(v4i*)(lds + slot_at(slot, r) + lane * 16) = whole || st < full ? held[hb][r].get(p) : held[hb][r].d;
  };
  auto issue = [&](int st, int hb, int slot, int r, bool whole) __attribute__((always_inline)) {
    if constexpr (REG) {
      stash(st, hb, slot, r, whole);
      fetch(st + 2, hb, r, whole);
      return;
    }
    const unsigned to = lds32 + slot_at(slot, r);
    const int8_t* base = (r < PW ? wbase : xbase) + (size_t)st * KB;
    const unsigned v = r < PW ? vw[r < PW ? r : 0] : vx[r < PW ? 0 : r - PW];
    if (whole || st < full)
      glds16_saddr(base, v, to);
    else if (st < nst)  // the end of K: zeros past it
      glds16_asm(st * KB + 16 * chunk < a.K ? base + v : zsrc, to);
  };

  acc_t acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = acc_t{0};
  v4i fw[2][NI][NV], fx[2][MJ][NV];
  const int sw = swizzle(lr);
  // read q of step `step` of a slot into buffer b (in the order of first use)
  auto read = [&](int slot, int step, int b, int q) __attribute__((always_inline)) {
    const int v = q % NV, f = q / NV, c = (step * NV + v) * 2 + lh;
    const int8_t* p = lds + slot * SLOT + 16 * (c ^ sw);
    if (f == 0)
      fw[b][0][v] = *(const v4i*)(p + (wn * NI * 32 + lr) * KB);
    else if (f <= MJ)
      fx[b][f - 1][v] = *(const v4i*)(p + TN * KB + ((wm * MJ + f - 1) * 32 + lr) * KB);
    else
      fw[b][f - MJ][v] = *(const v4i*)(p + ((wn * NI + f - MJ) * 32 + lr) * KB);
  };
  // e4m3 widened: the w fragment in use and the next, the x fragments of a step.
  // What comes next is widened while matrix instructions run that do not need it.
  typedef Mma<true> Wide;
  Wide::frag cw[2][NV], cx[MJ][NV];
  static_assert(NI == 1 || NI % 2 == 0, "a step starts with cw[0]");
  // one step's matrix instructions on buffer b; between them, in its first
  // half, the reads of the next step (rslot >= 0), and DMA pieces of stage dst
  // (dst >= 0)
  auto step = [&](int b, int rslot, int rstep, int dst, int hb, int dslot, bool whole) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < NM; ++t) {
      const int i = t / MJ, j = t % MJ;
      if (rslot >= 0) {
#pragma unroll
        for (int q = 0; q < NR; ++q)
          if (q * NM / (2 * NR) == t) read(rslot, rstep, b ^ 1, q);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (T == kF8) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          if (NM == 1) {  // a step is too short to wait for the next one's reads in it
            cw[0][v] = Wide::prep(fw[b][0][v]);
            cx[0][v] = Wide::prep(fx[b][0][v]);
          }
          acc[i][j] = MM::go(cw[i & 1][v], cx[j][v], acc[i][j]);
          __builtin_amdgcn_sched_barrier(0);
          if (NM == 1) continue;
          if (i + 1 == NI && rslot >= 0) cx[j][v] = Wide::prep(fx[b ^ 1][j][v]);
          if (j + 1 == MJ && i + 1 < NI) cw[(i + 1) & 1][v] = Wide::prep(fw[b][i + 1][v]);
          if (t + 1 == NM && rslot >= 0) cw[0][v] = Wide::prep(fw[b ^ 1][0][v]);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        acc[i][j] = MM::go(fw[b][i], fx[b][j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (dst >= 0) {
#pragma unroll
        for (int r = 0; r < PP; ++r)
          if (r * NM / PP == t) issue(dst, hb, dslot, r, whole);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // stage s, its first fragments in buffer b0; slot: where it lies, next: the
  // slot of s + 1.  Before its last step: stage s + 1 has landed everywhere,
  // and nobody reads stage s's slot any more, which stage s + SLOTS then takes.
  auto stage = [&](int s, int slot, int next, int b0, int hb, bool whole) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k + 1 < SPS; ++k) step((b0 + k) & 1, slot, k + 1, -1, 0, 0, false);
    if (REG) {  // this wave's writes of stage s + 1 are done; its loads go on
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    } else if (whole) {
      wait_vm_const<PP*(SLOTS - 2)>();  // and lgkmcnt(0)
    } else {
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    step((b0 + SPS - 1) & 1, next, 0, s + SLOTS, hb, slot, whole);
  };
  auto last_stage = [&](int slot, int b0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k + 1 < SPS; ++k) step((b0 + k) & 1, slot, k + 1, -1, 0, 0, false);
    step((b0 + SPS - 1) & 1, -1, 0, -1, 0, 0, false);
  };

  if constexpr (REG) {
#pragma unroll
    for (int st = 0; st < 2; ++st)
#pragma unroll
      for (int r = 0; r < PP; ++r) fetch(st, st, r, false);
  }
#pragma unroll
  for (int st = 0; st < SLOTS; ++st)
#pragma unroll
    for (int r = 0; r < PP; ++r) issue(st, st & 1, st, r, false);
  // the epilogue's operands, on their way before the sums begin
  const int cn = n0 + wn * NI * 32 + 4 * (lane % LPR), cr = lane / LPR;
  const bool in = cn < a.N;
  v4f ws = {0.f, 0.f, 0.f, 0.f}, bias = ws;
  if (in) {
    ws = column4(a.ws + (size_t)e * a.N, cn, a.N, a.vec);
    bias = column4(a.bias ? a.bias + (size_t)e * a.N : nullptr, cn, a.N, a.vec);
  }
  float sxr[MJ];
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int m = m0 + (wm * MJ + j) * 32 + lr;
    sxr[j] = a.xs && m < m1 ? a.xs[m] : 1.f;
  }
  if (REG)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  else if (nst >= SLOTS)
    wait_vm_const<PP*(SLOTS - 1)>();  // stage 0 has landed, the others may be under way
  else
    wait_vm0();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (nst > 0) {
#pragma unroll
    for (int q = 0; q < NR; ++q) read(0, 0, 0, q);
    if constexpr (T == kF8 && NM > 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        cw[0][v] = Wide::prep(fw[0][0][v]);
#pragma unroll
        for (int j = 0; j < MJ; ++j) cx[j][v] = Wide::prep(fx[0][j][v]);
      }
    }
    int s = 0, slot = 0;
    const auto after = [](int k) { return k + 1 == SLOTS ? 0 : k + 1; };
    // two stages at a time where a stage is an odd number of steps or goes
    // through registers: the buffers are then compile-time
    constexpr int AT = SPS % 2 || REG ? 2 : 1;
    for (; s + AT - 1 + SLOTS + (REG ? 2 : 0) < full; s += AT) {
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        stage(s + u, slot, after(slot), u * SPS & 1, (u + SLOTS) & 1, true);
        slot = after(slot);
      }
    }
    for (; s + AT < nst; s += AT) {
#pragma unroll
      for (int u = 0; u < AT; ++u) {
        stage(s + u, slot, after(slot), u * SPS & 1, (u + SLOTS) & 1, false);
        slot = after(slot);
      }
    }
    if (AT == 2 && s + 1 < nst) {
      stage(s, slot, after(slot), 0, SLOTS & 1, false);
      last_stage(after(slot), SPS & 1);
    } else {
      last_stage(slot, 0);
    }
  }
  __syncthreads();  // the slots become the epilogue's staging

  // Through LDS, a wave's 32 rows at a time, into rows: lane t then holds four
  // consecutive columns of one row, whole cache lines of y per instruction.
  // The row's scale rides in the pitch's padding.  The loop over the row code
  // is a real one (only the accumulator reads are per j): unrolled, with five
  // activations, the epilogue outgrew the instruction cache and cost as much
  // as 4096 of K.
  // A residual's loads (bf16: three j ahead; fp32: one) go in front
  // of the stores they would otherwise wait behind, and lie in LDS for the lane
  // that loaded them; rows and columns that do not exist repeat one that does.
  // 4096^3 int8 with a bf16 residual 73 us (loaded where it is added: 89; with
  // none 72), 8192 x 8192 x 2048 179 (243; 151).  Its own kernel: as a branch
  // of one, it cost products without a residual 2 us a round.
  int8_t* mine = lds + wave * 32 * PITCH;
  v4f* held_res = (v4f*)(lds + NW * 32 * PITCH + wave * NP * 1024) + lane;
  // bf16: j's in rw[j mod SB]; fp32: its halves in rw[0] and rw[1]
  constexpr int SB = MJ > 3 ? 3 : MJ;
  v2u rw[SB > 2 ? SB : 2][NP];
  const char* rbase = (const char*)uniform((const int8_t*)a.res + ((size_t)m0 * a.ldr) * (a.bf16 ? 2 : 4));
  const unsigned ldr = (unsigned)a.ldr * (a.bf16 ? 2 : 4), rcol = (unsigned)(in ? cn : 0) * (a.bf16 ? 2 : 4);
  const auto residual_at = [&](int j, int i) __attribute__((always_inline)) {
    int m = cr;
    asm volatile("" : "+v"(m));  // the addresses are made here, not all in front of the loop
    m += (wm * MJ + j) * 32 + i * RPI;
    const int last = m1 - 1 - m0;
    return rbase + ((unsigned)(m < last ? m : last) * ldr + rcol);
  };
  const auto fetch_bf16 = [&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < MJ) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        rw[j % SB][i] = *(const v2u*)residual_at(j, i);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  const auto fetch_f32 = [&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
    if constexpr (j < MJ) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const v4u v = *(const v4u*)residual_at(j, i);
        rw[0][i] = v2u{v[0], v[1]};
        rw[1][i] = v2u{v[2], v[3]};
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if (RES) {
    if (a.bf16) {
      fetch_bf16(std::integral_constant<int, 0>{});
      if constexpr (SB > 1) fetch_bf16(std::integral_constant<int, 1>{});
      if constexpr (SB > 2) fetch_bf16(std::integral_constant<int, 2>{});
    } else {
      fetch_f32(std::integral_constant<int, 0>{});
    }
  }
  auto stage_out = [&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)  // accumulator r: column (r & 3) + 8 (r >> 2) + 4 lh, row lr
        *(sum4*)(mine + lr * PITCH + (i * 32 + 8 * q + 4 * lh) * 4) =
            sum4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    if (lh == 0) *(float*)(mine + lr * PITCH + NI * 128) = sxr[j];
    if constexpr (RES) {
      if (a.bf16) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const v2u h = rw[j % SB][i];
          held_res[i * 64] = v4f{bf_lo(h[0]), bf_hi(h[0]), bf_lo(h[1]), bf_hi(h[1])};
        }
        fetch_bf16(std::integral_constant<int, j + SB>{});
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i)
          *(v4u*)&held_res[i * 64] = v4u{rw[0][i][0], rw[0][i][1], rw[1][i][0], rw[1][i][1]};
        fetch_f32(std::integral_constant<int, j + 1>{});
      }
    }
  };
#pragma unroll 1
  for (int j = 0; j < MJ; ++j) {
    if (j == 0) stage_out(std::integral_constant<int, 0>{});
    if constexpr (MJ > 1)
      if (j == 1) stage_out(std::integral_constant<int, 1>{});
    if constexpr (MJ > 2)
      if (j == 2) stage_out(std::integral_constant<int, 2>{});
    if constexpr (MJ > 3)
      if (j == 3) stage_out(std::integral_constant<int, 3>{});
    asm volatile("" ::: "memory");
    const int mj = m0 + (wm * MJ + j) * 32 + cr;
#pragma unroll 1
    for (int i = 0; i < NP; i += U) {
      v4f v[U], r[U];
      float sx[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int8_t* p = mine + ((i + u) * RPI + cr) * PITCH;
        const sum4 c = *(const sum4*)(p + 16 * (lane % LPR));
        v[u] = v4f{(float)c[0], (float)c[1], (float)c[2], (float)c[3]};
        sx[u] = *(const float*)(p + NI * 128);
        if (RES) r[u] = held_res[(i + u) * 64];
      }
      with_act(a.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = scaled4<decltype(act)::value>(v[u], sx[u], ws, bias);
      });
      if (RES || a.vec) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int m = mj + (i + u) * RPI;
          if (m < m1 && in) put4(a, m, cn, RES ? v[u] + r[u] : v[u]);
        }
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int m = mj + (i + u) * RPI;
          if (m < m1 && in) put4_any(a, m, cn, v[u]);
        }
      }
    }
    asm volatile("" ::: "memory");
  }
}

// The l-th tile of TN x TM in an order that shares operands: down groups of 4
// row blocks, column by column.  false: it has no rows.
template <int TN, int TM>
__device__ __forceinline__ bool tile_at(const LinearArgs& a, int l, int nbm, int nbn, int& e, int& m0, int& m1,
                                        int& n0) {
  constexpr int GROW = 4;
  const int grp = l / (GROW * nbn), r0 = grp * GROW;
  const int gsz = nbm - r0 < GROW ? nbm - r0 : GROW, li = l - grp * GROW * nbn;
  const int mt = r0 + li % gsz;
  n0 = li / gsz * TN;
  e = 0;
  m0 = mt * TM;
  m1 = a.M;
  if (a.E) {
    if (!expert_tile<TM>(a, mt, e, m0, m1)) return false;
    e = __builtin_amdgcn_readfirstlane(e);
    m0 = __builtin_amdgcn_readfirstlane(m0);
    m1 = __builtin_amdgcn_readfirstlane(m1);
  }
  return true;
}

template <int T, bool REG, int WN, int WM, int NI, int MJ, int NV, int KB, int SLOTS, int WPE, bool RES>
__global__ __launch_bounds__(WN* WM * 64, WPE) void linear_tile_kernel(const LinearArgs a, int nbm, int nbn) {
  __shared__ __attribute__((aligned(16))) int8_t lds[TileLds<WN, WM, NI, MJ, KB, SLOTS, RES>::BYTES];
  int e, m0, m1, n0;  // each XCD takes a run of tiles
  if (!tile_at<32 * WN * NI, 32 * WM * MJ>(a, xcd_remap(blockIdx.x, gridDim.x), nbm, nbn, e, m0, m1, n0)) return;
  linear_tile<T, REG, WN, WM, NI, MJ, NV, KB, SLOTS, RES>(a, e, m0, m1, n0, lds);
}

// 16-byte reads per fragment.  Widened e4m3 has the shortest in the large tiles:
// its widening runs behind more matrix instructions then, and spills nothing
// (8192^3: 760 us, 1020 with two; 128 x 128 tiles of 4096^3 143, 147 with two).
// A 64 x 64 tile's step has one product per fragment, and takes as long a one as
// registers allow (32 x 12288 x 4096: 16.4 us with four, 17.5 with two; through
// registers 4096 x 4096 x 4099 249 with two, 269 with four).
template <int T>
constexpr int kNv64 = T == kF8Cut ? 2 : 4;
template <int T>
constexpr int kNvReg64 = T == kF8 ? 2 : 4;
template <int T, int WIDE>
constexpr int kNv = T == kF8 ? 1 : WIDE;

// 256 x 256 tiles, from the `whole`-th on in four workgroups of 128 x 128, which
// start as CUs come free: a last round that would leave most of them idle takes
// a third of the time.  int8: 4096 x 5120 x 16384 335 -> 292 us, 4096 x 4608 x
// 4096 96 -> 87 (as a launch behind the first one it gained nothing: that waits
// for the slowest).
template <int T, bool RES>
__global__ __launch_bounds__(256, 1) void linear_tile_quarters_kernel(const LinearArgs a, int nbm, int nbn, int whole) {
  constexpr int B0 = TileLds<2, 2, 4, 4, 128, 2, RES>::BYTES, B1 = TileLds<2, 2, 2, 2, 128, 4, RES>::BYTES;
  __shared__ __attribute__((aligned(16))) int8_t lds[B0 > B1 ? B0 : B1];
  int e, m0, m1, n0;
  const int b = blockIdx.x;
  if (b < whole) {
    if (!tile_at<256, 256>(a, xcd_remap(b, whole), nbm, nbn, e, m0, m1, n0)) return;
    linear_tile<T, false, 2, 2, 4, 4, kNv<T, 2>, 128, 2, RES>(a, e, m0, m1, n0, lds);
  } else {
    const int q = b - whole;
    if (!tile_at<256, 256>(a, whole + q / 4, nbm, nbn, e, m0, m1, n0)) return;
    m0 += q % 2 * 128;
    n0 += q / 2 % 2 * 128;
    if (m0 >= m1 || n0 >= a.N) return;
    linear_tile<T, false, 2, 2, 2, 2, kNv<T, 4>, 128, 4, RES>(a, e, m0, m1, n0, lds);
  }
}

// row tiles of BM that the rows can need; grouped: each expert adds at most
// one part-filled tile, and no tile is empty
long row_tiles(const LinearArgs& a, int BM) {
  if (!a.E) return (a.M + BM - 1) / BM;
  const long t = a.M / BM + a.E;
  return t < a.M ? t : a.M;
}

// workgroups of tiles of tn columns by tm rows, 256 threads each: does a launch take them
bool tiles_fit(const LinearArgs& a, int tn, int tm) {
  return grid_fits(row_tiles(a, tm) * ((a.N + tn - 1) / tn), 256);
}

template <int T, bool REG, int WN, int WM, int NI, int MJ, int NV, int KB, int SLOTS, int WPE>
hipError_t launch_tile(const LinearArgs& a, hipStream_t s) {
  constexpr int TN = 32 * WN * NI, TM = 32 * WM * MJ;
  static_assert(WN * WM == 4, "256 threads");
  const long nbn = (a.N + TN - 1) / TN, nbm = row_tiles(a, TM);
  if (!tiles_fit(a, TN, TM)) return hipErrorInvalidConfiguration;
  const dim3 grid((unsigned)(nbm * nbn)), threads(WN * WM * 64);
  if (a.vec && a.res)
    hipLaunchKernelGGL((linear_tile_kernel<T, REG, WN, WM, NI, MJ, NV, KB, SLOTS, WPE, true>), grid, threads, 0, s, a,
                       (int)nbm, (int)nbn);
  else
    hipLaunchKernelGGL((linear_tile_kernel<T, REG, WN, WM, NI, MJ, NV, KB, SLOTS, WPE, false>), grid, threads, 0, s, a,
                       (int)nbm, (int)nbn);
  return hipGetLastError();
}

template <bool F8, bool ODD, int MI, int NJ, int WK, int U>
hipError_t launch_direct_as(const LinearArgs& a, hipStream_t s) {
  constexpr int BM = 16 * MI, BN = 16 * NJ;
  static_assert(WK == 4, "256 threads");
  const long nbn = (a.N + BN - 1) / BN;
  const long mt = row_tiles(a, BM);
  if (!tiles_fit(a, BN, BM)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((linear_direct_kernel<F8, ODD, MI, NJ, WK, U>), dim3((unsigned)(mt * nbn)), dim3(WK * 64), 0, s, a,
                     (int)mt);
  return hipGetLastError();
}

int num_cus() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0)
      v = 256;
    return v;
  }();
  return n;
}

// Which kernel.  us on one MI355X, weights from memory, 16-byte rows (int8; e4m3
// by the fp8 instructions within 10 %, 256 x 256 up to 15 % faster); then K odd,
// through registers.
//                        direct            tiles
//   M x N x K            16    32    64    64    128/4  128/2  256
//   1 x 4096 x 4096     5.8   8.8    15    12     21     33     55
//   16 x 4096 x 4096    6.8    10    16    12     21     33     55
//   32 x 4096 x 4096     10    12    18    13     22     34     57
//   32 x 12288 x 4096    26    21    20    16     24     35     58
//   64 x 4096 x 4096     18    11    21    15     24     35     58
//   256 x 4096 x 4096    59    33    21    14     26     35     62
//   512 x 4096 x 4096   115    61    34    21     26     35     62
//   1003 x 5000 x 2736  136    79    50    46     50     38     59
//   2276 x 953 x 16128  471   258   177    83     77    112    194
//   2048 x 4096 x 4096  450   232   125    70     54     42     62
//   4096 x 4096 x 4096  897   455   241   127    106     83     69
//   (256: the last round whole)
//   K odd:                                 64   128 x 64
//   32 x 4096 x 4099     16    19    32    26
//   64 x 4096 x 4099     27    18    39    29     39
//   256 x 4096 x 4099    88    51    33    28     37
//   1003 x 5000 x 2737  247   151   101    62     58
//   4096 x 4096 x 4099 1316   721   483   229    174
// e4m3 widened:          16    32    64    64    128/4  128/2  256
//   16 x 4096 x 4096    7.3   9.6    20    16     34     33     90
//   32 x 4096 x 4096     11    11    21    16     34     33     90
//   32 x 12288 x 4096    25    18    20    16     34     33     89
//   64 x 4096 x 4096     17    11    23    16     35     34     92
//   256 x 4096 x 4096    60    32    22    17     35     34     95
//   512 x 4096 x 4096   115    61    42    25     37     34     93
//   1003 x 5000 x 2736  133    84    70    49     56     42     80
//   2276 x 953 x 16128  473   255   206   113    119    117    339
//   2048 x 4096 x 4096  453   229   165    92     78     61     96
//   4096 x 4096 x 4096  902   456   322   177    153    122    111
//   K odd:                                 64   128 x 64
//   64 x 4096 x 4099     27    19    37    28     39
//   256 x 4096 x 4099    85    50    34    28     37
//   1003 x 5000 x 2737  246   140   109    62     62
//   4096 x 4096 x 4099 1343   774   511   249    212
// A tile's stage costs what its loads and its chain of steps take, nearly the
// same whatever else runs: so the tiles are compared by rounds of workgroups
// times a round's cost (us per 1024 of K with one and with two workgroups on a
// CU, and what a round costs besides).
struct TileCost {
  int tn, tm, per_cu;
  float one, two, fixed;
};
template <int T>
constexpr TileCost kDmaTiles[4] = {{64, 64, 2, 2.0f, 3.3f, 2.5f},   // 64 x 64, 5 slots
                                   {128, 128, 1, 4.5f, 5.2f, 5.f},  // 128 x 128, 4 slots
                                   {128, 128, 2, 5.0f, 9.0f, 4.f},  // 128 x 128, 2 slots
                                   {256, 256, 1, T == kS8 ? 15.f : 13.5f, T == kS8 ? 15.f : 13.5f, 9.f}};  // 256 x 256, 2 slots
template <>
constexpr TileCost kDmaTiles<kF8>[4] = {{64, 64, 2, 2.5f, 4.5f, 4.5f},
                                        {128, 128, 1, 6.9f, 6.9f, 7.f},
                                        {128, 128, 2, 6.6f, 12.2f, 7.f},
                                        {256, 256, 1, 21.7f, 21.7f, 15.f}};
constexpr TileCost kRegTiles[2] = {{64, 64, 2, 5.6f, 7.0f, 4.f}, {128, 64, 2, 8.0f, 9.9f, 5.f}};

// rows' tiles of height tm; grouped: as if each expert's last one were half full
float tiles_of_rows(const LinearArgs& a, int tm) {
  if (!a.E) return (float)((a.M + tm - 1) / tm);
  const float t = (float)a.M / tm + 0.5f * a.E;
  return t < a.M ? t : (float)a.M;
}

// Tiles of 256 x 256 whose last round, `rest` of them, runs in quarters of
// 128 x 128, one on a CU: what that takes.
float quarters_cost(const TileCost& t128, float rest, float cus, float k) {
  return __builtin_ceilf(4.f * rest / cus) * (t128.one * k + t128.fixed);
}

// The cheapest of the kinds whose tiles a launch takes.  whole: how many of its
// tiles stay whole if the others run in quarters (-1: all)
template <int N>
int best_tile(const LinearArgs& a, const TileCost (&tiles)[N], int& whole) {
  int best = 0;
  float least = INFINITY;
  whole = -1;
  const float cus = (float)num_cus(), k = a.K / 1024.f;
  for (int i = 0; i < N; ++i) {
    const TileCost& t = tiles[i];
    if (!tiles_fit(a, t.tn, t.tm)) continue;
    const float wgs = tiles_of_rows(a, t.tm) * (float)((a.N + t.tn - 1) / t.tn), round = cus * t.per_cu;
    const float rounds = __builtin_floorf(wgs / round), rest = wgs - rounds * round;
    float last = rest <= 0.f ? 0.f : (rest <= cus ? t.one : t.two) * k + t.fixed;
    bool quarters = false;
    if (t.tn == 256 && rounds > 0.f && rest > 0.f && grid_fits(4 * row_tiles(a, 256) * ((a.N + 255) / 256), 256)) {
      const float q = quarters_cost(tiles[1], rest, cus, k);
      quarters = q < last;
      if (quarters) last = q;
    }
    const float c = rounds * (t.two * k + t.fixed) + last;
    if (c < least) {
      least = c;
      best = i;
      whole = quarters ? (int)(rounds * round) : -1;
    }
  }
  return best;
}

template <int T>
hipError_t launch_quarters(const LinearArgs& a, int whole, hipStream_t s) {
  const long nbn = (a.N + 255) / 256, nbm = row_tiles(a, 256);
  if (whole > nbm * nbn) whole = (int)(nbm * nbn);
  const long grid = whole + 4 * (nbm * nbn - whole);
  if (!grid_fits(grid, 256)) return hipErrorInvalidConfiguration;
  if (a.vec && a.res)
    hipLaunchKernelGGL((linear_tile_quarters_kernel<T, true>), dim3((unsigned)grid), dim3(256), 0, s, a, (int)nbm,
                       (int)nbn, whole);
  else
    hipLaunchKernelGGL((linear_tile_quarters_kernel<T, false>), dim3((unsigned)grid), dim3(256), 0, s, a, (int)nbm,
                       (int)nbn, whole);
  return hipGetLastError();
}

template <int T>
hipError_t launch_best_tile(const LinearArgs& a, bool dma, hipStream_t s) {
  int whole;
  if (!dma) {
    if (best_tile(a, kRegTiles, whole) == 0) return launch_tile<T, true, 2, 2, 1, 1, kNvReg64<T>, 128, 2, 2>(a, s);
    return launch_tile<T, true, 2, 2, 2, 1, 2, 128, 2, 2>(a, s);
  }
  switch (best_tile(a, kDmaTiles<T>, whole)) {
    case 0: return launch_tile<T, false, 2, 2, 1, 1, kNv64<T>, 128, 5, 2>(a, s);
    case 1: return launch_tile<T, false, 2, 2, 2, 2, kNv<T, 4>, 128, 4, 1>(a, s);
    case 2: return launch_tile<T, false, 2, 2, 2, 2, kNv<T, 2>, 128, 2, 2>(a, s);
    default:
      return whole > 0 ? launch_quarters<T>(a, whole, s)
                       : launch_tile<T, false, 2, 2, 4, 4, kNv<T, 2>, 128, 2, 1>(a, s);
  }
}

template <bool F8, int MI, int NJ, int WK, int U>
hipError_t launch_direct(const LinearArgs& a, hipStream_t s) {
  return a.odd ? launch_direct_as<F8, true, MI, NJ, WK, U>(a, s) : launch_direct_as<F8, false, MI, NJ, WK, U>(a, s);
}

template <bool F8>
hipError_t launch_linear_any(const LinearArgs& a, bool dma, hipStream_t s) {
  const float rows = a.E ? (float)a.M / a.E : (float)a.M;  // rows that share weights
  const float cus = (float)num_cus();
  const auto wgs = [&](int t) { return tiles_of_rows(a, t) * (float)((a.N + t - 1) / t); };
  // tiles from half as many workgroups as CUs on; their rows' byte offsets are 32 bits
  if (rows > 16.f && wgs(64) >= 0.5f * cus && a.ldx <= (1 << 22) && a.ldw <= (1 << 22) && a.ldr <= (1 << 21)) {
    if constexpr (!F8)
      return launch_best_tile<kS8>(a, dma, s);
    else
      return a.cut ? launch_best_tile<kF8Cut>(a, dma, s) : launch_best_tile<kF8>(a, dma, s);
  }
  if ((rows <= 16.f || wgs(16) <= 2.f * cus) && tiles_fit(a, 16, 16)) return launch_direct<F8, 1, 1, 4, 4>(a, s);
  return wgs(64) < cus ? launch_direct<F8, 2, 2, 4, 4>(a, s) : launch_direct<F8, 4, 4, 4, 2>(a, s);
}

template <bool F8>
int linear_any(const char* who, const dlq_linear_desc* d, int E, const int32_t* off, const void* x, const float* xs,
               const void* w, const float* ws, const float* bias, const void* res, void* y, void* stream) {
  const auto bad = [&](const char* what) { return fail(DLQ_ERR_ARG, std::string(who) + ": " + what); };
  if (!d || d->M < 0 || d->N < 0 || d->K < 0) return bad("bad shape");
  if (d->K > 131071) return bad("K above 131071");
  // a row's or column's number plus a tile's height stays an int, here and in the kernels
  if (d->M > INT_MAX - 511 || d->N > INT_MAX - 511) return bad("M or N above 2^31 - 512");
  const int act = F8 ? d->act & ~DLQ_FP8_SUMS : d->act;
  if (act < DLQ_ACT_NONE || act > DLQ_ACT_SILU) return bad("bad act");
  if (d->out_type != DLQ_T_F32 && d->out_type != DLQ_T_BF16) return bad("bad out_type");
  if (d->ldx < d->K || d->ldw < d->K) return bad("row stride below K");
  if (d->ldy < d->N || (res && d->ldr < d->N)) return bad("row stride below N");
  if (E < 0 || E > 65535) return bad("experts outside 0..65535");
  if (d->M == 0 || d->N == 0 || (off && E == 0)) return DLQ_OK;
  if (!ws || !y || (d->K && (!x || !w))) return bad("null pointer");
  const uintptr_t es = d->out_type == DLQ_T_BF16 ? 2 : 4;
  if (((uintptr_t)xs | (uintptr_t)ws | (uintptr_t)bias | (uintptr_t)off) % 4 || ((uintptr_t)y | (uintptr_t)res) % es)
    return bad("pointer not aligned to its element type");
  if (res == y && res && d->ldr != d->ldy) return bad("residual is y with another row stride");
  LinearArgs a;
  a.x = (const int8_t*)x;
  a.w = (const int8_t*)w;
  a.xs = xs;
  a.ws = ws;
  a.bias = bias;
  a.res = res;
  a.y = y;
  a.M = d->M;
  a.N = d->N;
  a.K = d->K;
  a.ldx = d->ldx;
  a.ldw = d->ldw;
  a.ldy = d->ldy;
  a.ldr = res ? d->ldr : 0;
  a.act = act;
  a.cut = act != d->act;
  a.bf16 = d->out_type == DLQ_T_BF16;
  a.vec = ((uintptr_t)ws | (uintptr_t)bias) % 16 == 0 && ((uintptr_t)y | (uintptr_t)res) % (4 * es) == 0 &&
          d->N % 4 == 0 && d->ldy % 4 == 0 && (!res || d->ldr % 4 == 0);
  a.odd = ((uintptr_t)x | (uintptr_t)w | (uintptr_t)d->ldx | (uintptr_t)d->ldw) % 4 != 0;
  a.E = E;
  a.off = off;
  const bool dma = ((uintptr_t)x | (uintptr_t)w) % 16 == 0 && d->K % 16 == 0 && d->ldx % 16 == 0 && d->ldw % 16 == 0;
  const hipError_t e = launch_linear_any<F8>(a, dma, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration) return bad("more tiles than a launch takes");
  return e == hipSuccess ? DLQ_OK : fail(DLQ_ERR_LAUNCH, std::string(who) + " launch: " + hipGetErrorString(e));
}

}  // namespace
}  // namespace dlq

using namespace dlq;

extern "C" {

int dlq_linear_act_s8(const dlq_linear_desc* d, const int8_t* x, const float* x_scale, const int8_t* w,
                      const float* w_scale, const float* bias, const void* residual, void* y, void* stream) {
  return linear_any<false>("linear_act_s8", d, 0, nullptr, x, x_scale, w, w_scale, bias, residual, y, stream);
}

int dlq_linear_act_f8(const dlq_linear_desc* d, const uint8_t* x, const float* x_scale, const uint8_t* w,
                      const float* w_scale, const float* bias, const void* residual, void* y, void* stream) {
  return linear_any<true>("linear_act_f8", d, 0, nullptr, x, x_scale, w, w_scale, bias, residual, y, stream);
}

int dlq_linear_grouped_s8(const dlq_linear_desc* d, int E, const int32_t* offsets, const int8_t* x,
                          const float* x_scale, const int8_t* w, const float* w_scale, const float* bias,
                          const void* residual, void* y, void* stream) {
  if (!offsets) return fail(DLQ_ERR_ARG, "linear_grouped_s8: null offsets");
  return linear_any<false>("linear_grouped_s8", d, E, offsets, x, x_scale, w, w_scale, bias, residual, y, stream);
}

int dlq_linear_grouped_f8(const dlq_linear_desc* d, int E, const int32_t* offsets, const uint8_t* x,
                          const float* x_scale, const uint8_t* w, const float* w_scale, const float* bias,
                          const void* residual, void* y, void* stream) {
  if (!offsets) return fail(DLQ_ERR_ARG, "linear_grouped_f8: null offsets");
  return linear_any<true>("linear_grouped_f8", d, E, offsets, x, x_scale, w, w_scale, bias, residual, y, stream);
}

}  // extern "C"
