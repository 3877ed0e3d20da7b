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
  int act, bf16, vec;  // vec: y, res, ws and bias take aligned 4-element accesses
  int E;               // 0: one product over all rows
  const int* off;      // [E + 1], E > 0
};

__device__ __forceinline__ float act_of(float v, int act) {
  switch (act) {
    case DLQ_ACT_RELU: return v < 0.f ? 0.f : v;  // a NaN stays
    case DLQ_ACT_GELU: return 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    case DLQ_ACT_GELU_TANH: {  // 1 + tanh(u) = 2 / (1 + e^-2u)
      const float u = v * __builtin_fmaf(0.044715f * v, v, 1.f) * 1.5957691216057308f;
      return v / (1.f + expf(-u));
    }
    case DLQ_ACT_SILU: return v / (1.f + expf(-v));
    default: return v;
  }
}

// Four accumulators of row m, columns n..n+3 of expert e (0 if not grouped).
__device__ __forceinline__ void store4(const LinearArgs& a, int e, int m, int n, const float* acc) {
  const float sx = a.xs ? a.xs[m] : 1.f;
  const size_t en = (size_t)e * a.N + n, ym = (size_t)m * a.ldy + n, rm = (size_t)m * a.ldr + n;
  if (a.vec && n + 4 <= a.N) {
    const v4f ws = *(const v4f*)(a.ws + en);
    v4f b = {0.f, 0.f, 0.f, 0.f}, v;
    if (a.bias) b = *(const v4f*)(a.bias + en);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = act_of(__builtin_fmaf(acc[i], sx * ws[i], b[i]), a.act);
    if (a.bf16) {
      if (a.res) {
        const v2u r = *(const v2u*)((const uint16_t*)a.res + rm);
        v += v4f{bf_lo(r[0]), bf_hi(r[0]), bf_lo(r[1]), bf_hi(r[1])};
      }
      *(v2u*)((uint16_t*)a.y + ym) = v2u{bf_pack(v[0], v[1]), bf_pack(v[2], v[3])};
    } else {
      if (a.res) v += *(const v4f*)((const float*)a.res + rm);
      *(v4f*)((float*)a.y + ym) = v;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) break;
    float v = act_of(__builtin_fmaf(acc[i], sx * a.ws[en + i], a.bias ? a.bias[en + i] : 0.f), a.act);
    if (a.bf16) {
      if (a.res) v += __uint_as_float((unsigned)((const uint16_t*)a.res)[rm + i] << 16);
      ((uint16_t*)a.y)[ym + i] = (uint16_t)bf_pack(v, 0.f);
    } else {
      if (a.res) v += ((const float*)a.res)[rm + i];
      ((float*)a.y)[ym + i] = v;
    }
  }
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
// coarser than a 32-bit sum.  The codes are bf16 values as well, so here they
// are widened (one conversion per two codes) and multiplied as bf16, whose
// products are exact and sums fp32: twice the matrix instructions, in a kernel
// that waits for memory.
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
template <bool F8, int MI, int NJ, int WK>
__global__ __launch_bounds__(WK * 64) void linear_direct_kernel(const LinearArgs a) {
  typedef Mma<F8> MM;
  typedef typename MM::acc_t acc_t;
  constexpr int BM = 16 * MI, BN = 16 * NJ, KB = 64;
  __shared__ acc_t part[WK][MI * NJ][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, lr = lane & 15, lg = lane >> 4;
  const int nbn = (a.N + BN - 1) / BN;
  const int n0 = (int)(blockIdx.x % nbn) * BN, mt = blockIdx.x / nbn;
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
  for (int s = s0; s < s1; ++s) {
    v4i rx[MI], rw[NJ];
    if (s < full) {
#pragma unroll
      for (int i = 0; i < MI; ++i) rx[i] = *(const v4i_any*)(xp[i] + (size_t)s * KB);
#pragma unroll
      for (int j = 0; j < NJ; ++j) rw[j] = *(const v4i_any*)(wp[j] + (size_t)s * KB);
    } else {  // the end of K: zeros past it
      const int k = s * KB, avail = a.K - k - 16 * lg;
#pragma unroll
      for (int i = 0; i < MI; ++i) rx[i] = load_codes16(xp[i] + k, avail);
#pragma unroll
      for (int j = 0; j < NJ; ++j) rw[j] = load_codes16(wp[j] + k, avail);
    }
    typename MM::frag fx[MI], fw[NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i) fx[i] = MM::prep(rx[i]);
#pragma unroll
    for (int j = 0; j < NJ; ++j) fw[j] = MM::prep(rw[j]);
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[i][j] = MM::go(fw[j], fx[i], acc[i][j]);
  }
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
    const float v[4] = {(float)s[0], (float)s[1], (float)s[2], (float)s[3]};
    if (m < m1) store4(a, e, m, n, v);
  }
}

template <bool F8, int MI, int NJ, int WK>
hipError_t launch_direct(const LinearArgs& a, hipStream_t s) {
  constexpr int BM = 16 * MI, BN = 16 * NJ;
  const long nbn = (a.N + BN - 1) / BN;
  // grouped: each expert adds at most one part-filled tile, and no tile is empty
  long mt = (a.M + BM - 1) / BM;
  if (a.E) {
    mt = a.M / BM + a.E;
    if (mt > a.M) mt = a.M;
  }
  if (!grid_fits(mt * nbn, WK * 64)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((linear_direct_kernel<F8, MI, NJ, WK>), dim3((unsigned)(mt * nbn)), dim3(WK * 64), 0, s, a);
  return hipGetLastError();
}

template <bool F8>
int linear_any(const char* who, const dlq_linear_desc* d, int E, const int32_t* off, const void* x, const float* xs,
               const void* w, const float* ws, const float* bias, const void* res, void* y, void* stream) {
  const std::string p = std::string(who) + ": ";
  if (!d || d->M < 0 || d->N < 0 || d->K < 0) return fail(DLQ_ERR_ARG, p + "bad shape");
  if (d->K > 131071) return fail(DLQ_ERR_ARG, p + "K above 131071");
  if (d->act < DLQ_ACT_NONE || d->act > DLQ_ACT_SILU) return fail(DLQ_ERR_ARG, p + "bad act");
  if (d->out_type != DLQ_T_F32 && d->out_type != DLQ_T_BF16) return fail(DLQ_ERR_ARG, p + "bad out_type");
  if (d->ldx < d->K || d->ldw < d->K) return fail(DLQ_ERR_ARG, p + "row stride below K");
  if (d->ldy < d->N || (res && d->ldr < d->N)) return fail(DLQ_ERR_ARG, p + "row stride below N");
  if (E < 0 || E > 65535) return fail(DLQ_ERR_ARG, p + "experts outside 0..65535");
  if (d->M == 0 || d->N == 0 || (off && E == 0)) return DLQ_OK;
  if (!ws || !y || (d->K && (!x || !w))) return fail(DLQ_ERR_ARG, p + "null pointer");
  const uintptr_t es = d->out_type == DLQ_T_BF16 ? 2 : 4;
  if (((uintptr_t)xs | (uintptr_t)ws | (uintptr_t)bias | (uintptr_t)off) % 4 || ((uintptr_t)y | (uintptr_t)res) % es)
    return fail(DLQ_ERR_ARG, p + "pointer not aligned to its element type");
  if (res == y && res && d->ldr != d->ldy) return fail(DLQ_ERR_ARG, p + "residual is y with another row stride");
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
  a.act = d->act;
  a.bf16 = d->out_type == DLQ_T_BF16;
  a.vec = ((uintptr_t)ws | (uintptr_t)bias) % 16 == 0 && ((uintptr_t)y | (uintptr_t)res) % (4 * es) == 0 &&
          d->ldy % 4 == 0 && (!res || d->ldr % 4 == 0) && (E <= 1 || d->N % 4 == 0);
  a.E = E;
  a.off = off;
  const hipError_t e = launch_direct<F8, 1, 1, 4>(a, (hipStream_t)stream);
  return e == hipSuccess ? DLQ_OK : fail(DLQ_ERR_LAUNCH, p + "launch: " + hipGetErrorString(e));
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
