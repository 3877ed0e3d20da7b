// rowquant.hip -- dlq_quantize_rows_dyn_s8 / _f8: each row of fp32 or bf16
// values to int8 / e4m3 codes at a scale of its own, a = max |x|,
// s = a / m, q = rne(clamp(x * (1/s), +-m)), m = 127 | 448.
//
// The maximum is taken on the bits without their sign: as unsigned integers
// they are ordered as the magnitudes are, and an infinity or NaN comes out on
// top of every finite value, so one integer maximum finds both.
//
// Bound by memory: a row stays in registers between its maximum and its codes
// (one read), each lane's loads all on their way at once; a wave per row up to
// 2048 columns, 4 waves up to 16384, 16 above, rows past 65536 read again.
// 8192 x 8192: bf16 37.8 us, 5.3 TB/s read and written (a large copy: 5.2),
// fp32 73 us, 4.6 TB/s; keeping registers for 16384 columns there: 39.8 and 92.
#include "rowops_common.h"

namespace dlq {
namespace {

constexpr float kTiny = 0x1p-100f;  // below: the row counts as zero (1/s stays finite above)
typedef v2u v2u_any __attribute__((aligned(1)));
typedef unsigned u_any __attribute__((aligned(1)));

template <bool BF16>
__device__ __forceinline__ float row_value(const void* x, size_t i) {
  return BF16 ? __uint_as_float((unsigned)((const uint16_t*)x)[i] << 16) : ((const float*)x)[i];
}
template <bool F8>
__device__ __forceinline__ unsigned codes4(float a, float b, float c, float d) {
  return F8 ? enc4_f8(a, b, c, d, -448.f) : quant4(a, b, c, d, -127.f);
}

// One load of a lane: 16 bytes, 4 fp32 or 8 bf16 values.
template <bool BF16>
struct Vec {
  static constexpr int N = BF16 ? 8 : 4;
  v4i r;
  __device__ __forceinline__ void load(const void* x, size_t i) {
    r = *(const v4i_any*)((const char*)x + i * (BF16 ? 2 : 4));
  }
  // the last values of a row, from column c on; zeros behind them
  __device__ __forceinline__ void load_end(const void* x, size_t x0, unsigned c, unsigned cols) {
    constexpr int S = BF16 ? 2 : 4;
    const int left = (int)(cols - c) * S;
    r = load_tail16<false>((const char*)x + (x0 + c) * S, left < 16 ? left : 16, c < 16 ? (int)c * S : 16);
  }
  __device__ __forceinline__ unsigned most() const {
    unsigned u = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned w = (unsigned)r[k];
      if constexpr (BF16)
        u = max(u, max(w << 16 & 0x7fff0000u, w & 0x7fff0000u));
      else
        u = max(u, w & 0x7fffffffu);
    }
    return u;
  }
  template <bool F8>
  __device__ __forceinline__ v2u codes(float inv) const {
    if constexpr (BF16)
      return v2u{codes4<F8>(bf_lo(r[0]) * inv, bf_hi(r[0]) * inv, bf_lo(r[1]) * inv, bf_hi(r[1]) * inv),
                 codes4<F8>(bf_lo(r[2]) * inv, bf_hi(r[2]) * inv, bf_lo(r[3]) * inv, bf_hi(r[3]) * inv)};
    else
      return v2u{codes4<F8>(__int_as_float(r[0]) * inv, __int_as_float(r[1]) * inv, __int_as_float(r[2]) * inv,
                            __int_as_float(r[3]) * inv),
                 0u};
  }
};

// NW waves per row (a workgroup; 1: four rows per workgroup, no barriers),
// KEEP columns of it in registers.
template <bool BF16, bool F8, int NW, int KEEP>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void quantize_rows_dyn_kernel(
    const void* __restrict__ x, int rows, unsigned cols, int ldx, uint8_t* __restrict__ q, unsigned ldq,
    float* __restrict__ scale) {
  // columns are unsigned: cols and ldq end at 2^31 - 1, and a step beyond them must not wrap
  typedef Vec<BF16> V;
  constexpr int TPR = 64 * NW, N = V::N, SPAN = TPR * N;  // columns of one load of all lanes
  constexpr int NV = KEEP / SPAN;                         // loads kept in registers
  __shared__ unsigned wmax[NW];
  const unsigned t = threadIdx.x % TPR;
  const int row = NW == 1 ? (int)blockIdx.x * 4 + (int)(threadIdx.x >> 6) : (int)blockIdx.x;
  if (NW == 1 && row >= rows) return;
  const size_t x0 = (size_t)row * ldx;
  uint8_t* qr = q + (size_t)row * ldq;
  V v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const unsigned c = i * SPAN + t * N;
    if (c + N <= cols)
      v[i].load(x, x0 + c);
    else if (c < cols)
      v[i].load_end(x, x0, c, cols);
  }
  unsigned u = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * SPAN + t * N < cols) u = max(u, v[i].most());
  for (unsigned c = NV * SPAN + t * N; c < cols; c += SPAN) {
    V w;
    if (c + N <= cols)
      w.load(x, x0 + c);
    else
      w.load_end(x, x0, c, cols);
    u = max(u, w.most());
  }
  u = (unsigned)wave_join((int)u, 0, [](int a, int b) { return (int)max((unsigned)a, (unsigned)b); });
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) wmax[threadIdx.x >> 6] = u;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) u = max(u, wmax[i]);
  }
  const float a = __uint_as_float(u);
  const bool bad = u >= 0x7f800000u, none = bad || a < kTiny;
  const float s = bad ? __uint_as_float(0x7fc00000u) : none ? 1.f : __fdiv_rn(a, F8 ? 448.f : 127.f);
  const float inv = none ? 0.f : __fdiv_rn(1.f, s);
  if (t == 0) scale[row] = s;
  const auto put = [&](const V& w, unsigned c) {
    v2u o = w.template codes<F8>(inv);
    if (bad) o = v2u{0u, 0u};  // 0 * inf
    if (c + N <= cols) {
      if constexpr (BF16)
        *(v2u_any*)(qr + c) = o;
      else
        *(u_any*)(qr + c) = o[0];
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (c + k < cols) qr[c + k] = (uint8_t)(o[k >> 2] >> (8 * (k & 3)));
    }
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const unsigned c = i * SPAN + t * N;
    if (c < cols) put(v[i], c);
  }
  for (unsigned c = NV * SPAN + t * N; c < cols; c += SPAN) {
    V w;
    if (c + N <= cols)
      w.load(x, x0 + c);
    else
      w.load_end(x, x0, c, cols);
    put(w, c);
  }
  for (unsigned c = cols + t; c < ldq; c += TPR) qr[c] = 0;
}

template <bool BF16, bool F8, int NW, int KEEP>
hipError_t launch_as(const void* x, int rows, int cols, int ldx, uint8_t* q, int ldq, float* scale, hipStream_t s) {
  constexpr int ROWS = NW == 1 ? 4 : 1, THREADS = NW == 1 ? 256 : NW * 64;
  constexpr long long MOST = (1LL << 21) * ROWS;  // rows of one launch, whose work-items are 32 bits
  for (long long r = 0; r < rows; r += MOST) {
    const int n = (int)(rows - r < MOST ? rows - r : MOST);
    hipLaunchKernelGGL((quantize_rows_dyn_kernel<BF16, F8, NW, KEEP>), dim3((unsigned)((n + ROWS - 1) / ROWS)),
                       dim3(THREADS), 0, s, (const char*)x + (size_t)r * ldx * (BF16 ? 2 : 4), n, cols, ldx,
                       q + (size_t)r * ldq, ldq, scale + r);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <bool BF16, bool F8>
hipError_t launch_quantize(const void* x, int rows, int cols, int ldx, uint8_t* q, int ldq, float* scale,
                           hipStream_t s) {
  if (cols <= 2048) return launch_as<BF16, F8, 1, 2048>(x, rows, cols, ldx, q, ldq, scale, s);
  if (cols <= 8192) return launch_as<BF16, F8, 4, 8192>(x, rows, cols, ldx, q, ldq, scale, s);
  if (cols <= 16384) return launch_as<BF16, F8, 4, 16384>(x, rows, cols, ldx, q, ldq, scale, s);
  return launch_as<BF16, F8, 16, 65536>(x, rows, cols, ldx, q, ldq, scale, s);
}

template <bool F8>
int quantize_rows_dyn(const void* x, int x_type, int rows, int cols, int ldx, uint8_t* q, int ldq, float* scale,
                      void* stream) {
  if (rows < 0 || cols <= 0) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: bad shape");
  if (x_type != DLQ_T_F32 && x_type != DLQ_T_BF16) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: bad x_type");
  if (ldx < cols || ldq < cols) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: row stride below cols");
  if (rows == 0) return DLQ_OK;
  if (!x || !q || !scale) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: null pointer");
  if ((uintptr_t)x % (x_type == DLQ_T_BF16 ? 2 : 4) || (uintptr_t)scale % 4)
    return fail(DLQ_ERR_ARG, "quantize_rows_dyn: pointer not aligned to its element type");
  const hipError_t e = x_type == DLQ_T_BF16
                           ? launch_quantize<true, F8>(x, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream)
                           : launch_quantize<false, F8>(x, rows, cols, ldx, q, ldq, scale, (hipStream_t)stream);
  return e == hipSuccess ? DLQ_OK
                         : fail(DLQ_ERR_LAUNCH, std::string("quantize_rows_dyn launch: ") + hipGetErrorString(e));
}

}  // namespace
}  // namespace dlq

using namespace dlq;

extern "C" {

int dlq_quantize_rows_dyn_s8(const void* x, int x_type, int rows, int cols, int ldx, int8_t* q, int ldq, float* scale,
                             void* stream) {
  return quantize_rows_dyn<false>(x, x_type, rows, cols, ldx, (uint8_t*)q, ldq, scale, stream);
}

int dlq_quantize_rows_dyn_f8(const void* x, int x_type, int rows, int cols, int ldx, uint8_t* q, int ldq, float* scale,
                             void* stream) {
  return quantize_rows_dyn<true>(x, x_type, rows, cols, ldx, q, ldq, scale, stream);
}

}  // extern "C"
