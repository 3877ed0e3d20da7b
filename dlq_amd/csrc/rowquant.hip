// rowquant.hip -- dlq_quantize_rows_dyn_s8 / _f8: each row of fp32 or bf16
// values to int8 / e4m3 codes at a scale of its own, a = max |x|,
// s = a / m, q = rne(clamp(x * (1/s), +-m)), m = 127 | 448.
//
// The maximum is taken on the bits without their sign: as unsigned integers
// they are ordered as the magnitudes are, and an infinity or NaN comes out on
// top of every finite value, so one integer maximum finds both.
#include "rowops_common.h"

namespace dlq {
namespace {

constexpr float kTiny = 0x1p-100f;  // below: the row counts as zero (1/s stays finite above)

template <bool BF16>
__device__ __forceinline__ float row_value(const void* x, size_t i) {
  return BF16 ? __uint_as_float((unsigned)((const uint16_t*)x)[i] << 16) : ((const float*)x)[i];
}

template <bool BF16, bool F8>
__global__ __launch_bounds__(256) void quantize_rows_dyn_kernel(const void* __restrict__ x, int cols, int ldx,
                                                                uint8_t* __restrict__ q, int ldq,
                                                                float* __restrict__ scale) {
  __shared__ unsigned wmax[4];
  const int tid = threadIdx.x, row = blockIdx.x;
  const size_t x0 = (size_t)row * ldx;
  unsigned u = 0;
  for (int i = tid; i < cols; i += 256) {
    const unsigned b = __float_as_uint(row_value<BF16>(x, x0 + i)) & 0x7fffffffu;
    u = b > u ? b : u;
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const unsigned v = (unsigned)__shfl_xor((int)u, o);
    u = v > u ? v : u;
  }
  if ((tid & 63) == 0) wmax[tid >> 6] = u;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) u = wmax[i] > u ? wmax[i] : u;
  const float m = F8 ? 448.f : 127.f, a = __uint_as_float(u);
  const bool bad = u >= 0x7f800000u, none = bad || a < kTiny;
  const float s = bad ? __uint_as_float(0x7fc00000u) : none ? 1.f : __fdiv_rn(a, m);
  const float inv = none ? 0.f : __fdiv_rn(1.f, s);
  if (tid == 0) scale[row] = s;
  for (int i = tid; i < ldq; i += 256) {
    const float v = i < cols && !none ? row_value<BF16>(x, x0 + i) * inv : 0.f;
    q[(size_t)row * ldq + i] = (uint8_t)(F8 ? enc4_f8(v, 0.f, 0.f, 0.f, -448.f) : quant4(v, 0.f, 0.f, 0.f, -127.f));
  }
}

template <bool F8>
int quantize_rows_dyn(const void* x, int x_type, int rows, int cols, int ldx, uint8_t* q, int ldq, float* scale,
                      void* stream) {
  if (rows < 0 || cols <= 0) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: bad shape");
  if (x_type != DLQ_T_F32 && x_type != DLQ_T_BF16) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: bad x_type");
  if (ldx < cols || ldq < cols) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: row stride below cols");
  if (rows == 0) return DLQ_OK;
  if (!grid_fits(rows, 256)) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: too many rows");
  if (!x || !q || !scale) return fail(DLQ_ERR_ARG, "quantize_rows_dyn: null pointer");
  if ((uintptr_t)x % (x_type == DLQ_T_BF16 ? 2 : 4) || (uintptr_t)scale % 4)
    return fail(DLQ_ERR_ARG, "quantize_rows_dyn: pointer not aligned to its element type");
  if (x_type == DLQ_T_BF16)
    hipLaunchKernelGGL((quantize_rows_dyn_kernel<true, F8>), dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream,
                       x, cols, ldx, q, ldq, scale);
  else
    hipLaunchKernelGGL((quantize_rows_dyn_kernel<false, F8>), dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream,
                       x, cols, ldx, q, ldq, scale);
  const hipError_t e = hipGetLastError();
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
