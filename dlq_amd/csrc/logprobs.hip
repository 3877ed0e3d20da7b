// logprobs.hip -- dlq_logprobs: for each row of logits the log probability of
// a given token, the entropy and the `top` largest with their log
// probabilities.
//   m = max x, S = sum e^(x-m), T = sum e^(x-m) (x-m):
//   lp[j] = x[j] - m - log S,  entropy = log S - T / S.
// A masked logit (-inf) adds nothing to S and T; a row of nothing else has
// m = -inf, taken as 0 so that x - m stays -inf (S = 0: entropy 0).
#include "rowops_common.h"

namespace dlq {
namespace {

template <bool BF16>
__device__ __forceinline__ float logit(const void* x, size_t i) {
  return BF16 ? __uint_as_float((unsigned)((const uint16_t*)x)[i] << 16) : ((const float*)x)[i];
}

// The order of the alternatives as one unsigned number: the value's bits so
// turned that they are ordered as the values are (-0 as +0, NaN on top), then
// the index, the lowest largest.  0 is below every entry.
__device__ __forceinline__ unsigned value_key(float v) {
  const unsigned u = __float_as_uint(v + 0.f);
  return v != v ? 0xfffffffeu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long entry_key(float v, int j) {
  return (unsigned long long)value_key(v) << 32 | (unsigned)~j;
}

// sums over the 256 threads, in a fixed order
template <typename T, typename F>
__device__ __forceinline__ T block_join(T v, T* buf, F f) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = f(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  return f(f(buf[0], buf[1]), f(buf[2], buf[3]));
}

template <bool BF16>
__global__ __launch_bounds__(256) void logprobs_kernel(const void* __restrict__ x, int K, int ldx,
                                                       const int* __restrict__ tokens, int top,
                                                       float* __restrict__ logprob, float* __restrict__ entropy,
                                                       int* __restrict__ top_idx, float* __restrict__ top_logprob) {
  __shared__ float fb[4];
  __shared__ unsigned long long kb[4];
  const int tid = threadIdx.x, row = blockIdx.x;
  const size_t x0 = (size_t)row * ldx;
  const auto add = [](float a, float b) { return a + b; };
  float m = -INFINITY;
  for (int j = tid; j < K; j += 256) m = fmaxf(m, logit<BF16>(x, x0 + j));
  m = block_join(m, fb, [](float a, float b) { return fmaxf(a, b); });
  if (m == -INFINITY) m = 0.f;
  float S = 0.f, T = 0.f;
  for (int j = tid; j < K; j += 256) {
    const float d = logit<BF16>(x, x0 + j) - m, e = expf(d);
    S += e;
    T += e > 0.f ? e * d : 0.f;
  }
  S = block_join(S, fb, add);
  T = block_join(T, fb, add);
  const float ls = logf(S);
  if (tid == 0) {
    if (tokens) {
      const int t = tokens[row];
      float lp = 0.f;
      if (t >= K) lp = __uint_as_float(0x7fc00000u);
      else if (t >= 0) {
        const float d = logit<BF16>(x, x0 + t) - m;
        lp = S == 0.f || (d == -INFINITY && S == S) ? -INFINITY : d - ls;
      }
      logprob[row] = lp;
    }
    if (entropy) entropy[row] = S == 0.f ? 0.f : ls - T / S;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < top; ++k) {
    unsigned long long best = 0;
    for (int j = tid; j < K; j += 256) {
      const unsigned long long c = entry_key(logit<BF16>(x, x0 + j), j);
      if (c < last && c > best) best = c;
    }
    last = block_join(best, kb, [](unsigned long long a, unsigned long long b) { return a > b ? a : b; });
    if (tid == 0) {
      const int j = (int)~(unsigned)last;
      const float d = logit<BF16>(x, x0 + j) - m;
      top_idx[(size_t)row * top + k] = j;
      top_logprob[(size_t)row * top + k] = S == 0.f || (d == -INFINITY && S == S) ? -INFINITY : d - ls;
    }
  }
}

}  // namespace
}  // namespace dlq

using namespace dlq;

extern "C" {

size_t dlq_logprobs_workspace_bytes(int rows, int K, int top) {
  (void)rows;
  (void)K;
  (void)top;
  return 0;
}

int dlq_logprobs(const void* x, int x_type, int rows, int K, int ldx, const int32_t* tokens, int top, float* logprob,
                 float* entropy, int32_t* top_idx, float* top_logprob, void* workspace, size_t ws_bytes,
                 void* stream) {
  if (rows < 0 || K <= 0) return fail(DLQ_ERR_ARG, "logprobs: bad shape");
  if (x_type != DLQ_T_F32 && x_type != DLQ_T_BF16) return fail(DLQ_ERR_ARG, "logprobs: bad x_type");
  if (ldx < K) return fail(DLQ_ERR_ARG, "logprobs: row stride below K");
  if (top < 0 || top > 64 || top > K) return fail(DLQ_ERR_ARG, "logprobs: top outside 0..min(64, K)");
  if (rows == 0) return DLQ_OK;
  if (!grid_fits(rows, 256)) return fail(DLQ_ERR_ARG, "logprobs: too many rows");
  if (!x || !tokens != !logprob || (top && (!top_idx || !top_logprob)))
    return fail(DLQ_ERR_ARG, "logprobs: null pointer (tokens and logprob come together)");
  if ((uintptr_t)x % (x_type == DLQ_T_BF16 ? 2 : 4) ||
      ((uintptr_t)tokens | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_idx | (uintptr_t)top_logprob) % 4)
    return fail(DLQ_ERR_ARG, "logprobs: pointer not aligned to its element type");
  const size_t need = dlq_logprobs_workspace_bytes(rows, K, top);
  if (need && (!workspace || ws_bytes < need || (uintptr_t)workspace % 8))
    return fail(DLQ_ERR_ARG, "logprobs: workspace missing, too small or not 8-byte aligned");
  if (x_type == DLQ_T_BF16)
    hipLaunchKernelGGL(logprobs_kernel<true>, dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream, x, K, ldx,
                       tokens, top, logprob, entropy, top_idx, top_logprob);
  else
    hipLaunchKernelGGL(logprobs_kernel<false>, dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream, x, K, ldx,
                       tokens, top, logprob, entropy, top_idx, top_logprob);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? DLQ_OK : fail(DLQ_ERR_LAUNCH, std::string("logprobs launch: ") + hipGetErrorString(e));
}

}  // extern "C"
