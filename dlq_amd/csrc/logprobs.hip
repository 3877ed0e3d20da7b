// logprobs.hip -- dlq_logprobs: for each row of logits the log probability of
// a given token, the entropy and the `top` largest with their log
// probabilities.
//   m = max x, S = sum e^(x-m), T = sum e^(x-m) (x-m):
//   lp[j] = x[j] - m - log S,  entropy = log S - T / S.
// A masked logit (-inf) adds nothing to S and T; a row of nothing else has
// m = -inf, taken as 0 so that x - m stays -inf (S = 0: entropy 0).
//
// One pass over memory: a group of waves holds a chunk of a row in registers
// (32 logits per lane), so the maximum, the sums and the choice of the
// alternatives read it once.  A row of several chunks gets one workgroup per
// chunk (the split that fills the chip when there are few rows) and a second,
// small launch that joins the chunks' (m, S, T) and sorted alternatives in
// chunk order.
//
// The alternatives of a chunk: each of its NW waves finds the top/NW-th
// largest of its 64 lane maxima; the smallest of these has at least `top`
// logits at or above it, so only those -- one to two times `top` -- go to a
// list in LDS, and an entry's place is the number of larger entries.  Where
// that bound lets too many through (equal values, mostly masked rows) or a NaN
// is about, the exact bound is found: the top-th largest value bit by bit,
// counting over all logits of the chunk, then the index up to which the ones
// equal to it count.
#include "rowops_common.h"

namespace dlq {
namespace {

typedef unsigned long long u64;
constexpr int kLane = 32;   // logits per lane
constexpr int kList = 512;  // entries of the join's list
constexpr float kNan = __builtin_nanf("");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// What a wave leaves for the join.
struct Part {
  float m, S, T;
};

// f(m): sums S, T around m from a part's around its own p.m
__device__ __forceinline__ void add_part(Part p, float m, float& S, float& T) {
  if (p.m == -INFINITY && p.S == 0.f) return;  // nothing in it
  const float d = p.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
  S = __builtin_fmaf(p.S, f, S);
  if (f != 0.f) T = __builtin_fmaf(__builtin_fmaf(d, p.S, p.T), f, T);  // d may be -inf where f is 0
}

struct LogprobArgs {
  const void* x;
  int K, ldx, top, chunks;  // chunks per row
  const int* tokens;
  float* logprob;
  float* entropy;
  int* top_idx;
  float* top_logprob;
  u64* entries;  // [rows][chunks][top], chunks > 1
  Part* parts;   // [rows][chunks][4 waves]
};

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
__device__ __forceinline__ float key_value(unsigned k) {
  return k == 0xfffffffeu ? kNan : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 entry_key(float v, int j) { return (u64)value_key(v) << 32 | (unsigned)~j; }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float wave_max(float v) {
  return __int_as_float(wave_join(__float_as_int(v), __float_as_int(-INFINITY), [](int p, int q) {
    return __float_as_int(fmaxf(__int_as_float(p), __int_as_float(q)));
  }));
}
__device__ __forceinline__ float wave_sum(float v) {
  return __int_as_float(wave_join(__float_as_int(v), __float_as_int(-0.f), [](int p, int q) {
    return __float_as_int(__int_as_float(p) + __int_as_float(q));
  }));
}
__device__ __forceinline__ unsigned wave_min(unsigned v) {
  return (unsigned)wave_join((int)v, -1, [](int p, int q) { return (int)min((unsigned)p, (unsigned)q); });
}
__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const u64 w = __shfl_xor(v, o);
    v = w > v ? w : v;
  }
  return v;
}

// NW waves that work on one chunk: a whole workgroup (NW = 4), or one wave of
// it (NW = 1: the LDS of a wave needs no barrier, its accesses stay in order).
template <int NW>
__device__ __forceinline__ void group_sync() {
  if constexpr (NW > 1)
    __syncthreads();
  else
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
template <int NW, typename T, typename F>
__device__ __forceinline__ T group_join(T v, T* buf, F f) {  // v: already joined over the wave
  if constexpr (NW > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
    __syncthreads();
    v = buf[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = f(v, buf[i]);
  }
  return v;
}

// lp of a value whose distance to the row's maximum is d; ls = log S
__device__ __forceinline__ float log_prob(float d, float S, float ls) {
  return S == 0.f || (d == -INFINITY && S == S) ? -INFINITY : d - ls;
}

// The given token of a row and its logit: two loads, one behind the other, so
// they start before anything else.
struct Given {
  int token;
  float logit;
};
template <bool BF16>
__device__ __forceinline__ Given given_token(const LogprobArgs& a, int row) {
  Given g = {-1, 0.f};
  if (a.tokens) {
    g.token = a.tokens[row];
    if (g.token >= 0 && g.token < a.K) g.logit = logit<BF16>(a.x, (size_t)row * a.ldx + g.token);
  }
  return g;
}
// One lane of a row's group: the row's own numbers.  m: 0 for a row of -inf.
__device__ __forceinline__ void finish_row(const LogprobArgs& a, int row, Given g, float m, float S, float T) {
  const float ls = logf(S);
  if (a.tokens) a.logprob[row] = g.token < 0 ? 0.f : g.token >= a.K ? kNan : log_prob(g.logit - m, S, ls);
  if (a.entropy) a.entropy[row] = S == 0.f ? 0.f : ls - T / S;
}
__device__ __forceinline__ void put_alternative(const LogprobArgs& a, int row, int k, u64 key, float m, float S,
                                                float ls) {
  a.top_idx[(size_t)row * a.top + k] = (int)~(unsigned)key;
  a.top_logprob[(size_t)row * a.top + k] = log_prob(key_value((unsigned)(key >> 32)) - m, S, ls);
}

// Each of the n list entries that has fewer than `top` larger ones: put(place, key).
template <typename F>
__device__ __forceinline__ void place_entries(const u64* list, int n, int tid, int threads, int top, F put) {
  for (int i = tid; i < n; i += threads) {
    const u64 key = list[i];
    int larger = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) larger += list[j] > key;
    if (larger < top) put(larger, key);
  }
}

// A number that n of a wave's 64 keys reach, no larger than the nth largest and
// above the next smaller, bit by bit from above; 0 if fewer than n are not 0.
__device__ __forceinline__ unsigned wave_nth(unsigned key, int n) {
  unsigned bound = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const unsigned c = bound | 1u << b;
    const int reach = __popcll(__ballot(key >= c));
    if (reach >= n) bound = c;
    if (reach == n) break;
  }
  return bound;
}

template <bool BF16, int NW>
__global__ __launch_bounds__(256) void logprobs_chunk_kernel(const LogprobArgs a, int rows) {
  constexpr int G = 4 / NW, TPG = 64 * NW, NL = kLane, CHUNK = TPG * NL;
  constexpr int EPV = BF16 ? 8 : 4, NV = NL / EPV;  // logits per 16-byte load, loads per lane
  // entries of a group's list: with more, placing them costs more than the exact bound
  constexpr int kMany = NW == 1 ? 192 : 384;
  __shared__ u64 lists[G][kMany];
  __shared__ Part pbuf[4];
  __shared__ unsigned ubuf[4];
  __shared__ int counts[G];
  const int tid = threadIdx.x, g = tid / TPG, t = tid % TPG;
  const int row = G > 1 ? (int)blockIdx.x * G + g : (int)(blockIdx.x / (unsigned)a.chunks);
  const int chunk = G > 1 ? 0 : (int)(blockIdx.x % (unsigned)a.chunks);
  if (G > 1 && row >= rows) return;  // G > 1: no barriers below
  u64* list = lists[g];
  const int first = chunk * CHUNK, left = a.K - first;  // logits of this chunk on
  const size_t x0 = (size_t)row * a.ldx + first;
  if (t == 0) counts[g] = 0;

  const Given given = a.chunks == 1 ? given_token<BF16>(a, row) : Given{-1, 0.f};
  float x[NL];  // logit (v TPG + t) EPV + i of the chunk in x[v EPV + i]; those past K: -inf
  auto spread = [&](int v, v4i r) __attribute__((always_inline)) {
    if constexpr (BF16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[8 * v + 2 * i] = bf_lo((unsigned)r[i]);
        x[8 * v + 2 * i + 1] = bf_hi((unsigned)r[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * v + i] = __int_as_float(r[i]);
    }
  };
  const char* base = (const char*)a.x + x0 * (BF16 ? 2 : 4);
  if (left >= CHUNK) {
    v4i raw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = *(const v4i_any*)(base + (size_t)(v * TPG + t) * 16);
#pragma unroll
    for (int v = 0; v < NV; ++v) spread(v, raw[v]);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int j = (v * TPG + t) * EPV;
      if (j + EPV <= left) {
        spread(v, *(const v4i_any*)(base + (size_t)(v * TPG + t) * 16));
      } else {
        constexpr int SZ = BF16 ? 2 : 4;
        spread(v, load_tail16<false>(base + (size_t)(v * TPG + t) * 16, (left - j) * SZ, chunk ? 16 : j * SZ));
#pragma unroll
        for (int i = 0; i < EPV; ++i)
          if (j + i >= left) x[v * EPV + i] = -INFINITY;
      }
    }
  }

  float most[NL / 4], mine;  // of four logits each, of all (a NaN is never one)
#pragma unroll
  for (int q = 0; q < NL / 4; ++q) most[q] = max3(fmaxf(x[4 * q], x[4 * q + 1]), x[4 * q + 2], x[4 * q + 3]);
  mine = most[0];
#pragma unroll
  for (int q = 1; q + 1 < NL / 4; q += 2) mine = max3(mine, most[q], most[q + 1]);
  mine = fmaxf(mine, most[NL / 4 - 1]);

  // A wave's own sums, around its own maximum, in powers of two: the exponent
  // (x - m) log2(e) is one fma, x log2(e) - r with r = m log2(e) rounded once;
  // what that rounding shifts every term by is known and taken out of the sums.
  Part own;
  own.m = wave_max(mine);
  const float mw = own.m == -INFINITY ? 0.f : own.m;
  float S = 0.f, T = 0.f, shift = 0.f;
  if (__builtin_fabsf(mw) < 65536.f) {  // the shift stays below 2^-7
    const float r = mw * kLog2e;
    shift = __builtin_fmaf(mw, kLog2e, -r);
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      const float d = __builtin_fmaf(x[e], kLog2e, -r), p = __builtin_amdgcn_exp2f(d);
      S += p;
      T = __builtin_fmaf(p, fmaxf(d, -1e4f), T);  // a masked logit's 0 * -inf is 0 here; a NaN stays one in p
    }
  } else {
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      const float d = (x[e] - mw) * kLog2e, p = __builtin_amdgcn_exp2f(d);
      S += p;
      T = __builtin_fmaf(p, fmaxf(d, -1e4f), T);
    }
  }
  S = wave_sum(S);
  T = wave_sum(T);
  const float back = __builtin_amdgcn_exp2f(-shift);
  own.T = T = __builtin_fmaf(-shift, S, T) * (back * kLn2);
  own.S = S = S * back;
  const unsigned key = t * EPV < left ? value_key(mine) : 0u;
  unsigned bound = a.top ? wave_nth(key, (a.top + NW - 1) / NW) : 0u;
  float m = mw;
  bool plain = S != S;  // a NaN or +inf
  const bool whole = a.chunks == 1;
  if constexpr (NW > 1) {
    const int w = tid >> 6;
    if ((tid & 63) == 0) {
      if (whole)
        pbuf[w] = own;
      else
        a.parts[((size_t)row * a.chunks + chunk) * NW + w] = own;
      ubuf[w] = plain ? ~0u : bound;  // no bound is ~0
    }
    if (!whole && a.top == 0) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      plain |= ubuf[i] == ~0u;
      bound = min(bound, ubuf[i]);
    }
    if (whole) {
      float mg = pbuf[0].m;
#pragma unroll
      for (int i = 1; i < NW; ++i) mg = fmaxf(mg, pbuf[i].m);
      m = mg == -INFINITY ? 0.f : mg;
      S = T = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) add_part(pbuf[i], m, S, T);
    }
  }
  if (whole && t == 0) finish_row(a, row, given, m, S, T);
  if (a.top == 0) return;
  const float ls = whole ? logf(S) : 0.f;
  u64* out = whole ? nullptr : a.entries + ((size_t)row * a.chunks + chunk) * a.top;
  auto put = [&](int k, u64 key) {
    if (whole)
      put_alternative(a, row, k, key, m, S, ls);
    else
      out[k] = key;
  };

  int n = kMany + 1;
  if (!plain) {
    if (NW > 1 && bound == 0)  // a short last chunk leaves waves empty: one wave's top-th
      bound = group_join<NW>(wave_nth(key, a.top), ubuf, [](unsigned p, unsigned q) { return p > q ? p : q; });
    if (bound <= value_key(-INFINITY)) {
      // few logits, or few that are not masked: all of them, if they are not too many
      if (left <= kMany) {
#pragma unroll
        for (int e = 0; e < NL; ++e) {
          const int j = (e / EPV * TPG + t) * EPV + e % EPV;
          if (j < left) list[j] = entry_key(x[e], first + j);
        }
      }
      if (t == 0) counts[g] = left;
    } else {
      const float least = key_value(bound);  // those past K, as -inf, lie below
      if (mine >= least) {
#pragma unroll
        for (int q = 0; q < NL / 4; ++q)
          if (most[q] >= least) {
#pragma unroll
            for (int e = 4 * q; e < 4 * q + 4; ++e)
              if (x[e] >= least) {
                const int at = atomicAdd(&counts[g], 1);
                if (at < kMany) list[at] = entry_key(x[e], first + (e / EPV * TPG + t) * EPV + e % EPV);
              }
          }
      }
    }
    group_sync<NW>();
    n = counts[g];
  }
  if (n > kMany) {
    // keys in place of the logits, 0 past K: how many of the chunk reach c
    unsigned k[NL];
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      const int j = (e / EPV * TPG + t) * EPV + e % EPV;
      k[e] = j < left ? value_key(x[e]) : 0u;
    }
    const auto total = [&](int mine) {  // over the group, from the waves' counts
      if constexpr (NW > 1) mine = group_join<NW>(mine, (int*)ubuf, [](int p, int q) { return p + q; });
      return mine;
    };
    unsigned value = 0;
    int above = 0;  // keys above `value`
    bool exact = false;
#pragma unroll 1
    for (int b = 31; b >= 0 && !exact; --b) {
      const unsigned c = value | 1u << b;
      int reach = 0;
#pragma unroll
      for (int e = 0; e < NL; ++e) reach += __popcll(__ballot(k[e] >= c));
      reach = total(reach);
      if (reach >= a.top)
        value = c;
      else
        above = reach;
      exact = reach == a.top;
    }
    // of the keys equal to `value`, those at the lowest top - above places
    int place = CHUNK;  // all of them
    if (!exact) {
      place = 0;
#pragma unroll 1
      for (int b = CHUNK / 2; b > 0; b >>= 1) {
        int before = 0;
#pragma unroll
        for (int e = 0; e < NL; ++e)
          before += __popcll(__ballot(k[e] == value && (e / EPV * TPG + t) * EPV + e % EPV < place + b));
        if (total(before) <= a.top - above) place += b;
      }
    }
    group_sync<NW>();
    if (t == 0) counts[g] = 0;
    group_sync<NW>();
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      const int j = (e / EPV * TPG + t) * EPV + e % EPV;
      if (k[e] && (k[e] > value || (k[e] == value && j < place))) {
        const int at = atomicAdd(&counts[g], 1);
        if (at < kMany) list[at] = (u64)k[e] << 32 | (unsigned)~(first + j);
      }
    }
    group_sync<NW>();
    n = counts[g];
    if (n > kMany) n = kMany;
  }
  place_entries(list, n, t, TPG, a.top, put);
  // a last chunk shorter than `top`: empty entries behind its own
  for (int i = n + t; i < a.top; i += TPG) put(i, 0);
}

// The chunks of one row: a workgroup per row.
template <bool BF16>
__global__ __launch_bounds__(256) void logprobs_join_kernel(const LogprobArgs a) {
  constexpr int EARLY = 4;  // entries per thread that are loaded ahead
  __shared__ u64 list[kList];
  __shared__ u64 kbuf[4];
  __shared__ float fbuf[4];
  __shared__ v2f sbuf[4];
  __shared__ unsigned ubuf[4];
  __shared__ int count;
  const int tid = threadIdx.x, row = blockIdx.x;
  const int waves = 4 * a.chunks;
  const Part* parts = a.parts + (size_t)row * waves;
  const u64* entries = a.entries + (size_t)row * a.chunks * a.top;
  const int total = a.chunks * a.top;
  const Given given = given_token<BF16>(a, row);
  u64 early[EARLY];
#pragma unroll
  for (int r = 0; r < EARLY; ++r) early[r] = tid + 256 * r < total ? entries[tid + 256 * r] : 0;
  // A bound that at least `top` entries reach (the chunks' entries are sorted):
  // up to 64 chunks, the smallest of their (top/chunks)-th ones; more chunks,
  // from their first ones, as a chunk does it from its lanes' maxima.
  unsigned head = 0;
  const bool few = a.chunks <= 64;
  const int rank = few ? (a.top + a.chunks - 1) / a.chunks : 1;
  if (a.top)
    for (int c = tid; c < a.chunks; c += 256) {
      const unsigned e = (unsigned)(entries[(size_t)c * a.top + rank - 1] >> 32);
      head = e > head ? e : head;
    }
  if (tid == 0) count = 0;
  float mine = -INFINITY;
  for (int c = tid; c < waves; c += 256) mine = fmaxf(mine, parts[c].m);
  const float mg = group_join<4>(wave_max(mine), fbuf, [](float p, float q) { return fmaxf(p, q); });
  const float m = mg == -INFINITY ? 0.f : mg;
  float S = 0.f, T = 0.f;
  for (int c = tid; c < waves; c += 256) add_part(parts[c], m, S, T);
  const v2f st = group_join<4>(v2f{wave_sum(S), wave_sum(T)}, sbuf, [](v2f p, v2f q) { return p + q; });
  S = st[0];
  T = st[1];
  if (tid == 0) finish_row(a, row, given, m, S, T);
  if (a.top == 0) return;
  const float ls = logf(S);

  unsigned low = few ? (tid < a.chunks ? head : ~0u) : 0u;
  low = few ? wave_min(low) : wave_nth(head, (a.top + 3) / 4);
  const unsigned bound = group_join<4>(low, ubuf, [](unsigned p, unsigned q) { return p < q ? p : q; });
  const auto collect = [&](u64 e) {
    if (e && (unsigned)(e >> 32) >= bound) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) list[at] = e;
    }
  };
#pragma unroll
  for (int r = 0; r < EARLY; ++r) collect(early[r]);
  for (int i = tid + 256 * EARLY; i < total; i += 256) collect(entries[i]);
  __syncthreads();
  const int n = count;
  if (n <= kList) {
    place_entries(list, n, tid, 256, a.top, [&](int k, u64 key) { put_alternative(a, row, k, key, m, S, ls); });
    return;
  }
  u64 last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    u64 best = 0;
    for (int i = tid; i < total; i += 256) {
      const u64 e = entries[i];
      if (e < last && e > best) best = e;
    }
    last = group_join<4>(wave_max(best), kbuf, [](u64 p, u64 q) { return p > q ? p : q; });
    if (tid == 0) put_alternative(a, row, k, last, m, S, ls);
  }
}

// a row in one wave's registers, in a workgroup's, or in chunks of the latter
constexpr int kWaveChunk = 64 * kLane, kGroupChunk = 4 * kWaveChunk;
int chunks_of(int K) { return K <= kWaveChunk ? 1 : (K - 1) / kGroupChunk + 1; }

template <bool BF16>
hipError_t launch_logprobs(const LogprobArgs& a, int rows, hipStream_t s) {
  if (a.K <= kWaveChunk)
    hipLaunchKernelGGL((logprobs_chunk_kernel<BF16, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, rows);
  else
    hipLaunchKernelGGL((logprobs_chunk_kernel<BF16, 4>), dim3((unsigned)rows * (unsigned)a.chunks), dim3(256), 0, s, a,
                       rows);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.chunks == 1) return e;
  hipLaunchKernelGGL(logprobs_join_kernel<BF16>, dim3((unsigned)rows), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace dlq

using namespace dlq;

extern "C" {

size_t dlq_logprobs_workspace_bytes(int rows, int K, int top) {
  if (rows <= 0 || K <= 0 || top < 0) return 0;
  const size_t c = (size_t)chunks_of(K);
  return c == 1 ? 0 : (size_t)rows * c * (8 * (size_t)top + 4 * sizeof(Part));
}

int dlq_logprobs(const void* x, int x_type, int rows, int K, int ldx, const int32_t* tokens, int top, float* logprob,
                 float* entropy, int32_t* top_idx, float* top_logprob, void* workspace, size_t ws_bytes,
                 void* stream) {
  if (rows < 0 || K <= 0) return fail(DLQ_ERR_ARG, "logprobs: bad shape");
  if (x_type != DLQ_T_F32 && x_type != DLQ_T_BF16) return fail(DLQ_ERR_ARG, "logprobs: bad x_type");
  if (ldx < K) return fail(DLQ_ERR_ARG, "logprobs: row stride below K");
  if (top < 0 || top > 64 || top > K) return fail(DLQ_ERR_ARG, "logprobs: top outside 0..min(64, K)");
  if (rows == 0) return DLQ_OK;
  if (!x || !tokens != !logprob || (top && (!top_idx || !top_logprob)))
    return fail(DLQ_ERR_ARG, "logprobs: null pointer (tokens and logprob come together)");
  if ((uintptr_t)x % (x_type == DLQ_T_BF16 ? 2 : 4) ||
      ((uintptr_t)tokens | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_idx | (uintptr_t)top_logprob) % 4)
    return fail(DLQ_ERR_ARG, "logprobs: pointer not aligned to its element type");
  LogprobArgs a = {x, K, ldx, top, chunks_of(K), tokens, logprob, entropy, top_idx, top_logprob, nullptr, nullptr};
  if (!grid_fits((long long)rows * a.chunks, 256)) return fail(DLQ_ERR_ARG, "logprobs: too many rows");
  const size_t need = dlq_logprobs_workspace_bytes(rows, K, top);
  if (need && (!workspace || ws_bytes < need || (uintptr_t)workspace % 8))
    return fail(DLQ_ERR_ARG, "logprobs: workspace missing, too small or not 8-byte aligned");
  a.entries = (u64*)workspace;
  a.parts = (Part*)(a.entries + (size_t)rows * (a.chunks > 1 ? a.chunks : 0) * top);
  const hipError_t e = x_type == DLQ_T_BF16 ? launch_logprobs<true>(a, rows, (hipStream_t)stream)
                                            : launch_logprobs<false>(a, rows, (hipStream_t)stream);
  return e == hipSuccess ? DLQ_OK : fail(DLQ_ERR_LAUNCH, std::string("logprobs launch: ") + hipGetErrorString(e));
}

}  // extern "C"
