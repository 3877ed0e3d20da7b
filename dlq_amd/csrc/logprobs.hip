// logprobs.hip -- dlq_logprobs: for each row of logits the log probability of
// a given token, the entropy and the `top` largest with their log
// probabilities.
//   m = max x, S = sum e^(x-m), T = sum e^(x-m) (x-m):
//   lp[j] = x[j] - m - log S,  entropy = log S - T / S.
// A masked logit (-inf) adds nothing to S and T; a row of nothing else has
// m = -inf, taken as 0 so that x - m stays -inf (S = 0: entropy 0).
//
// One pass over memory, up to 32 logits per lane in registers, so the maximum,
// the sums and the alternatives' bound read a row once.  A row of up to 2048
// logits is one wave's and one of up to 8192 a workgroup's; both place the
// alternatives in the same launch.  A longer row gets one workgroup per chunk
// of 8192, what its registers hold, however many rows there are (so a few rows
// do not fill the chip: 4 x 100003 is 52 workgroups on 256 CUs).  Its waves
// work on their own, without a barrier: each leaves (m, S, T) and the largest
// logit of every four lanes (128 logits).  A second, small launch joins them in
// chunk order and reads again only those 128s that hold an alternative.
//
// What bounds it: memory for fp32; for bf16 the vector unit at the same time
// (per logit: unpack, half a maximum, fma, exp2, clamp, add, fma, of which the
// exp2 takes four times as long).  2048 x 65536 top 5: fp32 112 us, 4.8 TB/s;
// bf16 60 us, 4.5 TB/s (top 0: 105 and 52 us); alternatives placed by every
// chunk instead of by the join: bf16 79 us, top 64 128 instead of 75 us.
// 4 x 100003 fp32 top 20: 11.7 us, of which the first launch is 4 and the join,
// a chain of dependent steps, 8.  8192 x 8192 top 5: fp32 51 us, bf16 37 us.
// 16384 x 64 top 8: 12.5 us with 8 logits per lane, 21 with 32.
//
// The alternatives: some `top` of the lanes' (or groups') largest logits give a
// bound that as many logits reach, so only those at or above it -- one to two
// times `top` -- go to a list in LDS, and an entry's place is the number of
// larger entries.  Where that bound lets too many through (equal values, mostly
// masked rows) or a NaN is about, the row kernels find the exact one: the
// top-th largest value bit by bit, counting over all logits of the row, then
// the index up to which the ones equal to it count.
#include "rowops_common.h"

namespace dlq {
namespace {

typedef unsigned long long u64;
constexpr int kLane = 32;  // logits per lane, at most
// Up to so many alternatives, a workgroup's bound is the top-th of its 64 lane
// quads' largest (8192 x 8192 bf16 top 1: 33.9 us); for more, the smallest of
// the waves' (top / 4)-th of their 64 lanes' (36.9; equal at top 16).
constexpr int kFew = 16;
constexpr int kWaveChunk = 64 * kLane, kGroupChunk = 4 * kWaveChunk;
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
  float* heads;  // [rows][chunks][64], chunks > 1: the largest of a lane quad's logits
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
// fmaxf would first bring a signalling NaN to a quiet one; a row with a NaN
// takes none of its numbers from these.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
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
  unsigned bound = 0, bit = 1u << 31;
  int reach;
  do {  // on scalars: the vector unit has the logits to do
    const unsigned c = bound | bit;
    reach = __popcll(__ballot(key >= c));
    if (reach >= n) bound = c;
    bound = __builtin_amdgcn_readfirstlane(bound);
    bit >>= 1;
  } while (bit && reach != n);
  return bound;
}

// A lane's share of a chunk of TPG threads, from `base` on, `left` logits of the
// row: logit (v TPG + t) EPV + i in x[v EPV + i], -inf past the row's end.
// lead: the chunk's distance from the row's start.
template <bool BF16>
constexpr int kEpv = BF16 ? 8 : 4;  // logits per 16-byte load
template <bool BF16>
__device__ __forceinline__ void spread(v4i r, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      x[2 * i] = bf_lo((unsigned)r[i]);
      x[2 * i + 1] = bf_hi((unsigned)r[i]);
    } else {
      x[i] = __int_as_float(r[i]);
    }
  }
}
template <bool BF16, int TPG, int NL>
__device__ __forceinline__ void load_chunk(const char* base, int t, int left, bool lead, float (&x)[NL]) {
  constexpr int EPV = kEpv<BF16>, NV = NL / EPV, SZ = BF16 ? 2 : 4;
  if (left >= TPG * NL) {
    v4i raw[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = *(const v4i_any*)(base + (size_t)(v * TPG + t) * 16);
#pragma unroll
    for (int v = 0; v < NV; ++v) spread<BF16>(raw[v], x + EPV * v);
    return;
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int j = (v * TPG + t) * EPV;
    if (j + EPV <= left) {
      spread<BF16>(*(const v4i_any*)(base + (size_t)(v * TPG + t) * 16), x + EPV * v);
    } else {
      spread<BF16>(load_tail16<false>(base + (size_t)(v * TPG + t) * 16, (left - j) * SZ, lead ? 16 : j * SZ),
                   x + EPV * v);
#pragma unroll
      for (int i = 0; i < EPV; ++i)
        if (j + i >= left) x[v * EPV + i] = -INFINITY;
    }
  }
}
// The largest of each four logits, and of all (a NaN is never one).
template <int NL>
__device__ __forceinline__ float lane_max(const float (&x)[NL], float (&most)[NL / 4]) {
#pragma unroll
  for (int q = 0; q < NL / 4; ++q) most[q] = max3(max2(x[4 * q], x[4 * q + 1]), x[4 * q + 2], x[4 * q + 3]);
  float mine = most[0];
#pragma unroll
  for (int q = 1; q + 1 < NL / 4; q += 2) mine = max3(mine, most[q], most[q + 1]);
  return max2(mine, most[NL / 4 - 1]);
}
// A wave's own sums, around its own maximum m, in powers of two: the exponent
// (x - m) log2(e) is one fma, x log2(e) - r with r = m log2(e) rounded once;
// what that rounding shifts every term by is known and taken out of the sums.
template <int NL>
__device__ __forceinline__ Part wave_part(const float (&x)[NL], float m) {
  const float mw = m == -INFINITY ? 0.f : m;
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
  return {m, S * back, __builtin_fmaf(-shift, S, T) * (back * kLn2)};
}

// Whole rows: one per wave (NW = 1) or per workgroup (NW = 4).
template <bool BF16, int NW, int NL>
__global__ __launch_bounds__(256) void logprobs_row_kernel(const LogprobArgs a, int rows) {
  constexpr int G = 4 / NW, TPG = 64 * NW, EPV = kEpv<BF16>, CHUNK = TPG * NL;
  // entries of a group's list: with more, placing them costs more than the exact bound
  constexpr int kMany = NW == 1 ? 192 : 384;
  __shared__ u64 lists[G][kMany];
  __shared__ Part pbuf[4];
  __shared__ unsigned ubuf[4];
  __shared__ unsigned heads[64];
  __shared__ int counts[G];
  const int tid = threadIdx.x, g = tid / TPG, t = tid % TPG;
  const int row = (int)blockIdx.x * G + g;
  if (G > 1 && row >= rows) return;  // G > 1: no barriers below
  u64* list = lists[g];
  if (t == 0) counts[g] = 0;

  const Given given = given_token<BF16>(a, row);
  float x[NL], most[NL / 4];
  load_chunk<BF16, TPG>((const char*)a.x + (size_t)row * a.ldx * (BF16 ? 2 : 4), t, a.K, false, x);
  const float mine = lane_max(x, most);
  const float quad = quad_max(mine);
  const Part own = wave_part(x, wave_max_of_quads(quad));
  float S = own.S, T = own.T;
  const unsigned key = t * EPV < a.K ? value_key(mine) : 0u;
  const bool few = NW > 1 && a.top <= kFew;
  unsigned bound = a.top && !few ? wave_nth(key, (a.top + NW - 1) / NW) : 0u;
  float m = own.m == -INFINITY ? 0.f : own.m;
  bool plain = S != S;  // a NaN or +inf
  if constexpr (NW > 1) {
    const int w = tid >> 6;
    if ((tid & 63) == 0) {
      pbuf[w] = own;
      ubuf[w] = plain ? ~0u : bound;  // no bound is ~0
    }
    if (few && (tid & 3) == 3) heads[tid >> 2] = value_key(quad);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      plain |= ubuf[i] == ~0u;
      bound = min(bound, ubuf[i]);
    }
    if (few && a.top && !plain) bound = wave_nth(heads[tid & 63], a.top);
    float mg = pbuf[0].m;
#pragma unroll
    for (int i = 1; i < NW; ++i) mg = fmaxf(mg, pbuf[i].m);
    m = mg == -INFINITY ? 0.f : mg;
    S = T = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) add_part(pbuf[i], m, S, T);
  }
  if (t == 0) finish_row(a, row, given, m, S, T);
  if (a.top == 0) return;
  const float ls = logf(S);
  const auto put = [&](int k, u64 key) { put_alternative(a, row, k, key, m, S, ls); };

  int n = kMany + 1;
  if (!plain) {
    if (NW > 1 && bound <= value_key(-INFINITY))  // a short row leaves waves empty: one wave's top-th
      bound = group_join<NW>(wave_nth(key, a.top), ubuf, [](unsigned p, unsigned q) { return p > q ? p : q; });
    if (bound <= value_key(-INFINITY)) {
      // few logits, or few that are not masked: all of them, if they are not too many
      if (a.K <= kMany) {
#pragma unroll
        for (int e = 0; e < NL; ++e) {
          const int j = (e / EPV * TPG + t) * EPV + e % EPV;
          if (j < a.K) list[j] = entry_key(x[e], j);
        }
      }
      if (t == 0) counts[g] = a.K;
    } else {
      const float least = key_value(bound);  // those past the row's end, as -inf, lie below
      if (mine >= least) {
#pragma unroll
        for (int q = 0; q < NL / 4; ++q)
          if (most[q] >= least) {
#pragma unroll
            for (int e = 4 * q; e < 4 * q + 4; ++e)
              if (x[e] >= least) {
                const int at = atomicAdd(&counts[g], 1);
                if (at < kMany) list[at] = entry_key(x[e], (e / EPV * TPG + t) * EPV + e % EPV);
              }
          }
      }
    }
    group_sync<NW>();
    n = counts[g];
  }
  if (n > kMany) {
    // keys in place of the logits, 0 past the row's end: how many reach c
    unsigned k[NL];
#pragma unroll
    for (int e = 0; e < NL; ++e) {
      k[e] = t * EPV < a.K - (e / EPV * TPG * EPV + e % EPV) ? value_key(x[e]) : 0u;
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
          before += __popcll(__ballot(k[e] == value && t * EPV < place + b - (e / EPV * TPG * EPV + e % EPV)));
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
        if (at < kMany) list[at] = (u64)k[e] << 32 | (unsigned)~(j);
      }
    }
    group_sync<NW>();
    n = counts[g];
    if (n > kMany) n = kMany;
  }
  place_entries(list, n, t, TPG, a.top, put);
}

// One chunk of a long row per workgroup, its waves on their own: what the join
// needs of it.
template <bool BF16>
__global__ __launch_bounds__(256) void logprobs_chunk_kernel(const LogprobArgs a) {
  const int tid = threadIdx.x;
  const size_t at = blockIdx.x;  // row * chunks + chunk
  const int row = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks);
  const int first = chunk * kGroupChunk;
  float x[kLane], most[kLane / 4];
  const char* base = (const char*)a.x + ((size_t)row * a.ldx + first) * (BF16 ? 2 : 4);
  load_chunk<BF16, 256>(base, tid, a.K - first, true, x);  // a row's first chunk is a full one
  const float mine = lane_max(x, most), quad = quad_max(mine);
  float* head = a.heads + at * 64 + (tid >> 2);
  const bool last = a.top && (tid & 3) == 3;  // of a quad
  if (last) *head = quad;
  const Part own = wave_part(x, wave_max_of_quads(quad));
  if ((tid & 63) == 0) a.parts[at * 4 + (tid >> 6)] = own;
  if (a.top && own.S != own.S) {  // +inf, or a NaN, which is above all; read again, the registers are not kept for it
    unsigned k = value_key(mine);
#pragma unroll 1
    for (int e = 0; e < kLane; ++e) {
      const int j = (e / kEpv<BF16> * 256 + tid) * kEpv<BF16> + e % kEpv<BF16>;
      if (j < a.K - first) {
        const float v = logit<BF16>(base, j);
        if (v != v) k = value_key(v);
      }
    }
    k = max(k, (unsigned)__shfl_xor((int)k, 1));
    k = max(k, (unsigned)__shfl_xor((int)k, 2));
    if (last) *head = key_value(k);
  }
}

// A number that n and not many more of a wave's 256 keys reach; 0 if fewer than n are not 0.
__device__ __forceinline__ unsigned wave_nth(const unsigned (&key)[4], int n) {
  unsigned bound = 0, bit = 1u << 31;
  int reach;
  do {
    const unsigned c = bound | bit;
    reach = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) reach += __popcll(__ballot(key[i] >= c));
    if (reach >= n) bound = c;
    bound = __builtin_amdgcn_readfirstlane(bound);
    bit >>= 1;
  } while (bit && (reach < n || reach > n + n / 4 + 3));
  return bound;
}

// The chunks of one row: a workgroup per row.  Its alternatives: the largest of
// each group of logits is known, so that `top` of the 256 threads' largest ones
// give a bound that as many logits reach, and only the groups with a logit at
// or above it -- `top` or a few more -- are read again.  Where more logits reach
// it than the list holds, the list is cut to its `top` largest whenever it
// fills up; where many groups are at the bound (masked rows, equal logits), what
// equals it is taken in order, from the chunks that have a group at or above it
// (one below a larger logit of its group shows in no head).
template <bool BF16>
__global__ __launch_bounds__(256, 8) void logprobs_join_kernel(const LogprobArgs a) {
  constexpr int EPV = kEpv<BF16>, QUAD = 4 * kLane, SZ = BF16 ? 2 : 4;
  constexpr int STEP = 4;                    // heads, loads of a thread at a time
  constexpr int kFull = 256;                 // entries that a step may find in the list
  constexpr int kTied = 128;                 // groups at the bound that are not read one by one
  __shared__ u64 list[kFull + 1024];
  __shared__ u64 best[64];
  __shared__ int groups[256 * STEP];
  __shared__ Part pbuf[4];
  __shared__ __attribute__((aligned(16))) unsigned kbuf[256];
  __shared__ unsigned reached;
  __shared__ int count, found, start;
  const int tid = threadIdx.x, w = tid >> 6, row = blockIdx.x, top = a.top;
  const int waves = 4 * a.chunks, total = a.chunks * 64;
  const Part* parts = a.parts + (size_t)row * waves;
  const float* heads = a.heads + (size_t)row * total;
  const Given given = given_token<BF16>(a, row);
  float early[STEP];
  if (top) {
    unsigned head = 0;
#pragma unroll
    for (int r = 0; r < STEP; ++r) early[r] = tid + 256 * r < total ? heads[tid + 256 * r] : -INFINITY;
#pragma unroll
    for (int r = 0; r < STEP; ++r) head = max(head, value_key(early[r]));
    for (int i = tid + 256 * STEP; i < total; i += 256) head = max(head, value_key(heads[i]));
    kbuf[tid] = head;
  }
  Part own = {-INFINITY, 0.f, 0.f};
  if (w * 64 < waves) {
    for (int c = tid; c < waves; c += 256) own.m = fmaxf(own.m, parts[c].m);
    own.m = wave_max(own.m);
    const float m = own.m == -INFINITY ? 0.f : own.m;
    for (int c = tid; c < waves; c += 256) add_part(parts[c], m, own.S, own.T);
    own.S = wave_sum(own.S);
    own.T = wave_sum(own.T);
  }
  if ((tid & 63) == 0) pbuf[w] = own;
  if (tid == 0) {
    count = found = 0;
    start = 0x7fffffff;
  }
  __syncthreads();
  if (top && w == 0) {  // one wave for the bound, the next for the sums
    const v4u four = ((const v4u*)kbuf)[tid];
    const unsigned keys[4] = {four[0], four[1], four[2], four[3]};
    const unsigned b = wave_nth(keys, top);
    if (tid == 0) reached = b;
  }
  float m = fmaxf(fmaxf(pbuf[0].m, pbuf[1].m), fmaxf(pbuf[2].m, pbuf[3].m)), S = 0.f, T = 0.f;
  if (m == -INFINITY) m = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) add_part(pbuf[i], m, S, T);
  if (tid == 64) finish_row(a, row, given, m, S, T);
  if (top == 0) return;
  const float ls = logf(S);
  __syncthreads();

  // tied: the logits above v are listed here, of those equal to it the first
  // ones of the row behind the loop.  So are -inf, if fewer than top are more.
  const unsigned none = value_key(-INFINITY), v = max(reached, none);
  bool tied = v == none;
  u64 above = (u64)(v + tied) << 32;  // entries from here on count
  const size_t x0 = (size_t)row * a.ldx;
  for (int h0 = 0; h0 < total; h0 += 256 * STEP) {
    if (h0) {
      __syncthreads();
      if (tid == 0) found = 0;
      __syncthreads();
    }
    for (bool again = true; again;) {
#pragma unroll
      for (int r = 0; r < STEP; ++r) {
        const int h = h0 + 256 * r + tid;
        const unsigned k = h < total ? value_key(h0 ? heads[h] : early[r]) : 0u;
        if (k >= (unsigned)(above >> 32)) groups[atomicAdd(&found, 1)] = h;
        if (tied && k >= v) atomicMin(&start, h / 64);  // the first chunk that may hold one
      }
      __syncthreads();
      again = !tied && found > kTied && above == (u64)v << 32;
      if (again) {
        __syncthreads();
        if (tid == 0) found = 0;
        __syncthreads();
        tied = true;
        above = (u64)(v + 1) << 32;
      }
    }
    const int items = found * (QUAD / EPV);  // 16-byte loads
    for (int i0 = 0; i0 < items; i0 += 256 * STEP) {
      v4i raw[STEP];
      int at[STEP];
#pragma unroll
      for (int r = 0; r < STEP; ++r) {
        const int i = i0 + 256 * r + tid;
        at[r] = a.K;
        if (i < items) {
          const int h = groups[i / (QUAD / EPV)], o = i % (QUAD / EPV);
          const long long j = (long long)(h / 64) * kGroupChunk + ((o / 4) * 256 + h % 64 * 4 + o % 4) * EPV;
          if (j < a.K) at[r] = (int)j;
        }
        const char* p = (const char*)a.x + (x0 + at[r]) * SZ;
        raw[r] = v4i{};
        if (at[r] <= a.K - EPV)
          raw[r] = *(const v4i_any*)p;
        else if (at[r] < a.K)
          raw[r] = load_tail16<false>(p, (a.K - at[r]) * SZ, at[r] ? 16 : 0);
      }
#pragma unroll
      for (int u = 0; u < STEP * EPV / 4; ++u) {  // four logits per thread at a time
        const int r = u / (EPV / 4), e0 = u % (EPV / 4) * 4;
        if (i0 + 256 * r >= items) break;
        int n = 0;
        if (h0 || i0 || u) {  // the first step finds the list empty
          n = count;
          __syncthreads();
        }
        if (n > kFull) {
          place_entries(list, n, tid, 256, top, [&](int k, u64 key) { best[k] = key; });
          __syncthreads();
          if (tid < top) list[tid] = best[tid];
          above = best[top - 1] + 1;
          if (tid == 0) count = top;
          __syncthreads();
        }
        float l[EPV];
        spread<BF16>(raw[r], l);
#pragma unroll
        for (int e = e0; e < e0 + 4; ++e)
          if (at[r] < a.K - e) {
            const u64 key = entry_key(l[e], at[r] + e);
            if (key >= above) list[atomicAdd(&count, 1)] = key;
          }
        __syncthreads();
      }
    }
  }
  int have = count;
  __syncthreads();
  // the first step is most often enough, and leaves a short list
  long long j0 = v == none ? 0 : (long long)start * kGroupChunk;
  for (int step = 128; tied && have < top && j0 < a.K; j0 += step, step = 512 - (int)(j0 % 512)) {
    if (j0 % kGroupChunk == 0 &&
        !__syncthreads_or(value_key(heads[j0 / kGroupChunk * 64 + (tid & 63)]) >= v)) {
      step = kGroupChunk;
      continue;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const long long j = j0 + 256 * r + tid;
      const bool in = 256 * r + tid < step && j < a.K;
      const float l = in ? logit<BF16>(a.x, x0 + j) : 0.f;
      if (in && value_key(l) == v) list[atomicAdd(&count, 1)] = entry_key(l, (int)j);
    }
    __syncthreads();
    have = count;
    __syncthreads();
  }
  place_entries(list, count, tid, 256, top, [&](int k, u64 key) { put_alternative(a, row, k, key, m, S, ls); });
}

// a row in one wave's registers, in a workgroup's, or in chunks of the latter
int chunks_of(int K) { return K <= kWaveChunk ? 1 : (K - 1) / kGroupChunk + 1; }

template <bool BF16>
hipError_t launch_rows(const LogprobArgs& a, int rows, hipStream_t s) {
  const dim3 threads(256);
  if (a.chunks > 1) {
    hipLaunchKernelGGL(logprobs_chunk_kernel<BF16>, dim3((unsigned)rows * (unsigned)a.chunks), threads, 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(logprobs_join_kernel<BF16>, dim3((unsigned)rows), threads, 0, s, a);
  } else if (a.K <= kWaveChunk) {
    const dim3 grid((unsigned)((rows + 3) / 4));
    if (a.K <= kWaveChunk / 4)
      hipLaunchKernelGGL((logprobs_row_kernel<BF16, 1, kLane / 4>), grid, threads, 0, s, a, rows);
    else
      hipLaunchKernelGGL((logprobs_row_kernel<BF16, 1, kLane>), grid, threads, 0, s, a, rows);
  } else {
    const dim3 grid((unsigned)rows);
    if (a.K <= kGroupChunk / 2)
      hipLaunchKernelGGL((logprobs_row_kernel<BF16, 4, kLane / 2>), grid, threads, 0, s, a, rows);
    else
      hipLaunchKernelGGL((logprobs_row_kernel<BF16, 4, kLane>), grid, threads, 0, s, a, rows);
  }
  return hipGetLastError();
}

template <bool BF16>
hipError_t launch_logprobs(const LogprobArgs& all, int rows, hipStream_t s) {
  // rows of one launch, whose work-items are 32 bits: 2^22 workgroups at most
  const long long most = (1 << 22) / all.chunks;
  for (long long r = 0; r < rows; r += most) {
    LogprobArgs a = all;
    a.x = (const char*)a.x + (size_t)r * a.ldx * (BF16 ? 2 : 4);
    if (a.tokens) {
      a.tokens += r;
      a.logprob += r;
    }
    if (a.entropy) a.entropy += r;
    if (a.top) {
      a.top_idx += r * a.top;
      a.top_logprob += r * a.top;
    }
    if (a.chunks > 1) {
      a.heads += r * a.chunks * 64;
      a.parts += r * a.chunks * 4;
    }
    const hipError_t e = launch_rows<BF16>(a, (int)(rows - r < most ? rows - r : most), s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace
}  // namespace dlq

using namespace dlq;

extern "C" {

size_t dlq_logprobs_workspace_bytes(int rows, int K, int top) {
  if (rows <= 0 || K <= 0 || top < 0) return 0;
  const size_t c = (size_t)chunks_of(K);
  return c == 1 ? 0 : (size_t)rows * c * (4 * sizeof(Part) + (top ? 64 * sizeof(float) : 0));
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
  const int chunks = chunks_of(K);
  LogprobArgs a = {x, K, ldx, top, chunks, tokens, logprob, entropy, top_idx, top_logprob, nullptr, nullptr};
  const size_t need = dlq_logprobs_workspace_bytes(rows, K, top);
  if (need && (!workspace || ws_bytes < need || (uintptr_t)workspace % 8))
    return fail(DLQ_ERR_ARG, "logprobs: workspace missing, too small or not 8-byte aligned");
  a.parts = (Part*)workspace;
  a.heads = (float*)(a.parts + (size_t)rows * (chunks > 1 ? chunks : 0) * 4);
  const hipError_t e = x_type == DLQ_T_BF16 ? launch_logprobs<true>(a, rows, (hipStream_t)stream)
                                            : launch_logprobs<false>(a, rows, (hipStream_t)stream);
  return e == hipSuccess ? DLQ_OK : fail(DLQ_ERR_LAUNCH, std::string("logprobs launch: ") + hipGetErrorString(e));
}

}  // extern "C"
