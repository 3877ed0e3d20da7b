// rowops_common.h -- device helpers of the row operators (rowquant.hip,
// linear_act.hip, logprobs.hip): element types of rows, unaligned 16-byte
// loads, the products' epilogue.
#pragma once
#include "../../include/dlq.h"
#include "device_common.h"

namespace dlq {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
// 16 bytes at any address: gfx950 takes unaligned vector memory accesses, so
// this is one global_load_dwordx4 as well
typedef v4i v4i_any __attribute__((aligned(1)));

// 16 bytes of codes, those from `avail` on read as zero and not touched.
__device__ __forceinline__ v4i load_codes16(const int8_t* p, int avail) {
  if (avail >= 16) return *(const v4i_any*)p;
  v4i v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < avail) v[i >> 2] |= (int)((unsigned)(uint8_t)p[i] << (8 * (i & 3)));
  return v;
}

// value of a bf16 held in the low / high half of a dword
__device__ __forceinline__ float bf_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
// two values rounded to nearest even into one dword of bf16
__device__ __forceinline__ unsigned bf_pack(float a, float b) {
  const v2bf r = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, r);
}

// A wave's 64 values joined by f, the same in every lane: within rows of 16,
// then across them, by data-parallel primitives (no LDS round trips).  none:
// f(none, v) = v.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_move(int v, int none) {
  return __builtin_amdgcn_update_dpp(none, v, CTRL, ROWS, 0xf, false);
}
template <typename F>
__device__ __forceinline__ int wave_join(int v, int none, F f) {
  v = f(v, dpp_move<0x111, 0xf>(v, none));  // row_shr 1, 2, 4, 8
  v = f(v, dpp_move<0x112, 0xf>(v, none));
  v = f(v, dpp_move<0x114, 0xf>(v, none));
  v = f(v, dpp_move<0x118, 0xf>(v, none));
  v = f(v, dpp_move<0x142, 0xa>(v, none));  // row_bcast 15, 31
  v = f(v, dpp_move<0x143, 0xc>(v, none));
  return __builtin_amdgcn_readlane(v, 63);
}

// A launch's blocks * threads must stay below 2^32 (the dispatch packet's grid
// size is 32 bits of work-items).
inline bool grid_fits(long long blocks, int threads) { return blocks * threads < (1LL << 32); }

}  // namespace dlq
