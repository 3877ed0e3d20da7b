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
typedef v4i v4i_any __attribute__((aligned(1)));

// 16 bytes at any address: gfx950 takes them unaligned, but at a third of the
// rate where they do not start on a dword (12 x 16 x 11178 int8, rows 2 bytes
// off: 26.6 us, 8.8 on 8-byte rows).  ODD: the five dwords that hold them,
// moved into place when they are used; the fifth, where there are only four,
// is the fourth again, so that no dword is touched without a wanted byte in it.
template <bool ODD>
struct Raw16 {
  v4i d;
  __device__ __forceinline__ void load(const int8_t* p) { d = *(const v4i_any*)p; }
  __device__ __forceinline__ v4i get(const int8_t*) const { return d; }
};
template <>
struct Raw16<true> {
  typedef v4i v4i_dword __attribute__((aligned(4)));
  v4i d;
  int e;
  __device__ __forceinline__ void load(const int8_t* p) {
    const uintptr_t at = (uintptr_t)p;
    d = *(const v4i_dword*)(at & ~(uintptr_t)3);
    e = *(const int*)((at + 15) & ~(uintptr_t)3);
  }
  // p: any address that lies as the loaded one does to a dword
  __device__ __forceinline__ v4i get(const int8_t* p) const {
    const unsigned o = (unsigned)(uintptr_t)p & 3;
    return v4i{(int)__builtin_amdgcn_alignbyte((unsigned)d[1], (unsigned)d[0], o),
               (int)__builtin_amdgcn_alignbyte((unsigned)d[2], (unsigned)d[1], o),
               (int)__builtin_amdgcn_alignbyte((unsigned)d[3], (unsigned)d[2], o),
               (int)__builtin_amdgcn_alignbyte((unsigned)e, (unsigned)d[3], o)};
  }
};

// 16 bytes at p of which `avail` belong to the row, zeros in place of the
// others, which are not touched.  before: bytes of the row in front of p; with
// 16 up to the row's end the last 16 are loaded and moved down, one load
// instead of a chain of bytes.
template <bool ODD>
__device__ __forceinline__ v4i load_tail16(const void* at, int avail, int before) {
  const int8_t* p = (const int8_t*)at;
  v4i v = {0, 0, 0, 0};
  if (avail <= 0) return v;
  if (avail >= 16 || before + avail >= 16) {
    const int less = avail >= 16 ? 0 : 16 - avail;
    Raw16<ODD> r;
    r.load(p - less);
    v = r.get(p - less);
    if (less) {
      typedef unsigned long long u64;
      const u64 lo = (u64)(unsigned)v[1] << 32 | (unsigned)v[0], hi = (u64)(unsigned)v[3] << 32 | (unsigned)v[2];
      const int s = 8 * less;  // 8..120 bits
      const u64 l = s < 64 ? lo >> s | hi << (64 - s) : hi >> (s - 64), h = s < 64 ? hi >> s : 0;
      v = v4i{(int)l, (int)(l >> 32), (int)h, (int)(h >> 32)};
    }
    return v;
  }
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

// The same for floats, one instruction a step: lanes without a source keep what
// they have.  A step reads what the last one wrote after two wait states, the
// lane read after one.
#define DLQ_DPP_STEP(op, ctrl) "s_nop 1\n\t" op " %0, %0, %0 " ctrl " bank_mask:0xf\n\t"
#define DLQ_DPP_QUADS(op) DLQ_DPP_STEP(op, "row_shr:1 row_mask:0xf") DLQ_DPP_STEP(op, "row_shr:2 row_mask:0xf")
#define DLQ_DPP_REST(op)                                                                              \
  DLQ_DPP_STEP(op, "row_shr:4 row_mask:0xf")                                                          \
  DLQ_DPP_STEP(op, "row_shr:8 row_mask:0xf")                                                          \
  DLQ_DPP_STEP(op, "row_bcast:15 row_mask:0xa") DLQ_DPP_STEP(op, "row_bcast:31 row_mask:0xc") "s_nop 1"
__device__ __forceinline__ float lane63(float v) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_sum(float v) {
  asm(DLQ_DPP_QUADS("v_add_f32_dpp") DLQ_DPP_REST("v_add_f32_dpp") : "+v"(v));
  return lane63(v);
}
// Lane 4 i + 3: the largest of lanes 4 i to 4 i + 3 (a NaN is never one).
__device__ __forceinline__ float quad_max(float v) {
  asm(DLQ_DPP_QUADS("v_max_f32_dpp") "s_nop 1" : "+v"(v));
  return v;
}
__device__ __forceinline__ float wave_max_of_quads(float v) {
  asm(DLQ_DPP_REST("v_max_f32_dpp") : "+v"(v));
  return lane63(v);
}
__device__ __forceinline__ float wave_max(float v) { return wave_max_of_quads(quad_max(v)); }
#undef DLQ_DPP_STEP
#undef DLQ_DPP_QUADS
#undef DLQ_DPP_REST

// A launch's blocks * threads must stay below 2^32 (the dispatch packet's grid
// size is 32 bits of work-items).
inline bool grid_fits(long long blocks, int threads) { return blocks * threads < (1LL << 32); }

}  // namespace dlq
