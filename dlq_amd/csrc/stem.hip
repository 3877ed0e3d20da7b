// stem.hip -- fused ResNet-18 stem: input quantisation + conv1 7x7/s2/p3 (+BN,
// ReLU, requant) + maxpool 3x3/s2/p1 in one kernel.
//
// Replaces (RK = CUDA/resnet18-kernel-lab/cpp/fp32): the input upload
// (RK/runtime/infer_e2e.cu:255-256), conv2d_nchw_im2col_gemm for conv1
// (:259-270, im2col_nchw + sgemm_tiled), bn_launch + relu_forward (:272-280)
// and maxpool2d_3x3_s2p1_nchw (:282-293).  The 112x112x64 conv1 output never
// leaves the register file.
//
// K packing ("column units"): conv1's 147 taps per output pixel are 12 units
// of 16 bytes, unit (c, j) = channel c, input columns 2(ox-2+j) + {0, 1}
// (dx), the conv row's 8 input rows 2oy-3 .. 2oy+4 (kh): byte 2 kh + dx.
// K = 3 c x 4 j x 16 = 192 = 6 steps of v_mfma_i32_32x32x32_i8 (kw = 2j+dx-1
// = -1 and kh = 7 carry zero weights; the previous 2x2 space-to-depth packing
// padded 147 to 256).  Consecutive conv columns are consecutive units, so an
// A fragment is ONE aligned ds_read_b128 (2-byte-aligned 8-byte reads of a
// row-major plane cost 7x the LDS cycles: tools/probe/lds_tput_probe.hip).
// The units live in a ring of 8 conv-row buffers; the converter scatters
// each quantised input pixel pair (2 bytes, one ds_write_b16) into the 4
// conv rows whose window holds its input row.
//
// Input: every thread loads 2 pixels x 3 channels of one input row of one
// column unit (three 8-byte loads; a wave's 64 lanes are 16 units x 4 rows, so
// its ds_write_b16 scatter touches each bank at most twice) straight into
// registers, PD = 3 row quads ahead of their conversion.
//
// The two conv rows of a step are two interleaved MFMA chains sharing each
// k-step's weight fragment (6 weight reads per step instead of 12, two
// independent MFMAs in flight per wave): 72.8 -> 68.8 us per launch against
// one chain per row with PD = 4 (tools/ab.py, one box; PD = 3 alone 72.3).
//
// MFMA orientation D[px][oc]: A = 32 conv pixels of one conv row, B = the
// wave's 32 output channels (weight image in LDS, 208-byte rows).  A-row i is
// conv column c0 + pi(i) with pi chosen so that D register r of lane half h
// holds column c0 + 16h + r: each lane owns 16 consecutive columns of ONE
// channel, and the 3x3/s2 max pool runs on the int32 accumulators in
// registers (v_max3_i32).  Pooling before the epilogue is exact because the
// epilogue y = fma(acc, a, b) -> clamp -> rne is monotone non-decreasing in
// acc once a >= 0; channels with a < 0 have their weights (and a) negated at
// packing time (dlq_pack_stem_weights_s8).  Only the pooled values (1/4 of
// the conv outputs) are requantised.
//
// Work item = (image, band of pooled rows); workgroup = 8 waves = 4 column
// quarters x 2 channel tiles, two workgroups per CU.  Quarter q computes conv
// columns 28q-1 .. 28q+30 (32, of which 29 are used) and produces pooled
// columns 14q .. 14q+13.  A step computes conv rows 2p, 2p+1 and emits pooled
// row p.  Measured (tools/probe/stem_stamps.hip, N = 256, same box): 77.5 ->
// 72.5 us against the space-to-depth kernel; the launch runs at ~1.3 GHz
// (s_memtime cycles / wall), i.e. at the chip's power limit, not at HBM (the
// same input access pattern alone streams at 6.0 TB/s:
// tools/probe/stem_stream_probe.hip).
#include <cmath>
#include <type_traits>
#include <utility>

#include "device_common.h"

namespace dlq {
namespace {

constexpr int SNW = 8;                   // waves: 4 column quarters x 2 channel tiles
#ifndef DLQ_STEM_PD
#define DLQ_STEM_PD 3
#endif
constexpr int PD = DLQ_STEM_PD;          // row quads whose input loads are in flight ahead of the converter
constexpr int CR_SLOTS = 8;              // conv-row ring
constexpr int CR_PLANE = 128 * 16;       // one channel: units = super cols -4 .. 123 (0..3, 116..127 zero)
constexpr int CR_ROW = 3 * CR_PLANE + 64;  // conv-row slot pitch (+16 banks: adjacent slots' scatters on other banks)
constexpr int OFF_CR = 0;
constexpr int STG = 16 * 32;             // per wave: 16 pooled pixels x 32 channels of output staging
constexpr int OFF_STAGE = OFF_CR + CR_SLOTS * CR_ROW;
constexpr int WPITCH_S = 192 + 16;      // weight row pitch (13 units: a lane group's 16 rows on 16 bank quads)
constexpr int OFF_WST = OFF_STAGE + SNW * STG;  // the 64 x 192 B weight image
constexpr int LDS_STEM = OFF_WST + 64 * WPITCH_S;  // 66 KiB: two workgroups per CU
static_assert(2 * LDS_STEM <= 160 * 1024, "two workgroups per CU");
constexpr int SK = 192;                  // packed K per output channel
constexpr int kIntMin = (int)0x80000000;
typedef int v2i __attribute__((ext_vector_type(2)));

#ifdef DLQ_STAMPS
// timing-probe builds: per-wave cycle totals by section (no VM ops in the loop)
__device__ unsigned long long g_sstamps[512 * 8 * 8];
#define ST_DECL unsigned long long st_acc[6] = {0, 0, 0, 0, 0, 0}, st_prev = __builtin_amdgcn_s_memtime()
#define ST(k)                                                       \
  do {                                                              \
    const unsigned long long st_now = __builtin_amdgcn_s_memtime(); \
    st_acc[k] += st_now - st_prev;                                  \
    st_prev = st_now;                                               \
  } while (0)
#define ST_STORE()                                                                                       \
  do {                                                                                                   \
    if ((threadIdx.x & 63) == 0 && blockIdx.x < 512)                                                     \
      for (int q_ = 0; q_ < 6; ++q_) g_sstamps[(blockIdx.x * 8 + (threadIdx.x >> 6)) * 8 + q_] = st_acc[q_]; \
  } while (0)
#else
#define ST_DECL
#define ST(k) \
  do {        \
  } while (0)
#define ST_STORE() \
  do {             \
  } while (0)
#endif

struct StemArgs {
  const float* x;      // [N][3][224][224]
  const int8_t* w;     // [64 oc][6 k-steps][2 lane halves][16 B] (dlq_pack_stem_weights_s8)
  const float* alpha;  // [64] |alpha| (packed), output-grid units
  const float* beta;   // [64]
  int8_t* y;           // [N][56][56][64]
  float inv_s;         // 1 / input scale
  int N, nb, R;        // batch, bands per image, pooled rows per band
  Prefetch pf;         // the next launch's weights (engine forwards)
};


__device__ __forceinline__ int max3i(int a, int b, int c) {
  return __builtin_elementwise_max(__builtin_elementwise_max(a, b), c);
}

// F8: the fp8 path: the input is quantised to e4m3, the 6 i8
// k-steps become 3 v_mfma_f32_32x32x64_f8f6f4 (k-steps 2i, 2i+1 as the two
// halves of each 32-byte fragment, A and B alike), the pool runs on the fp32
// accumulators (max is exact; the e4m3 epilogue is monotone once alpha >= 0:
// dlq_pack_stem_weights_f8 flips the sign bits of the rows with alpha < 0).
template <bool F8>
__global__ __launch_bounds__(SNW * 64, 4) void stem_fused_kernel(StemArgs a) {
  using Acc = typename std::conditional<F8, v16f, v16i>::type;
  using Pv = typename std::conditional<F8, float, int>::type;
  __shared__ __attribute__((aligned(16))) int8_t lds[LDS_STEM];
  const unsigned lds32 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, lh = lane >> 5;
  const int ot = wave & 1, q = wave >> 1;  // channel tile, column quarter
  const int nitems = a.N * a.nb;

  // The weight image in LDS (B fragments re-read per conv row: the
  // registers hold the input loads in flight) and the channel's epilogue
  // constants.
  for (int i = tid; i < 64 * 12; i += SNW * 64)
    *(v4i*)(lds + OFF_WST + (i / 12) * WPITCH_S + (i % 12) * 16) = *(const v4i*)(a.w + i * 16);
  const unsigned w_row = lds32 + OFF_WST + (ot * 32 + lr) * WPITCH_S + lh * 16;
  const float al = a.alpha[ot * 32 + lr], be = a.beta[ot * 32 + lr];
  // the ring starts zeroed: a kh = 7 byte row (zero weight) read before its
  // first write must hold a valid code (an e4m3 NaN times 0 is NaN)
  for (int i = tid; i < CR_SLOTS * CR_ROW / 16; i += SNW * 64) *(v4i*)(lds + OFF_CR + i * 16) = v4i{0, 0, 0, 0};
  __syncthreads();
  // A-row permutation: lane row i -> conv column offset pi(i) (D reg r of half h = column 16h + r)
  const int pi = ((lr >> 3) << 2) + (lr & 3) + 16 * ((lr >> 2) & 1);
  const int ox = 28 * q - 1 + pi;  // this lane's conv column
  // k-step t, lane half lh reads unit (c = t >> 1, j = 2 (t & 1) + lh): super col ox - 2 + j
  const unsigned a_col = lds32 + OFF_CR + (unsigned)(ox + 2 + lh) * 16;
  int8_t* stg = lds + OFF_STAGE + wave * STG;

  // converter lanes: (input row r of the quad, unit u): a wave = 16 units x 4 rows
  const int cv_r = (tid >> 4) & 3, cv_u = (tid & 15) + 16 * (tid >> 6);

  ST_DECL;
  int item0, n_my;
  xcd_chunk(nitems, item0, n_my);
  for (int li = 0; li < n_my; ++li) {
    const int item = xcd_item(item0, li);
    const int n = item / a.nb, band = item - n * a.nb;
    const int py0 = band * a.R, py1 = min(56, py0 + a.R);
    if (py0 >= py1) continue;
    // quad k = input rows iy0 + 4k .. + 3 (iy0 = 4 py0 - 5); step t converts
    // quad t + 3 = rows 4p + 7 .. 4p + 10 (conv rows 2p + 2 .. 2p + 6) while it
    // reads conv rows 2p, 2p + 1, whose last rows came with quad t + 2
    const int iy0 = 4 * py0 - 5;
    const float* img = a.x + (size_t)n * 3 * 224 * 224;

    using F2 = float __attribute__((ext_vector_type(2)));
    F2 raw[PD + 1][3];
    // Branch-free input loads: one buffer resource per channel plane of the
    // image, and pixels outside it (padding rows and columns) take an
    // offset past the plane, which the buffer's range check returns as
    // zeros.  Without the branch the compiler's vmcnt accounting stays
    // exact, so a step waits only for the quad it converts (the branchy
    // form waited for every load in flight, vmcnt(0)): 64.7 -> 62.6 us per
    // launch (tools/ab.py, one box, bit-identical).
    __amdgpu_buffer_rsrc_t rs[3];
#pragma unroll
    for (int c = 0; c < 3; ++c)
      rs[c] = __builtin_amdgcn_make_buffer_rsrc((void*)(img + (size_t)c * 224 * 224), 0, 224 * 224 * 4, 0x00020000);
    const bool col_ok = (unsigned)(cv_u - 4) < 112u;
    auto load_quad = [&](int k, F2 (&r)[3]) {
      const int iy = iy0 + 4 * k + cv_r, sc = cv_u - 4;
      const int off = ((unsigned)iy < 224u && col_ok) ? (iy * 224 + 2 * sc) * 4 : 0x40000000;
#pragma unroll
      for (int c = 0; c < 3; ++c) r[c] = __builtin_bit_cast(F2, __builtin_amdgcn_raw_buffer_load_b64(rs[c], off, 0, 0));
    };
    // Quantise quad k and scatter each pixel pair into the 4 conv rows oy whose
    // window 2oy-3 .. 2oy+4 holds its input row iy (kh = iy - 2oy + 3).  Rows
    // of conv rows outside the band land in slots that the band's own rows
    // overwrite before they are read (tools: the stem parity tests at 1..14
    // bands per image).
    // Scatter addresses (int8): quad k's first conv row is ob0 + 2k (ob0 =
    // the lane's first conv row of quad 0), so its 4 rows' slots are
    // (ob0 + j) & 7 with j = (2k + e) & 7 -- static in the unrolled step
    // loop -- and kh = c0 - 2e with c0 in {6, 7} (the lane's row parity):
    // one table of 8 slot bases per lane and item, every scatter address an
    // immediate offset from one of them (per step ~120 -> ~100 VALU; stem
    // ~64.1 -> ~62.9 us per launch, medians of five A/B rounds on one box).
    const int ob0 = (iy0 + cv_r - 3) >> 1, kh0 = iy0 + cv_r - 2 * ob0 + 3;
    int sa[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sa[j] = OFF_CR + ((ob0 + j) & (CR_SLOTS - 1)) * CR_ROW + cv_u * 16 + 2 * kh0 - 12;
    auto convert_quad = [&](int k, const F2 (&r)[3], auto jc) {  // jc = (2k) & 7
      const int iy = iy0 + 4 * k + cv_r;
      unsigned v[3];
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        if constexpr (F8) {  // e4m3 codes of the two pixels; padding quantises to +0
          const float c0 = __builtin_amdgcn_fmed3f(r[c][0] * a.inv_s, -448.f, 448.f) + 0.0f;
          const float c1 = __builtin_amdgcn_fmed3f(r[c][1] * a.inv_s, -448.f, 448.f) + 0.0f;
          v[c] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c0, c1, 0, false);
        } else {  // clamp(x/s) + 1.5*2^23 -> rne'd int8 in the low byte
          const unsigned u0 = __float_as_uint(__builtin_amdgcn_fmed3f(r[c][0] * a.inv_s, -127.f, 127.f) + 12582912.0f);
          const unsigned u1 = __float_as_uint(__builtin_amdgcn_fmed3f(r[c][1] * a.inv_s, -127.f, 127.f) + 12582912.0f);
          v[c] = __builtin_amdgcn_perm(u1, u0, 0x0c0c0400u);
        }
      }
      if constexpr (!F8) {  // the 4 conv rows' slots from the item's table: immediates only
        constexpr int J = decltype(jc)::value;
        static_assert(PD == 3, "jc = (2k) & 7 is static because the step loop is unrolled by 4");
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int c = 0; c < 3; ++c)
            *(unsigned short*)(lds + sa[(J + e) & 7] + (12 - 4 * e + c * CR_PLANE)) = (unsigned short)v[c];
        }
        return;
      }
      const int oyb = (iy - 3) >> 1;  // ceil((iy - 4) / 2): the first of the 4 conv rows
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int oyc = oyb + e, kh = iy - 2 * oyc + 3;
        int8_t* dst = lds + OFF_CR + (oyc & (CR_SLOTS - 1)) * CR_ROW + cv_u * 16 + 2 * kh;
#pragma unroll
        for (int c = 0; c < 3; ++c) *(unsigned short*)(dst + c * CR_PLANE) = (unsigned short)v[c];
      }
    };
    // One conv row (global row oy): the wave's 32 px x 64 oc (two tiles), 6
    // k-steps; A fragments stream through a 3-deep ring of untracked
    // ds_read_b128 (inline asm: completion by explicit lgkmcnt waits).
    auto conv_row = [&](int oy) {
      Acc c0 = Acc{0};
      const unsigned ra = a_col + (oy & (CR_SLOTS - 1)) * CR_ROW;
      v4i fa[3];
      v4i fw[3];
#define STEM_RD(t)                                                                                               \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa[(t) % 3]) : "v"(ra), "n"(((t) >> 1) * CR_PLANE + ((t) & 1) * 32) \
               : "memory");                                                                                      \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fw[(t) % 3]) : "v"(w_row), "n"(32 * (t)) : "memory")
#define STEM_WAIT(t, n) asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(fa[(t) % 3]), "+v"(fw[(t) % 3]) : "n"(n) : "memory")
      if constexpr (F8) {  // k-steps 2i, 2i+1 = the two halves of one 64-deep fp8 MFMA
#define STEM_K8(i)                                                                                      \
  c0 = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(cat8(fa[(2 * (i)) % 3], fa[(2 * (i) + 1) % 3]),  \
                                                       cat8(fw[(2 * (i)) % 3], fw[(2 * (i) + 1) % 3]), c0, 0, 0, 0, 0, 0, 0)
        STEM_RD(0);
        STEM_RD(1);
        STEM_WAIT(0, 2);
        STEM_WAIT(1, 0);
        STEM_K8(0);
        STEM_RD(2);
        STEM_RD(3);
        STEM_WAIT(2, 2);
        STEM_WAIT(3, 0);
        STEM_K8(1);
        STEM_RD(4);
        STEM_RD(5);
        STEM_WAIT(4, 2);
        STEM_WAIT(5, 0);
        STEM_K8(2);
#undef STEM_K8
      } else {
#define STEM_K(t) c0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[(t) % 3], fw[(t) % 3], c0, 0, 0, 0)
        STEM_RD(0);
        STEM_RD(1);
        STEM_WAIT(0, 2);
        STEM_K(0);
        STEM_RD(2);
        STEM_WAIT(1, 2);
        STEM_K(1);
        STEM_RD(3);
        STEM_WAIT(2, 2);
        STEM_K(2);
        STEM_RD(4);
        STEM_WAIT(3, 2);
        STEM_K(3);
        STEM_RD(5);
        STEM_WAIT(4, 2);
        STEM_K(4);
        STEM_WAIT(5, 0);
        STEM_K(5);
#undef STEM_K
      }
#undef STEM_RD
#undef STEM_WAIT
      return c0;
    };
    // int8: conv rows oy, oy + 1 as two interleaved chains sharing each
    // k-step's weight fragment (6 weight reads instead of 12 per step, and two
    // independent MFMAs in flight per wave)
    auto conv_rows2 = [&](int oy, Acc& c0, Acc& c1) {
      c0 = Acc{0};
      c1 = Acc{0};
      const unsigned ra0 = a_col + (oy & (CR_SLOTS - 1)) * CR_ROW, ra1 = a_col + ((oy + 1) & (CR_SLOTS - 1)) * CR_ROW;
      v4i fa0[3], fa1[3], fw[3];
#define STEM_RD2(t)                                                                                               \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa0[(t) % 3]) : "v"(ra0), "n"(((t) >> 1) * CR_PLANE + ((t) & 1) * 32) \
               : "memory");                                                                                      \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa1[(t) % 3]) : "v"(ra1), "n"(((t) >> 1) * CR_PLANE + ((t) & 1) * 32) \
               : "memory");                                                                                      \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fw[(t) % 3]) : "v"(w_row), "n"(32 * (t)) : "memory")
#define STEM_WAIT2(t, n)                                                                                        \
  asm volatile("s_waitcnt lgkmcnt(%3)" : "+v"(fa0[(t) % 3]), "+v"(fa1[(t) % 3]), "+v"(fw[(t) % 3]) : "n"(n) : "memory")
#define STEM_K2(t)                                                              \
  c0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa0[(t) % 3], fw[(t) % 3], c0, 0, 0, 0); \
  c1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa1[(t) % 3], fw[(t) % 3], c1, 0, 0, 0)
      STEM_RD2(0);
      STEM_RD2(1);
      STEM_WAIT2(0, 3);
      STEM_K2(0);
      STEM_RD2(2);
      STEM_WAIT2(1, 3);
      STEM_K2(1);
      STEM_RD2(3);
      STEM_WAIT2(2, 3);
      STEM_K2(2);
      STEM_RD2(4);
      STEM_WAIT2(3, 3);
      STEM_K2(3);
      STEM_RD2(5);
      STEM_WAIT2(4, 3);
      STEM_K2(4);
      STEM_WAIT2(5, 0);
      STEM_K2(5);
#undef STEM_RD2
#undef STEM_WAIT2
#undef STEM_K2
    };
    auto mx3 = [](Pv x, Pv y, Pv z) -> Pv {
      if constexpr (F8)
        return __builtin_fmaxf(__builtin_fmaxf(x, y), z);
      else
        return max3i(x, y, z);
    };
    const Pv kLow = F8 ? (Pv)-INFINITY : (Pv)kIntMin;
    // Horizontal 3-max of a conv row, H[m] = max(local cols 2m, 2m+1, 2m+2):
    // half 0 takes column 16 from half 1; quarter 0's column 0 is conv column
    // -1 (pool padding).  Half 1's H[6], H[7] and half 0's beyond m=7 are unused.
    auto hpool = [&](const Acc& c, Pv (&H)[8]) {
      unsigned x0 = __builtin_bit_cast(unsigned, c[0]), c16 = x0;
      swap32(x0, c16);  // lanes 0-31: c16 = lanes 32-63's c[0]
      const Pv c0v = (q == 0 && lh == 0) ? kLow : c[0];
      H[0] = mx3(c0v, c[1], c[2]);
#pragma unroll
      for (int m = 1; m < 7; ++m) H[m] = mx3(c[2 * m], c[2 * m + 1], c[2 * m + 2]);
      H[7] = mx3(c[14], c[15], __builtin_bit_cast(Pv, c16));
    };

    // ---- prologue: quads 0..2 converted (input rows 4py0-5 .. 4py0+6),
    // quads 3 .. 2+PD loaded (quad k in register set k % (PD + 1)); H of
    // conv row 2py0-1.
    static_assert(PD >= 2, "the prologue converts quads 0..2 from their own sets");
#pragma unroll
    for (int k = 0; k <= PD; ++k) load_quad(k, raw[k]);
    convert_quad(0, raw[0], std::integral_constant<int, 0>{});
    load_quad(PD + 1, raw[0]);
    convert_quad(1, raw[1], std::integral_constant<int, 2>{});
    load_quad(PD + 2, raw[1]);
    convert_quad(2, raw[2], std::integral_constant<int, 4>{});
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): ring rows written (loads stay in flight)
    __builtin_amdgcn_s_barrier();
    Pv Hp[8];
    if (py0 == 0) {
#pragma unroll
      for (int m = 0; m < 8; ++m) Hp[m] = kLow;  // conv row -1: pool padding
    } else {
      hpool(conv_row(2 * py0 - 1), Hp);
    }

    // The staged output of step p is read back and stored during step p+1
    // (after its convert), so the LDS round trip and the store issue overlap
    // the next step instead of closing this one.
    const int pxl = lane >> 1, hf = lane & 1;
    // int8 staging [32 oc][16 px]: lane (oc lr, half lh) writes its 8 pooled
    // bytes as ONE ds_write_b64 (the 8-byte halves of rows with oc bit 3 set
    // swapped, so a 16-lane store group covers all 32 banks); the store side
    // reads it back transposed with two ds_read_b64_tr_b8 (16-lane group g,
    // lane i = 2r + h: row 8g' + r, px half h; lane i receives px i's 8 oc of
    // rows 8g' .. 8g' + 7), g' = g then g ^ 1, so the lanes of groups 0 and 2
    // hold 16 consecutive channels of px i.  Against 8 ds_write_b8 + one
    // ds_read_b128: ~26 fewer LDS cycles per wave and step (the stem's LDS
    // traffic -- 18 fragment reads, 12 scatter writes per wave and step --
    // rivals its MFMA time): 62.9-63.8 -> 61.7-62.0 us per launch, five A/B
    // rounds on one box, bit-identical.
    const int tg = lane >> 4, ti = lane & 15;
    const int8_t* tr1 = stg + (8 * tg + (ti >> 1)) * 16 + 8 * ((ti & 1) ^ (tg & 1));
    const int8_t* tr2 = stg + (8 * (tg ^ 1) + (ti >> 1)) * 16 + 8 * ((ti & 1) ^ ((tg ^ 1) & 1));
    auto store_row = [&](int p) {
      if constexpr (!F8) {
        const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)tr1);
        const v2i r2 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)tr2);
        if ((tg & 1) == 0 && ti < 14)
          *(v4i*)(a.y + (((size_t)n * 56 + p) * 56 + 14 * q + ti) * 64 + ot * 32 + 8 * tg) = v4i{r1[0], r1[1], r2[0], r2[1]};
        return;
      }
      const v4i o = *(const v4i*)(stg + pxl * 32 + hf * 16);
      if (lane < 28) *(v4i*)(a.y + (((size_t)n * 56 + p) * 56 + 14 * q + pxl) * 64 + ot * 32 + hf * 16) = o;
    };
    // step t (pooled row p = py0 + t): quad t+3 (register set (t+3) % (PD+1))
    // is quantised for the next step, quad t+3+PD is loaded into the set quad
    // t+2 freed, conv rows 2p and 2p+1 are computed and pooled.
    auto step = [&](int t, auto setc) {
      constexpr int S = decltype(setc)::value;  // == t % (PD + 1)
      const int p = py0 + t;
      ST(5);
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): last step's ring rows and staging
      __builtin_amdgcn_s_barrier();
      ST(0);
      auto ingest = [&]() {
        convert_quad(t + 3, raw[(S + 3) % (PD + 1)], std::integral_constant<int, (2 * S + 6) & 7>{});
        ST(1);
        if (t > 0) store_row(p - 1);
        load_quad(t + 3 + PD, raw[(S + 2) % (PD + 1)]);
        ST(2);
      };

      Pv He[8], Ho[8];
#ifndef DLQ_STEM_SERIAL
      if constexpr (!F8) {
        // The convert writes conv rows 2p+2 .. 2p+6 and the MFMAs read rows
        // 2p, 2p+1 (other ring slots), so within a step either may go first:
        // the MFMAs go first and the convert's VALU runs while they drain
        // (65.1-65.9 -> 63.7-64.0 us per launch, tools/ab.py, one box,
        // bit-identical; MFMAs first in waves 4-7 only: 66.8-67.5).
        Acc ce, co;
        conv_rows2(2 * p, ce, co);
        ingest();
        hpool(ce, He);
        hpool(co, Ho);
      } else
#endif
      {
        ingest();
        hpool(conv_row(2 * p), He);
        hpool(conv_row(2 * p + 1), Ho);
      }
      ST(3);
      // vertical max, epilogue on the pooled values, bytes -> staging
      if constexpr (!F8) {  // rne(clamp(y, 0, 127)) as v_cvt_pk_u8_f32(min(y, 127)) (quant4_relu), 8 bytes -> [oc][px]
        unsigned w[2] = {0u, 0u};
#pragma unroll
        for (int m = 0; m < 8; ++m) {
          const Pv v = mx3(Hp[m], He[m], Ho[m]);
          Hp[m] = Ho[m];
          const float y = __builtin_fmaf((float)v, al, be);
          w[m >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(__builtin_fminf(y, 127.f), m & 3, w[m >> 2]);
        }
        *(v2i*)(stg + lr * 16 + 8 * (lh ^ ((lr >> 3) & 1))) = v2i{(int)w[0], (int)w[1]};
        ST(4);
        return;
      }
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const Pv v = mx3(Hp[m], He[m], Ho[m]);
        Hp[m] = Ho[m];
        const float y = __builtin_fmaf((float)v, al, be);
        if constexpr (F8) {
          stg[(m + 8 * lh) * 32 + lr] = (int8_t)enc4_f8(y, 0.f, 0.f, 0.f, 0.f);
        } else {
          const unsigned u = __float_as_uint(__builtin_amdgcn_fmed3f(y, 0.f, 127.f) + 12582912.0f);
          stg[(m + 8 * lh) * 32 + lr] = (int8_t)u;
        }
      }
      // 14 pooled columns x 32 channels = 28 x 16 B, staged in LDS (written by
      // this wave: LDS is in order); stored during the next step
      ST(4);
    };
    const int nsteps = py1 - py0;
    static_assert(PD == 3 || PD == 4, "the step loop below is unrolled by PD + 1");
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    using I4 = std::integral_constant<int, 4>;
    int t = 0;
    for (; t + PD + 1 <= nsteps; t += PD + 1) {
      step(t, I0{});
      step(t + 1, I1{});
      step(t + 2, I2{});
      step(t + 3, I3{});
      if constexpr (PD == 4) step(t + 4, I4{});
    }
    if (t < nsteps) step(t, I0{});
    if (t + 1 < nsteps) step(t + 1, I1{});
    if (t + 2 < nsteps) step(t + 2, I2{});
    if constexpr (PD == 4) {
      if (t + 3 < nsteps) step(t + 3, I3{});
    }
    if (py1 > py0) store_row(py1 - 1);
    wait_vm0();
    __syncthreads();  // ring reuse by the next item
  }
  ST_STORE();
}

// int8 stem, one wave per column quarter computing BOTH channel tiles
// (stem2_kernel): 4 waves per workgroup, two workgroups per CU (two waves
// per SIMD, 256 VGPRs each).  Against stem_fused_kernel<false> (8 waves, one
// channel tile each): the wave keeps all 64 channels' weights in registers
// (48 VGPRs: no weight fragment reads) and reads each conv row's A fragment
// once for both tiles -- 12 instead of 36 ds_read_b128 per 24 MFMAs -- and
// its converter lanes take an input row PAIR (2oy-odd, +1), whose bytes of
// a conv row are 4 contiguous bytes (kh, kh + 1): one ds_write_b32 per conv
// row and channel where two lanes issued a ds_write_b16 each.  Same item
// walk, ring, band logic, pooling and numerics as stem_fused_kernel:
// 61.5-62.8 -> 59.2-60.6 us per launch (four A/B rounds, one box, round 4),
// bit-identical.  Its loop once went from ~197 to 160 non-MFMA VALU per step
// (24 MFMAs) -- packed multiply / add in the input conversion, packed fma in
// the requantisation, the pool pad as a min against a per-lane bound, one
// permlane32 swap without copies, no result selects in the store -- with the
// time unchanged (57.02 vs 57.09 us, profiles/r06_ab_stem_valu.txt): the stem
// is not bound by VALU issue.  Built without packed fp32 instructions the pairs
// are two scalar instructions each again, and the forward's time is what it was.
constexpr int S2W = 4;                          // waves: one per column quarter
constexpr int STG2 = 64 * 16;                   // per wave: [64 oc][16 px] bytes
constexpr int OFF_STAGE2 = OFF_CR + CR_SLOTS * CR_ROW;
constexpr int OFF_PF2 = OFF_STAGE2 + S2W * STG2;  // 1 KiB nobody reads: the prefetch pieces' destination
constexpr int LDS_STEM2 = OFF_PF2 + 1024;
static_assert(2 * LDS_STEM2 <= 160 * 1024, "two workgroups per CU");

__global__ __launch_bounds__(S2W * 64, 2) void stem2_kernel(StemArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t lds[LDS_STEM2];
  const unsigned lds32 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) int8_t*)lds;
  const int tid = threadIdx.x, lane = tid & 63, q = tid >> 6;  // q = column quarter = wave
  const int lr = lane & 31, lh = lane >> 5;
  const int nitems = a.N * a.nb;
  ST_DECL;

  // both channel tiles' weight fragments and epilogue constants, in registers
  v4i wr[2][6];
#pragma unroll
  for (int ot = 0; ot < 2; ++ot)
#pragma unroll
    for (int t = 0; t < 6; ++t) wr[ot][t] = *(const v4i*)(a.w + (ot * 32 + lr) * SK + t * 32 + lh * 16);
  using F2 = float __attribute__((ext_vector_type(2)));
  const F2 ab2[2] = {F2{a.alpha[lr], a.beta[lr]}, F2{a.alpha[32 + lr], a.beta[32 + lr]}};  // (alpha, beta) per channel tile
  for (int i = tid; i < CR_SLOTS * CR_ROW / 16; i += S2W * 64) *(v4i*)(lds + OFF_CR + i * 16) = v4i{0, 0, 0, 0};
  wait_vm_const<0>();
  __syncthreads();
  const int pi = ((lr >> 3) << 2) + (lr & 3) + 16 * ((lr >> 2) & 1);
  const int ox = 28 * q - 1 + pi;
  const unsigned a_col = lds32 + OFF_CR + (unsigned)(ox + 2 + lh) * 16;
  int8_t* stg = lds + OFF_STAGE2 + q * STG2;

  // converter lanes: (row pair cv_p of the quad, unit cv_u): a wave = 32 units x 2 pairs
  const int cv_p = (tid >> 5) & 1, cv_u = (tid & 31) + 32 * (tid >> 6);
  const bool col_ok = (unsigned)(cv_u - 4) < 112u;
  // staging read-back (store side): 16-lane group g, lane i; rows 16g + 8(g&1) + r, then 16g + 8(1 - (g&1)) + r
  const int tg = lane >> 4, ti = lane & 15;
  const int R1 = 16 * tg + 8 * (tg & 1) + (ti >> 1), R2 = 16 * tg + 8 * (1 - (tg & 1)) + (ti >> 1);
  const int8_t* tr1 = stg + R1 * 16 + 8 * ((ti & 1) ^ ((R1 >> 3) & 1));
  const int8_t* tr2 = stg + R2 * 16 + 8 * ((ti & 1) ^ ((R2 >> 3) & 1));
  // a 16-lane group's transposed reads depend only on its own lanes'
  // addresses: odd groups read R2's bytes first, so no select on the results
  const int8_t* trA = (tg & 1) ? tr2 : tr1;
  const int8_t* trB = (tg & 1) ? tr1 : tr2;

  int item0, n_my;
  xcd_chunk(nitems, item0, n_my);
  // the next launch's weights (the first layer1 block's), pulled towards the
  // CUs while this launch runs; the item loop's vmcnt(0) waits cover them
  prefetch_next(a.pf, q, S2W, lds32 + OFF_PF2);
  for (int li = 0; li < n_my; ++li) {
    const int item = xcd_item(item0, li);
    const int n = item / a.nb, band = item - n * a.nb;
    const int py0 = band * a.R, py1 = min(56, py0 + a.R);
    if (py0 >= py1) continue;
    const int iy0 = 4 * py0 - 5;  // odd: a pair starts on an odd input row
    const float* img = a.x + (size_t)n * 3 * 224 * 224;
    F2 raw[PD + 1][2][3];
    __amdgpu_buffer_rsrc_t rs[3];
#pragma unroll
    for (int c = 0; c < 3; ++c)
      rs[c] = __builtin_amdgcn_make_buffer_rsrc((void*)(img + (size_t)c * 224 * 224), 0, 224 * 224 * 4, 0x00020000);
    auto load_quad = [&](int k, F2 (&r)[2][3]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int iy = iy0 + 4 * k + 2 * cv_p + h, sc = cv_u - 4;
        const int off = ((unsigned)iy < 224u && col_ok) ? (iy * 224 + 2 * sc) * 4 : 0x40000000;
#pragma unroll
        for (int c = 0; c < 3; ++c)
          r[h][c] = __builtin_bit_cast(F2, __builtin_amdgcn_raw_buffer_load_b64(rs[c], off, 0, 0));
      }
    };
    // pair (iy, iy + 1), iy = iy0 + 4k + 2 cv_p odd: its conv rows are
    // oyb + e (e < 4), oyb = (iy - 3) / 2 = ob0 + 2k, and in conv row oyb + e
    // the pair's bytes are 12 - 4e .. 15 - 4e (kh = 6 - 2e, 7 - 2e)
    const int ob0 = ((iy0 - 3) >> 1) + cv_p;
    int sa[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) sa[j] = OFF_CR + ((ob0 + j) & (CR_SLOTS - 1)) * CR_ROW + cv_u * 16;
    // scatter addresses with the conv-row order rotated per 16-lane group:
    // write i of group g goes to conv row e = (i + g) & 3, so the four
    // groups' 4-byte writes land at chunk offsets 12 - 4e that differ mod 16
    // bytes -- 64 distinct banks per instruction, where the same e for every
    // lane put all four groups on the same 16 banks
    const int lg = (tid >> 4) & 3;
    int ra[4][4];
#pragma unroll
    for (int jj = 0; jj < 4; ++jj)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = (i + lg) & 3;
        int v = sa[(2 * jj) & 7];
        v = e == 1 ? sa[(2 * jj + 1) & 7] : v;
        v = e == 2 ? sa[(2 * jj + 2) & 7] : v;
        v = e == 3 ? sa[(2 * jj + 3) & 7] : v;
        ra[jj][i] = v + 12 - 4 * e;
      }
    // the scale multiply and the rounding add of a column pair at a time (two
    // scalar instructions each: the library is built without packed fp32 ones),
    // the clamp per value
    const F2 inv2 = {a.inv_s, a.inv_s}, mg2 = {12582912.0f, 12582912.0f};
    auto convert_quad = [&](const F2 (&r)[2][3], auto jc) {  // jc = (2k) & 7
      constexpr int J = decltype(jc)::value;
      unsigned v[3];
#pragma unroll
      for (int c = 0; c < 3; ++c) {
        unsigned u[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // rounding add before the clamp: fl(t + 1.5 2^23) is 1.5 2^23 +
          // rint(t) for |t| < 2^22 and beyond the clamp bounds otherwise, so
          // clamping the sum to 1.5 2^23 -+ 127 gives the same bits
          const F2 t = r[h][c] * inv2 + mg2;
          u[2 * h] = __float_as_uint(__builtin_amdgcn_fmed3f(t[0], 12582912.0f - 127.f, 12582912.0f + 127.f));
          u[2 * h + 1] = __float_as_uint(__builtin_amdgcn_fmed3f(t[1], 12582912.0f - 127.f, 12582912.0f + 127.f));
        }
        v[c] = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u) | __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 3; ++c) *(unsigned*)(lds + ra[J >> 1][i] + c * CR_PLANE) = v[c];
    };
    // conv rows oy, oy + 1 x both channel tiles: four chains per k-step on the
    // A fragments of the two rows (read once) and the resident weights
    auto conv_rows2 = [&](int oy, v16i (&c)[2][2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) c[i][0] = c[i][1] = v16i{0};
      const unsigned ra0 = a_col + (oy & (CR_SLOTS - 1)) * CR_ROW, ra1 = a_col + ((oy + 1) & (CR_SLOTS - 1)) * CR_ROW;
      v4i fa0[3], fa1[3];
#define STEM2_RD(t)                                                                                              \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa0[(t) % 3]) : "v"(ra0), "n"(((t) >> 1) * CR_PLANE + ((t) & 1) * 32) \
               : "memory");                                                                                      \
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa1[(t) % 3]) : "v"(ra1), "n"(((t) >> 1) * CR_PLANE + ((t) & 1) * 32) \
               : "memory")
#define STEM2_WAIT(t, n) asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(fa0[(t) % 3]), "+v"(fa1[(t) % 3]) : "n"(n) : "memory")
#define STEM2_K(t)                                                                          \
  c[0][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa0[(t) % 3], wr[0][t], c[0][0], 0, 0, 0); \
  c[0][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa0[(t) % 3], wr[1][t], c[0][1], 0, 0, 0); \
  c[1][0] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa1[(t) % 3], wr[0][t], c[1][0], 0, 0, 0); \
  c[1][1] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fa1[(t) % 3], wr[1][t], c[1][1], 0, 0, 0)
      STEM2_RD(0);
      STEM2_RD(1);
      STEM2_WAIT(0, 2);
      STEM2_K(0);
      STEM2_RD(2);
      STEM2_WAIT(1, 2);
      STEM2_K(1);
      STEM2_RD(3);
      STEM2_WAIT(2, 2);
      STEM2_K(2);
      STEM2_RD(4);
      STEM2_WAIT(3, 2);
      STEM2_K(3);
      STEM2_RD(5);
      STEM2_WAIT(4, 2);
      STEM2_K(4);
      STEM2_WAIT(5, 0);
      STEM2_K(5);
#undef STEM2_RD
#undef STEM2_WAIT
#undef STEM2_K
    };
    // column -1 (the pool's left pad) is masked by a min against the lane's
    // kb (INT_MIN on the image's left edge, else INT_MAX); lanes 0-31's
    // column 16 is lanes 32-63's column 0, brought over by one permlane32
    // swap whose other operand is column 1 (both dead once H[0] is formed)
    const int kb = (q == 0 && lh == 0) ? kIntMin : 0x7fffffff;
    auto hpool = [&](const v16i& c, int (&H)[8]) {
      H[0] = max3i(__builtin_elementwise_min(c[0], kb), c[1], c[2]);
#pragma unroll
      for (int m = 1; m < 7; ++m) H[m] = max3i(c[2 * m], c[2 * m + 1], c[2 * m + 2]);
      unsigned x0 = (unsigned)c[0], c16 = (unsigned)c[1];
      swap32(x0, c16);
      H[7] = max3i(c[14], c[15], (int)c16);
    };

    // prologue as stem_fused_kernel: quads 0..2 converted, 3 .. 2+PD loaded
#pragma unroll
    for (int k = 0; k <= PD; ++k) load_quad(k, raw[k]);
    convert_quad(raw[0], std::integral_constant<int, 0>{});
    load_quad(PD + 1, raw[0]);
    convert_quad(raw[1], std::integral_constant<int, 2>{});
    load_quad(PD + 2, raw[1]);
    convert_quad(raw[2], std::integral_constant<int, 4>{});
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    int Hp[2][8];
    if (py0 == 0) {
#pragma unroll
      for (int ot = 0; ot < 2; ++ot)
#pragma unroll
        for (int m = 0; m < 8; ++m) Hp[ot][m] = kIntMin;
    } else {
      // conv row 2py0 - 1 (its pair partner 2py0 is computed and discarded)
      v16i c[2][2];
      conv_rows2(2 * py0 - 1, c);
      hpool(c[0][0], Hp[0]);
      hpool(c[0][1], Hp[1]);
    }
    int8_t* const ybase = a.y + ((size_t)n * 56 * 56 + 14 * q + ti) * 64 + 16 * tg;
    auto store_row = [&](int p) {
      const v2i r1 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)trA);
      const v2i r2 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)trB);
      if (ti < 14) *(v4i*)(ybase + p * 56 * 64) = v4i{r1[0], r1[1], r2[0], r2[1]};
    };
    auto step = [&](int t, auto setc) {
      constexpr int S = decltype(setc)::value;
      const int p = py0 + t;
      __builtin_amdgcn_s_waitcnt(0xc07f);
      __builtin_amdgcn_s_barrier();
      ST(0);
      v16i c[2][2];
      conv_rows2(2 * p, c);
      ST(2);
      convert_quad(raw[(S + 3) % (PD + 1)], std::integral_constant<int, (2 * S + 6) & 7>{});
      ST(1);
      if (t > 0) store_row(p - 1);
      load_quad(t + 3 + PD, raw[(S + 2) % (PD + 1)]);
      ST(4);
#pragma unroll
      for (int ot = 0; ot < 2; ++ot) {
        int He[8], Ho[8];
        hpool(c[0][ot], He);
        hpool(c[1][ot], Ho);
        unsigned w[2] = {0u, 0u};
#pragma unroll
        // two pooled values at a time, two scalar fmas (an inline-asm packed form
        // broadcasting alpha / beta by op_sel gave ~25 differing bytes per B = 256
        // launch from run to run; tools/probe/stem_det.py)
        for (int m = 0; m < 8; m += 2) {
          const int v0 = max3i(Hp[ot][m], He[m], Ho[m]), v1 = max3i(Hp[ot][m + 1], He[m + 1], Ho[m + 1]);
          Hp[ot][m] = Ho[m];
          Hp[ot][m + 1] = Ho[m + 1];
          const F2 y = __builtin_elementwise_fma(F2{(float)v0, (float)v1}, F2{ab2[ot][0], ab2[ot][0]}, F2{ab2[ot][1], ab2[ot][1]});
          const float y0 = __builtin_fminf(y[0], 127.f), y1 = __builtin_fminf(y[1], 127.f);
          w[m >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(y0, m & 3, w[m >> 2]);
          w[m >> 2] = __builtin_amdgcn_cvt_pk_u8_f32(y1, (m + 1) & 3, w[m >> 2]);
        }
        const int row = ot * 32 + lr;
        *(v2i*)(stg + row * 16 + 8 * (lh ^ ((row >> 3) & 1))) = v2i{(int)w[0], (int)w[1]};
      }
      ST(3);
    };
    const int nsteps = py1 - py0;
    ST(5);
    static_assert(PD == 3, "the step loop below is unrolled by 4");
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    int t = 0;
    for (; t + 4 <= nsteps; t += 4) {
      step(t, I0{});
      step(t + 1, I1{});
      step(t + 2, I2{});
      step(t + 3, I3{});
    }
    if (t < nsteps) step(t, I0{});
    if (t + 1 < nsteps) step(t + 1, I1{});
    if (t + 2 < nsteps) step(t + 2, I2{});
    if (py1 > py0) store_row(py1 - 1);
    wait_vm0();
    __syncthreads();
  }
  ST_STORE();
}

int num_cus_stem() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
  }
  return n;
}

}  // namespace

size_t stem_packed_bytes() { return 64 * SK; }

// OIHW q[64][3][7][7] -> [64 oc][t 6][lh 2][16 B]: unit m = 2t + lh is
// (c = m >> 2, j = m & 3), byte b = 2 kh + dx is tap (kh, kw = 2j + dx - 1);
// kw = -1 and kh = 7 are zero (the K order of stem_fused_kernel's A
// fragments).  Rows of channels with alpha < 0 are negated and |alpha|
// returned, which keeps the fused stem's pool-before-epilogue exact.
template <typename T, typename Neg>
void pack_stem(const T* q, const float* alpha, T* out, float* alpha_abs, Neg neg_of) {
  for (int i = 0; i < 64 * SK; ++i) out[i] = 0;
  for (int o = 0; o < 64; ++o) {
    const bool neg = alpha[o] < 0.f;
    alpha_abs[o] = neg ? -alpha[o] : alpha[o];
    for (int m = 0; m < 12; ++m) {
      const int c = m >> 2, j = m & 3;
      for (int b = 0; b < 16; ++b) {
        const int kh = b >> 1, kw = 2 * j + (b & 1) - 1;
        if (kh > 6 || kw < 0 || kw > 6) continue;
        const T v = q[((o * 3 + c) * 7 + kh) * 7 + kw];
        out[o * SK + m * 16 + b] = neg ? neg_of(v) : v;
      }
    }
  }
}

void pack_stem_weights(const int8_t* q, const float* alpha, int8_t* out, float* alpha_abs) {
  pack_stem(q, alpha, out, alpha_abs, [](int8_t v) { return (int8_t)-v; });
}

// e4m3 twin: the sign bit is the negation.
void pack_stem_weights_f8(const uint8_t* q, const float* alpha, uint8_t* out, float* alpha_abs) {
  pack_stem(q, alpha, out, alpha_abs, [](uint8_t v) { return (uint8_t)(v ^ 0x80); });
}

hipError_t launch_stem_fused(const float* x, int N, const int8_t* w, const float* alpha, const float* beta,
                             float inv_s, int8_t* y, hipStream_t s, bool f8, const Prefetch* pf) {
  const int ncu = num_cus_stem();
  int nb = (2 * ncu + N - 1) / N;  // bands per image so that every CU gets two co-resident items
  nb = nb < 1 ? 1 : (nb > 14 ? 14 : nb);
  const int R = (56 + nb - 1) / nb;
  nb = (56 + R - 1) / R;
  StemArgs a{x, w, alpha, beta, y, inv_s, N, nb, R, pf && !f8 ? *pf : Prefetch{}};
  const int items = N * nb, grid = items < 2 * ncu ? items : 2 * ncu;
  if (f8)
    hipLaunchKernelGGL(stem_fused_kernel<true>, dim3(grid), dim3(SNW * 64), 0, s, a);
  else
    hipLaunchKernelGGL(stem2_kernel, dim3(grid), dim3(S2W * 64), 0, s, a);
  return hipGetLastError();
}

}  // namespace dlq
