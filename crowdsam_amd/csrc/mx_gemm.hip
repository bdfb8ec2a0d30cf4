// csam_mx_gemm: C[M,N] = act(A[M,K] W[N,K]^T + bias[n]) + R[m,n] with microscaled operands (A in E4M3 or E2M1, W in E2M1) on the
// scaled matrix instructions: the E8M0 byte of every block of 32 enters the MFMA as an operand, sums are fp32.
//
// One 32x32x64 MFMA takes two blocks of 32 per row, supplied (codes of E2M1, and always the scales) by lane groups g = 0, 1.  Which two
// blocks is free as long as A and W agree: instruction kk of a 128-wide step takes blocks kk and 2 + kk, so that a lane's two
// instructions read neighbouring blocks 2g, 2g + 1 and its two scale bytes are one aligned 16-bit load.  An E4M3 operand is spread
// differently: lane group g holds halves g (16 codes) of BOTH blocks.
// What the instruction keeps: E2M1 products are summed as fp32 sums them.  With an E4M3 operand it lines 16 neighbouring products up to
// the largest and drops bits below 2^-13 of that (measured: a product 2^-14 of its neighbour vanishes, one in the next 16 does not).  Of
// the result's norm: 4.5e-6 on gaussian rows, 1.2e-5 where 4 of 1024 channels are thirty times the others, 6e-5 where the channels' sizes are
// powers of two of a spread of 3; fp16's rounding is 2.1e-4, the rounding to E4M3 3e-2 to 6e-2.  16-bit results of many rows take that, at
// a third to a half of the time, unless the caller forbids it; otherwise both operands are multiplied as bf16, which holds them exactly.
// W rows are the instruction's row operand, A rows its columns: a lane ends up with 4 consecutive n of one row m.
#include <type_traits>
#include <utility>
#include <limits.h>
#include "mx_common.h"

namespace {

struct MxGemmArgs {
  const uint8_t* A; long lda; const uint8_t* As; long a_ss;
  const uint8_t* W; long ldw; const uint8_t* Ws; long w_ss;
  void* C; long ldc; int c_dt;
  const float* bias;
  const void* R; long ldr; int r_dt;
  int act, M, N, Kp;
  int cut;                                   // CSAM_MX_CUT: results may lose what the scaled instruction drops; CSAM_MX_WHOLE: they may not
  int past;                                  // C's rows begin on lines of 128 bytes: large tiles may store past the caches
};

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
__device__ __forceinline__ void glds16(const void* g, void* l) { __builtin_amdgcn_global_load_lds((gptr_t)g, (lptr_t)l, 16, 0, 0); }
__device__ __forceinline__ void glds4(const void* g, void* l) { __builtin_amdgcn_global_load_lds((gptr_t)g, (lptr_t)l, 4, 0, 0); }

__device__ __forceinline__ float mx_elem(const void* p, int dt, long i) {
  return dt == CSAM_DT_F32 ? ((const float*)p)[i] : dt == CSAM_DT_F16 ? (float)((const half_t*)p)[i] : (float)((const bf16_t*)p)[i];
}

__device__ __forceinline__ void mx_put(void* p, int dt, long i, float x) {
  if (dt == CSAM_DT_F32) ((float*)p)[i] = x;
  else if (dt == CSAM_DT_F16) ((half_t*)p)[i] = (half_t)x;
  else ((bf16_t*)p)[i] = (bf16_t)x;
}

// GELU = x Phi(x).  Results of 16 bits: Phi(-|x|) = 2^S(|x|), S a polynomial fitted to log2 of it for the least relative error up to 6.25.
// Within 6e-6 of the result there (half an fp16 step is 4.9e-4) and 1.3e-9 beyond, where the leading coefficient takes it to zero with no
// clamp: no error grows with |x|, +-inf and NaN come out as x (1 + erf(x / sqrt 2)) / 2 gives them.  Seven FMA, an exponential of quarter
// rate and four more: of 5330 x 4096 x 1024 5 us, a shorter polynomial of Phi with a clamp 4.  Results that stay fp32 take the erf form, off by
// 1.5e-7 / 2 |x| and its roundings.
__device__ __forceinline__ float mx_gelu16(float x) {
  const float k[8] = {-1.835283115e-06f, 6.160674093e-05f, -9.305833373e-04f, 8.508088067e-03f,
                      -5.396040156e-02f, -4.584641457e-01f, -1.151251078e+00f, -9.999952912e-01f};
  const float a = fabsf(x);
  float s = k[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) s = fmaf(s, a, k[i]);
  const float q = csam_exp2(s);
  return x * (x < 0.f ? q : 1.f - q);
}
__device__ __forceinline__ void mx_gelu4(floatx4& v, int c_dt) {
  if (c_dt == CSAM_DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = csam_gelu_erf(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mx_gelu16(v[i]);
  }
}

// a NaN stays one
__device__ __forceinline__ floatx4 mx_relu4(floatx4 v) {
  return floatx4{v[0] < 0.f ? 0.f : v[0], v[1] < 0.f ? 0.f : v[1], v[2] < 0.f ? 0.f : v[2], v[3] < 0.f ? 0.f : v[3]};
}

// 4 elements at any element's address
__device__ __forceinline__ floatx4 mx_load4(const void* p, int dt, long i) {
  if (dt == CSAM_DT_F32) return *(const csam_pack<float, 4>::at*)((const float*)p + i);
  if (dt == CSAM_DT_F16) {
    const auto h = *(const csam_pack<half_t, 4>::at*)((const half_t*)p + i);
    return floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
  }
  const auto h = *(const csam_pack<bf16_t, 4>::at*)((const bf16_t*)p + i);
  return floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}
template <bool NT = false>
__device__ __forceinline__ void mx_store4(void* p, int dt, long i, floatx4 v) {
  if (dt == CSAM_DT_F32) csam_put<NT>((csam_pack<float, 4>::at*)((float*)p + i), v);
  else if (dt == CSAM_DT_F16)
    csam_put<NT>((csam_pack<half_t, 4>::at*)((half_t*)p + i), csam_pack<half_t, 4>::vec{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]});
  else
    csam_put<NT>((csam_pack<bf16_t, 4>::at*)((bf16_t*)p + i), csam_pack<bf16_t, 4>::vec{(bf16_t)v[0], (bf16_t)v[1], (bf16_t)v[2], (bf16_t)v[3]});
}

// 4 consecutive columns n .. n + 3 of row m: bias, activation, residual, rounding, store
__device__ __forceinline__ void mx_epilogue4(const MxGemmArgs& p, int m, int n, floatx4 v) {
  if (m >= p.M || n >= p.N) return;
  const bool full = n + 4 <= p.N;
  if (p.bias) {
    if (full) v += mx_load4(p.bias, CSAM_DT_F32, n);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) v[i] += p.bias[n + i];
  }
  if (p.act == CSAM_ACT_GELU) mx_gelu4(v, p.c_dt);
  else if (p.act == CSAM_ACT_RELU) v = mx_relu4(v);
  if (full) {
    if (p.R) v += mx_load4(p.R, p.r_dt, (long)m * p.ldr + n);
    mx_store4(p.C, p.c_dt, (long)m * p.ldc + n, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i < p.N) {
      float x = v[i];
      if (p.R) x += mx_elem(p.R, p.r_dt, (long)m * p.ldr + n + i);
      mx_put(p.C, p.c_dt, (long)m * p.ldc + n + i, x);
    }
  }
}

// The large tiles' results go past the caches where every line of C belongs to one wave (16384 x 4096 x 4096 185 us, 170 so; 5330 x 4096 x
// 1024 with GELU 37.6, 35.9); lines that waves share have to meet in the L2 (6312 x 3178 x 206 28.2 us, past the caches 40.3).
// 4 consecutive columns of B rows STEP apart; every choice is uniform and made once for the B rows, but for the `left` < 4 last columns of
// rows whose length is no multiple of 4
template <int B, int STEP, bool NT>
__device__ __forceinline__ void mx_epilogue_rows(const MxGemmArgs& p, int m, int n, floatx4 bz, floatx4 (&v)[B]) {
  if (n >= p.N) return;
  const int left = p.N - n;
  floatx4 res[B];
  if (p.R && left < 4) {
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 3; ++i) res[b][i] = m + b * STEP < p.M && i < left ? mx_elem(p.R, p.r_dt, (long)(m + b * STEP) * p.ldr + n + i) : 0.f;
  } else if (p.R) {
    const long at = (long)m * p.ldr + n;
    if (p.r_dt == CSAM_DT_F32) {
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (m + b * STEP < p.M) res[b] = *(const csam_pack<float, 4>::at*)((const float*)p.R + at + (long)b * STEP * p.ldr);
    } else {
      uintx2 u[B];
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (m + b * STEP < p.M)
          u[b] = __builtin_bit_cast(uintx2, *(const csam_pack<half_t, 4>::at*)((const half_t*)p.R + at + (long)b * STEP * p.ldr));
#pragma unroll
      for (int b = 0; b < B; ++b) {
        if (p.r_dt == CSAM_DT_F16) {
          const half4_t h = __builtin_bit_cast(half4_t, u[b]);
          res[b] = floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        } else {
          res[b] = floatx4{csam_lo_bf16(u[b][0]), csam_hi_bf16(u[b][0]), csam_lo_bf16(u[b][1]), csam_hi_bf16(u[b][1])};
        }
      }
    }
  }
#pragma unroll
  for (int b = 0; b < B; ++b) v[b] += bz;
  if (p.act == CSAM_ACT_GELU) {
#pragma unroll
    for (int b = 0; b < B; ++b) mx_gelu4(v[b], p.c_dt);
  } else if (p.act == CSAM_ACT_RELU) {
#pragma unroll
    for (int b = 0; b < B; ++b) v[b] = mx_relu4(v[b]);
  }
  if (p.R) {
#pragma unroll
    for (int b = 0; b < B; ++b) v[b] += res[b];
  }
  if (left < 4) {
#pragma unroll
    for (int b = 0; b < B; ++b)
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (m + b * STEP < p.M && i < left) mx_put(p.C, p.c_dt, (long)(m + b * STEP) * p.ldc + n + i, v[b][i]);
  } else if (NT && p.past) {
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (m + b * STEP < p.M) mx_store4<true>(p.C, p.c_dt, (long)(m + b * STEP) * p.ldc + n, v[b]);
  } else {
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (m + b * STEP < p.M) mx_store4(p.C, p.c_dt, (long)(m + b * STEP) * p.ldc + n, v[b]);
  }
}

template <int FA, int KK>
__device__ __forceinline__ floatx16 mx_mfma32(const intx8& w, const intx8& a, floatx16 c, int sw, int sa) {
  constexpr int AF = FA == CSAM_MX_FP8 ? 0 : 4;
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w, a, c, 4, AF, KK, sw, KK, sa);
}
template <int FA, int J>
__device__ __forceinline__ floatx4 mx_mfma16(const intx8& w, const intx8& a, floatx4 c, int sw, int sa) {
  constexpr int AF = FA == CSAM_MX_FP8 ? 0 : 4;
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 4, AF, J, sw, J, sa);
}
__device__ __forceinline__ intx8 mx_frag(const void* lo) {
  const uintx4 a = *(const uintx4*)lo;
  return intx8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
}
__device__ __forceinline__ intx8 mx_frag(const void* lo, const void* hi) {
  const uintx4 a = *(const uintx4*)lo, b = *(const uintx4*)hi;
  return intx8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

template <int... I, typename F>
__device__ __forceinline__ void mx_for_each(std::integer_sequence<int, I...>, F f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, typename F>
__device__ __forceinline__ void mx_for(F f) { mx_for_each(std::make_integer_sequence<int, N>{}, f); }
#define MX_C(x) (std::integral_constant<int, (x)>{})

// An E4M3 part whose products are summed as fp32 sums them: both operands become bf16, which holds a scaled code of either format exactly,
// and four 32x32x16 instructions take the part.  Lane group g then holds codes 16g .. 16g + 15 of both blocks of the part: A's fragment is
// that already, W's group has 32 codes of one block and swaps halves with the other group, as the two groups' scales do.
__device__ __forceinline__ void mx_swap32(unsigned& a, unsigned& b) {          // a's upper half of lanes for b's lower
  const auto p = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = p[0];
  b = p[1];
}
typedef __bf16 mx_bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf8 __attribute__((ext_vector_type(8)));
template <int KK>
__device__ __forceinline__ void mx_scales(int s, unsigned (&byte)[2]) {        // of the part's two blocks
  byte[0] = byte[1] = (unsigned)s;
  mx_swap32(byte[0], byte[1]);
#pragma unroll
  for (int f = 0; f < 2; ++f) byte[f] = (byte[f] >> (8 * KK)) & 255u;
}
// a NaN block, or codes whose scale is so near the ends of the range that their product with it may not be a normal bf16
__device__ __forceinline__ bool mx_far(unsigned byte, unsigned codes) { return (byte == 255u) | ((byte - 32u >= 192u) & (codes != 0u)); }
__device__ __forceinline__ bool mx_far_a(const intx8& f, const unsigned (&byte)[2]) {
  return mx_far(byte[0], (unsigned)(f[0] | f[1] | f[2] | f[3])) | mx_far(byte[1], (unsigned)(f[4] | f[5] | f[6] | f[7]));
}
// the codes times their scales (byte 127: as they are)
__device__ __forceinline__ void mx_bf16_a(const intx8& f, const unsigned (&byte)[2], mx_bf8 (&out)[4]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const float sc = __builtin_bit_cast(float, byte[m / 2] << 23);
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const mx_bf2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * m + d], sc, false);
      const mx_bf2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(f[2 * m + d], sc, true);
      out[m][4 * d] = lo[0], out[m][4 * d + 1] = lo[1], out[m][4 * d + 2] = hi[0], out[m][4 * d + 3] = hi[1];
    }
  }
}
__device__ __forceinline__ void mx_swap_w(intx8& f) {                                     // the first 16 codes, the others
  unsigned q[4] = {(unsigned)f[0], (unsigned)f[1], (unsigned)f[2], (unsigned)f[3]};      // of the part's first block, of its second
  mx_swap32(q[0], q[2]);
  mx_swap32(q[1], q[3]);
#pragma unroll
  for (int m = 0; m < 4; ++m) f[m] = (int)q[m];
}
__device__ __forceinline__ bool mx_far_w(const intx8& f, const unsigned (&byte)[2]) {
  return mx_far(byte[0], (unsigned)(f[0] | f[1])) | mx_far(byte[1], (unsigned)(f[2] | f[3]));
}
__device__ __forceinline__ void mx_bf16_w(const intx8& f, const unsigned (&byte)[2], mx_bf8 (&out)[4]) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    const float sc = __builtin_bit_cast(float, byte[m / 2] << 23);
    const mx_bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)f[m], sc, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)f[m], sc, 1);
    const mx_bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)f[m], sc, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4((unsigned)f[m], sc, 3);
    out[m] = mx_bf8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
  }
}
// acc + t 2^(a + w - 254): the sum of a block's products of bare codes, by the blocks' E8M0 bytes
__device__ __forceinline__ float mx_add_scaled(float acc, float t, int a, int w) {
  return acc + (max(a, w) == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(t, a + w - 254));
}
// A part with far blocks: the bare codes are multiplied (every product is a multiple of 2^-10 below 2^12), each block's sum then takes its
// scales, so that whatever the scales are nothing is lost but what fp32 does not hold.
__device__ __forceinline__ void mx_far_part(const intx8& w, const unsigned (&wbyte)[2], const intx8& a, const unsigned (&abyte)[2],
                                            floatx16& acc, int g) {
  const unsigned bare[2] = {127u, 127u};
  mx_bf8 ab[4], wb[4];
  mx_bf16_a(a, bare, ab);
  mx_bf16_w(w, bare, wb);
  mx_for<2>([&](auto f_) {
    constexpr int f = decltype(f_)::value;
    floatx16 t = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[2 * f], ab[2 * f], t, 0, 0, 0);
    t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[2 * f + 1], ab[2 * f + 1], t, 0, 0, 0);
    int from = 4 * g;
    asm volatile("" : "+v"(from));                         // fetched anew for every tile: kept, W's scales would take 64 registers
    mx_for<16>([&](auto e_) {                              // register e holds W's row 8 (e / 4) + 4g + e % 4
      constexpr int e = decltype(e_)::value;
      acc[e] = mx_add_scaled(acc[e], t[e], (int)abyte[f], __shfl((int)wbyte[f], from + 8 * (e / 4) + e % 4));
      if constexpr (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);       // (four in flight: registers)
    });
  });
}

// --------------------------------------------------------------------------------------------------------------- tiled form
// TM x TN tile, WGM x WGN waves of 32x32 MFMA tiles, KS-wide steps through NS LDS stages filled by LDS-DMA (codes 16 bytes, scales 4
// bytes per lane).  LDS lines are 128 bytes: a row of the step (256 E2M1 or 128 E4M3 codes), or two rows of 128 E2M1 codes.  The LDS reads
// 256 bytes a cycle, sixteen lanes of 16 bytes: a row's pieces are turned by XOR with the index of its 256 bytes, on the DMA's source
// address and on the reads, so that sixteen lanes reading one column of pieces meet no bank twice.
// 16384 x 4096 x 4096: E2M1 183 us = 3.0 PFLOP/s, E4M3 267 us = 2.1; the matrix pipes are busy a third of the time.
template <int FA, int TM, int TN, int WGM, int WGN, int NS, int KS>
struct MxTile {
  static constexpr int NW = WGM * WGN;
  static constexpr int RA = FA == CSAM_MX_FP8 ? KS : KS / 2, RW = KS / 2;                // bytes of a row per step
  static constexpr int ABYTES = TM * RA, WBYTES = TN * RW, SBYTES = (TM + TN) * (KS / 32), STAGE = ABYTES + WBYTES + SBYTES;
  static constexpr int RUNS = (TM + TN) / 64 * (KS / 128);                               // scale fetches of 64 rows x 4 bytes
  static constexpr int LA = ABYTES / 1024 / NW, LW = WBYTES / 1024 / NW, LS = (RUNS + NW - 1) / NW;
  static constexpr int PER = LA + LW + LS;               // DMA instructions of a wave per stage: what a counted wait leaves in flight
  static constexpr int MI = TM / WGM / 32, NI = TN / WGN / 32;
  static constexpr int EPI = NW * 32 * (NI * 32 + 4) * 4;    // a wave's 32 rows of fp32 results on their way out, row by row
  static constexpr int LDS = NS * STAGE > EPI ? NS * STAGE : EPI;
  static_assert(LA * NW * 1024 == ABYTES && LW * NW * 1024 == WBYTES && TM % 64 == 0 && TN % 64 == 0, "whole DMA instructions per wave");
  static_assert((RA == 64 || RA == 128) && (RW == 64 || RW == 128), "line formats");
};

// tile of workgroup b: each XCD (b % 8) takes a contiguous run of the order, which walks GROUP tile rows column by column, so that the
// workgroups an XCD runs at once share operand panels in its L2
__device__ __forceinline__ void mx_tile_of(int b, int nm, int nn, int& tm, int& tn) {
  constexpr int GROUP = 8;
  const int n = nm * nn, x = b & 7, q = n >> 3, r = n & 7;
  const int i = x * q + min(x, r) + (b >> 3);
  const int per = GROUP * nn, grp = i / per, first = grp * GROUP, rows = min(GROUP, nm - first), j = i - grp * per;
  tn = j / rows;
  tm = first + j - tn * rows;
}

// byte of piece c (16 bytes) of row r in an operand whose rows are RB bytes
template <int RB>
__device__ __forceinline__ int mx_lds_piece(int r, int c) {
  return RB == 128 ? r * 128 + ((c ^ ((r >> 1) & 7)) << 4) : r * 64 + ((c ^ ((r >> 2) & 3)) << 4);
}

template <int FA, int TM, int TN, int WGM, int WGN, int NS, int KS, bool EXACT = false>
__global__ __launch_bounds__(WGM * WGN * 64, (TM / WGM) * (TN / WGN) > 128 * 64 ? 1 : 2) void mx_gemm_kernel(MxGemmArgs p) {
  using T = MxTile<FA, TM, TN, WGM, WGN, NS, KS>;
  constexpr int NW = T::NW, RA = T::RA, RW = T::RW, LA = T::LA, LW = T::LW, LS = T::LS, MI = T::MI, NI = T::NI, NH = KS / 64;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::LDS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN;
  int tm, tn;
  mx_tile_of(blockIdx.x, (p.M + TM - 1) / TM, (p.N + TN - 1) / TN, tm, tn);
  const int bm0 = tm * TM, bn0 = tn * TN;

  // DMA sources (32-bit offsets from the tile's first row; rows behind the last one are the last one again and never stored): lane l of
  // instruction i fills byte i * 1024 + l * 16, i.e. it fetches the piece that belongs there
  const uint8_t* abase = p.A + (long)bm0 * p.lda;
  const uint8_t* wbase = p.W + (long)bn0 * p.ldw;
  unsigned aoff[LA], woff[LW], soff[LS];
  const uint8_t* sbase[LS];
  long sstep[LS];
  int sdst[LS];
  auto source = [&](int at, int rb, int rows, unsigned ld) {        // piece at byte `at` of an operand's stage
    const int row = at / rb, c = (at % rb) >> 4, turned = rb == 128 ? c ^ ((row >> 1) & 7) : c ^ ((row >> 2) & 3);
    return (unsigned)min(row, rows - 1) * ld + turned * 16;
  };
#pragma unroll
  for (int i = 0; i < LA; ++i) aoff[i] = source((wave * LA + i) * 1024 + lane * 16, RA, p.M - bm0, (unsigned)p.lda);
#pragma unroll
  for (int i = 0; i < LW; ++i) woff[i] = source((wave * LW + i) * 1024 + lane * 16, RW, p.N - bn0, (unsigned)p.ldw);
#pragma unroll
  for (int i = 0; i < LS; ++i) {                          // a wave without a run of its own repeats the last one
    const int run = min(wave * LS + i, T::RUNS - 1), h = run / ((TM + TN) / 64), at = run % ((TM + TN) / 64);
    const bool isa = at < TM / 64;
    const int row = (isa ? at : at - TM / 64) * 64 + lane;
    sstep[i] = isa ? p.a_ss : p.w_ss;
    sbase[i] = (isa ? p.As + (long)bm0 * 4 : p.Ws + (long)bn0 * 4) + h * sstep[i];
    soff[i] = (unsigned)min(row, isa ? p.M - 1 - bm0 : p.N - 1 - bn0) * 4u;
    sdst[i] = T::ABYTES + T::WBYTES + run * 256;
  }
  // DMA instruction d of stage t (its source; a step behind the last one is the last one again) into stage `slot`
  auto dma = [&](auto d_, int slot, int t) {
    constexpr int d = decltype(d_)::value;
    uint8_t* base = smem + slot * T::STAGE;
    if constexpr (d < LA) glds16(abase + (long)t * RA + aoff[d], base + (wave * LA + d) * 1024);
    else if constexpr (d < LA + LW) glds16(wbase + (long)t * RW + woff[d - LA], base + T::ABYTES + (wave * LW + d - LA) * 1024);
    else glds4(sbase[d - LA - LW] + (long)t * (KS / 128) * sstep[d - LA - LW] + soff[d - LA - LW], base + sdst[d - LA - LW]);
  };

  floatx16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  // The main loop issues one stream per wave, in the order written here: part h of a step is MI * NI matrix instructions, and between them
  // go the LDS reads of the next part (a second fragment set) and a share of a later stage's DMA.  In a bunch behind the barrier the
  // DMAs of all waves queue for the one address unit of the CU while the matrix pipes wait.
  //   last part of step t:    reads of step t + 1's part 0; the first DMAs of step t + NS into stage t, which is read out
  //   other parts of step t:  reads of the next part; the rest of step t + NS - 1
  // Before the last part a wait and a barrier publish step t + 1: of the DMAs issued so far, steps t + 2 .. t + NS - 1 stay in flight.
  const int nt = p.Kp / KS;
  const int r = lane & 31, g = lane >> 5;
  constexpr int NQ = MI * NI, FR = FA == CSAM_MX_FP8 ? 2 : 1, NF = NI + MI * FR, NSC = MI + NI, PER = T::PER;
  intx8 af[2][MI], wf[2][NI];
  int sa[2][MI], sw[2][NI];                               // two bytes each: the scales of parts 2h and 2h + 1
  // LDS read k of part h: W fragments, A fragments (E4M3: two reads each); and scale read k of parts h and h + 1
  auto read = [&](auto k_, auto h_, int slot) {
    constexpr int k = decltype(k_)::value, h = decltype(h_)::value, set = h & 1;
    constexpr int c = (h >> 1) * 4 + (h & 1);                                               // E2M1: piece c + 2g of the row
    const uint8_t* base = smem + slot * T::STAGE;
    if constexpr (k < NI) {
      const uintx4 v = *(const uintx4*)(base + T::ABYTES + (wn * NI + k) * 32 * RW + mx_lds_piece<RW>(r, c + 2 * g));
#pragma unroll
      for (int e = 0; e < 4; ++e) wf[set][k][e] = (int)v[e];
    } else {
      constexpr int i = (k - NI) / FR, f = (k - NI) % FR;
      const int pc = FA == CSAM_MX_FP8 ? 4 * f + 2 * h + g : c + 2 * g;                        // E4M3: pieces 2h + g and 4 + 2h + g
      const uintx4 v = *(const uintx4*)(base + (wm * MI + i) * 32 * RA + mx_lds_piece<RA>(r, pc));
#pragma unroll
      for (int e = 0; e < 4; ++e) af[set][i][4 * f + e] = (int)v[e];
    }
  };
  auto read_scale = [&](auto k_, auto h_, auto ss_, int slot) {
    constexpr int k = decltype(k_)::value, h = decltype(h_)::value, ss = decltype(ss_)::value;
    const uint8_t* sb = smem + slot * T::STAGE + T::ABYTES + T::WBYTES + (h >> 1) * (TM + TN) * 4 + r * 4 + 2 * g;
    if constexpr (k < MI) sa[ss][k] = *(const unsigned short*)(sb + (wm * MI + k) * 128);
    else sw[ss][k - MI] = *(const unsigned short*)(sb + TM * 4 + (wn * NI + k - MI) * 128);
  };
  // part h: matrix instructions on scale set ss; between them the reads of part rh (scale set rs) from stage rslot and the DMAs
  // [d0, d1) of step dt into stage dslot.  The reads go first, so that they are done when the part is.
  auto part = [&](auto h_, auto ss_, auto rh_, auto rs_, int rslot, auto d0_, auto d1_, int dslot, int dt) __attribute__((always_inline)) {
    constexpr int h = decltype(h_)::value, ss = decltype(ss_)::value, rh = decltype(rh_)::value;
    constexpr int d0 = decltype(d0_)::value, d1 = decltype(d1_)::value;
    constexpr int S = (rh & 1) == 0 ? NSC : 0, NR = NF + S, ND = d1 - d0;
    mx_bf8 ab[EXACT ? MI : 1][4], wb[EXACT ? NI : 1][4];
    unsigned abyte[EXACT ? MI : 1][2], wbyte[EXACT ? NI : 1][2];
    bool far = false;
    if constexpr (EXACT) {
#pragma unroll
      for (int i = 0; i < MI; ++i) mx_scales<(h & 1)>(sa[ss][i], abyte[i]), far |= mx_far_a(af[h & 1][i], abyte[i]);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        mx_scales<(h & 1)>(sw[ss][j], wbyte[j]);
        mx_swap_w(wf[h & 1][j]);
        far |= mx_far_w(wf[h & 1][j], wbyte[j]);
      }
      far = __builtin_amdgcn_ballot_w64(far) != 0;        // uniform: matrix instructions do not heed the lanes' mask
    }
    constexpr int GAPS = NQ < 4 ? NQ : 4, RPG = (NR + GAPS - 1) / GAPS, G0 = NQ > 4 ? 2 : 0;
    constexpr int SCALED = 0, AS_BF16 = 1, FAR = 2;
    auto run = [&](auto form_) __attribute__((always_inline)) {
      constexpr int form = decltype(form_)::value;
      mx_for<NQ>([&](auto q_) {
        constexpr int q = decltype(q_)::value, i = q / NI, j = q % NI;
        if constexpr (form == FAR) {
          mx_far_part(wf[h & 1][j], wbyte[j], af[h & 1][i], abyte[i], acc[i][j], g);
        } else if constexpr (form == AS_BF16) {
#pragma unroll
          for (int m = 0; m < 4; ++m) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j][m], ab[i][m], acc[i][j], 0, 0, 0);
        } else {
          acc[i][j] = mx_mfma32<FA, (h & 1)>(wf[h & 1][j], af[h & 1][i], acc[i][j], sw[ss][j], sa[ss][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
        constexpr int r0 = q * RPG < NR ? q * RPG : NR, r1 = (q + 1) * RPG < NR ? (q + 1) * RPG : NR;
        constexpr int e0 = q < G0 ? 0 : (q - G0) * ND / (NQ - G0), e1 = q < G0 ? 0 : (q - G0 + 1) * ND / (NQ - G0);
        mx_for<r1 - r0>([&](auto x_) {
          constexpr int k = r0 + decltype(x_)::value;
          if constexpr (k < S) read_scale(MX_C(k), rh_, rs_, rslot);
          else read(MX_C(k - S), rh_, rslot);
        });
        mx_for<e1 - e0>([&](auto x_) { dma(MX_C(d0 + e0 + decltype(x_)::value), dslot, dt); });
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    if constexpr (EXACT) {
      if (!far) {
#pragma unroll
        for (int i = 0; i < MI; ++i) mx_bf16_a(af[h & 1][i], abyte[i], ab[i]);
#pragma unroll
        for (int j = 0; j < NI; ++j) mx_bf16_w(wf[h & 1][j], wbyte[j], wb[j]);
        run(MX_C(AS_BF16));
      } else {
        run(MX_C(FAR));
      }
    } else {
      run(MX_C(SCALED));
    }
  };
  constexpr int FIRST = (PER + NH - 1) / NH;              // DMAs of a stage that its first (the last) part issues
  mx_for<NS - 1>([&](auto s_) { mx_for<PER>([&](auto d_) { dma(d_, decltype(s_)::value, min(decltype(s_)::value, nt - 1)); }); });
  mx_for<FIRST>([&](auto d_) { dma(d_, NS - 1, min(NS - 1, nt - 1)); });
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * PER + FIRST) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  mx_for<NSC>([&](auto k_) { read_scale(k_, MX_C(0), MX_C(0), 0); });
  mx_for<NF>([&](auto k_) { read(k_, MX_C(0), 0); });
  // step t, t % UN = u: stages and scale sets are constants of the unrolled loop.  Scale sets: by step (NH = 2) or by pair of parts.
  constexpr int UN = NH == 2 && NS % 2 ? 2 * NS : NS;
  auto step = [&](int t, auto u_) __attribute__((always_inline)) {
    constexpr int u = decltype(u_)::value, slot = u % NS, next = (u + 1) % NS, prev = (u + NS - 1) % NS, us = u & 1;
    mx_for<NH - 1>([&](auto h_) {
      constexpr int h = decltype(h_)::value;
      constexpr int d0 = FIRST + h * (PER - FIRST) / (NH - 1), d1 = FIRST + (h + 1) * (PER - FIRST) / (NH - 1);
      part(h_, MX_C(NH == 2 ? us : (h >> 1) & 1), MX_C(h + 1), MX_C(((h + 1) >> 1) & 1), slot, MX_C(d0), MX_C(d1), prev, min(t + NS - 1, nt - 1));
    });
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * PER) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    part(MX_C(NH - 1), MX_C(NH == 2 ? us : 1), MX_C(0), MX_C(NH == 2 ? us ^ 1 : 0), next, MX_C(0), MX_C(FIRST), slot, min(t + NS, nt - 1));
  };
  for (int t = 0;;) {
    bool more = true;
    mx_for<UN>([&](auto u_) {
      if (more) {
        step(t, u_);
        more = ++t < nt;
      }
    });
    if (!more) break;
  }

  // Epilogue: a wave passes its results 32 rows at a time through LDS of its own and takes them out row by row, so that NI * 32
  // consecutive columns of a row move together (straight from the registers a store would touch 32 rows with 32 bytes each).
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");    // the repeated fetches have landed
  __builtin_amdgcn_s_barrier();                                 // ... everybody's, and every stage is read out
  asm volatile("" ::: "memory");
  constexpr int COLS = NI * 32, PITCH = COLS + 4;          // + 4 floats: rows start 4 banks apart
  constexpr int LPR = COLS / 4, RPI = 64 / LPR, B = 4;     // lanes of a row, rows of an access, accesses of a batch
  float* buf = (float*)smem + wave * 32 * PITCH;
  const int n = bn0 + wn * COLS + (lane % LPR) * 4, mr = bm0 + wm * MI * 32 + lane / LPR;
  floatx4 bz = {0.f, 0.f, 0.f, 0.f};
  if (p.bias && n + 4 <= p.N) bz = mx_load4(p.bias, CSAM_DT_F32, n);
  else if (p.bias)
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (n + j < p.N) bz[j] = p.bias[n + j];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(floatx4*)(buf + r * PITCH + j * 32 + 8 * e + 4 * g) =
            floatx4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
    const float* src = buf + lane / LPR * PITCH + (lane % LPR) * 4;
#pragma unroll 1
    for (int s = 0; s < 32 / RPI; s += B) {
      floatx4 v[B];
#pragma unroll
      for (int b = 0; b < B; ++b) v[b] = *(const floatx4*)(src + (s + b) * RPI * PITCH);
      mx_epilogue_rows<B, RPI, (TM >= 128)>(p, mr + i * 32 + s * RPI, n, bz, v);
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- direct form
// Few rows of A (up to MT * 16): no LDS staging.  A workgroup owns 16 rows of W; its NW waves take 256-wide steps of K in turn, each
// lane loading its own 32 consecutive bytes of a W row, and their partial sums are added through LDS in wave order.
// 16x16x128 instruction j of a step takes blocks 2g + j: lane group g = 0 .. 3 supplies the scales of its two blocks (one 16-bit load);
// an E4M3 operand's lane group holds half (g & 1) of logical blocks g / 2 and 2 + g / 2.
// Bound by the latency of a wave's few loads: 1 x 4096 x 1024 E4M3 3.5 us (EXACT 4.2), 32 x 4096 x 4096 E2M1 5.7 us (1.6 TB/s of weights).
// EXACT (an E4M3 operand whose products keep every bit): the bare codes as bf16, a block of 32 per 16x16x32 instruction, its sum scaled by
// the blocks' bytes.  A lane's two blocks of each operand are shared out among the lane groups, 8 codes each, by lane swaps.  us, the scaled
// instruction / so / 64x64 tiles: 1 x 1024 x 4096 4.4 / 6.6 / 24.5, 16 x 4096 x 4096 6.0 / 8.1 / 25, 32 x 4096 x 4096 7.9 / 11.2 / 25,
// 224 x 256 x 1024 3.8 / 4.5 / 9.0.
__device__ __forceinline__ void mx_swap16(unsigned& a, unsigned& b) {          // a's odd rows of 16 lanes for b's even ones
  const auto p = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = p[0];
  b = p[1];
}
// x[d] of lane group g for x[g] of lane group d
__device__ __forceinline__ void mx_turn(unsigned& x0, unsigned& x1, unsigned& x2, unsigned& x3) {
  mx_swap32(x0, x2);
  mx_swap32(x1, x3);
  mx_swap16(x0, x1);
  mx_swap16(x2, x3);
}
template <int FA, int MT, int NW, bool EXACT = false>
__global__ __launch_bounds__(NW * 64) void mx_gemm_rows_kernel(MxGemmArgs p) {
  static_assert(!EXACT || FA == CSAM_MX_FP8, "E2M1 products lose nothing");
  __shared__ floatx4 part[NW][MT][64];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 15, g = lane >> 4;
  const int tn_n = (p.N + 15) / 16;
  const int bn0 = (int)(blockIdx.x % tn_n) * 16, bm0 = (int)(blockIdx.x / tn_n) * (MT * 16);
  const long wrow = min(bn0 + r, p.N - 1);
  const uint8_t* wp = p.W + wrow * p.ldw + g * 32;
  const uint8_t* wsp = p.Ws + wrow * 4 + (long)(g >> 1) * p.w_ss + 2 * (g & 1);
  const uint8_t *ap[MT], *asp[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long row = min(bm0 + i * 16 + r, p.M - 1);
    ap[i] = p.A + row * p.lda + (EXACT ? g * 64 : FA == CSAM_MX_FP8 ? (g >> 1) * 64 + (g & 1) * 16 : g * 32);
    asp[i] = p.As + row * 4 + (EXACT ? 0 : (long)(g >> 1) * p.a_ss + 2 * (g & 1));
  }
  floatx4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int nt = p.Kp / 256;
  for (int t = wave; t < nt; t += NW) {
    if constexpr (EXACT) {
      unsigned w[2][4], sw[2][4];                          // of W: block 2b + j's codes 8g .. 8g + 7 at [j][b]; rows 4g + e's scales [half][e]
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uintx4 c = *(const uintx4*)(wp + (long)t * 128 + 16 * j);
#pragma unroll
        for (int d = 0; d < 4; ++d) w[j][d] = c[d];
#pragma unroll
        for (int e = 0; e < 4; ++e) sw[j][e] = *(const unsigned*)(p.Ws + (2L * t + j) * p.w_ss + 4L * min(bn0 + 4 * g + e, p.N - 1));
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) mx_turn(w[j][0], w[j][1], w[j][2], w[j][3]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        unsigned a[2][8], sa[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          sa[j] = *(const unsigned*)(asp[i] + (2L * t + j) * p.a_ss);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uintx4 c = *(const uintx4*)(ap[i] + (long)t * 256 + 32 * j + 16 * q);
#pragma unroll
            for (int d = 0; d < 4; ++d) a[j][4 * q + d] = c[d];
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mx_turn(a[j][0], a[j][2], a[j][4], a[j][6]);     // then block 2b + j's codes 8g .. 8g + 3 at [j][2b], the next four behind
          mx_turn(a[j][1], a[j][3], a[j][5], a[j][7]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const mx_bf2 a0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j][2 * b], 1.f, false), a1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j][2 * b], 1.f, true);
            const mx_bf2 a2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j][2 * b + 1], 1.f, false), a3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a[j][2 * b + 1], 1.f, true);
            const mx_bf2 w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j][b], 1.f, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j][b], 1.f, 1);
            const mx_bf2 w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j][b], 1.f, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[j][b], 1.f, 3);
            const floatx4 v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(mx_bf8{w0[0], w0[1], w1[0], w1[1], w2[0], w2[1], w3[0], w3[1]},
                                                                      mx_bf8{a0[0], a0[1], a1[0], a1[1], a2[0], a2[1], a3[0], a3[1]},
                                                                      floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            const int at = 8 * (2 * (b & 1) + j);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              acc[i][e] = mx_add_scaled(acc[i][e], v[e], (int)(sa[b >> 1] >> at & 255u), (int)(sw[b >> 1][e] >> at & 255u));
          }
        }
      }
    } else {
      const intx8 w0 = mx_frag(wp + (long)t * 128), w1 = mx_frag(wp + (long)t * 128 + 16);
      const int sw = *(const unsigned short*)(wsp + 2L * t * p.w_ss);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int sa = *(const unsigned short*)(asp[i] + 2L * t * p.a_ss);
        intx8 a0, a1;
        if constexpr (FA == CSAM_MX_FP8) {
          const uint8_t* a = ap[i] + (long)t * 256;        // logical block g of instruction j = block 2g + j of the step
          a0 = mx_frag(a, a + 128);
          a1 = mx_frag(a + 32, a + 160);
        } else {
          a0 = mx_frag(ap[i] + (long)t * 128);
          a1 = mx_frag(ap[i] + (long)t * 128 + 16);
        }
        acc[i] = mx_mfma16<FA, 0>(w0, a0, acc[i], sw, sa);
        acc[i] = mx_mfma16<FA, 1>(w1, a1, acc[i], sw, sa);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < MT; i += NW) {
    floatx4 v = part[0][i][lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) v += part[w][i][lane];
    mx_epilogue4(p, bm0 + i * 16 + r, bn0 + 4 * g, v);
  }
}

template <int FA, bool EXACT>
int mx_rows(hipStream_t st, const MxGemmArgs& p, long t16) {
  CSAM_REQUIRE(csam_launch_fits(t16, 256), "csam_mx_gemm: %d x %d is more than one launch takes", p.M, p.N);
  if (t16 <= 256 || p.M <= 16) mx_gemm_rows_kernel<FA, 1, 4, EXACT><<<(unsigned)t16, 256, 0, st>>>(p);
  else mx_gemm_rows_kernel<FA, 2, 4, EXACT><<<(unsigned)((long)csam_cdiv(p.M, 32) * csam_cdiv(p.N, 16)), 256, 0, st>>>(p);
  CSAM_LAUNCH_CHECK("csam_mx_gemm");
  return CSAM_OK;
}

template <int FA, int TM, int TN, int WGM, int WGN, int NS, int KS, bool EXACT = false>
int mx_tiles(hipStream_t st, const MxGemmArgs& p) {
  const long grid = (long)csam_cdiv(p.M, TM) * csam_cdiv(p.N, TN);
  CSAM_REQUIRE(csam_launch_fits(grid, WGM * WGN * 64), "csam_mx_gemm: %d x %d is more than one launch takes", p.M, p.N);
  mx_gemm_kernel<FA, TM, TN, WGM, WGN, NS, KS, EXACT><<<(unsigned)grid, WGM * WGN * 64, 0, st>>>(p);
  CSAM_LAUNCH_CHECK("csam_mx_gemm");
  return CSAM_OK;
}

// Which form.  The tiles move their operands from L2 to LDS at 6 to 9 TB/s while the matrix pipes are busy a third to a half of the time, at
// the clock that their power leaves: the largest tile wins that fills the chip, and where K is short, one that leaves room for a second
// workgroup per CU, whose main loop covers the first one's epilogue.  GELU makes the epilogue longer, so with it "short" goes further.
// us, fp16 out, each pair measured on one MI355X:
//   M x N x K              E2M1                                       E4M3
//   32 x 4096 x 4096       rows 5.7, 64x64 6.7                        rows 7.5, 64x64 7.8
//   224 x 4096 x 4096      64x64 7.8 (three stages 8.2), 128x64 10.2  64x64 9.2 (three stages 10.9), 64x128 11.4
//   512 x 4096 x 4096      64x64 11.7, 128x64 11.0, 128x128 16.8      64x64 15.3, 64x128 12.9, 128x256 22.0
//   1330 x 1024 x 4096     64x64 10.3, 128x64 10.1, 128x128 16.6      64x64 14.1, 64x128 11.8, 128x256 22.0
//   2048 x 4096 x 4096     64x64 34.7, 128x128 26.2, 256x256 32.6     64x64 50.6, 128x256 32.0, 256x256 45.9
//   2048 x 4096 x 1024     64x64 17.6, 128x128 13.6, 256x256 15.9     64x64 19.8, 128x256 14.6, 128x128 16.2
//   4096 x 4096 x 1024     256x256 22.8, 128x128 24.7                 256x256 25.0, 128x128 27.8
//   5330 x 4096 x 1024     128x128 29.3 (256-wide steps 31.5)         128x128 33.4, 128x256 34.3, 256x256 37.9
//     with GELU            128x128 33.0 (256-wide steps 37.5)         128x128 38.6, 128x256 41.7, 256x256 47.6
//   21320 x 4096 x 1024    128x128 92, 256x256 93, with GELU 106, 127     109, 113, with GELU 127, 145
//   16384 x 5120 x 1280    128x128 102, 256x256 91, with GELU 114, 121    120, 113, with GELU 135, 139
//   33000 x 4096 x 1792    128x128 201, 256x256 194, with GELU 223, 244   238, 247, with GELU 265, 290
//   8192 x 4096 x 2048     128x128 57.7, 256x256 51.5, with GELU 64.6, 61.3    69.1, 66.2, with GELU 77.5, 75.2
//   5330 x 4096 x 4096     128x128 68.2 (128-wide steps 76.7), 256x256 72.5    128x256 87.1, 128x128 97.8, 256x256 98.5
//   16384 x 4096 x 4096    128x128 218, 256x256 183                   128x256 292, 256x256 267
template <int FA>
int mx_gemm_launch(hipStream_t st, const MxGemmArgs& p) {
  const long t16 = (long)csam_cdiv(p.M, 16) * csam_cdiv(p.N, 16);
  const bool few = p.M <= 16 || t16 <= 512;
  if constexpr (FA == CSAM_MX_FP8) {
    // What the scaled instruction drops is kept in fp32 results and in results of few rows, which are bound by latency, unless the caller
    // lets it go, and in 16-bit results of many rows if the caller asks.  us to fp32 (M x N x K), as bf16 / scaled to fp16, the
    // conversion to bf16 taking most of the difference: 224 x 2048 x 1024 9.4 / 4.9, 5330 x 4096 x 1024 75 / 34.
    const bool whole = p.cut == CSAM_MX_WHOLE || (p.cut == 0 && (few || p.c_dt == CSAM_DT_F32));
    if (whole) {
      if (few) return mx_rows<FA, true>(st, p, t16);
      if ((long)csam_cdiv(p.M, 128) * csam_cdiv(p.N, 128) >= 256) return mx_tiles<FA, 128, 128, 2, 2, 2, 128, true>(st, p);
      return mx_tiles<FA, 64, 64, 2, 2, 4, 128, true>(st, p);
    }
  }
  if (few) return mx_rows<FA, false>(st, p, t16);
  const long t256 = (long)csam_cdiv(p.M, 256) * csam_cdiv(p.N, 256), rounds = (t256 + 255) / 256;
  const bool brief = p.Kp <= (p.act == CSAM_ACT_GELU ? 1792 : 1024);
  const bool large = brief ? t256 >= 240 && rounds == 1 : rounds >= 4 || t256 * 4 >= rounds * 256 * 3;
  if constexpr (FA == CSAM_MX_FP4) {
    const long t128 = (long)csam_cdiv(p.M, 128) * csam_cdiv(p.N, 128);
    if (large) return mx_tiles<FA, 256, 256, 2, 4, 3, 128>(st, p);
    if (t128 < 256) return mx_tiles<FA, 64, 64, 2, 2, 4, 256>(st, p);
    if (brief && t128 > 512) return mx_tiles<FA, 128, 128, 2, 2, 2, 128>(st, p);
    return mx_tiles<FA, 128, 128, 2, 2, 2, 256>(st, p);
  } else {
    const long wide = (long)csam_cdiv(p.M, 128) * csam_cdiv(p.N, 256);
    if (large) return mx_tiles<FA, 256, 256, 4, 2, 3, 128>(st, p);
    if (wide < 128) {
      const int n64 = csam_cdiv(p.N, 64), n128 = csam_cdiv(p.N, 128);       // (N = 137: 64x64 23.0, 64x128, half of it empty, 27.6)
      if ((long)csam_cdiv(p.M, 64) * n64 <= 256 || n128 * 15 > n64 * 8) return mx_tiles<FA, 64, 64, 2, 2, 4, 128>(st, p);
      return mx_tiles<FA, 64, 128, 2, 2, 4, 128>(st, p);
    }
    if (!brief || wide <= 256) return mx_tiles<FA, 128, 256, 2, 4, 3, 128>(st, p);
    return mx_tiles<FA, 128, 128, 2, 2, 2, 128>(st, p);
  }
}

}  // namespace

extern "C" int csam_mx_gemm(void* stream, const void* A, long lda, const void* A_scales, long a_scale_stride, int a_fmt, const void* W,
                            long ldw, const void* W_scales, long w_scale_stride, void* C, long ldc, int c_dtype, const float* bias,
                            const void* residual, long ldr, int r_dtype, int act, int M, int N, int K) {
  if (M == 0 || N == 0) return CSAM_OK;
  CSAM_REQUIRE(A && A_scales && W && W_scales && C, "csam_mx_gemm: null operand");
  CSAM_REQUIRE(M > 0 && N > 0 && K > 0, "csam_mx_gemm: bad sizes M %d N %d K %d", M, N, K);
  CSAM_REQUIRE(M <= INT_MAX - 255 && N <= INT_MAX - 255, "csam_mx_gemm: %d x %d is over 2^31 - 256 rows or columns", M, N);
  CSAM_REQUIRE(a_fmt == CSAM_MX_FP4 || a_fmt == CSAM_MX_FP8, "csam_mx_gemm: bad format %d", a_fmt);
  CSAM_REQUIRE(K <= (1 << 20), "csam_mx_gemm: K %d is over 2^20", K);
  const int Kp = csam_cdiv(K, 256) * 256;
  auto dt_ok = [](int dt) { return dt == CSAM_DT_F16 || dt == CSAM_DT_F32 || dt == CSAM_DT_BF16; };
  auto al = [](const void* q, long ld, int a) { return (uintptr_t)q % a == 0 && ld % a == 0; };
  CSAM_REQUIRE(dt_ok(c_dtype) && (!residual || dt_ok(r_dtype)), "csam_mx_gemm: bad dtype");
  const int cut = act & (CSAM_MX_CUT | CSAM_MX_WHOLE), plain = act & ~cut;
  CSAM_REQUIRE(cut != (CSAM_MX_CUT | CSAM_MX_WHOLE), "csam_mx_gemm: CSAM_MX_CUT and CSAM_MX_WHOLE exclude each other");
  CSAM_REQUIRE(plain == CSAM_ACT_NONE || plain == CSAM_ACT_GELU || plain == CSAM_ACT_RELU, "csam_mx_gemm: bad activation %d", act);
  CSAM_REQUIRE(lda >= (a_fmt == CSAM_MX_FP8 ? Kp : Kp / 2) && ldw >= Kp / 2, "csam_mx_gemm: code rows are shorter than %d padded columns", Kp);
  CSAM_REQUIRE(lda < (1 << 24) && ldw < (1 << 24), "csam_mx_gemm: code rows 16 MB apart or more");
  CSAM_REQUIRE(al(A, lda, 16) && al(W, ldw, 16), "csam_mx_gemm: codes and their row pitch have to be multiples of 16 bytes");
  CSAM_REQUIRE(al(A_scales, a_scale_stride, 4) && al(W_scales, w_scale_stride, 4) && a_scale_stride >= 4L * M && w_scale_stride >= 4L * N,
               "csam_mx_gemm: scale groups have to lie 4-byte aligned, at least 4 * rows bytes apart");
  CSAM_REQUIRE(ldc >= N && (!residual || ldr >= N), "csam_mx_gemm: an output row pitch is shorter than N");
  MxGemmArgs p = {(const uint8_t*)A, lda, (const uint8_t*)A_scales, a_scale_stride, (const uint8_t*)W, ldw, (const uint8_t*)W_scales,
                  w_scale_stride, C, ldc, c_dtype, bias, residual, ldr, r_dtype, plain, M, N, Kp, cut,
                  al(C, ldc * (c_dtype == CSAM_DT_F32 ? 4 : 2), 128)};
  return a_fmt == CSAM_MX_FP8 ? mx_gemm_launch<CSAM_MX_FP8>((hipStream_t)stream, p) : mx_gemm_launch<CSAM_MX_FP4>((hipStream_t)stream, p);
}
