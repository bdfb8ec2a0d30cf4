// Shared pieces of the microscaled (MX) operators and of the row operators that take bfloat16 beside fp16 / fp32.
//
// An MX operand of R rows and K columns (include/csam.h has the layout users see):
//   codes   [R][Kp / 2] (E2M1, element 2i in the low nibble) or [R][Kp] (E4M3), Kp = K rounded up to 256, zero codes behind K;
//   scales  [Kp / 128][R][4] E8M0 bytes: block b (32 elements) of row r at [b / 4][r][b % 4].  The four scales of a 128-wide step
//           of neighbouring rows lie side by side, so a wave fetches the scales of 32 or 64 rows as one run of whole cache lines;
//           row-major bytes would cost a 128-byte line per row and step.
#pragma once
#include "csam_common.h"

#define CSAM_DT_BF16 2
#define CSAM_MX_FP4 0
#define CSAM_MX_FP8 1
#define CSAM_MX_CUT 16
#define CSAM_MX_WHOLE 32

// A launch has fewer than 2^32 work items (HIP's limit on grid times workgroup in one dimension)
inline bool csam_launch_fits(long groups, int threads) { return groups <= 0xffffffffL / threads; }

typedef __bf16 bf16_t;
typedef unsigned uintx2 __attribute__((ext_vector_type(2)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float csam_lo_bf16(unsigned u) { return __builtin_bit_cast(float, u << 16); }
__device__ __forceinline__ float csam_hi_bf16(unsigned u) { return __builtin_bit_cast(float, u & 0xffff0000u); }

// N consecutive elements at an address that is a multiple of one element only: global accesses of any width take such addresses
template <typename T, int N>
struct csam_pack {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec at __attribute__((aligned(sizeof(T))));
};
// store; NT: past the caches' retention, for results that no cache would hold until they are read
template <bool NT, typename P, typename V>
__device__ __forceinline__ void csam_put(P* p, V v) {
  if constexpr (NT) __builtin_nontemporal_store(v, p);
  else *p = v;
}
// V = 4 or 8 consecutive elements as fp32; _tail: the first n of them (n may be <= 0), zeros behind
template <typename T, int V>
__device__ __forceinline__ void csam_load(const T* p, float (&v)[V]) {
  constexpr int N = sizeof(T) == 4 ? 4 : V;
#pragma unroll
  for (int j = 0; j < V; j += N) {
    const auto h = *(const typename csam_pack<T, N>::at*)(p + j);
#pragma unroll
    for (int i = 0; i < N; ++i) v[j + i] = (float)h[i];
  }
}
template <typename T, int V>
__device__ __forceinline__ void csam_load_tail(const T* p, int n, float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = i < n ? (float)p[i] : 0.f;
}
// V consecutive elements, rounded to nearest even
template <bool NT = false, typename T, int V>
__device__ __forceinline__ void csam_store(T* p, const float (&v)[V]) {
  constexpr int N = sizeof(T) == 4 ? 4 : V;
#pragma unroll
  for (int j = 0; j < V; j += N) {
    typename csam_pack<T, N>::vec h;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = (T)v[j + i];
    csam_put<NT>((typename csam_pack<T, N>::at*)(p + j), h);
  }
}
template <typename T, int V>
__device__ __forceinline__ void csam_store_tail(T* p, int n, const float (&v)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (i < n) p[i] = (T)v[i];
}

// value of an E8M0 byte: 2^(s - 127); 255 is NaN, 0 the subnormal 2^-127
__device__ __forceinline__ float csam_e8m0(unsigned s) {
  const unsigned bits = s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23;
  return __builtin_bit_cast(float, bits);
}

// DPP: a value of another lane of the quad, the eight or the row of sixteen
template <int CTRL>
__device__ __forceinline__ unsigned csam_dpp(unsigned v) {
  return (unsigned)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
}

// Quantises the V = 8 (4) values of this lane, whose quad (eight) of lanes holds one block of 32: returns the block's E8M0 byte and the
// codes (E2M1: 4 V bits in c[0]; E4M3: 8 V bits).
//   byte = max(exponent(amax) - emax, 0) on the biased fp32 exponent = floor(log2 amax) - emax + 127; a subnormal or zero amax has
//   exponent field 0, so its byte is 0; NaN and infinity have 255 -> byte 255 (every value of the block reads as NaN), codes 0.
// amax is an integer maximum of the magnitudes' bits: fmaxf would drop a NaN.  x / 2^(byte-127) is exact in fp32 (a power of two; the
// only results that could be subnormal come from elements 2^-100 below the block's largest, which round to zero in either format),
// so the one rounding is the converter's to E2M1 / E4M3, ties to even; both saturate (E4M3 by the clamp: the converter's own overflow
// would give NaN).
template <int FMT, int V>
__device__ __forceinline__ unsigned csam_mx_quant(const float (&v)[V], unsigned (&c)[2]) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m = max(m, __builtin_bit_cast(unsigned, v[i]) & 0x7fffffffu);
  m = max(m, csam_dpp<0xB1>(m));                          // quad_perm 1,0,3,2
  m = max(m, csam_dpp<0x4E>(m));                          // quad_perm 2,3,0,1
  if constexpr (V == 4) m = max(m, csam_dpp<0x141>(m));   // row_half_mirror: the other quad of the eight
  const unsigned e = m >> 23;
  constexpr unsigned EMAX = FMT == CSAM_MX_FP4 ? 2 : 8;
  const unsigned byte = e == 255u ? 255u : e > EMAX ? e - EMAX : 0u;
  c[0] = c[1] = 0u;
  if constexpr (FMT == CSAM_MX_FP4) {
    const float scale = __builtin_bit_cast(float, byte == 0u ? 0x00400000u : byte << 23);
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
    if constexpr (V == 8) {
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
      q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
    }
    c[0] = e == 255u ? 0u : q;
  } else {
    const float inv = __builtin_bit_cast(float, (254u - (byte > 253u ? 253u : byte)) << 23);
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      float w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_fmed3f(v[4 * j + i] * inv, -448.f, 448.f);
      int a = 0;
      a = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], a, false);
      a = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], a, true);
      c[j] = e == 255u ? 0u : (unsigned)a;
    }
  }
  return byte;
}

// Codes and scales of chunk `c` (V elements) of row `row`.  V = 8: 16 consecutive lanes hold a 128-wide group, so the four block bytes are
// put together with two rotations within 16 lanes and leave as one dword; V = 4: they are 32 lanes, and each block's byte leaves by itself.
template <int FMT, bool NT = false, int V>
__device__ __forceinline__ void csam_mx_store(const float (&v)[V], uint8_t* codes, long ldc, uint8_t* scales, long sstride, long row, int c) {
  unsigned q[2];
  unsigned s = csam_mx_quant<FMT>(v, q);
  uint8_t* to = codes + row * ldc + c * (FMT == CSAM_MX_FP4 ? V / 2 : V);
  if constexpr (FMT == CSAM_MX_FP8 && V == 8) csam_put<NT>((uintx2*)to, uintx2{q[0], q[1]});
  else if constexpr (FMT == CSAM_MX_FP8 || V == 8) csam_put<NT>((unsigned*)to, q[0]);
  else csam_put<NT>((unsigned short*)to, (unsigned short)q[0]);
  if constexpr (V == 8) {
    s <<= 8 * ((c >> 2) & 3);
    s |= csam_dpp<0x124>(s);                              // row_ror:4
    s |= csam_dpp<0x128>(s);                              // row_ror:8
    if ((c & 15) == 0) *(unsigned*)(scales + (long)(c >> 4) * sstride + row * 4) = s;
  } else {
    if ((c & 7) == 0) scales[(long)(c >> 5) * sstride + row * 4 + ((c >> 3) & 3)] = (uint8_t)s;
  }
}
