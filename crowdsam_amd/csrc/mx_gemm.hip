// csam_mx_gemm: C[M,N] = act(A[M,K] W[N,K]^T + bias[n]) + R[m,n] with microscaled operands (A in E4M3 or E2M1, W in E2M1) on the
// scaled matrix instructions: the E8M0 byte of every block of 32 enters the MFMA as an operand, sums are fp32.
//
// One 32x32x64 MFMA takes two blocks of 32 per row, supplied (codes of E2M1, and always the scales) by lane groups g = 0, 1.  Which two
// blocks is free as long as A and W agree: instruction kk of a 128-wide step takes blocks kk and 2 + kk, so that a lane's two
// instructions read neighbouring blocks 2g, 2g + 1 and its two scale bytes are one aligned 16-bit load.  An E4M3 operand is spread
// differently: lane group g holds halves g (16 codes) of BOTH blocks.
// W rows are the instruction's row operand, A rows its columns: a lane ends up with 4 consecutive n of one row m.
#include "mx_common.h"

namespace {

struct MxGemmArgs {
  const uint8_t* A; long lda; const uint8_t* As; long a_ss;
  const uint8_t* W; long ldw; const uint8_t* Ws; long w_ss;
  void* C; long ldc; int c_dt;
  const float* bias;
  const void* R; long ldr; int r_dt;
  int act, M, N, Kp;
  int vec;                                   // 4 consecutive columns of C (and R, bias) may move as one access
};

typedef const __attribute__((address_space(1))) void* gptr_t;
typedef __attribute__((address_space(3))) void* lptr_t;
__device__ __forceinline__ void glds16(const void* g, void* l) { __builtin_amdgcn_global_load_lds((gptr_t)g, (lptr_t)l, 16, 0, 0); }

__device__ __forceinline__ float mx_elem(const void* p, int dt, long i) {
  return dt == CSAM_DT_F32 ? ((const float*)p)[i] : dt == CSAM_DT_F16 ? (float)((const half_t*)p)[i] : (float)((const bf16_t*)p)[i];
}

// 4 consecutive columns n .. n + 3 of row m: bias, activation, residual, rounding, store
__device__ __forceinline__ void mx_epilogue4(const MxGemmArgs& p, int m, int n, floatx4 v) {
  if (m >= p.M || n >= p.N) return;
  const bool full = p.vec && n + 4 <= p.N;
  if (p.bias) {
    if (full) v += *(const floatx4*)(p.bias + n);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < p.N) v[i] += p.bias[n + i];
  }
  if (p.act != CSAM_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = csam_apply_act(v[i], p.act);
  }
  if (full) {
    if (p.R) {
      const long at = (long)m * p.ldr + n;
      if (p.r_dt == CSAM_DT_F32) v += *(const floatx4*)((const float*)p.R + at);
      else if (p.r_dt == CSAM_DT_F16) {
        const half4_t h = *(const half4_t*)((const half_t*)p.R + at);
        v += floatx4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
      } else {
        const uintx2 u = *(const uintx2*)((const bf16_t*)p.R + at);
        v += floatx4{csam_lo_bf16(u[0]), csam_hi_bf16(u[0]), csam_lo_bf16(u[1]), csam_hi_bf16(u[1])};
      }
    }
    const long at = (long)m * p.ldc + n;
    if (p.c_dt == CSAM_DT_F32) *(floatx4*)((float*)p.C + at) = v;
    else if (p.c_dt == CSAM_DT_F16) *(half4_t*)((half_t*)p.C + at) = half4_t{(half_t)v[0], (half_t)v[1], (half_t)v[2], (half_t)v[3]};
    else {
      typedef bf16_t bf16x4_t __attribute__((ext_vector_type(4)));
      *(bf16x4_t*)((bf16_t*)p.C + at) = bf16x4_t{(bf16_t)v[0], (bf16_t)v[1], (bf16_t)v[2], (bf16_t)v[3]};
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i < p.N) {
      float x = v[i];
      if (p.R) x += mx_elem(p.R, p.r_dt, (long)m * p.ldr + n + i);
      const long at = (long)m * p.ldc + n + i;
      if (p.c_dt == CSAM_DT_F32) ((float*)p.C)[at] = x;
      else if (p.c_dt == CSAM_DT_F16) ((half_t*)p.C)[at] = (half_t)x;
      else ((bf16_t*)p.C)[at] = (bf16_t)x;
    }
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

// --------------------------------------------------------------------------------------------------------------- tiled form
// TM x TN tile, WGM x WGN waves of 32x32 MFMA tiles, 128-wide K steps through NS = 2 LDS stages filled by 16-byte LDS-DMA.
// LDS lines of 128 bytes = one E4M3 row or two E2M1 rows of the step; slot ^= line & 7 on the DMA's source address and on the reads.
template <int FA, int TM, int TN, int WGM, int WGN>
__global__ __launch_bounds__(WGM * WGN * 64) void mx_gemm_kernel(MxGemmArgs p) {
  constexpr int NW = WGM * WGN;
  constexpr int RA = FA == CSAM_MX_FP8 ? 128 : 64, RW = 64;
  constexpr int ABYTES = TM * RA, STAGE = ABYTES + TN * RW;
  constexpr int LA = ABYTES / 1024 / NW, LW = TN * RW / 1024 / NW;
  static_assert(LA * NW * 1024 == ABYTES && LW * NW * 1024 == TN * RW, "whole DMA instructions per wave");
  constexpr int MI = TM / WGM / 32, NI = TN / WGN / 32;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * STAGE];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN;
  const int tn_n = (p.N + TN - 1) / TN;
  const int bm0 = (int)(blockIdx.x / tn_n) * TM, bn0 = (int)(blockIdx.x % tn_n) * TN;

  // DMA sources: lane l of instruction i fills line i * 8 + l / 8, slot l % 8, which holds piece (l % 8) ^ (line & 7)
  const int lg = (lane & 7) ^ (lane >> 3);
  const uint8_t *asrc[LA], *wsrc[LW];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int line = (wave * LA + i) * 8 + (lane >> 3);
    const int row = RA == 128 ? line : 2 * line + (lg >> 2), c = RA == 128 ? lg : lg & 3;
    asrc[i] = p.A + (long)min(bm0 + row, p.M - 1) * p.lda + c * 16;
  }
#pragma unroll
  for (int i = 0; i < LW; ++i) {
    const int line = (wave * LW + i) * 8 + (lane >> 3);
    wsrc[i] = p.W + (long)min(bn0 + 2 * line + (lg >> 2), p.N - 1) * p.ldw + (lg & 3) * 16;
  }
  auto stage = [&](int slot, int t) {
    uint8_t* base = smem + slot * STAGE;
#pragma unroll
    for (int i = 0; i < LA; ++i) glds16(asrc[i] + (long)t * RA, base + (wave * LA + i) * 1024);
#pragma unroll
    for (int i = 0; i < LW; ++i) glds16(wsrc[i] + (long)t * RW, base + ABYTES + (wave * LW + i) * 1024);
  };

  // fragment addresses within a stage (tile i, instruction kk): + i * 32 rows, ^ by kk
  const int r = lane & 31, g = lane >> 5;
  const int off64 = (r >> 1) * 128 + (((((r & 1) << 2) + 2 * g) ^ ((r >> 1) & 7)) << 4);       // E2M1: piece 2g + kk of the row
  const int off128 = r * 128 + ((g ^ (r & 7)) << 4);                                          // E4M3: pieces 2 kk + g and 4 + 2 kk + g
  const uint8_t *sap[MI], *swp[NI];
#pragma unroll
  for (int i = 0; i < MI; ++i) sap[i] = p.As + (long)min(bm0 + (wm * MI + i) * 32 + r, p.M - 1) * 4 + 2 * g;
#pragma unroll
  for (int j = 0; j < NI; ++j) swp[j] = p.Ws + (long)min(bn0 + (wn * NI + j) * 32 + r, p.N - 1) * 4 + 2 * g;

  floatx16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const int nt = p.Kp / 128;
  int sa[MI], sw[NI];
  stage(0, 0);
#pragma unroll
  for (int i = 0; i < MI; ++i) sa[i] = *(const unsigned short*)sap[i];
#pragma unroll
  for (int j = 0; j < NI; ++j) sw[j] = *(const unsigned short*)swp[j];
  for (int t = 0; t < nt; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // this wave's share of step t has landed
    __builtin_amdgcn_s_barrier();                          // ... and everybody's; step t - 1's stage is read out
    asm volatile("" ::: "memory");
    int na[MI], nw[NI];
    if (t + 1 < nt) {
      stage((t + 1) & 1, t + 1);
#pragma unroll
      for (int i = 0; i < MI; ++i) na[i] = *(const unsigned short*)(sap[i] + (long)(t + 1) * p.a_ss);
#pragma unroll
      for (int j = 0; j < NI; ++j) nw[j] = *(const unsigned short*)(swp[j] + (long)(t + 1) * p.w_ss);
    }
    const uint8_t* ab = smem + (t & 1) * STAGE + wm * MI * 32 * RA;
    const uint8_t* wb = smem + (t & 1) * STAGE + ABYTES + wn * NI * 32 * RW;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      intx8 af[MI], wf[NI];
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        if constexpr (RA == 128) af[i] = mx_frag(ab + i * 4096 + (off128 ^ (kk << 5)), ab + i * 4096 + (off128 ^ (kk << 5) ^ 64));
        else af[i] = mx_frag(ab + i * 2048 + (off64 ^ (kk << 4)));
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) wf[j] = mx_frag(wb + j * 2048 + (off64 ^ (kk << 4)));
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          acc[i][j] = kk ? mx_mfma32<FA, 1>(wf[j], af[i], acc[i][j], sw[j], sa[i]) : mx_mfma32<FA, 0>(wf[j], af[i], acc[i][j], sw[j], sa[i]);
    }
    if (t + 1 < nt) {
#pragma unroll
      for (int i = 0; i < MI; ++i) sa[i] = na[i];
#pragma unroll
      for (int j = 0; j < NI; ++j) sw[j] = nw[j];
    }
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = bm0 + (wm * MI + i) * 32 + r;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int n = bn0 + (wn * NI + j) * 32 + 4 * g;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mx_epilogue4(p, m, n + 8 * e, floatx4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]});
    }
  }
}

// -------------------------------------------------------------------------------------------------------------- direct form
// Few rows of A (up to MT * 16): no LDS staging.  A workgroup owns 16 rows of W; its NW waves take 256-wide steps of K in turn, each
// lane loading its own 32 consecutive bytes of a W row, and their partial sums are added through LDS in wave order.
// 16x16x128 instruction j of a step takes blocks 2g + j: lane group g = 0 .. 3 supplies the scales of its two blocks (one 16-bit load);
// an E4M3 operand's lane group holds half (g & 1) of logical blocks g / 2 and 2 + g / 2.
template <int FA, int MT, int NW>
__global__ __launch_bounds__(NW * 64) void mx_gemm_rows_kernel(MxGemmArgs p) {
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
    ap[i] = p.A + row * p.lda + (FA == CSAM_MX_FP8 ? (g >> 1) * 64 + (g & 1) * 16 : g * 32);
    asp[i] = p.As + row * 4 + (long)(g >> 1) * p.a_ss + 2 * (g & 1);
  }
  floatx4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int nt = p.Kp / 256;
  for (int t = wave; t < nt; t += NW) {
    const intx8 w0 = mx_frag(wp + (long)t * 128), w1 = mx_frag(wp + (long)t * 128 + 16);
    const int sw = *(const unsigned short*)(wsp + 2L * t * p.w_ss);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int sa = *(const unsigned short*)(asp[i] + 2L * t * p.a_ss);
      intx8 a0, a1;
      if constexpr (FA == CSAM_MX_FP8) {
        const uint8_t* a = ap[i] + (long)t * 256;          // logical block g of instruction j = block 2g + j of the step
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

template <int FA>
int mx_gemm_launch(hipStream_t st, const MxGemmArgs& p) {
  const long tn16 = csam_cdiv(p.N, 16);
  if (p.M <= 64) {
    if (p.M <= 16) mx_gemm_rows_kernel<FA, 1, 4><<<(unsigned)tn16, 256, 0, st>>>(p);
    else if (p.M <= 32) mx_gemm_rows_kernel<FA, 2, 4><<<(unsigned)tn16, 256, 0, st>>>(p);
    else mx_gemm_rows_kernel<FA, 4, 4><<<(unsigned)tn16, 256, 0, st>>>(p);
  } else {
    const long grid = (long)csam_cdiv(p.M, 128) * csam_cdiv(p.N, 128);
    CSAM_REQUIRE(grid < (1L << 31), "csam_mx_gemm: too many tiles");
    mx_gemm_kernel<FA, 128, 128, 2, 2><<<(unsigned)grid, 256, 0, st>>>(p);
  }
  CSAM_LAUNCH_CHECK("csam_mx_gemm");
  return CSAM_OK;
}

}  // namespace

extern "C" int csam_mx_gemm(void* stream, const void* A, long lda, const void* A_scales, long a_scale_stride, int a_fmt, const void* W,
                            long ldw, const void* W_scales, long w_scale_stride, void* C, long ldc, int c_dtype, const float* bias,
                            const void* residual, long ldr, int r_dtype, int act, int M, int N, int K) {
  if (M == 0 || N == 0) return CSAM_OK;
  CSAM_REQUIRE(A && A_scales && W && W_scales && C, "csam_mx_gemm: null operand");
  CSAM_REQUIRE(M > 0 && N > 0 && K > 0, "csam_mx_gemm: bad sizes M %d N %d K %d", M, N, K);
  CSAM_REQUIRE(a_fmt == CSAM_MX_FP4 || a_fmt == CSAM_MX_FP8, "csam_mx_gemm: bad format %d", a_fmt);
  CSAM_REQUIRE(K <= (1 << 20), "csam_mx_gemm: K %d is over 2^20", K);
  const int Kp = csam_cdiv(K, 256) * 256;
  auto dt_ok = [](int dt) { return dt == CSAM_DT_F16 || dt == CSAM_DT_F32 || dt == CSAM_DT_BF16; };
  auto al = [](const void* q, long ld, int a) { return (uintptr_t)q % a == 0 && ld % a == 0; };
  CSAM_REQUIRE(dt_ok(c_dtype) && (!residual || dt_ok(r_dtype)), "csam_mx_gemm: bad dtype");
  CSAM_REQUIRE(act == CSAM_ACT_NONE || act == CSAM_ACT_GELU || act == CSAM_ACT_RELU, "csam_mx_gemm: bad activation %d", act);
  CSAM_REQUIRE(lda >= (a_fmt == CSAM_MX_FP8 ? Kp : Kp / 2) && ldw >= Kp / 2, "csam_mx_gemm: code rows are shorter than %d padded columns", Kp);
  CSAM_REQUIRE(al(A, lda, 16) && al(W, ldw, 16), "csam_mx_gemm: codes and their row pitch have to be multiples of 16 bytes");
  CSAM_REQUIRE(al(A_scales, a_scale_stride, 4) && al(W_scales, w_scale_stride, 4) && a_scale_stride >= 4L * M && w_scale_stride >= 4L * N,
               "csam_mx_gemm: scale groups have to lie 4-byte aligned, at least 4 * rows bytes apart");
  CSAM_REQUIRE(ldc >= N && (!residual || ldr >= N), "csam_mx_gemm: an output row pitch is shorter than N");
  auto es = [](int dt) { return dt == CSAM_DT_F32 ? 4 : 2; };
  const int vec = al(C, ldc * es(c_dtype), 4 * es(c_dtype)) && (!residual || al(residual, ldr * es(r_dtype), 4 * es(r_dtype))) &&
                  (!bias || (uintptr_t)bias % 16 == 0);
  MxGemmArgs p = {(const uint8_t*)A, lda, (const uint8_t*)A_scales, a_scale_stride, (const uint8_t*)W, ldw, (const uint8_t*)W_scales,
                  w_scale_stride, C, ldc, c_dtype, bias, residual, ldr, r_dtype, act, M, N, Kp, vec};
  return a_fmt == CSAM_MX_FP8 ? mx_gemm_launch<CSAM_MX_FP8>((hipStream_t)stream, p) : mx_gemm_launch<CSAM_MX_FP4>((hipStream_t)stream, p);
}
