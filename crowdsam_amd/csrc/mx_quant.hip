// Quantisation to and from microscaled (MX) operands, and the root-mean-square norm that can hand its rows out as one.
// All of it is bound by memory: a pass reads each input once and writes each output once.
#include <limits.h>
#include <type_traits>
#include "mx_common.h"

namespace {

// ---------------------------------------------------------------------------------------------------------------- quantise
// A workgroup takes 8 R rows x 256 columns: 512 bytes (16-bit inputs) of a row per half-wave.  With R = 4 the scale dwords of its 32
// neighbouring rows are a whole 128-byte line per 128 columns, and no line is shared between XCDs; R = 1 where that would leave CUs idle
// (333 x 1001: 44 workgroups or 168, 5.3 or 2.5 us).  NT: codes that the L2s would not
// hold are stored past them (21320 x 4096 fp16 to E4M3: 52.4 us, 47.5 so = 5.6 TB/s; the product that reads them takes the same either way).
constexpr int Q_COLS = 256;

template <typename T, int FMT, int R, bool NT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, long ldx, uint8_t* __restrict__ codes, long ldc,
                                                          uint8_t* __restrict__ scales, long sstride, int M, int K, int nseg) {
  const int seg = blockIdx.x % nseg, r0 = (blockIdx.x / nseg) * (8 * R) + (threadIdx.x >> 5);
  const int c8 = seg * (Q_COLS / 8) + (threadIdx.x & 31), k = c8 * 8;
  float v[R][8];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + 8 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
    if (row < M && k < K) {
      if (k + 8 <= K) csam_load(x + (long)row * ldx + k, v[i]);
      else csam_load_tail(x + (long)row * ldx + k, K - k, v[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + 8 * i;
    if (row < M) csam_mx_store<FMT, NT>(v[i], codes, ldc, scales, sstride, row, c8);       // whole half-waves share a row
  }
}

// values of V = 4 or 8 consecutive codes, times their block's scale
template <int FMT, int V>
__device__ __forceinline__ void mx_values(const uint8_t* codes, float scale, float (&v)[V]) {
  float2_t w[V / 2];
  if constexpr (FMT == CSAM_MX_FP4) {
    unsigned q;
    if constexpr (V == 8) q = *(const unsigned*)codes;
    else q = *(const unsigned short*)codes;
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 0);
    w[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 1);
    if constexpr (V == 8) {
      w[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 2);
      w[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, 1.0f, 3);
    }
  } else {
    unsigned q[V / 4];
    if constexpr (V == 8) {
      const uintx2 d = *(const uintx2*)codes;
      q[0] = d[0], q[1] = d[1];
    } else q[0] = *(const unsigned*)codes;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      w[2 * i] = __builtin_amdgcn_cvt_pk_f32_fp8(q[i], false);
      w[2 * i + 1] = __builtin_amdgcn_cvt_pk_f32_fp8(q[i], true);
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = w[i / 2][i % 2] * scale;
}

// The same segments of 256 columns, a lane's V elements one 16-byte store (fp32: 20000 x 4096 from E2M1 118 us with two stores of a lane
// side by side, 55.0 so).  NT: results that the L2s would not hold go past them if their rows are whole lines (fp16: the same operand
// 38.0 us, 31.6 so; rows of 4100: 45.4, past the caches 59.3).
template <typename T, int FMT, int R, bool NT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, long ldc, const uint8_t* __restrict__ scales,
                                                            long sstride, T* __restrict__ y, long ldy, int M, int K, int nseg) {
  constexpr int V = 16 / sizeof(T), LANES = Q_COLS / V, ROWS = 256 / LANES;
  const int seg = blockIdx.x % nseg, r0 = (blockIdx.x / nseg) * (ROWS * R) + threadIdx.x / LANES;
  const int k = seg * Q_COLS + threadIdx.x % LANES * V;
  if (k >= K) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int row = r0 + ROWS * i;
    if (row >= M) continue;
    const unsigned s = scales[(long)(k >> 7) * sstride + (long)row * 4 + ((k >> 5) & 3)];
    float v[V];
    mx_values<FMT, V>(codes + row * ldc + (FMT == CSAM_MX_FP4 ? k / 2 : k), csam_e8m0(s), v);
    T* to = y + (long)row * ldy + k;
    if (k + V <= K) {
      typename csam_pack<T, V>::vec h;
#pragma unroll
      for (int e = 0; e < V; ++e) h[e] = (T)v[e];
      csam_put<NT>((typename csam_pack<T, V>::at*)to, h);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (k + e < K) to[e] = (T)v[e];
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------- RMS norm
// h = x + r, y = h * rsqrt(mean(h^2) + eps) * gamma: the row stays in registers between the sum and the scaling (one read of x and
// r, one write of h and y).  NW waves share a row of up to NW * MAXC * 512 columns; NW = 1 needs no barrier.  h is summed and scaled in
// fp32 before it is rounded to r's type.  Bound by memory: 65536 x 1280 bfloat16 with residual 112 us = 6.0 TB/s, 5330 x 1024 fp16 with an
// fp32 residual to E4M3 12 us = 5.0 TB/s.  A wave takes one row: with up to 16 rows in turn, gamma held in registers, the loads of a row
// waited for the stores of the last (143 us).
struct RmsArgs {
  const void* x; long ldx;
  const void* r; long ldr;
  void* h; long ldh;
  const float* gamma;
  float eps;
  void* y; long ldy; int y_kind;          // CSAM_DT_*, or RMS_MX + CSAM_MX_*
  uint8_t* scales; long sstride;
  int M, D, Dp;
};
constexpr int RMS_MX = 16;
// RK: 0 no residual, 1 residual of x's type, 2 fp32 residual.  A lane's chunks are V elements: 8, or 4 where a stream of a row is fp32, so
// that every access of a wave is one run (the two 16-byte halves of a lane's 8 fp32 values would part it: 65536 x 512 with an
// fp32 residual 85 us, 68 so, and with all of a row's loads in flight).
template <typename T, int RK, int NW, int MAXC, int V, bool NT>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void rms_norm_kernel(RmsArgs p) {
  typedef typename std::conditional<RK == 2, float, T>::type R;
  constexpr int SLOTS = NW == 1 ? 4 : 1;
  __shared__ float part[NW];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int slot = NW == 1 ? wave : 0;
  const int c0 = NW == 1 ? lane : (int)threadIdx.x;
  constexpr int STEP = NW * 64;
  const long row = (long)blockIdx.x * SLOTS + slot;
  if (row >= p.M) return;                                  // uniform over the waves that share the row
  const int D = p.D;
  const T* xr = (const T*)p.x + row * p.ldx;
  const R* rr = (const R*)p.r + row * p.ldr;
  // Where a whole chunk begins; lanes without one load the row's first and drop it, so that no branch parts the loads and all of a row's
  // are in flight at once (65536 x 1280 fp16 with an fp32 residual to E4M3: 202 us with a branch at every chunk, 169 so).
  auto at = [&](int j) {
    const int k = (c0 + j * STEP) * V;
    return k + V <= D ? k : 0;
  };
  float v[MAXC][V], g[MAXC][V];
  float s = 0.f;
  if (D >= V) {
    typename csam_pack<T, V>::vec x[MAXC];
    typename csam_pack<R, V>::vec r[MAXC];
#pragma unroll
    for (int j = 0; j < MAXC; ++j) {
      x[j] = *(const typename csam_pack<T, V>::at*)(xr + at(j));
      if constexpr (RK != 0) r[j] = *(const typename csam_pack<R, V>::at*)(rr + at(j));
    }
    if constexpr (NW < 16) {
#pragma unroll
      for (int j = 0; j < MAXC; ++j) csam_load(p.gamma + at(j), g[j]);
    }
#pragma unroll
    for (int j = 0; j < MAXC; ++j) {
      const bool full = (c0 + j * STEP) * V + V <= D;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float h = (float)x[j][e];
        if constexpr (RK != 0) h += (float)r[j][e];
        v[j][e] = full ? h : 0.f;
        if constexpr (NW < 16) g[j][e] = full ? g[j][e] : 0.f;     // (columns behind D are zero, whatever gamma holds)
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < MAXC; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] = g[j][e] = 0.f;
  }
  if (D % V != 0) {
#pragma unroll
    for (int j = 0; j < MAXC; ++j) {
      const int k = (c0 + j * STEP) * V;
      if (k < D && k + V > D) {
        csam_load_tail(xr + k, D - k, v[j]);
        if constexpr (NW < 16) csam_load_tail(p.gamma + k, D - k, g[j]);
        if constexpr (RK != 0) {
          float r[V];
          csam_load_tail(rr + k, D - k, r);
#pragma unroll
          for (int e = 0; e < V; ++e) v[j][e] += r[e];
        }
      }
    }
  }
  if constexpr (RK != 0) {
#pragma unroll
    for (int j = 0; j < MAXC; ++j) {
      const int k = (c0 + j * STEP) * V;
      R* hp = (R*)p.h + row * p.ldh + k;
      if (k + V <= D) csam_store<NT>(hp, v[j]);
      else csam_store_tail(hp, D - k, v[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < MAXC; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) s = fmaf(v[j][e], v[j][e], s);
  s = csam_wave_sum(s);
  if constexpr (NW > 1) {
    if (lane == 0) part[wave] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += part[w];
  }
  const float rstd = 1.0f / sqrtf(s * (1.0f / (float)D) + p.eps);
#pragma unroll
  for (int j = 0; j < MAXC; ++j) {
    const int c = c0 + j * STEP, k = c * V;
    if constexpr (NW == 16) {                              // (fewer registers: 4000 x 32768 bfloat16 266 us with gamma held from the start, 204 so)
      if (k + V <= D) csam_load(p.gamma + k, g[j]);
      else csam_load_tail(p.gamma + k, D - k, g[j]);
    }
    float y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = v[j][e] * rstd * g[j][e];
    if (p.y_kind >= RMS_MX) {
      if (k < p.Dp) {                                    // whole blocks of lanes: Dp is a multiple of 256
        if (p.y_kind == RMS_MX + CSAM_MX_FP8) csam_mx_store<CSAM_MX_FP8, NT>(y, (uint8_t*)p.y, p.ldy, p.scales, p.sstride, row, c);
        else csam_mx_store<CSAM_MX_FP4, NT>(y, (uint8_t*)p.y, p.ldy, p.scales, p.sstride, row, c);
      }
    } else if (k < D) {
      const bool full = k + V <= D;
      if (p.y_kind == CSAM_DT_F16) {
        half_t* yp = (half_t*)p.y + row * p.ldy + k;
        if (full) csam_store<NT>(yp, y); else csam_store_tail(yp, D - k, y);
      } else if (p.y_kind == CSAM_DT_BF16) {
        bf16_t* yp = (bf16_t*)p.y + row * p.ldy + k;
        if (full) csam_store<NT>(yp, y); else csam_store_tail(yp, D - k, y);
      } else {
        float* yp = (float*)p.y + row * p.ldy + k;
        if (full) csam_store<NT>(yp, y); else csam_store_tail(yp, D - k, y);
      }
    }
  }
}

template <typename T, int RK, int V, bool NT>
int rms_launch_v(hipStream_t st, const RmsArgs& p) {
  const int chunks = csam_cdiv(p.Dp ? p.Dp : p.D, 8);      // of 8
  CSAM_REQUIRE(chunks <= 256 ? csam_launch_fits(csam_cdiv(p.M, 4), 256) : csam_launch_fits(p.M, chunks <= 1024 ? 256 : 1024),
               "csam_rms_norm: %d rows of %d are more than one launch takes", p.M, p.D);
#define RMS_GO(NW, MAXC) rms_norm_kernel<T, RK, NW, MAXC * 8 / V, V, NT><<<csam_cdiv(p.M, NW == 1 ? 4 : 1), NW == 1 ? 256 : NW * 64, 0, st>>>(p)
  if (chunks <= 64) RMS_GO(1, 1);
  else if (chunks <= 128) RMS_GO(1, 2);
  else if (chunks <= 192) RMS_GO(1, 3);
  else if (chunks <= 256) RMS_GO(1, 4);
  else if (chunks <= 512) RMS_GO(4, 2);
  else if (chunks <= 1024) RMS_GO(4, 4);
  else RMS_GO(16, 4);
#undef RMS_GO
  CSAM_LAUNCH_CHECK("csam_rms_norm");
  return CSAM_OK;
}

template <typename T, int RK>
int rms_launch(hipStream_t st, const RmsArgs& p) {
  const long yb = p.y_kind >= RMS_MX ? 1 : p.y_kind == CSAM_DT_F32 ? 4 : 2, hb = RK == 0 ? 0 : RK == 2 ? 4 : (long)sizeof(T);
  // Results that the last-level cache would not hold go past the caches, whole lines or not (us through them / past them: 65536 x 1280
  // bfloat16 with residual 118 / 107, x 1279 168 / 153, x 1284 141 / 129; fp16 with an fp32 residual to E4M3 x 1280 167.5 / 163.7, x 1279
  // 182 / 175; 40000 x 4100 bfloat16 352 / 345); smaller ones stay for their reader (21320 x 1024 fp16 with an fp32 residual to E4M3: 43 us,
  // 39 past the caches, but with the product that reads both 83, past the caches 88).
  const bool past = (long)p.M * p.D * (yb + hb) > (256L << 20);
  if constexpr (sizeof(T) == 4 || RK == 2) return past ? rms_launch_v<T, RK, 4, true>(st, p) : rms_launch_v<T, RK, 4, false>(st, p);
  else if (p.y_kind == CSAM_DT_F32) return past ? rms_launch_v<T, RK, 4, true>(st, p) : rms_launch_v<T, RK, 4, false>(st, p);
  else return past ? rms_launch_v<T, RK, 8, true>(st, p) : rms_launch_v<T, RK, 8, false>(st, p);
}

bool aligned(const void* p, long ld_bytes, int a) { return ((uintptr_t)p % a) == 0 && ld_bytes % a == 0; }
int dt_bytes(int dt) { return dt == CSAM_DT_F32 ? 4 : 2; }
bool dt_ok(int dt) { return dt == CSAM_DT_F16 || dt == CSAM_DT_F32 || dt == CSAM_DT_BF16; }

// checks shared by everything that reads or writes an MX operand
int mx_check(const char* who, const void* codes, long ldc, const void* scales, long sstride, int fmt, int M, int K) {
  CSAM_REQUIRE(codes && scales, "%s: null operand", who);
  CSAM_REQUIRE(fmt == CSAM_MX_FP4 || fmt == CSAM_MX_FP8, "%s: format %d is neither CSAM_MX_FP4 nor CSAM_MX_FP8", who, fmt);
  CSAM_REQUIRE(M <= INT_MAX - 255 && K <= INT_MAX - 255, "%s: %d x %d is over 2^31 - 256 rows or columns", who, M, K);
  const long Kp = (K + 255L) / 256 * 256;
  CSAM_REQUIRE(ldc >= (fmt == CSAM_MX_FP4 ? Kp / 2 : Kp), "%s: code rows of %ld bytes are shorter than %ld padded columns", who, ldc, Kp);
  CSAM_REQUIRE(aligned(codes, ldc, 16), "%s: codes and their row pitch have to be multiples of 16 bytes", who);
  CSAM_REQUIRE(aligned(scales, sstride, 4) && sstride >= 4L * M, "%s: scale groups have to lie 4-byte aligned, at least 4 * rows bytes apart", who);
  return CSAM_OK;
}

}  // namespace

extern "C" {

int csam_mx_quantize(void* stream, const void* x, long ldx, int x_dtype, void* codes, long ldcodes, void* scales, long scale_stride,
                     int fmt, int M, int K) {
  if (M == 0) return CSAM_OK;
  CSAM_REQUIRE(x, "csam_mx_quantize: null operand");
  CSAM_REQUIRE(M > 0 && K > 0 && ldx >= K, "csam_mx_quantize: bad sizes M %d K %d ldx %ld", M, K, ldx);
  CSAM_REQUIRE(dt_ok(x_dtype), "csam_mx_quantize: bad dtype %d", x_dtype);
  if (int rc = mx_check("csam_mx_quantize", codes, ldcodes, scales, scale_stride, fmt, M, K)) return rc;
  const int nseg = csam_cdiv(K, Q_COLS);
  const long grid = (long)nseg * csam_cdiv(M, 8);
  CSAM_REQUIRE(csam_launch_fits((long)nseg * csam_cdiv(M, 32), 256), "csam_mx_quantize: %d x %d is more than one launch takes", M, K);
  hipStream_t st = (hipStream_t)stream;
#define GO(T, F)                                                                                                         \
  do {                                                                                                                   \
    const unsigned g4 = (unsigned)((long)nseg * csam_cdiv(M, 32));                                                       \
    if ((long)M * ldcodes > (32L << 20)) mx_quantize_kernel<T, F, 4, true><<<g4, 256, 0, st>>>((const T*)x, ldx, (uint8_t*)codes, ldcodes, (uint8_t*)scales, scale_stride, M, K, nseg); \
    else if (grid >= 2048) mx_quantize_kernel<T, F, 4, false><<<g4, 256, 0, st>>>((const T*)x, ldx, (uint8_t*)codes, ldcodes, (uint8_t*)scales, scale_stride, M, K, nseg); \
    else mx_quantize_kernel<T, F, 1, false><<<(unsigned)grid, 256, 0, st>>>((const T*)x, ldx, (uint8_t*)codes, ldcodes, (uint8_t*)scales, scale_stride, M, K, nseg); \
  } while (0)
  if (fmt == CSAM_MX_FP4) {
    if (x_dtype == CSAM_DT_F16) GO(half_t, CSAM_MX_FP4);
    else if (x_dtype == CSAM_DT_F32) GO(float, CSAM_MX_FP4);
    else GO(bf16_t, CSAM_MX_FP4);
  } else {
    if (x_dtype == CSAM_DT_F16) GO(half_t, CSAM_MX_FP8);
    else if (x_dtype == CSAM_DT_F32) GO(float, CSAM_MX_FP8);
    else GO(bf16_t, CSAM_MX_FP8);
  }
#undef GO
  CSAM_LAUNCH_CHECK("csam_mx_quantize");
  return CSAM_OK;
}

int csam_mx_dequantize(void* stream, const void* codes, long ldcodes, const void* scales, long scale_stride, int fmt, void* y, long ldy,
                       int y_dtype, int M, int K) {
  if (M == 0) return CSAM_OK;
  CSAM_REQUIRE(y, "csam_mx_dequantize: null operand");
  CSAM_REQUIRE(M > 0 && K > 0 && ldy >= K, "csam_mx_dequantize: bad sizes M %d K %d ldy %ld", M, K, ldy);
  CSAM_REQUIRE(dt_ok(y_dtype), "csam_mx_dequantize: bad dtype %d", y_dtype);
  if (int rc = mx_check("csam_mx_dequantize", codes, ldcodes, scales, scale_stride, fmt, M, K)) return rc;
  const int nseg = csam_cdiv(K, Q_COLS);
  const long grid = (long)nseg * csam_cdiv(M, 8);
  CSAM_REQUIRE(csam_launch_fits((long)nseg * csam_cdiv(M, y_dtype == CSAM_DT_F32 ? 16 : 32), 256),
               "csam_mx_dequantize: %d x %d is more than one launch takes", M, K);
  hipStream_t st = (hipStream_t)stream;
#define GO(T, F)                                                                                                         \
  do {                                                                                                                   \
    constexpr int ROWS = sizeof(T) == 4 ? 4 : 8;                                                                         \
    const unsigned g1 = (unsigned)((long)nseg * csam_cdiv(M, ROWS)), g4 = (unsigned)((long)nseg * csam_cdiv(M, 4 * ROWS)); \
    const bool past = (long)M * ldy * sizeof(T) > (32L << 20) && aligned(y, ldy * sizeof(T), 128);                      \
    if (past) mx_dequantize_kernel<T, F, 4, true><<<g4, 256, 0, st>>>((const uint8_t*)codes, ldcodes, (const uint8_t*)scales, scale_stride, (T*)y, ldy, M, K, nseg); \
    else if (grid >= 2048) mx_dequantize_kernel<T, F, 4, false><<<g4, 256, 0, st>>>((const uint8_t*)codes, ldcodes, (const uint8_t*)scales, scale_stride, (T*)y, ldy, M, K, nseg); \
    else mx_dequantize_kernel<T, F, 1, false><<<g1, 256, 0, st>>>((const uint8_t*)codes, ldcodes, (const uint8_t*)scales, scale_stride, (T*)y, ldy, M, K, nseg); \
  } while (0)
  if (fmt == CSAM_MX_FP4) {
    if (y_dtype == CSAM_DT_F16) GO(half_t, CSAM_MX_FP4);
    else if (y_dtype == CSAM_DT_F32) GO(float, CSAM_MX_FP4);
    else GO(bf16_t, CSAM_MX_FP4);
  } else {
    if (y_dtype == CSAM_DT_F16) GO(half_t, CSAM_MX_FP8);
    else if (y_dtype == CSAM_DT_F32) GO(float, CSAM_MX_FP8);
    else GO(bf16_t, CSAM_MX_FP8);
  }
#undef GO
  CSAM_LAUNCH_CHECK("csam_mx_dequantize");
  return CSAM_OK;
}

static int rms_any(hipStream_t st, RmsArgs& p, int x_dtype, int r_dtype, const char* who) {
  CSAM_REQUIRE(p.x && p.gamma && p.y, "%s: null operand", who);
  CSAM_REQUIRE((p.r == nullptr) == (p.h == nullptr), "%s: the residual and the sum's output come together", who);
  CSAM_REQUIRE(p.M > 0 && p.D > 0 && p.D <= 32768, "%s: bad sizes M %d D %d (D <= 32768)", who, p.M, p.D);
  CSAM_REQUIRE(p.ldx >= p.D && (!p.r || (p.ldr >= p.D && p.ldh >= p.D)), "%s: a row pitch is shorter than the row", who);
  CSAM_REQUIRE(dt_ok(x_dtype), "%s: bad dtype %d", who, x_dtype);
  CSAM_REQUIRE(!p.r || r_dtype == x_dtype || r_dtype == CSAM_DT_F32, "%s: the residual is fp32 or of x's type", who);
  CSAM_REQUIRE(p.eps > 0.f, "%s: eps has to be positive", who);
  const int rk = !p.r ? 0 : (r_dtype == CSAM_DT_F32 && x_dtype != CSAM_DT_F32) ? 2 : 1;
#define GO(T) return rk == 0 ? rms_launch<T, 0>(st, p) : rk == 1 ? rms_launch<T, 1>(st, p) : rms_launch<T, 2>(st, p)
  if (x_dtype == CSAM_DT_F16) GO(half_t);
  if (x_dtype == CSAM_DT_BF16) GO(bf16_t);
#undef GO
  return rk == 0 ? rms_launch<float, 0>(st, p) : rms_launch<float, 1>(st, p);
}

int csam_rms_norm(void* stream, const void* x, long ldx, int x_dtype, const void* residual, long ldr, int r_dtype, void* h, long ldh,
                  const float* gamma, float eps, void* y, long ldy, int y_dtype, int M, int D) {
  if (M == 0) return CSAM_OK;
  CSAM_REQUIRE(dt_ok(y_dtype) && ldy >= D, "csam_rms_norm: bad output dtype %d or row pitch %ld", y_dtype, ldy);
  RmsArgs p = {x, ldx, residual, ldr, h, ldh, gamma, eps, y, ldy, y_dtype, nullptr, 0, M, D, 0};
  return rms_any((hipStream_t)stream, p, x_dtype, r_dtype, "csam_rms_norm");
}

int csam_rms_norm_mx(void* stream, const void* x, long ldx, int x_dtype, const void* residual, long ldr, int r_dtype, void* h, long ldh,
                     const float* gamma, float eps, void* codes, long ldcodes, void* scales, long scale_stride, int fmt, int M, int D) {
  if (M == 0) return CSAM_OK;
  CSAM_REQUIRE(D > 0, "csam_rms_norm_mx: bad width %d", D);
  if (int rc = mx_check("csam_rms_norm_mx", codes, ldcodes, scales, scale_stride, fmt, M, D)) return rc;
  RmsArgs p = {x, ldx, residual, ldr, h, ldh, gamma, eps, codes, ldcodes, RMS_MX + fmt, (uint8_t*)scales, scale_stride, M, D,
               csam_cdiv(D, 256) * 256};
  return rms_any((hipStream_t)stream, p, x_dtype, r_dtype, "csam_rms_norm_mx");
}

}  // extern "C"
