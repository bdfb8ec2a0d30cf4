// Rotary positions with several axes: the q and k heads of token-major rows, rotated by angles that are the products of a token's
// position along an axis (row, column, time) and a frequency per pair of elements.
#include "mx_common.h"

namespace {

struct RotaryArgs {
  const void* q; void* qo; long ldq, ldqo;          // row pitches in elements
  const void* k; void* ko; long ldk, ldko;
  int hsq, hsqo, hsk, hsko;                         // head pitches in elements
  const void* pos; long pos_stride; int pos_f32;    // [axes][Tp]
  const double* freq; const int* axis;              // [P] radians per unit, axis of each pair
  int T, Tp, Hq, Hk, hd, P, axes;
  int units, split;                                 // units of a head, head phases of a token
};

// cos and sin of pos * freq.  The product and its reduction to one turn are in fp64: at a position of 1e5 an fp32 angle is off by
// 4e-3 radians.  What is left is in [-1/2, 1/2] turns, where the fp32 functions are exact to an ulp.
__device__ __forceinline__ void rotary_angle(const RotaryArgs& p, int t, int pair, float& c, float& s) {
  const int ax = min(max(p.axis[pair], 0), p.axes - 1);
  const long at = (long)ax * p.pos_stride + t % p.Tp;
  const double x = p.pos_f32 ? (double)((const float*)p.pos)[at] : (double)((const int*)p.pos)[at];
  const double turns = x * p.freq[pair] * 0.15915494309189533577;
  const float f = 2.0f * (float)(turns - __builtin_rint(turns));
  c = cospif(f);
  s = sinpif(f);
}

// One thread = one unit of one token for every `split`-th head: the angles are computed once and used for all of its heads.
//   VEC, half:        VW elements of the first half of the pairs and their VW partners, or VW elements that pass through;
//   VEC, interleaved: VW consecutive elements = VW / 2 pairs;
//   scalar:           one pair, or one element that passes through.
// Consecutive threads hold consecutive units of a head, then the next head phase: a wave touches whole runs of the row.
template <typename T, bool HALF, bool VEC>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  constexpr int VW = VEC ? 16 / sizeof(T) : 1;
  typedef T vec_t __attribute__((ext_vector_type(VW)));
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const unsigned tw = idx / p.units;
  const int u = idx - tw * p.units;
  const unsigned t = tw / p.split;
  const int s0 = tw - t * p.split;
  if (t >= (unsigned)p.T) return;
  const int H = p.Hq + p.Hk;

  // where the unit's elements are and what happens to them
  int i0, i1 = -1;                                   // i1 < 0: only VW elements at i0
  constexpr int NP = VEC ? (HALF ? VW : VW / 2) : 1;
  float cs[NP], sn[NP];
  bool turn = true;
  if constexpr (VEC && HALF) {
    turn = u * VW < p.P;
    i0 = turn ? u * VW : u * VW + p.P;
    if (turn) i1 = i0 + p.P;
  } else if constexpr (VEC) {
    i0 = u * VW;
    turn = i0 < 2 * p.P;
  } else {
    turn = u < p.P;
    i0 = turn ? (HALF ? u : 2 * u) : u + p.P;
    if (turn) i1 = i0 + (HALF ? p.P : 1);
  }
  const int pair0 = VEC && !HALF ? u * NP : u * (VEC ? VW : 1);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    cs[i] = 1.f, sn[i] = 0.f;
    if (turn && pair0 + i < p.P) rotary_angle(p, (int)t, pair0 + i, cs[i], sn[i]);
  }
  for (int h = s0; h < H; h += p.split) {
    const bool isq = h < p.Hq;
    const T* src = isq ? (const T*)p.q + (long)t * p.ldq + (long)h * p.hsq : (const T*)p.k + (long)t * p.ldk + (long)(h - p.Hq) * p.hsk;
    T* dst = isq ? (T*)p.qo + (long)t * p.ldqo + (long)h * p.hsqo : (T*)p.ko + (long)t * p.ldko + (long)(h - p.Hq) * p.hsko;
    if constexpr (VEC && !HALF) {
      vec_t v = *(const vec_t*)(src + i0);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (pair0 + i < p.P) {                       // a pair behind the last one passes through bit for bit
          const float a = (float)v[2 * i], b = (float)v[2 * i + 1];
          v[2 * i] = (T)(a * cs[i] - b * sn[i]);
          v[2 * i + 1] = (T)(a * sn[i] + b * cs[i]);
        }
      }
      *(vec_t*)(dst + i0) = v;
    } else {
      vec_t v = *(const vec_t*)(src + i0);
      if (i1 >= 0) {
        vec_t w = *(const vec_t*)(src + i1);
#pragma unroll
        for (int i = 0; i < VW; ++i) {
          const float a = (float)v[i], b = (float)w[i];
          v[i] = (T)(a * cs[i] - b * sn[i]);
          w[i] = (T)(a * sn[i] + b * cs[i]);
        }
        *(vec_t*)(dst + i1) = w;
      }
      *(vec_t*)(dst + i0) = v;
    }
  }
}

template <typename T>
int rotary_launch(hipStream_t st, RotaryArgs& p, int half) {
  constexpr int VW = 16 / sizeof(T);
  auto al = [&](const void* b, long ld, long hs) { return !b || ((uintptr_t)b % 16 == 0 && ld % VW == 0 && hs % VW == 0); };
  const bool vec = al(p.q, p.ldq, p.hsq) && al(p.qo, p.ldqo, p.hsqo) && al(p.k, p.ldk, p.hsk) && al(p.ko, p.ldko, p.hsko) &&
                   p.hd % VW == 0 && (!half || p.P % VW == 0);
  p.units = !vec ? p.P + (p.hd - 2 * p.P) : half ? (p.hd - p.P) / VW : p.hd / VW;
  const int H = p.Hq + p.Hk;
  p.split = csam_cdiv(H, 4);
  const long n = (long)p.T * p.units * p.split;
  CSAM_REQUIRE(n < (1L << 31), "csam_rotary: too many elements");
  const unsigned grid = (unsigned)csam_cdiv(n, 256);
  if (vec) {
    if (half) rotary_kernel<T, true, true><<<grid, 256, 0, st>>>(p);
    else rotary_kernel<T, false, true><<<grid, 256, 0, st>>>(p);
  } else {
    if (half) rotary_kernel<T, true, false><<<grid, 256, 0, st>>>(p);
    else rotary_kernel<T, false, false><<<grid, 256, 0, st>>>(p);
  }
  CSAM_LAUNCH_CHECK("csam_rotary");
  return CSAM_OK;
}

}  // namespace

extern "C" int csam_rotary(void* stream, const void* q, long ldq, int hsq, void* q_out, long ldqo, int hsqo, int Hq, const void* k,
                           long ldk, int hsk, void* k_out, long ldko, int hsko, int Hk, int dtype, const void* pos, long pos_stride,
                           int pos_is_f32, const double* freq, const int* axis, int axes, int pairs, int interleaved, int T, int T_pos,
                           int head_dim) {
  if (T == 0) return CSAM_OK;
  CSAM_REQUIRE(q && q_out && pos && freq && axis && (!Hk || (k && k_out)), "csam_rotary: null operand");
  CSAM_REQUIRE(T > 0 && Hq > 0 && Hk >= 0 && head_dim > 0 && axes > 0, "csam_rotary: bad sizes T %d Hq %d Hk %d head_dim %d axes %d", T, Hq, Hk,
               head_dim, axes);
  CSAM_REQUIRE(pairs > 0 && 2 * (long)pairs <= head_dim, "csam_rotary: %d pairs do not fit a head of %d", pairs, head_dim);
  CSAM_REQUIRE(T_pos > 0 && T % T_pos == 0 && pos_stride >= T_pos, "csam_rotary: %d tokens are not a multiple of %d positions", T, T_pos);
  CSAM_REQUIRE(dtype == CSAM_DT_F16 || dtype == CSAM_DT_F32 || dtype == CSAM_DT_BF16, "csam_rotary: bad dtype %d", dtype);
  CSAM_REQUIRE(hsq >= head_dim && hsqo >= head_dim && (!Hk || (hsk >= head_dim && hsko >= head_dim)), "csam_rotary: heads overlap");
  RotaryArgs p = {q, q_out, ldq, ldqo, Hk ? k : nullptr, Hk ? k_out : nullptr, ldk, ldko, hsq, hsqo, hsk, hsko, pos, pos_stride, pos_is_f32,
                  freq, axis, T, T_pos, Hq, Hk, head_dim, pairs, axes, 0, 0};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CSAM_DT_F16) return rotary_launch<half_t>(st, p, !interleaved);
  if (dtype == CSAM_DT_BF16) return rotary_launch<bf16_t>(st, p, !interleaved);
  return rotary_launch<float>(st, p, !interleaved);
}
