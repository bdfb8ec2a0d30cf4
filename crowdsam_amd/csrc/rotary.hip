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
  sincospif(f, &s, &c);
}

// One thread = one unit of one token for every `split`-th head: the angles are computed once and used for all of its heads, HB of which are
// fetched together (the first HB before the angles are computed).
//   half:        VW elements of the first half of the pairs and their VW partners, or VW elements that pass through;
//   interleaved: VW consecutive elements = VW / 2 pairs.
// Consecutive threads hold consecutive units of a head, then the next head phase: a wave touches whole runs of the row.
template <typename T, bool HALF, int VW>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  typedef typename csam_pack<T, VW>::vec vec_t;
  typedef typename csam_pack<T, VW>::at vec_at;
  constexpr int HB = 4;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const unsigned tw = idx / p.units;
  const int u = idx - tw * p.units;
  const unsigned t = tw / p.split;
  const int s0 = tw - t * p.split;
  if (t >= (unsigned)p.T) return;
  const int H = p.Hq + p.Hk;

  // where the unit's elements are and what happens to them
  constexpr int NP = HALF ? VW : VW / 2;
  const int pair0 = u * NP;
  const bool turn = pair0 < p.P;
  const int i0 = HALF && !turn ? u * VW + p.P : u * VW;
  vec_t v[HB], w[HB];
  const bool lone = !HALF && VW == 2 && i0 + 1 == p.hd;        // the last element of a head of odd width
  auto head = [&](int h, bool out) {
    if (h < p.Hq) {
      return out ? (char*)p.qo + ((long)t * p.ldqo + (long)h * p.hsqo) * (long)sizeof(T) : (char*)p.q + ((long)t * p.ldq + (long)h * p.hsq) * (long)sizeof(T);
    }
    h -= p.Hq;
    return out ? (char*)p.ko + ((long)t * p.ldko + (long)h * p.hsko) * (long)sizeof(T) : (char*)p.k + ((long)t * p.ldk + (long)h * p.hsk) * (long)sizeof(T);
  };
  auto fetch = [&](int h0) {
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int h = h0 + b * p.split;
      if (h < H) {
        const T* src = (const T*)head(h, false);
        if (!HALF && VW == 2 && lone) v[b][0] = src[i0];
        else v[b] = *(const vec_at*)(src + i0);
        if (HALF && turn) w[b] = *(const vec_at*)(src + i0 + p.P);
      }
    }
  };
  fetch(s0);
  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    cs[i] = 1.f, sn[i] = 0.f;
    if (pair0 + i < p.P) rotary_angle(p, (int)t, pair0 + i, cs[i], sn[i]);
  }
  for (int h0 = s0; h0 < H; h0 += HB * p.split) {
    if (h0 != s0) fetch(h0);
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int h = h0 + b * p.split;
      if (h >= H) break;
      T* dst = (T*)head(h, true);
      if constexpr (HALF) {
        if (turn) {
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            const float x = (float)v[b][i], y = (float)w[b][i];
            v[b][i] = (T)(x * cs[i] - y * sn[i]);
            w[b][i] = (T)(x * sn[i] + y * cs[i]);
          }
          *(vec_at*)(dst + i0 + p.P) = w[b];
        }
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (pair0 + i < p.P) {                     // a pair behind the last one passes through bit for bit
            const float x = (float)v[b][2 * i], y = (float)v[b][2 * i + 1];
            v[b][2 * i] = (T)(x * cs[i] - y * sn[i]);
            v[b][2 * i + 1] = (T)(x * sn[i] + y * cs[i]);
          }
        }
      }
      if (!HALF && VW == 2 && lone) dst[i0] = v[b][0];
      else *(vec_at*)(dst + i0) = v[b];
    }
  }
}

template <typename T, bool HALF, int VW>
int rotary_go(hipStream_t st, RotaryArgs& p) {
  p.units = csam_cdiv(HALF ? p.hd - p.P : p.hd, VW);
  // heads of a thread: the angles cost a thread about as much as eight heads, but a small call wants threads more than it minds angles
  const int H = p.Hq + p.Hk;
  const long per_head = (long)p.T * p.units;
  p.split = per_head * csam_cdiv(H, 8) >= 262144 ? csam_cdiv(H, 8) : per_head * csam_cdiv(H, 4) >= 65536 ? csam_cdiv(H, 4) : H;
  const long n = per_head * p.split;
  CSAM_REQUIRE(n < (1L << 31), "csam_rotary: too many elements");
  rotary_kernel<T, HALF, VW><<<(unsigned)csam_cdiv(n, 256), 256, 0, st>>>(p);
  CSAM_LAUNCH_CHECK("csam_rotary");
  return CSAM_OK;
}

// the widest accesses that units of whole accesses allow (addresses need no alignment beyond an element's)
template <typename T>
int rotary_launch(hipStream_t st, RotaryArgs& p, int half) {
  constexpr int W = 16 / sizeof(T);
  const int odd = half ? p.P | p.hd : p.hd;
  if (odd % W == 0) return half ? rotary_go<T, true, W>(st, p) : rotary_go<T, false, W>(st, p);
  if (W == 8 && odd % 4 == 0) return half ? rotary_go<T, true, 4>(st, p) : rotary_go<T, false, 4>(st, p);
  if (!half) return rotary_go<T, false, 2>(st, p);
  return odd % 2 == 0 ? rotary_go<T, true, 2>(st, p) : rotary_go<T, true, 1>(st, p);
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
