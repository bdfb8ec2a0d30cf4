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
  int tokens, heads, splits;                        // tokens and heads of a workgroup, workgroups that share a token's heads
  int units, turning, Pp;                           // units of a head, those that rotate (half); P rounded up to whole units' table reads
  unsigned by_unit, by_token, by_pair;              // ceil(2^32 / d) for d = units, heads * units, P
};
constexpr int ROT_TABLE = 2048;                     // (cos, sin) entries of a workgroup's table: 16 KB (and one unit's over)

// n / d by d's reciprocal: exact while n * d < 2^32, and every n here is below 2^16
__device__ __forceinline__ unsigned rot_div(unsigned n, unsigned r, int d) { return d == 1 ? n : __umulhi(n, r); }

// cos and sin of pos * freq.  The product and its reduction to one turn are in fp64: at a position of 1e5 an fp32 angle is off by
// 4e-3 radians.  What is left is in [-1/2, 1/2] turns, where the fp32 functions are exact to an ulp.
__device__ __forceinline__ float2_t rotary_angle(const RotaryArgs& p, int t, int pair) {
  // a token's positions do not depend on the pair's axis: those of the first four axes are fetched beside it
  const int at = t % p.Tp;
  int w[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) w[a] = a < p.axes ? ((const int*)p.pos)[(long)a * p.pos_stride + at] : 0;
  const double f = p.freq[pair];
  const int ax = min(max(p.axis[pair], 0), p.axes - 1);
  int v = ax == 0 ? w[0] : ax == 1 ? w[1] : ax == 2 ? w[2] : w[3];
  if (ax > 3) v = ((const int*)p.pos)[(long)ax * p.pos_stride + at];
  const double x = p.pos_f32 ? (double)__builtin_bit_cast(float, v) : (double)v;
  const double turns = x * f * 0.15915494309189533577;
  float c, s;
  sincospif(2.0f * (float)(turns - __builtin_rint(turns)), &s, &c);
  return float2_t{c, s};
}

// Bound by memory: 16384 tokens x 32 heads of 80 fp16, interleaved, 34 us = 4.9 TB/s; 32 heads of 128, half, 42 us = 6.4 TB/s.
// A workgroup takes `tokens` tokens x `heads` heads: it puts cos and sin of each of its tokens and pairs into LDS once, and walks its
// units, HB of a thread's at a time, the first of them fetched before the angles are computed:
//   half:        VW elements of the first half of the pairs and their VW partners, or VW elements that pass through;
//   interleaved: VW consecutive elements = VW / 2 pairs.
// What is left of a run of the head behind its whole units (PIECES) is units of VW / 2, VW / 4, .. 1 elements, as its length has bits
// (16384 tokens x 32 heads of 64 with 17 pairs, half, fp16: 48.0 us; with accesses of one element throughout 93.3).
// Consecutive threads hold consecutive units of a head, then the next head: a wave touches whole runs of the row.
template <int VW>
__device__ __forceinline__ int rotary_unit(int u, int n, int& size) {         // unit u of a run of n elements: where it begins, its size
  const int whole = n / VW, j = u - whole;
  size = VW;
  if (j < 0) return u * VW;
  int at = whole * VW, k = 0;
#pragma unroll
  for (int s = VW / 2, found = 0; s; s >>= 1) {
    const bool bit = n & s, mine = bit && k == j;
    if (mine) size = s, found = 1;
    at += bit && !found ? s : 0;
    k += bit;
  }
  return at;
}
template <typename T, int VW, int N>
__device__ __forceinline__ void rotary_take(const T* p, int size, typename csam_pack<T, VW>::vec& v) {
  if (size == N) {
    const auto h = *(const typename csam_pack<T, N>::at*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = h[i];
  }
  if constexpr (N > 1) rotary_take<T, VW, N / 2>(p, size, v);
}
template <typename T, int VW, int N, bool NT>
__device__ __forceinline__ void rotary_give(T* p, int size, const typename csam_pack<T, VW>::vec& v) {
  if (size == N) {
    typename csam_pack<T, N>::vec h;
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = v[i];
    csam_put<NT>((typename csam_pack<T, N>::at*)p, h);
  }
  if constexpr (N > 1) rotary_give<T, VW, N / 2, NT>(p, size, v);
}

template <typename T, bool HALF, int VW, bool PIECES, bool NT>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  typedef typename csam_pack<T, VW>::vec vec_t;
  typedef typename csam_pack<T, VW>::at vec_at;
  constexpr int HB = 4, NP = HALF ? VW : VW / 2;
  __shared__ __attribute__((aligned(16))) float2_t table[ROT_TABLE + NP];
  const int hb = blockIdx.x % p.splits * p.heads;
  const int t0 = (int)(blockIdx.x / p.splits) * p.tokens, nt = min(p.tokens, p.T - t0);
  const int H = p.Hq + p.Hk, per_token = p.heads * p.units, total = nt * per_token;

  vec_t v[HB], w[HB];
  T* dst[HB];                                       // where the unit goes; null: no unit
  short pair0[HB], tl[HB], size[HB];                // its first pair, token and elements
  auto fetch = [&](int first) {
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      const int idx = first + b * 256;
      dst[b] = nullptr;
      if (idx >= total) continue;
      const int tk = (int)rot_div(idx, p.by_token, per_token), r = idx - tk * per_token, hl = (int)rot_div(r, p.by_unit, p.units), u = r - hl * p.units;
      const int h = hb + hl;
      if (h >= H) continue;
      const long t = t0 + tk;
      const bool turn = !HALF || u < p.turning;     // of a half layout's units, the first `turning` rotate, the others pass through
      int i0, sz = VW;
      if constexpr (PIECES) i0 = turn ? rotary_unit<VW>(u, HALF ? p.P : p.hd, sz) : rotary_unit<VW>(u - p.turning, p.hd - 2 * p.P, sz);
      else i0 = (turn ? u : u - p.turning) * VW;
      pair0[b] = (short)(turn ? (HALF ? i0 : i0 >> 1) : p.P);
      if (!turn) i0 += 2 * p.P;
      tl[b] = (short)tk;
      size[b] = (short)sz;
      const bool isq = h < p.Hq;
      const T* src = (isq ? (const T*)p.q + t * p.ldq + (long)h * p.hsq : (const T*)p.k + t * p.ldk + (long)(h - p.Hq) * p.hsk) + i0;
      dst[b] = (isq ? (T*)p.qo + t * p.ldqo + (long)h * p.hsqo : (T*)p.ko + t * p.ldko + (long)(h - p.Hq) * p.hsko) + i0;
      if constexpr (PIECES) {
        rotary_take<T, VW, VW>(src, sz, v[b]);
        if (HALF && turn) rotary_take<T, VW, VW>(src + p.P, sz, w[b]);
      } else {
        v[b] = *(const vec_at*)src;
        if (HALF && turn) w[b] = *(const vec_at*)(src + p.P);
      }
    }
  };
  auto store = [&](T* to, int sz, const vec_t& x) {
    if constexpr (PIECES) rotary_give<T, VW, VW, NT>(to, sz, x);
    else csam_put<NT>((vec_at*)to, x);
  };
  fetch(threadIdx.x);
  for (int i = threadIdx.x; i < nt * p.P; i += 256) {
    const int tk = (int)rot_div(i, p.by_pair, p.P), pair = i - tk * p.P;
    table[tk * p.Pp + pair] = rotary_angle(p, t0 + tk, pair);
  }
  __syncthreads();
  for (int first = threadIdx.x; first < total; first += 256 * HB) {
    if (first != (int)threadIdx.x) fetch(first);
#pragma unroll
    for (int b = 0; b < HB; ++b) {
      if (!dst[b]) continue;
      const bool turn = pair0[b] < p.P;
      float2_t cs[NP];                              // (entries behind the last pair are read and not used)
      if (turn) {
#pragma unroll
        for (int i = 0; i < NP; ++i) cs[i] = table[tl[b] * p.Pp + pair0[b] + i];
      }
      if constexpr (HALF) {
        if (turn) {
#pragma unroll
          for (int i = 0; i < VW; ++i) {
            const float x = (float)v[b][i], y = (float)w[b][i];
            v[b][i] = (T)(x * cs[i][0] - y * cs[i][1]);
            w[b][i] = (T)(x * cs[i][1] + y * cs[i][0]);
          }
          store(dst[b] + p.P, size[b], w[b]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          if (pair0[b] + i < p.P) {                  // a pair behind the last one passes through bit for bit
            const float x = (float)v[b][2 * i], y = (float)v[b][2 * i + 1];
            v[b][2 * i] = (T)(x * cs[i][0] - y * cs[i][1]);
            v[b][2 * i + 1] = (T)(x * cs[i][1] + y * cs[i][0]);
          }
        }
      }
      store(dst[b], size[b], v[b]);
    }
  }
}

// the widest accesses, at any element's address
template <typename T, bool HALF>
int rotary_launch(hipStream_t st, RotaryArgs& p) {
  constexpr int VW = 16 / sizeof(T), NP = HALF ? VW : VW / 2, HB = 4;
  const int rest = p.hd - 2 * p.P;
  const bool pieces = HALF ? p.P % VW || rest % VW : p.hd % VW;
  auto units = [](int n) { return n / VW + __builtin_popcount((unsigned)n % VW); };
  p.turning = HALF ? units(p.P) : 0;
  p.units = HALF ? p.turning + units(rest) : units(p.hd);
  p.Pp = csam_cdiv(p.P, NP) * NP;
  const int H = p.Hq + p.Hk;
  // A workgroup's units: one batch of its threads (16384 tokens x 32 heads of 80: 39.8 us, 45.4 with two batches).  A token with more is
  // shared by workgroups, tokens with fewer share one; a call that would not give every CU a workgroup this way is cut finer.
  const long all = (long)p.T * H * p.units, want = all >= 256L * 256 * HB ? 256 * HB : max(256L, all / 256);
  p.heads = (int)max(1L, min((long)H, want / p.units));
  p.splits = csam_cdiv(H, p.heads);
  p.tokens = (int)max(1L, min(min((long)p.T, (long)ROT_TABLE / p.Pp), want / ((long)p.heads * p.units)));
  auto recip = [](long d) { return (unsigned)(((1ULL << 32) + d - 1) / d); };
  p.by_unit = recip(p.units);
  p.by_token = recip((long)p.heads * p.units);
  p.by_pair = recip(p.P);
  const long grid = (long)csam_cdiv(p.T, p.tokens) * p.splits;
  CSAM_REQUIRE(csam_launch_fits(grid, 256), "csam_rotary: %d tokens x %d heads of %d are more than one launch takes", p.T, H, p.hd);
  // Results beyond the L2s' size that do not overwrite their input are stored past the caches where lines belong to one store each: lines
  // that two stores fill have to meet in the L2.  us through the caches / past them, fp16:
  //   half, runs of whole lines of 128 bytes: 16384 tokens x 32 heads of 128 with 64 pairs 49.0 / 42.3; in place 44.7 / 48.9
  //   the same 16 bytes off the lines: 51.4 / 99.0; runs of 64 bytes (heads of 64 with 32 pairs) 24.3 / 27.2, of 80 (80 with 40) 32.3 / 61.6
  //   interleaved: a wave's stores are one run over the heads, only its ends share lines: 32 heads of 128 48.3 / 41.6, 6 bytes off the lines
  //   54.8 / 45.0, of 80 30.3 / 28.6, in place 31.1 / 31.0
  //   interleaved with pieces, which share a line each: 64 heads of 36 33.6 / 50.3, 32 of 97 46.0 / 49.0, 20 of 250 86.4 / 69.6; fp32: 64
  //   heads of 34 69.7 / 50.6, 32 of 97 89.6 / 66.5
  constexpr long LINE = 128;
  auto whole = [&](const void* to, long ld, long hs) { return (uintptr_t)to % LINE == 0 && ld * sizeof(T) % LINE == 0 && hs * sizeof(T) % LINE == 0; };
  const bool lines = HALF ? p.P * sizeof(T) % LINE == 0 && rest * sizeof(T) % LINE == 0 && whole(p.qo, p.ldqo, p.hsqo) &&
                                (!p.Hk || whole(p.ko, p.ldko, p.hsko))
                          : !pieces || p.hd * (long)sizeof(T) >= LINE;
  const bool past = lines && p.qo != p.q && (long)p.T * H * p.hd * (long)sizeof(T) > (32L << 20);
  if (pieces && past) {                              // (half layouts of whole lines have no pieces)
    if constexpr (!HALF) rotary_kernel<T, HALF, VW, true, true><<<(unsigned)grid, 256, 0, st>>>(p);
  } else if (pieces) rotary_kernel<T, HALF, VW, true, false><<<(unsigned)grid, 256, 0, st>>>(p);
  else if (past) rotary_kernel<T, HALF, VW, false, true><<<(unsigned)grid, 256, 0, st>>>(p);
  else rotary_kernel<T, HALF, VW, false, false><<<(unsigned)grid, 256, 0, st>>>(p);
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
  CSAM_REQUIRE(head_dim <= 2 * ROT_TABLE, "csam_rotary: heads of %d elements (at most %d)", head_dim, 2 * ROT_TABLE);
  CSAM_REQUIRE(T_pos > 0 && T % T_pos == 0 && pos_stride >= T_pos, "csam_rotary: %d tokens are not a multiple of %d positions", T, T_pos);
  CSAM_REQUIRE(dtype == CSAM_DT_F16 || dtype == CSAM_DT_F32 || dtype == CSAM_DT_BF16, "csam_rotary: bad dtype %d", dtype);
  CSAM_REQUIRE(hsq >= head_dim && hsqo >= head_dim && (!Hk || (hsk >= head_dim && hsko >= head_dim)), "csam_rotary: heads overlap");
  RotaryArgs p = {q, q_out, ldq, ldqo, Hk ? k : nullptr, Hk ? k_out : nullptr, ldk, ldko, hsq, hsqo, hsk, hsko, pos, pos_stride, pos_is_f32,
                  freq, axis, T, T_pos, Hq, Hk, head_dim, pairs, axes};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CSAM_DT_F16) return interleaved ? rotary_launch<half_t, false>(st, p) : rotary_launch<half_t, true>(st, p);
  if (dtype == CSAM_DT_BF16) return interleaved ? rotary_launch<bf16_t, false>(st, p) : rotary_launch<bf16_t, true>(st, p);
  return interleaved ? rotary_launch<float, false>(st, p) : rotary_launch<float, true>(st, p);
}
