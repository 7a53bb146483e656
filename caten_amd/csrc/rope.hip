// Rotary positions of a ragged batch's rows: every row has a position of its own (cthip_kv_plan_paged writes them), queries and keys are slices of
// one product, the angles come from a table of frequencies.  The reference rotates whole heads, neighbouring channels, at consecutive
// positions (nn/positional-encoding.lisp:3-64: cthip_rope).
//
// A pair (a, b) at angle t = position * frequency becomes m (a cos t - b sin t, a sin t + b cos t).  t is a 64-bit product, and a whole number of quarter
// turns is taken off it in 64 bits, so that sine and cosine are as exact at position 10^6 as at 1 (in 32 bits t alone would be off by 0.03 there; in 64 its rounding, 2^-53 of it, comes
// to theirs, 2^-23, at 2^30 radians).  A thread
// works out the angles of its channels once and turns them in every head it takes, four channels (halves: eight) in one access of 16 bytes each, one head
// after the other (outputs may be the inputs, so a head's loads stay behind the stores of the one before; the other wavefronts run meanwhile).  Bound by the rows: read and written once.
//   6001 rows of 64 + 8 heads of 128, halves (442 MB): 84 us = 5.2 TB/s, where a copy of 4 GiB reaches 4.7.
//   48 rows of 32 + 4 heads of 64, pairs: 2.9 us, a launch and three round trips (position, frequencies, the rows).
#include <algorithm>

#include "common.h"

namespace cthip {

struct RopeRows {
  float *q_out, *k_out;
  const float *q, *k;
  int64_t q_out_stride, k_out_stride, q_stride, k_stride;
  const int *positions;
  const double *frequencies;
  float magnitude;
  int H, heads, Dh, rotary;  // heads: of q and k
  int units, per_block;      // pieces of a head that a thread takes, and how many of them a workgroup has side by side
  int at_once, rounds;       // heads that a workgroup takes at a time, and how many times
};

// sine and cosine: the nearest multiple of a quarter turn taken off in 64 bits (two terms of pi / 2, fused: what is left is as exact as the angle),
// Taylor's series on the eighth of a turn that is left (|x| <= pi / 4: x^11 / 11! below 2^-28 of x, x^12 / 12! below 2^-32)
__device__ __forceinline__ void sincos_far(double angle, float &sn, float &cs) {
  const double quarter = rint(angle * 0.63661977236758134308);
  const float x = (float)fma(-quarter, 6.123233995736766e-17, fma(-quarter, 1.5707963267948966, angle)), y = x * x;
  float s = fmaf(y, 2.75573192e-6f, -1.98412698e-4f);
  s = fmaf(y, s, 8.33333333e-3f);
  s = fmaf(y, s, -1.66666667e-1f);
  s = fmaf(x * y, s, x);
  float c = fmaf(y, -2.75573192e-7f, 2.48015873e-5f);
  c = fmaf(y, c, -1.38888889e-3f);
  c = fmaf(y, c, 4.16666667e-2f);
  c = fmaf(y * y, c, fmaf(y, -0.5f, 1.0f));
  const int k = (int)(quarter - 4.0 * floor(0.25 * quarter));  // 0 .. 3
  sn = k & 1 ? c : s;
  cs = k & 1 ? s : c;
  if (k & 2) sn = -sn;
  if (k == 1 || k == 2) cs = -cs;
}

template <int N>
struct Floats;
template <>
struct Floats<4> {
  typedef f4_any type;
};
template <>
struct Floats<2> {
  typedef float type __attribute__((ext_vector_type(2), aligned(4)));
};
template <>
struct Floats<1> {
  typedef float type __attribute__((ext_vector_type(1), aligned(4)));
};

// A unit: neighbouring pairs: V channels; halves: V channels and the V that are rotary / 2 further on.  Behind the rotary part, V channels that stay.
template <bool HALVES, int V>
__global__ __launch_bounds__(256) void k_rope_rows(RopeRows a) {
  typedef typename Floats<V>::type vec;
  constexpr int ANGLES = HALVES ? V : V / 2;
  const int row = blockIdx.x, position = a.positions[row];
  if (position < 0) return;
  const int unit = blockIdx.z * 256 + threadIdx.x % a.per_block;
  const int mine = threadIdx.x / a.per_block, h0 = (int)blockIdx.y * a.rounds * a.at_once + mine;
  if (unit >= a.units || mine >= a.at_once) return;
  const int turned = HALVES ? a.rotary / (2 * V) : a.rotary / V;  // units of the rotary part
  const bool turns = unit < turned;
  const int c0 = turns ? unit * V : a.rotary + (unit - turned) * V, c1 = HALVES && turns ? c0 + a.rotary / 2 : c0;
  float sn[ANGLES], cs[ANGLES];
  if (turns) {
#pragma unroll
    for (int i = 0; i < ANGLES; i++) {
      sincos_far((double)position * a.frequencies[(HALVES ? c0 : c0 / 2) + i], sn[i], cs[i]);
      sn[i] *= a.magnitude, cs[i] *= a.magnitude;
    }
  }
  const float *q = a.q + (int64_t)row * a.q_stride, *k = a.k + (int64_t)row * a.k_stride;
  float *q_out = a.q_out + (int64_t)row * a.q_out_stride, *k_out = a.k_out + (int64_t)row * a.k_out_stride;
#pragma unroll 4
  for (int i = 0; i < a.rounds; i++) {
    const int h = h0 + i * a.at_once;
    if (h >= a.heads) break;
    const float *from = h < a.H ? q + (int64_t)h * a.Dh : k + (int64_t)(h - a.H) * a.Dh;
    float *to = h < a.H ? q_out + (int64_t)h * a.Dh : k_out + (int64_t)(h - a.H) * a.Dh;
    vec x = *(const vec *)(from + c0);
    if constexpr (HALVES) {
      if (turns) {
        vec y = *(const vec *)(from + c1);
#pragma unroll
        for (int e = 0; e < V; e++) {
          const float u = x[e], w = y[e];
          x[e] = fmaf(u, cs[e], -(w * sn[e]));
          y[e] = fmaf(u, sn[e], w * cs[e]);
        }
        *(vec *)(to + c1) = y;
      }
    } else if (turns) {
#pragma unroll
      for (int e = 0; e < ANGLES; e++) {
        const float u = x[2 * e], w = x[2 * e + 1];
        x[2 * e] = fmaf(u, cs[e], -(w * sn[e]));
        x[2 * e + 1] = fmaf(u, sn[e], w * cs[e]);
      }
    }
    *(vec *)(to + c0) = x;
  }
}

}  // namespace cthip

using namespace cthip;

extern "C" {

int cthip_rope_frequencies(double *frequencies, int rotary_dim, double base, double factor, int trained, double slow, double fast) {
  CTHIP_ARG(rotary_dim >= 0 && rotary_dim % 2 == 0 && (rotary_dim == 0 || frequencies) && base > 0.0 && base < INFINITY && factor > 0.0 && factor < INFINITY);
  CTHIP_ARG(trained >= 0 && (trained == 0 || (slow >= 0.0 && fast > slow && fast < INFINITY)));
  for (int i = 0; i < rotary_dim / 2; i++) {
    const double f = pow(base, -2.0 * i / rotary_dim);
    const double turns = trained * f * 0.15915494309189533577;
    const double keep = trained == 0 ? 0.0 : turns <= slow ? 0.0 : turns >= fast ? 1.0 : (turns - slow) / (fast - slow);
    frequencies[i] = f * (keep + (1.0 - keep) / factor);
  }
  return 0;
}

int cthip_rope_rows(float *q_out, int64_t q_out_stride, float *k_out, int64_t k_out_stride, const float *q, int64_t q_stride, const float *k, int64_t k_stride,
                    const int *positions, int n_rows, int H, int Hkv, int Dh, int rotary_dim, int layout, const double *frequencies, float magnitude) {
  CTHIP_REQUIRE_INIT();
  CTHIP_ARG(n_rows >= 0 && H >= 0 && Hkv >= 0 && Dh >= 0 && rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= Dh);
  CTHIP_ARG(layout == CTHIP_ROPE_PAIRS || layout == CTHIP_ROPE_HALVES);
  if (n_rows > (1 << 23) || H > 65535 || Hkv > 65535 || Dh > 65535)
    return fail(CTHIP_E_UNSUPPORTED, "cthip_rope_rows: %d rows of %d and %d heads of %d (at most 2^23 rows, 65535 heads and channels)", n_rows, H, Hkv, Dh);
  CTHIP_ARG(H == 0 || n_rows == 0 || Dh == 0 || (q && q_out && q_stride >= (int64_t)H * Dh && q_out_stride >= (int64_t)H * Dh));
  CTHIP_ARG(Hkv == 0 || n_rows == 0 || Dh == 0 || (k && k_out && k_stride >= (int64_t)Hkv * Dh && k_out_stride >= (int64_t)Hkv * Dh));
  CTHIP_ARG((q != q_out || q_stride == q_out_stride || H == 0) && (k != k_out || k_stride == k_out_stride || Hkv == 0));
  if (n_rows == 0 || H + Hkv == 0 || Dh == 0) return 0;
  CTHIP_ARG(positions && (rotary_dim == 0 || frequencies));
  const bool halves = layout == CTHIP_ROPE_HALVES;
  // four channels a thread where a head's parts are whole fours, else the least that a pair allows
  const bool fours = (halves ? rotary_dim / 2 : rotary_dim) % 4 == 0 && (Dh - rotary_dim) % 4 == 0;
  if (!fours && !halves && (Dh - rotary_dim) % 2 != 0)
    return fail(CTHIP_E_UNSUPPORTED, "cthip_rope_rows: heads of %d channels, an odd number", Dh);
  const int V = fours ? 4 : halves ? 1 : 2;
  RopeRows a = {q_out, k_out, q, k, q_out_stride, k_out_stride, q_stride, k_stride, positions, frequencies, magnitude, H, H + Hkv, Dh, rotary_dim};
  a.units = (halves ? rotary_dim / 2 : rotary_dim) / V + (Dh - rotary_dim) / V;
  a.per_block = a.units < 256 ? a.units : 256;
  a.at_once = 256 / a.per_block;
  // A row's heads go to as many workgroups as the card runs at once, eight a compute unit, or to one, which works its angles out once.  64 + 8 heads of
  // 128, by one workgroup a row and so: 48 rows 5.0 and 3.5 us, 200 rows 5.6 and 4.7, 600 rows 8.6 and 7.8; with four times as many 1500
  // rows of 32 + 4 heads of 64 take 7.1 instead of 5.9.
  const int rounds = (a.heads + a.at_once - 1) / a.at_once, chunks = std::max(1, std::min(rounds, 8 * state().compute_units / n_rows));
  a.rounds = (rounds + chunks - 1) / chunks;
  const dim3 grid((unsigned)n_rows, (unsigned)chunks, (unsigned)((a.units + 255) / 256)), block(256);
#define ROPE(HALVES_, V_) hipLaunchKernelGGL((k_rope_rows<HALVES_, V_>), grid, block, 0, state().stream, a)
  if (halves && V == 4) ROPE(true, 4);
  else if (halves) ROPE(true, 1);
  else if (V == 4) ROPE(false, 4);
  else ROPE(false, 2);
#undef ROPE
  CTHIP_LAUNCH_CHECK();
  return 0;
}

}  // extern "C"
