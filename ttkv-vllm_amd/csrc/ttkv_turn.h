// Rotary positions from frequencies, without a table of angles: the pairs of a row turned by
// position * turns[j] revolutions. gfx950 / CDNA4.
//
// The angle is formed in 64 bits, in revolutions: the product of a position below 2^31 and a frequency
// of at most one revolution is off by 2^-53 of itself, 2^-22 of a revolution at worst and less than fp32
// resolves where frequencies are those of a model (1 / (2 pi) at most). Whole and quarter revolutions are
// taken off exactly; what is left, at most an eighth, goes to radians and to fp32 and into the Taylor
// series of the sine and the cosine.
#pragma once

#include "ttkv_device.h"

namespace ttkv {

constexpr int kTurnHalf = 512;              // frequencies that the LDS holds
constexpr int64_t kTurnPositions = 1ll << 31;

// Cosine and sine of t revolutions. Series up to x^10 and x^9 at |x| <= pi / 4: off by 5e-10 and 2e-9.
__device__ __forceinline__ void turn_angle(double t, float& c, float& s) {
  t -= rint(t);
  const double k = rint(4.0 * t);
  const float x = (float)((t - 0.25 * k) * 6.283185307179586), y = x * x;
  const float sn = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), 1.f);
  const float cn = fmaf(
      y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f), -0.5f), 1.f);
  const int q = (int)k & 3;  // quarters, -2 .. 2
  const float a = q & 1 ? sn : cn, b = q & 1 ? cn : sn;
  c = q == 1 || q == 2 ? -a : a;
  s = q & 2 ? -b : b;
}

// Rows that are turned: up to two sets of heads (queries and keys) of one dtype.
struct TurnArgs {
  const void* x[2];
  void* y[2];
  int heads[2];
  int64_t x_stride[2], y_stride[2];
  int dtype, d, half, adjacent;
  const int64_t* pos;
  const double* turns;
  float amplitude;
  int32_t* err;
};

// Cosines and sines of token `tok` into cs[0 .. half), by the workgroup's threads; NaN where its
// position is refused, which is returned. The caller synchronises before they are read.
__device__ __forceinline__ bool turn_table(const int64_t* pos, const double* turns, int half, float amplitude,
                                           int64_t tok, int tid, int threads, float2v* cs) {
  const int64_t p = *gbl(pos + tok);
  const bool ok = p >= 0 && p < kTurnPositions;
  for (int j = tid; j < half; j += threads) {
    float c, s;
    turn_angle((double)p * *gbl(turns + j), c, s);
    cs[j] = ok ? float2v{c * amplitude, s * amplitude} : float2v{NAN, NAN};
  }
  return ok;
}

// One token's rows, an element or a pair per thread.
__device__ __forceinline__ void turn_token(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  const bool ok = turn_table(a.pos, a.turns, a.half, a.amplitude, tok, tid, threads, cs);
  if (!ok && tid == 0) atomicOr(a.err, TTKV_ERR_BAD_POSITION);
  __syncthreads();
  const int per = a.d - a.half;  // pairs, then the dims that are copied
  for (int i = tid; i < (a.heads[0] + a.heads[1]) * per; i += threads) {
    const int head = i / per, j = i - head * per, set = head >= a.heads[0];
    const int64_t hd = (int64_t)(set ? head - a.heads[0] : head) * a.d;
    const int64_t from = tok * a.x_stride[set] + hd, to = tok * a.y_stride[set] + hd;
    if (j >= a.half) {
      const float v = load_act(a.x[set], a.dtype, from + j + a.half);
      store_act(a.y[set], a.dtype, to + j + a.half, ok ? v : NAN);
      continue;
    }
    const int u = a.adjacent ? 2 * j : j, v = a.adjacent ? 2 * j + 1 : j + a.half;
    const float x = load_act(a.x[set], a.dtype, from + u), y = load_act(a.x[set], a.dtype, from + v);
    const float c = cs[j][0], s = cs[j][1];
    store_act(a.y[set], a.dtype, to + u, x * c - y * s);
    store_act(a.y[set], a.dtype, to + v, y * c + x * s);
  }
}

}  // namespace ttkv
