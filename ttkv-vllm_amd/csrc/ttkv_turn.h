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
  int pieces;  // rows go in pieces of 8 elements
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

// One token's rows by the threads of a workgroup, in pieces of 8 elements: rows whose pieces are 16-byte
// aligned, pairs that lie in one piece or in two. A thread keeps its piece's frequencies from head to head;
// kTurnBatch heads' loads are in flight at a time, the first ones asked for before the angles are formed.
constexpr int kTurnBatch = 4;
template <int DT>
__device__ __forceinline__ void turn_pieces(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  const bool adj = a.adjacent;
  const int nch = adj ? a.half >> 2 : a.half >> 3;  // pieces (by halves: pairs of them) that are turned
  const int slots = threads / nch, heads = a.heads[0] + a.heads[1];
  const int slot = tid / nch, p = tid - slot * nch, mate = adj ? 0 : a.half;
  const bool on = slot < slots;
  auto place = [&](int head, bool out, int64_t& at) -> const void* {
    const int set = head >= a.heads[0];
    at = tok * (out ? a.y_stride : a.x_stride)[set] + (int64_t)(set ? head - a.heads[0] : head) * a.d;
    return out ? a.y[set] : a.x[set];
  };
  Act8<DT> x[kTurnBatch], y[kTurnBatch];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int b = 0; b < kTurnBatch; ++b) {
      const int head = h0 + b * slots + slot;
      if (on && head < heads) {
        int64_t at;
        const void* src = place(head, false, at);
        x[b] = load_act8<DT>(src, at + 8 * p);
        if (!adj) y[b] = load_act8<DT>(src, at + 8 * p + mate);
      }
    }
  };
  fetch(0);
  const bool ok = turn_table(a.pos, a.turns, a.half, a.amplitude, tok, tid, threads, cs);
  if (!ok && tid == 0) atomicOr(a.err, TTKV_ERR_BAD_POSITION);
  __syncthreads();
  float c[8], s[8];  // (adjacent pairs: four)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2v w = cs[adj ? 4 * p + (i & 3) : on ? 8 * p + i : 0];
    c[i] = w[0];
    s[i] = w[1];
  }
  for (int h0 = 0; h0 < heads; h0 += kTurnBatch * slots) {
#pragma unroll
    for (int b = 0; b < kTurnBatch; ++b) {
      const int head = h0 + b * slots + slot;
      if (on && head < heads) {
        int64_t at;
        void* dst = const_cast<void*>(place(head, true, at));
        float u[8], v[8];
        if (adj) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float xi = act8_get<DT>(x[b], 2 * i), yi = act8_get<DT>(x[b], 2 * i + 1);
            u[2 * i] = xi * c[i] - yi * s[i];
            u[2 * i + 1] = yi * c[i] + xi * s[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float xi = act8_get<DT>(x[b], i), yi = act8_get<DT>(y[b], i);
            u[i] = xi * c[i] - yi * s[i];
            v[i] = yi * c[i] + xi * s[i];
          }
          store_act8<DT>(dst, at + 8 * p + mate, v);
        }
        store_act8<DT>(dst, at + 8 * p, u);
      }
    }
    fetch(h0 + kTurnBatch * slots);
  }
  const int rest = (a.d - 2 * a.half) >> 3;  // pieces that are copied
  for (int i = tid; i < heads * rest; i += threads) {
    const int head = i / rest, x0 = 2 * a.half + (i - head * rest) * 8;
    int64_t from, to;
    const void* src = place(head, false, from);
    void* dst = const_cast<void*>(place(head, true, to));
    if (dst == src && from == to && ok) continue;  // in place
    const Act8<DT> z = load_act8<DT>(src, from + x0);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ok ? act8_get<DT>(z, k) : NAN;
    store_act8<DT>(dst, to + x0, v);
  }
}

// One token's rows, in pieces or an element or a pair per thread.
__device__ __forceinline__ void turn_token(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  if (a.pieces) {
    if (a.dtype == TTKV_DTYPE_BF16) turn_pieces<TTKV_DTYPE_BF16>(a, tok, tid, threads, cs);
    else if (a.dtype == TTKV_DTYPE_F16) turn_pieces<TTKV_DTYPE_F16>(a, tok, tid, threads, cs);
    else turn_pieces<TTKV_DTYPE_F32>(a, tok, tid, threads, cs);
    return;
  }
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
