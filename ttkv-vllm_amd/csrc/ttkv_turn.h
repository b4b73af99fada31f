// Rotary positions from frequencies, without a table of angles: the pairs of a row turned by
// position * turns[j] revolutions. gfx950 / CDNA4.
//
// The angle is formed in 64 bits, in revolutions: the product of a position below 2^31 and a frequency
// of at most one revolution is off by 2^-53 of itself, 2^-22 of a revolution at worst and less than fp32
// resolves where frequencies are those of a model (1 / (2 pi) at most). Whole and quarter revolutions are
// taken off exactly; what is left, at most an eighth, goes to radians and to fp32 and into the Taylor
// series of the sine and the cosine. Bound by memory: 8,192 tokens of 40 heads of 128 in bf16, 168 MB, 31 us
// (pairs in two halves; adjacent 32), 5.4 TB/s; 8 tokens 2.8 us in a graph, where a launch that does nothing takes 2.0.
#pragma once

#include <type_traits>

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

// Whether position p is taken.
__device__ __forceinline__ bool turn_place(int64_t p) { return p >= 0 && p < kTurnPositions; }

// Cosine and sine of frequency j at position p; NaN where that is refused.
__device__ __forceinline__ float2v turn_at(const double* turns, int j, int64_t p, float amplitude) {
  float c, s;
  turn_angle((double)p * *gbl(turns + j), c, s);
  return turn_place(p) ? float2v{c * amplitude, s * amplitude} : float2v{NAN, NAN};
}

// 16 bytes of a row, by a store that does not stay in the caches: rows are whole lines, and drain while others
// are turned (40 heads of 128 in bf16: 512 tokens 3.8 us with stores that stay, 3.5 so; 4,096 15.8, 15.0;
// adjacent pairs, 8,192 tokens: 31.5, 31.8).
__device__ __forceinline__ void turn_store16(void* p, u32x4 w) { __builtin_nontemporal_store(w, gblw((u32x4*)p)); }

// Eight consecutive elements, rounded once by the hardware's conversions.
template <int DT>
__device__ __forceinline__ void turn_store8(void* p, int64_t i, const float v[8]) {
  if constexpr (DT == TTKV_DTYPE_F32) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      turn_store16((float*)p + i + 4 * j,
                   __builtin_bit_cast(u32x4, float4v{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]}));
  } else {
    typedef std::conditional_t<DT == TTKV_DTYPE_F16, _Float16, __bf16> T;
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 w;
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = (T)v[k];
    turn_store16((uint16_t*)p + i, __builtin_bit_cast(u32x4, w));
  }
}

// One token's rows in pieces of 8 elements: rows whose pieces are 16-byte aligned, pairs that lie in one
// piece (adjacent) or in two. A thread keeps its piece's frequencies from head to head; kTurnBatch heads'
// loads are in flight at a time, the first ones asked for before the angles are formed. Two of them (four:
// 8,192 tokens of 40 heads 38.1 us, 36.0 with two, whose fewer registers hold more tokens on a CU), and a
// workgroup of four waves per token at every size (a wave per token: 38.1, 512 tokens 9.1 against 4.9 us).
// STREAM: loads that do not stay in the caches, for rows of more bytes than those hold (kTurnStream).
constexpr int kTurnBatch = 2;
template <int DT, bool ADJ, bool STREAM>
__device__ __forceinline__ void turn_pieces(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  constexpr int kFreqs = ADJ ? 4 : 8;  // of an item: a piece, or a pair of pieces
  const int items = a.half / kFreqs, heads = a.heads[0] + a.heads[1];
  const int slots = threads / items, slot = tid / items, p = tid - slot * items;
  const int e0 = 8 * p, e1 = e0 + a.half;
  const int rest = (a.d - 2 * a.half) >> 3;  // pieces of a head that are copied
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
      if (slot < slots && head < heads) {
        int64_t at;
        const void* src = place(head, false, at);
        x[b] = load_act8<DT, STREAM>(src, at + e0);
        if (!ADJ) y[b] = load_act8<DT, STREAM>(src, at + e1);
      }
    }
  };
  fetch(0);
  const int64_t pos = *gbl(a.pos + tok);
  const bool ok = turn_place(pos);
  // Pieces that are copied, bit by bit (NaN where the position is refused), while the first ones to be turned
  // and the frequencies arrive; none in place.
  const bool in_place = ok && a.x[0] == a.y[0] && a.x[1] == a.y[1];
  for (int i0 = in_place ? heads * rest : tid; i0 < heads * rest; i0 += kTurnBatch * threads) {
    Act8<DT> z[kTurnBatch];
#pragma unroll
    for (int b = 0; b < kTurnBatch; ++b) {
      const int i = i0 + b * threads, head = i / rest;
      int64_t at;
      if (i < heads * rest) {
        const void* src = place(head, false, at);
        z[b] = load_act8<DT, STREAM>(src, at + 2 * a.half + (i - head * rest) * 8);
      }
    }
#pragma unroll
    for (int b = 0; b < kTurnBatch; ++b) {
      const int i = i0 + b * threads, head = i / rest;
      int64_t at;
      if (i < heads * rest) {
        char* dst = (char*)const_cast<void*>(place(head, true, at));
        at += 2 * a.half + (i - head * rest) * 8;
#pragma unroll
        for (int j = 0; j < (DT == TTKV_DTYPE_F32 ? 2 : 1); ++j)
          turn_store16(dst + at * (DT == TTKV_DTYPE_F32 ? 4 : 2) + 16 * j,
                       ok ? z[b].raw[j] : u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu});
      }
    }
  }
  for (int j = tid; j < a.half; j += threads) cs[j] = turn_at(a.turns, j, pos, a.amplitude);
  if (!ok && tid == 0) atomicOr(a.err, TTKV_ERR_BAD_POSITION);
  __syncthreads();
  float c[kFreqs], s[kFreqs];
#pragma unroll
  for (int i = 0; i < kFreqs; ++i) {
    const float2v w = cs[kFreqs * p + i];
    c[i] = w[0];
    s[i] = w[1];
  }
  for (int h0 = 0; h0 < heads; h0 += kTurnBatch * slots) {
#pragma unroll
    for (int b = 0; b < kTurnBatch; ++b) {
      const int head = h0 + b * slots + slot;
      if (slot < slots && head < heads) {
        int64_t at;
        void* dst = const_cast<void*>(place(head, true, at));
        float u[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xi = act8_get<DT>(x[b], i), yi = ADJ ? act8_get<DT>(x[b], i ^ 1) : act8_get<DT>(y[b], i);
          const float ci = c[ADJ ? i / 2 : i], si = s[ADJ ? i / 2 : i];
          u[i] = ADJ && (i & 1) ? xi * ci + yi * si : xi * ci - yi * si;
          v[i] = yi * ci + xi * si;
        }
        turn_store8<DT>(dst, at + e0, u);
        if (!ADJ) turn_store8<DT>(dst, at + e1, v);
      }
    }
    fetch(h0 + kTurnBatch * slots);
  }
}

template <bool STREAM>
__device__ __forceinline__ void turn_pieces(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  auto run = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (a.adjacent) turn_pieces<DT, true, STREAM>(a, tok, tid, threads, cs);
    else turn_pieces<DT, false, STREAM>(a, tok, tid, threads, cs);
  };
  if (a.dtype == TTKV_DTYPE_BF16) run(std::integral_constant<int, TTKV_DTYPE_BF16>{});
  else if (a.dtype == TTKV_DTYPE_F16) run(std::integral_constant<int, TTKV_DTYPE_F16>{});
  else run(std::integral_constant<int, TTKV_DTYPE_F32>{});
}

// One token's rows, an element or a pair per thread of the workgroup.
__device__ __forceinline__ void turn_elements(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  const int64_t pos = *gbl(a.pos + tok);
  const bool ok = turn_place(pos);
  for (int j = tid; j < a.half; j += threads) cs[j] = turn_at(a.turns, j, pos, a.amplitude);
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

// A token's rows by a workgroup.
template <bool STREAM>
__device__ __forceinline__ void turn_token(const TurnArgs& a, int64_t tok, int tid, int threads, float2v* cs) {
  if (a.pieces) turn_pieces<STREAM>(a, tok, tid, threads, cs);
  else turn_elements(a, tok, tid, threads, cs);
}

}  // namespace ttkv
