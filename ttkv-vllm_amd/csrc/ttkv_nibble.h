// The 4-bit cache: 16-bit codes-and-scale records of rotated keys and values, one record per tile
// of 16 slots and KV head.
//
// A group of 32 dims of a token's key (or value) row x is stored as 32 codes of 4 bits and one
// 16-bit parameter:
//   lo = min(0, min x), hi = max(0, max x)            (x clamped to +-32640 first)
//   s  = (hi - lo) / 15, in 64 bits, rounded up to 7 significant bits, at least 2^-14
//   z  = rint(-lo / s) in [0, 15],  c = clamp(rint(x / s) + z, 0, 15),  value = (c - z) * s
// s is an fp16 number whose low four mantissa bits are zero; the parameter holds z there. c - z has
// 4 bits and s 7, so a value is exact in fp16: the reads feed it to the matrix units unrounded. A
// group that holds a NaN or an infinity has the parameter 0x7e00 (s = NaN) and reads back as NaN.
//
// The slots of a block are taken 16 at a time (the block size is a multiple of 16); such a tile's
// bytes are its slots' bytes together, H records of 2,304 bytes (144 bytes per slot and head).
// Within a record the codes lie as the read's matrix operands want them, a lane's share of the
// tile in 16 consecutive bytes:
//      0  key codes: dword (qd * 16 + u) * 4 + g holds token u's dims 32 g + 8 qd + j (j = 0..7) at
//         bits 4 (j / 2) + 16 (j % 2): a shift and a mask give two consecutive dims as 16-bit halves
//   1024  value codes: dword ((q4 * 16 + n) * 2 + pair) * 2 + quad holds, in its low half, token
//         4 q4 + 2 pair and, in its high half, the next one: each dims 32 (2 quad + gg) + 2 n + b at
//         bits 4 (2 gg + b): the same shift and mask give two tokens of one dim
//   2048  key parameters, u * 4 + g
//   2176  value parameters, (q4 * 4 + g) * 4 + u % 4
#pragma once

#include "ttkv_device.h"

namespace ttkv {

constexpr int kNibTile = 16;       // slots per tile
constexpr int kNibGroup = 32;      // dims per parameter
constexpr int kNibRecord = 2304;   // bytes of a tile's record of one head
constexpr int kNibSlot = kNibRecord / kNibTile;  // bytes per slot and head
constexpr int kNibV = 1024;        // record offsets: value codes,
constexpr int kNibKp = 2048;       // key parameters,
constexpr int kNibVp = 2176;       // value parameters
constexpr float kNibMax = 32640.f;       // values are clamped to this: 7.5 steps of the largest scale
constexpr float kNibMinScale = 0x1p-14f; // the smallest normal fp16

// (c - z) * s of two codes as an fp16 pair, exactly: the codes' nibbles at bit 4 m of x's halves,
// biased by 1024 (one unit in fp16's last place there), z likewise in zb = nib_biased(parameters),
// s = nib_scales(parameters). The difference has 4 bits and s 7, so neither operation rounds.
// The masks come in registers (one scalar, one vector: an instruction takes one constant from
// outside the vector registers), so each is a single v_and_or_b32.
struct NibMasks {
  uint32_t nib, one;  // 0x000f000f (uniform), 0x64006400 (in a vector register)
};
__device__ __forceinline__ NibMasks nib_masks() {
  NibMasks k{0x000f000fu, 0x64006400u};
  asm("" : "+s"(k.nib), "+v"(k.one));
  return k;
}
__device__ __forceinline__ half2v nib_biased(uint32_t x, const NibMasks& k) {
  return __builtin_bit_cast(half2v, (x & k.nib) | k.one);
}
__device__ __forceinline__ half2v nib_scales(uint32_t p2) {
  return __builtin_bit_cast(half2v, p2 & 0xfff0fff0u);
}
__device__ __forceinline__ half2v nib_pair(uint32_t x, int m, half2v zb, half2v s,
                                           const NibMasks& k) {
  return (nib_biased(x >> (4 * m), k) - zb) * s;
}

// A query row's share of a lane, the operand of the score products: dims 32 g + 8 q4 + (0..7) as
// qf[g], lanes q4 = 0..3 of one row together. qs: what a product's result is multiplied by, never
// negative (the query takes the scale's sign, so the largest product is the largest score).
// bf16 comes to fp16 at a power of two per row that brings its largest value to [1, 2): exact but for
// values below 2^-14 of the largest, which keep an error of at most 2^-25 of it. `on`: false for
// columns without a row, which are 0.
struct NibRow {
  u32x4 raw[4];
};
__device__ __forceinline__ NibRow nib_load_row(const uint16_t* row, int q4) {
  NibRow x;
#pragma unroll
  for (int g = 0; g < 4; ++g) x.raw[g] = *gbl((const u32x4*)(row + 32 * g + 8 * q4));
  return x;
}
template <int QDT>
__device__ __forceinline__ void nib_query(const NibRow& in, float scale_log2, bool on, half8 qf[4],
                                          float& qs) {
  const auto& raw = in.raw;
  qs = fabsf(scale_log2);
  if constexpr (QDT == TTKV_DTYPE_F16) {
#pragma unroll
    for (int g = 0; g < 4; ++g) qf[g] = __builtin_bit_cast(half8, raw[g]);
  } else {
    float x[32], mx = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const uint32_t w = raw[i >> 3][(i & 7) >> 1];
      x[i] = bf16_bits_to_float(w & 0xffffu);
      x[i + 1] = bf16_bits_to_float(w >> 16);
      mx = fmaxf(fmaxf(mx, fabsf(x[i])), fabsf(x[i + 1]));
    }
    mx = cross_row_max(mx);
    const int e = mx > 0.f && mx < INFINITY ? ilogbf(mx) : 0;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const half2v p = {(_Float16)ldexpf(x[i], -e), (_Float16)ldexpf(x[i + 1], -e)};
      qf[i >> 3][i & 7] = p[0];
      qf[i >> 3][(i & 7) + 1] = p[1];
    }
    qs = ldexpf(qs, e);
  }
  const bool none = qs == 0.f || !on;  // (a scale of 0 must not meet a masked score)
  if (none) qs = 1.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    if (scale_log2 < 0.f) qf[g] = -qf[g];
    if (none) qf[g] = half8{};
  }
}

// Softmax weights are 2^(score * qs - m), m a running maximum. Formed in one fma, the exponent of a key
// whose score is the maximum is what the rounding of m left over, 2^-25 |m| at most: a common factor of
// the row's weights, but one that leaves fp16 where |m| is about 2^29. Rows of |m| above kNibFar take the
// product rounded by itself: equal scores then weigh the same and the largest exactly 1, whatever their
// size. A maximum before the first visible key is the lowest float.
constexpr float kNibFar = 4096.f;
constexpr float kNibNone = -3.402823466e38f;
__device__ __forceinline__ bool nib_far(float m) { return fabsf(m) > kNibFar && m > kNibNone; }
// Other rows have m the maximum less `lift`: weights down to 2^-(14 + lift) of the largest are normal
// fp16 numbers, and smaller ones are rounded to 2^-(25 + lift) of it. (With m the maximum itself 2,000
// tokens at 2^-20.6 beside one came out 2.8 % off, at 2^-26 as nothing.) m has to move once a key's weight
// is 2^(16 - lift) times the largest of when it last moved.
constexpr float kNibMost = 8 * 65504.f;  // a lane's sum of eight weights; beyond it one is infinite
__device__ __forceinline__ float nib_max(float m, float scores, float lift) {
  return fmaxf(m, nib_far(scores) ? scores : scores - lift);
}
__device__ __forceinline__ float nib_apart(float score, float qs, float m) {
#pragma clang fp contract(off)
  const float p = score * qs;
  return p - m;
}

// Inclusive prefix sum over the wave's lanes (all active), on DPP: within rows of 16, then the rows.
__device__ __forceinline__ int nib_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // last lane of rows 0, 2 to 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // of row 1 to rows 2 and 3
  return v;
}

// Two floats of another workgroup's partial result (see ld_agent).
__device__ __forceinline__ float2v ld_agent2(const float* p) {
  const uint64_t w =
      __hip_atomic_load((const uint64_t*)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return __builtin_bit_cast(float2v, w);
}

// Four floats of other workgroups' partial results, at byte `at` of `bytes` from a wave-uniform base:
// one 16-byte load of the cache policy of an agent-scope load (sc1). ld_agent's atomic loads are of
// 8 bytes at most; a join is bound by how much it has in flight.
__device__ __forceinline__ float4v ld_agent16(const float* base, uint32_t bytes, uint32_t at) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00027000);
  const auto w = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)at, 0, 16);
  return __builtin_bit_cast(float4v, w);
}

}  // namespace ttkv
