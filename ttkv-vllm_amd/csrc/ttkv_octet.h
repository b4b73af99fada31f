// The 8-bit cache: e4m3 codes with one power of two per 32 dims, of rotated keys and values, one record
// per tile of 16 slots and KV head.
//
// A group of 32 dims x of a token's key (or value) row is stored as 32 codes and one byte:
//   2^e the smallest power of two with max |x| <= 448 * 2^e, e >= -117     (x clamped to +-1.75 * 2^127)
//   code = e4m3(x / 2^e), rounded to the nearest, ties to even;  byte = e + 127;  value = code * 2^e
// A value has 4 significant bits and lies in [2^-126, 1.75 * 2^127] or is 0: it is exact in bf16 and
// never subnormal there, so the reads feed it to the matrix units unrounded. A group that holds a NaN or
// an infinity has NaN codes and the byte 127.
//
// The slots of a block are taken 16 at a time (the block size is a multiple of 16); such a tile's bytes
// are its slots' bytes together, H records of 33 d bytes. Within a record the codes lie as the read's
// matrix operands want them, a lane's share of the tile in pieces of 16 consecutive bytes (lane = 16 q + u
// or 16 q + n):
//   0       key codes: token u's dims q d/4 + 16 p + (0..15) at ((p * 4 + q) * 16 + u) * 16
//   16 d    value codes: with N = d / 16, bytes b = N i + e of lane (q, n) are token 4 q + i's dim
//           N n + e, at (b / 16 * 64 + 16 q + n) * 16 + b % 16
//   32 d    key exponents: group g of token u at (g / P * 16 + u) * P + g % P, P = max(1, d / 128)
//   32.5 d  value exponents: g * 16 + u
#pragma once

#include "ttkv_device.h"

namespace ttkv {

constexpr int kOctTile = 16;   // slots per tile
constexpr int kOctMinByte = 127 - 117;
constexpr uint32_t kOctNanCode = 0x7f, kOctNanByte = 127;
constexpr float kOctMax = 0x1.cp127f;

template <int D>
struct Oct {
  static_assert(D == 64 || D == 128 || D == 256, "head dims of 64, 128 and 256");
  static constexpr int kRecord = 33 * D;       // bytes of a tile's record of one head
  static constexpr int kPair = D >= 128 ? D / 128 : 1;  // key exponents of a lane
  static constexpr int kDims = D / 16;         // a lane's value dims per token
  static constexpr int kV = 16 * D;            // record offsets: value codes,
  static constexpr int kKp = 32 * D;           // key exponents,
  static constexpr int kVp = 32 * D + D / 2;   // value exponents

  static __device__ __forceinline__ int key(int u, int x) {
    return ((x % (D / 4) / 16 * 4 + x / (D / 4)) * 16 + u) * 16 + x % 16;
  }
  static __device__ __forceinline__ int value(int u, int x) {
    const int b = u % 4 * kDims + x % kDims;
    return kV + (b / 16 * 64 + u / 4 * 16 + x / kDims) * 16 + b % 16;
  }
  static __device__ __forceinline__ int key_power(int u, int g) {
    return kKp + (g / kPair * 16 + u) * kPair + g % kPair;
  }
  static __device__ __forceinline__ int value_power(int u, int g) { return kVp + g * 16 + u; }
};

// 2^(byte - 127); bytes that no write leaves (0, 255) give 0 and infinity.
__device__ __forceinline__ float oct_power(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Two codes (the low or high half of a dword) times their power of two, as a bf16 pair, exactly.
template <bool HIGH>
__device__ __forceinline__ bf16x2 oct_pair(uint32_t codes, float power) {
  return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, power, HIGH);
}

}  // namespace ttkv
