// Write of new keys and values into the 4-bit cache (format: ttkv_nibble.h). gfx950 / CDNA4.
//
// One wave per (token, KV head): lanes 0..31 hold the key row, 4 consecutive dims each, lanes
// 32..63 the value row, so a group of 32 dims is 8 neighbouring lanes and its minimum and maximum
// are three DPP steps.
//
// Codes are decided exactly. For 16-bit inputs the quotients x / s and -lo / s are taken in 32
// bits: x has at most 11 significant bits and s 7, so a quotient that is not on a rounding border
// k + 1/2 is at least 6e-5 from it, and the correctly rounded division is within 1e-6 (and exact
// on a border). 32-bit inputs are divided in 64 bits. The scale's range and its quotient by 15 are
// taken in 64 bits for every type.
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_nibble.h"

namespace ttkv {

struct NibWriteArgs {
  const void* k;
  const void* v;
  int k_dtype, v_dtype;
  int64_t k_row_stride, v_row_stride;
  const int64_t* slots;
  int num_tokens, H;
  uint8_t* page;
  int64_t n_slots, slot_stride;
  _Float16* k_out;
  _Float16* v_out;
  int32_t* err;
};

// A neighbour's value within groups of 8 lanes: xor 1, xor 2, and the mirrored lane of the 8.
template <int STEP>
__device__ __forceinline__ int dpp8(int v) {
  constexpr int ctrl = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : 0x141;
  return __builtin_amdgcn_update_dpp(0, v, ctrl, 0xF, 0xF, false);
}
template <int STEP>
__device__ __forceinline__ float dpp8f(float v) {
  return __builtin_bit_cast(float, dpp8<STEP>(__builtin_bit_cast(int, v)));
}

// (hi - lo) / 15 rounded up to 7 significant bits, at least 2^-14.
__device__ __forceinline__ float nib_step(float lo, float hi) {
  const double t = ((double)hi - (double)lo) / 15.0;
  const uint64_t low = (1ull << 46) - 1;
  const uint64_t b = (__builtin_bit_cast(uint64_t, t) + low) & ~low;
  return fmaxf((float)__builtin_bit_cast(double, b), kNibMinScale);
}

template <bool WIDE>
__device__ __forceinline__ float nib_quot(float x, float s) {
  if constexpr (WIDE) return (float)rint((double)x / (double)s);
  return rintf(x / s);
}

template <bool WIDE>
__device__ __forceinline__ void nib_write_row(const NibWriteArgs& a, int64_t tok, int h,
                                              int64_t slot, int lane) {
  const bool val = lane >= 32;
  const int i = lane & 31;  // dims 4 i .. 4 i + 3
  const int g = i >> 3;
  const void* src = val ? a.v : a.k;
  const int dt = val ? a.v_dtype : a.k_dtype;
  const int64_t at = tok * (val ? a.v_row_stride : a.k_row_stride) + (int64_t)h * kD + 4 * i;
  const bool vec = act_rows_aligned(src, dt, val ? a.v_row_stride : a.k_row_stride);
  float x[4];
  load_act_n<4>(src, dt, at, vec, x);
  int bad = 0;
  float lo = 0.f, hi = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bad |= !(fabsf(x[j]) < INFINITY);
    x[j] = fminf(fmaxf(x[j], -kNibMax), kNibMax);
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  bad |= dpp8<0>(bad);
  bad |= dpp8<1>(bad);
  bad |= dpp8<2>(bad);
  lo = fminf(lo, dpp8f<0>(lo));
  lo = fminf(lo, dpp8f<1>(lo));
  lo = fminf(lo, dpp8f<2>(lo));
  hi = fmaxf(hi, dpp8f<0>(hi));
  hi = fmaxf(hi, dpp8f<1>(hi));
  hi = fmaxf(hi, dpp8f<2>(hi));
  if (bad) {
    lo = hi = 0.f;
    x[0] = x[1] = x[2] = x[3] = 0.f;
  }
  const float s = nib_step(lo, hi);
  const float z = nib_quot<WIDE>(-lo, s);
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    c[j] = (uint32_t)fminf(fmaxf(nib_quot<WIDE>(x[j], s) + z, 0.f), 15.f);
  const uint32_t par =
      bad ? 0x7e00u : __builtin_bit_cast(uint16_t, (_Float16)s) | (uint32_t)z;

  _Float16* outp = val ? a.v_out : a.k_out;
  if (outp) {
    const float f = bad ? NAN : s;
    half4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (_Float16)(((float)c[j] - z) * f);
    *gblw((half4*)(outp + (tok * a.H + h) * kD + 4 * i)) = o;
  }
  uint8_t* rec = a.page + (slot >> 4) * (kNibTile * a.slot_stride) + h * kNibRecord;
  const int u = (int)(slot & 15);
  if (!val) {
    uint32_t w = (c[0] | (c[1] << 16) | (c[2] << 4) | (c[3] << 20)) << (8 * (i & 1));
    w |= (uint32_t)dpp8<0>((int)w);
    if (!(i & 1)) *gblw((uint32_t*)rec + (((i & 7) >> 1) * 16 + u) * 4 + g) = w;
    if (!(i & 7)) *gblw((uint16_t*)(rec + kNibKp) + u * 4 + g) = (uint16_t)par;
  } else {
    const int q4 = u >> 2, pair = (u >> 1) & 1, n = 2 * (i & 7);
    uint8_t* b = rec + kNibV + (((q4 * 16 + n) * 2 + pair) * 2 + (g >> 1)) * 4 + 2 * (u & 1) + (g & 1);
    *gblw(b) = (uint8_t)(c[0] | (c[1] << 4));
    *gblw(b + 16) = (uint8_t)(c[2] | (c[3] << 4));
    if (!(i & 7)) *gblw((uint16_t*)(rec + kNibVp) + (q4 * 4 + g) * 4 + (u & 3)) = (uint16_t)par;
  }
}

__global__ __launch_bounds__(256) void nibble_write_kernel(NibWriteArgs a) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t tok = row / a.H;
  if (tok >= a.num_tokens) return;
  const int64_t slot = a.slots[tok];
  if (slot < 0) return;  // a padded token
  if (slot >= a.n_slots) {
    if ((threadIdx.x & 63) == 0) atomicOr(a.err, TTKV_ERR_BAD_SLOT);
    return;
  }
  const int h = (int)(row % a.H), lane = threadIdx.x & 63;
  if (a.k_dtype == TTKV_DTYPE_F32 || a.v_dtype == TTKV_DTYPE_F32)
    nib_write_row<true>(a, tok, h, slot, lane);
  else
    nib_write_row<false>(a, tok, h, slot, lane);
}

int nibble_check_page(int H, int d, const uint8_t* page, int64_t n_slots, int64_t slot_stride) {
  if (d != kD) return host_fail(TTKV_E_UNSUPPORTED, "head dim must be 128");
  if (H <= 0) return host_fail(TTKV_E_INVALID, "H must be positive");
  if (!page) return host_fail(TTKV_E_INVALID, "null page");
  if (slot_stride < (int64_t)kNibSlot * H)
    return host_fail(TTKV_E_INVALID, "slot stride is smaller than the slot (144 H bytes)");
  if ((uintptr_t)page % 16 || slot_stride % 16)
    return host_fail(TTKV_E_INVALID, "the page and its slot stride must be 16-byte aligned");
  if (n_slots <= 0 || n_slots % kNibTile)
    return host_fail(TTKV_E_INVALID, "the page must hold a positive multiple of 16 slots");
  return TTKV_OK;
}

int nibble_write_paged(int H, int d, const void* key, int k_dtype, int64_t k_row_stride,
                       const void* val, int v_dtype, int64_t v_row_stride, const int64_t* slots,
                       int num_tokens, uint8_t* page, int64_t n_slots, int64_t slot_stride,
                       void* k_out, void* v_out, int32_t* err, hipStream_t st) {
  if (int rc = nibble_check_page(H, d, page, n_slots, slot_stride)) return rc;
  for (int dt : {k_dtype, v_dtype})
    if (dt != TTKV_DTYPE_F32 && dt != TTKV_DTYPE_F16 && dt != TTKV_DTYPE_BF16)
      return host_fail(TTKV_E_INVALID, "key / value dtype must be fp32, fp16 or bf16");
  if (num_tokens < 0) return host_fail(TTKV_E_INVALID, "negative num_tokens");
  if (num_tokens == 0) return TTKV_OK;
  if (!key || !val || !slots || !err) return host_fail(TTKV_E_INVALID, "null pointer argument");
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
    return host_fail(TTKV_E_INVALID, "key_out / value_out must be 16-byte aligned");
  const int64_t rows = (int64_t)num_tokens * H, grid = (rows + 3) / 4;
  if (grid > 0x7fffffff) return host_fail(TTKV_E_INVALID, "too many tokens for one call");
  NibWriteArgs a{key,   val,  k_dtype, v_dtype,     k_row_stride,     v_row_stride,     slots, num_tokens,
                 H,     page, n_slots, slot_stride, (_Float16*)k_out, (_Float16*)v_out, err};
  hipLaunchKernelGGL(nibble_write_kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("nibble write launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
