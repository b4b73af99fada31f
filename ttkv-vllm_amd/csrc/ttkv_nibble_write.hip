// Write of new keys and values into the 4-bit cache (format: ttkv_nibble.h). gfx950 / CDNA4.
//
// One wave per pair of tokens and KV head: 16 lanes per row of 128 dims, 8 dims each, keys in lanes
// 0..31 and values in lanes 32..63, so a group of 32 dims is 4 neighbouring lanes and its minimum and
// maximum are two DPP steps. A workgroup is 8 tokens of one head, whose slots in a row share a record.
//
// Codes are decided exactly. For 16-bit inputs the quotients x / s and -lo / s are taken in 32
// bits: x has at most 11 significant bits and s 7, so a quotient that is not on a rounding border
// k + 1/2 is at least 6e-5 from it. q = x r with r = 1 / s to an ulp, corrected once by its residual
// x - q s, is within 1e-6, and exact on a border: there the corrected value differs from a number
// that fp32 holds by less than q 2^-44 before it is rounded. 32-bit inputs are divided in 64 bits.
// The scale's range and its quotient by 15 are taken in 64 bits for every type.
//
// Bound by the instructions of the quantisation, 306 per wave: 2,048 tokens of 8 heads in bf16, 19 MB with
// the stored values returned, 7.6 us with vector issue at 90 % (a row over 32 lanes and library divisions:
// 13; fp32 9.4, fp16 with bf16 9.7); a few tokens are one chain of round trips, 3.5 us.
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

// The lane's value by xor 1 (STEP 0) or 2 (STEP 1) within 4 lanes.
template <int STEP>
__device__ __forceinline__ float dpp4(float v) {
  const int w = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, w, STEP ? 0x4E : 0xB1, 0xF, 0xF, false));
}

// (hi - lo) / 15 rounded up to 7 significant bits, at least 2^-14.
__device__ __forceinline__ float nib_step(float lo, float hi) {
  const double t = ((double)hi - (double)lo) / 15.0;
  const uint64_t low = (1ull << 46) - 1;
  const uint64_t b = (__builtin_bit_cast(uint64_t, t) + low) & ~low;
  return fmaxf((float)__builtin_bit_cast(double, b), kNibMinScale);
}

// rint(x / s); r is 1 / s to an ulp.
template <bool WIDE>
__device__ __forceinline__ float nib_quot(float x, float s, float r) {
  if constexpr (WIDE) return (float)rint((double)x / (double)s);
  const float q = x * r;
  return rintf(fmaf(fmaf(-q, s, x), r, q));
}

// DT: the type of keys and values, or -1 where they differ (then by the arguments, as 32-bit inputs).
template <int DT>
__global__ __launch_bounds__(256) void nibble_write_kernel(NibWriteArgs a) {
  constexpr bool WIDE = DT < 0 || DT == TTKV_DTYPE_F32;
  const int lane = threadIdx.x & 63, i = lane & 15, g = i >> 2;  // dims 8 i .. 8 i + 7, of group g
  const bool val = lane >= 32;
  const int h = (int)(blockIdx.x % (unsigned)a.H);
  const int64_t tok = (int64_t)(blockIdx.x / (unsigned)a.H) * 8 + (threadIdx.x >> 6) * 2 + ((lane >> 4) & 1);
  if (tok >= a.num_tokens) return;
  const int64_t slot = *gbl(a.slots + tok);
  if (slot < 0) return;  // a padded token
  if (slot >= a.n_slots) {
    if ((lane & 47) == 0) atomicOr(a.err, TTKV_ERR_BAD_SLOT);
    return;
  }
  const void* src = val ? a.v : a.k;
  const int dt = DT >= 0 ? DT : val ? a.v_dtype : a.k_dtype;
  const int64_t stride = val ? a.v_row_stride : a.k_row_stride;
  float x[8];
  load_act_n<8>(src, dt, tok * stride + (int64_t)h * kD + 8 * i, act_rows_aligned(src, dt, stride), x);
  float odd = 0.f;  // NaN where an input is not finite
  float lo = 0.f, hi = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    odd = fmaf(x[j], 0.f, odd);
    x[j] = fminf(fmaxf(x[j], -kNibMax), kNibMax);
    lo = fminf(lo, x[j]);
    hi = fmaxf(hi, x[j]);
  }
  odd += dpp4<0>(odd);
  odd += dpp4<1>(odd);
  lo = fminf(lo, dpp4<0>(lo));
  lo = fminf(lo, dpp4<1>(lo));
  hi = fmaxf(hi, dpp4<0>(hi));
  hi = fmaxf(hi, dpp4<1>(hi));
  const bool bad = odd != odd;
  if (bad) lo = hi = 0.f;
  const float s = nib_step(lo, hi), r = __builtin_amdgcn_rcpf(s);
  const float z = nib_quot<WIDE>(-lo, s, r);
  float c[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    c[j] = bad ? 0.f : fminf(fmaxf(nib_quot<WIDE>(x[j], s, r) + z, 0.f), 15.f);
  const uint32_t par =
      bad ? 0x7e00u : __builtin_bit_cast(uint16_t, (_Float16)s) | (uint32_t)z;

  _Float16* outp = val ? a.v_out : a.k_out;
  if (outp) {
    const float f = bad ? NAN : s;
    half8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (_Float16)((c[j] - z) * f);
    *gblw((half8*)(outp + (tok * a.H + h) * kD + 8 * i)) = o;
  }
  uint8_t* rec = a.page + (slot >> 4) * (kNibTile * a.slot_stride) + (int64_t)h * kNibRecord;
  const int u = (int)(slot & 15), n = i & 3;
  // codes are joined as integers below 2^24 that fp32 holds exactly
  if (!val) {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      w[j] = (uint32_t)fmaf(c[4 * j + 3], 1048576.f,
                            fmaf(c[4 * j + 1], 65536.f, fmaf(c[4 * j + 2], 16.f, c[4 * j])));
    *gblw((uint32_t*)rec + (n * 16 + u) * 4 + g) = w[0] | (w[1] << 8);
    if (n == 0) *gblw((uint16_t*)(rec + kNibKp) + u * 4 + g) = (uint16_t)par;
  } else {
    const int q4 = u >> 2, pair = (u >> 1) & 1;
    uint8_t* b = rec + kNibV + (((q4 * 16 + 4 * n) * 2 + pair) * 2 + (g >> 1)) * 4 + 2 * (u & 1) + (g & 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) *gblw(b + 16 * j) = (uint8_t)fmaf(c[2 * j + 1], 16.f, c[2 * j]);
    if (n == 0) *gblw((uint16_t*)(rec + kNibVp) + (q4 * 4 + g) * 4 + (u & 3)) = (uint16_t)par;
  }
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
  const int64_t grid = ((int64_t)num_tokens + 7) / 8 * H;
  if (grid > 0x7fffffff) return host_fail(TTKV_E_INVALID, "too many tokens for one call");
  NibWriteArgs a{key,   val,  k_dtype, v_dtype,     k_row_stride,     v_row_stride,     slots, num_tokens,
                 H,     page, n_slots, slot_stride, (_Float16*)k_out, (_Float16*)v_out, err};
  auto kernel = k_dtype != v_dtype               ? nibble_write_kernel<-1>
                : k_dtype == TTKV_DTYPE_F32 ? nibble_write_kernel<TTKV_DTYPE_F32>
                : k_dtype == TTKV_DTYPE_F16 ? nibble_write_kernel<TTKV_DTYPE_F16>
                                            : nibble_write_kernel<TTKV_DTYPE_BF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("nibble write launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
