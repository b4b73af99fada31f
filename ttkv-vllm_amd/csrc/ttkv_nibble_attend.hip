// Attention over the 4-bit cache (format: ttkv_nibble.h). gfx950 / CDNA4.
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_nibble.h"

namespace ttkv {

struct NibAttendArgs {
  int H, HQ, G;
  float scale_log2;
  const void* q;
  int dtype;
  int64_t q_row_stride;
  const uint8_t* page;
  int64_t num_blocks, slot_stride;
  int bs;
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* seq_lens;
  const int32_t* qsl;
  const int32_t* req_index;
  int num_reqs, max_q, max_seq;
  bool decode;
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  int32_t* err;
};

__device__ __forceinline__ float nib_scale(uint32_t p) { return f16_bits_to_float(p & 0xfff0u); }
__device__ __forceinline__ float nib_zero(uint32_t p) { return (float)(p & 15u); }

// One wave per (request, query, query head): lane l owns dims 2 l and 2 l + 1.
__global__ __launch_bounds__(64) void nibble_attend_kernel(NibAttendArgs a) {
  const int lane = threadIdx.x;
  const int hq = blockIdx.x, j = blockIdx.y, rr = blockIdx.z;
  const int r = a.req_index ? a.req_index[rr] : rr;
  const int h = hq / a.G;
  const int64_t q0 = a.qsl[r];
  const int Q = a.decode ? 1 : a.qsl[r + 1] - (int)q0;
  if (j >= Q) return;
  int n = max(a.seq_lens[r], 0), bits = 0;
  if (n > a.max_seq || (j == 0 && Q > a.max_q)) bits |= TTKV_ERR_SEQ_LEN;
  n = min(n, a.max_seq);
  bool bad = !a.decode && n < Q;
  if (bad) bits |= TTKV_ERR_SEQ_LEN;
  const int last = a.decode ? n : n - Q + j + 1;  // keys this query sees
  const int64_t at = (q0 + j) * a.q_row_stride + (int64_t)hq * kD + 2 * lane;
  const float qa = load_act(a.q, a.dtype, at) * a.scale_log2;
  const float qb = load_act(a.q, a.dtype, at + 1) * a.scale_log2;
  float m = -INFINITY, l = 0.f, oa = 0.f, ob = 0.f;
  const int g = lane >> 4, jj = (2 * lane) & 7, qd = (lane & 15) >> 2, nn = lane & 15;
  for (int t = 0; t < last && !bad; ++t) {
    const int blk = a.bt[(int64_t)r * a.bt_row_stride + t / a.bs];
    if (blk < 0 || blk >= a.num_blocks) {
      bits |= TTKV_ERR_BAD_BLOCK;
      bad = true;
      break;
    }
    const int64_t slot = (int64_t)blk * a.bs + t % a.bs;
    const uint8_t* rec = a.page + (slot >> 4) * (kNibTile * a.slot_stride) + h * kNibRecord;
    const int u = (int)(slot & 15);
    const uint32_t kw = *((const uint32_t*)rec + (qd * 16 + u) * 4 + g) >> (2 * jj);
    const uint32_t kp = *((const uint16_t*)(rec + kNibKp) + u * 4 + g);
    const float ks = nib_scale(kp), kz = nib_zero(kp);
    float s = qa * (((float)(kw & 15u) - kz) * ks) + qb * (((float)((kw >> 16) & 15u) - kz) * ks);
    s = wave_sum(s);
    const uint32_t vw = *((const uint32_t*)(rec + kNibV) +
                          (((u >> 2) * 16 + nn) * 2 + ((u >> 1) & 1)) * 2 + (g >> 1)) >>
                        (16 * (u & 1) + 8 * (g & 1));
    const uint32_t vp = *((const uint16_t*)(rec + kNibVp) + ((u >> 2) * 4 + g) * 4 + (u & 3));
    const float vs = nib_scale(vp), vz = nib_zero(vp);
    const float mn = fmaxf(m, s);
    const float f = m == -INFINITY ? 0.f : exp2f(m - mn), p = exp2f(s - mn);
    l = l * f + p;
    oa = oa * f + p * (((float)(vw & 15u) - vz) * vs);
    ob = ob * f + p * (((float)((vw >> 4) & 15u) - vz) * vs);
    m = mn;
  }
  if (bits && lane == 0) atomicOr(a.err, bits);
  const float inv = bad ? NAN : last <= 0 ? 0.f : 1.f / l;
  const int64_t to = (q0 + j) * a.out_row_stride + (int64_t)hq * kD + 2 * lane;
  store_act(a.out, a.out_dtype, to, oa * inv);
  store_act(a.out, a.out_dtype, to + 1, ob * inv);
}

int nibble_check_read(int H, int HQ, int d, const void* q, int q_dtype,
                               int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                               int64_t slot_stride, int bs, const int32_t* bt, int max_blocks,
                               const int32_t* seq_lens, const int32_t* qsl, int num_reqs,
                               int max_seq, const void* out, int out_dtype,
                               int64_t out_row_stride, const int32_t* err) {
  if (int rc = nibble_check_page(H, d, page, n_slots, slot_stride)) return rc;
  if (HQ <= 0 || HQ % H) return host_fail(TTKV_E_INVALID, "num_heads is not a multiple of H");
  if (HQ / H > 16)
    return host_fail(TTKV_E_UNSUPPORTED, "more than 16 query heads per KV head");
  for (int dt : {q_dtype, out_dtype})
    if (dt != TTKV_DTYPE_F16 && dt != TTKV_DTYPE_BF16)
      return host_fail(TTKV_E_INVALID, "query / out dtype must be fp16 or bf16");
  if (bs <= 0 || bs % kNibTile || n_slots % bs)
    return host_fail(TTKV_E_INVALID, "the block size must be a multiple of 16 that divides the "
                                     "page's slots");
  if (n_slots / kNibTile > 0x7fffffff)
    return host_fail(TTKV_E_UNSUPPORTED, "more than 2^31 tiles of 16 slots");
  if (num_reqs < 0 || max_seq < 0 || max_blocks < 0)
    return host_fail(TTKV_E_INVALID, "negative count");
  if ((int64_t)max_blocks * bs < max_seq)
    return host_fail(TTKV_E_INVALID, "max_seq_len needs more blocks than the block table holds");
  if (num_reqs && (!q || !bt || !seq_lens || !qsl || !out || !err))
    return host_fail(TTKV_E_INVALID, "null pointer argument");
  if (((uintptr_t)q | (uintptr_t)out) % 16 || q_row_stride % 8 || out_row_stride % 8)
    return host_fail(TTKV_E_INVALID, "query / out rows must be 16-byte aligned");
  return TTKV_OK;
}

static int nibble_attend(int H, int HQ, float scale, const void* q, int q_dtype,
                         int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                         int64_t slot_stride, int bs, const int32_t* bt, int64_t bt_row_stride,
                         const int32_t* seq_lens, const int32_t* qsl, const int32_t* req_index,
                         int num_reqs, int max_q, int max_seq, bool decode, void* out,
                         int out_dtype, int64_t out_row_stride, int32_t* err, hipStream_t st) {
  NibAttendArgs a{H, HQ, HQ / H, scale * 1.4426950408889634f, q, q_dtype, q_row_stride, page,
                  n_slots / bs, slot_stride, bs, bt, bt_row_stride, seq_lens, qsl, req_index,
                  num_reqs, max_q, max_seq, decode, out, out_dtype, out_row_stride, err};
  hipLaunchKernelGGL(nibble_attend_kernel, dim3(HQ, max_q, num_reqs), dim3(64), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("nibble attend launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

int64_t nibble_prefill_workspace_bytes(int H, int HQ, int num_reqs, int max_q, int max_seq) {
  return 256;
}

int nibble_prefill_paged(int H, int HQ, int d, float scale, const void* q, int q_dtype,
                         int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                         int64_t slot_stride, int bs, const int32_t* bt, int64_t bt_row_stride,
                         int max_blocks, const int32_t* seq_lens, const int32_t* qsl,
                         const int32_t* req_index, int num_reqs, int max_q, int max_seq,
                         void* out, int out_dtype, int64_t out_row_stride, void* ws,
                         int64_t ws_bytes, int32_t* err, hipStream_t st) {
  if (int rc = nibble_check_read(H, HQ, d, q, q_dtype, q_row_stride, page, n_slots, slot_stride,
                                   bs, bt, max_blocks, seq_lens, qsl, num_reqs, max_seq, out,
                                   out_dtype, out_row_stride, err))
    return rc;
  if (max_q < 0) return host_fail(TTKV_E_INVALID, "negative max_q_len");
  if (max_q > max_seq) return host_fail(TTKV_E_INVALID, "max_q_len is longer than max_seq_len");
  const int64_t need = nibble_prefill_workspace_bytes(H, HQ, num_reqs, max_q, max_seq);
  if (!ws || ws_bytes < need || (uintptr_t)ws % 256)
    return host_fail(TTKV_E_WORKSPACE, "prefill workspace needs " + std::to_string(need) +
                                           " bytes, 256-aligned");
  if (num_reqs == 0 || max_q == 0) return TTKV_OK;
  return nibble_attend(H, HQ, scale, q, q_dtype, q_row_stride, page, n_slots, slot_stride, bs, bt,
                       bt_row_stride, seq_lens, qsl, req_index, num_reqs, max_q, max_seq, false,
                       out, out_dtype, out_row_stride, err, st);
}

}  // namespace ttkv
