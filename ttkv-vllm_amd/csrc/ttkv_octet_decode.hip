// Attention of new tokens over the 8-bit cache (format: ttkv_octet.h): one query per request, or a few
// drafts. gfx950 / CDNA4.
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_octet.h"

namespace ttkv {

constexpr int kODMaxQ = 16;  // queries per request

struct OctDecodeArgs {
  int H, G;
  float scale;
  const void* q;
  int q_dtype;
  int64_t q_row_stride;
  int num_tokens;
  const uint8_t* page;
  int64_t tile_stride;
  int num_blocks, tpb;
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* seq_lens;
  const int32_t* qsl;
  int max_q, max_seq, window;
  const float* sinks;
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  float* lse;
  int32_t* err;
};

// One workgroup per (request, query, query head); a wave per key in turn, joined in LDS.
template <int D>
__global__ __launch_bounds__(256) void octet_decode_kernel(OctDecodeArgs a) {
  using F = Oct<D>;
  constexpr int N = D / 64;
  __shared__ float sh[4][D + 2];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, HQ = a.H * a.G;
  const int hq = (int)(blockIdx.x % (unsigned)HQ), h = hq / a.G;
  const int j = (int)(blockIdx.x / (unsigned)HQ % (unsigned)a.max_q), r = (int)(blockIdx.x / (unsigned)HQ / (unsigned)a.max_q);
  const int n = min(max(a.seq_lens[r], 0), a.max_seq), row0 = a.qsl[r], Q = a.qsl[r + 1] - row0;
  const bool first = threadIdx.x == 0 && hq == 0 && j == 0;
  if (first && (a.seq_lens[r] > a.max_seq || Q > a.max_q || (n > 0 && n < Q))) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
  if (j >= Q) return;
  const int64_t row = (int64_t)row0 + j;
  if (row < 0 || row >= a.num_tokens) {
    if (threadIdx.x == 0 && hq == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
    return;
  }
  const int at = n - Q + j, lo = a.window > 0 ? max(0, at - a.window + 1) : 0;
  float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
  for (int k = 0; k < N; ++k) q[k] = load_act(a.q, a.q_dtype, row * a.q_row_stride + (int64_t)hq * D + lane * N + k);
  bool bad = n > 0 && n < Q;
  for (int t = lo + wv; t <= at; t += 4) {
    const int tile = t / kOctTile, b = tile / a.tpb, u = t % kOctTile, id = a.bt[r * a.bt_row_stride + b];
    if ((uint32_t)id >= (uint32_t)a.num_blocks) {
      if (lane == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
      bad = true;
      break;
    }
    const uint8_t* rec = a.page + ((int64_t)id * a.tpb + tile - b * a.tpb) * a.tile_stride + (int64_t)h * F::kRecord;
    float s = 0.f, v[N];
    for (int k = 0; k < N; ++k) {
      const int x = lane * N + k;
      s = fmaf(q[k], (float)oct_pair<false>(rec[F::key(u, x)], oct_power(rec[F::key_power(u, x / 32)]))[0], s);
      v[k] = (float)oct_pair<false>(rec[F::value(u, x)], oct_power(rec[F::value_power(u, x / 32)]))[0];
    }
    s = wave_sum(s) * a.scale;
    const float mn = fmaxf(m, s), f = m == mn ? 1.f : expf(m - mn), p = expf(s - mn);
    l = l * f + p;
    for (int k = 0; k < N; ++k) o[k] = o[k] * f + p * v[k];
    m = mn;
  }
  if (bad) l = NAN;
  for (int k = 0; k < N; ++k) sh[wv][lane * N + k] = o[k];
  if (lane == 0) {
    sh[wv][D] = m;
    sh[wv][D + 1] = l;
  }
  __syncthreads();
  float M = a.sinks ? a.sinks[hq] : -INFINITY;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sh[w][D]);
  float total = a.sinks && M > -INFINITY ? expf(a.sinks[hq] - M) : 0.f;
  float x = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float f = sh[w][D] == -INFINITY ? 0.f : expf(sh[w][D] - M);
    total += sh[w][D + 1] != sh[w][D + 1] ? NAN : sh[w][D + 1] * f;
    if (threadIdx.x < D) x += f == 0.f ? 0.f : sh[w][threadIdx.x] * f;
  }
  if (threadIdx.x < D)
    store_act(a.out, a.out_dtype, row * a.out_row_stride + (int64_t)hq * D + threadIdx.x, total == 0.f ? 0.f : x / total);
  if (a.lse && threadIdx.x == 0) a.lse[row * HQ + hq] = total == 0.f ? -INFINITY : M + logf(total);
}

int64_t octet_decode_workspace_bytes(int H, int HQ, int d, int num_reqs, int max_q, int max_seq) { return 256; }

int octet_decode_paged(int H, int HQ, int d, float scale, const void* q, int q_dtype, int64_t q_row_stride,
                       int num_tokens, const uint8_t* page, int64_t n_slots, int64_t slot_stride, int bs,
                       const int32_t* bt, int64_t bt_row_stride, int max_blocks, const int32_t* seq_lens,
                       const int32_t* qsl, int num_reqs, int max_q, int max_seq, int window,
                       const float* sinks, void* out, int out_dtype, int64_t out_row_stride, float* lse,
                       void* ws, int64_t ws_bytes, int32_t* err, hipStream_t st) {
  if (int rc = octet_check_page(H, d, page, n_slots, slot_stride)) return rc;
  if (int rc = octet_check_table(bs, n_slots, num_reqs, max_blocks, max_seq)) return rc;
  if (HQ <= 0 || HQ % H) return host_fail(TTKV_E_INVALID, "num_heads is not a multiple of H");
  if (HQ / H > 16) return host_fail(TTKV_E_UNSUPPORTED, "more than 16 query heads per KV head");
  for (int dt : {q_dtype, out_dtype})
    if (dt != TTKV_DTYPE_F16 && dt != TTKV_DTYPE_BF16)
      return host_fail(TTKV_E_INVALID, "query / out dtype must be fp16 or bf16");
  if (num_tokens < 0 || max_q < 0) return host_fail(TTKV_E_INVALID, "negative count");
  if (max_q > kODMaxQ) return host_fail(TTKV_E_UNSUPPORTED, "more than 16 queries per request");
  if (window < 0) return host_fail(TTKV_E_INVALID, "negative window");
  if (num_reqs && (!q || !bt || !seq_lens || !qsl || !out || !err))
    return host_fail(TTKV_E_INVALID, "null pointer argument");
  if (((uintptr_t)q | (uintptr_t)out) % 16 || q_row_stride % 8 || out_row_stride % 8)
    return host_fail(TTKV_E_INVALID, "query / out rows must be 16-byte aligned");
  const int64_t need = octet_decode_workspace_bytes(H, HQ, d, num_reqs, max_q, max_seq);
  if (!ws || ws_bytes < need || (uintptr_t)ws % 256)
    return host_fail(TTKV_E_WORKSPACE, "decode workspace needs " + std::to_string(need) + " bytes, 256-aligned");
  if (num_reqs == 0 || num_tokens == 0 || max_q == 0) return TTKV_OK;
  if (window >= max_seq) window = 0;  // no window
  OctDecodeArgs a{H,        HQ / H,     scale,          q,   q_dtype,       q_row_stride, num_tokens, page,
                  kOctTile * slot_stride, (int)(n_slots / bs), bs / kOctTile, bt, bt_row_stride, seq_lens, qsl, max_q,
                  max_seq,  window,     sinks,          out, out_dtype,     out_row_stride, lse,    err};
  auto kernel = d == 64 ? octet_decode_kernel<64> : d == 128 ? octet_decode_kernel<128> : octet_decode_kernel<256>;
  const int64_t grid = (int64_t)num_reqs * max_q * HQ;
  if (grid > 0x7fffffff) return host_fail(TTKV_E_INVALID, "too many requests for one call");
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("octet decode launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
