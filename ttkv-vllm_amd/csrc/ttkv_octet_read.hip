// Read of stored keys and values out of the 8-bit cache (format: ttkv_octet.h) as rows. gfx950 / CDNA4.
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_octet.h"

namespace ttkv {

struct OctReadArgs {
  int H;
  const uint8_t* page;
  int64_t tile_stride;
  int num_blocks, tpb;  // tpb: tiles per block
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* starts;
  const int32_t* first;
  int max_seq, num_rows;
  void* k_out;
  void* v_out;
  int64_t k_stride, v_stride;
  int out_dtype;
  int32_t* err;
};

// One workgroup per (request, KV head); a thread per 8 dims of a row.
template <int D>
__global__ __launch_bounds__(256) void octet_read_kernel(OctReadArgs a) {
  using F = Oct<D>;
  constexpr int kLanes = D / 8;
  const int h = (int)(blockIdx.x % (unsigned)a.H), r = (int)(blockIdx.x / (unsigned)a.H);
  const int i = threadIdx.x % kLanes, x = 8 * i;
  const int64_t row0 = a.starts[r], rows = (int64_t)a.starts[r + 1] - row0;
  const int64_t t0 = a.first ? a.first[r] : 0;
  for (int64_t k = threadIdx.x / kLanes; k < rows; k += 256 / kLanes) {
    const int64_t row = row0 + k, t = t0 + k;
    if (row < 0 || row >= a.num_rows) {
      if (h == 0 && i == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
      continue;
    }
    float kv[2][8];
    for (int j = 0; j < 8; ++j) kv[0][j] = kv[1][j] = NAN;
    if (t < 0 || t >= a.max_seq) {
      if (h == 0 && i == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
    } else {
      const int tile = (int)(t / kOctTile), b = tile / a.tpb, u = (int)(t % kOctTile);
      const int id = a.bt[r * a.bt_row_stride + b];
      if ((uint32_t)id >= (uint32_t)a.num_blocks) {
        if (h == 0 && i == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
      } else {
        const uint8_t* rec =
            a.page + ((int64_t)id * a.tpb + tile - b * a.tpb) * a.tile_stride + (int64_t)h * F::kRecord;
        const float kp = oct_power(rec[F::key_power(u, x / 32)]), vp = oct_power(rec[F::value_power(u, x / 32)]);
        for (int j = 0; j < 8; ++j) {
          kv[0][j] = (float)oct_pair<false>(rec[F::key(u, x + j)], kp)[0];
          kv[1][j] = (float)oct_pair<false>(rec[F::value(u, x + j)], vp)[0];
        }
      }
    }
    for (int j = 0; j < 8; ++j) {
      store_act(a.k_out, a.out_dtype, row * a.k_stride + h * D + x + j, kv[0][j]);
      store_act(a.v_out, a.out_dtype, row * a.v_stride + h * D + x + j, kv[1][j]);
    }
  }
}

int octet_check_table(int bs, int64_t n_slots, int num_reqs, int max_blocks, int max_seq) {
  if (bs <= 0 || bs % kOctTile || n_slots % bs)
    return host_fail(TTKV_E_INVALID, "the block size must be a multiple of 16 that divides the page's slots");
  if (n_slots / kOctTile > 0x7fffffff)
    return host_fail(TTKV_E_UNSUPPORTED, "more than 2^31 tiles of 16 slots");
  if (max_seq > (1 << 26)) return host_fail(TTKV_E_UNSUPPORTED, "max_seq_len beyond 2^26");
  if (num_reqs < 0 || max_seq < 0 || max_blocks < 0) return host_fail(TTKV_E_INVALID, "negative count");
  if ((int64_t)max_blocks * bs < max_seq)
    return host_fail(TTKV_E_INVALID, "max_seq_len needs more blocks than the block table holds");
  return TTKV_OK;
}

int octet_read_paged(int H, int d, const uint8_t* page, int64_t n_slots, int64_t slot_stride, int bs,
                     const int32_t* bt, int64_t bt_row_stride, int max_blocks, const int32_t* starts,
                     const int32_t* first, int num_reqs, int max_seq, int num_rows, void* k_out,
                     int64_t k_stride, void* v_out, int64_t v_stride, int out_dtype, int32_t* err,
                     hipStream_t st) {
  if (int rc = octet_check_page(H, d, page, n_slots, slot_stride)) return rc;
  if (int rc = octet_check_table(bs, n_slots, num_reqs, max_blocks, max_seq)) return rc;
  if (out_dtype != TTKV_DTYPE_F32 && out_dtype != TTKV_DTYPE_F16 && out_dtype != TTKV_DTYPE_BF16)
    return host_fail(TTKV_E_INVALID, "key_out / value_out dtype must be fp32, fp16 or bf16");
  if (num_rows < 0) return host_fail(TTKV_E_INVALID, "negative count");
  if (num_reqs == 0 || num_rows == 0) return TTKV_OK;
  if (!bt || !starts || !k_out || !v_out || !err) return host_fail(TTKV_E_INVALID, "null pointer argument");
  if ((int64_t)num_reqs * H > 0x7fffffff) return host_fail(TTKV_E_INVALID, "too many requests for one call");
  OctReadArgs a{H,     page,    kOctTile * slot_stride, (int)(n_slots / bs), bs / kOctTile, bt,       bt_row_stride,
                starts, first,  max_seq,                num_rows,            k_out,         v_out,    k_stride,
                v_stride, out_dtype, err};
  auto kernel = d == 64 ? octet_read_kernel<64> : d == 128 ? octet_read_kernel<128> : octet_read_kernel<256>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(num_reqs * H)), dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("octet read launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
