// Read of stored keys and values out of the 8-bit cache (format: ttkv_octet.h) as rows. gfx950 / CDNA4.
// Bound by memory: every stored byte read and every row written once. 4 x 7,656 tokens of 8 heads, 190 MB,
// 31.0 us, 6.1 TB/s (a copy whose stores stay in the caches reaches 5.0); 700 tokens
// 4.4 us, a chain of scan, block id, record and store.
#include <math.h>

#include <type_traits>

#include "ttkv_host.h"
#include "ttkv_nibble.h"
#include "ttkv_octet.h"

namespace ttkv {

struct OctReadArgs {
  int H, num_reqs;
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

// A request's rows that the outputs hold, and the tiles of their tokens.
struct OctReadRows {
  int64_t t0;        // output row k holds token t0 + k,
  int row0, lo, hi;  // k in [lo, hi)
  int tile, tiles;
};
__device__ __forceinline__ OctReadRows oct_read_rows(const OctReadArgs& a, int r, bool& clipped) {
  OctReadRows x;
  x.row0 = a.starts[r];
  const int end = a.starts[r + 1];
  x.t0 = (int64_t)(a.first ? a.first[r] : 0) - x.row0;
  x.lo = max(0, x.row0);
  x.hi = min(end, a.num_rows);
  clipped = end < x.row0 || (end > x.row0 && (x.row0 < 0 || end > a.num_rows));
  x.tile = (int)((x.t0 + x.lo) >> 4);
  x.tiles = x.hi > x.lo ? (int)((x.t0 + x.hi - 1) >> 4) - x.tile + 1 : 0;
  return x;
}

// Eight elements of a row, rounded once, by stores that do not stay in the caches: rows are whole lines, and
// what is read beside them stays instead (8 x 8,000 tokens of 64 dims: 44.3 us with stores that stay, 31.5 so; 4 x
// 4,000 of 256 46.8, 31.5; loads that do not stay cost up to a quarter).
template <int DT>
__device__ __forceinline__ void oct_read_store(void* out, int64_t i, const float f[8]) {
  if constexpr (DT == TTKV_DTYPE_F32) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      __builtin_nontemporal_store(float4v{f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]},
                                  gblw((float4v*)((float*)out + i) + j));
  } else {
    typedef std::conditional_t<DT == TTKV_DTYPE_F16, _Float16, __bf16> T;
    typedef T T8 __attribute__((ext_vector_type(8)));
    T8 w;
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = (T)f[j];
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, w), gblw((u32x4*)((uint16_t*)out + i)));
  }
}

// A wave per (tile, KV head): its lanes take 8 dims of a row each, d / 8 lanes a row, so that rows are
// stored whole, and every load of the record is under way before the first is used.
template <int D, int DT, bool VEC>
__global__ __launch_bounds__(256) void octet_read_kernel(OctReadArgs a) {
  using F = Oct<D>;
  constexpr int kLanes = D / 8, kRows = 64 / kLanes, kRounds = 16 / kRows;
  const int lane = threadIdx.x & 63;
  const int i = lane % kLanes, x = 8 * i;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);; item += waves) {
    const int64_t want = item / a.H;
    const int h = (int)(item - want * a.H);
    // the request whose tiles hold number `want`
    int r = -1;
    int64_t before = 0;
    OctReadRows rq{};
    for (int r0 = 0; r0 < a.num_reqs && r < 0; r0 += 64) {
      bool clipped = false;
      OctReadRows mine{};
      if (r0 + lane < a.num_reqs) mine = oct_read_rows(a, r0 + lane, clipped);
      if (clipped && item == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
      const int incl = nib_scan(mine.tiles);
      const int64_t at = want - before;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(at < incl && mine.tiles > 0);
      if (hit) {
        const int ln = __builtin_ctzll(hit);
        r = r0 + ln;
        rq.row0 = __builtin_amdgcn_readlane(mine.row0, ln);
        rq.lo = __builtin_amdgcn_readlane(mine.lo, ln);
        rq.hi = __builtin_amdgcn_readlane(mine.hi, ln);
        rq.t0 = (int64_t)(a.first ? a.first[r] : 0) - rq.row0;
        rq.tile = __builtin_amdgcn_readlane(mine.tile, ln) + (int)at - __builtin_amdgcn_readlane(incl - mine.tiles, ln);
      }
      before += __builtin_amdgcn_readlane(incl, 63);
      if (item == 0 && r >= 0)  // (the requests behind the first hit are looked at for their rows, too)
        for (int k = r0 + 64 + lane; k < a.num_reqs; k += 64) {
          oct_read_rows(a, k, clipped);
          if (clipped) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
        }
    }
    if (r < 0) return;
    const int64_t tok = (int64_t)rq.tile * 16;
    // a token outside the call's lengths or a block outside the cache: NaN
    const int b = rq.tile < 0 ? 0 : rq.tile / a.tpb;
    int id = -1;
    if (tok >= 0 && tok < a.max_seq) {
      id = a.bt[r * a.bt_row_stride + b];
      if ((uint32_t)id >= (uint32_t)a.num_blocks) {
        id = -1;
        if (lane == 0 && h == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
      }
    }
    const uint8_t* rec = a.page + ((int64_t)max(id, 0) * a.tpb + max(rq.tile, 0) - b * a.tpb) * a.tile_stride +
                         (int64_t)h * F::kRecord;
    u32x2v c[2][kRounds];
    uint8_t pw[2][kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int u = k * kRows + lane / kLanes;
      c[0][k] = *gbl((const u32x2v*)(rec + F::key(u, x)));
      pw[0][k] = *gbl(rec + F::key_power(u, x / 32));
      if constexpr (D == 64) {
        c[1][k][0] = *gbl((const uint32_t*)(rec + F::value(u, x)));
        c[1][k][1] = *gbl((const uint32_t*)(rec + F::value(u, x + 4)));
      } else {
        c[1][k] = *gbl((const u32x2v*)(rec + F::value(u, x)));
      }
      pw[1][k] = *gbl(rec + F::value_power(u, x / 32));
    }
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int64_t t = tok + k * kRows + lane / kLanes, at = t - rq.t0;
      if (at < rq.lo || at >= rq.hi) continue;
      const bool in = t >= 0 && t < a.max_seq;
      if (!in && h == 0 && i == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
      const bool nan = id < 0 || !in;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const float p = oct_power(pw[kv][k]);
        bf16x2 o[4] = {oct_pair<false>(c[kv][k][0], p), oct_pair<true>(c[kv][k][0], p),
                       oct_pair<false>(c[kv][k][1], p), oct_pair<true>(c[kv][k][1], p)};
        const int64_t to = at * (kv ? a.v_stride : a.k_stride) + (int64_t)h * D + x;
        void* out = kv ? a.v_out : a.k_out;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = nan ? NAN : (float)o[j >> 1][j & 1];
        if constexpr (VEC) {
          oct_read_store<DT>(out, to, f);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) store_act(out, DT, to + j, f[j]);
        }
      }
    }
  }
}

template <int D, int DT>
static void oct_read_launch(const OctReadArgs& a, unsigned grid, bool vec, hipStream_t st) {
  if (vec)
    hipLaunchKernelGGL((octet_read_kernel<D, DT, true>), dim3(grid), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((octet_read_kernel<D, DT, false>), dim3(grid), dim3(256), 0, st, a);
}
template <int D>
static void oct_read_launch(const OctReadArgs& a, unsigned grid, bool vec, hipStream_t st) {
  if (a.out_dtype == TTKV_DTYPE_F32) oct_read_launch<D, TTKV_DTYPE_F32>(a, grid, vec, st);
  else if (a.out_dtype == TTKV_DTYPE_F16) oct_read_launch<D, TTKV_DTYPE_F16>(a, grid, vec, st);
  else oct_read_launch<D, TTKV_DTYPE_BF16>(a, grid, vec, st);
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
  const int64_t eb = out_dtype == TTKV_DTYPE_F32 ? 4 : 2;
  if (rows_meet(k_out, k_stride * eb, H * d * eb, v_out, v_stride * eb, H * d * eb, num_rows))
    return host_fail(TTKV_E_INVALID, "key_out and value_out overlap");
  if (rows_fold(k_stride, H * d, num_rows) || rows_fold(v_stride, H * d, num_rows))
    return host_fail(TTKV_E_INVALID, "rows of an output overlap one another");
  // wide stores where every row starts 16-byte aligned; else an element at a time
  const bool vec = ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0 && (k_stride * eb | v_stride * eb) % 16 == 0;
  OctReadArgs a{H,     num_reqs, page,    kOctTile * slot_stride, (int)(n_slots / bs), bs / kOctTile, bt, bt_row_stride,
                starts, first,   max_seq, num_rows,               k_out,               v_out,         k_stride, v_stride,
                out_dtype, err};
  // a wave per (tile, head), of rows that start anywhere in a tile; those beyond the grid in turn
  const int64_t items = ((int64_t)num_rows / kOctTile + 2 * (int64_t)num_reqs) * H;
  const unsigned grid = (unsigned)std::min<int64_t>((items + 3) / 4, 1 << 20);
  if (d == 64) oct_read_launch<64>(a, grid, vec, st);
  else if (d == 128) oct_read_launch<128>(a, grid, vec, st);
  else oct_read_launch<256>(a, grid, vec, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("octet read launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
