// A serving step's bookkeeping: block tables, slot map and positions from the requests' lengths
// (step_plan), and rotary positions with one to four axes (rotary_axes). gfx950 / CDNA4.
#include <math.h>

#include "ttkv_device.h"
#include "ttkv_host.h"

namespace ttkv {

// ------------------------------------------------------------------------------- step plan
// One launch. Request r has c stored and n new tokens: it holds have = ceil(c / bs) blocks and needs
// ceil((c + n) / bs); its fresh ones come from the free list at the sum of the requests' before it.
// Every workgroup forms the two prefix sums (new tokens, fresh blocks) over all requests in LDS (a
// few thousand integers from L2, cheaper than a second launch that waits for a first) and then
// takes its share of the tokens, finding each one's request by bisection. A token of a fresh block
// reads its block id from the free list and not from the table, which other workgroups are writing.
// Bound by the chain of dependent reads: 3 us for 8 single tokens, 8.7 for 256 requests of up to 120
// (the scan over the workgroup, then for each of a thread's four tokens eight steps of bisection in LDS
// and two reads); a few KB move.
constexpr int kPlanThreads = 256;
constexpr int kPlanTokens = 4;        // tokens per thread the grid is sized for
constexpr int kPlanMaxReqs = 8000;    // two prefix arrays within 64 KB of LDS
constexpr int kPlanCap = (1 << 30) - 1;  // lengths and their sums saturate here

struct PlanArgs {
  const int32_t* computed;
  const int32_t* qlens;
  int R;
  int32_t* bt;
  int64_t bt_row_stride;
  int W;
  const int32_t* free_ids;
  int F;
  int bs;
  int64_t num_blocks;
  int T;
  int32_t* qsl;
  int32_t* seq;
  int64_t* slots;
  int64_t* pos;
  int32_t* used;
  int32_t* err;
};

__device__ __forceinline__ int sat_add(int a, int b) { return min(a + b, kPlanCap); }
__device__ __forceinline__ int plan_len(int v) { return min(max(v, 0), kPlanCap); }
__device__ __forceinline__ int div_up(int a, int b) { return a / b + (a % b != 0); }

// Last index r in [0, n) with v[r] <= x; v ascends and v[0] = 0 <= x.
__device__ __forceinline__ int last_not_above(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (v[m] <= x) lo = m;
    else hi = m;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void step_plan_kernel(PlanArgs a) {
  extern __shared__ int sh[];
  int* qstart = sh;             // [R] first token of each request
  int* fstart = sh + a.R;       // [R] its first fresh block in the free list
  __shared__ int wsum[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int per = (a.R + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(tid * per, a.R), r1 = min(r0 + per, a.R);
  int sq = 0, sf = 0, bits = 0;
  for (int r = r0; r < r1; ++r) {
    const int cr = a.computed[r], nr = a.qlens[r];
    const int c = plan_len(cr), n = plan_len(nr);
    if (c != cr || n != nr) bits |= TTKV_ERR_SEQ_LEN;
    const int s = sat_add(c, n);
    const int have = min(div_up(c, a.bs), a.W), need = min(div_up(s, a.bs), a.W);
    if (div_up(s, a.bs) > a.W) bits |= TTKV_ERR_SEQ_LEN;
    qstart[r] = sq;
    fstart[r] = sf;
    sq = sat_add(sq, n);
    sf = sat_add(sf, need - have);
  }
  // inclusive scans of the threads' sums over the workgroup
  int iq = sq, jf = sf;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int tq = __shfl_up(iq, o), tf = __shfl_up(jf, o);
    if (lane >= o) {
      iq = sat_add(iq, tq);
      jf = sat_add(jf, tf);
    }
  }
  if (lane == 63) {
    wsum[0][wv] = iq;
    wsum[1][wv] = jf;
  }
  __syncthreads();
  int bq = 0, bf = 0, total = 0, fresh = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wv) {
      bq = sat_add(bq, wsum[0][w]);
      bf = sat_add(bf, wsum[1][w]);
    }
    total = sat_add(total, wsum[0][w]);
    fresh = sat_add(fresh, wsum[1][w]);
  }
  const int uq = __shfl_up(iq, 1), uf = __shfl_up(jf, 1);
  bq = sat_add(bq, lane ? uq : 0);
  bf = sat_add(bf, lane ? uf : 0);
  for (int r = r0; r < r1; ++r) {
    qstart[r] = sat_add(qstart[r], bq);
    fstart[r] = sat_add(fstart[r], bf);
  }
  __syncthreads();
  const int gid = blockIdx.x * kPlanThreads + tid;
  const int step = gridDim.x * kPlanThreads;
  if (total > a.T) bits |= TTKV_ERR_SEQ_LEN;
  if (fresh > a.F) bits |= TTKV_ERR_NO_BLOCK;
  for (int r = gid; r < a.R; r += step) {
    a.qsl[r] = min(qstart[r], a.T);
    a.seq[r] = sat_add(plan_len(a.computed[r]), plan_len(a.qlens[r]));
  }
  if (gid == 0) {
    a.qsl[a.R] = min(total, a.T);
    *a.used = min(fresh, a.F);
  }
  for (int f = gid; f < fresh; f += step) {
    const int r = last_not_above(fstart, a.R, f);
    const int col = div_up(plan_len(a.computed[r]), a.bs) + f - fstart[r];
    const int id = f < a.F ? a.free_ids[f] : -1;
    a.bt[(int64_t)r * a.bt_row_stride + col] = id;
  }
  for (int i = gid; i < a.T; i += step) {
    int64_t slot = -1, pos = 0;
    if (i < total) {
      const int r = last_not_above(qstart, a.R, i);
      const int c = plan_len(a.computed[r]);
      const int p = sat_add(c, i - qstart[r]);
      const int have = div_up(c, a.bs), col = p / a.bs;
      pos = p;
      if (col < a.W) {
        int id = -1;
        if (col < have) {
          id = a.bt[(int64_t)r * a.bt_row_stride + col];
        } else {
          const int f = fstart[r] + col - have;
          if (f < a.F) id = a.free_ids[f];
        }
        if (id >= 0 && id < a.num_blocks)
          slot = (int64_t)id * a.bs + p % a.bs;
        else if (col < have || fstart[r] + col - have < a.F)
          bits |= TTKV_ERR_BAD_BLOCK;
      }
    }
    a.slots[i] = slot;
    a.pos[i] = pos;
  }
  if (bits) atomicOr(a.err, bits);
}

int step_plan(const int32_t* computed, const int32_t* qlens, int R, int32_t* bt,
              int64_t bt_row_stride, int W, const int32_t* free_ids, int F, int bs,
              int64_t num_blocks, int T, int32_t* qsl, int32_t* seq, int64_t* slots, int64_t* pos,
              int32_t* used, int32_t* err, hipStream_t st) {
  if (R < 0 || T < 0 || F < 0 || W < 0 || num_blocks < 0)
    return host_fail(TTKV_E_INVALID, "negative count");
  if (R > kPlanMaxReqs)
    return host_fail(TTKV_E_UNSUPPORTED, "step_plan takes at most 8000 requests");
  if (bs <= 0) return host_fail(TTKV_E_INVALID, "block_size must be positive");
  if (bt_row_stride < W) return host_fail(TTKV_E_INVALID, "block table rows overlap");
  if (T > kPlanCap || num_blocks > 0x7fffffff)
    return host_fail(TTKV_E_INVALID, "too many tokens or blocks for one call");
  if (!qsl || !used || !err || (R && (!computed || !qlens || !seq)) || (R && W && !bt) ||
      (F && !free_ids) || (T && (!slots || !pos)))
    return host_fail(TTKV_E_INVALID, "null pointer argument");
  // Every workgroup reads the lengths and the free list while others write, so no output may lie in
  // them, nor in another output. Ranges in bytes; the table's rows may have gaps between them.
  struct Range {
    uintptr_t at, end;
    bool meets(const Range& o) const { return at < o.end && o.at < end; }
  };
  auto range = [](const void* p, int64_t bytes) { return Range{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes}; };
  const Range outs[] = {range(qsl, ((int64_t)R + 1) * 4), range(seq, (int64_t)R * 4), range(used, 4),
                        range(slots, (int64_t)T * 8), range(pos, (int64_t)T * 8)};
  const Range lens[] = {range(computed, (int64_t)R * 4), range(qlens, (int64_t)R * 4)};
  const Range ids = range(free_ids, (int64_t)F * 4);
  auto in_table = [&](const Range& x) {
    const uintptr_t t0 = (uintptr_t)bt;
    if (!R || !W || x.at >= x.end || x.end <= t0) return false;
    const uint64_t row = (uint64_t)bt_row_stride * 4, from = x.at > t0 ? x.at - t0 : 0, to = x.end - t0;
    if (from / row >= (uint64_t)R) return false;
    return from % row < (uint64_t)W * 4 || (from / row + 1 < (uint64_t)R && to > (from / row + 1) * row);
  };
  for (const Range& x : outs)
    if (x.meets(lens[0]) || x.meets(lens[1]))
      return host_fail(TTKV_E_INVALID, "an output lies in one of the length inputs");
  if (in_table(lens[0]) || in_table(lens[1]))
    return host_fail(TTKV_E_INVALID, "the block table holds one of the length inputs");
  if (in_table(ids)) return host_fail(TTKV_E_INVALID, "the free list lies in the block table");
  for (const Range& x : outs) {
    if (x.meets(ids)) return host_fail(TTKV_E_INVALID, "an output lies in the free list");
    if (in_table(x)) return host_fail(TTKV_E_INVALID, "an output lies in the block table");
    for (const Range& y : outs)
      if (&x != &y && x.meets(y)) return host_fail(TTKV_E_INVALID, "two outputs overlap");
  }
  PlanArgs a{computed, qlens, R, bt,  bt_row_stride, W,     free_ids, F,   bs,
             num_blocks, T,   qsl, seq, slots, pos, used, err};
  const int grid = std::max(1, (T + kPlanThreads * kPlanTokens - 1) / (kPlanThreads * kPlanTokens));
  hipLaunchKernelGGL(step_plan_kernel, dim3(grid), dim3(kPlanThreads), (size_t)R * 8, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("step plan launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

// ----------------------------------------------------------------------------- rotary axes
// y[j] = x[j] cos - x[j + half] sin,  y[j + half] = x[j + half] cos + x[j] sin for j < half =
// rot / 2, the angle row taken at the token's position on frequency j's axis; dims past rot are
// copied. Products and sums in 32 bits, rounded once to the row's type.
constexpr int kRotAxes = 4;

struct RotArgs {
  const void* q;
  const void* k;
  void* qo;
  void* ko;
  int dtype, HQ, H, d, half, N;
  int64_t q_stride, k_stride, qo_stride, ko_stride;
  const int64_t* pos;
  int64_t pos_stride;  // between axes
  int axes, interleaved;
  int sec[kRotAxes];
  const float* cs;
  int64_t max_pos;
  int32_t* err;
};

__device__ __forceinline__ int rot_axis(const RotArgs& a, int j) {
  if (a.interleaved) {
    const int ax = j % a.axes;
    int n = a.sec[0];
#pragma unroll
    for (int i = 1; i < kRotAxes; ++i) n = ax == i ? a.sec[i] : n;
    return j < a.axes * n ? ax : 0;
  }
  int ax = 0, end = a.sec[0];
#pragma unroll
  for (int i = 1; i < kRotAxes; ++i) {
    if (i < a.axes && j >= end) ax = i;
    end += a.sec[i];
  }
  return ax;
}

// The token's position on each axis; false where one is outside the table.
__device__ __forceinline__ bool rot_positions(const RotArgs& a, int64_t tok,
                                              int64_t p[kRotAxes]) {
  bool ok = true;
#pragma unroll
  for (int i = 0; i < kRotAxes; ++i) {
    p[i] = i < a.axes ? a.pos[i * a.pos_stride + tok] : 0;
    if (p[i] < 0 || p[i] >= a.max_pos) {
      ok = false;
      p[i] = 0;
    }
  }
  if (!ok && threadIdx.x == 0) atomicOr(a.err, TTKV_ERR_BAD_POSITION);
  return ok;
}

// Eight consecutive elements of a 16-byte aligned row piece, in registers and as floats.
template <int DT>
struct Rot8 {
  u32x4 raw[DT == TTKV_DTYPE_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Rot8<DT> rot_load8(const void* p, int64_t i) {
  Rot8<DT> x;
  const char* at = (const char*)p + i * (DT == TTKV_DTYPE_F32 ? 4 : 2);
#pragma unroll
  for (int j = 0; j < (DT == TTKV_DTYPE_F32 ? 2 : 1); ++j)
    x.raw[j] = __builtin_nontemporal_load(gbl((const u32x4*)at + j));
  return x;
}
template <int DT>
__device__ __forceinline__ float rot_get(const Rot8<DT>& x, int i) {
  if constexpr (DT == TTKV_DTYPE_F32) {
    const uint32_t w = x.raw[i >> 2][i & 3];  // (by value: a bit cast of an element reads the first)
    return __builtin_bit_cast(float, w);
  }
  const uint32_t w = x.raw[0][i >> 1], b = i & 1 ? w >> 16 : w & 0xffffu;
  return DT == TTKV_DTYPE_F16 ? f16_bits_to_float(b) : bf16_bits_to_float(b);
}
template <int DT>
__device__ __forceinline__ void rot_store8(void* p, int64_t i, const float v[8]) {
  if constexpr (DT == TTKV_DTYPE_F32) {
    store_act4(p, DT, i, float4v{v[0], v[1], v[2], v[3]}, true);
    store_act4(p, DT, i + 4, float4v{v[4], v[5], v[6], v[7]}, true);
  } else {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float lo = v[2 * k], hi = v[2 * k + 1];
      if constexpr (DT == TTKV_DTYPE_F16)
        w[k] = __builtin_bit_cast(uint32_t, half2v{(_Float16)lo, (_Float16)hi});
      else
        w[k] = (uint32_t)float_to_bf16_bits(lo) | ((uint32_t)float_to_bf16_bits(hi) << 16);
    }
    *gblw((u32x4*)((uint16_t*)p + i)) = w;
  }
}

// One wave per token. Lane j first looks up frequency j's cosine and sine (one load each, whatever
// the axes) and leaves them in LDS; then the lanes take (head, 8 frequencies) pairs of 16-byte pieces,
// four heads' loads in flight at a time, the first four asked for before the lookup. Bound by memory:
// every query and key byte read and written once. 8,192 tokens of 40 heads in bf16, 171 MB: 36.9 us,
// 4.6 TB/s (a copy reaches 4.8; loads that stay in the cache 41.3, the kernel below, a pair per thread,
// 90).
constexpr int kRotHalf = 128;  // frequencies the LDS holds
constexpr int kRotBatch = 4;
template <int DT>
__global__ __launch_bounds__(64) void rotary_rows_kernel(RotArgs a) {
  __shared__ float cs[2][kRotHalf];
  const int64_t tok = blockIdx.x;
  const int lane = threadIdx.x;
  const int nch = a.half >> 3, slots = 64 / nch, heads = a.HQ + a.H;
  const int slot = lane / nch, j0 = (lane - slot * nch) * 8;
  const bool on = slot < slots;
  auto place = [&](int head, bool out, int64_t& at) -> const void* {
    const bool is_q = head < a.HQ;
    const int64_t stride = out ? (is_q ? a.qo_stride : a.ko_stride)
                               : (is_q ? a.q_stride : a.k_stride);
    at = tok * stride + (int64_t)(is_q ? head : head - a.HQ) * a.d;
    return out ? (is_q ? a.qo : a.ko) : (is_q ? a.q : a.k);
  };
  Rot8<DT> x[kRotBatch], y[kRotBatch];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int b = 0; b < kRotBatch; ++b) {
      const int head = h0 + b * slots + slot;
      if (on && head < heads) {
        int64_t at;
        const void* src = place(head, false, at);
        x[b] = rot_load8<DT>(src, at + j0);
        y[b] = rot_load8<DT>(src, at + j0 + a.half);
      }
    }
  };
  fetch(0);
  int64_t p[kRotAxes];
  const bool ok = rot_positions(a, tok, p);
  for (int j = lane; j < a.half; j += 64) {
    const int ax = rot_axis(a, j);
    int64_t q = p[0];
#pragma unroll
    for (int i = 1; i < kRotAxes; ++i) q = ax == i ? p[i] : q;
    const float* row = a.cs + q * (2 * a.half) + j;
    const float c = *gbl(row), s = *gbl(row + a.half);
    cs[0][j] = ok ? c : NAN;
    cs[1][j] = ok ? s : NAN;
  }
  __syncthreads();
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = cs[0][j0 + i];
    s[i] = cs[1][j0 + i];
  }
  for (int h0 = 0; h0 < heads; h0 += kRotBatch * slots) {
#pragma unroll
    for (int b = 0; b < kRotBatch; ++b) {
      const int head = h0 + b * slots + slot;
      if (on && head < heads) {
        int64_t at;
        void* dst = const_cast<void*>(place(head, true, at));
        float u[8], v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xi = rot_get<DT>(x[b], i), yi = rot_get<DT>(y[b], i);
          u[i] = xi * c[i] - yi * s[i];
          v[i] = yi * c[i] + xi * s[i];
        }
        rot_store8<DT>(dst, at + j0, u);
        rot_store8<DT>(dst, at + j0 + a.half, v);
      }
    }
    fetch(h0 + kRotBatch * slots);
  }
  const int rest = (a.d - 2 * a.half) >> 3;  // pieces that are copied
  for (int i = lane; i < heads * rest; i += 64) {
    const int head = i / rest, x0 = 2 * a.half + (i - head * rest) * 8;
    int64_t from, to;
    const void* src = place(head, false, from);
    void* dst = const_cast<void*>(place(head, true, to));
    const Rot8<DT> z = rot_load8<DT>(src, from + x0);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = ok ? rot_get<DT>(z, k) : NAN;
    rot_store8<DT>(dst, to + x0, v);
  }
}

// Rows whose pieces of 8 are not 16-byte aligned, or longer than the wave kernel's table: one pair
// per thread. 8,192 tokens of 40 heads in bf16 90 us, where aligned rows on the same card take 39.
__global__ __launch_bounds__(256) void rotary_axes_kernel(RotArgs a) {
  const int64_t tok = blockIdx.x;
  int64_t p[kRotAxes];
  const bool ok = rot_positions(a, tok, p);
  const int per = a.half + (a.d - 2 * a.half);  // pairs, then the dims that are copied
  for (int i = threadIdx.x; i < (a.HQ + a.H) * per; i += 256) {
    const int head = i / per, j = i % per;
    const bool is_q = head < a.HQ;
    const void* src = is_q ? a.q : a.k;
    void* dst = is_q ? a.qo : a.ko;
    const int64_t hd = (int64_t)(is_q ? head : head - a.HQ) * a.d;
    const int64_t from = tok * (is_q ? a.q_stride : a.k_stride) + hd;
    const int64_t to = tok * (is_q ? a.qo_stride : a.ko_stride) + hd;
    if (j >= a.half) {
      const int x = j + a.half;
      store_act(dst, a.dtype, to + x, ok ? load_act(src, a.dtype, from + x) : NAN);
      continue;
    }
    const int64_t row = p[rot_axis(a, j)] * (2 * a.half);
    const float c = ok ? a.cs[row + j] : NAN, s = a.cs[row + j + a.half];
    const float x = load_act(src, a.dtype, from + j), y = load_act(src, a.dtype, from + j + a.half);
    store_act(dst, a.dtype, to + j, x * c - y * s);
    store_act(dst, a.dtype, to + j + a.half, y * c + x * s);
  }
}

// Whether rows of `a` and of `b` share bytes: n rows each, of wa and wb bytes at strides sa and sb. Rows
// of unlike strides are only looked at where they begin.
static bool rot_rows_meet(const void* a, int64_t sa, int64_t wa, const void* b, int64_t sb, int64_t wb,
                          int64_t n) {
  if (!wa || !wb || !a || !b) return false;
  const int64_t off = (int64_t)((uintptr_t)b - (uintptr_t)a);
  auto meet = [&](int64_t o) { return o < wa && -o < wb; };
  if (n == 1 || sa != sb || sa <= 0) return meet(off);
  const int64_t k0 = -off / sa;  // row i + k of b lies nearest to row i of a
  for (int64_t k = k0 - 1; k <= k0 + 1; ++k)
    if (k > -n && k < n && meet(off + k * sa)) return true;
  return false;
}

int rotary_axes(const void* q, const void* k, void* qo, void* ko, int dtype, int N, int HQ, int H,
                int d, int64_t q_stride, int64_t k_stride, int64_t qo_stride, int64_t ko_stride,
                const int64_t* pos, int64_t pos_stride, int axes, const int32_t* sections,
                int interleaved, const float* cs, int64_t max_pos, int rot, int32_t* err,
                hipStream_t st) {
  if (dtype != TTKV_DTYPE_F32 && dtype != TTKV_DTYPE_F16 && dtype != TTKV_DTYPE_BF16)
    return host_fail(TTKV_E_INVALID, "dtype must be fp32, fp16 or bf16");
  if (N < 0 || HQ < 0 || H < 0 || d <= 0) return host_fail(TTKV_E_INVALID, "negative count");
  if (rot <= 0 || rot % 2 || rot > d)
    return host_fail(TTKV_E_INVALID, "the rotary dims must be even and at most the head dim");
  if (axes < 1 || axes > kRotAxes) return host_fail(TTKV_E_INVALID, "one to four axes");
  if (!sections) return host_fail(TTKV_E_INVALID, "null sections");
  int sum = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0) return host_fail(TTKV_E_INVALID, "negative section");
    sum += sections[i];
    if (interleaved && i && sections[i] && i + axes * (sections[i] - 1) >= rot / 2)
      return host_fail(TTKV_E_INVALID, "an interleaved section runs past the frequencies");
  }
  if (sum != rot / 2)
    return host_fail(TTKV_E_INVALID, "the sections must add up to half the rotary dims");
  if (max_pos <= 0) return host_fail(TTKV_E_INVALID, "empty cos_sin_cache");
  if (N == 0 || HQ + H == 0) return TTKV_OK;
  if ((HQ && (!q || !qo)) || (H && (!k || !ko)) || !pos || !cs || !err)
    return host_fail(TTKV_E_INVALID, "null pointer argument");
  // a row is written while others are still to be read: an output is its input as it stands, or apart
  const int64_t eb = dtype == TTKV_DTYPE_F32 ? 4 : 2, qw = (int64_t)HQ * d * eb, kw = (int64_t)H * d * eb;
  const int64_t qs = q_stride * eb, ks = k_stride * eb, qos = qo_stride * eb, kos = ko_stride * eb;
  if ((!(qo == q && (qos == qs || N == 1)) && rot_rows_meet(qo, qos, qw, q, qs, qw, N)) ||
      (!(ko == k && (kos == ks || N == 1)) && rot_rows_meet(ko, kos, kw, k, ks, kw, N)))
    return host_fail(TTKV_E_INVALID, "an output overlaps its input without being it");
  if (rot_rows_meet(qo, qos, qw, k, ks, kw, N) || rot_rows_meet(ko, kos, kw, q, qs, qw, N) ||
      rot_rows_meet(qo, qos, qw, ko, kos, kw, N))
    return host_fail(TTKV_E_INVALID, "one of query and key overlaps the other's output");
  RotArgs a{q,        k,        qo,         ko,   dtype,      HQ,   H,           d, rot / 2, N,
            q_stride, k_stride, qo_stride, ko_stride, pos, pos_stride, axes, interleaved != 0};
  for (int i = 0; i < axes; ++i) a.sec[i] = sections[i];
  a.cs = cs;
  a.max_pos = max_pos;
  a.err = err;
  bool rows = rot % 16 == 0 && d % 8 == 0 && rot / 2 <= kRotHalf;
  for (const void* p : {q, k, (const void*)qo, (const void*)ko}) rows &= (uintptr_t)p % 16 == 0;
  for (int64_t s : {q_stride, k_stride, qo_stride, ko_stride}) rows &= s * eb % 16 == 0;
  if (!rows)
    hipLaunchKernelGGL(rotary_axes_kernel, dim3(N), dim3(256), 0, st, a);
  else if (dtype == TTKV_DTYPE_F32)
    hipLaunchKernelGGL(rotary_rows_kernel<TTKV_DTYPE_F32>, dim3(N), dim3(64), 0, st, a);
  else if (dtype == TTKV_DTYPE_F16)
    hipLaunchKernelGGL(rotary_rows_kernel<TTKV_DTYPE_F16>, dim3(N), dim3(64), 0, st, a);
  else
    hipLaunchKernelGGL(rotary_rows_kernel<TTKV_DTYPE_BF16>, dim3(N), dim3(64), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("rotary launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

}  // namespace ttkv
