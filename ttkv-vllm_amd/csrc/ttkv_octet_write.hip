// Write of new keys and values into the 8-bit cache (format: ttkv_octet.h), the keys rotated on the way
// where the call has positions, its queries with them; and the rotation by itself. gfx950 / CDNA4.
//
// A workgroup of 256 threads takes the keys and values of 1024 / d tokens of one head, 8 dims a thread:
// a group of 32 dims is 4 neighbouring lanes. Tokens of one workgroup that follow each other in a tile
// write whole 128-byte lines of its record. Rotated keys go from the turn into the quantisation in 32 bits,
// and the queries' workgroups run beside the others in the same launch: a decode step needs one call for both.
//
// Kernels in graph replays: 8 tokens of 8 KV and 32 query heads, rotated, 3.5 us (a launch that does nothing
// 2.0); 2,048 tokens of 8 heads that come rotated, stored values returned, 21 MB, 5.2 us, one chain of slot, row
// and store over a full chip; 3,321 tokens of 4 heads of 256 dims and 16 query heads, rotated, 75 MB, 18.5 us,
// 4.1 TB/s with vector issue at 67 %. The kernel without a rotation is one of its own: it has 20 registers where
// the queries' code takes 84 (2,048 tokens 6.7 us with it).
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_octet.h"
#include "ttkv_turn.h"

namespace ttkv {

struct OctWriteArgs {
  const void* k;
  const void* v;
  int k_dtype, v_dtype;
  int64_t k_row_stride, v_row_stride;
  const int64_t* slots;
  int num_tokens, H;
  uint8_t* page;
  int64_t n_slots, slot_stride;
  uint16_t* k_out;
  uint16_t* v_out;
  int32_t* err;
  int write_blocks;  // workgroups before those of the queries
  TurnArgs turn;     // half == 0: keys come rotated
};

// The lane's value by xor 1 (STEP 0) or 2 (STEP 1) within 4 lanes.
template <int STEP>
__device__ __forceinline__ float quad_xor(float v) {
  const int w = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, w, STEP ? 0x4E : 0xB1, 0xF, 0xF, false));
}

// DT: the type of keys and values, or -1 where they differ (then by the arguments).
template <int D, int DT, bool TURN>
__global__ __launch_bounds__(256) void octet_write_kernel(OctWriteArgs a) {
  using F = Oct<D>;
  constexpr int kTokens = 1024 / D, kLanes = D / 8;
  __shared__ __align__(16) float2v cs[TURN ? kTurnHalf : 1];
  const int tid = threadIdx.x;
  if (TURN && (int)blockIdx.x >= a.write_blocks) {
    turn_token<false>(a.turn, (int)blockIdx.x - a.write_blocks, tid, 256, cs);
    return;
  }
  const int row = tid / kLanes, i = tid % kLanes, t = row % kTokens;  // dims 8 i .. 8 i + 7
  const bool val = row >= kTokens;
  const int h = (int)(blockIdx.x % (unsigned)a.H);
  const int64_t tok0 = (int64_t)(blockIdx.x / (unsigned)a.H) * kTokens, tok = tok0 + t;
  const bool on = tok < a.num_tokens;
  const void* src = val ? a.v : a.k;
  const int dt = DT >= 0 ? DT : val ? a.v_dtype : a.k_dtype;
  const int64_t stride = val ? a.v_row_stride : a.k_row_stride, at = tok * stride + (int64_t)h * D;
  const bool vec = act_rows_aligned(src, dt, stride);
  const int half = TURN ? a.turn.half : 0;
  // a lane's dims and, in a piece of 8 where the halves are made of such, the others of their pairs: a second
  // load, asked for with the first (through LDS and a token's table at a time 8 x 1 tokens took 6.2 us, 3.5 so)
  const bool whole = a.turn.adjacent || half % 8 == 0, mated = !val && !a.turn.adjacent && whole && 8 * i < 2 * half;
  const int mate = 8 * i < half ? 8 * i + half : 8 * i - half;
  float x[8] = {}, y[8] = {};
  if (on) {
    load_act_n<8>(src, dt, at + 8 * i, vec, x);
    if (mated) load_act_n<8>(src, dt, at + mate, vec, y);
  }
  const int64_t slot = on ? *gbl(a.slots + tok) : -1;  // negative: a padded token
  if (slot >= a.n_slots && !val && i == 0) atomicOr(a.err, TTKV_ERR_BAD_SLOT);
  const bool keep = slot >= 0 && slot < a.n_slots;
  if constexpr (TURN) {
    for (int e = tid; e < kTokens * half; e += 256) {  // (kTokens * half <= 512)
      const int n = e / half, j = e - n * half;
      if (tok0 + n >= a.num_tokens) break;
      const int64_t p = *gbl(a.turn.pos + tok0 + n);
      cs[e] = turn_at(a.turn.turns, j, p, a.turn.amplitude);
      if (j == 0 && h == 0 && !turn_place(p)) atomicOr(a.err, TTKV_ERR_BAD_POSITION);
    }
    __syncthreads();
    if (!val && keep) {
      const float2v* w = cs + t * half;
      const bool refused = w[0][0] != w[0][0];
      if (a.turn.adjacent) {
#pragma unroll
        for (int j = 0; j < 8; j += 2)
          if (8 * i + j < 2 * half) {
            const float2v f = w[4 * i + j / 2];
            const float u = x[j] * f[0] - x[j + 1] * f[1], v = x[j + 1] * f[0] + x[j] * f[1];
            x[j] = u;
            x[j + 1] = v;
          }
      } else if (whole) {
        if (mated) {
          const bool first = 8 * i < half;
          const int j0 = first ? 8 * i : 8 * i - half;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float2v f = w[j0 + j];
            x[j] = first ? x[j] * f[0] - y[j] * f[1] : x[j] * f[0] + y[j] * f[1];
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int e = 8 * i + j;
          if (e < 2 * half) {
            const bool first = e < half;
            const float2v f = w[first ? e : e - half];
            const float m = load_act(src, dt, at + (first ? e + half : e - half));
            x[j] = first ? x[j] * f[0] - m * f[1] : x[j] * f[0] + m * f[1];
          }
        }
      }
      if (refused)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = NAN;
    }
  }
  if (!keep) return;
  float odd = 0.f, top = 0.f;  // odd: NaN where a value is not finite
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    odd = fmaf(x[j], 0.f, odd);
    x[j] = fminf(fmaxf(x[j], -kOctMax), kOctMax);
    top = fmaxf(top, fabsf(x[j]));
  }
  odd += quad_xor<0>(odd);
  odd += quad_xor<1>(odd);
  top = fmaxf(top, quad_xor<0>(top));
  top = fmaxf(top, quad_xor<1>(top));
  const bool bad = odd != odd;
  // 448 = 1.75 * 2^8: the exponent less 8, and one more where the mantissa is above 1.75
  const uint32_t e = ((__builtin_bit_cast(uint32_t, top) + 0x1fffffu) >> 23) - 8;
  const uint32_t byte = bad ? kOctNanByte : max((int)e, kOctMinByte);
  const float by = oct_power(254 - byte);
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * by, x[4 * j + 1] * by, 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * by, x[4 * j + 3] * by, c, true);
    w[j] = bad ? kOctNanCode * 0x01010101u : (uint32_t)c;
  }
  uint16_t* outp = val ? a.v_out : a.k_out;
  if (outp) {
    const float p = oct_power(byte);
    const bf16x2 o[4] = {oct_pair<false>(w[0], p), oct_pair<true>(w[0], p), oct_pair<false>(w[1], p),
                         oct_pair<true>(w[1], p)};
    const u32x4 all = {__builtin_bit_cast(uint32_t, o[0]), __builtin_bit_cast(uint32_t, o[1]),
                       __builtin_bit_cast(uint32_t, o[2]), __builtin_bit_cast(uint32_t, o[3])};
    turn_store16(outp + (tok * a.H + h) * D + 8 * i, all);  // (2,048 tokens of 8 heads 5.8 us with stores that stay, 5.2)
  }
  uint8_t* rec = a.page + (slot >> 4) * (kOctTile * a.slot_stride) + (int64_t)h * F::kRecord;
  const int u = (int)(slot & 15), g = i >> 2;
  if (!val) {
    *gblw((u32x2v*)(rec + F::key(u, 8 * i))) = u32x2v{w[0], w[1]};
    if ((i & 3) == 0) *gblw(rec + F::key_power(u, g)) = (uint8_t)byte;
  } else {
    if constexpr (F::kDims >= 8) {
      *gblw((u32x2v*)(rec + F::value(u, 8 * i))) = u32x2v{w[0], w[1]};
    } else {
      *gblw((uint32_t*)(rec + F::value(u, 8 * i))) = w[0];
      *gblw((uint32_t*)(rec + F::value(u, 8 * i + 4))) = w[1];
    }
    if ((i & 3) == 0) *gblw(rec + F::value_power(u, g)) = (uint8_t)byte;
  }
}

// A workgroup per token.
template <bool STREAM>
__global__ __launch_bounds__(256) void rotary_scaled_kernel(TurnArgs a) {
  __shared__ __align__(16) float2v cs[kTurnHalf];
  turn_token<STREAM>(a, blockIdx.x, threadIdx.x, 256, cs);
}

// Rows that are read and written past this go by loads that do not stay in the caches (bf16, 40 heads of
// 128: 8,192 tokens, 168 MB, 36.0 us so and 37.5 with loads that stay; 4,096 tokens, 84 MB, 21.3 and 17.9).
constexpr int64_t kTurnStream = 128 << 20;

// The rows from token t on.
static TurnArgs turn_from(TurnArgs a, int64_t t) {
  const int64_t eb = a.dtype == TTKV_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < 2; ++i)
    if (a.heads[i]) {
      a.x[i] = (const char*)a.x[i] + t * a.x_stride[i] * eb;
      a.y[i] = (char*)a.y[i] + t * a.y_stride[i] * eb;
    }
  a.pos += t;
  return a;
}

// Whether rows go in pieces of 8 elements: aligned, and pairs that lie in one or two of them.
static bool turn_pieces_apply(const TurnArgs& a) {
  const int64_t eb = a.dtype == TTKV_DTYPE_F32 ? 4 : 2;
  const int unit = a.adjacent ? 4 : 8;
  bool pieces = a.d % (2 * unit) == 0 && a.half % unit == 0 && a.d / (2 * unit) <= 256;
  for (int i = 0; i < 2; ++i)
    if (a.heads[i])
      pieces &= ((uintptr_t)a.x[i] | (uintptr_t)a.y[i]) % 16 == 0 && a.x_stride[i] * eb % 16 == 0 &&
                a.y_stride[i] * eb % 16 == 0;
  return pieces;
}

static bool act_dtype(int dt) {
  return dt == TTKV_DTYPE_F32 || dt == TTKV_DTYPE_F16 || dt == TTKV_DTYPE_BF16;
}

// The rotation's own arguments; `limit`: dims of a row.
static int turn_check(const int64_t* pos, const double* turns, int rot, int limit) {
  if (rot <= 0 || rot % 2 || rot > limit)
    return host_fail(TTKV_E_INVALID, "the rotary dims must be even and at most the head dim");
  if (rot / 2 > kTurnHalf) return host_fail(TTKV_E_UNSUPPORTED, "more than 1024 rotary dims");
  if (!pos || !turns) return host_fail(TTKV_E_INVALID, "null positions or turns");
  if ((uintptr_t)turns % 8) return host_fail(TTKV_E_INVALID, "turns must be 8-byte aligned");
  return TTKV_OK;
}

// A set's output may be its input, at its stride, or lie apart from it.
static bool turn_clash(const void* x, int64_t xs, const void* y, int64_t ys, int64_t width, int64_t eb, int64_t n) {
  return !(x == y && (xs == ys || n == 1)) && rows_meet(y, ys * eb, width, x, xs * eb, width, n);
}

int rotary_scaled(const void* q, const void* k, void* qo, void* ko, int dtype, int N, int HQ, int H, int d,
                  int64_t q_stride, int64_t k_stride, int64_t qo_stride, int64_t ko_stride, const int64_t* pos,
                  const double* turns, int rot, float amplitude, int adjacent, int32_t* err, hipStream_t st) {
  if (!act_dtype(dtype)) return host_fail(TTKV_E_INVALID, "dtype must be fp32, fp16 or bf16");
  if (N < 0 || HQ < 0 || H < 0 || d <= 0) return host_fail(TTKV_E_INVALID, "negative count");
  if (N == 0 || HQ + H == 0) return TTKV_OK;
  if (int rc = turn_check(pos, turns, rot, d)) return rc;
  if ((HQ && (!q || !qo)) || (H && (!k || !ko)) || !err) return host_fail(TTKV_E_INVALID, "null pointer argument");
  const int64_t eb = dtype == TTKV_DTYPE_F32 ? 4 : 2, qw = HQ ? (int64_t)HQ * d * eb : 0,
                kw = H ? (int64_t)H * d * eb : 0;
  if (turn_clash(q, q_stride, qo, qo_stride, qw, eb, N) || turn_clash(k, k_stride, ko, ko_stride, kw, eb, N))
    return host_fail(TTKV_E_INVALID, "an output overlaps its input without being it");
  if (rows_meet(qo, qo_stride * eb, qw, k, k_stride * eb, kw, N) ||
      rows_meet(ko, ko_stride * eb, kw, q, q_stride * eb, qw, N) ||
      rows_meet(qo, qo_stride * eb, qw, ko, ko_stride * eb, kw, N))
    return host_fail(TTKV_E_INVALID, "one of query and key overlaps the other's output");
  if (rows_fold(qo_stride * eb, qw, N) || rows_fold(ko_stride * eb, kw, N))
    return host_fail(TTKV_E_INVALID, "rows of an output overlap one another");
  TurnArgs a{{q, k}, {qo, ko}, {HQ, H}, {q_stride, k_stride}, {qo_stride, ko_stride}, dtype, d, rot / 2, adjacent != 0,
             0,      pos,      turns,   amplitude,            err};
  a.pieces = turn_pieces_apply(a);
  auto kernel = 2 * (qw + kw) * N > kTurnStream ? rotary_scaled_kernel<true> : rotary_scaled_kernel<false>;
  for (int64_t t = 0; t < N; t += kMaxGrid) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(N - t, kMaxGrid)), dim3(256), 0, st, turn_from(a, t));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return host_fail(TTKV_E_LAUNCH, std::string("scaled rotary launch: ") + hipGetErrorString(e));
  }
  return TTKV_OK;
}

int octet_check_page(int H, int d, const uint8_t* page, int64_t n_slots, int64_t slot_stride) {
  if (d != 64 && d != 128 && d != 256) return host_fail(TTKV_E_UNSUPPORTED, "head dim must be 64, 128 or 256");
  if (H <= 0) return host_fail(TTKV_E_INVALID, "H must be positive");
  if (!page) return host_fail(TTKV_E_INVALID, "null page");
  if (slot_stride < ((int64_t)33 * d * H + 15) / 16)
    return host_fail(TTKV_E_INVALID, "slot stride is smaller than the slot (33 d H / 16 bytes)");
  if ((uintptr_t)page % 16) return host_fail(TTKV_E_INVALID, "the page must be 16-byte aligned");
  if (n_slots <= 0 || n_slots % kOctTile)
    return host_fail(TTKV_E_INVALID, "the page must hold a positive multiple of 16 slots");
  return TTKV_OK;
}

template <int D, bool TURN>
static void oct_write_launch(const OctWriteArgs& a, unsigned grid, int dt, hipStream_t st) {
  auto kernel = dt == TTKV_DTYPE_F32    ? octet_write_kernel<D, TTKV_DTYPE_F32, TURN>
                : dt == TTKV_DTYPE_F16  ? octet_write_kernel<D, TTKV_DTYPE_F16, TURN>
                : dt == TTKV_DTYPE_BF16 ? octet_write_kernel<D, TTKV_DTYPE_BF16, TURN>
                                        : octet_write_kernel<D, -1, TURN>;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), 0, st, a);
}
template <int D>
static void oct_write_launch(const OctWriteArgs& a, unsigned grid, int dt, hipStream_t st) {
  if (a.turn.half) oct_write_launch<D, true>(a, grid, dt, st);
  else oct_write_launch<D, false>(a, grid, dt, st);
}

int octet_write_paged(int H, int d, const void* key, int k_dtype, int64_t k_row_stride, const void* val,
                      int v_dtype, int64_t v_row_stride, const int64_t* slots, int num_tokens, uint8_t* page,
                      int64_t n_slots, int64_t slot_stride, void* k_out, void* v_out, const int64_t* pos,
                      const double* turns, int rot, float amplitude, int adjacent, const void* q, int q_dtype,
                      int64_t q_stride, int HQ, void* qo, int64_t qo_stride, int32_t* err, hipStream_t st) {
  if (int rc = octet_check_page(H, d, page, n_slots, slot_stride)) return rc;
  if (!act_dtype(k_dtype) || !act_dtype(v_dtype))
    return host_fail(TTKV_E_INVALID, "key / value dtype must be fp32, fp16 or bf16");
  if (num_tokens < 0 || HQ < 0) return host_fail(TTKV_E_INVALID, "negative count");
  if (rot < 0) return host_fail(TTKV_E_INVALID, "negative rotary dims");
  if (HQ && !rot) return host_fail(TTKV_E_INVALID, "queries are taken to be rotated: they need rotary dims");
  if (num_tokens == 0) return TTKV_OK;
  if (!key || !val || !slots || !err) return host_fail(TTKV_E_INVALID, "null pointer argument");
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
    return host_fail(TTKV_E_INVALID, "key_out / value_out must be 16-byte aligned");
  if (rot)
    if (int rc = turn_check(pos, turns, rot, d)) return rc;
  // Rows are read while others are written: key_out may be the key as it stands, value_out the value, and
  // nothing else overlaps.
  const int64_t kb = k_dtype == TTKV_DTYPE_F32 ? 4 : 2, vb = v_dtype == TTKV_DTYPE_F32 ? 4 : 2, row = (int64_t)H * d;
  auto meets = [&](const void* y, int64_t ys, int64_t width, const void* x, int64_t xs, int64_t xw) {
    return rows_meet(y, ys, width, x, xs, xw, num_tokens);
  };
  auto same = [&](const void* y, const void* x, int64_t xs, int64_t xb) {
    return y == x && xb == 2 && (xs == row || num_tokens == 1);
  };
  if ((k_out && !same(k_out, key, k_row_stride, kb) && meets(k_out, 2 * row, 2 * row, key, k_row_stride * kb, row * kb)) ||
      (v_out && !same(v_out, val, v_row_stride, vb) && meets(v_out, 2 * row, 2 * row, val, v_row_stride * vb, row * vb)) ||
      meets(k_out, 2 * row, 2 * row, val, v_row_stride * vb, row * vb) ||
      meets(v_out, 2 * row, 2 * row, key, k_row_stride * kb, row * kb) ||
      meets(k_out, 2 * row, 2 * row, v_out, 2 * row, 2 * row))
    return host_fail(TTKV_E_INVALID, "key_out or value_out overlaps the keys, the values or the other");
  if (HQ) {
    if (!act_dtype(q_dtype)) return host_fail(TTKV_E_INVALID, "query dtype must be fp32, fp16 or bf16");
    if (!q || !qo) return host_fail(TTKV_E_INVALID, "null pointer argument");
    const int64_t eb = q_dtype == TTKV_DTYPE_F32 ? 4 : 2, qw = (int64_t)HQ * d * eb;
    if (turn_clash(q, q_stride, qo, qo_stride, qw, eb, num_tokens))
      return host_fail(TTKV_E_INVALID, "query_out overlaps the query without being it");
    if (meets(qo, qo_stride * eb, qw, key, k_row_stride * kb, row * kb) ||
        meets(qo, qo_stride * eb, qw, val, v_row_stride * vb, row * vb) ||
        meets(qo, qo_stride * eb, qw, k_out, 2 * row, 2 * row) || meets(qo, qo_stride * eb, qw, v_out, 2 * row, 2 * row) ||
        meets(q, q_stride * eb, qw, k_out, 2 * row, 2 * row) || meets(q, q_stride * eb, qw, v_out, 2 * row, 2 * row))
      return host_fail(TTKV_E_INVALID, "query_out overlaps the keys or values, or the query their outputs");
    if (rows_fold(qo_stride * eb, qw, num_tokens))
      return host_fail(TTKV_E_INVALID, "rows of query_out overlap one another");
  }
  TurnArgs turn{{q, nullptr},  {qo, nullptr}, {HQ, 0}, {q_stride, 0}, {qo_stride, 0}, q_dtype, d, rot / 2,
                adjacent != 0, 0,             pos,     turns,         amplitude,      err};
  turn.pieces = HQ && turn_pieces_apply(turn);
  const int dt = k_dtype == v_dtype ? k_dtype : -1;
  // of `tokens` tokens and a head each, and one per token for the queries
  const int64_t tokens = 1024 / d, most = std::max<int64_t>(1, kMaxGrid / (H + tokens)) * tokens;
  for (int64_t t = 0; t < num_tokens; t += most) {
    const int n = (int)std::min(num_tokens - t, most);
    const int64_t blocks = (n + tokens - 1) / tokens * H;
    OctWriteArgs a{(const char*)key + t * k_row_stride * kb,
                   (const char*)val + t * v_row_stride * vb,
                   k_dtype,
                   v_dtype,
                   k_row_stride,
                   v_row_stride,
                   slots + t,
                   n,
                   H,
                   page,
                   n_slots,
                   slot_stride,
                   k_out ? (uint16_t*)k_out + t * row : nullptr,
                   v_out ? (uint16_t*)v_out + t * row : nullptr,
                   err,
                   (int)blocks,
                   turn_from(turn, t)};
    const unsigned grid = (unsigned)(blocks + (HQ ? n : 0));
    if (d == 64) oct_write_launch<64>(a, grid, dt, st);
    else if (d == 128) oct_write_launch<128>(a, grid, dt, st);
    else oct_write_launch<256>(a, grid, dt, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return host_fail(TTKV_E_LAUNCH, std::string("octet write launch: ") + hipGetErrorString(e));
  }
  return TTKV_OK;
}

}  // namespace ttkv
