// Attention of new tokens over the 8-bit cache (format: ttkv_octet.h): one query per request, or a few
// drafts. gfx950 / CDNA4.
//
// The rows of a (request, KV head) are its (query, query head) pairs, row = j G + p. Work item = (request,
// block of RG groups of 16 rows, chunk of the request's 32-token steps, KV head), one workgroup of W waves that
// take the chunk's steps in turn: W is 4 or 8 (od_waves), RG 1 or 2 (od_groups). The chunk length comes from a plan that every workgroup computes alike from the
// batch's lengths: the shortest that spreads the batch's steps over the resident workgroups, so a ragged
// batch fills the chip by its total work. Items of a (block, head) leave unnormalised partials in the
// workspace; the last to arrive joins them.
//
// One step of a wave, two tiles of 16 tokens:
//   S^T [token, row] = K Q^T on v_mfma_f32_16x16x32_bf16: a lane's d / 4 key code bytes of a tile are its A
//     operand of the d / 32 products (token lane % 16), made bf16 at their power of two by one instruction
//     per pair, exactly; the queries are the B operand, held in registers (fp16 ones as two bf16 parts,
//     exactly). Columns without a row are zero.
//   softmax in the result's own registers: lane column = row, 8 tokens of it. Weights are taken against
//     the maximum as it stands, which moves only when their sum is large, so most steps need no maximum
//     and no exchange between lanes; the sum stays per lane until the end. bf16 has fp32's range, so no
//     weight leaves it; three parts of a weight keep its 24 bits.
//   O^T [dim, row] += V^T P^T, a product per dim of a lane's d / 16 and weight part: the scores' layout is
//     the B operand's as it stands. A lane holds dims of four tokens per tile; their bf16 pairs of two dims
//     become pairs of two tokens by one byte permutation each. The result's column is the row again, so
//     the rescale is a lane's factor.
// A step is 66 d bytes. Bound by memory where calls are large: 8 x 14,402 tokens of 8 heads of 128, 243 MB,
// 46.1 us, of which a prologue takes 5 and the join 3: 6.4 TB/s between them (vector issue 40 %, matrix units
// 19 %); 61 requests of 70 to 2,900 37.3 us for 178 MB. Smaller calls are a chain of round trips: one key tile
// 5.3 us, a split and its join 2.3 to 4 more; 1 x 1,082 8.8 us.
#include <math.h>

#include <atomic>

#include "ttkv_host.h"
#include "ttkv_nibble.h"
#include "ttkv_octet.h"

namespace ttkv {

constexpr int kODMaxQ = 16;  // queries per request
constexpr int kODStep = 2 * kOctTile;  // tokens per wave step
constexpr int kODPlanLanes = 4;        // requests per lane in the plan: 256 per launch
constexpr int kODClasses = 8;          // of chunk lengths, for the items' order
constexpr int kODRows = 16;            // rows of a group: a matrix product's columns
constexpr float kODNone = -3.402823466e38f;  // the maximum before the first visible key
constexpr float kODMost = 0x1p10f;     // a lane's sum of eight weights before the maximum moves
// One query per request; several, whose rows are one block; or more blocks, whose bytes stay in the caches for
// each other (6 x 5 queries of four query heads over 4,000 keys, d = 256: 25.1 us with loads that do not stay,
// 23.3; where there is one block they cost: 30 x 3 over 200 to 4,000 30.1, 32.6). Blocks of two groups of rows
// take loads that do not stay however many there are (with such and with ones that stay, 60 x 8 queries of eight
// query heads over 1,500 keys: of 128 dims 76.4 us and 74.2, of 256 90.3 and 85.9, of 64 48.2 and 49.2; 40 x 16
// of four over 2,000 70.3 and 71.4).
enum { kODSingle = 0, kODOwn = 1, kODShared = 2 };
// What a chunk's join costs per row and dim against a step (1 x 14,000 tokens: 16.4 us with 6e-4, 14.1 so; 1 x
// 60,000 of one KV head of eight query heads 70 without it, 19.4 so).
constexpr float kODJoin = 9e-4f;
// bf16 parts of a weight: its 24 bits, as where values cancel an output shows what the weights are off by. Two, of
// 16 bits, take 1 to 4 % less (8 x 14,402 tokens 45.7 and 45.9 us, 61 of 70 to 2,900 37.0 and 37.3, 6 x 5 queries
// of 256 dims 26.3 and 27.3), 9 % where 64 rows share a KV head (60 x 8 over 1,500 keys 66.1 and 72.3); the pairs of figures elsewhere in this
// file compare variants of two parts.
constexpr int kODParts = 3;
constexpr float kLog2e = 1.4426950408889634f;

struct OctDecodeArgs {
  int H, G;
  float scale_log2;
  const uint16_t* q;
  int64_t q_row_stride;
  int num_tokens;
  const uint8_t* page;
  int64_t tile_stride;
  int num_blocks;
  int tpb;  // tiles per block
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* seq_lens;
  const int32_t* qsl;
  int num_reqs, max_q, max_seq;
  int window;  // 0: none
  const float* sinks;
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  float* lse;
  int* ws_cnt;
  int cnt_stride;    // between counters: cache lines of their own where there is room (atomics on one line wait
                     // for each other: 1 x 14,000 tokens 14.2 us side by side, 12.5 so)
  float* ws_o;       // [split items][part_rows][D]
  float* ws_ml;      // [split items][part_rows][2]
  uint32_t o_bytes;  // size of ws_o
  int part_rows;     // rows of an item's partials
  float by_H;            // 1 / H
  float by_target;       // 1 / the items that the plan aims at
  int resident;          // what the chip holds at once
  float join;            // what a chunk's join costs against a step
  int32_t* err;
};

struct OctPlan {
  int r, rb, c, h;   // batch row, row block, chunk, KV head
  int n, Q, q0;      // keys, queries and the first one's row
  int s0, steps;     // the request's steps: the first and how many
  int nch;           // the block's chunks
  int part, block;   // the block's first split item and its number, both before the head
  bool none;
};

// x / d for 0 <= x < 2^24 and by = 1 / d to an ulp.
__device__ __forceinline__ int od_div(int x, int d, float by) {
  int k = (int)((float)x * by);
  k -= k * d > x;
  return k + ((k + 1) * d <= x);
}

template <int W, int RB>  // waves of a workgroup, rows of a block
__device__ __forceinline__ OctPlan od_plan(const OctDecodeArgs& a) {
  const int lane = threadIdx.x & 63;
  int n[kODPlanLanes], q0[kODPlanLanes], Q[kODPlanLanes], s0[kODPlanLanes], st[kODPlanLanes], rb[kODPlanLanes];
  int total = 0, longest = 0, whole = 0;
  bool falls = false;  // a request's queries end before they begin: none are taken
#pragma unroll
  for (int i = 0; i < kODPlanLanes; ++i) {
    n[i] = q0[i] = Q[i] = 0;
    const int r = lane + 64 * i;
    if (64 * i >= a.num_reqs || r >= a.num_reqs) continue;
    n[i] = a.seq_lens[r];
    q0[i] = a.qsl[r];
    const int q1 = a.qsl[r + 1];
    falls |= q1 < q0[i];
    Q[i] = q1 < q0[i] ? -1 : (int)min((uint32_t)q1 - (uint32_t)q0[i], 0x7fffffffu);
  }
  if (blockIdx.x == 0 && threadIdx.x < 64 && falls) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
#pragma unroll
  for (int i = 0; i < kODPlanLanes; ++i) {
    s0[i] = st[i] = rb[i] = 0;
    if (64 * i >= a.num_reqs) continue;
    const int nn = min(max(n[i], 0), a.max_seq), qq = min(max(Q[i], 0), a.max_q), p0 = nn - Q[i];
    s0[i] = a.window && p0 >= a.window ? (p0 - a.window + 1) / kODStep : 0;
    st[i] = p0 >= 0 && qq > 0 ? (p0 + qq - 1) / kODStep + 1 - s0[i] : 0;
    rb[i] = (qq * a.G + RB - 1) / RB;
    total += st[i] * rb[i];
    longest = max(longest, st[i]);
    whole += rb[i];
  }
  // (a lane has less than 2^28 steps, and its sums below fp32's 2^24 are whole)
  float all = (float)wave_sum_i(total & 4095);
  if (__builtin_amdgcn_ballot_w64(total >> 12)) all += 4096.f * (float)wave_sum_i(total >> 12);
  whole = wave_sum_i(whole);
  // whole rounds of the workgroup's waves. (Never shorter than the batch's share: the grid and the workspace are
  // made for that; fp32 is off by less than the factor.)
  all *= (float)a.H * 1.000001f;
  int C = (max(1, (int)ceilf(all * a.by_target)) + W - 1) / W * W;
  // A step costs its chunk's wave about a, a chunk its join about b per row and dim: the two together are
  // least at sqrt(4 steps b / a) steps.
  C = max(C, (int)(sqrtf((float)wave_max_i(longest) * a.join) / W + 0.5f) * W);
  // Never more than steps / C rounded up; and two rounds of the waves longer rather than a chunk more, whose
  // hand-over costs as much (24 x 256 keys: 10.2 us with it, 7.0 so; 1 x 300 7.6, 6.8; 61 of 70 to 2,900 39.2, 36.6).
  float by_C;
  auto length = [&](int c) {
    C = c;
    by_C = __builtin_amdgcn_rcpf((float)c) * 0.9999995f;
  };
  auto chunks = [&](int steps) { return max(1, (int)((float)(steps + C - 1 - 2 * W) * by_C)); };
  length(C);
  // Longer chunks rather than a second round of workgroups, where the batch has not more blocks anyway (6 x 5
  // queries, d = 256: 45.2 us, 32.1 so). There are at most `whole` chunks more than the steps have lengths of C.
  if (whole * a.H <= a.resident && (float)(whole * a.H) + all * by_C * 1.000001f > (float)a.resident) {
    while (true) {
      int items = 0;
#pragma unroll
      for (int i = 0; i < kODPlanLanes; ++i)
        if (64 * i < a.num_reqs) items += rb[i] * chunks(st[i]);
      if (wave_sum_i(items) * a.H <= a.resident) break;
      length(C + max(1, C / (16 * W)) * W);
    }
  }
  OctPlan P{};
  P.none = true;
  const int it = blockIdx.x;
  // Long chunks first, so that a compute unit's workgroups are not all long (64 of 100 to 3,000 keys: 46.2 us in
  // the batch's order, 43.6 so): classes by the chunk's eighth of C, in the batch's order within each. Not where
  // chunks are short or requests many, whose scans cost more (200 of 50 to 600: 34.3, 40.5).
  const int classes = a.num_reqs > 64 || C <= 8 ? 1 : kODClasses;
  int nch[kODPlanLanes], cls[kODPlanLanes];
#pragma unroll
  for (int i = 0; i < kODPlanLanes; ++i) {
    nch[i] = cls[i] = 0;
    if (64 * i >= a.num_reqs) continue;
    nch[i] = chunks(st[i]);
    if (classes > 1) {
      const float eighths = (float)st[i] * __builtin_amdgcn_rcpf((float)nch[i]) * by_C * kODClasses;
      cls[i] = kODClasses - 1 - min(kODClasses - 1, (int)eighths);
    }
  }
  int carry = 0, ln = 0;
  for (int k = 0; k < classes && P.none; ++k) {
#pragma unroll
    for (int i = 0; i < kODPlanLanes; ++i) {
      if (64 * i >= a.num_reqs) break;
      const int items = cls[i] == k ? rb[i] * nch[i] * a.H : 0;
      if (!__builtin_amdgcn_ballot_w64(items > 0)) continue;
      const int incl = nib_scan(items), ex = carry + incl - items;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(ex <= it && it < ex + items);
      if (hit) {
        ln = __builtin_ctzll(hit);
        P.none = false;
        P.r = 64 * i + ln;
        P.n = __builtin_amdgcn_readlane(n[i], ln);
        P.Q = __builtin_amdgcn_readlane(Q[i], ln);
        P.q0 = __builtin_amdgcn_readlane(q0[i], ln);
        P.s0 = __builtin_amdgcn_readlane(s0[i], ln);
        P.steps = __builtin_amdgcn_readlane(st[i], ln);
        P.nch = __builtin_amdgcn_readlane(nch[i], ln);
        const int local = it - __builtin_amdgcn_readlane(ex, ln), blocks = __builtin_amdgcn_readlane(rb[i], ln);
        // Workgroups go to the eight XCDs in turn: the row blocks of a (chunk, KV head) lie eight items apart, so
        // that they share its bytes in one L2 (of up to eight such units the last ones lie closer).
        int unit = local;
        if (blocks > 1) {
          const int units = P.nch * a.H;
          const int group = od_div(local, 8 * blocks, __builtin_amdgcn_rcpf(8.f * (float)blocks));
          const int rest = local - group * 8 * blocks, wide = min(8, units - group * 8);
          P.rb = od_div(rest, wide, __builtin_amdgcn_rcpf((float)wide));
          unit = group * 8 + rest - P.rb * wide;
        }
        P.c = od_div(unit, a.H, a.by_H);
        P.h = unit - P.c * a.H;
        break;
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  // the blocks, and the split ones' items, of the requests before
  if (P.nch > 1) {
    int blocks = 0, parts = 0;
#pragma unroll
    for (int i = 0; i < kODPlanLanes; ++i)
      if (64 * i + lane < P.r) {
        blocks += rb[i];
        parts += nch[i] > 1 ? rb[i] * nch[i] : 0;
      }
    P.block = wave_sum_i(blocks) + P.rb;
    P.part = wave_sum_i(parts) + P.rb * P.nch;
  }
  return P;
}

// One step's bytes of a lane: per tile its token's key codes and exponents, and its dims' value codes and
// exponents of four tokens.
template <int D>
struct OctStep {
  u32x4 k[2][D / 64], v[2][D / 64];
  uint32_t kp[2], vp[2];
};

// STREAM: a load that does not stay in the caches.
template <bool STREAM, typename T>
__device__ __forceinline__ T od_load(const T* p) {
  return STREAM ? __builtin_nontemporal_load(gbl(p)) : *gbl(p);
}

// Four tokens' values of one dim, and of the next, from the tokens' pairs of those dims.
__device__ __forceinline__ uint32_t od_low(bf16x2 a, bf16x2 b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x05040100u);
}
__device__ __forceinline__ uint32_t od_high(bf16x2 a, bf16x2 b) {
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}

template <int D, int W, int QDT, int MODE, int RG>
__global__ __launch_bounds__(64 * W, W > 4 ? W / 4 : D == 256 ? 3 - RG : D == 128 ? 2 : 5 - RG) void octet_decode_kernel(OctDecodeArgs a) {
  using F = Oct<D>;
  constexpr int N = F::kDims, KS = D / 32, PIECES = D / 64, PARTS = QDT == TTKV_DTYPE_F16 ? 2 : 1;
  constexpr bool CHUNK = MODE != kODSingle;
  constexpr int kThreads = 64 * W, RB = kODRows * RG;
  constexpr int RS = D + 4;  // floats of a row in LDS: the rows' columns start in different banks
  extern __shared__ __align__(16) float red_all[];  // [waves][rows][RS]: the waves' results, then the join's
  float(*red_o)[RB][RS] = (float(*)[RB][RS])red_all;
  __shared__ float red_m[W][RB], red_l[W][RB];
  __shared__ int last_sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const OctPlan P = od_plan<W, RB>(a);
  if (P.none) return;
  const int h = P.h, G = a.G, HQ = a.H * a.G;
  const int n = min(max(P.n, 0), a.max_seq), Q = min(P.Q, a.max_q);
  const int p0 = n - P.Q;  // position of query 0
  const int row0 = P.rb * RB, nrow = min(RB, Q * G - row0);  // the block's rows
  const bool outside = P.q0 < 0 || (int64_t)P.q0 + Q > a.num_tokens;
  if (tid == 0 && h == 0 && P.c == 0 && P.rb == 0 &&
      (P.n < 0 || P.n > a.max_seq || P.Q > a.max_q || (n > 0 && p0 < 0) || outside))
    atomicOr(a.err, TTKV_ERR_SEQ_LEN);
  // row `r` of the block in the query and the output, and whether it has a place there
  auto row_at = [&](int r, int64_t stride) -> int64_t {
    const int row = row0 + r, j = CHUNK ? row / G : 0;
    return ((int64_t)P.q0 + j) * stride + (int64_t)(h * G + row - j * G) * D;
  };
  auto has = [&](int r) {
    const int64_t t = (int64_t)P.q0 + (CHUNK ? (row0 + r) / G : 0);
    return !outside || (t >= 0 && t < a.num_tokens);
  };
  // The end of a row: the sink joins its sum. `o` of dims d .. d + 3, not yet divided by l.
  auto finish = [&](int r, int d, float4v o, float m, float l) {
    if (!has(r)) return;
    const int row = row0 + r, j = CHUNK ? row / G : 0, hq = h * G + row - j * G;
    if (a.sinks) {
      const float s = a.sinks[hq] * kLog2e, mn = fmaxf(m, s), f = exp2f(m - mn);
      l = l * f + exp2f(s - mn);
      o *= f;
      m = mn;
    }
    // no weight: no key, or keys whose scores all lie below fp32, which leave nothing to go by
    const float by = l == 0.f ? (n > 0 ? NAN : 0.f) : 1.f / l;
    store_act4(a.out, a.out_dtype, row_at(r, a.out_row_stride) + d, o * by, true);
    if (a.lse && d == 0)
      a.lse[((int64_t)P.q0 + j) * HQ + hq] = l == 0.f ? (n > 0 ? NAN : -INFINITY) : (m + log2f(l)) * 0.6931471805599453f;
  };
  if (p0 < 0) {  // an empty request's rows are 0; fewer keys than queries are refused
    for (int i = tid; i < nrow * (D / 4); i += kThreads)
      finish(i / (D / 4), i % (D / 4) * 4, float4v{}, kODNone, n > 0 ? NAN : 0.f);
    return;
  }
  const int col = lane & 15, q4 = lane >> 4;

  // The queries, row 16 g + `col` of group g, as the B operand of the score products: dims q4 D / 4 + 8 s + (0..7)
  bf16x8 qf[RG][PARTS][KS];
  float m[RG], l[RG];
  int lim[RG], low[RG];  // last key the lane's row sees, and the one before its first
  float4v acc[RG][N];    // [g][e][i]: dim (4 q4 + i) N + e of the lane's row
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const int my = min(kODRows * g + col, nrow - 1);
    const bool on = kODRows * g + col < nrow && has(my);
    const uint16_t* src = a.q + row_at(my, a.q_row_stride) + q4 * (D / 4);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 raw = {};
      if (on) raw = *gbl((const u32x4*)(src + 8 * s));
      if constexpr (QDT == TTKV_DTYPE_BF16) {
        qf[g][0][s] = __builtin_bit_cast(bf16x8, raw);
      } else {
        const half8 x = __builtin_bit_cast(half8, raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // 11 bits are 8 and the 3 that they leave
          const __bf16 hi = (__bf16)(float)x[j];
          qf[g][0][s][j] = hi;
          qf[g][PARTS - 1][s][j] = (__bf16)((float)x[j] - (float)hi);
        }
      }
    }
    lim[g] = p0 + (CHUNK ? (row0 + my) / G : 0);
    low[g] = a.window ? lim[g] - a.window : -1;
    m[g] = kODNone;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) acc[g][e] = float4v{};
  }
  const int see_all = p0 + (CHUNK ? row0 / G : 0);  // no row of the block sees less than to here
  const int low_all = a.window ? p0 + (CHUNK ? (row0 + nrow - 1) / G : 0) - a.window : -1;  // and from behind here

  // the block's steps in equal parts, the first ones a step longer
  const int each = od_div(P.steps, P.nch, __builtin_amdgcn_rcpf((float)P.nch)), more = P.steps - each * P.nch;
  const int s0 = P.s0 + each * P.c + min(P.c, more);
  const int s1 = s0 + each + (P.c < more);
  const int first_tile = a.window ? max(p0 - a.window + 1, 0) / kOctTile : 0;
  bool bad = false;

  const uint8_t* base = a.page + (int64_t)h * F::kRecord;
  const int32_t* bt = a.bt + (int64_t)P.r * a.bt_row_stride;
  // tile ids of this wave's next 64 steps, one step per lane (-1: a block outside the cache)
  const float by_tpb = __builtin_amdgcn_rcpf((float)a.tpb);
  int tid0 = 0, tid1 = 0;
  auto fetch_ids = [&](int s) {
    const int mine = min(s + W * lane, s1 - 1);  // (past the chunk: its last step's again)
    // (no tile outside the keys that some row sees: a window's past blocks may be gone)
    const int t0 = max(2 * mine, first_tile), t1 = min(max(2 * mine + 1, first_tile), (n - 1) / kOctTile);
    const int b0 = od_div(t0, a.tpb, by_tpb), b1 = od_div(t1, a.tpb, by_tpb);
    const int i0 = bt[b0], i1 = bt[b1];
    tid0 = (uint32_t)i0 < (uint32_t)a.num_blocks ? i0 * a.tpb + t0 - b0 * a.tpb : -1;
    tid1 = (uint32_t)i1 < (uint32_t)a.num_blocks ? i1 * a.tpb + t1 - b1 * a.tpb : -1;
  };
  auto record = [&](int k, int t) {  // of the wave's k-th step since fetch_ids
    const int id = __builtin_amdgcn_readlane(t ? tid1 : tid0, k);
    bad |= id < 0;
    return base + (int64_t)max(id, 0) * a.tile_stride;
  };
  auto load_keys = [&](int k, OctStep<D>& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* rec = record(k, t);
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
        x.k[t][p] = od_load<MODE != kODShared>((const u32x4*)(rec + 1024 * p + 16 * lane));
      if constexpr (D == 256)
        x.kp[t] = od_load<MODE != kODShared>((const uint16_t*)(rec + F::kKp) + lane);
      else
        x.kp[t] = od_load<MODE != kODShared>(rec + F::kKp + (D == 64 ? (lane >> 5) * 16 + col : lane));
    }
  };
  auto load_values = [&](int k, OctStep<D>& x) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint8_t* rec = record(k, t);
#pragma unroll
      for (int p = 0; p < PIECES; ++p)
        x.v[t][p] = od_load<MODE != kODShared>((const u32x4*)(rec + F::kV + 1024 * p + 16 * lane));
      x.vp[t] = od_load<MODE != kODShared>((const uint32_t*)(rec + F::kVp + col * N / 32 * 16) + q4);
    }
  };
  auto load = [&](int k, OctStep<D>& x) {
    load_keys(k, x);
    load_values(k, x);
  };
  auto step = [&](int s, OctStep<D>& x, auto&& keys_done) {
    float4v sc[RG][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int g = 0; g < RG; ++g) sc[g][t] = float4v{};
      const float pw[2] = {oct_power(x.kp[t] & 0xffu), oct_power(x.kp[t] >> 8)};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const float p = pw[D == 256 ? ks / 4 : 0];
        bf16x8 kf;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint32_t c = x.k[t][ks / 2][ks % 2 * 2 + w];
          const bf16x2 lo = oct_pair<false>(c, p), hi = oct_pair<true>(c, p);
          kf[4 * w] = lo[0];
          kf[4 * w + 1] = lo[1];
          kf[4 * w + 2] = hi[0];
          kf[4 * w + 3] = hi[1];
        }
#pragma unroll
        for (int g = 0; g < RG; ++g)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            sc[g][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[g][part][ks], sc[g][t], 0, 0, 0);
      }
#pragma unroll
      for (int g = 0; g < RG; ++g) sc[g][t] *= a.scale_log2;
    }
    keys_done();
    const int tok = s * kODStep + 4 * q4;
    uint32_t note = 0;  // bit 4 t + i: the lane's dims of that token are NaN
    if ((s + 1) * kODStep - 1 > see_all || s * kODStep <= low_all) {
      // Some row does not see all of this step: no score outside its keys. A weight of 0 must not meet a
      // NaN: values that no row sees become 0, and with several queries a group that is NaN becomes 0
      // too and is noted for the rows that see it.
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = tok + 16 * t + i;
#pragma unroll
          for (int g = 0; g < RG; ++g)
            if (tk > lim[g] || tk <= low[g]) sc[g][t][i] = -INFINITY;
          bool drop = tk > lim[0] || tk <= low[0];
          if constexpr (CHUNK) {
            drop = tk >= n || (a.window && tk <= p0 - a.window);
            const uint32_t c = x.v[t][i * N / 16][i * N % 16 / 4] & 0x7fu;  // (a group is NaN as a whole)
            if (!drop && c == kOctNanCode) {
              note |= 1u << (4 * t + i);
              drop = true;
            }
          }
          if (drop) {
#pragma unroll
            for (int w = 0; w < N / 4; ++w) x.v[t][(i * N / 4 + w) / 4][(i * N / 4 + w) % 4] = 0;
            x.vp[t] = (x.vp[t] & ~(0xffu << (8 * i))) | (127u << (8 * i));
          }
        }
    }
    // Weights against the maximum as it stands; it moves where a lane's sum of eight is large (or NaN). A
    // score's product with the scale is rounded by itself, so that equal scores weigh the same.
    float p[RG][8], sum[RG];
    auto weights = [&](int g) {
#pragma clang fp contract(off)
      sum[g] = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[g][4 * t + i] = fast_exp2(sc[g][t][i] - m[g]);
          sum[g] += p[g][4 * t + i];
        }
    };
    bool fits = true;
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      weights(g);
      fits &= sum[g] <= kODMost;
    }
    if (__builtin_amdgcn_ballot_w64(!fits)) {
#pragma unroll
      for (int g = 0; g < RG; ++g) {
        float mt = kODNone;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) mt = fmaxf(mt, sc[g][t][i]);
        const float mn = fmaxf(m[g], cross_row_max(mt)), f = exp2f(m[g] - mn);
        m[g] = mn;
        l[g] *= f;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[g][e] *= f;
        weights(g);
      }
    }
    bf16x8 part[RG][kODParts];  // the weights' 24 bits
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      l[g] += sum[g];
#pragma unroll
      for (int k = 0; k < kODParts; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          part[g][k][i] = (__bf16)p[g][i];
          p[g][i] -= (float)part[g][k][i];
        }
    }
    float vp[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) vp[t][i] = oct_power((x.vp[t] >> (8 * i)) & 0xffu);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      u32x4 lo, hi;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        bf16x2 pr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int b = i * N + e;
          const uint32_t c = x.v[t][b / 16][b % 16 / 4];
          pr[i] = b & 2 ? oct_pair<true>(c, vp[t][i]) : oct_pair<false>(c, vp[t][i]);
        }
        lo[2 * t] = od_low(pr[0], pr[1]);
        lo[2 * t + 1] = od_low(pr[2], pr[3]);
        hi[2 * t] = od_high(pr[0], pr[1]);
        hi[2 * t + 1] = od_high(pr[2], pr[3]);
      }
      const bf16x8 v0 = __builtin_bit_cast(bf16x8, lo), v1 = __builtin_bit_cast(bf16x8, hi);
#pragma unroll
      for (int g = 0; g < RG; ++g)
#pragma unroll
        for (int k = 0; k < kODParts; ++k) {
          acc[g][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, part[g][k], acc[g][e], 0, 0, 0);
          acc[g][e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, part[g][k], acc[g][e + 1], 0, 0, 0);
        }
    }
    if (CHUNK && __builtin_amdgcn_ballot_w64(note != 0)) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // tokens 16 (k / 4) + 4 (0..3) + k % 4, lanes' dims N lane % 16
        const uint64_t of = __builtin_amdgcn_ballot_w64((note >> k) & 1);
        if (!of) continue;
        for (int b = 0; b < 4; ++b) {
          const uint32_t lanes = (uint32_t)(of >> (16 * b)) & 0xffffu;
          const int tk = s * kODStep + 16 * (k / 4) + 4 * b + k % 4;
#pragma unroll
          for (int g = 0; g < RG; ++g)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (tk <= lim[g] && tk > low[g] && ((lanes >> (4 * q4 + i)) & 1))
#pragma unroll
                for (int e = 0; e < N; ++e) acc[g][e][i] = NAN;
        }
      }
    }
  };

  for (int s = s0 + wv; s < s1;) {
    fetch_ids(s);
    const int cnt = min(64, (s1 - s + W - 1) / W);  // steps of this wave in the set
    if constexpr (D == 256 || (D == 128 && CHUNK)) {
      // One register set: the next step's keys are asked for once the scores are formed, a step's values when it
      // begins. Fewer registers, so heads of 256 dims have two waves per SIMD (24 x 1,000 keys 16.8 us with two
      // sets, 14.7 so; 6 x 5 queries over 4,000 30.5, 28.6; of 128 dims 22.9, 21.6; single queries of 128 dims gain
      // nothing, 64 of 100 to 3,000 43.4, 45.3).
      OctStep<D> x;
      load_keys(0, x);
      for (int k = 0; k < cnt; ++k) {
        load_values(k, x);
        __builtin_amdgcn_sched_barrier(0);
        step(s + W * k, x, [&]() {
          __builtin_amdgcn_sched_barrier(0);
          load_keys(min(k + 1, cnt - 1), x);
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    } else {
      OctStep<D> xa, xb;
      auto none = []() {};
      load(0, xa);
      int k = 0;
      while (true) {
        load(min(k + 1, cnt - 1), xb);
        __builtin_amdgcn_sched_barrier(0);
        step(s + W * k, xa, none);
        if (++k >= cnt) break;
        load(min(k + 1, cnt - 1), xa);
        __builtin_amdgcn_sched_barrier(0);
        step(s + W * k, xb, none);
        if (++k >= cnt) break;
      }
    }
    s += W * 64;
  }
  if (bad && lane == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
#pragma unroll
  for (int g = 0; g < RG; ++g) l[g] = bad ? NAN : cross_row_sum(l[g]);

  // ---- the waves' results, joined in LDS
  if (q4 == 0) {
#pragma unroll
    for (int g = 0; g < RG; ++g) {
      red_m[wv][kODRows * g + col] = m[g];
      red_l[wv][kODRows * g + col] = l[g];
    }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < RG; ++g) {
    const int r = kODRows * g + col;
    float M = kODNone;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, red_m[w][r]);
    const float f = exp2f(m[g] - M);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < N; e += 4)
        *(float4v*)&red_o[wv][r][(4 * q4 + i) * N + e] =
            float4v{acc[g][e][i] * f, acc[g][e + 1][i] * f, acc[g][e + 2][i] * f, acc[g][e + 3][i] * f};
  }
  __syncthreads();
  const int PR = a.part_rows;
  const int64_t part = ((int64_t)P.part + P.c) * a.H + h;  // (where the block is split)
  for (int i = tid; i < nrow * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float mm = kODNone, ll = 0.f;
    float4v o = {};
#pragma unroll
    for (int w = 0; w < W; ++w) mm = fmaxf(mm, red_m[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      ll += red_l[w][r] * exp2f(red_m[w][r] - mm);
      o += *(const float4v*)&red_o[w][r][d];
    }
    if (P.nch == 1) {
      finish(r, d, o, mm, ll);
    } else {
      store_agent16(a.ws_o + (part * PR + r) * D + d, o);
      if (d == 0) store_agent8(a.ws_ml + (part * PR + r) * 2, float2v{mm, ll});
    }
  }
  if (P.nch == 1) return;

  // ---- the last workgroup of a (block, head) joins its chunks' partials
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* cnt = a.ws_cnt + (P.block * a.H + h) * a.cnt_stride;
    const int prev = arrive(cnt);
    last_sh = prev == P.nch - 1;
    if (last_sh) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_sh) return;
  // d / 4 lanes take a row, four dims each, chunk after chunk with a running maximum; where rows are few,
  // 2^share such teams take every 2^share-th chunk of a row and are joined in LDS.
  constexpr int LPR = D / 4, TEAMS = kThreads / LPR, AHEAD = 8;
  const int team = tid / LPR, d4 = tid % LPR * 4;
  int share = 0;
  while (nrow << (share + 1) <= TEAMS && 2 << share <= P.nch) ++share;
  const int64_t part0 = (int64_t)P.part * a.H + h;
  const int sub = team & ((1 << share) - 1);
  for (int r0 = 0; r0 < nrow; r0 += TEAMS >> share) {
    const int r = r0 + (team >> share);
    float mm = kODNone, ll = 0.f;
    float4v o = {};
    if (r < nrow)
      for (int c0 = sub; c0 < P.nch; c0 += AHEAD << share) {
        float4v x[AHEAD];
        float2v ml[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int c = min(c0 + (u << share), P.nch - 1);
          const int64_t at = (part0 + (int64_t)c * a.H) * PR + r;
          ml[u] = ld_agent2(a.ws_ml + at * 2);
          x[u] = ld_agent16(a.ws_o, a.o_bytes, (uint32_t)((at * D + d4) * 4));
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (c0 + (u << share) < P.nch) {
            const float mn = fmaxf(mm, ml[u][0]), f = exp2f(mm - mn), g = exp2f(ml[u][0] - mn);
            o = o * f + x[u] * g;
            ll = ll * f + ml[u][1] * g;
            mm = mn;
          }
      }
    if (share) {  // (one round: rows << share fit the teams)
      float* at = red_all + team * (D + 8);
      *(float4v*)(at + d4) = o;
      if (d4 == 0) {
        at[D] = mm;
        at[D + 1] = ll;
      }
      __syncthreads();
      if (sub || r >= nrow) return;
      for (int u = 1; u < 1 << share; ++u) {
        const float* y = at + u * (D + 8);
        const float mn = fmaxf(mm, y[D]), f = exp2f(mm - mn), g = exp2f(y[D] - mn);
        o = o * f + *(const float4v*)(y + d4) * g;
        ll = ll * f + y[D + 1] * g;
        mm = mn;
      }
    }
    if (r < nrow) finish(r, d4, o, mm, ll);
  }
}

// The plan's item target: two workgroups per compute unit, one of the larger ones. Three of the smaller would
// fit, but shorter chunks pay their prologue and their join more often (8 x 14,402 tokens: 45.3 us with two,
// 50 with three; 8 x 5 queries over 3,000 keys 21, 25).
static int od_target(int d, int waves) { return (d == 256 || waves > 4 ? 1 : 2) * device_cu_count(); }

// Waves of a workgroup: four, or eight where the (block, head) pairs are about as many as the compute units,
// so that few are split, and their keys of a middle length. Measured with four and with eight (us, eight KV
// heads of 128 and 64 dims): 24 x 700 keys 13.8 and 11.9, 10.8 and 8.5; 24 x 3,000 35.6 and 29.0, 22.2 and
// 22.4; 32 x 2,000 28.6 and 27.2, 17.9 and 15.7; but 24 x 512 9.0 and 10.1, 7.1 and 7.4; 32 of 600 to 11,000
// 72.8 and 79.0, 42.6 and 47.8; 8 x 1,024 10.1 and 11.5; 16 x 1,024 11.9 and 12.6, 9.6 and 9.0. (Heads of 256
// dims have registers for four.)
static int od_waves(int d, int64_t pairs, int max_seq, int max_q, int window, int groups) {
  const int span = window ? std::min(max_seq, window + max_q - 1) : max_seq, steps = (span + kODStep - 1) / kODStep;
  const int cus = device_cu_count();
  return d < 256 && groups == 1 && 8 * pairs > 5 * cus && pairs <= cus && steps > 16 && steps <= 96 ? 8 : 4;
}

// Groups of 16 rows in a block: one, or two where blocks of one are more than the plan aims at; both share the
// keys' and values' conversion, but a small call waits longer for its larger join (us, with one and two, eight
// KV heads of 128 dims: 60 x 8 queries over 1,500 keys 45.2, 38.1; 30 x 5 over 1,500 25.5, 27.8; 6 x 5 over
// 4,000 20.8, 25.3; four of 256 dims: 60 x 8 62.6, 43.9; 30 x 5 32.9, 33.4). Of fp16 queries of 256 dims there
// are registers for one.
static int od_groups(int H, int d, int q_dtype, int num_reqs, int rows) {
  if (rows <= kODRows || (d == 256 && q_dtype == TTKV_DTYPE_F16)) return 1;
  return (int64_t)num_reqs * H * ((rows + kODRows - 1) / kODRows) > od_target(d, 4) ? 2 : 1;
}

// Requests per launch, of `blocks` row blocks each: the plan's lanes, and a counter per (block, head).
static int od_slice(int H, int blocks, int num_reqs) {
  return std::max(1, std::min({num_reqs, kODPlanLanes * 64, kMaxCounters / (H * blocks)}));
}

// Items of split blocks, at most, of `pairs` (block, head) pairs. A chunk has at least total / target
// steps, and a split block of st steps has less than st / C + 1 < 2 st / C chunks: less than 2 target of
// them in all; and whole rounds of a request's waves, four where they are fewest.
static int64_t od_max_chunks(int max_seq) {
  const int64_t round = kODStep * 4;
  return std::max<int64_t>(1, (max_seq + round - 1) / round + 1);  // (a window's first step may be cut)
}
static int64_t od_parts(int d, int64_t pairs, int max_seq) {
  return std::min<int64_t>(2 * od_target(d, 4), pairs * od_max_chunks(max_seq));
}

int64_t octet_decode_workspace_bytes(int H, int HQ, int d, int num_reqs, int max_q, int max_seq) {
  if (num_reqs == 0 || max_q == 0) return 256;
  // (sizes that grow with every argument: layers of unlike heads share a workspace)
  return kCounterBytes + (int64_t)2 * 2 * device_cu_count() * 2 * kODRows * (d + 2) * 4;
}

template <int D, int W, int QDT>
static auto od_kernel(int mode, int groups) {
  if constexpr (W == 4 && !(D == 256 && QDT == TTKV_DTYPE_F16))
    if (groups == 2) return octet_decode_kernel<D, W, QDT, kODOwn, 2>;
  return mode == kODSingle ? octet_decode_kernel<D, W, QDT, kODSingle, 1>
         : mode == kODOwn  ? octet_decode_kernel<D, W, QDT, kODOwn, 1>
                           : octet_decode_kernel<D, W, QDT, kODShared, 1>;
}

template <int D, int W>
static int od_launch(OctDecodeArgs a, unsigned grid, int q_dtype, int mode, int groups, hipStream_t st) {
  auto kernel = q_dtype == TTKV_DTYPE_F16 ? od_kernel<D, W, TTKV_DTYPE_F16>(mode, groups)
                                          : od_kernel<D, W, TTKV_DTYPE_BF16>(mode, groups);
  const int smem = W * kODRows * groups * (D + 4) * 4;
  if (smem > 65536 - 4096)
    if (int rc = raise_smem_limit((const void*)kernel, smem)) return rc;
  // workgroups per CU, by kernel (the same on every device of a process; a race writes the same number)
  static std::atomic<int> fit[2][4];
  std::atomic<int>& known = fit[q_dtype == TTKV_DTYPE_F16][groups == 2 ? 3 : mode];
  int per = known.load(std::memory_order_relaxed);
  if (!per) {
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, 64 * W, smem) != hipSuccess || per < 1) per = 1;
    known.store(per, std::memory_order_relaxed);
  }
  a.resident = std::max(per * device_cu_count(), od_target(D, W));
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * W), smem, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("octet decode launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}
template <int D>
static int od_launch(const OctDecodeArgs& a, int waves, unsigned grid, int q_dtype, int mode, int groups,
                     hipStream_t st) {
  if (waves == 4) return od_launch<D, 4>(a, grid, q_dtype, mode, groups, st);
  return od_launch<D, D == 256 ? 4 : 8>(a, grid, q_dtype, mode, groups, st);
}

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
  if (H > kMaxCounters / (kODMaxQ * 16 / kODRows)) return host_fail(TTKV_E_UNSUPPORTED, "too many KV heads");
  if (window < 0) return host_fail(TTKV_E_INVALID, "negative window");
  if (num_reqs && (!q || !bt || !seq_lens || !qsl || !out || !err))
    return host_fail(TTKV_E_INVALID, "null pointer argument");
  if (((uintptr_t)q | (uintptr_t)out) % 16 || q_row_stride % 8 || out_row_stride % 8)
    return host_fail(TTKV_E_INVALID, "query / out rows must be 16-byte aligned");
  if (q && out && !(out == q && (out_row_stride == q_row_stride || num_tokens == 1)) &&
      rows_meet(out, 2 * out_row_stride, 2ll * HQ * d, q, 2 * q_row_stride, 2ll * HQ * d, num_tokens))
    return host_fail(TTKV_E_INVALID, "out overlaps the query without being it");
  if (rows_fold(out_row_stride, (int64_t)HQ * d, num_tokens))
    return host_fail(TTKV_E_INVALID, "rows of out overlap one another");
  const int64_t need = octet_decode_workspace_bytes(H, HQ, d, num_reqs, max_q, max_seq);
  if (!ws || ws_bytes < need || (uintptr_t)ws % 256)
    return host_fail(TTKV_E_WORKSPACE, "decode workspace needs " + std::to_string(need) + " bytes, 256-aligned");
  if (num_reqs == 0 || num_tokens == 0 || max_q == 0) return TTKV_OK;
  if (window >= max_seq) window = 0;  // no window
  const int rows = HQ / H * max_q, groups = od_groups(H, d, q_dtype, num_reqs, rows);
  const int blocks = (rows + kODRows * groups - 1) / (kODRows * groups);
  const int mode = max_q == 1 ? kODSingle : blocks == 1 ? kODOwn : kODShared;
  const int slice = od_slice(H, blocks, num_reqs);
  const int64_t parts = od_parts(d, (int64_t)slice * H * blocks, max_seq);
  OctDecodeArgs a{};
  a.H = H;
  a.G = HQ / H;
  a.scale_log2 = scale * kLog2e;
  a.q = (const uint16_t*)q;
  a.q_row_stride = q_row_stride;
  a.num_tokens = num_tokens;
  a.page = page;
  a.tile_stride = kOctTile * slot_stride;
  a.num_blocks = (int)(n_slots / bs);
  a.tpb = bs / kOctTile;
  a.bt_row_stride = bt_row_stride;
  a.max_q = max_q;
  a.max_seq = max_seq;
  a.window = window;
  a.sinks = sinks;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_row_stride = out_row_stride;
  a.lse = lse;
  a.part_rows = std::min(rows, kODRows * groups);
  a.ws_cnt = (int*)ws;
  a.ws_o = (float*)((char*)ws + kCounterBytes);
  a.ws_ml = a.ws_o + parts * a.part_rows * d;
  a.o_bytes = (uint32_t)(parts * a.part_rows * d * 4);
  a.join = (float)(a.part_rows * d) * kODJoin;
  a.err = err;
  for (int r0 = 0; r0 < num_reqs; r0 += slice) {
    a.num_reqs = std::min(slice, num_reqs - r0);
    a.seq_lens = seq_lens + r0;
    a.qsl = qsl + r0;
    a.bt = bt + (int64_t)r0 * bt_row_stride;
    // an item per (block, head), and what the split ones have more
    const int64_t pairs = (int64_t)a.num_reqs * H * blocks;
    a.cnt_stride = (int)std::max<int64_t>(1, std::min<int64_t>(32, kMaxCounters / pairs));
    const int waves = od_waves(d, pairs, max_seq, max_q, window, groups), target = od_target(d, waves);
    a.by_target = 1.f / (float)target;
    a.by_H = 1.f / (float)H;
    const unsigned grid = (unsigned)std::min(pairs + target, pairs * od_max_chunks(max_seq));
    const int rc = d == 64    ? od_launch<64>(a, waves, grid, q_dtype, mode, groups, st)
                   : d == 128 ? od_launch<128>(a, waves, grid, q_dtype, mode, groups, st)
                              : od_launch<256>(a, waves, grid, q_dtype, mode, groups, st);
    if (rc != TTKV_OK) return rc;
  }
  return TTKV_OK;
}

}  // namespace ttkv
