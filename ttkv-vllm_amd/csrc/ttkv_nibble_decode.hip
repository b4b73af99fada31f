// Decode attention over the 4-bit cache (format: ttkv_nibble.h): one query per request, and short
// chunks of queries. gfx950 / CDNA4.
//
// The rows of a (request, KV head) are its query heads, or (chunk) its (query, query head) pairs, row
// = j G + p. Work item = (request, block of 16 rows or of two groups of 16, chunk of the block's
// 32-token steps, KV head),
// one workgroup of 4 waves that take the chunk's steps in turn. The chunk length comes from a plan
// that every workgroup computes alike from the batch's lengths: the shortest that spreads the batch's
// steps over the resident workgroups, so a ragged batch fills the chip by its total work. Items of a
// (block, head) leave unnormalised partials in the workspace; the last to arrive joins them.
//
// One step of a wave, two tiles of 16 tokens:
//   S^T [token, row] = K Q^T, four v_mfma_f32_16x16x32_f16 per tile and group of rows: a lane's 16 key code
//     bytes are its A operand of all four (token lane % 16, 8 dims of each group of 32), unpacked by a
//     shift and a mask per pair and dequantised exactly in packed fp16; the queries are the B operand,
//     held in registers. Columns without a row are zero.
//   softmax in the result's own registers: lane column = row, 8 tokens of it. Weights are taken against
//     the maximum as it stands, which moves only when a weight leaves fp16 (2^8 growth), so most
//     steps need no maximum and no exchange between lanes; the sum stays per lane until the end.
//   O^T [dim, row] += V^T P^T, eight MFMAs: the scores' layout is the B operand's as it
//     stands, and a lane's 16 value code bytes per tile are its A operand of all eight (a dim pair of
//     each group, four tokens). The result's column is the row again, so the rescale is a lane's factor.
// Bytes per step 4,608; the two register sets keep the next step's loads in flight. Bound by memory: 8 x
// 14,402 tokens of 8 heads, 133 MB, 30.2 to 33 us by card, 4.4 TB/s at best (a copy reaches 4.8); the
// loads alone took 26 us of a profiled 33. 61 requests of 70 to 2,900 tokens 27.6 us for 98 MB; one of
// 1,082 tokens 9 us, the chain of plan, block ids, codes, hand-off and join.
#include <math.h>

#include <type_traits>

#include "ttkv_host.h"
#include "ttkv_nibble.h"

namespace ttkv {

constexpr int kNDThreads = 256;
constexpr int kNDWaves = 4;
constexpr int kNDStep = 2 * kNibTile;  // tokens per wave step
constexpr int kNDPlanLanes = 4;        // requests per lane in the plan: 256 per launch
constexpr int kNDClasses = 8;          // of chunk lengths, for the items' order
constexpr int kNDShortRows = 256;      // rows of a chunk that may come here
constexpr int64_t kNDShortWork = 17000;  // and steps of all its blocks,
constexpr int64_t kNDFewWork = 24000;    // where they are few
constexpr int64_t kNDWideWork = 36000;   // from which two groups of 16 rows share a block
constexpr int kNDRows = 16;            // rows of a block: a matrix product's columns
constexpr float kNDLift = 8.f;         // of the weights (nib_max)

struct NibDecodeArgs {
  int H, G;
  float scale_log2;
  const uint16_t* q;
  int64_t q_row_stride;
  const uint8_t* page;
  int64_t tile_stride;
  int num_blocks;
  int tpb;  // tiles per block
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* seq_lens;
  const int32_t* qsl;
  const int32_t* req_index;  // chunks
  int num_reqs, max_q, max_seq;
  int num_starts;  // entries of qsl (decode)
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  int* ws_cnt;
  float* ws_o;        // [split items][part_rows][kD]
  float* ws_ml;       // [split items][part_rows][2]
  uint32_t o_bytes;   // size of ws_o
  int part_rows;      // rows of an item's partials
  int target;
  int32_t* err;
};

struct NibDecodePlan {
  int r, rb, c, h;      // batch row, row block, chunk, KV head
  int n, Q, rows, nch;  // keys, queries, rows of all blocks, the block's chunks
  int q0;               // the request's first row of the query
  int part, block;      // the block's first split item and its number, both before the head
  bool none;
};

// Chunks of at most C steps, by 1 / C to an ulp: never more than the quotient rounded up, and one less
// only where it is whole, alike for every workgroup (the chunks are cut equal from their number).
__device__ __forceinline__ int nd_chunks(int steps, int C, float by_C) {
  return max(1, (int)((float)(steps + C - 1) * by_C));
}

// RB: rows of a block.
template <bool CHUNK, int RB>
__device__ __forceinline__ NibDecodePlan nd_plan(const NibDecodeArgs& a, int item) {
  const int lane = threadIdx.x & 63;
  int idx[kNDPlanLanes], n[kNDPlanLanes], q0[kNDPlanLanes], Q[kNDPlanLanes];
  int st[kNDPlanLanes], rb[kNDPlanLanes];
  int total = 0, longest = 0, whole = 0;
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    idx[i] = n[i] = q0[i] = Q[i] = st[i] = rb[i] = 0;
    if (64 * i >= a.num_reqs) continue;
    const int r = lane + 64 * i;
    const bool on = r < a.num_reqs;
    idx[i] = CHUNK && a.req_index && on ? a.req_index[r] : on ? r : 0;
    n[i] = on ? a.seq_lens[idx[i]] : 0;
    q0[i] = on ? a.qsl[idx[i]] : 0;
    // decode: no query where the next request's row is the same one
    Q[i] = !on ? 0 : CHUNK ? a.qsl[idx[i] + 1] - q0[i] : r + 1 >= a.num_starts || a.qsl[r + 1] != q0[i];
  }
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    if (64 * i >= a.num_reqs) continue;
    const int nn = min(max(n[i], 0), a.max_seq);
    st[i] = Q[i] != 0 ? (nn + kNDStep - 1) / kNDStep : 0;
    if (CHUNK && nn < Q[i]) st[i] = 1;
    rb[i] = CHUNK ? (min(max(Q[i], 0), a.max_q) * a.G + RB - 1) / RB : Q[i];
    total += st[i] * rb[i];
    longest = max(longest, st[i]);
    whole += rb[i];
  }
  total = wave_sum_i(total);
  // whole rounds of the four waves
  const int64_t all = (int64_t)total * a.H;
  const int per = all < 0x40000000 ? (int)((uint32_t)all + a.target - 1) / a.target
                                   : (int)fminf((float)all / (float)a.target * 1.00001f, 1e8f) + 1;
  int C = max(1, (per + kNDWaves - 1) / kNDWaves) * kNDWaves;
  // A chunk's step costs the request about 0.2 us and a chunk about as much in the join: where the
  // batch would fill the chip with shorter ones, the root of the steps, rounded down for 16 rows, whose
  // steps cost more (1 x 14,000 tokens of 8 heads: 21.1 us, 16.6 so; of 2 heads 28.9, 16.7).
  C = max(C, (int)(sqrtf((float)wave_max_i(longest)) / kNDWaves + (CHUNK ? 0.25f : 0.75f)) * kNDWaves);
  if (CHUNK) {
    // Two workgroups of chunks fill a CU (decode: three): longer chunks rather than a second round of
    // them, where the batch has not more blocks anyway (6 x 32 queries over 600 keys: 27.5 us, 17.0 so).
    whole = wave_sum_i(whole);
    while ((int64_t)whole * a.H <= a.target) {
      int items = 0;
      const float by_C = __builtin_amdgcn_rcpf((float)C);
#pragma unroll
      for (int i = 0; i < kNDPlanLanes; ++i)
        if (64 * i < a.num_reqs) items += rb[i] * nd_chunks(st[i], C, by_C);
      if ((int64_t)wave_sum_i(items) * a.H <= a.target) break;
      C += max(1, C / (16 * kNDWaves)) * kNDWaves;
    }
  }
  NibDecodePlan P{};
  P.h = item % a.H;
  const int it = item / a.H;
  P.none = true;
  // Long chunks first: the short ones fill the gaps that they leave at the end (61 requests of 70 to
  // 2,900 tokens: 30.2 us in the batch's order, 28.3 so). Classes by the chunk's eighth of C, in the
  // batch's order within each.
  int nch[kNDPlanLanes], cls[kNDPlanLanes], bex[kNDPlanLanes], pex[kNDPlanLanes];
  int blocks = 0, parts = 0;
  const float by_C = __builtin_amdgcn_rcpf((float)C);
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    if (64 * i >= a.num_reqs) break;
    nch[i] = nd_chunks(st[i], C, by_C);
    const float eighths = (float)st[i] * __builtin_amdgcn_rcpf((float)nch[i]) * by_C * kNDClasses;
    cls[i] = kNDClasses - 1 - min(kNDClasses - 1, (int)eighths);
    const int split = nch[i] > 1 ? rb[i] * nch[i] : 0;
    const int bincl = CHUNK ? nib_scan(rb[i]) : 0, pincl = nib_scan(split);
    bex[i] = CHUNK ? blocks + bincl - rb[i] : 64 * i + lane;
    pex[i] = parts + pincl - split;
    parts += __builtin_amdgcn_readlane(pincl, 63);
    if (CHUNK) blocks += __builtin_amdgcn_readlane(bincl, 63);
  }
  int carry = 0;
  for (int k = 0; k < kNDClasses && P.none; ++k) {
#pragma unroll
    for (int i = 0; i < kNDPlanLanes; ++i) {
      if (64 * i >= a.num_reqs) break;
      const int items = cls[i] == k ? rb[i] * nch[i] : 0;
      if (!__builtin_amdgcn_ballot_w64(items > 0)) continue;
      const int incl = nib_scan(items), ex = carry + incl - items;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(items > 0 && ex <= it && it < ex + items);
      if (hit) {
        const int ln = __builtin_ctzll(hit);
        P.none = false;
        P.r = __builtin_amdgcn_readlane(idx[i], ln);
        P.n = __builtin_amdgcn_readlane(n[i], ln);
        P.Q = __builtin_amdgcn_readlane(Q[i], ln);
        P.q0 = __builtin_amdgcn_readlane(q0[i], ln);
        P.nch = __builtin_amdgcn_readlane(nch[i], ln);
        const int local = it - __builtin_amdgcn_readlane(ex, ln);
        P.rb = CHUNK ? local / P.nch : 0;
        P.c = local - P.rb * P.nch;
        P.rows = CHUNK ? min(max(P.Q, 0), a.max_q) * a.G : a.G;
        P.part = __builtin_amdgcn_readlane(pex[i], ln) + P.rb * P.nch;
        P.block = __builtin_amdgcn_readlane(bex[i], ln) + P.rb;
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
  }
  return P;
}

// One step's bytes of a lane: per tile its 16 key and 16 value code bytes, its token's four key
// parameters and its four tokens' value parameters.
struct NibStep {
  u32x4 k[2], v[2];
  u32x2v kp[2];
  u32x4 vp[2][2];
};

// RG: groups of 16 rows that a block has, one column of a product each.
template <int QDT, bool CHUNK, int RG>
__global__ __launch_bounds__(kNDThreads, 2) void nibble_decode_kernel(NibDecodeArgs a) {
  constexpr int RB = kNDRows * RG;
  extern __shared__ __align__(16) float red_all[];  // [waves][RB][kD]: the waves' results, then the join's
  float(*red_o)[RB][kD] = (float(*)[RB][kD])red_all;
  __shared__ float red_m[kNDWaves][RB], red_l[kNDWaves][RB];
  __shared__ int last_sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const NibDecodePlan P = nd_plan<CHUNK, RB>(a, blockIdx.x);
  if (P.none) return;
  const int h = P.h, G = a.G;
  const int n = min(max(P.n, 0), a.max_seq);
  const int p0 = CHUNK ? n - P.Q : n - 1;  // position of query 0
  if (tid == 0 && h == 0 && P.c == 0 && P.rb == 0 &&
      (P.n > a.max_seq || (CHUNK && (P.Q > a.max_q || p0 < 0))))
    atomicOr(a.err, TTKV_ERR_SEQ_LEN);
  const int64_t q0 = P.q0;
  const int row0 = P.rb * RB, nrow = min(RB, P.rows - row0);  // the block's rows
  // row `r` of the block in the query and the output
  auto row_at = [&](int r, int64_t stride) -> int64_t {
    const int row = row0 + r, j = CHUNK ? row / G : 0;
    return (q0 + j) * stride + (int64_t)(h * G + row - j * G) * kD;
  };
  if (CHUNK ? p0 < 0 : n == 0) {  // fewer keys than queries; an empty request's attention is 0
    for (int i = tid; i < nrow * kD; i += kNDThreads)
      store_act(a.out, a.out_dtype, row_at(i / kD, a.out_row_stride) + i % kD, CHUNK ? NAN : 0.f);
    return;
  }
  const int col = lane & 15, q4 = lane >> 4;

  // The queries, row 16 r + `col` of group r, as the B operand of the four score products
  half8 qf[RG][4];
  float qs[RG], m[RG], l[RG];
  int lim[RG];  // last key the lane's row sees
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const int row = min(kNDRows * r + col, nrow - 1);
    const NibRow qrow = nib_load_row(a.q + row_at(row, a.q_row_stride), q4);
    nib_query<QDT>(qrow, a.scale_log2, kNDRows * r + col < nrow, qf[r], qs[r]);
    m[r] = kNibNone;
    l[r] = 0.f;
    lim[r] = CHUNK ? p0 + (row0 + row) / G : p0;
  }
  const int see_min = CHUNK ? p0 + row0 / G : p0;                     // and every row
  float4v acc[RG][8];  // [group][dim of the pair]: dims 32 g + 8 q4 + 2 i + b of the lane's rows
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[r][i] = float4v{};

  const int steps = (CHUNK ? p0 + (row0 + nrow - 1) / G : p0) / kNDStep + 1;
  // the block's steps in equal parts
  const int s0 = (int)((int64_t)steps * P.c / P.nch);
  const int s1 = (int)((int64_t)steps * (P.c + 1) / P.nch);
  bool bad = false;
  float most = kNibMost;  // below every sum from the wave's first far maximum on

  const NibMasks masks = nib_masks();
  const uint8_t* base = a.page + (int64_t)h * kNibRecord;
  const int32_t* bt = a.bt + (int64_t)P.r * a.bt_row_stride;
  // tile ids of this wave's next 64 steps, one step per lane (-1: a block outside the cache)
  int tid0 = 0, tid1 = 0;
  auto fetch_ids = [&](int s) {
    const int mine = min(s + kNDWaves * lane, s1 - 1);  // (past the chunk: its last step's again)
    const int t0 = 2 * mine, t1 = min(2 * mine + 1, (n - 1) / kNibTile);
    const int b0 = t0 / a.tpb, b1 = t1 / a.tpb;
    const int i0 = bt[b0], i1 = bt[b1];
    tid0 = (uint32_t)i0 < (uint32_t)a.num_blocks ? i0 * a.tpb + t0 - b0 * a.tpb : -1;
    tid1 = (uint32_t)i1 < (uint32_t)a.num_blocks ? i1 * a.tpb + t1 - b1 * a.tpb : -1;
  };
  auto load = [&](int k, NibStep& x) {  // the wave's k-th step since fetch_ids
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int id = __builtin_amdgcn_readlane(t ? tid1 : tid0, k);
      const uint8_t* rec = base + (int64_t)max(id, 0) * a.tile_stride;
      x.k[t] = __builtin_nontemporal_load(gbl((const u32x4*)(rec + 16 * lane)));
      x.kp[t] = __builtin_nontemporal_load(gbl((const u32x2v*)(rec + kNibKp + 8 * col)));
      x.v[t] = __builtin_nontemporal_load(gbl((const u32x4*)(rec + kNibV + 16 * lane)));
      x.vp[t][0] = __builtin_nontemporal_load(gbl((const u32x4*)(rec + kNibVp + 32 * q4)));
      x.vp[t][1] = __builtin_nontemporal_load(gbl((const u32x4*)(rec + kNibVp + 32 * q4 + 16)));
      bad |= id < 0;
    }
  };
  auto step = [&](int s, NibStep& x) {
    float4v sc[RG][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < RG; ++r) sc[r][t] = float4v{};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const half2v zz = nib_biased(x.kp[t][g >> 1], masks), sg = nib_scales(x.kp[t][g >> 1]);
        const half2v zb = {zz[g & 1], zz[g & 1]}, ss = {sg[g & 1], sg[g & 1]};
        half8 kf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const half2v v = nib_pair(x.k[t][g], j, zb, ss, masks);
          kf[2 * j] = v[0];
          kf[2 * j + 1] = v[1];
        }
#pragma unroll
        for (int r = 0; r < RG; ++r)
          sc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[r][g], sc[r][t], 0, 0, 0);
      }
    }
    const int tok = s * kNDStep + 4 * q4;
    uint32_t note = 0;  // bit 16 t + 4 i + g: that group of the lane's token is NaN
    if ((s + 1) * kNDStep - 1 > see_min) {
      // Some row does not see all of this step: no score past its last key. A weight of 0 must not
      // meet a NaN: values past the last key become 0, and in a chunk a group that is NaN becomes 0
      // too and is noted for the rows that see it.
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tk = tok + 16 * t + i;
#pragma unroll
          for (int r = 0; r < RG; ++r)
            if (tk > lim[r]) sc[r][t][i] = -INFINITY;
          const uint32_t keep = i & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int at = 2 * (g & 1) + (i >> 1);
            const uint32_t w = x.vp[t][g >> 1][at], p = i & 1 ? w >> 16 : w & 0xffffu;
            const bool nan = CHUNK && (p & 0x7c00u) == 0x7c00u;
            if (tk >= n || nan) x.vp[t][g >> 1][at] = w & keep;
            if (CHUNK && nan && tk < n) note |= 1u << (16 * t + 4 * i + g);
          }
        }
    }
    // Weights against the maximum as it stands. It has to move only where a weight leaves fp16 and so
    // makes its lane's sum of eight infinite (or NaN): the scores' own maximum is taken in that case
    // alone, or where a row of the wave has a far one.
    half8 pf[RG];
    float sum[RG];
    auto weights = [&](int r, bool apart) {
      sum[r] = 0.f;
      auto exponent = [&](float s) {
        const float e = fmaf(s, qs[r], -m[r]);
        return apart ? nib_apart(s, qs[r], m[r]) : e;
      };
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          // the one rounding on the way to the output, to the value product's 16-bit operand (low parts
          // in a second product would double it); the sum takes the rounded weights
          const half2v p = {(_Float16)fast_exp2(exponent(sc[r][t][i])),
                            (_Float16)fast_exp2(exponent(sc[r][t][i + 1]))};
          sum[r] = __builtin_amdgcn_fdot2(p, half2v{(_Float16)1.f, (_Float16)1.f}, sum[r], false);
          pf[r][4 * t + i] = p[0];
          pf[r][4 * t + i + 1] = p[1];
        }
    };
    bool fits = true;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      weights(r, false);
      fits &= sum[r] <= most;
    }
    if (__builtin_amdgcn_ballot_w64(!fits)) {
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        float mt = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) mt = fmaxf(mt, sc[r][t][i]);
        const float mn = nib_max(m[r], cross_row_max(mt * qs[r]), kNDLift);
        const float f = exp2f(m[r] - mn);
        m[r] = mn;
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r][i] *= f;
        weights(r, nib_far(mn));
        if (__builtin_amdgcn_ballot_w64(nib_far(mn))) most = -1.f;
      }
    }
#pragma unroll
    for (int r = 0; r < RG; ++r) l[r] += sum[r];
#pragma unroll
    for (int quad = 0; quad < 2; ++quad)
#pragma unroll
      for (int gg = 0; gg < 2; ++gg) {
        const int g = 2 * quad + gg;
        half8 vf[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int pair = 0; pair < 2; ++pair) {
            const uint32_t p2 = x.vp[t][g >> 1][2 * (g & 1) + pair];
            const half2v zb = nib_biased(p2, masks), ss = nib_scales(p2);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              const half2v v = nib_pair(x.v[t][2 * pair + quad], 2 * gg + b, zb, ss, masks);
              vf[b][4 * t + 2 * pair] = v[0];
              vf[b][4 * t + 2 * pair + 1] = v[1];
            }
          }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < RG; ++r)
            acc[r][2 * g + b] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pf[r], acc[r][2 * g + b], 0, 0, 0);
      }
    if (CHUNK && __builtin_amdgcn_ballot_w64(note != 0)) {
      for (int k = 0; k < kNDStep; ++k) {  // token 16 t + 4 q + i
        const int of = __builtin_amdgcn_readlane((int)note, 16 * ((k >> 2) & 3));
        const int groups = (of >> (16 * (k >> 4) + 4 * (k & 3))) & 15;
        if (!groups) continue;
#pragma unroll
        for (int r = 0; r < RG; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if ((groups >> (i >> 1) & 1) && s * kNDStep + k <= lim[r]) acc[r][i] += NAN;
      }
    }
  };

  for (int s = s0 + wv; s < s1;) {
    fetch_ids(s);
    const int cnt = min(64, (s1 - s + kNDWaves - 1) / kNDWaves);  // steps of this wave in the set
    NibStep xa, xb;
    load(0, xa);
    int k = 0;
    while (true) {
      load(min(k + 1, cnt - 1), xb);
      __builtin_amdgcn_sched_barrier(0);
      step(s + kNDWaves * k, xa);
      if (++k >= cnt) break;
      load(min(k + 1, cnt - 1), xa);
      __builtin_amdgcn_sched_barrier(0);
      step(s + kNDWaves * k, xb);
      if (++k >= cnt) break;
    }
    s += kNDWaves * 64;
  }
  if (bad && lane == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
#pragma unroll
  for (int r = 0; r < RG; ++r) l[r] = bad ? NAN : cross_row_sum(l[r]);

  // ---- the four waves' results, joined in LDS
  if (q4 == 0) {
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      red_m[wv][kNDRows * r + col] = m[r];
      red_l[wv][kNDRows * r + col] = l[r];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const int row = kNDRows * r + col;
    float M = kNibNone;
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) M = fmaxf(M, red_m[w][row]);
    const float f = exp2f(m[r] - M);
    if (row < nrow) {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2v o = {acc[r][2 * g][i] * f, acc[r][2 * g + 1][i] * f};
          *(float2v*)&red_o[wv][row][32 * g + 8 * q4 + 2 * i] = o;
        }
    }
  }
  __syncthreads();
  const int PR = a.part_rows;
  const int64_t part = ((int64_t)P.part + P.c) * a.H + h;  // (where the block is split)
  for (int e = 4 * tid; e < nrow * kD; e += 4 * kNDThreads) {
    const int p = e / kD, d = e % kD;
    float mm = kNibNone, ll = 0.f;
    float4v o = {};
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) mm = fmaxf(mm, red_m[w][p]);
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) ll += red_l[w][p] * exp2f(red_m[w][p] - mm);
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) o += *(const float4v*)&red_o[w][p][d];
    if (P.nch == 1) {
      store_act4(a.out, a.out_dtype, row_at(p, a.out_row_stride) + d, o * (1.f / ll), true);
    } else {
      store_agent16(a.ws_o + (part * PR + p) * kD + d, o);
      if (d == 0) store_agent8(a.ws_ml + (part * PR + p) * 2, float2v{mm, ll});
    }
  }
  if (P.nch == 1) return;

  // ---- the last workgroup of a (block, head) joins its chunks' partials
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* cnt = a.ws_cnt + P.block * a.H + h;
    const int prev = arrive(cnt);
    last_sh = prev == P.nch - 1;
    if (last_sh) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_sh) return;
  // Half a wave takes a row, a lane four dims of it; lane % 32 first holds a chunk's maximum and sum.
  // All of a wave's rows are under way together. With four rows or less and more chunks than a half wave
  // has in flight, 2, 4 or 8 of them share a row's chunks and are joined in LDS (1 x 60,000 tokens of one
  // head: 22.2 us, 18.9 so; 4 x 9,000 of 8: 20.7, 19.7).
  constexpr int ROWS = RB / (2 * kNDWaves);  // per half wave
  const int c32 = lane & 31, lead = lane & 32;
  const int64_t part0 = (int64_t)P.part * a.H + h;
  // log2 of the half waves per row
  const int share = min(nrow > 4 ? 0 : nrow > 2 ? 1 : nrow > 1 ? 2 : 3,
                        P.nch <= 8 ? 0 : P.nch <= 16 ? 1 : P.nch <= 32 ? 2 : 3);
  auto join = [&](auto rows_c, auto shared_c) {
    constexpr bool SHARED = decltype(shared_c)::value;
    constexpr int K = decltype(rows_c)::value;
    // chunks of every row in flight (one row: 8 heads per KV head, 2 x 12,000 tokens: 20.4 us with 8, 19.3;
    // shared, 4 x 9,000: 18.6 with 8, 19.1)
    constexpr int AHEAD = K == 1 && !SHARED ? 16 : K == 4 ? 4 : 8;
    const int half = 2 * wv + (lane >> 5), sh = SHARED ? share : 0;
    const int sub = SHARED ? half & ((1 << share) - 1) : 0;
    // by half waves or, unshared, by waves (one of whose rows may be the last one again)
    auto on = [&](int k) { return SHARED ? half >> sh < nrow : 2 * (wv + kNDWaves * k) < nrow; };
    float mm[K], ll[K];
    float4v o[K];
    int row[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      row[k] = min((half >> sh) + 2 * kNDWaves * k, nrow - 1);
      mm[k] = kNibNone;
      ll[k] = 0.f;
      o[k] = float4v{};
    }
    for (int c0 = 0; c0 < P.nch; c0 += 32) {
      const int nb = min(32, P.nch - c0);
      float4v x[K][AHEAD];
      auto fetch = [&](int j) {  // chunks j + sub, j + sub + 2^sh, ...
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (on(k))
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
              const int c = j + sub + (u << sh);
              if (c < nb)
                x[k][u] = ld_agent16(
                    a.ws_o, a.o_bytes,
                    (uint32_t)((((part0 + (int64_t)(c0 + c) * a.H) * PR + row[k]) * kD + 4 * c32) * 4));
            }
      };
      float2v ml[K];
      float wc[K];
#pragma unroll
      for (int k = 0; k < K; ++k)
        ml[k] = ld_agent2(a.ws_ml + ((part0 + (int64_t)(c0 + min(c32, nb - 1)) * a.H) * PR + row[k]) * 2);
      fetch(0);  // (a round trip that the weights' does not come before)
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float x0, x1;
        swap16(row_max(c32 < nb ? ml[k][0] : kNibNone), x0, x1);
        const float mn = fmaxf(mm[k], fmaxf(x0, x1));
        const float keep = exp2f(mm[k] - mn);
        wc[k] = c32 < nb ? exp2f(ml[k][0] - mn) : 0.f;
        swap16(row_sum(c32 < nb ? ml[k][1] * wc[k] : 0.f), x0, x1);
        ll[k] = ll[k] * keep + x0 + x1;
        o[k] *= keep;
        mm[k] = mn;
      }
      for (int j = 0; j < nb; j += AHEAD << sh) {
        if (j) fetch(j);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int c = j + sub + (u << sh);
          if (SHARED || c < nb)
#pragma unroll
            for (int k = 0; k < K; ++k) {
              const float w = __shfl(wc[k], lead + (c & 31));
              if (on(k) && c < nb) o[k] += x[k][u] * w;
            }
        }
      }
    }
    if (SHARED) {
      float* sums = red_all;  // [half wave][kD]
      *(float4v*)(sums + half * kD + 4 * c32) = o[0];
      __syncthreads();
      if (sub) return;
      for (int u = 1; u < 1 << sh; ++u) o[0] += *(const float4v*)(sums + (half + u) * kD + 4 * c32);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if ((half >> sh) + 2 * kNDWaves * k < nrow)
        store_act4(a.out, a.out_dtype, row_at(row[k], a.out_row_stride) + 4 * c32, o[k] * (1.f / ll[k]), true);
  };
  if (share) join(std::integral_constant<int, 1>{}, std::true_type{});
  else if (nrow <= 2 * kNDWaves) join(std::integral_constant<int, 1>{}, std::false_type{});
  else join(std::integral_constant<int, ROWS>{}, std::false_type{});
}

// The plan's item target: two workgroups per CU. A third would fit beside them, but shorter chunks
// pay their prologue and join more often (8 x 14,402 tokens on one card: 30.7 us at two per CU, 35.7 at
// two and a half, 32.8 at three; 61 requests of 70 to 2,900: 28.6, 28.2, 31.0).
static int nd_target() { return 2 * device_cu_count(); }

// Requests per launch, of `blocks` row blocks each: the plan's lanes, and a counter per (block, head).
static int nd_slice(int H, int blocks, int num_reqs) {
  return std::max(1, std::min({num_reqs, kNDPlanLanes * 64, kMaxCounters / (H * blocks)}));
}

// Chunks of a block at most: whole rounds of the four waves.
static int64_t nd_max_chunks(int max_seq) {
  const int64_t round = kNDStep * kNDWaves;
  return std::max<int64_t>(1, (max_seq + round - 1) / round);
}

// Items of split blocks, at most, of `pairs` (block, head) pairs. A chunk has at least total / target
// steps, and a split block of st steps has less than st / C + 1 < 2 st / C chunks: less than 2 target of
// them in all.
static int64_t nd_parts(int64_t pairs, int max_seq) {
  const int64_t most = nd_max_chunks(max_seq);
  return most <= 1 ? 0 : std::min<int64_t>(2 * nd_target(), pairs * most);
}

static int nd_blocks(int rows, int groups) {
  return (rows + kNDRows * groups - 1) / (kNDRows * groups);
}

// Groups of 16 rows per block: one, or two where a chunk has 17 to 32 rows and the call is large; both
// of a block's groups share the dequantised keys and values, but a small call waits longer for its
// larger join (us, with one and two: 60 x 8 queries of four heads per KV head over 1,500 keys 49.5, 35.5;
// 16 x 8 over 6,000 48.0, 40.0; 60 x 8 over 300 26.4, 18.5; 4 x 8 over 14,000 33.3, 34.6; 30 x 8 over 100
// 11.2, 12.3. Longer chunks gain less: 16 x 16 over 2,000 32.3 in the prefill kernel, 30.2).
static int nd_groups(int H, int num_reqs, int rows, int max_seq) {
  if (rows <= kNDRows || rows > 2 * kNDRows) return 1;
  const int64_t items = (int64_t)num_reqs * H * 2, steps = (max_seq + kNDStep - 1) / kNDStep;
  return items > nd_target() || items * steps > kNDWideWork ? 2 : 1;
}

// Rows of a (request, KV head) per query position at most, whatever the KV heads: the sizes below grow
// with every argument, so that layers of unlike heads share a workspace.
static int nd_most_rows(int HQ) { return std::min(HQ, 16); }

int64_t nibble_decode_workspace_bytes(int H, int HQ, int num_reqs, int max_seq) {
  if (num_reqs == 0) return 256;
  const int64_t pairs = (int64_t)nd_slice(H, 1, num_reqs) * H;
  return kCounterBytes + nd_parts(pairs, max_seq) * nd_most_rows(HQ) * (kD + 2) * 4;
}

// Chunks of at most 32 rows take this kernel, and longer ones while the whole call is short: it reads
// and dequantises a key for 16 rows, the prefill kernel for 128 to 384, but it has no tiles in LDS, no
// second launch and a smaller join. A call's items before any split are its (block, head) pairs, its
// work their steps. Measured here and there (us, four query heads and eight KV heads):
//   two blocks   30 x 8 queries over 100 keys 11.5, 13.5; 16 x 8 over 6,000 40.0, 61.3; 60 x 8 over 300
//     18.5, 24.3
//   more, one round of items, 24,000 steps of few of them   1 x 32 over 12,000 29.8, 35.2; 1 x 64 over
//     5,000 26.8, 28.2; 1 x 64 over 6,000 30.3, 30.3; 2 x 20 over 14,000 38.7, 37.2
//   or 17,000 of many   4 x 60 over 300 15.4, 18.1; 20 x 12 over 900 21.7, 34.0; 4 x 32 over 2,000 23.7,
//     24.5; 4 x 32 over 2,500 26.3, 25.6; 5 x 20 over 4,000 35.3, 30.6; two rounds: 30 x 16 over 300 25.6, 16.0
bool nibble_short_applies(int H, int HQ, int num_reqs, int max_q, int max_seq) {
  const int64_t rows = (int64_t)max_q * (HQ / H);
  if (rows > kNDShortRows) return false;
  const int64_t blocks = nd_blocks((int)rows, 1), steps = (max_seq + kNDStep - 1) / kNDStep;
  if (H * blocks > kMaxCounters) return false;
  if (blocks <= 2) return true;
  const int64_t items = (int64_t)num_reqs * H * blocks;
  return items <= nd_target() && items * steps <= (items <= nd_target() / 4 ? kNDFewWork : kNDShortWork);
}

// Bytes of partial results of such a chunk call at most, growing with every argument.
int64_t nibble_short_part_bytes(int H, int HQ, int num_reqs, int max_q, int max_seq) {
  const int rows = (int)std::min<int64_t>((int64_t)max_q * nd_most_rows(HQ), kNDShortRows);
  const int64_t pairs = std::min<int64_t>(
      std::min<int64_t>(num_reqs, kMaxCounters) * std::min(H, kMaxCounters) * nd_blocks(rows, 1), kMaxCounters);
  return nd_parts(pairs, max_seq) * std::min(rows, 2 * kNDRows) * (kD + 2) * 4;
}

template <bool CHUNK, int RG>
static int nd_launch(const NibDecodeArgs& a, unsigned grid, int q_dtype, hipStream_t st) {
  constexpr int smem = kNDWaves * kNDRows * RG * kD * 4;
  auto kernel = q_dtype == TTKV_DTYPE_F16 ? nibble_decode_kernel<TTKV_DTYPE_F16, CHUNK, RG>
                                          : nibble_decode_kernel<TTKV_DTYPE_BF16, CHUNK, RG>;
  if (RG > 1)
    if (int rc = raise_smem_limit((const void*)kernel, smem)) return rc;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kNDThreads), smem, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("nibble decode launch: ") + hipGetErrorString(e));
  return TTKV_OK;
}

// The arguments have been checked. max_q == 0: decode, of num_starts entries in qsl.
int nibble_decode_launch(int H, int HQ, float scale, const void* q, int q_dtype,
                         int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                         int64_t slot_stride, int bs, const int32_t* bt, int64_t bt_row_stride,
                         const int32_t* seq_lens, const int32_t* qsl, int num_starts,
                         const int32_t* req_index, int num_reqs, int max_q, int max_seq, void* out,
                         int out_dtype, int64_t out_row_stride, void* ws, int32_t* err,
                         hipStream_t st) {
  const int rows = HQ / H * std::max(max_q, 1), groups = nd_groups(H, num_reqs, rows, max_seq);
  const int blocks = nd_blocks(rows, groups);
  const int slice = nd_slice(H, blocks, num_reqs);
  const int64_t parts = nd_parts((int64_t)slice * H * blocks, max_seq);
  NibDecodeArgs a{};
  a.H = H;
  a.G = HQ / H;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.q = (const uint16_t*)q;
  a.q_row_stride = q_row_stride;
  a.page = page;
  a.tile_stride = kNibTile * slot_stride;
  a.num_blocks = (int)(n_slots / bs);
  a.tpb = bs / kNibTile;
  a.bt = bt;
  a.bt_row_stride = bt_row_stride;
  a.seq_lens = seq_lens;
  a.qsl = qsl;
  a.max_q = max_q;
  a.max_seq = max_seq;
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_row_stride = out_row_stride;
  a.part_rows = std::min(rows, kNDRows * groups);
  a.ws_cnt = (int*)ws;
  a.ws_o = (float*)((char*)ws + kCounterBytes);
  a.ws_ml = a.ws_o + parts * a.part_rows * kD;
  a.o_bytes = (uint32_t)(parts * a.part_rows * kD * 4);
  a.target = nd_target();
  a.err = err;
  for (int r0 = 0; r0 < num_reqs; r0 += slice) {
    a.num_reqs = std::min(slice, num_reqs - r0);
    a.num_starts = num_starts - r0;
    if (req_index) {
      a.req_index = req_index + r0;
    } else {
      a.seq_lens = seq_lens + r0;
      a.qsl = qsl + r0;
      a.bt = bt + (int64_t)r0 * bt_row_stride;
    }
    // an item per (block, head), and what the split ones have more
    const int64_t pairs = (int64_t)a.num_reqs * H * blocks;
    const unsigned grid = (unsigned)std::min(pairs + nd_target(), pairs * nd_max_chunks(max_seq));
    const int rc = max_q == 0    ? nd_launch<false, 1>(a, grid, q_dtype, st)
                   : groups == 1 ? nd_launch<true, 1>(a, grid, q_dtype, st)
                                 : nd_launch<true, 2>(a, grid, q_dtype, st);
    if (rc != TTKV_OK) return rc;
  }
  return TTKV_OK;
}

int nibble_decode_paged(int H, int HQ, int d, float scale, const void* q, int q_dtype,
                        int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                        int64_t slot_stride, int bs, const int32_t* bt, int64_t bt_row_stride,
                        int max_blocks, const int32_t* seq_lens, const int32_t* qsl, int num_starts,
                        int num_reqs, int max_seq, void* out, int out_dtype, int64_t out_row_stride, void* ws,
                        int64_t ws_bytes, int32_t* err, hipStream_t st) {
  if (int rc = nibble_check_read(H, HQ, d, q, q_dtype, q_row_stride, page, n_slots, slot_stride,
                                 bs, bt, max_blocks, seq_lens, qsl, num_reqs, max_seq, out,
                                 out_dtype, out_row_stride, err))
    return rc;
  if (H > kMaxCounters) return host_fail(TTKV_E_UNSUPPORTED, "too many KV heads");
  if (num_starts < num_reqs) return host_fail(TTKV_E_INVALID, "fewer query starts than requests");
  const int64_t need = nibble_decode_workspace_bytes(H, HQ, num_reqs, max_seq);
  if (!ws || ws_bytes < need || (uintptr_t)ws % 256)
    return host_fail(TTKV_E_WORKSPACE, "decode workspace needs " + std::to_string(need) +
                                           " bytes, 256-aligned");
  if (num_reqs == 0) return TTKV_OK;
  return nibble_decode_launch(H, HQ, scale, q, q_dtype, q_row_stride, page, n_slots, slot_stride,
                              bs, bt, bt_row_stride, seq_lens, qsl, num_starts, nullptr, num_reqs, 0, max_seq,
                              out, out_dtype, out_row_stride, ws, err, st);
}

}  // namespace ttkv
