// Attention of chunks of queries over the 4-bit cache (format: ttkv_nibble.h), causal. gfx950 / CDNA4.
//
// Flash attention. The rows of a (request, KV head) are its (query, query head) pairs, row = j G + p,
// so the G heads of a KV head share every key read. A workgroup of 8 waves holds 128, 256 or 384 of
// them (NG = 1 to 3 groups of 16 per wave) and walks a part of the request's keys in tiles of 64:
//   dequantise  waves 0..3 the tile's keys, waves 4..7 its values, 16 code bytes per thread, exactly
//               (ttkv_nibble.h) to fp16 in LDS: keys [token][dim], values transposed [dim][token] in
//               the order of the products' operands. Once per tile and 128 NG rows.
//   S^T = K Q^T on v_mfma_f32_16x16x32_f16, 32 tokens at a time: a key fragment read from LDS serves
//               the wave's NG groups. Lane column = row, so a row's softmax state is a lane's own.
//   softmax     as in the decode kernel: weights against a maximum that moves seldom, rounded to fp16
//               once, and their sum is of the rounded ones.
//   O^T += V^T P^T: the scores' layout is the weights' operand layout as it stands.
// One barrier per tile (two tile buffers); the next tile's codes are in flight in registers. Waves
// 0..3 compute before they dequantise and waves 4..7 after, so that the two waves of a SIMD are
// out of step and one's matrix products run under the other's vector work.
//
// Bound by instruction issue: per tile of 384 rows a SIMD's two waves have 192 products of 16 cycles and
// about 750 vector instructions (softmax, dequantisation) that take 4 cycles each beside them; 5,900
// cycles in all, with the clock near 1.95 GHz when every CU works. 1 x 2,048 queries of 32 heads over 12,345
// keys: 270 to 283 us by card, 1,050 TFLOP/s at best (a large library product 1,250); 4 x 256 of 24 heads
// over 7,656: 105 to 111.
//
// The keys of a row block are split over several workgroups where the batch has too few row blocks
// to fill the chip: the split comes from a plan that every workgroup computes alike from the lengths
// on the device. The parts' unnormalised results are joined by a second launch, 32 rows per workgroup
// (a row block's last part cannot join them itself in good time: one CU draws about 45 GB/s from what
// other XCDs wrote, and 384 rows of four parts are 0.8 MB; 1 x 512 queries with their own keys: 24 us
// for the join by the last part's workgroup).
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_nibble.h"

namespace ttkv {

constexpr int kNPThreads = 512;
constexpr int kNPWaves = 8;
constexpr int kNPTile = 64;        // keys per tile
constexpr int kNPPlanLanes = 4;    // requests per lane in the plan: 256 per launch
constexpr int kNPMaxSplit = 32;
constexpr int kNPMinTiles = 4;     // keys per part, in tiles (batches that are not searched)
constexpr int kNPSearch = 16;      // requests up to which the plan searches for the number of parts
// Lift of the weights (nib_max): a wave moves its maxima when any of its 48 rows has to. 1 x 2,048 over
// 12,345 and 4 x 256 over 7,656 took 270.4 and 105.9 us with 0 or 4, 274.5 and 107.7 with 6, 277.7 and 110.2
// with 8 (decode, bound by memory, 8 in the same time).
constexpr float kNPLift = 4.f;
// Rows of partial results a launch may leave, 66.0 MB: a workspace stays below 64 MiB, and calls that
// would leave more have row blocks enough to fill the chip with fewer parts.
constexpr int64_t kNPPartRows = 127000;
constexpr int kNPKBytes = kNPTile * kD * 2;
constexpr int kNPSmem = 4 * kNPKBytes;  // two buffers of keys and values

struct NibPrefillArgs {
  int H, G;
  float scale_log2;
  const uint16_t* q;
  int64_t q_row_stride;
  const uint8_t* page;
  int64_t tile_stride;
  int num_blocks, tpb;
  const int32_t* bt;
  int64_t bt_row_stride;
  const int32_t* seq_lens;
  const int32_t* qsl;
  const int32_t* req_index;
  int num_reqs, max_q, max_seq;
  uint32_t g_mul, g_shift;  // row / G = (2 row g_mul / 2^32) >> g_shift
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  uint8_t* ws_flag;       // [row blocks][RW / 32]: a piece that the join has to take
  struct NibPrefillJoin* ws_join;  // [row blocks]
  float* ws_o;   // [part rows][kD]
  float* ws_ml;  // [part rows][2]
  int64_t part_rows;
  int target, grid;
  int32_t* err;
};

// A row block whose keys were split: what its join needs.
struct NibPrefillJoin {
  int64_t part, q0;  // its first part row, the chunk's first query row
  int ns, rows;      // parts, and rows between them
  int row0, nrow, h;
};
constexpr int kNPJoinRows = 32;     // rows per workgroup of the join
constexpr int kNPJoinThreads = 256;

struct NibPrefillPlan {
  int r, h, rb, sp, ns;  // batch row, KV head, row block, key part and how many
  int n, Q, rows;        // keys, the chunk's queries, rows processed
  int block;             // the row block's number in the launch
  int64_t part, q0;      // first part row of the (request, head), the chunk's first query row
  bool none;
};

// Parts of a request's tiles, C of them each but for rounding (a reciprocal: near a whole quotient it may
// be one off, alike for every workgroup, and the parts are cut equal from their number; 1 for C >= tiles).
__device__ __forceinline__ int np_parts(int tiles, int C, float by_C) {
  return min(max(1, (int)((float)(tiles + C - 1) * by_C)), kNPMaxSplit);
}

// Tiles per part of `parts` parts of T tiles, rounded up or one more.
__device__ __forceinline__ int np_each(int T, int parts) {
  return max(1, (int)((float)T * __builtin_amdgcn_rcpf((float)parts) + 0.999f));
}

// An estimate of a launch's time in us, from what these kernels measured: a tile of a row block takes
// 1.55, 2.05 and 3.0 us with one, two and three groups of rows per wave (16 x 384 rows over 24,000 and
// 48,000 keys; eight KV heads, 256 CUs) and a block 5 us beside its tiles (4 x 1,432 rows over 180 keys,
// 8 heads); the items, of `load` tiles in all, take whole rounds of the CUs, and no less than the longest;
// a split costs its join and, per partial row, 520 bytes written and read.
__host__ __device__ inline float np_cost(int ng, float longest, float load, float items, float cus,
                                         float need) {
  const float tile = ng == 1 ? 1.55f : ng == 2 ? 2.05f : 3.0f;
#ifdef __HIP_DEVICE_COMPILE__
  const float rounds = ceilf(items * __builtin_amdgcn_rcpf(cus)), each = load * __builtin_amdgcn_rcpf(items);
#else
  const float rounds = ceilf(items / cus), each = load / items;
#endif
  return 5.f * rounds + tile * fmaxf(longest, rounds * each) + (need > 0.f ? 5.f + 1.5e-4f * need : 0.f);
}
// Tiles that a row block of a chunk of Q queries over T tiles has on average.
__host__ __device__ inline float np_mean_tiles(int T, int Q) {
  const float less = (float)Q / (2 * kNPTile);
  return (float)T - (less < 0.5f * T ? less : 0.5f * T);
}

// Parts of at least C tiles. For few requests every number of parts of the longest one, from 1 to 32, is
// priced, one per lane; many requests have row blocks enough, and get the shortest parts that spread
// their tiles over the target's workgroups. Either way the partial results have to fit the workspace,
// and the items the grid.
template <int RW>
__device__ __forceinline__ NibPrefillPlan np_plan(const NibPrefillArgs& a, int item) {
  constexpr int NG = RW / (16 * kNPWaves);
  const int lane = threadIdx.x & 63;
  int idx[kNPPlanLanes], n[kNPPlanLanes], q0[kNPPlanLanes], Q[kNPPlanLanes];
  int rows[kNPPlanLanes], tiles[kNPPlanLanes];
#pragma unroll
  for (int i = 0; i < kNPPlanLanes; ++i) {
    idx[i] = n[i] = q0[i] = Q[i] = 0;
    if (64 * i >= a.num_reqs) continue;
    const int r = lane + 64 * i;
    const bool on = r < a.num_reqs;
    idx[i] = on ? (a.req_index ? a.req_index[r] : r) : 0;
    n[i] = on ? a.seq_lens[idx[i]] : 0;
    q0[i] = on ? a.qsl[idx[i]] : 0;
    Q[i] = on ? a.qsl[idx[i] + 1] - q0[i] : 0;
  }
  float work = 0.f, most_work = 0.f;  // tiles of all row blocks: that they see, and of their requests
#pragma unroll
  for (int i = 0; i < kNPPlanLanes; ++i) {
    rows[i] = tiles[i] = 0;
    if (64 * i >= a.num_reqs) continue;
    const int nn = min(max(n[i], 0), a.max_seq);
    rows[i] = min(max(Q[i], 0), a.max_q) * a.G;
    tiles[i] = nn < Q[i] ? 1 : (nn + kNPTile - 1) / kNPTile;
    work += (float)((rows[i] + RW - 1) / RW) * np_mean_tiles(tiles[i], Q[i]);
    most_work += (float)((rows[i] + RW - 1) / RW) * (float)tiles[i];
  }
  int C;
  if (a.num_reqs <= kNPSearch) {
    const int most = wave_max_i(rows[0] > 0 ? tiles[0] : 1);
    const int parts = (lane & (kNPMaxSplit - 1)) + 1, c = np_each(most, parts);
    float longest = 0.f, items = 0.f, need = 0.f;
    const float by_c = __builtin_amdgcn_rcpf((float)c);
    const int blocks = (rows[0] + RW - 1) / RW;
    work = wave_sum(work) * (float)a.H;
    // a half wave takes every other request, four of them at a time (lanes past the last hold none)
    for (int r = 0; r < a.num_reqs; r += 8) {
#pragma unroll
      for (int k = r; k < r + 8; k += 2) {
        auto of = [&](int v) {
          const int even = __builtin_amdgcn_readlane(v, k), odd = __builtin_amdgcn_readlane(v, k + 1);
          return lane < 32 ? even : odd;
        };
        const int T = of(tiles[0]), rw = of(rows[0]);
        const float ns = (float)np_parts(T, c, by_c);
        longest = fmaxf(longest, rw > 0 ? (float)T * __builtin_amdgcn_rcpf(ns) : 0.f);
        items += (float)of(blocks) * ns;
        need += ns > 1.f ? (float)rw * ns : 0.f;
      }
    }
    longest = fmaxf(longest, __shfl_xor(longest, 32));
    items += __shfl_xor(items, 32);
    need += __shfl_xor(need, 32);
    items *= (float)a.H;
    need *= (float)a.H;
    const bool fits = need <= (float)a.part_rows && items <= (float)a.grid;  // (one part always does)
    const float us = np_cost(NG, longest, work, fmaxf(items, 1.f), (float)a.target, need);
    const int price = fits ? (int)fminf(us * 16.f, 3e7f) : 0x3ffffff;  // sixteenths
    const int best = -wave_max_i(-(price * 32 + parts - 1)) & 31;
    C = np_each(most, best + 1);
  } else {
    // at most work / C items beside one per row block: within the grid
    C = max(kNPMinTiles, (int)ceilf(wave_sum(most_work) * (float)a.H / (float)a.target));
    while (true) {
      float need = 0.f;
#pragma unroll
      for (int i = 0; i < kNPPlanLanes; ++i) {
        const int ns = np_parts(tiles[i], C, __builtin_amdgcn_rcpf((float)C));
        need += ns > 1 ? (float)rows[i] * (float)ns : 0.f;
      }
      need = wave_sum(need) * (float)a.H;
      if (need <= (float)a.part_rows) break;
      C += (C >> 2) + 1;
    }
  }
  NibPrefillPlan P{};
  P.none = true;
  P.h = item % a.H;
  const int it = item / a.H;
  int carry = 0, blocks = 0, prows = 0;
  const float by_C = __builtin_amdgcn_rcpf((float)C);
#pragma unroll
  for (int i = 0; i < kNPPlanLanes; ++i) {
    if (64 * i >= a.num_reqs) break;
    const int rb = (rows[i] + RW - 1) / RW, ns = np_parts(tiles[i], C, by_C), items = rb * ns;
    const int pr = ns > 1 ? rows[i] * ns : 0;
    const int incl = nib_scan(items), ex = carry + incl - items;
    const int bincl = nib_scan(rb), pincl = nib_scan(pr);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(items > 0 && ex <= it && it < ex + items);
    if (hit) {
      const int ln = __builtin_ctzll(hit);
      const int local = it - __builtin_amdgcn_readlane(ex, ln);
      const int nrb = __builtin_amdgcn_readlane(rb, ln);
      P.none = false;
      P.r = __builtin_amdgcn_readlane(idx[i], ln);
      P.n = __builtin_amdgcn_readlane(n[i], ln);
      P.Q = __builtin_amdgcn_readlane(Q[i], ln);
      P.q0 = __builtin_amdgcn_readlane(q0[i], ln);
      P.rows = __builtin_amdgcn_readlane(rows[i], ln);
      P.ns = __builtin_amdgcn_readlane(ns, ln);
      P.rb = nrb - 1 - local / P.ns;  // the last rows see the most keys: first
      P.sp = local % P.ns;
      P.block = (blocks + __builtin_amdgcn_readlane(bincl - rb, ln) + P.rb) * a.H + P.h;
      P.part = (int64_t)(prows + __builtin_amdgcn_readlane(pincl - pr, ln)) * a.H +
               (int64_t)P.h * P.ns * P.rows;
    }
    carry += __builtin_amdgcn_readlane(incl, 63);
    blocks += __builtin_amdgcn_readlane(bincl, 63);
    prows += __builtin_amdgcn_readlane(pincl, 63);
  }
  return P;
}

// Tile buffers, by byte address: keys [token][16 chunks of 8 dims], 256 bytes a token, then values
// [dim][8 chunks of 8 token slots], 128 bytes a dim. A row's 16-byte chunks are exchanged by XOR with
// the row's number, so that a fragment's 16 rows lie in distinct banks; chunk 4 s + q4 of the row is
// then the address of chunk q4 with s << 6 exchanged in. Addresses are formed from the tile's buffer
// each time, since kept ones spill the matrix operands.
constexpr uint32_t kNPBuf = 2 * kNPKBytes;  // bytes of a tile
template <typename T>
__device__ __forceinline__ T np_get(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)(uintptr_t)at;
}
template <typename T>
__device__ __forceinline__ void np_put(uint32_t at, T v) {
  *(__attribute__((address_space(3))) T*)(uintptr_t)at = v;
}
// Barrier for LDS alone: global loads stay in flight across it.
__device__ __forceinline__ void np_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// row / G for rows below 2^31, with g_mul = ceil(2^(31 + g_shift) / G) and 2^g_shift >= G: row times
// what the rounding adds is below 2^(31 + g_shift).
__device__ __forceinline__ int np_by_g(const NibPrefillArgs& a, int row) {
  return (int)(__umulhi(2u * (uint32_t)row, a.g_mul) >> a.g_shift);
}
// Row `row` of a chunk that begins at query row q0, KV head h, in the query or the output.
__device__ __forceinline__ int64_t np_row_at(const NibPrefillArgs& a, int64_t q0, int h, int row,
                                             int64_t stride) {
  const int j = np_by_g(a, row);
  return (q0 + j) * stride + (int64_t)(h * a.G + row - j * a.G) * kD;
}
template <int QDT, int NG>
__global__ __launch_bounds__(kNPThreads, 2) void nibble_prefill_kernel(NibPrefillArgs a) {
  constexpr int RW = kNPWaves * 16 * NG;
  extern __shared__ __align__(1024) unsigned char smem[];  // (the XORs above count on whole rows)
  __shared__ uint32_t nan_sh[2][kNPTile / 4];  // per token of a masked tile: its groups that are NaN
  __shared__ int bad_sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const NibPrefillPlan P = np_plan<RW>(a, blockIdx.x);
  if (P.none) return;
  const int h = P.h;
  const int n = min(max(P.n, 0), a.max_seq);
  const int64_t q0 = P.q0;
  const int nrow = min(RW, P.rows - P.rb * RW);
  if (tid == 0 && h == 0 && P.sp == 0 && P.rb == 0 &&
      (P.n > a.max_seq || P.Q > a.max_q || n < P.Q))
    atomicOr(a.err, TTKV_ERR_SEQ_LEN);
  if (n < P.Q) {  // fewer keys than queries
    for (int e = tid; e < nrow * kD; e += kNPThreads) {
      const int row = P.rb * RW + e / kD;
      store_act(a.out, a.out_dtype,
                np_row_at(a, q0, h, row, a.out_row_stride) + e % kD, NAN);
    }
    return;
  }
  const int col = lane & 15, q4 = lane >> 4;
  const int row0 = P.rb * RW + wv * 16 * NG;  // the wave's first row
  const bool active = row0 < P.rows;
  const int p0 = n - P.Q;  // position of query 0
  const int see_min = p0 + np_by_g(a, row0),
            see_max = p0 + np_by_g(a, min(row0 + 16 * NG - 1, P.rows - 1));

  // the block's tiles and this part of them
  const int tiles = (p0 + np_by_g(a, P.rb * RW + nrow - 1)) / kNPTile + 1;
  const int t0 = (int)((int64_t)tiles * P.sp / P.ns), t1 = (int)((int64_t)tiles * (P.sp + 1) / P.ns);
  const int wg_see = p0 + np_by_g(a, P.rb * RW);  // last key that every row of the block sees
  const uint8_t* base = a.page + (int64_t)h * kNibRecord;
  const int32_t* bt = a.bt + (int64_t)P.r * a.bt_row_stride;
  const NibMasks masks = nib_masks();
  const uint32_t smem_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const uint32_t krow = smem_at + col * 256 + ((q4 ^ col) << 4);  // token col, chunk q4
  const bool values = wv >= 4;
  const int tt = wv & 3;  // this wave's record of a tile
  const int last_rec = (n - 1) / kNibTile;
  bool bad = false;
  float most = kNibMost;  // below every sum from the wave's first far maximum on
  int ids = 0;
  auto fetch_ids = [&](int t) {  // record ids of the next 64 tiles, one per lane (-1: bad block)
    const int rec = min(4 * (t + lane) + tt, last_rec);
    const int b = rec / a.tpb, id = bt[b];
    ids = (uint32_t)id < (uint32_t)a.num_blocks ? id * a.tpb + rec - b * a.tpb : -1;
  };
  u32x4 code;
  u32x4 par[2];
  int ids_at = t0;
  auto load = [&](int t) {
    if (t >= t1) return;
    if (t - ids_at >= 64) {
      ids_at = t;
      fetch_ids(t);
    }
    const int id = __builtin_amdgcn_readlane(ids, t - ids_at);
    bad |= id < 0;
    const uint8_t* rec = base + (int64_t)max(id, 0) * a.tile_stride;
    if (values) {
      code = *gbl((const u32x4*)(rec + kNibV + 16 * lane));
      par[0] = *gbl((const u32x4*)(rec + kNibVp + 32 * q4));
      par[1] = *gbl((const u32x4*)(rec + kNibVp + 32 * q4 + 16));
    } else {
      code = *gbl((const u32x4*)(rec + 16 * lane));
      const u32x2v kp = *gbl((const u32x2v*)(rec + kNibKp + 8 * col));
      par[0][0] = kp[0];
      par[0][1] = kp[1];
    }
  };
  if (t0 < t1) fetch_ids(t0);
  // The query rows are asked for behind the first tile's record ids, and wait behind its codes.
  NibRow qrow[NG];
  int lim[NG];  // last key the lane's row sees
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    const int row = min(row0 + 16 * gr + col, P.rows - 1);
    lim[gr] = p0 + np_by_g(a, row);
    qrow[gr] = nib_load_row(a.q + np_row_at(a, q0, h, row, a.q_row_stride), q4);
  }
  load(t0);
  half8 qf[NG][4];
  float qs[NG], m[NG], l[NG];
  float4v acc[NG][8];
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) {
    nib_query<QDT>(qrow[gr], a.scale_log2, true, qf[gr], qs[gr]);
    m[gr] = kNibNone;
    l[gr] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[gr][i] = float4v{};
  }
  auto dequant_keys = [&](int t) {
    if (t >= t1) return;
    const uint32_t at = krow + (t & 1) * kNPBuf + tt * (16 * 256);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const half2v zz = nib_biased(par[0][g >> 1], masks), sg = nib_scales(par[0][g >> 1]);
      const half2v zb = {zz[g & 1], zz[g & 1]}, ss = {sg[g & 1], sg[g & 1]};
      half8 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const half2v v = nib_pair(code[g], j, zb, ss, masks);
        o[2 * j] = v[0];
        o[2 * j + 1] = v[1];
      }
      np_put(at ^ (g << 6), o);
    }
  };
  auto dequant_values = [&](int t) {
    if (t >= t1) return;
    const int tok = t * kNPTile + 16 * tt + 4 * q4;  // the lane's four tokens
    if ((t + 1) * kNPTile - 1 > wg_see) {
      // Some row does not see all of this tile. A weight of 0 must not meet a NaN: values past the
      // last key become 0, and a group that is NaN becomes 0 too and is noted for the rows that see it.
      uint32_t note = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int at = 2 * (g & 1) + (i >> 1);
          const uint32_t w = par[g >> 1][at], p = i & 1 ? w >> 16 : w & 0xffffu;
          const bool nan = (p & 0x7c00u) == 0x7c00u;
          if (tok + i >= n || nan) {
            par[g >> 1][at] = w & (i & 1 ? 0x0000ffffu : 0xffff0000u);
            note |= tok + i < n ? 1u << (8 * i + g) : 0u;
          }
        }
      if (col == 0) nan_sh[t & 1][4 * tt + q4] = note;
    }
    // chunk 4 (tt / 2) + q4 of dim 2 col + b, its half tt % 2
    const uint32_t vb = smem_at + (t & 1) * kNPBuf + kNPKBytes + 8 * (tt & 1);
    uint32_t at[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int dim = 2 * col + b;
      at[b] = vb + dim * 128 + (((4 * (tt >> 1) + q4) ^ (dim & 7)) << 4);
    }
#pragma unroll
    for (int quad = 0; quad < 2; ++quad)
#pragma unroll
      for (int gg = 0; gg < 2; ++gg) {
        const int g = 2 * quad + gg;
        half4 o[2];
#pragma unroll
        for (int pair = 0; pair < 2; ++pair) {
          const uint32_t p2 = par[g >> 1][2 * (g & 1) + pair];
          const half2v zb = nib_biased(p2, masks), ss = nib_scales(p2);
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const half2v v = nib_pair(code[2 * pair + quad], 2 * gg + b, zb, ss, masks);
            o[b][2 * pair] = v[0];
            o[b][2 * pair + 1] = v[1];
          }
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) np_put(at[b] + 32 * 128 * g, o[b]);
      }
  };
  auto compute = [&](int t) {
    if (!active || t * kNPTile > see_max) return;
    const uint32_t kb = krow + (t & 1) * kNPBuf;
    const uint32_t vb = smem_at + (t & 1) * kNPBuf + kNPKBytes + col * 128 + ((q4 ^ (col & 7)) << 4);
    const bool masked = (t + 1) * kNPTile - 1 > see_min;
    // Fragments are asked for a few products ahead (rings of four and three, the order pinned by the
    // scheduling barriers): with their loads next to their use, every third product waited for LDS.
    auto key_frag = [&](int ks, int f) {  // f: tokens 16 (f / 4), dims 32 (f % 4)
      return np_get<half8>((kb ^ ((f & 3) << 6)) + (32 * ks + 16 * (f >> 2)) * 256);
    };
    auto value_frag = [&](int ks, int db) {
      return np_get<half8>((vb ^ (ks << 6)) + 16 * 128 * db);
    };
    half8 kf[4], vf[3];
#pragma unroll
    for (int f = 0; f < 4; ++f) kf[f] = key_frag(0, f);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      float4v sc[NG][2];
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) sc[gr][0] = sc[gr][1] = float4v{};
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int f = 0; f < 8; ++f) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          sc[gr][f >> 2] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[f & 3], qf[gr][f & 3], sc[gr][f >> 2], 0, 0, 0);
        if (f < 4) kf[f & 3] = key_frag(ks, f + 4);
        else if (f < 7) vf[f - 4] = value_frag(ks, f - 4);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      if (masked) {
        const int tok = t * kNPTile + 32 * ks + 4 * q4;
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
#pragma unroll
          for (int tg = 0; tg < 2; ++tg)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (tok + 16 * tg + i > lim[gr]) sc[gr][tg][i] = -INFINITY;
      }
      // Weights against the maximum as it stands. It has to move only where a weight leaves fp16 and
      // so makes its lane's sum of eight infinite (or NaN): the scores' own maximum is taken in that
      // case alone, or where a row of the wave has a far one.
      half8 pf[NG];
      float sum[NG];
      auto weights = [&](int gr, bool apart) {
        sum[gr] = 0.f;
        auto exponent = [&](float s) {
          const float e = fmaf(s, qs[gr], -m[gr]);
          return apart ? nib_apart(s, qs[gr], m[gr]) : e;
        };
#pragma unroll
        for (int tg = 0; tg < 2; ++tg)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            // the one rounding on the way to the output, to the value product's 16-bit operand (low
            // parts in a second product would double it); the sum takes the rounded weights
            const half2v p = {(_Float16)fast_exp2(exponent(sc[gr][tg][i])),
                              (_Float16)fast_exp2(exponent(sc[gr][tg][i + 1]))};
            sum[gr] = __builtin_amdgcn_fdot2(p, half2v{(_Float16)1.f, (_Float16)1.f}, sum[gr], false);
            pf[gr][4 * tg + i] = p[0];
            pf[gr][4 * tg + i + 1] = p[1];
          }
      };
      bool fits = true;
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) {
        weights(gr, false);
        fits &= sum[gr] <= most;
      }
      if (__builtin_amdgcn_ballot_w64(!fits)) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr) {
          float mt = -INFINITY;
#pragma unroll
          for (int tg = 0; tg < 2; ++tg)
#pragma unroll
            for (int i = 0; i < 4; ++i) mt = fmaxf(mt, sc[gr][tg][i]);
          const float mn = nib_max(m[gr], cross_row_max(mt * qs[gr]), kNPLift);
          const float f = exp2f(m[gr] - mn);
          m[gr] = mn;
          l[gr] *= f;
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[gr][i] *= f;
          weights(gr, nib_far(mn));
          if (__builtin_amdgcn_ballot_w64(nib_far(mn))) most = -1.f;
        }
      }
#pragma unroll
      for (int gr = 0; gr < NG; ++gr) l[gr] += sum[gr];
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int db = 0; db < 8; ++db) {
#pragma unroll
        for (int gr = 0; gr < NG; ++gr)
          acc[gr][db] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[db % 3], pf[gr], acc[gr][db], 0, 0, 0);
        if (db < 5) vf[db % 3] = value_frag(ks, db + 3);
        if (db >= 4 && ks == 0) kf[db - 4] = key_frag(1, db - 4);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if ((t + 1) * kNPTile - 1 > wg_see) {  // NaN groups of a tile with masked keys
      const uint32_t mine = nan_sh[t & 1][lane & 15];
      if (__builtin_amdgcn_ballot_w64(mine != 0)) {
        for (int k = 0; k < kNPTile; ++k) {
          const uint32_t note = (nan_sh[t & 1][k >> 2] >> (8 * (k & 3))) & 15u;
          if (!note) continue;
#pragma unroll
          for (int gr = 0; gr < NG; ++gr)
#pragma unroll
            for (int db = 0; db < 8; ++db)
              if ((note >> (db >> 1) & 1) && t * kNPTile + k <= lim[gr]) acc[gr][db] += NAN;
        }
      }
    }
  };

  if (tid == 0) bad_sh = 0;
  if (t0 < t1) {
    if (!values) {
      dequant_keys(t0);
      load(t0 + 1);
    }
    // The value waves enter the loop half a turn early: they dequantise tile t + 1 (at t = t0 - 1 the
    // first tile) before they compute tile t, the key waves after it.
    for (int t = t0 - 1; t < t1; ++t) {
      if (values) {
        dequant_values(t + 1);
        load(t + 2);
      }
      if (t >= t0) compute(t);
      if (!values && t >= t0) {
        dequant_keys(t + 1);
        load(t + 2);
      }
      np_barrier();
    }
  } else {
    np_barrier();
  }
  if (bad) {
    bad_sh = 1;
    if (lane == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
  }
  __syncthreads();
  const bool nan_rows = bad_sh != 0;
#pragma unroll
  for (int gr = 0; gr < NG; ++gr) l[gr] = nan_rows ? NAN : cross_row_sum(l[gr]);

  if (P.ns == 1) {
    if (!active) return;
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const int row = row0 + 16 * gr + col;
      if (row >= P.rows) continue;
      const float inv = 1.f / l[gr];
      const int64_t at = np_row_at(a, q0, h, row, a.out_row_stride);
#pragma unroll
      for (int db = 0; db < 8; ++db)
        store_act4(a.out, a.out_dtype, at + 16 * db + 4 * q4, acc[gr][db] * inv, true);
    }
    return;
  }
  if (active) {
#pragma unroll
    for (int gr = 0; gr < NG; ++gr) {
      const int row = row0 + 16 * gr + col;
      if (row >= P.rows) continue;
      const int64_t pr = P.part + (int64_t)P.sp * P.rows + row;
#pragma unroll
      for (int db = 0; db < 8; ++db)
        *gblw((float4v*)(a.ws_o + pr * kD + 16 * db + 4 * q4)) = acc[gr][db];
      if (q4 == 0) *gblw((float2v*)(a.ws_ml + 2 * pr)) = float2v{m[gr], l[gr]};
    }
  }
  if (P.sp == 0) {
    if (tid == 0)
      a.ws_join[P.block] = NibPrefillJoin{P.part + P.rb * RW, q0, P.ns, P.rows, P.rb * RW, nrow, h};
    constexpr int PIECES = RW / kNPJoinRows;
    if (tid < PIECES && tid * kNPJoinRows < nrow) a.ws_flag[P.block * PIECES + tid] = 1;
  }
}

// Joins the parts of 32 rows: out = sum_s w_s o_s / sum_s w_s l_s, w_s = 2^(m_s - max m). Its flag is
// set by the attention launch and cleared here, so the flags are zero between calls. A chain of round
// trips to memory (flag, sums, parts), so parts are asked for B at a time, without a branch between them
// (past one the compiler waits for all that is in flight), the first before the sums are there.
template <int RW>
__global__ __launch_bounds__(kNPJoinThreads) void nibble_join_kernel(NibPrefillArgs a) {
  constexpr int PIECES = RW / kNPJoinRows;
  __shared__ float2v wgt[kNPMaxSplit][kNPJoinRows];  // weight, sum
  __shared__ float inv_sh[kNPJoinRows];
  const int tid = threadIdx.x;
  const int block = blockIdx.x / PIECES, piece = blockIdx.x % PIECES;
  uint8_t* flag = a.ws_flag + blockIdx.x;
  const uint8_t on = *flag;
  const NibPrefillJoin J = a.ws_join[block];  // (meaningless without the flag)
  if (!on) return;
  const int r0 = piece * kNPJoinRows, nr = min(kNPJoinRows, J.nrow - r0);
  const int64_t first = J.part + r0;
  constexpr int UNITS = kNPJoinRows * kD / 4 / kNPJoinThreads;  // four floats each
  const int d = 4 * (tid % (kD / 4));
  auto join = [&](auto b_c) {
    constexpr int B = decltype(b_c)::value;
    float4v x[B][UNITS], o[UNITS];
    auto fetch = [&](int s0) {
#pragma unroll
      for (int k = 0; k < B; ++k)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const int row = min((tid + u * kNPJoinThreads) / (kD / 4), nr - 1);
          x[k][u] = *gbl((const float4v*)(
              a.ws_o + (first + (int64_t)min(s0 + k, J.ns - 1) * J.rows + row) * kD + d));
        }
    };
    fetch(0);
    for (int e = tid; e < J.ns * kNPJoinRows; e += kNPJoinThreads) {
      const int s = e / kNPJoinRows, row = min(e % kNPJoinRows, nr - 1);
      wgt[s][e % kNPJoinRows] =
          *gbl((const float2v*)(a.ws_ml + 2 * (first + (int64_t)s * J.rows + row)));
    }
    __syncthreads();
    if (tid == 0) *flag = 0;
    if (tid < kNPJoinRows) {
      float mm = kNibNone, ll = 0.f;
#pragma unroll 8
      for (int s = 0; s < J.ns; ++s) mm = fmaxf(mm, wgt[s][tid][0]);
#pragma unroll 8
      for (int s = 0; s < J.ns; ++s) {
        const float2v ml = wgt[s][tid];
        const float w = exp2f(ml[0] - mm);
        ll += w * ml[1];
        wgt[s][tid][0] = w;
      }
      inv_sh[tid] = 1.f / ll;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < UNITS; ++u) o[u] = float4v{};
    for (int s0 = 0; s0 < J.ns; s0 += B) {
      if (s0) fetch(s0);
#pragma unroll
      for (int k = 0; k < B; ++k) {
        const int s = min(s0 + k, J.ns - 1);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const float w = wgt[s][(tid + u * kNPJoinThreads) / (kD / 4)][0];
          o[u] += x[k][u] * (s0 + k < J.ns ? w : 0.f);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int row = (tid + u * kNPJoinThreads) / (kD / 4);
      if (row >= nr) break;
      const int rr = J.row0 + r0 + row;
      store_act4(a.out, a.out_dtype,
                 np_row_at(a, J.q0, J.h, rr, a.out_row_stride) + d,
                 o[u] * inv_sh[row], true);
    }
  };
  if (J.ns == 2) join(std::integral_constant<int, 2>{});
  else if (J.ns <= 4) join(std::integral_constant<int, 4>{});
  else join(std::integral_constant<int, 8>{});
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
  if (max_seq > (1 << 26))
    return host_fail(TTKV_E_UNSUPPORTED, "max_seq_len beyond 2^26");
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

// Requests per launch: the plan's lanes and a flag per 32 rows of every row block and head; with no
// room for one request's flags, its keys are not split.
struct NibPrefillSlice {
  int ng, reqs;
  int64_t blocks;  // row blocks of a launch, at most
  bool split;
};
// Parts of a request at most.
static int64_t np_max_parts(int max_seq) {
  const int64_t tiles = (max_seq + kNPTile - 1) / kNPTile;
  return std::min<int64_t>(kNPMaxSplit, tiles);
}

static NibPrefillSlice np_slice(int H, int HQ, int num_reqs, int max_q, int max_seq) {
  const int64_t rows = (int64_t)max_q * (HQ / H), cus = device_cu_count();
  const int T = (max_seq + kNPTile - 1) / kNPTile;
  NibPrefillSlice best{};
  float least = 0.f;
  int parts = 1;
  for (int ng = 3; ng >= 1; --ng) {
    NibPrefillSlice s{};
    s.ng = ng;
    const int64_t rw = kNPWaves * 16 * ng;
    const int64_t per = (rows + rw - 1) / rw * H;              // row blocks of one request
    const int64_t flags = kCounterBytes / (rw / kNPJoinRows);  // row blocks the flags serve
    s.split = per <= flags && np_max_parts(max_seq) > 1;
    s.reqs = std::min(num_reqs, kNPPlanLanes * 64);
    if (s.split) s.reqs = (int)std::min<int64_t>(s.reqs, flags / per);
    s.blocks = per * s.reqs;
    // the plan's search with every request at its longest
    const float load = (float)(per * num_reqs) * np_mean_tiles(T, max_q);
    for (int k = 1; k <= (s.split ? np_max_parts(max_seq) : 1); ++k) {
      const int64_t need = k > 1 ? rows * H * num_reqs * k : 0;
      if (k > 1 && (need > kNPPartRows || per * num_reqs * (k - 1) > cus)) break;
      const float us = np_cost(ng, (float)((T + k - 1) / k), load, (float)(per * num_reqs * k), (float)cus,
                               (float)need);
      if (best.ng == 0 || us < least) {
        best = s;
        least = us;
        parts = k;
      }
    }
  }
  // One request whose keys need no split at its longest: no second launch (1 x 256 over 256: 20.2
  // us, 18.7 so).
  if (num_reqs == 1 && parts == 1) best.split = false;
  return best;
}

static int64_t np_part_rows(int HQ, int reqs, int max_q, int max_seq) {
  return std::min(kNPPartRows, np_max_parts(max_seq) * std::min<int64_t>(reqs, kNPPartRows) *
                                   std::min<int64_t>(max_q, kNPPartRows) * HQ);
}

static int64_t np_join_bytes(const NibPrefillSlice& s) {
  return (s.blocks * (int64_t)sizeof(NibPrefillJoin) + 255) / 256 * 256;
}

// An upper bound that grows with every argument, so that a workspace for the largest batch serves the
// others: a join record for every row block that the flags can serve, of 128 rows each (a request has
// max_q HQ / 128 of them and, for what its heads round up, less than H more), and the parts of either
// kernel.
int64_t nibble_prefill_workspace_bytes(int H, int HQ, int num_reqs, int max_q, int max_seq) {
  if (num_reqs == 0 || max_q == 0) return 256;
  const int64_t rw = kNPWaves * 16, most = kCounterBytes / (rw / kNPJoinRows);
  const int64_t per = std::min((int64_t)max_q * HQ / rw + H, most);
  const int64_t blocks = std::min(per * std::min<int64_t>(num_reqs, most), most);
  const int64_t joins = (blocks * (int64_t)sizeof(NibPrefillJoin) + 255) / 256 * 256;
  const int64_t parts = np_part_rows(HQ, num_reqs, max_q, max_seq) * (kD + 2) * 4;
  return kCounterBytes + std::max(joins + parts, nibble_short_part_bytes(H, HQ, num_reqs, max_q, max_seq));
}

template <int QDT, int NG>
static int np_launch(const NibPrefillArgs& a, unsigned grid, unsigned blocks, hipStream_t st) {
  if (int rc = raise_smem_limit((const void*)nibble_prefill_kernel<QDT, NG>, kNPSmem)) return rc;
  hipLaunchKernelGGL((nibble_prefill_kernel<QDT, NG>), dim3(grid), dim3(kNPThreads), kNPSmem, st, a);
  if (a.part_rows) {
    constexpr int RW = kNPWaves * 16 * NG;
    hipLaunchKernelGGL((nibble_join_kernel<RW>), dim3(blocks * (RW / kNPJoinRows)),
                       dim3(kNPJoinThreads), 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return host_fail(TTKV_E_LAUNCH, std::string("nibble prefill launch: ") + hipGetErrorString(e));
  return TTKV_OK;
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
  if (nibble_short_applies(H, HQ, num_reqs, max_q, max_seq))
    return nibble_decode_launch(H, HQ, scale, q, q_dtype, q_row_stride, page, n_slots, slot_stride,
                                bs, bt, bt_row_stride, seq_lens, qsl, 0, req_index, num_reqs, max_q,
                                max_seq, out, out_dtype, out_row_stride, ws, err, st);
  const NibPrefillSlice s = np_slice(H, HQ, num_reqs, max_q, max_seq);
  const int64_t items =
      s.split ? std::min(s.blocks + device_cu_count() + 8, s.blocks * np_max_parts(max_seq)) : s.blocks;
  if (items > 0x7fffffff) return host_fail(TTKV_E_INVALID, "too many queries for one call");
  NibPrefillArgs a{};
  a.H = H;
  a.G = HQ / H;
  while ((1 << a.g_shift) < a.G) ++a.g_shift;
  a.g_mul = (uint32_t)(((1ull << (31 + a.g_shift)) + a.G - 1) / a.G);
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
  a.part_rows = s.split ? np_part_rows(HQ, s.reqs, max_q, max_seq) : 0;
  a.ws_flag = (uint8_t*)ws;
  a.ws_join = (NibPrefillJoin*)((char*)ws + kCounterBytes);
  a.ws_o = (float*)((char*)ws + kCounterBytes + np_join_bytes(s));
  a.ws_ml = a.ws_o + a.part_rows * kD;
  a.target = device_cu_count();  // a workgroup fills a CU
  a.grid = (int)items;
  a.err = err;
  for (int r0 = 0; r0 < num_reqs; r0 += s.reqs) {
    a.num_reqs = std::min(s.reqs, num_reqs - r0);
    if (req_index) {
      a.req_index = req_index + r0;
    } else {
      a.seq_lens = seq_lens + r0;
      a.qsl = qsl + r0;
      a.bt = bt + (int64_t)r0 * bt_row_stride;
    }
    const unsigned grid = (unsigned)items;
    const bool f16 = q_dtype == TTKV_DTYPE_F16;
    int rc = TTKV_OK;
    switch (s.ng) {
      case 1: rc = f16 ? np_launch<TTKV_DTYPE_F16, 1>(a, grid, (unsigned)s.blocks, st) : np_launch<TTKV_DTYPE_BF16, 1>(a, grid, (unsigned)s.blocks, st); break;
      case 2: rc = f16 ? np_launch<TTKV_DTYPE_F16, 2>(a, grid, (unsigned)s.blocks, st) : np_launch<TTKV_DTYPE_BF16, 2>(a, grid, (unsigned)s.blocks, st); break;
      default: rc = f16 ? np_launch<TTKV_DTYPE_F16, 3>(a, grid, (unsigned)s.blocks, st) : np_launch<TTKV_DTYPE_BF16, 3>(a, grid, (unsigned)s.blocks, st); break;
    }
    if (rc != TTKV_OK) return rc;
  }
  return TTKV_OK;
}

}  // namespace ttkv
