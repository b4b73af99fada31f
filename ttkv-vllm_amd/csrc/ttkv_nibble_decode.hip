// Decode attention over the 4-bit cache (format: ttkv_nibble.h): one query per request. gfx950 / CDNA4.
//
// Work item = (request, KV head, chunk of the request's 32-token steps), one workgroup of 4 waves
// that take the chunk's steps in turn. The chunk length comes from a plan that every workgroup
// computes alike from the batch's lengths: the shortest that spreads the batch's steps over the
// resident workgroups, so a ragged batch fills the chip by its total work. Items of a (request,
// head) leave unnormalised partials in the workspace; the last to arrive joins them.
//
// One step of a wave, two tiles of 16 tokens:
//   S^T [token, query] = K Q^T, four v_mfma_f32_16x16x32_f16 per tile: a lane's 16 key code bytes are
//     its A operand of all four (token lane % 16, 8 dims of each group of 32), unpacked by a shift and
//     a mask per pair and dequantised exactly in packed fp16; the query is the B operand, held in
//     registers. The 16 columns are the G query heads (the rest are zero).
//   softmax in the result's own registers: lane column = query, 8 tokens of it; the running maximum
//     moves only when a score exceeds it by 8 (weights stay below 2^8), so most steps need no
//     exchange between lanes, and the sum stays per lane until the end.
//   O^T [dim, query] += V^T P^T, eight MFMAs: the scores' layout is the B operand's as it stands, and
//     a lane's 16 value code bytes per tile are its A operand of all eight (a dim pair of each group,
//     four tokens). The result's column is the query again, so the rescale is a factor of the lane's.
// Bytes per step 4,608; the two register sets keep the next step's loads in flight.
#include <math.h>

#include "ttkv_host.h"
#include "ttkv_nibble.h"

namespace ttkv {

constexpr int kNDThreads = 256;
constexpr int kNDWaves = 4;
constexpr int kNDStep = 2 * kNibTile;  // tokens per wave step
constexpr int kNDPlanLanes = 4;        // requests per lane in the plan: 256 per launch
constexpr float kNDLazy = 8.f;         // log2 of the largest softmax weight before a rescale
constexpr int kNDPart = kD + 2;        // floats of a partial row: o, max, sum

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
  int num_reqs, max_seq;
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  int* ws_cnt;
  float* ws_part;
  int target;
  int32_t* err;
};

// Item -> (request, chunk, head); `steps`: 32-token steps of the request, C of them per chunk.
struct NibDecodePlan {
  int C, r, c, h, n, n_chunks, first;
  bool none;
};

__device__ __forceinline__ NibDecodePlan nd_plan(const NibDecodeArgs& a, int item) {
  const int lane = threadIdx.x & 63;
  int n[kNDPlanLanes], st[kNDPlanLanes], total = 0;
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    const int r = lane + 64 * i;
    n[i] = r < a.num_reqs ? a.seq_lens[r] : 0;
  }
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    st[i] = (min(max(n[i], 0), a.max_seq) + kNDStep - 1) / kNDStep;
    total += st[i];
  }
  total = wave_sum_i(total);
  NibDecodePlan P{};
  // whole rounds of the four waves
  const int64_t all = (int64_t)total * a.H;
  const int64_t per = (all + a.target - 1) / a.target;
  P.C = max(1, (int)((per + kNDWaves - 1) / kNDWaves)) * kNDWaves;
  P.h = item % a.H;
  const int it = item / a.H;  // among (request, chunk)
  int carry = 0;
  P.none = true;
#pragma unroll
  for (int i = 0; i < kNDPlanLanes; ++i) {
    if (64 * i >= a.num_reqs) break;
    const int r = lane + 64 * i;
    const int nch = r < a.num_reqs ? max(1, (st[i] + P.C - 1) / P.C) : 0;
    const int incl = nib_scan(nch), ex = carry + incl - nch;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(nch > 0 && ex <= it && it < ex + nch);
    if (hit) {
      const int ln = __builtin_ctzll(hit);
      P.none = false;
      P.r = 64 * i + ln;
      P.first = __builtin_amdgcn_readlane(ex, ln);
      P.c = it - P.first;
      P.n = __builtin_amdgcn_readlane(n[i], ln);
      P.n_chunks = __builtin_amdgcn_readlane(nch, ln);
    }
    carry += __builtin_amdgcn_readlane(incl, 63);
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

template <int QDT>
__global__ __launch_bounds__(kNDThreads, 2) void nibble_decode_kernel(NibDecodeArgs a) {
  __shared__ float red_o[kNDWaves][16][kD];
  __shared__ float red_m[kNDWaves][16], red_l[kNDWaves][16];
  __shared__ int last_sh;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const NibDecodePlan P = nd_plan(a, blockIdx.x);
  if (P.none) return;
  const int r = P.r, h = P.h, G = a.G;
  const int n = min(max(P.n, 0), a.max_seq);
  if (P.n > a.max_seq && P.c == 0 && h == 0 && tid == 0) atomicOr(a.err, TTKV_ERR_SEQ_LEN);
  const int64_t row = a.qsl[r];
  if (n == 0) {  // no keys: the attention is 0
    for (int i = tid; i < G * kD; i += kNDThreads)
      store_act(a.out, a.out_dtype, row * a.out_row_stride + (int64_t)h * G * kD + i, 0.f);
    return;
  }
  const int col = lane & 15, q4 = lane >> 4;

  // The query, column `col`, as the B operand of the four score products: dims 32 g + 8 q4 ...
  half8 qf[4];
  float qs;
  nib_load_query<QDT>(a.q + row * a.q_row_stride + (int64_t)(h * G + min(col, G - 1)) * kD, q4,
                      a.scale_log2, col < G, qf, qs);

  const int steps = (n + kNDStep - 1) / kNDStep;
  // the request's steps in equal parts
  const int s0 = (int)((int64_t)steps * P.c / P.n_chunks);
  const int s1 = (int)((int64_t)steps * (P.c + 1) / P.n_chunks);
  float4v acc[8];  // [group][dim of the pair]: dims 32 g + 8 q4 + 2 i + b of the column's query
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = float4v{};
  float m = -INFINITY, l = 0.f;
  bool bad = false;

  const NibMasks masks = nib_masks();
  const uint8_t* base = a.page + (int64_t)h * kNibRecord;
  const int32_t* bt = a.bt + (int64_t)r * a.bt_row_stride;
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
      x.kp[t] = *gbl((const u32x2v*)(rec + kNibKp + 8 * col));
      x.v[t] = __builtin_nontemporal_load(gbl((const u32x4*)(rec + kNibV + 16 * lane)));
      x.vp[t][0] = *gbl((const u32x4*)(rec + kNibVp + 32 * q4));
      x.vp[t][1] = *gbl((const u32x4*)(rec + kNibVp + 32 * q4 + 16));
      bad |= id < 0;
    }
  };
  auto step = [&](int s, NibStep& x) {
    float4v sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = float4v{};
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
        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], sc[t], 0, 0, 0);
      }
    }
    const int tok = s * kNDStep + 4 * q4;
    if ((s + 1) * kNDStep > n) {  // the last step: no score and no value past the last token
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (tok + 16 * t + i >= n) {
            sc[t][i] = -INFINITY;
            const uint32_t keep = i & 1 ? 0x0000ffffu : 0xffff0000u;
#pragma unroll
            for (int g = 0; g < 4; ++g) x.vp[t][g >> 1][2 * (g & 1) + (i >> 1)] &= keep;
          }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mt = fmaxf(mt, sc[t][i]);
      }
    mt *= qs;
    if (__builtin_amdgcn_ballot_w64(mt > m + kNDLazy)) {
      const float mn = fmaxf(m, cross_row_max(mt));
      const float f = m == -INFINITY ? 0.f : exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= f;
    }
    half8 pf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        // the one rounding on the way to the output; the sum takes the rounded weights
        const half2v p = {(_Float16)fast_exp2(fmaf(sc[t][i], qs, -m)),
                          (_Float16)fast_exp2(fmaf(sc[t][i + 1], qs, -m))};
        l = __builtin_amdgcn_fdot2(p, half2v{(_Float16)1.f, (_Float16)1.f}, l, false);
        pf[4 * t + i] = p[0];
        pf[4 * t + i + 1] = p[1];
      }
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
          acc[2 * g + b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[b], pf, acc[2 * g + b], 0, 0, 0);
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
  if (bad) {
    l = NAN;
    if (lane == 0) atomicOr(a.err, TTKV_ERR_BAD_BLOCK);
  }
  l = cross_row_sum(l);

  // ---- the four waves' results, joined in LDS
  if (q4 == 0) {
    red_m[wv][col] = m;
    red_l[wv][col] = l;
  }
  __syncthreads();
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kNDWaves; ++w) M = fmaxf(M, red_m[w][col]);
  const float f = m == -INFINITY ? 0.f : exp2f(m - M);
  if (col < G) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2v o = {acc[2 * g][i] * f, acc[2 * g + 1][i] * f};
        *(float2v*)&red_o[wv][col][32 * g + 8 * q4 + 2 * i] = o;
      }
  }
  __syncthreads();
  const int64_t orow = row * a.out_row_stride + (int64_t)h * G * kD;
  const int64_t item = ((int64_t)P.first + P.c) * a.H + h;
  float* part = a.ws_part + item * G * kNDPart;
  for (int e = 2 * tid; e < G * kD; e += 2 * kNDThreads) {  // (a wave covers one row)
    const int p = e / kD, d = e % kD;
    float mm = -INFINITY, ll = 0.f;
    float2v o = {};
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) mm = fmaxf(mm, red_m[w][p]);
#pragma unroll
    for (int w = 0; w < kNDWaves; ++w) {
      ll += red_m[w][p] == -INFINITY && red_l[w][p] == 0.f ? 0.f
                                                           : red_l[w][p] * exp2f(red_m[w][p] - mm);
      o += *(const float2v*)&red_o[w][p][d];
    }
    if (P.n_chunks == 1) {
      const float inv = 1.f / ll;
      store_act(a.out, a.out_dtype, orow + e, o[0] * inv);
      store_act(a.out, a.out_dtype, orow + e + 1, o[1] * inv);
    } else {
      store_agent8(part + p * kNDPart + d, o);
      if (d == 0) store_agent8(part + p * kNDPart + kD, float2v{mm, ll});
    }
  }
  if (P.n_chunks == 1) return;

  // ---- the last workgroup of a (request, head) joins its chunks' partials
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    int* cnt = a.ws_cnt + r * a.H + h;
    const int prev = arrive(cnt);
    last_sh = prev == P.n_chunks - 1;
    if (last_sh) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_sh) return;
  const int64_t cstride = (int64_t)a.H * G * kNDPart;
  for (int p = wv; p < G; p += kNDWaves) {
    const float* pp = a.ws_part + ((int64_t)P.first * a.H + h) * G * kNDPart + p * kNDPart;
    float mm = -INFINITY, ll = 0.f;
    float2v o = {};
    for (int c0 = 0; c0 < P.n_chunks; c0 += 64) {
      const int nb = min(64, P.n_chunks - c0);
      const float* pl = pp + (c0 + min(lane, nb - 1)) * cstride + kD;
      const float2v ml = ld_agent2(pl);
      const float mc = lane < nb ? ml[0] : -INFINITY, lc = ml[1];
      const float mn = fmaxf(mm, wave_max(mc));
      const float keep = mm == -INFINITY ? 0.f : exp2f(mm - mn);
      const float wc = lane < nb ? exp2f(mc - mn) : 0.f;
      ll = ll * keep + wave_sum(lane < nb ? lc * wc : 0.f);
      o *= keep;
      for (int j = 0; j < nb; j += 8) {
        float2v x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float* po = pp + (c0 + min(j + u, nb - 1)) * cstride + 2 * lane;
          x[u] = ld_agent2(po);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float w = __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wc), min(j + u, 63)));
          if (j + u < nb) o += x[u] * w;
        }
      }
      mm = mn;
    }
    const float inv = 1.f / ll;
    store_act(a.out, a.out_dtype, orow + p * kD + 2 * lane, o[0] * inv);
    store_act(a.out, a.out_dtype, orow + p * kD + 2 * lane + 1, o[1] * inv);
  }
}

// The plan's item target: two workgroups per CU. A third would fit, but shorter chunks pay their
// prologue and join more often (8 x 14,402 tokens: 31.2 us at two per CU, 32.8 at three, 36.2 at
// four; 61 requests of 70 to 2,900: 33.4, 35.0, 34.6).
static int nd_target() {
  static int slots = 0;
  if (!slots) {
    int per_cu = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(
            &per_cu, nibble_decode_kernel<TTKV_DTYPE_F16>, kNDThreads, 0) != hipSuccess ||
        per_cu < 1)
      per_cu = 2;
    slots = std::min(per_cu, 2) * device_cu_count();
  }
  return slots;
}

// Requests per launch: the plan's lanes, and a counter per (request, head).
static int nd_slice(int H, int num_reqs) {
  return std::max(1, std::min({num_reqs, kNDPlanLanes * 64, kMaxCounters / H}));
}

// Items a launch of nr requests can plan: the target's share and a rounding per (request, head),
// and never more than one per round of the four waves.
static int64_t nd_max_items(int H, int nr, int max_seq) {
  const int64_t round = kNDStep * kNDWaves;
  const int64_t most = std::max<int64_t>(1, (max_seq + round - 1) / round);
  return std::min((int64_t)nd_target() + (int64_t)nr * H, (int64_t)nr * H * most);
}

int64_t nibble_decode_workspace_bytes(int H, int HQ, int num_reqs, int max_seq) {
  if (num_reqs == 0) return 256;
  return kCounterBytes + nd_max_items(H, nd_slice(H, num_reqs), max_seq) * (HQ / H) * kNDPart * 4;
}

int nibble_decode_paged(int H, int HQ, int d, float scale, const void* q, int q_dtype,
                        int64_t q_row_stride, const uint8_t* page, int64_t n_slots,
                        int64_t slot_stride, int bs, const int32_t* bt, int64_t bt_row_stride,
                        int max_blocks, const int32_t* seq_lens, const int32_t* qsl, int num_reqs,
                        int max_seq, void* out, int out_dtype, int64_t out_row_stride, void* ws,
                        int64_t ws_bytes, int32_t* err, hipStream_t st) {
  if (int rc = nibble_check_read(H, HQ, d, q, q_dtype, q_row_stride, page, n_slots, slot_stride,
                                 bs, bt, max_blocks, seq_lens, qsl, num_reqs, max_seq, out,
                                 out_dtype, out_row_stride, err))
    return rc;
  if (H > kMaxCounters) return host_fail(TTKV_E_UNSUPPORTED, "too many KV heads");
  const int64_t need = nibble_decode_workspace_bytes(H, HQ, num_reqs, max_seq);
  if (!ws || ws_bytes < need || (uintptr_t)ws % 256)
    return host_fail(TTKV_E_WORKSPACE, "decode workspace needs " + std::to_string(need) +
                                           " bytes, 256-aligned");
  const int slice = nd_slice(H, num_reqs);
  for (int r0 = 0; r0 < num_reqs; r0 += slice) {
    const int nr = std::min(slice, num_reqs - r0);
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
    a.bt = bt + (int64_t)r0 * bt_row_stride;
    a.bt_row_stride = bt_row_stride;
    a.seq_lens = seq_lens + r0;
    a.qsl = qsl + r0;
    a.num_reqs = nr;
    a.max_seq = max_seq;
    a.out = out;
    a.out_dtype = out_dtype;
    a.out_row_stride = out_row_stride;
    a.ws_cnt = (int*)ws;
    a.ws_part = (float*)((char*)ws + kCounterBytes);
    a.target = nd_target();
    a.err = err;
    const dim3 grid((unsigned)nd_max_items(H, nr, max_seq));
    if (q_dtype == TTKV_DTYPE_F16)
      hipLaunchKernelGGL((nibble_decode_kernel<TTKV_DTYPE_F16>), grid, dim3(kNDThreads), 0, st, a);
    else
      hipLaunchKernelGGL((nibble_decode_kernel<TTKV_DTYPE_BF16>), grid, dim3(kNDThreads), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
      return host_fail(TTKV_E_LAUNCH, std::string("nibble decode launch: ") + hipGetErrorString(e));
  }
  return TTKV_OK;
}

}  // namespace ttkv
