// Attention weights that cached tokens gather: weights[b, h, j] += sum over the query rows r of kv head h that see token j of
// exp(score(r, j) - lse[r]), the rows' log-sum-exps being those of the attention call before. What an eviction goes by.
//
// Keys only: per token and kv head 72 bytes (head_dim 128; 144 at 256, 256 as FP8) are read and 4 bytes of weights read and
// written, against 144 of an attention step. As in the decode kernel the (request, kv head) sequences form one stream of units
// of 32 tokens that is cut into equal parts, here one per WARP (to 16 query rows; one per CTA beyond): nothing is merged, every
// weight belongs to one warp, so there is no order to depend on. A warp fetches its units ahead through a ring of its own and
// computes S^T = K Q^T per 16 tokens with mma.m16n8k16, the keys dequantised in registers (code * scale is exact in f16). Query
// rows beyond those of a pass are taken in further passes over the keys.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "hkv_common.cuh"

namespace hkv {

int record_cuda(cudaError_t e);
int noalloc_workspace(void** ws);

constexpr int kWtWarps = 4;
constexpr int kWtThreads = kWtWarps * 32;
// (cost / least units of 4 / 2, 2 / 2 and 2 / 1: four requests of 2048 tokens, 8 kv heads x 128, 9.2, 7.6 and 6.8 us; 8 / 2: 12.5)
constexpr int kWtCost = 2;           // what a sequence costs a warp beyond its units (its queries and log-sum-exps), in units
constexpr int kWtMin = 1;            // least units of a warp

struct WeightsParams {
  const __nv_bfloat16* q;
  const uint8_t* kd;
  const uint8_t* ksf;
  long long dst, dsh, ssh;
  unsigned dsp, ssp;
  const int* bt;
  const int* seq_lens;
  const int* qsl;
  const float* gk;
  const float* lse;
  const float* signs;
  float* w;
  long long w_b, w_h;
  int* status;
  int MP, B, KVH, G, qlmax, lps, row0, max_len, W, window, sinks;
  float scale_log2, rot_scale;
};

// LAYOUT as in the decode kernel: 0 rows of [codes | scales] back to back, 1 codes and scales in regions of their own, 3 rows
// at any stride, copied one by one; 2 FP8 keys (rows at any stride)
template <int D, int LAYOUT>
struct WtGeo {
  static constexpr bool K8 = LAYOUT == 2;
  static constexpr bool ROWCOPY = LAYOUT >= 2;
  static constexpr int SD = K8 ? D : D / 2, SS = K8 ? 0 : D / 16;
  static constexpr int UT = 32;
  static constexpr int ROW = LAYOUT == 1 ? SD : SD + SS;             // byte stride between token rows of a stage
  static constexpr int SF_BASE = LAYOUT == 1 ? UT * SD : SD, SF_ROW = LAYOUT == 1 ? SS : ROW;
  static constexpr int STAGE = UT * (SD + SS);
  static constexpr int NS = 2;         // (8 requests of 131072, 8 x 128: 139.2 us with two stages, 139.8 with three or four)
  static constexpr int KS = D / 16, NBL = D / 64, KB = K8 ? 16 : 8;
  // 72-byte rows: as in the decode kernel, so that the lanes' loads touch every bank once
  __device__ static constexpr int tok(int i) {
    return (D == 128 && LAYOUT != 1) ? ((i & 5) | ((i & 2) << 2) | ((i & 8) >> 2)) : i;
  }
};

struct WtReq {
  int U, L, ql, q0;                    // units, context, query tokens, first query row
  int su, skip;                        // units from su on lie `skip` units further
};
__device__ __forceinline__ WtReq wt_req(const WeightsParams& p, int b) {
  WtReq r;
  r.q0 = __ldg(p.qsl + b);
  int ql = __ldg(p.qsl + b + 1) - r.q0;
  ql = (ql < 0 || ql > p.qlmax || p.G * ql <= p.row0) ? 0 : ql;
  r.ql = ql;
  r.L = ql > 0 ? min(max(__ldg(p.seq_lens + b), 0), p.max_len) : 0;
  const int all = (min(r.L, p.W) + 31) >> 5;        // (tokens behind the weights gather nothing)
  const int lo = p.window > 0 ? max(0, r.L - ql + p.row0 / p.G - p.window + 1) : 0;      // first token of the first row's window
  const int su = min(all, (min(lo, p.sinks) + 31) >> 5), wu = min(all, lo >> 5);
  r.su = su;
  r.skip = max(0, wu - su);
  r.U = all - r.skip;
  return r;
}

// The request b0 that holds the start of a part of the stream of weights (units + COST of the requests, kv head by kv head), and the
// weight of the requests before it, per kv head; part(total) cuts the stream and returns the part's start, or -1 where it is empty
// (for the whole CTA after the last __syncthreads).
template <int COST, class Part>
__device__ __forceinline__ bool wt_locate(const WeightsParams& p, int* coarse, Part part, int& b0, int& base0, WtReq& first) {
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5, B = p.B, KVH = p.KVH;
  auto wt = [](int U) { return U > 0 ? U + COST : 0; };
  if (B <= 32) {                       // a lane per request, every warp for itself
    const WtReq r = wt_req(p, min(lane, B - 1));
    const int u = lane < B ? wt(r.U) : 0;
    int incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    __syncthreads();                   // (the barriers are set up)
    const long long lo = part((long long)__shfl_sync(0xffffffffu, incl, 31) * KVH);
    if (lo < 0) return false;
    b0 = __ffs(__ballot_sync(0xffffffffu, (long long)incl * KVH > lo)) - 1;
    base0 = __shfl_sync(0xffffffffu, incl - u, b0);
    first.U = __shfl_sync(0xffffffffu, r.U, b0);
    first.L = __shfl_sync(0xffffffffu, r.L, b0);
    first.ql = __shfl_sync(0xffffffffu, r.ql, b0);
    first.q0 = __shfl_sync(0xffffffffu, r.q0, b0);
    first.su = __shfl_sync(0xffffffffu, r.su, b0);
    first.skip = __shfl_sync(0xffffffffu, r.skip, b0);
  } else {
    // prefix over groups of 32 requests
    const int ngrp = (B + 31) >> 5;
    for (int grp = wp; grp < ngrp; grp += kWtWarps) {
      const int b = grp * 32 + lane;
      int u = b < B ? wt(wt_req(p, b).U) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) u += __shfl_xor_sync(0xffffffffu, u, o);
      if (lane == 0) coarse[grp + 1] = u;
    }
    __syncthreads();
    if (wp == 0) {
      const int per_lane = (ngrp + 31) >> 5;
      int s = 0;
      for (int i = 0; i < per_lane; ++i) {
        const int k = lane * per_lane + i;
        s += k < ngrp ? coarse[k + 1] : 0;
      }
      int incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      int run = incl - s;
      for (int i = 0; i < per_lane; ++i) {
        const int k = lane * per_lane + i;
        if (k < ngrp) {
          run += coarse[k + 1];
          coarse[k + 1] = run;
        }
      }
      if (lane == 0) coarse[0] = 0;
    }
    __syncthreads();
    const long long lo = part((long long)coarse[ngrp] * KVH);
    if (lo < 0) return false;
    int lo_g = 0, hi_g = ngrp;
    while (hi_g - lo_g > 1) {
      const int m = (lo_g + hi_g) >> 1;
      if ((long long)coarse[m] * KVH <= lo) lo_g = m; else hi_g = m;
    }
    const int b = lo_g * 32 + lane;
    const int u = b < B ? wt(wt_req(p, b).U) : 0;
    int incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    const int j = __ffs(__ballot_sync(0xffffffffu, (long long)(coarse[lo_g] + incl) * KVH > lo)) - 1;
    b0 = lo_g * 32 + j;
    base0 = coarse[lo_g] + __shfl_sync(0xffffffffu, incl - u, j);
    first = wt_req(p, b0);
  }
  return true;
}

// One query row's channels of a lane (a quarter of them, in the order of the key blocks) as f16 fragments, rotated where the keys are
template <int D>
__device__ __forceinline__ void wt_query(const WeightsParams& p, const __nv_bfloat16* qrow, bool have, bool flip, int c, uint32_t (*qa)[2]) {
  constexpr int NQ = 16 * (D / 64);
  float qf[NQ];
#pragma unroll
  for (int u = 0; u < 2 * (D / 64); ++u) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (have) x = __ldg(reinterpret_cast<const uint4*>(qrow + NQ * c) + u);
    const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qf[8 * u + 2 * i] = __uint_as_float(ws[i] << 16);
      qf[8 * u + 2 * i + 1] = __uint_as_float(ws[i] & 0xffff0000u);
    }
  }
  if (p.signs != nullptr) {
    // bf16(FWHT(q * signs) * head_dim^-0.5) in the stage order of the decode kernel: the same bits
#pragma unroll
    for (int i = 0; i < NQ; i += 4) {
      const float4 y = __ldg(reinterpret_cast<const float4*>(p.signs + NQ * c + i));
      qf[i] = __fmul_rn(qf[i], y.x);
      qf[i + 1] = __fmul_rn(qf[i + 1], y.y);
      qf[i + 2] = __fmul_rn(qf[i + 2], y.z);
      qf[i + 3] = __fmul_rn(qf[i + 3], y.w);
    }
#pragma unroll
    for (int hh = 1; hh < NQ; hh *= 2)
#pragma unroll
      for (int i = 0; i < NQ; ++i)
        if ((i & hh) == 0) {
          const float a = qf[i], b = qf[i + hh];
          qf[i] = __fadd_rn(a, b);
          qf[i + hh] = __fsub_rn(a, b);
        }
#pragma unroll
    for (int m = 1; m < 4; m *= 2) {
      const bool upper = (c & m) != 0;
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        const float o2 = __shfl_xor_sync(0xffffffffu, qf[i], m);
        qf[i] = upper ? __fsub_rn(o2, qf[i]) : __fadd_rn(qf[i], o2);
      }
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) qf[i] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(qf[i], p.rot_scale)));
  }
#pragma unroll
  for (int i = 0; i < NQ / 2; ++i) {
    const float a = flip ? -qf[2 * i] : qf[2 * i], b = flip ? -qf[2 * i + 1] : qf[2 * i + 1];
    qa[i >> 1][i & 1] = pack_f16x2_sat(a, b);
  }
}

// QT: 8-row query tiles of a pass, one or two.
//
// What bounds it (8 requests of 131072 tokens, 8 x 128, group 8; 0.74 of the copy peak): instruction issue, 65 % used, and dependency
// latency; 186 warp instructions per 16 tokens, 64 of them the conversions and scale products of the keys (ALU pipe 53 %). More CTAs
// at fewer registers are slower: 126 registers 139 us, 96 165, 80 169. Rolling a unit's two blocks, for the instruction cache, gained
// nothing (16 rows over 131072: 188 -> 197 us).
template <int D, int LAYOUT, int QT>
__global__ void __launch_bounds__(kWtThreads, D == 128 ? (QT == 1 ? 4 : 3) : QT == 1 ? 3 : 2) weights_kernel(const WeightsParams p) {
  using Gm = WtGeo<D, LAYOUT>;
  constexpr int NS = Gm::NS, UT = Gm::UT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kWtWarps * NS];
  int* coarse = reinterpret_cast<int*>(smem + kWtWarps * NS * Gm::STAGE);
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int KVH = p.KVH, B = p.B, G = p.G;
  if (tid < kWtWarps * NS) mbar_init(bars + tid, Gm::ROWCOPY ? 32 : 1);
  pdl_wait();
  pdl_launch_dependents();

  // the part [lo, hi) of this warp in the stream of weights
  auto wt = [](int U) { return U > 0 ? U + kWtCost : 0; };
  const long long parts = (long long)gridDim.x * kWtWarps;
  long long lo, hi;
  auto part = [&](long long total) {
    const long long per = max((long long)(kWtMin + kWtCost), (total + parts - 1) / parts);
    lo = ((long long)blockIdx.x + (long long)wp * gridDim.x) * per;
    hi = min(total, lo + per);
    return lo < hi ? lo : -1ll;
  };
  int b0, base0;
  WtReq first;                         // of b0
  fence_barrier_init();
  if (!wt_locate<kWtCost>(p, coarse, part, b0, base0, first)) return;
  // A walk over the units of [lo, hi): the fetching side runs NS units ahead of the computing one
  struct Walk {
    int b, h, u, end;                  // the next unit of sequence (b, h), one past its last here
    long long seq0;                    // stream position of the sequence: kWtCost slots, then its units
    WtReq r;
  };
  auto enter = [&](Walk& x, long long pos) {        // from stream position pos on; false: nothing left
    while (pos < hi) {
      const long long u0 = x.seq0 + kWtCost, e = u0 + x.r.U;
      const long long from = max(pos, u0), to = min(hi, e);
      if (x.r.U > 0 && from < to) {
        x.u = (int)(from - u0);
        x.end = (int)(to - u0);
        return true;
      }
      if (hi <= e) return false;
      x.seq0 = e;
      pos = max(pos, e);
      if (++x.h == KVH) {
        x.h = 0;
        do {
          if (++x.b >= B) return false;
          x.r = wt_req(p, x.b);
        } while (x.r.U <= 0);
      }
    }
    return false;
  };
  Walk cw;
  cw.b = b0;
  cw.r = first;
  cw.h = (int)((lo - (long long)base0 * KVH) / wt(cw.r.U));
  cw.seq0 = (long long)base0 * KVH + (long long)cw.h * wt(cw.r.U);
  bool more = enter(cw, lo);
  Walk fw = cw;
  bool f_more = more;

  const uint32_t ring_a = smem_u32(smem + wp * NS * Gm::STAGE), bars_a = smem_u32(bars + wp * NS);
  const int PSM = (1 << p.lps) - 1;
  // units fetched ahead; the next stage to fetch into and to consume, and the latter's phase
  int ahead = 0, f_st = 0, c_st = 0;
  uint32_t c_par = 0;
  const uint8_t *f_kd, *f_ks;          // keys of the fetching side's kv head
  auto f_head = [&]() {
    f_kd = p.kd + (long long)fw.h * p.dsh;
    f_ks = p.ksf + (long long)fw.h * p.ssh;
  };
  f_head();
  // page ids of the next 16 units (two 16-token blocks each) of the fetching side's sequence, a lane each; -1: no row sees the block
  int pg = 0, pg_first = 0, pg_end = -1;
  auto look_up = [&]() {
    const int u = fw.u + (lane >> 1), t = (u + (u >= fw.r.su ? fw.r.skip : 0)) * UT + 16 * (lane & 1);
    const int lo_w = p.window > 0 ? max(0, fw.r.L - fw.r.ql + p.row0 / G - p.window + 1) : 0;
    pg = u < fw.end && t < min(fw.r.L, p.W) && (t + 16 > lo_w || t < p.sinks) ? __ldg(p.bt + (long long)fw.b * p.MP + (t >> p.lps)) : -1;
    pg_first = fw.u;
    pg_end = min(fw.end, fw.u + 16);
  };
  // fetches the next unit, 16-token blocks that hold a visible token only
  auto fetch = [&]() {
    const uint32_t bar = bars_a + 8 * f_st, st = ring_a + f_st * Gm::STAGE;
    const int tok0 = (fw.u + (fw.u >= fw.r.su ? fw.r.skip : 0)) * UT;
    if (fw.u >= pg_end) look_up();
    int page[2];
#pragma unroll
    for (int bi = 0; bi < 2; ++bi) page[bi] = __shfl_sync(0xffffffffu, pg, 2 * (fw.u - pg_first) + bi);
    if (Gm::ROWCOPY) {
      // two lanes per token row (of a 16-token block)
      constexpr int CB = D == 128 ? 8 : 16, N = (Gm::SD + Gm::SS) / CB;
      const int row = lane >> 1;
#pragma unroll
      for (int bi = 0; bi < 2; ++bi)
        if (page[bi] >= 0) {
          const uint8_t* src = f_kd + (unsigned long long)(unsigned)page[bi] * p.dsp + (((tok0 + 16 * bi) & PSM) + row) * p.dst;
          const uint32_t d = st + (16 * bi + row) * Gm::ROW;
          for (int j = lane & 1; j < N; j += 2) cp_async<CB>(d + j * CB, src + j * CB);
        }
      cp_async_mbar_arrive_noinc(bar);
    } else if (elect_one()) {
      const int nb = (page[0] >= 0) + (page[1] >= 0);
      mbar_expect_tx_u32(bar, nb * 16 * (Gm::SD + Gm::SS));
#pragma unroll
      for (int bi = 0; bi < 2; ++bi)
        if (page[bi] >= 0) {
          const unsigned pos = (tok0 + 16 * bi) & PSM;
          const uint8_t* src = f_kd + (unsigned long long)(unsigned)page[bi] * p.dsp + pos * (unsigned)Gm::ROW;
          if (LAYOUT == 0) {
            bulk_g2s_u32(st + bi * 16 * Gm::ROW, src, 16 * Gm::ROW, bar);
          } else {
            bulk_g2s_u32(st + bi * 16 * Gm::SD, src, 16 * Gm::SD, bar);
            bulk_g2s_u32(st + UT * Gm::SD + bi * 16 * Gm::SS, f_ks + (unsigned long long)(unsigned)page[bi] * p.ssp + pos * (unsigned)Gm::SS,
                         16 * Gm::SS, bar);
          }
        }
    }
    ++ahead;
    if (++f_st == NS) f_st = 0;
    if (++fw.u == fw.end) {
      f_more = enter(fw, fw.seq0 + kWtCost + fw.end);
      f_head();
      pg_end = -1;
    }
  };
  while (f_more && ahead < NS) fetch();

  const int r0 = Gm::tok(g), r1 = Gm::tok(g + 8);
  const uint32_t koff_d = r0 * Gm::ROW + Gm::KB * Gm::NBL * c, koff_s = Gm::SF_BASE + r0 * Gm::SF_ROW + Gm::NBL * c;
  constexpr int KR1 = Gm::tok(8) - Gm::tok(0);
  bool dead = false;
  while (more && !dead) {
    // the queries of this sequence: rows 8 q + g, channels of this lane's key blocks, as f16; rows 2 c, 2 c + 1 of the scores
    const int L = cw.r.L, ql = cw.r.ql, q0 = cw.r.q0, h = cw.h;
    const int R = min(8 * QT, G * ql - p.row0);
    float le[QT][2];
    int lim[QT][2];
#pragma unroll
    for (int q = 0; q < QT; ++q)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = 8 * q + 2 * c + k, row = p.row0 + r;
        const bool is = r < R;
        const int tr = is ? row / G : 0;
        le[q][k] = is ? __ldg(p.lse + (long long)(q0 + tr) * (KVH * G) + h * G + row - tr * G)
                      : __int_as_float(0x7f800000);              // (a row that does not exist: its scores are 0 - inf)
        lim[q][k] = is ? L - ql + tr + 1 : 0;       // sees the keys below this one
      }
    const float sc_signed = p.scale_log2 * __ldg(p.gk + h);
    const bool flip = sc_signed < 0.0f;
    const float sc = fabsf(sc_signed);
    uint32_t qa[QT][Gm::KS][2];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      const bool have = g + 8 * q < R;
      const int t = have ? (p.row0 + g + 8 * q) / G : 0, gq = have ? p.row0 + g + 8 * q - t * G : 0;
      const __nv_bfloat16* qrow = p.q + ((long long)(q0 + t) * (KVH * G) + h * G + gq) * D;
      wt_query<D>(p, qrow, have, flip, c, qa[q]);
    }
#pragma unroll
    for (int q = 0; q < QT; ++q) {
      le[q][0] *= 1.4426950408889634f;
      le[q][1] *= 1.4426950408889634f;
    }
    // tokens of [w_hi, t_lo) and whole sinks are seen by every row that exists
    const int t_lo = L - ql + p.row0 / G + 1;
    const int w_hi = p.window > 0 ? L - ql + (p.row0 + R - 1) / G + 1 - p.window : 0;
    const int lo_w = p.window > 0 ? L - ql + p.row0 / G + 1 - p.window : 0;
    float* wrow = p.w + (long long)cw.b * p.w_b + (long long)h * p.w_h;
    while (true) {
      const uint32_t bar = bars_a + 8 * c_st, st = ring_a + c_st * Gm::STAGE;
      const int tok0 = (cw.u + (cw.u >= cw.r.su ? cw.r.skip : 0)) * UT;
      // this lane's token of the unit, whose weight it adds to: block c / 2, row r0 or r1
      const int mine = tok0 + 16 * (c >> 1) + (c & 1 ? r1 : r0);
      const bool masked = tok0 + UT > t_lo || (tok0 < w_hi && tok0 + UT > p.sinks);
      const bool add = mine < min(L, p.W) && (mine >= lo_w || mine < p.sinks);
      float old = add ? wrow[mine] : 0.0f;
      if (!mbar_try_wait_u32(bar, c_par) && !mbar_wait_bounded_u32(bar, c_par)) {
        if (lane == 0) atomicExch(p.status, HKV_ERR_DEVICE_WAIT);
        dead = true;
        break;
      }
      float sum[2][2];                              // [block][row r0 / r1], over this lane's query rows
#pragma unroll
      for (int bi = 0; bi < 2; ++bi) {
        const uint32_t kd_ = st + koff_d + bi * 16 * Gm::ROW, ks_ = st + koff_s + bi * 16 * Gm::SF_ROW;
        float x[QT][4];
#pragma unroll
        for (int q = 0; q < QT; ++q) x[q][0] = x[q][1] = x[q][2] = x[q][3] = 0.0f;
        if (Gm::K8) {
#pragma unroll
          for (int u = 0; u < Gm::NBL; ++u) {
            const uint4 a = lds128(kd_ + 16 * u), b = lds128(kd_ + KR1 * Gm::ROW + 16 * u);
            const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t A[4];
              e4m3x4_to_f16x2(wa[v], A[0], A[2]);
              e4m3x4_to_f16x2(wb[v], A[1], A[3]);
#pragma unroll
              for (int q = 0; q < QT; ++q) mma_f16(x[q], A[0], A[1], A[2], A[3], qa[q][4 * u + v][0], qa[q][4 * u + v][1]);
            }
          }
        } else {
          uint2 w0[Gm::NBL], w1[Gm::NBL];
          uint32_t h0[(Gm::NBL + 1) / 2], h1[(Gm::NBL + 1) / 2];
          if (Gm::NBL == 2) {
            w0[0] = lds64(kd_);
            w0[1] = lds64(kd_ + 8);
            w1[0] = lds64(kd_ + KR1 * Gm::ROW);
            w1[1] = lds64(kd_ + KR1 * Gm::ROW + 8);
            h0[0] = e4m3x2_to_f16x2(lds16(ks_));
            h1[0] = e4m3x2_to_f16x2(lds16(ks_ + KR1 * Gm::SF_ROW));
          } else {
#pragma unroll
            for (int j = 0; j < Gm::NBL / 2; ++j) {
              const uint4 a = lds128(kd_ + 16 * j), b = lds128(kd_ + KR1 * Gm::ROW + 16 * j);
              w0[2 * j] = make_uint2(a.x, a.y);
              w0[2 * j + 1] = make_uint2(a.z, a.w);
              w1[2 * j] = make_uint2(b.x, b.y);
              w1[2 * j + 1] = make_uint2(b.z, b.w);
            }
            e4m3x4_to_f16x2(lds32(ks_), h0[0], h0[(Gm::NBL - 1) / 2]);
            e4m3x4_to_f16x2(lds32(ks_ + KR1 * Gm::SF_ROW), h1[0], h1[(Gm::NBL - 1) / 2]);
          }
#pragma unroll
          for (int u = 0; u < Gm::NBL; ++u) {
            const __half2 p0 = u32_as_h2(h0[u >> 1]), p1 = u32_as_h2(h1[u >> 1]);
            const __half2 sf0 = (u & 1) ? __high2half2(p0) : __low2half2(p0);
            const __half2 sf1 = (u & 1) ? __high2half2(p1) : __low2half2(p1);
            uint32_t e0[4], e1[4], e2[4], e3[4];
            e2m1x8_to_f16x2(w0[u].x, e0);
            e2m1x8_to_f16x2(w0[u].y, e1);
            e2m1x8_to_f16x2(w1[u].x, e2);
            e2m1x8_to_f16x2(w1[u].y, e3);
#pragma unroll
            for (int v = 0; v < 4; ++v) {           // k-step v: channels 4 v .. 4 v + 3 of the block
              const uint32_t a0 = hmul2h(v < 2 ? e0[2 * v & 3] : e1[2 * v & 3], sf0), a1 = hmul2h(v < 2 ? e2[2 * v & 3] : e3[2 * v & 3], sf1);
              const uint32_t a2 = hmul2h(v < 2 ? e0[(2 * v & 3) + 1] : e1[(2 * v & 3) + 1], sf0),
                             a3 = hmul2h(v < 2 ? e2[(2 * v & 3) + 1] : e3[(2 * v & 3) + 1], sf1);
#pragma unroll
              for (int q = 0; q < QT; ++q) mma_f16(x[q], a0, a1, a2, a3, qa[q][4 * u + v][0], qa[q][4 * u + v][1]);
            }
          }
        }
        sum[bi][0] = sum[bi][1] = 0.0f;
        const int ta = tok0 + 16 * bi + r0, tb = tok0 + 16 * bi + r1;
#pragma unroll
        for (int q = 0; q < QT; ++q) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float pa = fast_exp2(fmaf(x[q][k], sc, -le[q][k])), pb = fast_exp2(fmaf(x[q][2 + k], sc, -le[q][k]));
            if (masked) {                           // (warp-uniform)
              auto sees = [&](int t) { return t < lim[q][k] && (p.window == 0 || t >= lim[q][k] - p.window || t < p.sinks); };
              pa = sees(ta) ? pa : 0.0f;
              pb = sees(tb) ? pb : 0.0f;
            }
            sum[bi][0] += pa;
            sum[bi][1] += pb;
          }
        }
      }
      // the four lanes of a token sum up their rows; lane c ends with block c / 2, row r0 (c even) or r1
      const bool up = c & 2, odd = c & 1;
      float s0 = up ? sum[1][0] : sum[0][0], s1 = up ? sum[1][1] : sum[0][1];
      s0 += __shfl_xor_sync(0xffffffffu, up ? sum[0][0] : sum[1][0], 2);
      s1 += __shfl_xor_sync(0xffffffffu, up ? sum[0][1] : sum[1][1], 2);
      const float s = (odd ? s1 : s0) + __shfl_xor_sync(0xffffffffu, odd ? s0 : s1, 1);
      if (add) wrow[mine] = old + s;
      --ahead;
      if (++c_st == NS) {
        c_st = 0;
        c_par ^= 1;
      }
      __syncwarp();
      if (f_more) fetch();                          // (into the stage just read)
      if (++cw.u == cw.end) {
        more = enter(cw, cw.seq0 + kWtCost + cw.end);
        break;
      }
    }
  }
  if (dead)                                         // nothing of this warp's may still be on its way when the CTA ends
    for (; ahead > 0; --ahead) {
      (void)mbar_wait_bounded_u32(bars_a + 8 * c_st, c_par);
      if (++c_st == NS) {
        c_st = 0;
        c_par ^= 1;
      }
    }
}

// Passes of 32 rows (17 to 64 query rows a kv head). With the kernel above every warp would prepare 32 rows for itself and hold their
// fragments in 128 registers (at head_dim 256). Here the part of the stream belongs to a CTA: its warps prepare a tile of eight rows
// each, put the fragments into shared memory and take the units by turns; a unit's two blocks share each fragment that is read.
// 32 requests of 1k to 16k tokens, 2 x 256, group 8 x 4 tokens: 50 us in two passes of 16 rows, 34 with the fragments in registers,
// 29.3 so. What bounds it: of 45000 clocks 9000 locate, fetch and prepare, then a unit takes a warp 4400 with the tensor pipe two
// thirds busy (mma.sync; 128 instructions a unit). Two CTAs an SM 29.8 us, three 29.3, four 30.6 (128 registers, spills); with the
// blocks of channels rolled 30.1; queries prefetched before the pages are looked up 30.5; a sequence's cost at 5 to 8 units 29.4 to 30.
// Passes of 16 rows gain little by it (the same with two tokens 22.9 -> 22.1, 300 requests to 300 tokens 12.7 -> 14.5) and keep theirs.
constexpr int kWdCost = 3;           // what a sequence costs a CTA beyond its units, in units
constexpr int kWdMin = 4;

template <int D, int LAYOUT>
__global__ void __launch_bounds__(kWtThreads, LAYOUT == 2 ? 2 : 3) wide_weights_kernel(const WeightsParams p) {
  using Gm = WtGeo<D, LAYOUT>;
  constexpr int NS = Gm::NS, UT = Gm::UT, QT = 4, W = kWtWarps;
  static_assert(W == QT, "a tile of rows per warp");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[W * NS];
  __shared__ __align__(8) float s_le[8 * QT];       // log-sum-exps (base 2) of the rows
  __shared__ __align__(8) int s_lim[8 * QT];        // a row sees the keys below this one
  uint8_t* sq = smem + W * NS * Gm::STAGE;          // fragments of the sequence's queries
  const uint32_t sq_a = smem_u32(sq);
  int* coarse = reinterpret_cast<int*>(sq + QT * Gm::KS * 256);
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int KVH = p.KVH, B = p.B, G = p.G;
  if (tid < W * NS) mbar_init(bars + tid, Gm::ROWCOPY ? 32 : 1);
  pdl_wait();
  pdl_launch_dependents();

  auto wt = [](int U) { return U > 0 ? U + kWdCost : 0; };
  long long lo, hi;
  auto part = [&](long long total) {
    const long long per = max((long long)(kWdMin + kWdCost), (total + gridDim.x - 1) / gridDim.x);
    lo = (long long)blockIdx.x * per;
    hi = min(total, lo + per);
    return lo < hi ? lo : -1ll;
  };
  int b0, base0;
  WtReq first;
  fence_barrier_init();
  if (!wt_locate<kWdCost>(p, coarse, part, b0, base0, first)) return;
  // A walk over the sequences of [lo, hi): units [u, end) of sequence (b, h), n units of the CTA before them. The unit u + i is the
  // warp's with number (n + i) % 4.
  struct Walk {
    int b, h, u, end, n;
    long long seq0;
    WtReq r;
  };
  auto enter = [&](Walk& x, long long pos) {
    while (pos < hi) {
      const long long u0 = x.seq0 + kWdCost, e = u0 + x.r.U;
      const long long from = max(pos, u0), to = min(hi, e);
      if (x.r.U > 0 && from < to) {
        x.u = (int)(from - u0);
        x.end = (int)(to - u0);
        return true;
      }
      if (hi <= e) return false;
      x.seq0 = e;
      pos = max(pos, e);
      if (++x.h == KVH) {
        x.h = 0;
        do {
          if (++x.b >= B) return false;
          x.r = wt_req(p, x.b);
        } while (x.r.U <= 0);
      }
    }
    return false;
  };
  auto next = [&](Walk& x) {
    x.n += x.end - x.u;
    return enter(x, x.seq0 + kWdCost + x.end);
  };
  auto own = [&](const Walk& x) { return x.u + ((wp - x.n) & (W - 1)); };
  Walk cw;
  cw.b = b0;
  cw.r = first;
  cw.n = 0;
  cw.h = (int)((lo - (long long)base0 * KVH) / wt(cw.r.U));
  cw.seq0 = (long long)base0 * KVH + (long long)cw.h * wt(cw.r.U);
  bool more = enter(cw, lo);
  Walk fw = cw;
  bool f_more = more;
  int fu = own(fw);

  const uint32_t ring_a = smem_u32(smem + wp * NS * Gm::STAGE), bars_a = smem_u32(bars + wp * NS);
  const int PSM = (1 << p.lps) - 1;
  int ahead = 0, f_st = 0, c_st = 0;
  uint32_t c_par = 0;
  // page ids of this warp's next 16 units, two 16-token blocks each; -1: no row sees the block
  int pg = 0, pg_first = 0, pg_end = -1;
  auto seek = [&]() {                  // to a sequence that has a unit for this warp
    while (f_more && fu >= fw.end) {
      f_more = next(fw);
      fu = own(fw);
      pg_end = -1;
    }
  };
  auto fetch = [&]() {
    const uint32_t bar = bars_a + 8 * f_st, st = ring_a + f_st * Gm::STAGE;
    const int tok0 = (fu + (fu >= fw.r.su ? fw.r.skip : 0)) * UT;
    if (fu >= pg_end) {
      const int u = fu + W * (lane >> 1), t = (u + (u >= fw.r.su ? fw.r.skip : 0)) * UT + 16 * (lane & 1);
      const int lo_w = p.window > 0 ? max(0, fw.r.L - fw.r.ql + p.row0 / G - p.window + 1) : 0;
      pg = u < fw.end && t < min(fw.r.L, p.W) && (t + 16 > lo_w || t < p.sinks) ? __ldg(p.bt + (long long)fw.b * p.MP + (t >> p.lps)) : -1;
      pg_first = fu;
      pg_end = fu + W * 16;
    }
    int page[2];
#pragma unroll
    for (int bi = 0; bi < 2; ++bi) page[bi] = __shfl_sync(0xffffffffu, pg, 2 * ((fu - pg_first) / W) + bi);
    const uint8_t* f_kd = p.kd + (long long)fw.h * p.dsh;
    if (Gm::ROWCOPY) {
      constexpr int CB = D == 128 ? 8 : 16, N = (Gm::SD + Gm::SS) / CB;
      const int row = lane >> 1;
#pragma unroll
      for (int bi = 0; bi < 2; ++bi)
        if (page[bi] >= 0) {
          const uint8_t* src = f_kd + (unsigned long long)(unsigned)page[bi] * p.dsp + (((tok0 + 16 * bi) & PSM) + row) * p.dst;
          const uint32_t d = st + (16 * bi + row) * Gm::ROW;
          for (int j = lane & 1; j < N; j += 2) cp_async<CB>(d + j * CB, src + j * CB);
        }
      cp_async_mbar_arrive_noinc(bar);
    } else if (elect_one()) {
      const int nb = (page[0] >= 0) + (page[1] >= 0);
      mbar_expect_tx_u32(bar, nb * 16 * (Gm::SD + Gm::SS));
#pragma unroll
      for (int bi = 0; bi < 2; ++bi)
        if (page[bi] >= 0) {
          const unsigned pos = (tok0 + 16 * bi) & PSM;
          const uint8_t* src = f_kd + (unsigned long long)(unsigned)page[bi] * p.dsp + pos * (unsigned)Gm::ROW;
          if (LAYOUT == 0) {
            bulk_g2s_u32(st + bi * 16 * Gm::ROW, src, 16 * Gm::ROW, bar);
          } else {
            const uint8_t* f_ks = p.ksf + (long long)fw.h * p.ssh;
            bulk_g2s_u32(st + bi * 16 * Gm::SD, src, 16 * Gm::SD, bar);
            bulk_g2s_u32(st + UT * Gm::SD + bi * 16 * Gm::SS, f_ks + (unsigned long long)(unsigned)page[bi] * p.ssp + pos * (unsigned)Gm::SS,
                         16 * Gm::SS, bar);
          }
        }
    }
    ++ahead;
    if (++f_st == NS) f_st = 0;
    fu += W;
    seek();
  };
  seek();
  while (f_more && ahead < NS) fetch();

  const int r0 = Gm::tok(g), r1 = Gm::tok(g + 8);
  const uint32_t koff_d = r0 * Gm::ROW + Gm::KB * Gm::NBL * c, koff_s = Gm::SF_BASE + r0 * Gm::SF_ROW + Gm::NBL * c;
  constexpr int KR1 = Gm::tok(8) - Gm::tok(0);
  bool dead = false;                                // (of this warp; it keeps meeting the others)
  while (more) {
    const int L = cw.r.L, ql = cw.r.ql, q0 = cw.r.q0, h = cw.h;
    const int R = min(8 * QT, G * ql - p.row0);
    const float sc_signed = p.scale_log2 * __ldg(p.gk + h);
    const bool flip = sc_signed < 0.0f;
    const float sc = fabsf(sc_signed);
    {
      const bool have = g + 8 * wp < R;
      const int t = have ? (p.row0 + g + 8 * wp) / G : 0, gq = have ? p.row0 + g + 8 * wp - t * G : 0;
      uint32_t qa[Gm::KS][2];
      wt_query<D>(p, p.q + ((long long)(q0 + t) * (KVH * G) + h * G + gq) * D, have, flip, c, qa);
      __syncthreads();                              // the sequence before is done with its fragments
#pragma unroll
      for (int k = 0; k < Gm::KS; k += 2)           // two k-steps a lane together
        *reinterpret_cast<uint4*>(sq + (wp * Gm::KS + k) * 256 + 16 * lane) = make_uint4(qa[k][0], qa[k][1], qa[k + 1][0], qa[k + 1][1]);
      if (tid < 8 * QT) {
        const int row = p.row0 + tid;
        const bool is = tid < R;
        const int tr = is ? row / G : 0;
        s_le[tid] = is ? 1.4426950408889634f * __ldg(p.lse + (long long)(q0 + tr) * (KVH * G) + h * G + row - tr * G)
                       : __int_as_float(0x7f800000);             // (a row that does not exist: its scores are 0 - inf)
        s_lim[tid] = is ? L - ql + tr + 1 : 0;
      }
      __syncthreads();
    }
    // tokens of [w_hi, t_lo) and whole sinks are seen by every row that exists
    const int t_lo = L - ql + p.row0 / G + 1;
    const int w_hi = p.window > 0 ? L - ql + (p.row0 + R - 1) / G + 1 - p.window : 0;
    const int lo_w = p.window > 0 ? L - ql + p.row0 / G + 1 - p.window : 0;
    float* wrow = p.w + (long long)cw.b * p.w_b + (long long)h * p.w_h;
    for (int cu = own(cw); cu < cw.end && !dead; cu += W) {
      const uint32_t bar = bars_a + 8 * c_st, st = ring_a + c_st * Gm::STAGE;
      const int tok0 = (cu + (cu >= cw.r.su ? cw.r.skip : 0)) * UT;
      // this lane's token of the unit, whose weight it adds to: block c / 2, row r0 or r1
      const int mine = tok0 + 16 * (c >> 1) + (c & 1 ? r1 : r0);
      const bool masked = tok0 + UT > t_lo || (tok0 < w_hi && tok0 + UT > p.sinks);
      const bool add = mine < min(L, p.W) && (mine >= lo_w || mine < p.sinks);
      const float old = add ? wrow[mine] : 0.0f;
      if (!mbar_try_wait_u32(bar, c_par) && !mbar_wait_bounded_u32(bar, c_par)) {
        if (lane == 0) atomicExch(p.status, HKV_ERR_DEVICE_WAIT);
        dead = true;
        break;
      }
      float x[2][QT][4];
#pragma unroll
      for (int bi = 0; bi < 2; ++bi)
#pragma unroll
        for (int q = 0; q < QT; ++q) x[bi][q][0] = x[bi][q][1] = x[bi][q][2] = x[bi][q][3] = 0.0f;
      const uint32_t kd_ = st + koff_d, ks_ = st + koff_s;
#pragma unroll
      for (int j = 0; j < Gm::NBL / 2; ++j) {       // two blocks of channels of this lane
        uint32_t h0[2], h1[2];                      // their scales, of rows r0, r1 of both blocks of tokens
        uint32_t wd[2][2][2][Gm::K8 ? 4 : 2];       // and codes: [token block][row r0 / r1][channel block]
#pragma unroll
        for (int bi = 0; bi < 2; ++bi)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t a = kd_ + (bi * 16 + r * KR1) * Gm::ROW + 2 * Gm::KB * j;
            if (!Gm::K8) (r ? h1 : h0)[bi] = e4m3x2_to_f16x2(lds16(ks_ + (bi * 16 + r * KR1) * Gm::SF_ROW + 2 * j));
            if (D == 128) {                         // (rows of 72 bytes)
#pragma unroll
              for (int uu = 0; uu < 2; ++uu) {
                const uint2 y = lds64(a + 8 * uu);
                wd[bi][r][uu][0] = y.x, wd[bi][r][uu][1] = y.y;
              }
            } else if (Gm::K8) {
#pragma unroll
              for (int uu = 0; uu < 2; ++uu) {
                const uint4 y = lds128(a + 16 * uu);
                wd[bi][r][uu][0] = y.x, wd[bi][r][uu][1] = y.y;
                if constexpr (Gm::K8) wd[bi][r][uu][2] = y.z, wd[bi][r][uu][3] = y.w;
              }
            } else {
              const uint4 y = lds128(a);
              wd[bi][r][0][0] = y.x, wd[bi][r][0][1] = y.y, wd[bi][r][1][0] = y.z, wd[bi][r][1][1] = y.w;
            }
          }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {            // k-steps 8 j + 2 kk and the next
          const int uu = kk >> 1, vv = kk & 1;
          uint32_t A[2][2][4];
#pragma unroll
          for (int bi = 0; bi < 2; ++bi) {
            if (Gm::K8) {
              e4m3x4_to_f16x2(wd[bi][0][uu][2 * vv], A[bi][0][0], A[bi][0][2]);
              e4m3x4_to_f16x2(wd[bi][1][uu][2 * vv], A[bi][0][1], A[bi][0][3]);
              e4m3x4_to_f16x2(wd[bi][0][uu][2 * vv + 1], A[bi][1][0], A[bi][1][2]);
              e4m3x4_to_f16x2(wd[bi][1][uu][2 * vv + 1], A[bi][1][1], A[bi][1][3]);
            } else {
              const __half2 p0 = u32_as_h2(h0[bi]), p1 = u32_as_h2(h1[bi]);
              const __half2 sf0 = uu ? __high2half2(p0) : __low2half2(p0);
              const __half2 sf1 = uu ? __high2half2(p1) : __low2half2(p1);
              uint32_t e0[4], e1[4];
              e2m1x8_to_f16x2(wd[bi][0][uu][vv], e0);
              e2m1x8_to_f16x2(wd[bi][1][uu][vv], e1);
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                A[bi][v][0] = hmul2h(e0[2 * v], sf0);
                A[bi][v][1] = hmul2h(e1[2 * v], sf1);
                A[bi][v][2] = hmul2h(e0[2 * v + 1], sf0);
                A[bi][v][3] = hmul2h(e1[2 * v + 1], sf1);
              }
            }
          }
          uint4 f[QT];
#pragma unroll
          for (int q = 0; q < QT; ++q) f[q] = lds128(sq_a + (q * Gm::KS + 8 * j + 2 * kk) * 256 + 16 * lane);
#pragma unroll
          for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int bi = 0; bi < 2; ++bi)
              mma_f16(x[bi][q], A[bi][0][0], A[bi][0][1], A[bi][0][2], A[bi][0][3], f[q].x, f[q].y);
#pragma unroll
          for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int bi = 0; bi < 2; ++bi)
              mma_f16(x[bi][q], A[bi][1][0], A[bi][1][1], A[bi][1][2], A[bi][1][3], f[q].z, f[q].w);
        }
      }
      float sum[2][2] = {};                         // [block][row r0 / r1], over this lane's query rows
#pragma unroll
      for (int q = 0; q < QT; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float le = s_le[8 * q + 2 * c + k];
          const int lim = masked ? s_lim[8 * q + 2 * c + k] : 0;
#pragma unroll
          for (int bi = 0; bi < 2; ++bi) {
            float pa = fast_exp2(fmaf(x[bi][q][k], sc, -le)), pb = fast_exp2(fmaf(x[bi][q][2 + k], sc, -le));
            if (masked) {                           // (warp-uniform)
              auto sees = [&](int t) { return t < lim && (p.window == 0 || t >= lim - p.window || t < p.sinks); };
              pa = sees(tok0 + 16 * bi + r0) ? pa : 0.0f;
              pb = sees(tok0 + 16 * bi + r1) ? pb : 0.0f;
            }
            sum[bi][0] += pa;
            sum[bi][1] += pb;
          }
        }
      // the four lanes of a token sum up their rows; lane c ends with block c / 2, row r0 (c even) or r1
      const bool up = c & 2, odd = c & 1;
      float s0 = up ? sum[1][0] : sum[0][0], s1 = up ? sum[1][1] : sum[0][1];
      s0 += __shfl_xor_sync(0xffffffffu, up ? sum[0][0] : sum[1][0], 2);
      s1 += __shfl_xor_sync(0xffffffffu, up ? sum[0][1] : sum[1][1], 2);
      const float sum_ = (odd ? s1 : s0) + __shfl_xor_sync(0xffffffffu, odd ? s0 : s1, 1);
      if (add) wrow[mine] = old + sum_;
      --ahead;
      if (++c_st == NS) {
        c_st = 0;
        c_par ^= 1;
      }
      __syncwarp();
      if (f_more) fetch();                          // (into the stage just read)
    }
    more = next(cw);
  }
  if (dead)                                         // nothing of this warp's may still be on its way when the CTA ends
    for (; ahead > 0; --ahead) {
      (void)mbar_wait_bounded_u32(bars_a + 8 * c_st, c_par);
      if (++c_st == NS) {
        c_st = 0;
        c_par ^= 1;
      }
    }
}

template <int D, int LAYOUT, int QT>
static int launch_weights(const WeightsParams& p, cudaStream_t st) {
  using Gm = WtGeo<D, LAYOUT>;
  void (*k)(WeightsParams);
  if constexpr (QT == 4) k = wide_weights_kernel<D, LAYOUT>;
  else k = weights_kernel<D, LAYOUT, QT>;
  const size_t smem = kWtWarps * Gm::NS * Gm::STAGE + (QT == 4 ? QT * Gm::KS * 256 : 0) + (kMaxBatch / 32 + 2) * 4;
  int dev = 0, sms = 0, ctas = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, k, kWtThreads, smem);
  if (e != cudaSuccess) return record_cuda(e);
  if (ctas < 1) return HKV_ERR_UNSUPPORTED;
  return record_cuda(launch_pdl(k, dim3((unsigned)(sms * ctas)), dim3(kWtThreads), smem, st, p));
}

template <int QT>
static int launch_weights_any(const WeightsParams& p, int D, int layout, cudaStream_t st) {
  if (D == 128) return layout == 0 ? launch_weights<128, 0, QT>(p, st) : layout == 1 ? launch_weights<128, 1, QT>(p, st) : launch_weights<128, 3, QT>(p, st);
  return layout == 0 ? launch_weights<256, 0, QT>(p, st) : layout == 1 ? launch_weights<256, 1, QT>(p, st)
         : layout == 2 ? launch_weights<256, 2, QT>(p, st) : launch_weights<256, 3, QT>(p, st);
}

}  // namespace hkv

extern "C" int hkv_accumulate_weights(const void* q, const void* kd, const void* ksf, const int64_t strides[6], int PS,
                                      const int32_t* block_tables, int MP, const int32_t* seq_lens, const int32_t* query_start_loc,
                                      int B, int KVH, int G, int D, int qlmax, float sm_scale, const float* gk, const float* lse,
                                      float* weights, int64_t w_b, int64_t w_h, int W, int window, int sinks, const float* signs,
                                      int k8, void* workspace, void* stream) {
  using namespace hkv;
  if (B < 0 || MP < 0 || W < 0 || window < 0 || sinks < 0) return HKV_ERR_RANGE;
  if (B == 0) return HKV_OK;
  if (!q || !kd || !ksf || !strides || !block_tables || !seq_lens || !query_start_loc || !gk || !lse || !weights) return HKV_ERR_NULL;
  if ((D != 128 && D != 256) || (k8 && (D != 256 || signs))) return HKV_ERR_UNSUPPORTED;
  if (KVH < 1 || G < 1 || qlmax < 1 || (int64_t)G * qlmax > 64) return HKV_ERR_UNSUPPORTED;
  if (PS < 16 || (PS & (PS - 1)) != 0) return HKV_ERR_UNSUPPORTED;
  if (B > kMaxBatch) return HKV_ERR_RANGE;
  const int SD = D / 2, SS = D / 16;
  const int64_t dsp = strides[0], dst = strides[1], dsh = strides[2], ssp = strides[3], sst = strides[4], ssh = strides[5];
  const bool together = !k8 && sst == dst && dsp == ssp && dsh == ssh && (const uint8_t*)ksf == (const uint8_t*)kd + SD;
  int layout;
  if (k8) layout = 2;
  else if (together && dst == SD + SS) layout = 0;
  else if (dst == SD && sst == SS) layout = 1;
  else if (together) layout = 3;
  else return HKV_ERR_UNSUPPORTED;
  const int a = layout == 3 && D == 128 ? 7 : 15;
  if (((uintptr_t)kd | (uintptr_t)dsp | (uintptr_t)dsh | (layout >= 2 ? (uintptr_t)dst : 0)) & a) return HKV_ERR_ALIGN;
  if (layout == 1 && (((uintptr_t)ksf | (uintptr_t)ssp | (uintptr_t)ssh) & 15)) return HKV_ERR_ALIGN;
  if (((uintptr_t)q & 15) || (signs && ((uintptr_t)signs & 15)) || (((uintptr_t)lse | (uintptr_t)weights) & 3) ||
      ((uintptr_t)workspace & 255))
    return HKV_ERR_ALIGN;
  if (!rows_apart(B, KVH, W, w_b, w_h)) return HKV_ERR_UNSUPPORTED;
  if (dsp < 0 || ssp < 0 || dst < 0 || dsp >= (1ll << 31) || ssp >= (1ll << 31) || dst >= (1ll << 31)) return HKV_ERR_RANGE;
  if (!workspace) {
    const int rc = noalloc_workspace(&workspace);
    if (rc != HKV_OK) return rc;
  }
  WeightsParams p;
  p.q = (const __nv_bfloat16*)q;
  p.kd = (const uint8_t*)kd; p.ksf = (const uint8_t*)ksf;
  p.dsp = (unsigned)dsp; p.ssp = (unsigned)ssp; p.dst = dst; p.dsh = dsh; p.ssh = ssh;
  p.bt = block_tables; p.seq_lens = seq_lens; p.qsl = query_start_loc; p.gk = gk; p.lse = lse; p.signs = signs;
  p.w = weights; p.w_b = w_b; p.w_h = w_h;
  p.status = &((Header*)workspace)->status;
  p.MP = MP; p.B = B; p.KVH = KVH; p.G = G; p.qlmax = qlmax;
  p.lps = 0;
  while ((1 << p.lps) < PS) ++p.lps;
  p.max_len = (int)std::min((long long)MP * PS, 0x7fffff00ll);      // (a length beyond the table is cut there)
  p.W = W;
  p.window = window >= p.max_len ? 0 : window;            // (everything is seen)
  p.sinks = sinks;
  if (p.window > (1 << 30)) return HKV_ERR_RANGE;
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.rot_scale = (float)(1.0 / sqrt((double)D));
  cudaStream_t st = (cudaStream_t)stream;
  // query rows of a pass: 8, 16 or 32
  const int QT = G * qlmax <= 8 ? 1 : G * qlmax <= 16 ? 2 : 4;
  for (p.row0 = 0; p.row0 < G * qlmax; p.row0 += 8 * QT) {
    const int rc = QT == 1 ? launch_weights_any<1>(p, D, layout, st) : QT == 2 ? launch_weights_any<2>(p, D, layout, st)
                                                                         : launch_weights_any<4>(p, D, layout, st);
    if (rc != HKV_OK) return rc;
  }
  return HKV_OK;
}
