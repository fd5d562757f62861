// Eviction from the paged cache by gathered attention weight: per (request, kv head) the first `sinks` tokens, the last
// `recent` and, of those between, the heaviest stay, in their order; their slots move to the front of the sequence.
//
// Two launches:
//   select_kernel  which tokens stay. A cluster of 1 to 8 CTAs per (request, kv head) finds the weight of the last one by a radix
//                  selection over the fp32 values as ordered integers (11 + 11 + 10 bits): every CTA counts its share of the
//                  tokens into a shared-memory histogram, the CTAs read one another's through distributed shared memory and all
//                  come to the same digit. Two passes do unless weights agree in 22 bits. Ranks come from ballots and the counts
//                  of the warps and CTAs before; `kept` takes the positions in ascending order.
//   move_kernel    the kept tokens' slots and weights to their new places, byte for byte
// No sums are formed and nothing depends on an order of atomics: the histogram counts are whole numbers.
//
// In place (a request's new pages are its own first ones) one CTA may write a slot that another one reads. A token's rank never
// exceeds its position, so the moves are cut into rounds of ascending rank by ONE cluster per (request, kv head): a round's slots
// are all read before the first of them is written (cluster barrier between), and later rounds read positions that are at least
// as high as their ranks, above every rank written so far. Moves to other pages need no order: all warps work on their own.
#include <algorithm>
#include <type_traits>

#include "hkv_common.cuh"

namespace hkv {

int record_cuda(cudaError_t e);

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kEvBins = 2048;
constexpr int kEvCluster = 8;
constexpr int kSelRegs = 32;                        // weights of a thread that stay in registers
constexpr int kSmall = 32 * kSelRegs;               // tokens that one warp selects from
constexpr int kMoveThreads = 256, kMoveWarps = kMoveThreads / 32;

struct EvictParams {
  uint8_t* kd;
  uint8_t* ksf;
  uint8_t* vd;
  uint8_t* vsf;
  long long dsp, dst, dsh, ssp, sst, ssh;
  const int* bt;
  const int* out_bt;
  const int* seq_lens;
  int* out_lens;
  const float* w;
  float* ow;
  long long w_b, w_h, ow_b, ow_h;                   // element strides of the weights
  int* kept;
  int B, MP, OMP, lps, KVH, keep, sinks, recent, max_len, W, OW;
  int bulk, split;                                  // a tile's new rows lie back to back and 16-byte aligned; codes apart from scales
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();                                     // (.aligned: the warp's lanes come together)
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int peer_load(const int* p, uint32_t rank) {   // *p of another CTA of the cluster
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

__device__ __forceinline__ void peer_store(int* p, uint32_t rank, int v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
// sum of v over the lanes up to this one
__device__ __forceinline__ int scan_warp(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// The candidates are the tokens between the first and the last ones that have a weight: [sinks, this). Those without one are lighter
// than all of them, so that where the candidates are no more than may stay, the first tokens from `sinks` on stay
__device__ __forceinline__ int candidates_end(int L, int W, int sinks, int recent) { return min(L - recent, max(W, sinks)); }
// fp32 -> unsigned integers of the same order; both zeros are one, every NaN lies above infinity
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w);
  if (w != w) return 0xffffffffu;
  if (u == 0x80000000u) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// At most kSmall candidates, by one warp: the threshold bit by bit, every bit a count over the lanes' registers, no
// barrier. Right for more (request, kv head) pairs than the CTAs of select_kernel fill SMs in one wave: 2048 pairs of 300 tokens, 100 stay,
// 36 us against 80 (both launches), of 800 and 300 78 against 113; 512 of 300 19 against 22. A few pairs of 1000: 19 against 12.
__device__ __forceinline__ void select_small(const float* w, int W, int* kept, int lane, int L, int keep, int sinks, int recent) {
  const int n = min(L, keep);
  if (L <= keep) {
    for (int r = lane; r < keep; r += 32) kept[r] = r < n ? r : -1;
    return;
  }
  for (int i = lane; i < sinks; i += 32) kept[i] = i;
  for (int i = lane; i < recent; i += 32) kept[keep - recent + i] = L - recent + i;
  const int cnt = candidates_end(L, W, sinks, recent) - sinks, need = keep - sinks - recent, turns = (cnt + 31) >> 5;
  if (need >= cnt || need == 0) {
    for (int i = lane; i < need; i += 32) kept[sinks + i] = sinks + i;
    return;
  }
  w += sinks;
  uint32_t key[kSelRegs];
#pragma unroll
  for (int g = 0; g < kSelRegs; g += 8) {
    float x[8];
    if (g < turns) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = w[min(32 * (g + u) + lane, cnt - 1)];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) key[g + u] = g < turns && 32 * (g + u) + lane < cnt ? weight_key(x[u]) : 0u;
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int g = 0; g < kSelRegs; g += 4)
      if (g < turns) {
#pragma unroll
        for (int u = g; u < g + 4; ++u) f(u, key[u]);
      }
  };
  uint32_t low = 0;                                 // the need-th largest key, and whether others are equal to it
  bool ties = true;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit != 0 && ties; bit >>= 1) {
    int c = 0;
    each([&](int, uint32_t k) { c += k >= (low | bit); });
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= need) low |= bit;
    ties = c != need;                               // (else exactly those stay)
  }
  int left = 0;
  if (ties) {
    int c = 0;
    each([&](int, uint32_t k) { c += k > low; });
    left = need - __reduce_add_sync(0xffffffffu, c);
  } else {
    --low;
  }
  const unsigned below = (1u << lane) - 1;
  int gb = 0, eb = 0;
  kept += sinks;
  each([&](int u, uint32_t k) {
    const unsigned bg = __ballot_sync(0xffffffffu, k > low), be = __ballot_sync(0xffffffffu, ties && k == low);
    const int e = eb + __popc(be & below);
    if (k > low || (ties && k == low && e < left)) kept[gb + __popc(bg & below) + min(e, left)] = sinks + 32 * u + lane;
    gb += __popc(bg);
    eb += __popc(be);
  });
}
__global__ void __launch_bounds__(kMoveThreads) select_small_kernel(const EvictParams p) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, pair = blockIdx.x * kMoveWarps + (threadIdx.x >> 5);
  const int b = pair / p.KVH, h = pair - b * p.KVH;
  if (b >= p.B) return;
  const int L = min(max(__ldg(p.seq_lens + b), 0), p.max_len);
  if (h == 0 && lane == 0) p.out_lens[b] = min(L, p.keep);
  select_small(p.w + b * p.w_b + h * p.w_h, p.W, p.kept + (long long)pair * p.keep, lane, L, p.keep, p.sinks, p.recent);
}

// A warp has a run of the CTA's tokens, 32 at a time, a lane one of them: the order of (warp, turn, lane) is that of the tokens.
// The first kSelRegs turns stay in registers from pass to pass, further ones (contexts of more than 16384 tokens
// a CTA of the cluster) are read again, one by one.
// What bounds it: the longest context's chain of phases. One CTA, 14400 tokens (clocks): 7000 for the loads, 13000 for the first
// pass (shared-memory atomics; a weight's leading bits agree with several of its neighbours'), 1000 for each look at the bins, 1000
// for the second pass, 5000 for counts and ranks. Loads behind a branch each took 23000. 256 threads (one wave of CTAs where 512 take
// two) took 41 us instead of 27 for 64 requests of 1.5k to 16k tokens, 1024 threads 31 to 36: the long ones decide.
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(const EvictParams p) {
  __shared__ __align__(16) int hist[kEvBins];
  __shared__ int wsum[kSelWarps], counts[2 * kSelWarps], totals[2], found[3], slice;
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5;
  const int nc = (int)cluster_size(), cr = (int)cluster_rank(), h = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  const int L = min(max(__ldg(p.seq_lens + b), 0), p.max_len), n = min(L, p.keep);
  const float* w = p.w + b * p.w_b + h * p.w_h;
  int* kept = p.kept + ((long long)b * p.KVH + h) * p.keep;
  const int t0 = cr * kSelThreads + tid, step = nc * kSelThreads;
  if (cr == 0 && h == 0 && tid == 0) p.out_lens[b] = n;
  if (L <= p.keep) {                                // (the whole cluster leaves)
    for (int r = t0; r < p.keep; r += step) kept[r] = r < n ? r : -1;
    return;
  }
  for (int i = t0; i < p.sinks; i += step) kept[i] = i;
  for (int i = t0; i < p.recent; i += step) kept[p.keep - p.recent + i] = L - p.recent + i;
  // candidates, of which so many stay
  const int mid = candidates_end(L, p.W, p.sinks, p.recent) - p.sinks, need = p.keep - p.sinks - p.recent;
  if (need >= mid || need == 0) {                   // (again the whole cluster)
    for (int i = t0; i < need; i += step) kept[p.sinks + i] = p.sinks + i;
    return;
  }
  const int share = (mid + nc - 1) / nc, m0 = min(mid, cr * share), cnt = min(mid, m0 + share) - m0;
  const int turns = ((cnt + kSelWarps - 1) / kSelWarps + 31) >> 5;                   // of a warp
  const int i0 = wp * turns * 32 + lane, first = p.sinks + m0 + i0;                  // this lane's first token, of the CTA's and of all
  const float* wl = w + first;
  // (0: no token; no weight has this key)
  auto fetch = [&](int u) { return i0 + 32 * u < cnt ? weight_key(wl[32 * u]) : 0u; };
  uint32_t key[kSelRegs];
#pragma unroll
  for (int g = 0; g < kSelRegs; g += 8) {           // (eight loads at a time, none of them behind a branch)
    float x[8];
    if (g < turns) {
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = w[p.sinks + m0 + min(i0 + 32 * (g + u), cnt - 1)];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) key[g + u] = g + u < turns && i0 + 32 * (g + u) < cnt ? weight_key(x[u]) : 0u;
  }
  auto each = [&](auto f) {                         // f(turn, key) over this lane's tokens
#pragma unroll
    for (int g = 0; g < kSelRegs; g += 4)
      if (g < turns) {
#pragma unroll
        for (int u = g; u < g + 4; ++u) f(u, key[u]);
      }
#pragma unroll 1
    for (int u = kSelRegs; u < turns; ++u) f(u, fetch(u));
  };
  uint32_t prefix = 0;                              // the leading bits of the threshold
  int left = need, shift = 32;                      // tokens to take among those that share them
  bool ties = true;
#pragma unroll 1
  for (int pass = 0; pass < 3 && ties; ++pass) {
    const int from = shift, width = pass < 2 ? 11 : 10;
    shift -= width;
    reinterpret_cast<int4*>(hist)[tid] = make_int4(0, 0, 0, 0);
    __syncthreads();
    if (pass == 0) {
      each([&](int, uint32_t k) {
        if (k) atomicAdd(&hist[k >> 21], 1);
      });
    } else {
      const uint32_t mask = (1u << width) - 1;
      each([&](int, uint32_t k) {
        if (k >> from == prefix) atomicAdd(&hist[(k >> shift) & mask], 1);
      });
    }
    // The bin that holds the left-th key from the top, and how many of it are wanted. A CTA of a cluster sums up its share of the
    // bins over all CTAs and scans it; the one whose share holds the key tells the others.
    const int share_b = kEvBins / nc, nb = max(1, share_b / kSelThreads);              // bins of a CTA, of a thread (1, 2 or 4)
    if (nc == 1) __syncthreads(); else cluster_sync();
    int c[4] = {0, 0, 0, 0}, s = 0;
    const int top = kEvBins - 1 - cr * share_b - tid * nb;                             // this thread's bins, downwards
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < nb && tid < share_b) {
        if (nc == 1) c[u] = hist[top - u];
        else
          for (int r = 0; r < nc; ++r) c[u] += peer_load(hist + top - u, (cr + r) & (nc - 1));
        s += c[u];
      }
    const int incl = scan_warp(s, lane);
    if (lane == 31) wsum[wp] = incl;
    __syncthreads();
    int above = incl - s + __reduce_add_sync(0xffffffffu, lane < wp ? wsum[lane] : 0);
    if (nc > 1) {
      if (tid == kSelThreads - 1) slice = above + s;
      cluster_sync();
      above += __reduce_add_sync(0xffffffffu, lane < cr ? peer_load(&slice, lane) : 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u < nb && above < left && left <= above + c[u])
        for (int r = 0; r < nc; ++r) {
          peer_store(&found[0], r, top - u);
          peer_store(&found[1], r, left - above);
          peer_store(&found[2], r, c[u]);
        }
      above += c[u];
    }
    if (nc == 1) __syncthreads(); else cluster_sync();
    prefix = (prefix << width) | (uint32_t)found[0];
    left = found[1];
    ties = found[2] != left;                        // (else the whole bin stays)
  }
  // who stays: keys above `low`, and with ties (all 32 bits are known then) the first `left` of those equal to it
  const uint32_t low = ties ? prefix : (prefix << shift) - 1;
  int gt = 0, eq = 0;
  each([&](int, uint32_t k) {
    gt += k > low;
    eq += k == low;
  });
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    counts[2 * wp] = gt;
    counts[2 * wp + 1] = eq;
  }
  __syncthreads();
  // of the tokens before this warp's
  const int gw = lane < kSelWarps ? counts[2 * lane] : 0, ew = lane < kSelWarps ? counts[2 * lane + 1] : 0;
  int gb = __reduce_add_sync(0xffffffffu, lane < wp ? gw : 0), eb = __reduce_add_sync(0xffffffffu, lane < wp ? ew : 0);
  if (nc > 1) {
    if (wp == 0) {
      const int gt_all = __reduce_add_sync(0xffffffffu, gw), eq_all = __reduce_add_sync(0xffffffffu, ew);
      if (lane == 0) {
        totals[0] = gt_all;
        totals[1] = eq_all;
      }
    }
    cluster_sync();
    gb += __reduce_add_sync(0xffffffffu, lane < cr ? peer_load(&totals[0], lane) : 0);
    eb += __reduce_add_sync(0xffffffffu, lane < cr ? peer_load(&totals[1], lane) : 0);
  }
  const unsigned below = (1u << lane) - 1;
  if (!ties) {
    int r = p.sinks + gb;
    each([&](int u, uint32_t k) {
      const unsigned bg = __ballot_sync(0xffffffffu, k > low);
      if (k > low) kept[r + __popc(bg & below)] = first + 32 * u;
      r += __popc(bg);
    });
  } else {
    each([&](int u, uint32_t k) {
      const unsigned bg = __ballot_sync(0xffffffffu, k > low), be = __ballot_sync(0xffffffffu, k == low);
      const int er = eb + __popc(be & below);
      if (k > low || (k == low && er < left)) kept[p.sinks + gb + __popc(bg & below) + min(er, left)] = first + 32 * u;
      gb += __popc(bg);
      eb += __popc(be);
    });
  }
  if (nc > 1) cluster_sync();                       // (the totals have been read)
}

// A tile of moves: 16 tokens (8 at head_dim 256) whose new places lie in one 16-token block of a page. A warp gathers their rows
// into shared memory, piece by piece (PB bytes: 8 at head_dim 128, whose rows are 8-byte aligned, 16 at 256; a row is 8 pieces of codes, FP8 keys
// 16 before them, and one of scales), and writes the tile out: with one bulk copy a side where rows lie back to back in the
// cache, else piece by piece. The rows hold no registers on their way, so that a warp has the next tile in flight while it
// writes this one. 64 requests of 1.5k to 16k tokens cut to 2048, 8 kv heads x 128 (302 MB moved): 83 us with the rows in
// registers and 8-byte stores, which the L1 and the address arithmetic bound; 67 to 72 now (profiled), for 363 MB of DRAM traffic:
// rows of 72 bytes here and there cost whole 32-byte sectors. In one piece (nothing evicted) the launch moves the 302 MB in 54 us. Eight
// tokens a tile at head_dim 256, where sixteen leave room for fewer warps: 71 -> 65 us (8 requests of 131072 to 16384, 2 x 256).
template <int D, bool K8>
struct EvGeo {
  static constexpr int PB = D == 128 ? 8 : 16;
  static constexpr int NP = K8 ? 25 : 9;            // pieces of a row
  static constexpr int TOK = D == 128 ? 16 : 8;     // tokens of a tile
  static constexpr int ROWS = K8 ? TOK : 2 * TOK;   // rows of a tile: keys, then values (K8: both in one)
  static constexpr int PIECES = ROWS * NP, TURNS = (PIECES + 31) / 32;
  static constexpr int TILE = PIECES * PB;
  static constexpr int WARP = 2 * (TILE + 16 * TOK);               // shared memory of a warp: two tiles, the rows' old places (codes, scales)
};

__device__ __forceinline__ void bulk_s2g(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

// CLUSTER: calls in place; else a row in place, which the caller may mix in, is one CTA's work
template <int D, bool K8, bool CLUSTER, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, 32 / WARPS) move_kernel(const EvictParams p) {
  using Gm = EvGeo<D, K8>;
  constexpr int PB = Gm::PB, NP = Gm::NP, T = Gm::TOK;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5, h = blockIdx.y, b = blockIdx.z;
  const int L = min(max(__ldg(p.seq_lens + b), 0), p.max_len), n = min(L, p.keep);      // (older than the preceding launch)
  const int* bt = p.bt + (long long)b * p.MP;
  const int* obt = p.out_bt + (long long)b * p.OMP;
  pdl_wait();
  pdl_launch_dependents();
  if (n == 0) return;
  const float* w = p.w + b * p.w_b + h * p.w_h;
  float* ow = p.ow + b * p.ow_b + h * p.ow_h;
  const int* kept = p.kept + ((long long)b * p.KVH + h) * p.keep;
  const bool own_pages = __ldg(bt) == __ldg(obt), own_weights = ow == w, in_place = own_pages || own_weights;
  if (own_pages && own_weights && L <= p.keep) return;             // everything stays where it is
  const int cl = CLUSTER ? (int)cluster_size() : 1;
  if (in_place && (int)blockIdx.x >= cl) return;    // one cluster's work
  const int ctas = in_place ? cl : (int)gridDim.x, PSM = (1 << p.lps) - 1;
  const long long dh = h * p.dsh, sh = h * p.ssh;
  uint8_t* const mine = smem + wp * Gm::WARP;
  const uint32_t tiles_a = smem_u32(mine);
  long long* const places = reinterpret_cast<long long*>(mine + 2 * Gm::TILE);           // [tile][codes, scales][T]
  // piece x of a tile: its row, its place in the row, and where that lies in shared memory
  auto row_of = [](int x) { return x / NP; };
  auto base_of = [&](int row, int pc) -> uint8_t* {
    if (K8) return pc < 16 ? p.kd + pc * 16 : pc == 24 ? p.vsf : p.vd + (pc - 16) * 16;
    return pc == 8 ? (row < T ? p.ksf : p.vsf) : (row < T ? p.kd : p.vd) + pc * PB;
  };
  auto at = [&](int x, int row, int pc) {           // (split: codes and scales have regions of their own)
    return K8 || !p.split ? x * PB : pc < 8 ? row * 8 * PB + pc * PB : (2 * T * 8 + row) * PB;
  };
  // The old place of a token hangs on two loads one after the other (position, page), its rows on those: the positions are
  // fetched two tiles ahead, the rows one. (Every CTA of a cluster takes every round, so that all of them meet at its barrier.)
  const int stride = ctas * WARPS * T;
  int rt = (blockIdx.x * WARPS + wp) * T;
  auto position = [&](int r) { return lane < T && r + lane < n ? __ldg(kept + r + lane) : -1; };
  int j = position(rt);
  float wv = 0.0f, wn = 0.0f;
  bool still = false, still_n = false;              // (the tile stays where it is)
  auto gather = [&](int buf, int r, float& weight, bool& same) {      // the rows of tokens r .. r + T - 1, at positions j
    const int left = n - r;
    // (positions ascend: the tile's last one tells whether all of them are their ranks)
    same = own_pages && left >= T && __shfl_sync(0xffffffffu, j, T - 1) == r + T - 1;
    if (left > 0 && !same) {
      if (j >= 0) {
        const long long pg = __ldg(bt + (j >> p.lps));
        const int so = j & PSM;
        places[buf * 2 * T + lane] = pg * p.dsp + so * p.dst + dh;
        places[buf * 2 * T + T + lane] = pg * p.ssp + so * p.sst + sh;
      }
      __syncwarp();
#pragma unroll
      for (int u = 0; u < Gm::TURNS; ++u) {
        const int x = u * 32 + lane, row = row_of(x), pc = x - row * NP, i = row & (T - 1);
        const bool scales = pc == NP - 1;
        if ((Gm::PIECES % 32 == 0 || x < Gm::PIECES) && i < left)
          cp_async<PB>(tiles_a + buf * Gm::TILE + at(x, row, pc), base_of(row, pc) + places[buf * 2 * T + (scales ? T : 0) + i]);
      }
    }
    if (j >= 0) weight = j < p.W ? w[j] : 0.0f;
    asm volatile("cp.async.commit_group;" ::: "memory");
    j = position(r + stride);
  };
  gather(0, rt, wv, still);
  int buf = 0;
  for (int base = 0; base < n; base += stride, rt += stride, buf ^= 1) {
    // (the copy out of the other buffer, a turn ago, must have read it)
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    gather(buf ^ 1, rt + stride, wn, still_n);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (in_place) {
      if (CLUSTER) cluster_sync();
      else __syncthreads();
    }
    const int left = n - rt;
    if (left > 0 && !still) {
      const long long og = __ldg(obt + (rt >> p.lps));
      const int oo = rt & PSM;
      const long long to = og * p.dsp + oo * p.dst + dh, to_s = og * p.ssp + oo * p.sst + sh;
      const uint32_t tile = tiles_a + buf * Gm::TILE;
      if (p.bulk && left >= T) {
        fence_proxy_async();
        __syncwarp();
        if (K8) {
          if (lane == 0) bulk_s2g(p.kd + to, tile, Gm::TILE);
        } else if (!p.split) {
          if (lane < 2) bulk_s2g((lane ? p.vd : p.kd) + to, tile + lane * T * NP * PB, T * NP * PB);
        } else if (lane < 2) {
          bulk_s2g((lane ? p.vd : p.kd) + to, tile + lane * T * 8 * PB, T * 8 * PB);
          bulk_s2g((lane ? p.vsf : p.ksf) + to_s, tile + (2 * T * 8 + lane * T) * PB, T * PB);
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      } else {
        __syncwarp();
#pragma unroll 3
        for (int u = 0; u < Gm::TURNS; ++u) {
          const int x = u * 32 + lane, row = row_of(x), pc = x - row * NP, i = row & (T - 1);
          if ((Gm::PIECES % 32 == 0 || x < Gm::PIECES) && i < left) {
            uint8_t* d = base_of(row, pc) + (pc == NP - 1 ? to_s + i * p.sst : to + i * p.dst);
            const uint32_t s = tile + at(x, row, pc);
            if (PB == 8) *reinterpret_cast<uint2*>(d) = lds64(s);
            else *reinterpret_cast<uint4*>(d) = lds128(s);
          }
        }
      }
    }
    if (lane < T && rt + lane < n) ow[rt + lane] = wv;
    wv = wn;
    still = still_n;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  // (in place: the last barrier lies behind every read)
  for (int r = n + blockIdx.x * 32 * WARPS + tid; r < min(L, p.OW); r += ctas * 32 * WARPS) ow[r] = 0.0f;
}

template <typename K>
static int launch_clusters(K k, const EvictParams& p, unsigned x, unsigned y, unsigned z, unsigned cluster, int threads, size_t smem,
                           cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(x, y, z);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return record_cuda(cudaLaunchKernelEx(&cfg, k, p));
}

}  // namespace hkv

extern "C" int hkv_evict(void* kd, void* ksf, void* vd, void* vsf, const int64_t strides[6], int PS, const int32_t* block_tables,
                         int MP, const int32_t* seq_lens, int B, int KVH, int D, int k8, const float* weights, int64_t w_b,
                         int64_t w_h, int W, int keep, int sinks, int recent, const int32_t* out_tables, int OMP, int32_t* kept,
                         int32_t* out_lens, float* out_weights, int64_t ow_b, int64_t ow_h, int OW, void* stream) {
  using namespace hkv;
  if (B < 0 || MP < 0 || OMP < 0 || W < 0 || OW < 0) return HKV_ERR_RANGE;
  if (B == 0) return HKV_OK;
  if (!kd || !ksf || !vd || !vsf || !strides || !block_tables || !seq_lens || !weights || !out_tables || !kept || !out_lens ||
      !out_weights)
    return HKV_ERR_NULL;
  if ((D != 128 && D != 256) || (k8 && D != 256)) return HKV_ERR_UNSUPPORTED;
  if (KVH < 1 || KVH > 1024 || PS < 16 || (PS & (PS - 1))) return HKV_ERR_UNSUPPORTED;
  if (B > kMaxBatch) return HKV_ERR_RANGE;
  if (keep < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep) return HKV_ERR_RANGE;
  if ((int64_t)keep > (int64_t)OMP * PS || keep > OW) return HKV_ERR_RANGE;      // the new pages, the new weights
  auto apart = [](uintptr_t x, int64_t nx, uintptr_t y, int64_t ny) {      // of so many 4-byte numbers each
    return x + 4 * (uintptr_t)nx <= y || y + 4 * (uintptr_t)ny <= x;
  };
  // other heads read the old length while the new one is written
  if (!apart((uintptr_t)seq_lens, B, (uintptr_t)out_lens, B)) return HKV_ERR_UNSUPPORTED;
  const uintptr_t a = (uintptr_t)kd | (uintptr_t)vd | (uintptr_t)vsf | (k8 ? 0 : (uintptr_t)ksf) | (uintptr_t)strides[0] |
                      (uintptr_t)strides[1] | (uintptr_t)strides[2] | (uintptr_t)strides[3] | (uintptr_t)strides[4] |
                      (uintptr_t)strides[5];
  if (a & (D == 128 ? 7 : 15)) return HKV_ERR_ALIGN;
  if (((uintptr_t)weights | (uintptr_t)out_weights) & 3) return HKV_ERR_ALIGN;
  if (!rows_apart(B, KVH, OW, ow_b, ow_h)) return HKV_ERR_UNSUPPORTED;
  // new weights where the old ones are read: only in place, rank by rank
  const bool same = weights == out_weights && (B == 1 || w_b == ow_b) && (KVH == 1 || w_h == ow_h);
  if (!same && !apart((uintptr_t)weights, (B - 1) * w_b + (KVH - 1) * w_h + W, (uintptr_t)out_weights, (B - 1) * ow_b + (KVH - 1) * ow_h + OW))
    return HKV_ERR_UNSUPPORTED;
  EvictParams p;
  p.kd = (uint8_t*)kd; p.ksf = (uint8_t*)ksf; p.vd = (uint8_t*)vd; p.vsf = (uint8_t*)vsf;
  p.dsp = strides[0]; p.dst = strides[1]; p.dsh = strides[2];
  p.ssp = strides[3]; p.sst = strides[4]; p.ssh = strides[5];
  p.bt = block_tables; p.out_bt = out_tables; p.seq_lens = seq_lens; p.out_lens = out_lens;
  p.w = weights; p.ow = out_weights; p.w_b = w_b; p.w_h = w_h; p.ow_b = ow_b; p.ow_h = ow_h;
  p.kept = kept;
  p.B = B; p.MP = MP; p.OMP = OMP; p.KVH = KVH; p.keep = keep; p.sinks = sinks; p.recent = recent; p.OW = OW;
  // rows back to back, and bulk copies' 16-byte alignment (a tile begins at a multiple of 16 tokens)
  const int64_t SD = k8 ? D + D / 2 : D / 2, SS = D / 16, row = SD + SS;
  const bool al16 = (((uintptr_t)kd | (uintptr_t)vd | (uintptr_t)strides[0] | (uintptr_t)strides[2]) & 15) == 0;
  const bool together = strides[1] == row && strides[4] == row && strides[0] == strides[3] && strides[2] == strides[5];
  const bool slots = k8 ? together && (uint8_t*)vd == (uint8_t*)kd + D && (uint8_t*)vsf == (uint8_t*)vd + D / 2
                        : together && (uint8_t*)ksf == (uint8_t*)kd + SD && (uint8_t*)vsf == (uint8_t*)vd + SD;
  p.split = !k8 && !slots && strides[1] == SD && strides[4] == SS &&
            (((uintptr_t)ksf | (uintptr_t)vsf | (uintptr_t)strides[3] | (uintptr_t)strides[5]) & 15) == 0;
  p.bulk = al16 && (slots || p.split);
  p.split = p.split && p.bulk;
  p.lps = 0;
  while ((1 << p.lps) < PS) ++p.lps;
  p.max_len = (int)std::min((long long)MP * PS, 0x7fffff00ll);      // (a length beyond the table is cut there)
  p.W = W;
  const int widest = p.max_len < W ? p.max_len : W;       // tokens to select from
  const long long pairs = (long long)B * KVH;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return record_cuda(e);
  // CTAs per (request, kv head) for the selection. A cluster divides the work of a long context but meets four times a pass, and one
  // CTA holds 16384 weights in registers. Both launches, one CTA and four (us): a request of 8 heads x 128, 8192 tokens 21.2 and 21.5,
  // 10240 21.5 and 23.5, 12288 23.7 and 25.0, 14336 25.6 and 25.6, 16384 25.6 and 23.5, 24576 42 and 26; 8 requests of 2 x 256 23.5 and
  // 25.6, 27.6 and 27.8, 29.7 and 29.7, 29.7 and 27.7, 32.6 and 31.7, 50 and 34. Two are slower than one as long as that one's registers
  // do (16 requests of 8 x 128, 16384 tokens 68.6 and 70.7, 24576 105 and 95). No more CTAs than two an SM, which run at once: 128 pairs
  // to 20000 tokens take 50.9 us with two each, 60.8 with four; 512 pairs 107 with one each, 121 with two.
  int nc = kEvCluster;
  while (nc > 1 && (pairs * nc > 2 * sms || widest < nc * 2048 || widest <= (nc == 2 ? kSelThreads * kSelRegs : 12288))) nc /= 2;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = widest <= kSmall && pairs > 2 * sms ? record_cuda(launch_pdl(select_small_kernel, dim3((unsigned)((pairs + kMoveWarps - 1) / kMoveWarps)),
                                                        dim3(kMoveThreads), 0, st, p))
                               : launch_clusters(select_kernel, p, nc, KVH, B, nc, kSelThreads, 0, st);
  if (rc != HKV_OK) return rc;
  const int T = D == 128 ? 16 : 8, warp_smem = k8 ? EvGeo<256, true>::WARP : D == 128 ? EvGeo<128, false>::WARP : EvGeo<256, false>::WARP;
  const long long most = keep < p.max_len ? keep : p.max_len;
  void (*mk)(const EvictParams) = nullptr;
  if (out_tables == block_tables || out_weights == weights) {
    // In place: a cluster per (request, kv head), no larger than a round's work and no more CTAs than fill the GPU (512 pairs to 2048
    // tokens: 105 us with two CTAs a cluster, 112 with eight). A round waits for its slowest read, so few pairs with many rounds take
    // as many warps as fit: 16 pairs to 16384 tokens at head_dim 256 167 -> 125 us (to other pages 65), to 7000 at 128 36 -> 31; two
    // rounds gain nothing (2048 tokens: 18.9 -> 21.5).
    int nm = kEvCluster;
    while (nm > 1 && (nm / 2 * kMoveWarps * T >= most || pairs * nm > 4 * sms)) nm /= 2;
    const bool wide = pairs * nm <= sms && most > 4 * nm * kMoveWarps * T;
    if (k8) mk = wide ? move_kernel<256, true, true, 32> : move_kernel<256, true, true, kMoveWarps>;
    else if (D == 128) mk = wide ? move_kernel<128, false, true, 32> : move_kernel<128, false, true, kMoveWarps>;
    else mk = wide ? move_kernel<256, false, true, 32> : move_kernel<256, false, true, kMoveWarps>;
    const int warps = wide ? 32 : kMoveWarps;
    rc = record_cuda(cudaFuncSetAttribute((const void*)mk, cudaFuncAttributeMaxDynamicSharedMemorySize, warps * warp_smem));
    return rc != HKV_OK ? rc : launch_clusters(mk, p, nm, KVH, B, nm, 32 * warps, (size_t)warps * warp_smem, st);
  }
  if (k8) mk = move_kernel<256, true, false, kMoveWarps>;
  else mk = D == 128 ? move_kernel<128, false, false, kMoveWarps> : move_kernel<256, false, false, kMoveWarps>;
  const int smem = kMoveWarps * warp_smem;
  rc = record_cuda(cudaFuncSetAttribute((const void*)mk, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (rc != HKV_OK) return rc;
  // As many CTAs as run at once, four an SM, or as find work at once; rounded down, since a few behind the first wave cost as much as
  // another wave (160 pairs to 20000 tokens: 592 / 160 up 70.4 us, down 59.9; 128 pairs 50.9, 44.4), but two a pair while there are
  // fewer than four pairs an SM (512 pairs to 2048 tokens: one each 104.5, two 98.2).
  const long long round = kMoveWarps * T, fit = std::max(4 * sms / pairs, std::min(2ll, (4 * sms + pairs - 1) / pairs));
  const long long x = std::max(1ll, std::min((most + round - 1) / round, fit));
  return record_cuda(launch_pdl(mk, dim3((unsigned)x, (unsigned)KVH, (unsigned)B), dim3(kMoveThreads), smem, st, p));
}
