// Eviction from the paged cache by gathered attention weight: per (request, kv head) the first `sinks` tokens, the last
// `recent` and, of those between, the heaviest stay, in their order; their slots move to the front of the sequence.
//
// One cluster of 1 to 8 CTAs per (request, kv head) does all of it in one launch:
//   select   the weight that the last token to stay has, by a radix selection over the fp32 values as ordered integers
//            (11 + 11 + 10 bits). Every CTA counts its share of the tokens into a shared-memory histogram; the CTAs read one
//            another's through distributed shared memory and all come to the same digit.
//   list     which tokens stay, ascending: ranks from ballots and the counts of the warps and CTAs before, written to `kept`
//   move     the kept tokens' slots and weights to their new places, byte for byte
// No sums are formed and nothing depends on an order of atomics: the histogram counts are whole numbers.
//
// In place (a request's new pages are its own first ones) a slot may be read by one CTA and written by another. A token's rank
// never exceeds its position, so the moves are cut into rounds of ascending rank, a round's slots are all read before the first
// of them is written (cluster barrier between), and what a round writes lies at or below every position that later rounds read
// only where it has been read already: position j of rank r' >= r(round end) > any rank written so far.
#include <type_traits>

#include "hkv_common.cuh"

namespace hkv {

int record_cuda(cudaError_t e);

constexpr int kEvThreads = 512, kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048;
constexpr int kEvCluster = 8;
constexpr int kEvKeys = 20480;                      // weights that a CTA keeps in shared memory (80 KB; the rest is read again)

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
  int MP, OMP, lps, KVH, keep, sinks, recent, max_len, OW, cap;
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
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int peer_load(const int* p, uint32_t rank) {   // *p of another CTA of the cluster
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// fp32 -> unsigned integers of the same order; both zeros are one, every NaN lies above infinity
__device__ __forceinline__ uint32_t weight_key(float w) {
  const uint32_t u = __float_as_uint(w);
  if (w != w) return 0xffffffffu;
  if (u == 0x80000000u) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// PB: bytes of a piece of a slot (8 at head_dim 128, whose rows are 8-byte aligned; 16 at 256). A slot's side is NP pieces of
// codes (FP8 keys: 16) and one of scales; NP + 1 lanes copy a side.
template <int D, bool K8>
struct EvGeo {
  static constexpr int PB = D == 128 ? 8 : 16;
  static constexpr int NP = 8;                      // pieces of D / 2 code bytes
  static constexpr int LANES = K8 ? 16 + NP + 1 : 3 * (NP + 1);      // a token; or three sides of tokens
  static constexpr int SIDES = K8 ? 1 : 3;          // sides (K8: tokens) a warp copies at a time
  static constexpr int U = 8;                       // of those in flight
  static constexpr int TOK = K8 ? U : U * 3 / 2;    // tokens of a warp and round
};

template <int D, bool K8>
__global__ void __launch_bounds__(kEvThreads, 2) evict_kernel(const EvictParams p) {
  using Gm = EvGeo<D, K8>;
  using Piece = typename std::conditional<Gm::PB == 8, uint2, uint4>::type;
  extern __shared__ uint32_t keys[];
  __shared__ int hist[kEvBins];
  __shared__ int wsum[kEvWarps], counts[2 * kEvWarps], totals[2], found[3];
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5;
  const int nc = (int)cluster_size(), cr = (int)cluster_rank(), h = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_launch_dependents();
  const int L = min(max(__ldg(p.seq_lens + b), 0), p.max_len), n = min(L, p.keep);
  const float* w = p.w + b * p.w_b + h * p.w_h;
  float* ow = p.ow + b * p.ow_b + h * p.ow_h;
  int* kept = p.kept + ((long long)b * p.KVH + h) * p.keep;
  const int* bt = p.bt + (long long)b * p.MP;
  const int* obt = p.out_bt + (long long)b * p.OMP;
  if (cr == 0 && h == 0 && tid == 0) p.out_lens[b] = n;

  if (L <= p.keep) {
    for (int r = cr * kEvThreads + tid; r < p.keep; r += nc * kEvThreads) kept[r] = r < n ? r : -1;
  } else {
    const int mid = L - p.sinks - p.recent, need = p.keep - p.sinks - p.recent;      // candidates, of which so many stay
    const int share = (mid + nc - 1) / nc, m0 = min(mid, cr * share), m1 = min(mid, m0 + share), first = p.sinks + m0, cnt = m1 - m0;
    for (int i = tid; i < cnt; i += kEvThreads)
      if (i < p.cap) keys[i] = weight_key(w[first + i]);
    auto key = [&](int i) { return i < p.cap ? keys[i] : weight_key(w[first + i]); };
    uint32_t prefix = 0;                            // the leading bits of the threshold
    int left = need, shift = 32;                    // tokens to take among those that share them
    const int widths[3] = {11, 11, 10};
#pragma unroll 1
    for (int pass = 0; pass < 3 && need > 0; ++pass) {
      const int from = shift;
      shift -= widths[pass];
      for (int i = tid; i < kEvBins; i += kEvThreads) hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < cnt; i += kEvThreads) {
        const uint32_t k = key(i);
        if (from == 32 || k >> from == prefix) atomicAdd(&hist[(k >> shift) & ((1 << widths[pass]) - 1)], 1);
      }
      cluster_sync();
      // the bins of all CTAs; thread t has the bins 4 t .. 4 t + 3 counted from the top
      int c[4], s = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int bin = kEvBins - 1 - (4 * tid + u);
        c[u] = 0;
        for (int r = 0; r < nc; ++r) c[u] += peer_load(&hist[bin], (cr + r) % nc);
        s += c[u];
      }
      int incl = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      if (lane == 31) wsum[wp] = incl;
      __syncthreads();
      int above = incl - s;
      for (int i = 0; i < wp; ++i) above += wsum[i];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (above < left && left <= above + c[u]) {
          found[0] = kEvBins - 1 - (4 * tid + u);
          found[1] = left - above;
          found[2] = c[u];
        }
        above += c[u];
      }
      cluster_sync();                               // (the histograms have been read)
      prefix = (prefix << widths[pass]) | (uint32_t)found[0];
      left = found[1];
      if (found[2] == left) break;                  // the whole bin stays
    }
    // who stays: key >> shift above the prefix, and the first `left` of those equal to it
    auto rel = [&](int i) {                         // 2: above, 1: equal, 0: below
      if (need == 0) return 0;
      const uint32_t k = key(i) >> shift;
      return k > prefix ? 2 : k == prefix ? 1 : 0;
    };
    const int part = (cnt + kEvWarps - 1) / kEvWarps, i0 = min(cnt, wp * part), i1 = min(cnt, i0 + part);
    int gt = 0, eq = 0;
    for (int i = i0; i < i1; i += 32) {
      const int v = i + lane < i1 ? rel(i + lane) : 0;
      gt += __popc(__ballot_sync(0xffffffffu, v == 2));
      eq += __popc(__ballot_sync(0xffffffffu, v == 1));
    }
    if (lane == 0) {
      counts[2 * wp] = gt;
      counts[2 * wp + 1] = eq;
    }
    __syncthreads();
    if (tid < 2) {
      int t = 0;
      for (int i = 0; i < kEvWarps; ++i) t += counts[2 * i + tid];
      totals[tid] = t;
    }
    cluster_sync();
    int gb = 0, eb = 0;
    for (int r = 0; r < cr; ++r) {
      gb += peer_load(&totals[0], r);
      eb += peer_load(&totals[1], r);
    }
    for (int i = 0; i < wp; ++i) {
      gb += counts[2 * i];
      eb += counts[2 * i + 1];
    }
    const unsigned below = (1u << lane) - 1;
    for (int i = i0; i < i1; i += 32) {
      const int v = i + lane < i1 ? rel(i + lane) : 0;
      const unsigned bg = __ballot_sync(0xffffffffu, v == 2), be = __ballot_sync(0xffffffffu, v == 1);
      const int g = gb + __popc(bg & below), e = eb + __popc(be & below);
      if (v == 2 || (v == 1 && e < left)) kept[p.sinks + g + min(e, left)] = first + i + lane;
      gb += __popc(bg);
      eb += __popc(be);
    }
    for (int i = cr * kEvThreads + tid; i < p.sinks; i += nc * kEvThreads) kept[i] = i;
    for (int i = cr * kEvThreads + tid; i < p.recent; i += nc * kEvThreads) kept[p.keep - p.recent + i] = L - p.recent + i;
  }
  cluster_sync();                                   // the list is complete, also where another CTA wrote it

  if (n > 0) {
    // a request's own first pages, or weights that move within their row: read before written
    const bool in_place = ow == w || __ldg(bt) == __ldg(obt);
    const int PSM = (1 << p.lps) - 1;
    const long long dh = h * p.dsh, sh = h * p.ssh;
    // what this lane copies of a (token, side): pieces 0 .. 7 codes, 8 scales; K8: 0 .. 15 keys, then the same of the values
    const int sub = K8 ? 0 : lane / (Gm::NP + 1), pc = K8 ? lane : lane - sub * (Gm::NP + 1);
    const bool on = lane < Gm::LANES;
    constexpr int ROUND = kEvWarps * Gm::TOK;
    for (int r0 = cr * ROUND; r0 - cr * ROUND < n; r0 += nc * ROUND) {
      Piece v[Gm::U];
      uint8_t* to[Gm::U];
      const int rw = r0 + wp * Gm::TOK;
#pragma unroll
      for (int u = 0; u < Gm::U; ++u) {
        const int item = u * Gm::SIDES + sub, r = rw + (K8 ? item : item >> 1), side = K8 ? 0 : item & 1;
        to[u] = nullptr;
        if (on && r < n) {
          const int j = __ldcg(kept + r);
          const long long pg = __ldg(bt + (j >> p.lps)), og = __ldg(obt + (r >> p.lps));
          const int so = j & PSM, oo = r & PSM;
          const bool scales = K8 ? pc == 24 : pc == 8;
          uint8_t* base;
          if (K8) base = pc < 16 ? p.kd + pc * 16 : scales ? p.vsf : p.vd + (pc - 16) * 16;
          else base = scales ? (side ? p.vsf : p.ksf) : (side ? p.vd : p.kd) + pc * Gm::PB;
          const uint8_t* from;
          if (scales) {
            from = base + pg * p.ssp + so * p.sst + sh;
            to[u] = base + og * p.ssp + oo * p.sst + sh;
          } else {
            from = base + pg * p.dsp + so * p.dst + dh;
            to[u] = base + og * p.dsp + oo * p.dst + dh;
          }
          if (from == to[u]) to[u] = nullptr;       // it stays where it is
          else v[u] = *reinterpret_cast<const Piece*>(from);
        }
      }
      float wv = 0.0f;
      const int rt = rw + lane;
      const bool mine = lane < Gm::TOK && rt < n;
      if (mine) wv = w[__ldcg(kept + rt)];
      if (in_place) cluster_sync();
#pragma unroll
      for (int u = 0; u < Gm::U; ++u)
        if (to[u]) *reinterpret_cast<Piece*>(to[u]) = v[u];
      if (mine) ow[rt] = wv;
    }
    // (CTAs beyond the last round's ranks have nothing to read but meet the others at every barrier: the loop's bound is the
    // cluster's first rank of the round)
  }
  for (int r = n + cr * kEvThreads + tid; r < min(L, p.OW); r += nc * kEvThreads) ow[r] = 0.0f;
}

template <int D, bool K8>
static int launch_evict(const EvictParams& p, int B, int nc, size_t smem, cudaStream_t st) {
  auto k = evict_kernel<D, K8>;
  int rc = record_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvKeys * 4));
  if (rc != HKV_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)nc, (unsigned)p.KVH, (unsigned)B);
  cfg.blockDim = dim3(kEvThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)nc;
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
  if (seq_lens == out_lens) return HKV_ERR_UNSUPPORTED;   // other heads read the old length while the new one is written
  const uintptr_t a = (uintptr_t)kd | (uintptr_t)vd | (uintptr_t)vsf | (k8 ? 0 : (uintptr_t)ksf) | (uintptr_t)strides[0] |
                      (uintptr_t)strides[1] | (uintptr_t)strides[2] | (uintptr_t)strides[3] | (uintptr_t)strides[4] |
                      (uintptr_t)strides[5];
  if (a & (D == 128 ? 7 : 15)) return HKV_ERR_ALIGN;
  if (((uintptr_t)weights | (uintptr_t)out_weights) & 3) return HKV_ERR_ALIGN;
  EvictParams p;
  p.kd = (uint8_t*)kd; p.ksf = (uint8_t*)ksf; p.vd = (uint8_t*)vd; p.vsf = (uint8_t*)vsf;
  p.dsp = strides[0]; p.dst = strides[1]; p.dsh = strides[2];
  p.ssp = strides[3]; p.sst = strides[4]; p.ssh = strides[5];
  p.bt = block_tables; p.out_bt = out_tables; p.seq_lens = seq_lens; p.out_lens = out_lens;
  p.w = weights; p.ow = out_weights; p.w_b = w_b; p.w_h = w_h; p.ow_b = ow_b; p.ow_h = ow_h;
  p.kept = kept;
  p.MP = MP; p.OMP = OMP; p.KVH = KVH; p.keep = keep; p.sinks = sinks; p.recent = recent; p.OW = OW;
  p.lps = 0;
  while ((1 << p.lps) < PS) ++p.lps;
  const long long reach = (long long)MP * PS;
  p.max_len = (int)(reach < W ? reach : W);               // (a length beyond the table or the weights is cut there)
  const long long pairs = (long long)B * KVH;
  int nc = kEvCluster;
  while (nc > 1 && (pairs * nc > 600 || p.max_len < nc * 1024)) nc /= 2;
  const int share = (p.max_len + nc - 1) / nc;
  p.cap = share < kEvKeys ? share : kEvKeys;
  const size_t smem = (size_t)(p.cap > 0 ? p.cap : 1) * 4;
  cudaStream_t st = (cudaStream_t)stream;
  return k8 ? launch_evict<256, true>(p, B, nc, smem, st)
            : D == 128 ? launch_evict<128, false>(p, B, nc, smem, st) : launch_evict<256, false>(p, B, nc, smem, st);
}
