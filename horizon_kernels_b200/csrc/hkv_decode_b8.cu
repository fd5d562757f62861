// Decode attention over the 8-bit cache: tiles of 16 tokens of one kv head and side, D code bytes a token (E4M3 or int8, 16-byte
// chunk j of token t at chunk j ^ (t % 8)) and one power-of-two scale a tile (include/hkv.h).
//
// The kernels are the decode kernel's body (hkv_decode.cu: stream of units cut into equal partitions, private rings of bulk copies,
// S^T = K Q^T and O^T += V^T P^T with mma.m16n8k16, merge inside the launch) over this layout. What differs:
//   * a code is converted to f16 and used as it is. The key scale of a block multiplies its scores; the value scale enters the
//     exponent of the weights, p = 2^(s + e_v - max), and the sum of the weights takes it out again, so that neither costs an
//     instruction per element. Both are exact; a weight, f16, keeps its 11 bits down to 2^-14 of the largest product of a weight and
//     a value scale, and is off by at most 2^-25 of that product below.
//   * the chunks of a tile are permuted in the cache, so that a bulk copy brings rows of 128 or 256 bytes whose 16-byte loads touch every
//     bank once, both along the channels (keys) and along the tokens (values).
//
// B200, back to back: 8 requests of 65536 tokens, 8 kv heads x 128, group 8, 174 us (6.2 TB/s, 0.95 of a copy), 64 of 1024 to 32768 197
// (0.93); 96 of 500 to 16384, 2 x 256, group 8, 85 (0.81), with two query tokens 95 (int8: 97). The memory bounds the long ones; the
// others lose 10 to 15 us to the start and the end of the launch, sixteen rows at head_dim 256 also to dependency latency at 255 registers
// and eight warps an SM. More than sixteen rows read the cache once per sixteen: 64 of 1024 to 16384, 8 x 128, group 8, with 1 / 2 / 4 query
// tokens 125 / 132 / 264.
#include <algorithm>
#include <atomic>
#include <mutex>

#define HKV_DECODE_BODY_ONLY
#include "hkv_decode.cu"

namespace hkv {

template <int D, int LAYOUT, int QT, bool WIN>
__global__ void __launch_bounds__(NTHREADS, QT == 2 ? 2 : Geo<D, LAYOUT>::MINB) b8_kernel(const DecodeParams p) {
  decode_body<D, LAYOUT, QT, WIN>(p);
}

struct B8Variant {
  void (*kernel)(const DecodeParams);
  int smem, most;                                    // most: CTAs per SM that the decode workspace is sized for
};
template <int D, int LAYOUT, int QT, bool WIN>
static B8Variant variant() {
  return {b8_kernel<D, LAYOUT, QT, WIN>, Smem<D, LAYOUT, QT>::TOTAL, QT == 2 ? 2 : Geo<D, LAYOUT>::MINB};
}
// (sixteen rows at head_dim 128 in units of 32 tokens: 64 requests of 500 to 8000 tokens, group 8 x 2 query tokens, 79 us, 85 in units of 16)
template <int D, int FMT>
static B8Variant variant_of(bool two, bool win) {
  constexpr int L1 = 4 + FMT, L2 = (D == 128 ? 6 : 4) + FMT;
  return two ? (win ? variant<D, L2, 2, true>() : variant<D, L2, 2, false>())
             : win ? variant<D, L1, 1, true>() : variant<D, L1, 1, false>();
}
static B8Variant variant_of(int D, int fmt, bool two, bool win) {
  return D == 128 ? (fmt ? variant_of<128, 1>(two, win) : variant_of<128, 0>(two, win))
                  : fmt ? variant_of<256, 1>(two, win) : variant_of<256, 0>(two, win);
}

struct B8Device {
  int sms = 0;
  int ctas[2][2][2][2];                              // [D == 256][fmt][two][win]
  std::atomic<bool> ready{false};
};
static B8Device g_b8_dev[64];
static std::mutex g_b8_mutex;

static int b8_device(const B8Device** out) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return record_cuda(e);
  if (dev < 0 || dev >= 64) return HKV_ERR_RANGE;
  B8Device& d = g_b8_dev[dev];
  if (!d.ready.load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(g_b8_mutex);
    if (!d.ready.load(std::memory_order_relaxed)) {
      e = cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev);
      if (e != cudaSuccess) return record_cuda(e);
      for (int i = 0; i < 16; ++i) {
        const B8Variant v = variant_of(i & 8 ? 256 : 128, i >> 2 & 1, i & 2, i & 1);
        int n = 0;
        e = cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem);
        if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, v.kernel, NTHREADS, v.smem);
        if (e != cudaSuccess) return record_cuda(e);
        d.ctas[i >> 3][i >> 2 & 1][i >> 1 & 1][i & 1] = std::min(n, v.most);
      }
      d.ready.store(true, std::memory_order_release);
    }
  }
  *out = &d;
  return HKV_OK;
}

}  // namespace hkv

extern "C" int hkv_decode_b8(const void* q, const void* kt, const void* vt, const int64_t strides[2], int PS,
                             const int32_t* block_tables, int MP, const int32_t* seq_lens, const int32_t* query_start_loc, int B,
                             int KVH, int G, int D, int qlmax, float sm_scale, float v_scale, const float* gk, const float* gv,
                             void* workspace, size_t workspace_bytes, int splits, int fmt, int window, int sinks, float* lse,
                             void* out, void* stream) {
  using namespace hkv;
  if (B < 0 || MP < 0 || window < 0 || sinks < 0) return HKV_ERR_RANGE;
  if (B == 0) return HKV_OK;
  if (!q || !kt || !vt || !strides || !block_tables || !seq_lens || !query_start_loc || !gk || !gv || !workspace || !out)
    return HKV_ERR_NULL;
  if ((D != 128 && D != 256) || (fmt != HKV_B8_E4M3 && fmt != HKV_B8_INT8)) return HKV_ERR_UNSUPPORTED;
  if (KVH < 1 || G < 1 || qlmax < 1 || G > kMaxRows || qlmax > kMaxRows || G * qlmax > kMaxRows) return HKV_ERR_UNSUPPORTED;
  if (PS < 16 || (PS & (PS - 1)) != 0) return HKV_ERR_UNSUPPORTED;
  if (B > kMaxBatch || splits < 0) return HKV_ERR_RANGE;
  if (splits > 64) return HKV_ERR_SPLITS;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)kt | (uintptr_t)vt) & 15) return HKV_ERR_ALIGN;
  if ((strides[0] | strides[1]) & 15) return HKV_ERR_ALIGN;
  if (((uintptr_t)workspace & 255) || ((uintptr_t)lse & 3)) return HKV_ERR_ALIGN;
  if (strides[0] < 0 || strides[0] >= (1ll << 31)) return HKV_ERR_RANGE;       // a page is far below 2 GB
  if ((long long)window >= (long long)MP * PS) window = 0;                     // everything is seen
  if (window > (1 << 30)) return HKV_ERR_RANGE;
  const B8Device* dev;
  int rc = b8_device(&dev);
  if (rc != HKV_OK) return rc;
  const bool win = window > 0 || lse != nullptr;
  auto parts_of = [&](int cps) {
    long long n = std::min<long long>((long long)dev->sms * cps, kMaxParts);
    if (splits > 0) n = std::min<long long>(n, (long long)B * KVH * splits);
    return n < 1 ? 1 : n;
  };
  // more than eight query rows per kv head: sixteen a pass, where the workspace holds their partials
  const int two_tiles = dev->ctas[D == 256][fmt][1][win];
  const bool two = G * qlmax > RPAD && two_tiles > 0 &&
                   workspace_bytes >= WorkspaceLayout((int)parts_of(two_tiles), 2 * RPAD, D).total;
  const int rows_per_pass = two ? 2 * RPAD : RPAD, cps = two ? two_tiles : dev->ctas[D == 256][fmt][0][win];
  if (cps < 1) return HKV_ERR_UNSUPPORTED;
  const long long n_parts = parts_of(cps);
  if (workspace_bytes < WorkspaceLayout((int)n_parts, rows_per_pass, D).total) return HKV_ERR_WORKSPACE;
  DecodeParams p = {};
  p.q = (const __nv_bfloat16*)q;
  p.kd = p.ksf = (const uint8_t*)kt;
  p.vd = p.vsf = (const uint8_t*)vt;
  p.dsp = p.ssp = (unsigned)strides[0];
  p.dsh = p.ssh = strides[1];
  p.bt = block_tables; p.seq_lens = seq_lens; p.qsl = query_start_loc;
  p.gk = gk; p.gv = gv;
  p.ws = (uint8_t*)workspace;
  p.out = (__nv_bfloat16*)out;
  p.MP = MP; p.B = B; p.KVH = KVH; p.G = G; p.qlmax = qlmax; p.PS = PS;
  p.early_meta = early_metadata();
  p.max_len = (int)std::min<long long>((long long)MP * PS, 0x7fffffffll);
  p.scale_log2 = sm_scale * 1.4426950408889634f;
  p.v_scale = v_scale;
  p.window = window;
  p.sinks = sinks;
  p.lse = lse;
  const B8Variant v = variant_of(D, fmt, two, win);
  for (int row0 = 0; row0 < G * qlmax; row0 += rows_per_pass) {
    p.row0 = row0;
    rc = record_cuda(launch_pdl(v.kernel, dim3((unsigned)n_parts), dim3(NTHREADS), (size_t)v.smem, (cudaStream_t)stream, p));
    if (rc != HKV_OK) return rc;
  }
  return HKV_OK;
}
