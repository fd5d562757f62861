// Appending keys and values to the 8-bit cache: tiles of 16 tokens of one kv head and side under one power-of-two scale
// (include/hkv.h), with the position rotation of keys and queries on the way (hkv_rotary.cuh).
//
// A warp has one tile: the call's tokens that fall into it (neighbours in `slots`), their largest magnitude, the tile's scale, the
// codes. Rows of a tile that the call does not name keep their codes unless the scale grows; then the same warp rounds them to
// the new one. A scale is a power of two, so that codes times scales are exact in 16 bits (prefill operands), and growing costs an
// E4M3 code nothing but its last subnormal bits.
#include <cuda_fp8.h>

#include "hkv_common.cuh"
#include "hkv_rotary.cuh"

namespace hkv {

int record_cuda(cudaError_t e);

struct B8WriteParams {
  const __nv_bfloat16* key;
  const __nv_bfloat16* val;
  long long ks0, ks1, vs0, vs1;
  uint8_t* kt;
  uint8_t* vt;
  long long dsp, dsh;                                // byte strides between pages and kv heads
  const long long* slots;
  const float* gk;
  const float* gv;
  int n, KVH, lps;                                   // tokens with a slot; log2 of the page size
  int per;                                           // tokens whose tiles a warp starts (1 to 16)
};

// the smallest exponent e of the cache's range with a <= 2^e times the largest code (448 = 1.75 * 2^8, 127 = 1.984375 * 2^6)
template <bool INT8>
__device__ __forceinline__ int tile_exponent(float a) {
  const uint32_t b = __float_as_uint(a) & 0x7fffffffu;
  const int e = (int)(b >> 23) - 127 - (INT8 ? 6 : 8) + ((b & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u));
  return min(max(e, INT8 ? HKV_B8_INT8_MIN : HKV_B8_E4M3_MIN), INT8 ? HKV_B8_INT8_MAX : HKV_B8_E4M3_MAX);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// four values -> four codes, round to nearest even; beyond the largest code: that one. A NaN stays one (int8: 0)
template <bool INT8>
__device__ __forceinline__ uint32_t codes4(const float (&y)[4]) {
  uint32_t w;
  if (INT8) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = y[i] == y[i] ? fminf(fmaxf(y[i], -127.0f), 127.0f) : 0.0f;
      c[i] = __float_as_uint(__fadd_rn(v, 12582912.0f));             // 1.5 * 2^23: the integer in the low bits
    }
    w = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  } else {
    asm("{\n\t.reg .b16 l, h;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\t"
        "mov.b32 %0, {l, h};\n\t}"
        : "=r"(w)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]));
  }
  return w;
}
// four codes under a scale 2^-d as large (f = 2^-d): rounded to the new one
template <bool INT8>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float f) {
  uint32_t h[2];
  b8_to_f16x2<INT8>(w, h[0], h[1]);
  float y[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    y[2 * i] = __fmul_rn(__low2float(u32_as_h2(h[i])), f);
    y[2 * i + 1] = __fmul_rn(__high2float(u32_as_h2(h[i])), f);
  }
  return codes4<INT8>(y);
}

// RN(x / g) by three multiply-adds with r = RN(1 / g): exact where nothing over- or underflows on the way (Markstein), which
// `fast` states: 2^-60 <= |g| <= 2^60 and magnitudes up to 2^60; quotients below 2^-60 may differ, and get code 0 whatever they are
struct Divisor {
  float g, r;
  bool fast;
  __device__ __forceinline__ float operator()(float x) const {
    if (!fast) return __fdiv_rn(x, g);
    const float y = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-g, y, x), r, y);
  }
};

template <int D, bool INT8, bool ROT>
__global__ void __launch_bounds__(256) b8_write_kernel(const B8WriteParams p, const RotaryParams r) {
  constexpr int LPR = D / 16, RPP = 32 / LPR, NP = 16 / RPP;         // lanes of a row, rows at a time, times
  pdl_wait();                                        // inputs and the cache may come from the preceding launch
  pdl_launch_dependents();
  if (ROT && blockIdx.x >= r.first_block) {
    rotate_queries<D>(r, (long long)(blockIdx.x - r.first_block) * 256 + threadIdx.x);
    return;
  }
  const int lane = threadIdx.x & 31;
  const unsigned warp = blockIdx.x * 8 + (threadIdx.x >> 5), sides = 2 * p.KVH;
  const unsigned set = warp / sides, hs = warp - set * sides;
  const long long t0 = (long long)set * p.per;       // tiles that begin, in the list, with one of these tokens
  if (t0 >= p.n) return;
  const int side = hs >= (unsigned)p.KVH, h = side ? hs - p.KVH : hs;
  const int j = lane % LPR, rr = lane / LPR;
  const LaneTurn lt = lane_turn<D>(j, ROT && !side ? r.rot : 0, ROT && !side ? r.neighbours : 0);
  const __nv_bfloat16* src = side ? p.val + h * p.vs1 : p.key + h * p.ks1;
  const long long s0 = side ? p.vs0 : p.ks0;
  uint8_t* const base = (side ? p.vt : p.kt) + h * p.dsh;
  Divisor div;
  div.g = __ldg((side ? p.gv : p.gk) + h);
  div.r = __frcp_rn(div.g);
  const bool g_ok = fabsf(div.g) >= 0x1p-60f && fabsf(div.g) <= 0x1p60f;

  // lane i looks at token t0 - 1 + i
  auto slot_of = [&](long long t) { return t >= 0 && t < p.n ? __ldg(p.slots + t) : -1ll; };
  const long long slot = slot_of(t0 - 1 + lane), tile = slot < 0 ? -1 : slot >> 4;
  const long long before = __shfl_up_sync(0xffffffffu, tile, 1);
  unsigned leaders = __ballot_sync(0xffffffffu, lane >= 1 && lane <= p.per && tile >= 0 && tile != before);
  while (leaders) {
    const int j0 = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const long long mine = __shfl_sync(0xffffffffu, tile, j0);
    // the run of tokens in this tile, and the last of them for every row: lane i < 16 gets that of row i, or -1
    int tok = -1;
    {
      unsigned in = __ballot_sync(0xffffffffu, tile == mine) >> j0;
      int len = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
      const int first = (int)__shfl_sync(0xffffffffu, slot, j0) & 15;
      // (a prompt's or a draft's: ascending)
      const bool plain = __all_sync(0xffffffffu, lane < j0 || lane >= j0 + len || ((int)slot & 15) == first + lane - j0);
      if (plain) {
        if (lane >= first && lane < first + len && lane < 16) tok = (int)(t0 - 1) + j0 + lane - first;
      } else {
        for (int i = j0; i < j0 + len; ++i)
          if (lane == ((int)__shfl_sync(0xffffffffu, slot, i) & 15)) tok = (int)(t0 - 1) + i;
      }
      // runs past the lanes' tokens: only those that lie well inside a set, or name a row twice
      for (long long t = t0 + 31; j0 + len == 32 && t < p.n; t += 32) {
        const long long more = slot_of(t + lane);
        in = __ballot_sync(0xffffffffu, more >= 0 && more >> 4 == mine);
        const int n = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
        for (int i = 0; i < n; ++i)
          if (lane == ((int)__shfl_sync(0xffffffffu, more, i) & 15)) tok = (int)t + i;
        if (n < 32) break;
      }
      if (lane >= 16) tok = -1;
    }
    const unsigned named = __ballot_sync(0xffffffffu, tok >= 0);
    const bool fresh = named & 1u;                   // the tile begins anew
    const long long at = mine << 4, page = at >> p.lps;
    uint8_t* const t_ = base + page * p.dsp + ((at & ((1ll << p.lps) - 1)) >> 4) * (16 * D + 16);
    uint32_t* const t_scale = reinterpret_cast<uint32_t*>(t_ + 16 * D);
    const int was = fresh ? -127 : (int)(*t_scale >> 23 & 255u) - 127;

    // the rows: sixteen channels of NP rows in a lane, as bf16 pairs
    uint4 a[NP], b[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int t = __shfl_sync(0xffffffffu, tok, i * RPP + rr);
      a[i] = b[i] = make_uint4(0, 0, 0, 0);
      if (t >= 0) {
        const __nv_bfloat16* row = src + t * s0;
        a[i] = *reinterpret_cast<const uint4*>(row + 8 * lt.ga);
        b[i] = *reinterpret_cast<const uint4*>(row + 8 * lt.gb);
        if (ROT && lt.kind) {
          Angles an;
          load_angles(r, table_row(r, t), lt, an);
          turn_groups(a[i], b[i], lt, an);
        }
      }
    }
    __nv_bfloat162 top = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const uint32_t w[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t m = w[k] & 0x7fff7fffu;
        top = __hmax2(top, *reinterpret_cast<const __nv_bfloat162*>(&m));      // (a NaN does not count)
      }
    }
    const float amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(__low2float(top), __high2float(top)))));
    div.fast = g_ok && amax <= 0x1p60f;
    const int need = tile_exponent<INT8>(__fdiv_rn(amax, div.g));
    const int old = min(max(was, INT8 ? HKV_B8_INT8_MIN : HKV_B8_E4M3_MIN), INT8 ? HKV_B8_INT8_MAX : HKV_B8_E4M3_MAX);
    const int e = fresh ? need : max(need, old);

    auto where = [&](int row, int g) {               // eight code bytes of a row
      return reinterpret_cast<uint2*>(t_ + row * D + (((g >> 1) ^ (row & 7)) << 4) + (g & 1) * 8);
    };
    if (!fresh && e > old) {
      const float f = two_to(old - e);
#pragma unroll 1
      for (int i = 0; i < NP; ++i) {
        const int row = i * RPP + rr;
        if (named >> row & 1u) continue;
        uint2 *pa = where(row, lt.ga), *pb = where(row, lt.gb);
        const uint2 x = *pa, y = *pb;
        *pa = make_uint2(recode4<INT8>(x.x, f), recode4<INT8>(x.y, f));
        *pb = make_uint2(recode4<INT8>(y.x, f), recode4<INT8>(y.y, f));
      }
    }
    const float inv = two_to(-e);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int row = i * RPP + rr;
      if (!(named >> row & 1u)) continue;
      const uint32_t w[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
      uint32_t c[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y[4];
        bf16x2_floats(w[2 * k], y[0], y[1]);
        bf16x2_floats(w[2 * k + 1], y[2], y[3]);
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = __fmul_rn(div(y[u]), inv);
        c[k] = codes4<INT8>(y);
      }
      *where(row, lt.ga) = make_uint2(c[0], c[1]);
      *where(row, lt.gb) = make_uint2(c[2], c[3]);
    }
    if (lane == 0 && e != was) *t_scale = (uint32_t)(e + 127) << 23;
    __syncwarp();
  }
}

}  // namespace hkv

extern "C" int hkv_write_b8(const void* key, const void* val, int64_t ks0, int64_t ks1, int64_t vs0, int64_t vs1, void* kt, void* vt,
                            const int64_t strides[2], int PS, const int64_t* slots, int64_t n_slots, const float* gk, const float* gv,
                            int KVH, int D, int fmt, const hkv_rotary* rotary, void* stream) {
  using namespace hkv;
  if (n_slots < 0 || n_slots >= (1ll << 31) - 64) return HKV_ERR_RANGE;
  if (n_slots == 0 && (!rotary || rotary->n_tokens == 0)) return HKV_OK;
  if (!key || !val || !kt || !vt || !strides || !slots || !gk || !gv) return HKV_ERR_NULL;
  if ((D != 128 && D != 256) || (fmt != HKV_B8_E4M3 && fmt != HKV_B8_INT8)) return HKV_ERR_UNSUPPORTED;
  if (KVH < 1 || KVH > 1024 || PS < 16 || (PS & (PS - 1)) != 0) return HKV_ERR_UNSUPPORTED;
  if (((uintptr_t)key | (uintptr_t)val | (uintptr_t)kt | (uintptr_t)vt | (uintptr_t)strides[0] | (uintptr_t)strides[1]) & 15)
    return HKV_ERR_ALIGN;
  if ((ks0 | ks1 | vs0 | vs1) & 7) return HKV_ERR_ALIGN;
  RotaryParams r = {};
  if (rotary) {
    const int rc = rotary_params(rotary, D, n_slots, key, ks0, ks1, val, vs0, vs1, KVH, &r);
    if (rc != HKV_OK) return rc;
  }
  B8WriteParams p;
  p.key = (const __nv_bfloat16*)key;
  p.val = (const __nv_bfloat16*)val;
  p.ks0 = ks0; p.ks1 = ks1; p.vs0 = vs0; p.vs1 = vs1;
  p.kt = (uint8_t*)kt; p.vt = (uint8_t*)vt;
  p.dsp = strides[0]; p.dsh = strides[1];
  p.slots = (const long long*)slots;
  p.gk = gk; p.gv = gv;
  p.n = (int)n_slots; p.KVH = KVH;
  p.lps = 0;
  while ((1 << p.lps) < PS) ++p.lps;
  p.per = n_slots * 2 * KVH <= 8192 ? 1 : 16;
  const long long warps = (n_slots + p.per - 1) / p.per * 2 * KVH, blocks = (warps + 7) / 8;
  r.first_block = (unsigned)blocks;
  const long long all = blocks + (rotary ? (query_threads(r, D) + 255) / 256 : 0);
  if (all > 0x7fffffffll || warps > 0xffffffffll - 64) return HKV_ERR_RANGE;
  void (*k)(const B8WriteParams, const RotaryParams);
  const bool i8 = fmt == HKV_B8_INT8;
  if (D == 128) k = rotary ? (i8 ? b8_write_kernel<128, true, true> : b8_write_kernel<128, false, true>)
                           : i8 ? b8_write_kernel<128, true, false> : b8_write_kernel<128, false, false>;
  else k = rotary ? (i8 ? b8_write_kernel<256, true, true> : b8_write_kernel<256, false, true>)
                  : i8 ? b8_write_kernel<256, true, false> : b8_write_kernel<256, false, false>;
  return record_cuda(launch_pdl(k, dim3((unsigned)all), dim3(256), 0, (cudaStream_t)stream, p, r));
}
