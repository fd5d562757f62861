// Appending keys and values to the 8-bit cache: tiles of 16 tokens of one kv head and side under one power-of-two scale
// (include/hkv.h), with the position rotation of keys and queries on the way (hkv_rotary.cuh).
//
// A warp has one tile: the call's tokens that fall into it (neighbours in `slots`), their largest magnitude, the tile's scale, the
// codes. Rows of a tile that the call does not name keep their codes unless the scale grows; then the same warp rounds them to
// the new one. A scale is a power of two, so that codes times scales are exact in 16 bits (prefill operands), and growing costs an
// E4M3 code nothing but its last subnormal bits.
//
// What bounds it: the chain of latencies of a tile (slots, rows, the largest of them, stores) over the warps that an SM holds, and the
// instructions of the rotation. B200, 8 kv heads x 128, back to back: 17108 tokens of twelve prompts 24 us (4.4 TB/s), with the
// rotation of the keys and 32 query heads 69 us (5.7 TB/s; the queries alone take 44); four single tokens 1.9 and 2.4 us. With the rows
// in registers instead of shared memory a key warp took 128 of them: 97 us for the prompts; angles from global memory for every head: the same.
// Without a rotation a prompt's floor is 16 us, and a warp has one tile on its way at a time: rows, the largest magnitude, codes.
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
  int per;                                           // tokens of a set: a CTA has the tiles that begin with one of them (1 to 16)
  unsigned groups;                                   // CTAs of a set, each with a warp per kv head and side
};

// the smallest exponent e of the cache's range with a <= 2^e times the largest code (448 = 1.75 * 2^8, 127 = 1.984375 * 2^6)
template <bool INT8>
__device__ __forceinline__ int tile_exponent(float a) {
  const uint32_t b = __float_as_uint(a) & 0x7fffffffu;
  const int e = (int)(b >> 23) - 127 - (INT8 ? 6 : 8) + ((b & 0x7fffffu) > (INT8 ? 0x7e0000u : 0x600000u));
  return min(max(e, INT8 ? HKV_B8_INT8_MIN : HKV_B8_E4M3_MIN), INT8 ? HKV_B8_INT8_MAX : HKV_B8_E4M3_MAX);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }


// four values -> four codes, round to nearest even; beyond the largest code: that one. A NaN stays one (int8: 0; the values are within
// the codes then, see sound_pair)
template <bool INT8>
__device__ __forceinline__ uint32_t codes4(const float (&y)[4]) {
  uint32_t w;
  if (INT8) {
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(__fadd_rn(y[i], 12582912.0f));   // 1.5 * 2^23: the integer in the low bits
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
    if (INT8) {                                      // (-128 is no code of the writer's)
      y[2 * i] = fmaxf(y[2 * i], -127.0f);
      y[2 * i + 1] = fmaxf(y[2 * i + 1], -127.0f);
    }
  }
  return codes4<INT8>(y);
}

// What a row's values are turned into codes with: y = x / g * 2^-e.
//   g = 2^k (as 1, the usual one): one packed multiplication by 2^(-k - e), exact
//   otherwise g = m 2^k, 1 < m < 2: RN(x / m) by three multiply-adds with r = RN(1 / m) (Markstein; nothing overflows, and an
//   infinity has been replaced by the largest number), times the same power of two. RN(x / g) but for quotients below fp32's normal range
struct ToCode {
  float m, r, f;
  __nv_bfloat162 f2;
  bool unit;
};
__device__ __forceinline__ ToCode to_code(float g, int e) {
  const uint32_t b = __float_as_uint(g);
  ToCode t;
  t.unit = (b & 0x7fffffu) == 0;
  t.m = __uint_as_float((b & 0x807fffffu) | 0x3f800000u);            // with the sign of g
  t.r = __frcp_rn(t.m);
  t.f = two_to(min(max(127 - (int)(b >> 23 & 255u) - e, -126), 127));
  const float s = t.unit ? copysignf(t.f, g) : t.f;
  t.f2 = __floats2bfloat162_rn(s, s);
  return t;
}
// int8: NaN -> 0, and within +-127
__device__ __forceinline__ uint32_t sound_pair(uint32_t w) {
  const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&w);
  w &= __heq2_mask(x, x);
  const __nv_bfloat162 top = __floats2bfloat162_rn(127.0f, 127.0f), low = __floats2bfloat162_rn(-127.0f, -127.0f);
  const __nv_bfloat162 y = __hmin2(__hmax2(*reinterpret_cast<const __nv_bfloat162*>(&w), low), top);
  return *reinterpret_cast<const uint32_t*>(&y);
}
// eight values -> eight codes
template <bool INT8>
__device__ __forceinline__ uint2 codes8(const uint4& v, const ToCode& t) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float y[8];
  if (t.unit) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), t.f2);
      uint32_t u = *reinterpret_cast<const uint32_t*>(&p);
      if (INT8) u = sound_pair(u);
      bf16x2_floats(u, y[2 * i], y[2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) bf16x2_floats(w[i], y[2 * i], y[2 * i + 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float q = __fmul_rn(y[i], t.r);
      float x = __fmaf_rn(__fmaf_rn(-t.m, q, y[i]), t.r, q);
      if (!INT8) x = copysignf(x, q);                // (a zero's own sign: its remainder is +0, and so is the sum with q = -0)
      y[i] = __fmul_rn(x, t.f);
      if (INT8) y[i] = y[i] == y[i] ? fminf(fmaxf(y[i], -127.0f), 127.0f) : 0.0f;
    }
  }
  const float lo[4] = {y[0], y[1], y[2], y[3]}, hi[4] = {y[4], y[5], y[6], y[7]};
  return make_uint2(codes4<INT8>(lo), codes4<INT8>(hi));
}
// the larger magnitudes of two pairs; a NaN does not count
__device__ __forceinline__ __nv_bfloat162 larger(__nv_bfloat162 top, uint32_t w) {
  return __hmax2(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
}
// infinities -> the largest number; a NaN stays one
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  const uint32_t top = 0x7f7f7f7fu, low = 0xff7fff7fu;
  const __nv_bfloat162 x = __hmin2_nan(__hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&low)),
                                       *reinterpret_cast<const __nv_bfloat162*>(&top));
  return *reinterpret_cast<const uint32_t*>(&x);
}

// one side of one kv head, as a warp goes through its tiles
template <int D>
struct B8Side {
  const __nv_bfloat16* src;
  long long s0;                                      // elements between tokens
  uint8_t* base;
  float g;
  LaneTurn lt;
  int rr;                                            // this lane's row of those that are worked on at a time
};

// A tile's exponent from the largest magnitude among the call's rows, and whether there is an infinity among them. `was`: the tile's
// scale word. One that this writer has left is a power of two; a tile whose first slot nobody has written may hold any word, of which the
// exponent counts, and which is replaced as a whole: the word is compared, not its exponent.
struct TileScale {
  int e, old;
  bool inf;
  __device__ __forceinline__ uint32_t word() const { return (uint32_t)(e + 127) << 23; }
};
template <bool INT8>
__device__ __forceinline__ TileScale tile_scale(float g, float amax, bool fresh, uint32_t was) {
  const int need = tile_exponent<INT8>(__fdiv_rn(amax, g));
  TileScale t;
  t.old = min(max((int)(was >> 23 & 255u) - 127, INT8 ? HKV_B8_INT8_MIN : HKV_B8_E4M3_MIN), INT8 ? HKV_B8_INT8_MAX : HKV_B8_E4M3_MAX);
  t.e = fresh ? need : max(need, t.old);
  t.inf = amax > 3.38953139e38f;
  return t;
}
__device__ __forceinline__ float larger_half(__nv_bfloat162 top) { return fmaxf(__low2float(top), __high2float(top)); }
__device__ __forceinline__ float warp_largest(__nv_bfloat162 top) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(larger_half(top))));
}
// eight code bytes of a row
template <int D>
__device__ __forceinline__ uint2* code_bytes(uint8_t* tile, int row, int g) {
  return reinterpret_cast<uint2*>(tile + row * D + (((g >> 1) ^ (row & 7)) << 4) + (g & 1) * 8);
}
// rows first, first + step, .. that the call does not name, under a scale that grows
template <int D, bool INT8>
__device__ __forceinline__ void recode_rows(const B8Side<D>& s, uint8_t* tile, unsigned named, int by, int first, int step) {
  const float f = two_to(-by);
#pragma unroll 1
  for (int row = first; row < 16; row += step) {
    if (named >> row & 1u) continue;
    uint2 *pa = code_bytes<D>(tile, row, s.lt.ga), *pb = code_bytes<D>(tile, row, s.lt.gb);
    const uint2 x = *pa, y = *pb;
    *pa = make_uint2(recode4<INT8>(x.x, f), recode4<INT8>(x.y, f));
    *pb = make_uint2(recode4<INT8>(y.x, f), recode4<INT8>(y.y, f));
  }
}
template <int D, bool INT8>
__device__ __forceinline__ void store_row(const B8Side<D>& s, uint8_t* tile, int row, uint4 a, uint4 b, const ToCode& tc, bool inf) {
  if (inf) {
    a = make_uint4(finite_pair(a.x), finite_pair(a.y), finite_pair(a.z), finite_pair(a.w));
    b = make_uint4(finite_pair(b.x), finite_pair(b.y), finite_pair(b.z), finite_pair(b.w));
  }
  *code_bytes<D>(tile, row, s.lt.ga) = codes8<INT8>(a, tc);
  *code_bytes<D>(tile, row, s.lt.gb) = codes8<INT8>(b, tc);
}
__device__ __forceinline__ __nv_bfloat162 largest(__nv_bfloat162 top, const uint4& v) {
  return larger(larger(larger(larger(top, v.x), v.y), v.z), v.w);
}

// The byte of page 0 and head 0's tiles that a slot's tile begins with
template <int D>
__device__ __forceinline__ long long tile_offset(const B8WriteParams& p, long long tile) {
  const long long at = tile << 4, page = at >> p.lps;
  return page * p.dsp + ((at & ((1ll << p.lps) - 1)) >> 4) * (16 * D + 16);
}

// Single tokens, each in a tile of its own (lanes `leaders` of the list; `slot`, `angle` theirs): RPP of them at a time, a tile for the
// D / 16 lanes of a row. 1024 tokens of 8 kv heads x 128: 3.8 us, one after another 8.7.
template <int D, bool INT8, bool ROT>
__device__ __forceinline__ void write_singles(const B8WriteParams& p, const B8Side<D>& s, const RotaryParams& r, bool turned, unsigned leaders,
                                              long long slot, int angle, long long t0) {
  constexpr int LPR = D / 16, RPP = 512 / D;
  while (leaders) {
    unsigned m = leaders;
#pragma unroll
    for (int i = 1; i < RPP; ++i)
      if (i <= s.rr) m &= m - 1;
    const bool mine = m != 0;                        // (the rr-th of them)
    const int j = mine ? __ffs(m) - 1 : 0, at = __shfl_sync(0xffffffffu, angle, j);
    const long long sl = __shfl_sync(0xffffffffu, slot, j);
    const int row = (int)sl & 15;
    uint8_t* const tile = s.base + tile_offset<D>(p, sl >> 4);
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    uint32_t was = 0;
    if (mine) {
      const __nv_bfloat16* src = s.src + (t0 - 1 + j) * s.s0;
      a = *reinterpret_cast<const uint4*>(src + 8 * s.lt.ga);
      b = *reinterpret_cast<const uint4*>(src + 8 * s.lt.gb);
      if (row) was = *reinterpret_cast<const uint32_t*>(tile + 16 * D);
    }
    if (ROT && turned && mine && s.lt.kind) {
      Angles an;
      load_angles(r, table_row(r, at), s.lt, an);
      turn_groups(a, b, s.lt, an);
    }
    float amax = larger_half(largest(largest(__floats2bfloat162_rn(0.0f, 0.0f), a), b));
#pragma unroll
    for (int x = 1; x < LPR; x <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, x));
    if (mine) {
      const TileScale sc = tile_scale<INT8>(s.g, amax, row == 0, was);
      if (row && sc.e > sc.old) recode_rows<D, INT8>(s, tile, 1u << row, sc.e - sc.old, 0, 1);
      store_row<D, INT8>(s, tile, row, a, b, to_code(s.g, sc.e), sc.inf);
      if ((threadIdx.x & (LPR - 1)) == 0 && sc.word() != was) *reinterpret_cast<uint32_t*>(tile + 16 * D) = sc.word();
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < RPP; ++i) leaders &= leaders - 1;
  }
}

// The rows of one tile. Lane i < 16 has row i's token (or -1) and its angles: copy number `angle` in shared memory, or row ~angle of
// the table.
//
// A few rows (RPP: as many as the warp's lanes have at a time), of drafts and prompts' ends: in registers.
template <int D, bool INT8, bool ROT>
__device__ __forceinline__ void write_few(const B8Side<D>& s, const RotaryParams& r, bool turned, int tok, int angle, unsigned named,
                                          uint8_t* tile, uint32_t was) {
  constexpr int RPP = 512 / D;
  unsigned m = named;
#pragma unroll
  for (int i = 1; i < RPP; ++i)
    if (i <= s.rr) m &= m - 1;
  const bool mine = m != 0;                          // (the rr-th of the rows)
  const int row = mine ? __ffs(m) - 1 : 0, t = __shfl_sync(0xffffffffu, tok, row), at = __shfl_sync(0xffffffffu, angle, row);
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (mine) {
    const __nv_bfloat16* src = s.src + t * s.s0;
    a = *reinterpret_cast<const uint4*>(src + 8 * s.lt.ga);
    b = *reinterpret_cast<const uint4*>(src + 8 * s.lt.gb);
  }
  if (ROT && turned && mine && s.lt.kind) {
    Angles an;
    load_angles(r, table_row(r, ~at), s.lt, an);
    turn_groups(a, b, s.lt, an);
  }
  const TileScale sc = tile_scale<INT8>(s.g, warp_largest(largest(largest(__floats2bfloat162_rn(0.0f, 0.0f), a), b)), named & 1u, was);
  if (!(named & 1u) && sc.e > sc.old) recode_rows<D, INT8>(s, tile, named, sc.e - sc.old, s.rr, RPP);
  if (mine) store_row<D, INT8>(s, tile, row, a, b, to_code(s.g, sc.e), sc.inf);
  if ((threadIdx.x & 31) == 0 && sc.word() != was) *reinterpret_cast<uint32_t*>(tile + 16 * D) = sc.word();
}

// More rows go through the warp's 16 rows of shared memory: a lane copies what it alone works on, all rows at once, so that a warp has 4
// or 8 KB on their way at few registers. Then, RPP rows at a time: keys are turned and the largest magnitude found; once the scale is
// known, the codes. `copies`: the angles are still being copied (every warp of the CTA comes by here then).
template <int D, bool INT8, bool ROT>
__device__ __forceinline__ void write_tile(const B8Side<D>& s, const RotaryParams& r, bool turned, const uint8_t* angles, bool& copies,
                                           uint8_t* rows, int tok, int angle, unsigned named, uint8_t* tile, uint32_t was) {
  constexpr int RPP = 512 / D;
  uint8_t* const my = rows + s.rr * (2 * D);         // this lane's row of the first ones; its groups lie at 16 * ga and 16 * gb
  auto any = [&](int i) { return (named >> i & ((1u << RPP) - 1)) != 0; };    // (i: first row of a pass)
#pragma unroll 1
  for (int i = 0; i < 16; i += RPP) {
    if (!any(i)) continue;
    const int t = __shfl_sync(0xffffffffu, tok, i + s.rr);
    if (t >= 0) {
      const __nv_bfloat16* row = s.src + t * s.s0;
      cp_async<16>(smem_u32(my) + i * (2 * D) + 16 * s.lt.ga, row + 8 * s.lt.ga);
      cp_async<16>(smem_u32(my) + i * (2 * D) + 16 * s.lt.gb, row + 8 * s.lt.gb);
    }
  }
  cp_async_wait();
  if (ROT && copies) {
    __syncthreads();
    copies = false;
  }
  __nv_bfloat162 top = __floats2bfloat162_rn(0.0f, 0.0f), top2 = top;
#pragma unroll 1
  for (int i = 0; i < 16; i += RPP) {
    if (!any(i)) continue;
    const int at = ROT ? __shfl_sync(0xffffffffu, angle, i + s.rr) : 0;
    if (named >> (i + s.rr) & 1u) {
      uint4 *pa = reinterpret_cast<uint4*>(my + i * (2 * D) + 16 * s.lt.ga), *pb = reinterpret_cast<uint4*>(my + i * (2 * D) + 16 * s.lt.gb);
      uint4 a = *pa, b = *pb;
      if (ROT && turned && s.lt.kind) {
        Angles an;
        load_angles<true>(r, at >= 0 ? angles + at * (4 * D) : table_row(r, ~at), s.lt, an);
        turn_groups(a, b, s.lt, an);
        *pa = a;
        *pb = b;
      }
      top = largest(top, a);
      top2 = largest(top2, b);
    }
  }
  const TileScale sc = tile_scale<INT8>(s.g, warp_largest(__hmax2(top, top2)), named & 1u, was);
  if (!(named & 1u) && sc.e > sc.old) recode_rows<D, INT8>(s, tile, named, sc.e - sc.old, s.rr, RPP);
  const ToCode tc = to_code(s.g, sc.e);
#pragma unroll 1
  for (int i = 0; i < 16; i += RPP)
    if (named >> (i + s.rr) & 1u)
      store_row<D, INT8>(s, tile, i + s.rr, *reinterpret_cast<const uint4*>(my + i * (2 * D) + 16 * s.lt.ga),
                         *reinterpret_cast<const uint4*>(my + i * (2 * D) + 16 * s.lt.gb), tc, sc.inf);
  if ((threadIdx.x & 31) == 0 && sc.word() != was) *reinterpret_cast<uint32_t*>(tile + 16 * D) = sc.word();
}
// The first part, 32 rows of angles, is for the kernels of sets of 16 tokens. Those of smaller sets read angles where they need them and leave
// it unused, which costs them CTAs: at head_dim 256 with eight warps 96 KB allow two an SM where 64 would allow three.
template <int D>
constexpr int b8_write_smem(bool rot, int warps) { return (rot ? 32 * 4 * D : 0) + warps * 32 * D; }

// A CTA has the tiles that begin with one of `per` neighbouring tokens, of up to eight kv heads and sides: a warp for each. In sets of 16
// (FEW false) the keys' angles are copied into shared memory, once for all of its heads, while the rows are on their way.
template <int D, bool INT8, bool ROT, bool FEW>
__global__ void __launch_bounds__(256, FEW || D == 256 ? 3 : 4) b8_write_kernel(const B8WriteParams p, const RotaryParams r) {
  constexpr int LPR = D / 16;                        // lanes of a row
  extern __shared__ __align__(16) uint8_t b8_smem[];
  uint8_t *const angles = b8_smem, *const rows = b8_smem + (ROT ? 32 * 4 * D : 0) + (threadIdx.x >> 5) * (32 * D);
  pdl_wait();                                        // inputs and the cache may come from the preceding launch
  pdl_launch_dependents();
  unsigned block = blockIdx.x;
  if (ROT && query_block<false>(r, block)) {
    rotate_queries<D>(r, (long long)block * blockDim.x + threadIdx.x);
    return;
  }
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const unsigned set = block / p.groups, h0 = (block - set * p.groups) * warps, hs = h0 + w, sides = 2 * p.KVH;
  const long long t0 = (long long)set * p.per;
  // lane i looks at token t0 - 1 + i
  auto slot_of = [&](long long t) { return t >= 0 && t < p.n ? __ldg(p.slots + t) : -1ll; };
  const long long slot = slot_of(t0 - 1 + lane);
  const bool side = hs >= (unsigned)p.KVH;
  bool copies = ROT && h0 < (unsigned)p.KVH && !FEW;        // (a single token's angles are read where they are needed)
  int angle = 0;
  if (ROT && h0 < (unsigned)p.KVH && t0 - 1 + lane >= 0 && t0 - 1 + lane < p.n) angle = table_index(r, t0 - 1 + lane);
  const int h = hs >= sides ? 0 : side ? hs - p.KVH : hs;
  B8Side<D> s;
  s.src = side ? p.val + h * p.vs1 : p.key + h * p.ks1;
  s.s0 = side ? p.vs0 : p.ks0;
  s.base = (side ? p.vt : p.kt) + h * p.dsh;
  s.g = __ldg((side ? p.gv : p.gk) + h);
  s.lt = lane_turn<D>(lane % LPR, ROT && !side ? r.rot : 0, ROT && !side ? r.neighbours : 0);
  s.rr = lane / LPR;

  const long long tile = slot < 0 ? -1 : slot >> 4;
  const long long before = __shfl_up_sync(0xffffffffu, tile, 1);
  unsigned leaders = __ballot_sync(0xffffffffu, lane >= 1 && lane <= p.per && tile >= 0 && tile != before);
  if (copies && leaders) {                           // tokens of the set, and those behind it in its last tile
    const long long last = __shfl_sync(0xffffffffu, tile, p.per);
    const unsigned more = __ballot_sync(0xffffffffu, tile == last && tile >= 0) >> p.per;
    const int end = p.per + max(1, more == 0xffffffffu ? 32 : __ffs(~more) - 1), bytes = r.rot * (r.bf16 ? 2 : 4);
    for (int i = 1 + w; i < min(end, 32); i += warps) {
      const uint8_t* row = table_row(r, __shfl_sync(0xffffffffu, angle, i));
      for (int c = 16 * lane; c < bytes; c += 512) cp_async<16>(smem_u32(angles) + i * (4 * D) + c, row + c);
    }
  }
  // No head for this warp. Only a set's last CTA of eight warps has such, where 2 * KVH is no multiple of eight: it begins at side
  // 8 * floor(2 * KVH / 8) >= KVH (KVH >= 5), so that it copies no angles and no barrier waits for this warp.
  if (hs >= sides) return;
  if (FEW && (__ballot_sync(0xffffffffu, tile >= 0 && tile == before) & leaders << 1) == 0) {      // no tile has a second token
    write_singles<D, INT8, ROT>(p, s, r, ROT && !side, leaders, slot, angle, t0);
    return;
  }
  while (leaders) {
    const int j0 = __ffs(leaders) - 1;
    leaders &= leaders - 1;
    const long long mine = __shfl_sync(0xffffffffu, tile, j0);
    uint8_t* const t_ = s.base + tile_offset<D>(p, mine);
    const uint32_t was_bits = *reinterpret_cast<const uint32_t*>(t_ + 16 * D);
    // the run of tokens in this tile, and the last of them for every row: lane i < 16 gets that of row i, or -1
    int tok = -1, ang = 0;
    {
      unsigned in = __ballot_sync(0xffffffffu, tile == mine) >> j0;
      const int len = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
      const int first = (int)__shfl_sync(0xffffffffu, slot, j0) & 15;
      // (a prompt's or a draft's: ascending)
      const bool plain = __all_sync(0xffffffffu, lane < j0 || lane >= j0 + len || ((int)slot & 15) == first + lane - j0);
      if (plain) {
        if (lane >= first && lane < first + len) tok = (int)(t0 - 1) + j0 + lane - first;
        ang = (j0 + lane - first) & 31;
      } else {
        for (int i = j0; i < j0 + len; ++i)
          if (lane == ((int)__shfl_sync(0xffffffffu, slot, i) & 15)) {
            tok = (int)(t0 - 1) + i;
            ang = i;
          }
      }
      if (ROT && FEW) ang = ~__shfl_sync(0xffffffffu, angle, ang);
      // runs past the lanes' tokens: only those that lie well inside a set, or name a row twice
      for (long long t = t0 + 31; j0 + len == 32 && t < p.n; t += 32) {
        const long long more = slot_of(t + lane);
        in = __ballot_sync(0xffffffffu, more >= 0 && more >> 4 == mine);
        const int n = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
        for (int i = 0; i < n; ++i)
          if (lane == ((int)__shfl_sync(0xffffffffu, more, i) & 15)) tok = (int)t + i;
        if (ROT && !side && tok >= t) ang = ~table_index(r, tok);
        if (n < 32) break;
      }
      if (lane >= 16) tok = -1;
    }
    const unsigned named = __ballot_sync(0xffffffffu, tok >= 0);
    const uint32_t was = named & 1u ? 0 : was_bits;
    if (FEW && __popc(named) <= 512 / D) write_few<D, INT8, ROT>(s, r, ROT && !side, tok, ang, named, t_, was);
    else write_tile<D, INT8, ROT>(s, r, ROT && !side, angles, copies, rows, tok, ang, named, t_, was);
    __syncwarp();
  }
}

template <int D, bool FEW>
static auto b8_write(bool int8, bool rot) -> void (*)(const B8WriteParams, const RotaryParams) {
  return int8 ? (rot ? b8_write_kernel<D, true, true, FEW> : b8_write_kernel<D, true, false, FEW>)
              : rot ? b8_write_kernel<D, false, true, FEW> : b8_write_kernel<D, false, false, FEW>;
}

}  // namespace hkv

extern "C" int hkv_write_b8(const void* key, const void* val, int64_t ks0, int64_t ks1, int64_t vs0, int64_t vs1, void* kt, void* vt,
                            const int64_t strides[2], int PS, const int64_t* slots, int64_t n_slots, const float* gk, const float* gv,
                            int KVH, int D, int fmt, const hkv_rotary* rotary, void* stream) {
  using namespace hkv;
  if (n_slots < 0 || n_slots >= (1ll << 31) - 64) return HKV_ERR_RANGE;
  if (n_slots == 0 && (!rotary || rotary->n_tokens == 0)) return HKV_OK;
  if (n_slots > 0 && (!key || !val || !slots)) return HKV_ERR_NULL;
  if (!kt || !vt || !strides || !gk || !gv) return HKV_ERR_NULL;
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
  // Tokens of a set. A set of one has a warp for each of its tokens' rows, which is best while the GPU holds these warps at once (148 SMs
  // with three CTAs of eight); larger sets leave fewer warps without a tile to begin, and take several tiles of single tokens at a time.
  // us at 1 / 4 / 8 tokens a set, e4m3, caches larger than the L2, rows = 2 * KVH * tokens:
  //   2 x 256, rotating, 512 tokens (2048 rows) single 6.1 / 5.4 / 7.8, in pairs 6.1 / 6.7 / 10.1
  //   8 x 128, rotating, 256 tokens (4096) single 6.1 / 3.7 / 4.9, in pairs 5.1 / 6.0 / 9.0; 512 (8192) 9.0 / 4.5 / 5.8, 7.9 / 7.1 / 10.7
  //   2 x 256, 1024 tokens (4096) in pairs 4.4 / 5.2 / 7.8; 3000 (12000) 8.4 / 5.9 / 8.4; 4096 (16384) 10.4 / 9.3 / 9.0
  //   8 x 128, 1536 tokens (24576) of a prompt 11.1 / 6.4 / 5.8; 1 x 128, 4096 (8192) in drafts of four 6.3 / 3.7 / 5.2
  // From 8192 tokens on a call is of prompts: sets of 16, in whose kernel the keys' angles are copied once for all heads. There 8 / 16 tokens a
  // set take 39 / 34 (a prompt of 8192 tokens, 8 x 128, rotating) and 15.6 / 13.3 (not rotating), but 46 / 103 were they all single.
  const int64_t rows = n_slots * 2 * KVH, at_once = 148 * 24;
  p.per = n_slots >= 8192 ? 16 : rows <= at_once ? 1 : rows <= 4 * at_once ? 4 : 8;
  const int warps = 2 * KVH < 8 ? 2 * KVH : 8;
  p.groups = (unsigned)((2 * KVH + warps - 1) / warps);
  const long long blocks = (n_slots + p.per - 1) / p.per * p.groups;
  const long long all = rotary ? with_queries(r, D, blocks, 32 * warps) : blocks;
  if (all > 0x7fffffffll) return HKV_ERR_RANGE;
  void (*k)(const B8WriteParams, const RotaryParams);
  const bool i8 = fmt == HKV_B8_INT8;
  if (p.per < 16) k = D == 128 ? b8_write<128, true>(i8, rotary) : b8_write<256, true>(i8, rotary);
  else k = D == 128 ? b8_write<128, false>(i8, rotary) : b8_write<256, false>(i8, rotary);
  const int smem = D == 128 ? b8_write_smem<128>(rotary, warps) : b8_write_smem<256>(rotary, warps);
  if (smem > 48 * 1024) {
    const int rc = record_cuda(cudaFuncSetAttribute((const void*)k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (rc != HKV_OK) return rc;
  }
  return record_cuda(launch_pdl(k, dim3((unsigned)all), dim3(32 * warps), smem, (cudaStream_t)stream, p, r));
}
