// Position rotation of query and key rows on their way (hkv_rotary in include/hkv.h): pairs of channels (x1, x2) become
// (x1 c - x2 s, x2 c + x1 s), products and sums rounded singly in fp32 and the result once to bf16, which is what a launch that
// rotates before the write leaves in memory.
#pragma once

#include <cuda_bf16.h>

#include <initializer_list>
#include <numeric>

#include "hkv_common.cuh"
#include "hkv_f32x2.cuh"

namespace hkv {

struct RotaryParams {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  long long qs0, qs1, os0, os1;
  const long long* positions;
  const uint8_t* table;                              // row p: cosines of rot / 2 pairs, then their sines
  long long rows;                                    // of the table
  long long n_tokens;
  int HQ, rot, bf16, neighbours;
  unsigned others;                                   // CTAs that do not rotate queries
  unsigned long long share;                          // of those that do, times 2^32, rounded up
};

// True for a CTA that rotates queries; `index` counts the CTAs of its kind. Queries are a matter of memory bandwidth. ALTERNATE: their CTAs
// lie between those that write the cache, so that an SM has both at a time, which pays where these are bound by their instructions
// (NVFP4, 16384 tokens, 32 + 2 x 8 heads x 128: 93 us, 102 with the queries last, 106 with them first); else they come last, and
// fill the SMs that the others leave (the 8-bit cache, 2048 tokens: 12.9 us against 14.8).
template <bool ALTERNATE>
__device__ __forceinline__ bool query_block(const RotaryParams& r, unsigned& index) {
  if (!ALTERNATE) {
    index = blockIdx.x < r.others ? blockIdx.x : blockIdx.x - r.others;
    return blockIdx.x >= r.others;
  }
  const unsigned before = (unsigned)(blockIdx.x * r.share >> 32), with = (unsigned)((blockIdx.x + 1ull) * r.share >> 32);
  index = with > before ? before : blockIdx.x - before;
  return with > before;
}

// (a position outside the table takes the nearest row)
__device__ __forceinline__ int table_index(const RotaryParams& r, long long token) {
  const long long pos = __ldg(r.positions + token);
  return (int)(pos < 0 ? 0 : pos >= r.rows ? r.rows - 1 : pos);
}
__device__ __forceinline__ const uint8_t* table_row(const RotaryParams& r, int index) {
  return r.table + (long long)index * r.rot * (r.bf16 ? 2 : 4);
}
__device__ __forceinline__ void bf16x2_floats(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ uint32_t floats_bf16x2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
template <bool SHARED, typename T>
__device__ __forceinline__ T table_load(const T* p) {                // SHARED: the row may be a copy in shared memory
  if (SHARED) return *p;
  else return __ldg(p);
}
// N (4 or 8) neighbouring numbers of a table row, from number `at` (a multiple of N) on
template <int N, bool SHARED = false>
__device__ __forceinline__ void table_numbers(const RotaryParams& r, const uint8_t* row, int at, float (&x)[N]) {
  if (r.bf16) {
    uint32_t w[N / 2];
    if (N == 8) {
      const uint4 v = table_load<SHARED>(reinterpret_cast<const uint4*>(row + 2 * at));
      w[0] = v.x; w[1] = v.y; w[N / 2 - 2] = v.z; w[N / 2 - 1] = v.w;
    } else {
      const uint2 v = table_load<SHARED>(reinterpret_cast<const uint2*>(row + 2 * at));
      w[0] = v.x; w[1] = v.y;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) bf16x2_floats(w[i], x[2 * i], x[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = table_load<SHARED>(reinterpret_cast<const float4*>(row + 4 * at) + i);
      x[4 * i] = v.x; x[4 * i + 1] = v.y; x[4 * i + 2] = v.z; x[4 * i + 3] = v.w;
    }
  }
}
// x c - y s, pairwise, each product and the difference rounded: an fma by -1, which cannot absorb the packed product that feeds its
// first operand, and single products for its addend. (With packed products for both, ptxas 12.9 rounded once where this has to round
// twice: a bit of one turned value in a few thousand.)
__device__ __forceinline__ f32x2 turn2(f32x2 x, f32x2 y, f32x2 c, f32x2 s) {
  return fma2(mul2(y, s), 0xbf800000bf800000ull, pk(__fmul_rn(lo(x), lo(c)), __fmul_rn(hi(x), hi(c))));
}
constexpr f32x2 kSigns = 0x8000000080000000ull;
__device__ __forceinline__ f32x2 bf16x2_pair(uint32_t w) { return (f32x2)(w & 0xffff0000u) << 32 | (w << 16); }
__device__ __forceinline__ uint32_t pair_bf16x2(f32x2 v) { return floats_bf16x2(lo(v), hi(v)); }
// two neighbouring values, turned as one of the "neighbours" pairs
__device__ __forceinline__ uint32_t turn_neighbours(uint32_t w, float c, float s) {
  const f32x2 v = bf16x2_pair(w);
  return pair_bf16x2(turn2(v, pk(hi(v), lo(v)), pk(c, c), pk(s, -s)));
}

// Cosines and sines of a lane's two groups of eight channels. A row is spread over D / 16 lanes; lane j has two groups such that
// both halves of its pairs are its own: "halves" groups j and j + rot / 16 where j < rot / 16, and two groups that stay as they are
// otherwise; "neighbours" groups j and j + D / 16, either turned or not.
struct LaneTurn {
  int ga, gb;                                        // groups of eight channels
  int kind;                                          // 0: none, 1: halves, 2: neighbours
  bool ta, tb;                                       // neighbours: group a / b is turned
};
template <int D>
__device__ __forceinline__ LaneTurn lane_turn(int j, int rot, int neighbours) {
  LaneTurn t;
  const int half = neighbours ? 0 : rot / 16;        // groups of eight in half the rotated channels
  if (j < half) {
    t.ga = j;
    t.gb = j + half;
  } else {
    t.ga = half + j;                                 // = 2 half + (j - half)
    t.gb = t.ga + D / 16 - half;
  }
  t.kind = neighbours ? 2 : j < half ? 1 : 0;
  t.ta = neighbours && 8 * t.ga < rot;
  t.tb = neighbours && 8 * t.gb < rot;
  return t;
}
struct Angles {
  float c[8], s[8];                                  // halves: of the eight pairs; neighbours: four of group a, four of group b
};
template <bool SHARED = false>
__device__ __forceinline__ void load_angles(const RotaryParams& r, const uint8_t* row, const LaneTurn& t, Angles& a) {
  const int half = r.rot / 2;
  if (t.kind == 1) {
    table_numbers<8, SHARED>(r, row, 8 * t.ga, a.c);
    table_numbers<8, SHARED>(r, row, half + 8 * t.ga, a.s);
  } else if (t.kind == 2) {
    float c[4], s[4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if (g ? t.tb : t.ta) {
        table_numbers<4, SHARED>(r, row, 4 * (g ? t.gb : t.ga), c);
        table_numbers<4, SHARED>(r, row, half + 4 * (g ? t.gb : t.ga), s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          a.c[4 * g + i] = c[i];
          a.s[4 * g + i] = s[i];
        }
      }
    }
  }
}
// the lane's two groups, eight bf16 values each, turned in place
__device__ __forceinline__ void turn_groups(uint4& a, uint4& b, const LaneTurn& t, const Angles& an) {
  uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
  if (t.kind == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 x = bf16x2_pair(wa[i]), y = bf16x2_pair(wb[i]), c = pk(an.c[2 * i], an.c[2 * i + 1]), s = pk(an.s[2 * i], an.s[2 * i + 1]);
      wa[i] = pair_bf16x2(turn2(x, y, c, s));
      wb[i] = pair_bf16x2(turn2(y, x, c, s ^ kSigns));
    }
  } else if (t.kind == 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (t.ta) wa[i] = turn_neighbours(wa[i], an.c[i], an.s[i]);
      if (t.tb) wb[i] = turn_neighbours(wb[i], an.c[4 + i], an.s[4 + i]);
    }
  }
  a = make_uint4(wa[0], wa[1], wa[2], wa[3]);
  b = make_uint4(wb[0], wb[1], wb[2], wb[3]);
}

// Group `g` (eight channels, in w) of the row at `src` on its own: the channels it is paired with are read here
__device__ __forceinline__ void turn_own_group(const RotaryParams& r, const uint8_t* angles, const __nv_bfloat16* src, int g, uint32_t* w) {
  if (8 * g >= r.rot) return;
  const int half = r.rot / 2;
  if (r.neighbours) {
    float c[4], s[4];
    table_numbers<4>(r, angles, 4 * g, c);
    table_numbers<4>(r, angles, half + 4 * g, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = turn_neighbours(w[i], c[i], s[i]);
  } else {
    const bool second = 8 * g >= half;
    const int at = second ? 8 * g - half : 8 * g;     // first of the group's pairs
    const uint4 o = *reinterpret_cast<const uint4*>(src + (second ? at : at + half));
    const uint32_t wo[4] = {o.x, o.y, o.z, o.w};
    float c[8], s[8];
    table_numbers<8>(r, angles, at, c);
    table_numbers<8>(r, angles, half + at, s);
    const f32x2 sign = second ? kSigns : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = pair_bf16x2(turn2(bf16x2_pair(w[i]), bf16x2_pair(wo[i]), pk(c[2 * i], c[2 * i + 1]), pk(s[2 * i], s[2 * i + 1]) ^ sign));
  }
}

// Query rows: D / 16 threads have up to kHeadsAtOnce heads of a token, under the same angles. `at`: thread number among those that
// rotate queries. In place is fine: a thread stores what it alone has read.
constexpr int kHeadsAtOnce = 4;
template <int D>
__device__ __forceinline__ void rotate_queries(const RotaryParams& r, long long at) {
  constexpr int LPR = D / 16;
  const int sets = (r.HQ + kHeadsAtOnce - 1) / kHeadsAtOnce;
  const long long item = at / LPR, token = item / sets;
  if (token >= r.n_tokens) return;
  const int h0 = (int)(item - token * sets) * kHeadsAtOnce;
  const LaneTurn t = lane_turn<D>((int)(at % LPR), r.rot, r.neighbours);
  const __nv_bfloat16* src = r.q + token * r.qs0 + h0 * r.qs1;
  __nv_bfloat16* dst = r.out + token * r.os0 + h0 * r.os1;
  uint4 a[kHeadsAtOnce], b[kHeadsAtOnce];
#pragma unroll
  for (int i = 0; i < kHeadsAtOnce; ++i) {
    if (h0 + i >= r.HQ) break;
    a[i] = *reinterpret_cast<const uint4*>(src + i * r.qs1 + 8 * t.ga);
    b[i] = *reinterpret_cast<const uint4*>(src + i * r.qs1 + 8 * t.gb);
  }
  Angles an;
  load_angles(r, table_row(r, table_index(r, token)), t, an);
#pragma unroll
  for (int i = 0; i < kHeadsAtOnce; ++i) {
    if (h0 + i >= r.HQ) break;
    turn_groups(a[i], b[i], t, an);
    *reinterpret_cast<uint4*>(dst + i * r.os1 + 8 * t.ga) = a[i];
    *reinterpret_cast<uint4*>(dst + i * r.os1 + 8 * t.gb) = b[i];
  }
}
// CTAs of the launch, of which `blocks` do something else than rotate queries
inline long long with_queries(RotaryParams& r, int D, long long blocks, int threads) {
  const long long n = r.n_tokens * ((r.HQ + kHeadsAtOnce - 1) / kHeadsAtOnce) * (D / 16), q = (n + threads - 1) / threads, all = blocks + q;
  r.others = (unsigned)blocks;
  r.share = all > 0 && all < (1ll << 31) ? (((unsigned long long)q << 32) + all - 1) / all : 0;
  return all;
}

// ----------------------------------------------------------------------------------------------------- host side
// rows of D 16-bit numbers: row (i, h), i < n, h < heads, at p + 2 * (i * s0 + h * s1) bytes
struct RowSet {
  const void* p;
  int64_t s0, s1, n, heads;
};
// Whether two sets of rows have no byte in common, by one of three rules: they lie apart as a whole; they are columns of the same long rows
// (queries and keys of a fused product); or they are columns of something smaller (heads of queries, keys and values in turn): every
// stride is a multiple of g, and modulo g a row of one set lies beside a row of the other.
inline bool rows_disjoint(const RowSet& a, const RowSet& b, int64_t D) {
  if (a.n < 1 || b.n < 1) return true;
  const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
  const int64_t a_span = (a.heads - 1) * a.s1 + D, b_span = (b.heads - 1) * b.s1 + D;
  if (pa + 2 * (uint64_t)((a.n - 1) * a.s0 + a_span) <= pb || pb + 2 * (uint64_t)((b.n - 1) * b.s0 + b_span) <= pa) return true;
  const bool first = pa <= pb;
  const uint64_t apart = first ? pb - pa : pa - pb;
  auto beside = [apart](int64_t m, int64_t lo_span, int64_t hi_span) {
    const uint64_t off = apart % (2 * (uint64_t)m);
    return off >= 2 * (uint64_t)lo_span && off + 2 * (uint64_t)hi_span <= 2 * (uint64_t)m;
  };
  if (a.s0 == b.s0 && a.s0 > 0 && beside(a.s0, first ? a_span : b_span, first ? b_span : a_span)) return true;
  int64_t g = 0;
  for (const RowSet* r : {&a, &b}) {
    if (r->n > 1) g = std::gcd(g, r->s0);
    if (r->heads > 1) g = std::gcd(g, r->s1);
  }
  return g > 0 && beside(g, D, D);
}
// checks a caller's hkv_rotary; keys and values (n tokens of KVH heads) must not be where the queries go
inline int rotary_params(const hkv_rotary* u, int D, int64_t n_slots, const void* key, int64_t ks0, int64_t ks1, const void* val,
                         int64_t vs0, int64_t vs1, int KVH, RotaryParams* r) {
  if (!u->query || !u->query_out || !u->positions || !u->table) return HKV_ERR_NULL;
  if (u->n_tokens < n_slots || u->n_tokens >= (1ll << 31) || u->rows < 1 || u->rows >= (1ll << 31)) return HKV_ERR_RANGE;
  if (u->HQ < 1 || u->HQ > 65536 || u->rot < 16 || u->rot > D || u->rot % 16) return HKV_ERR_UNSUPPORTED;
  if (u->qs0 < 0 || u->qs1 < 0 || u->os0 < 0 || u->os1 < 0) return HKV_ERR_RANGE;
  if (((uintptr_t)u->query | (uintptr_t)u->query_out | (uintptr_t)u->table) & 15) return HKV_ERR_ALIGN;
  if (((uintptr_t)u->positions & 7) || ((u->qs0 | u->qs1 | u->os0 | u->os1) & 7)) return HKV_ERR_ALIGN;
  const int64_t n = u->n_tokens;
  const RowSet out{u->query_out, u->os0, u->os1, n, u->HQ};
  // rows that are written must not overlap one another, nor what else is read
  if (!rows_apart((int)n, u->HQ, D, u->os0, u->os1)) return HKV_ERR_RANGE;
  // (a stride between one row and no other says nothing)
  const bool same = u->query == u->query_out && (n < 2 || u->qs0 == u->os0) && (u->HQ < 2 || u->qs1 == u->os1);
  if (!same && !rows_disjoint({u->query, u->qs0, u->qs1, n, u->HQ}, out, D)) return HKV_ERR_RANGE;
  if (ks0 >= 0 && ks1 >= 0 && !rows_disjoint({key, ks0, ks1, n_slots, KVH}, out, D)) return HKV_ERR_RANGE;
  if (vs0 >= 0 && vs1 >= 0 && !rows_disjoint({val, vs0, vs1, n_slots, KVH}, out, D)) return HKV_ERR_RANGE;
  r->q = (const __nv_bfloat16*)u->query;
  r->out = (__nv_bfloat16*)u->query_out;
  r->qs0 = u->qs0; r->qs1 = u->qs1; r->os0 = u->os0; r->os1 = u->os1;
  r->positions = (const long long*)u->positions;
  r->table = (const uint8_t*)u->table;
  r->rows = u->rows;
  r->n_tokens = n;
  r->HQ = u->HQ; r->rot = u->rot; r->bf16 = u->table_bf16 != 0; r->neighbours = u->interleaved != 0;
  return HKV_OK;
}

}  // namespace hkv
