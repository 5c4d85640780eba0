// na_cache_attend.hip — attention of new tokens against a paged cache held in 8 bits
// (serving).
//
// Query token j of sample b is token t = len_b - Lq + j of its sequence and sees
// tokens max(0, t - W + 1) .. t:  out = softmax(scale q k^T) v,  lse the log of the
// softmax's sum.  Token i lies in slot i mod T of page tables[b][i / T]; keys and values
// are e4m3 codes times their page's and head's power of two, which every bf16 holds
// exactly: they become bf16 as they are read, and products run on the bf16 matrix
// cores.  Queries and probabilities meet them in parts of 8 bits each: bf16 queries in
// one and fp16 ones in two (both exactly), float32 in three (24 bits); probabilities of
// 16-bit queries in two (16 bits), of float32 in three.  Scores, sums and outputs are
// float32, probabilities lose half a step of their parts, out is rounded once.
//
// The rows of a sample and key/value head (its query heads of all its new tokens)
// are cut into tiles; a tile and the keys its rows see are an item, cut into units of
// 64 keys.  The chip's workgroups share all units evenly, in order: lengths lie on the
// device, so each finds its part by adding up the items' units, and ragged lengths
// leave no workgroup waiting.  An item that lies in one workgroup is written by it;
// the others leave (m, l, o) -- reference point, sum and unnormalised output of an
// online softmax, float32 -- per workgroup, and k_cache_join adds those of a row.
// Where tables are short, each item has a workgroup of its own and nothing is joined.
//
// A token each of 32 samples of 8192 tokens, 8 heads of 128, 537 MB: 101 us with the
// join, 5.3 TB/s (memory); 2 x 1024 tokens of 32 heads at 8192 tokens: 352 us, 0.73
// PFLOP/s in 1.5 products for one, 1.10 of the matrix cores, which bound it (a large
// bf16 product reaches 1.09 to 1.15; probabilities of 8 bits: 265 us).
#include "na_cache.h"
#include "na_chunk.h"
#include "na_launch.h"
#include "na_lean.h"

#include <algorithm>
#include <type_traits>

namespace na {
namespace {

constexpr int kUnit = 64;   // keys
constexpr int kTile = 32;   // keys of a narrow wave's tile
// Units of an even share up to which each workgroup takes one chunk of one item.  Ragged
// lengths, us (with 0): 8 x 128 tokens of 4 heads of 64, a window of 4095: 48.0 (50.5); a
// token each of 8 samples of up to 4096, 8 heads of 128: 16.9 (18.9).  At 80, 32 samples of
// up to 16384: 119, at 24 110.
constexpr int kAligned = 24;
constexpr int kEntries = 512;  // of a sample's table at a time, 4 KB of a wide workgroup's LDS
constexpr int kJoin = 8;    // parts that a thread of the join loads at once

struct CacheProb {
  int32_t B, Lq, H, Hkv, rep, D;
  int32_t Mo, rows, rt;       // rows of a sample and key/value head, of a tile; tiles
  int32_t items;              // B * rt
  int32_t pages, lgT, M, W;   // W: window
  int32_t wgs, least;         // workgroups (0: one an item), units that one takes at least
  float sl2;                  // scale * log2(e)
  FastDiv frep, frt;
  int64_t qs[3];              // sample, token, head
  int64_t ts;
  const int32_t *tables, *lens;
  CachePages k, v;
};

struct CacheArgs {
  const void *q;
  void *out;
  float *lse;    // or null
  float *po;     // [2 wgs][rows][D] parts: of an item begun before, of one begun here
  float2 *pml;   // [2 wgs][rows] their reference points and sums
  int2 *span;    // [Hkv][items] first and last workgroup
};

// Keys, of full tables or a window, up to which each item of narrow tiles has a workgroup
// of its own: what a second launch costs weighs more than what idle CUs would do.  `many`
// where there are items for half of the CUs.  One token, up to so many keys, us (shared
// out and joined): 4 x 2 heads of 64: 512 6.7 (11.7), 1280 9.5 (12.0), 2048 12.7 (12.2);
// 1 x 8 of 128: 512 8.1 (12.0), 1280 12.6 (12.4), 2048 17.0 (12.5); 16 x 8 of 128: 1536
// 16.6 (21.0), 2048 20.3 (22.9), 2560 22.9 (25.2), of lengths from 1 on 15.9 (16.4), 18.9
// (20.1), 21.3 (22.0), in float32 19.3 (18.7), 23.4 (22.6), 26.4 (24.5); 4 x 4 of 256: 256
// 10.2 (14.3), 512 15.0 (14.7).
struct CacheWhole {
  int keys, many, waves;
};
constexpr CacheWhole cache_whole(int D) {
  return D > 128 ? CacheWhole{384, 384, 4} : CacheWhole{1280, 2048, 8};
}

// The keys that an item's rows see, and units over them.
struct CacheItem {
  int b, row0, row1;     // rows of the sample
  int len;
  int k0, lo, hi;        // keys [lo, hi) of some row, units from k0
  int lo_max, hi_min;    // keys that every row sees
  int units;
};

__device__ __forceinline__ int cache_len(const CacheProb &P, int i) {
  return min(max(P.lens[fdiv((uint32_t)i, P.frt)], 0), P.M << P.lgT);
}

__device__ __forceinline__ CacheItem cache_item(const CacheProb &P, int i, int len) {
  CacheItem w;
  w.b = (int)fdiv((uint32_t)i, P.frt);
  const int r = i - w.b * P.rt;
  w.len = len;
  w.row0 = r * P.rows;
  w.row1 = min(w.row0 + P.rows, P.Mo);
  const int first = w.len - P.Lq + (int)fdiv((uint32_t)w.row0, P.frep);
  const int last = w.len - P.Lq + (int)fdiv((uint32_t)(w.row1 - 1), P.frep);
  w.lo = max(first - P.W + 1, 0);
  w.hi = max(last + 1, 0);
  w.lo_max = max(last - P.W + 1, 0);
  w.hi_min = max(first + 1, 0);
  w.k0 = w.lo & ~(kUnit - 1);
  w.units = w.hi > w.lo ? (w.hi - w.k0 + kUnit - 1) / kUnit : 0;
  return w;
}

// Inclusive sum over the wave's lanes up to this one.
__device__ __forceinline__ int wave_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(x, off, 64);
    x += lane >= off ? y : 0;
  }
  return x;
}

// A value that all lanes hold, as one scalar (quotients come in vector registers).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ void cache_uniform(CacheItem &w) {
  for (int *x : {&w.b, &w.row0, &w.row1, &w.len, &w.k0, &w.lo, &w.hi, &w.lo_max, &w.hi_min, &w.units})
    *x = uniform(*x);
}

// The items of a head in order, 64 at a time, their chunks of `size` units added up.
struct CacheScan {
  int i0 = -64, size = 0, units = 0, len = 0;  // first item, the lane's units
  int mine = 0, sum = 0, all = 0;    // the lane's chunks, up to it, of all 64
  __device__ __forceinline__ void load(const CacheProb &P, int first, int chunk) {
    if (first != i0) {
      i0 = first;
      size = 0;
      const int i = i0 + (threadIdx.x & 63);
      len = i < P.items ? cache_len(P, i) : 0;
      units = i < P.items ? cache_item(P, i, len).units : 0;
    }
    if (chunk == size) return;
    size = chunk;
    mine = (int)((unsigned)(units + size - 1) / (unsigned)size);
    sum = wave_scan(mine);
    all = __builtin_amdgcn_readlane(sum, 63);
  }
  __device__ __forceinline__ CacheItem item(const CacheProb &P, int i) const {
    return cache_item(P, i, (uint32_t)(i - i0) < 64u ? __builtin_amdgcn_readlane(len, i - i0)
                                                     : cache_len(P, i));
  }
  // Chunks of all items.
  __device__ __forceinline__ int total(const CacheProb &P, int chunk) {
    int t = 0;
    for (int i = 0; i < P.items; i += 64) {
      load(P, i, chunk);
      t += all;
    }
    return t;
  }
  // The item that chunk u lies in; u becomes the chunk within it.
  __device__ __forceinline__ int find(const CacheProb &P, int &u, int chunk) {
    for (int i = 0; i < P.items; i += 64) {
      load(P, i, chunk);
      if (u < all) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(sum > u));
        u -= __builtin_amdgcn_readlane(sum - mine, at);
        return i0 + at;
      }
      u -= all;
    }
    return P.items;  // not reached: u is less than the total
  }
};

// Entry i of a sample's table: the page or -1, and the bytes of its scales.
struct CacheEntry {
  int page, k, v;
  __device__ __forceinline__ CacheEntry(const CacheProb &P, int sample, int g, int i) {
    page = i < P.M ? P.tables[sample * P.ts + i] : -1;
    k = v = 0;
    if ((uint32_t)page >= (uint32_t)P.pages) {
      page = -1;
    } else {
      k = P.k.scale[page * P.k.sc[0] + g * P.k.sc[1]];
      v = P.v.scale[page * P.v.sc[0] + g * P.v.sc[1]];
    }
  }
};

// Both scales' bytes, of keys and above of values, in the range that the append keeps to,
// where the append takes them for held ones too.  (Unwritten pages may hold others.)
__device__ __forceinline__ int cache_scales(int k, int v) {
  constexpr int low = kScaleBias + kScaleLow, high = kScaleBias + kScaleHigh;
  return min(max(k, low), high) | min(max(v, low), high) << 8;
}

// As the wide workgroups' table holds it.
__device__ __forceinline__ int2 cache_entry(const CacheProb &P, int sample, int g, int i) {
  const CacheEntry e(P, sample, g, i);
  return make_int2(e.page, cache_scales(e.k, e.v));
}

// 64 entries of a sample's table, one a lane.  The scales' bytes stay as they are loaded,
// so that the first keys' loads do not wait for them.
struct PageWindow {
  int base, page, k, v;
  __device__ __forceinline__ void load(const CacheProb &P, int sample, int g, int first) {
    base = first;
    const CacheEntry e(P, sample, g, first + (threadIdx.x & 63));
    page = e.page;
    k = e.k;
    v = e.v;
  }
  // Whether it holds table entry i (uniform).
  __device__ __forceinline__ bool holds(int i) const { return (uint32_t)(i - base) < 64u; }
  __device__ __forceinline__ int page_of(int i) const {
    return __builtin_amdgcn_readlane(page, i - base);
  }
  __device__ __forceinline__ int scales_of(int i) const {
    return cache_scales(__builtin_amdgcn_readlane(k, i - base), __builtin_amdgcn_readlane(v, i - base));
  }
};

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef L16<bf16_t> M16;

__device__ __forceinline__ float scale_of(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// Eight codes times a power of two.
__device__ __forceinline__ bf8 decode8(uint32_t a, uint32_t b, float s) {
  union {
    bf2 p[4];
    bf8 v;
  } o;
  o.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, false);
  o.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, s, true);
  o.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, false);
  o.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, s, true);
  return o.v;
}

// Parts of a query, and of a probability: one of 8 bits is off by up to half a step of
// bf16 outputs themselves (0.0023 of the outputs against 64 bits, with two 0.0017, which is
// their own rounding).
template <typename T>
constexpr int cache_parts() {
  return std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, f16_t>::value ? 2 : 3;
}
template <typename T>
constexpr int cache_prob_parts() {
  return sizeof(T) == 2 ? 2 : 3;
}

// Eight probabilities as sums of parts.
template <int NP>
__device__ __forceinline__ void split8(const float (&x)[8], bf8 (&o)[NP]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[p][i] = (__bf16)r[i];
      if (p + 1 < NP) r[i] -= (float)o[p][i];
    }
}

// Eight channels of a query: the first part of what would round to an infinity is the
// largest bf16, and what is not finite has no further parts.
template <int NP>
__device__ __forceinline__ void split_query8(const float (&x)[8], bf8 (&o)[NP]) {
  constexpr float kMost = 0x1.fep127f;
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool finite = fabsf(x[i]) < INFINITY;
    o[0][i] = (__bf16)(finite ? fminf(fmaxf(x[i], -kMost), kMost) : x[i]);
    r[i] = finite ? x[i] - (float)o[0][i] : 0.f;
  }
#pragma unroll
  for (int p = 1; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[p][i] = (__bf16)r[i];
      if (p + 1 < NP) r[i] -= (float)o[p][i];
    }
}

// Eight channels of a query row, as they lie and as sums of parts.
template <typename T>
struct Query8 {
  u4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T *p, bool live) {
    typedef typename Mem16<sizeof(T)>::t m4;  // any alignment of the elements
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      r[i] = u4{0, 0, 0, 0};
      if (live) r[i] = *reinterpret_cast<const m4 *>(p + 4 * i);
    }
  }
  template <int NP>
  __device__ __forceinline__ void parts(bf8 (&o)[NP]) const {
    if constexpr (std::is_same<T, bf16_t>::value) {
      o[0] = __builtin_bit_cast(bf8, r[0]);
    } else {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = sizeof(T) == 4 ? __uint_as_float(r[i / 4 % (sizeof(T) / 2)][i % 4])
                              : (float)__builtin_bit_cast(f16_t, (uint16_t)(r[0][i / 2] >> (16 * (i & 1))));
      split_query8<NP>(x, o);
    }
  }
};

// Four results of a row, rounded.
template <typename T>
__device__ __forceinline__ void cache_store4(T *p, f32x4 x) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4 *>(p) = x;
  } else {
    typename L16<T>::v4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (typename L16<T>::e)x[r];
    *reinterpret_cast<typename L16<T>::v4 *>(p) = o;
  }
}

// Index in lse of row r of sample b and key/value head g.
__device__ __forceinline__ int64_t cache_out_row(const CacheProb &P, int b, int g, int r) {
  const int j = (int)fdiv((uint32_t)r, P.frep);
  return ((int64_t)b * P.Lq + j) * P.H + g * P.rep + (r - j * P.rep);
}

// Where a workgroup's rows of an item go: to out, or to its part.
template <typename T>
__device__ __forceinline__ void cache_put(const CacheProb &P, const CacheArgs &A, const CacheItem &w,
                                          int g, int part, int r, int c, f32x4 o, float l) {
  if (c >= P.D) return;
  if (part >= 0) {
    *reinterpret_cast<f32x4 *>(A.po + ((int64_t)part * P.rows + r) * P.D + c) = o;
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    cache_store4(static_cast<T *>(A.out) + cache_out_row(P, w.b, g, w.row0 + r) * P.D + c, o * inv);
  }
}
__device__ __forceinline__ void cache_put_ml(const CacheProb &P, const CacheArgs &A,
                                             const CacheItem &w, int g, int part, int r, float m,
                                             float l) {
  if (part >= 0)
    A.pml[(int64_t)part * P.rows + r] = make_float2(m, l);
  else if (A.lse != nullptr)
    A.lse[cache_out_row(P, w.b, g, w.row0 + r)] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Online softmax step of a lane's N scores of one row (the four lanes of a row hold
// the others): scores to probabilities in place, m, l and o rescaled where the
// reference point m moves.  It may trail the maximum by 8 (a factor 2^8 in p): exact
// after the division by l.
template <int N, int NDB>
__device__ __forceinline__ void cache_softmax(float (&p)[N], float sl2, float &m, float &l,
                                              f32x4 (&o)[NDB]) {
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, p[i]);
  mx = quad_max(mx) * sl2;
  if (__builtin_amdgcn_ballot_w64(mx > m + 8.f) != 0) {
    const float mn = fmaxf(m, mx);
    const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    l *= alpha;
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    m = mn;
  }
  const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], sl2, -mu));
    l += p[i];
  }
}

// Takes the NaNs out of 16 codes; a bit for each.  A value that some rows of a tile
// see and others do not may be one, which a probability of zero would not take out.
__device__ __forceinline__ uint32_t take_nans(u4 &x) {
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = ((x[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // codes 7f and ff
    x[i] &= ~(t | (t - (t >> 7)));
    mask |= ((t >> 7) * 0x01020408u >> 24) << (4 * i);
  }
  return mask;
}

// What take_nans took out of a tile's values, back into the outputs of the rows that
// see it: nan[key * D / 16 + unit], the lane's row sees keys [lo, lo + n) of `keys`.
template <int D, int NDB>
__device__ __forceinline__ void put_nans(const uint16_t *nan, int keys, int lo, int n, int gq,
                                         f32x4 (&o)[NDB]) {
  static_assert(NDB == D / 16, "a unit is a block of 16 channels");
#pragma unroll 1
  for (int key = 0; key < keys; ++key)
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const uint32_t bits = (uint32_t)nan[key * NDB + db] >> (4 * gq);
      const bool sees = (unsigned)(key - lo) < (unsigned)n;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (sees && (bits >> c & 1)) o[db][c] = __uint_as_float(0x7fc00000u);
      __builtin_amdgcn_sched_barrier(0);  // few registers rather than loads ahead
    }
}

// A row's queries, and the keys [lo, lo + n) that it sees.
template <typename T>
struct CacheRow {
  const T *q;
  int lo, n;
  __device__ __forceinline__ CacheRow(const CacheProb &P, const CacheArgs &A, const CacheItem &w,
                                      int g, int row) {
    const int r = min(row, w.row1 - 1);
    const int j = (int)fdiv((uint32_t)r, P.frep), i = r - j * P.rep;
    q = static_cast<const T *>(A.q) + w.b * P.qs[0] + j * P.qs[1] + (int64_t)(g * P.rep + i) * P.qs[2];
    const int t = w.len - P.Lq + j;
    lo = max(t - P.W + 1, 0);
    n = max(t + 1 - lo, 0);
  }
};

// Narrow: 16 NQ rows, the waves take different tiles of 32 keys of [ka, kb): keys go
// from memory into the matrix operand, values through the wave's own LDS (its
// transposing read), no barrier until the waves' results meet.
template <typename T, int D, int NQ, int NW>
__device__ __forceinline__ void cache_narrow(const CacheProb &P, const CacheArgs &A,
                                             const CacheItem &w, int g, int ka, int kb, int part,
                                             char *smem) {
  constexpr int NP = cache_parts<T>(), PP = cache_prob_parts<T>();
  constexpr int NS = D / 64, NDB = D / 16, RS = D + 8;
  constexpr int UPR = D / 16, RPP = 64 / UPR, NU = kTile / RPP;  // V: units per row, rows per pass
  const int tid = threadIdx.x, wv = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 15, gq = lane >> 4;
  __bf16 *const vs = reinterpret_cast<__bf16 *>(smem) + wv * (kTile * RS);  // the wave's own
  uint16_t *const nan = reinterpret_cast<uint16_t *>(smem + sizeof(__bf16) * NW * kTile * RS) +
                        wv * (kTile * UPR);
  Query8<T> qr[NQ][2 * NS];
  int lo[NQ], cnt[NQ];
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const CacheRow<T> row(P, A, w, g, w.row0 + 16 * qi + n);
    lo[qi] = row.lo;
    cnt[qi] = row.n;
#pragma unroll
    for (int s = 0; s < 2 * NS; ++s) {
      const int c = 64 * (s / 2) + 16 * gq + 8 * (s & 1);
      qr[qi][s].load(row.q + c, c < P.D);
    }
  }
  bf8 qf[NQ][2 * NS][NP];
  const int vc = lane % UPR, vr = lane / UPR;
  u4 kr[2][NS], vr8[NU];
  int entry[2];  // of the table, of the loaded tile's halves
  bool bad = false;
  PageWindow win;
  win.base = -64;
  const uint8_t *const kg = P.k.code + g * P.k.st[1], *const vg = P.v.code + g * P.v.st[1];
  const uint32_t ko = (uint32_t)(n * (int)P.k.st[2] + 16 * gq);
  const uint32_t vo = (uint32_t)(vr * (int)P.v.st[2] + 16 * vc);
  // Keys that no row sees are not read: zeros (0 times them is 0).
  const int seen0 = max(ka, w.lo), seen1 = min(kb, w.hi);
  auto load = [&](int t0) {
    const bool whole = t0 >= seen0 && t0 + kTile <= seen1 && P.D == D;
    int page[2];
    entry[0] = t0 >> P.lgT;
    entry[1] = (t0 + 16) >> P.lgT;
    if (!win.holds(entry[0]) || !win.holds(entry[1])) win.load(P, w.b, g, entry[0]);
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) page[hh] = win.page_of(entry[hh]);
    bad = page[0] < 0 || page[1] < 0;
    const int mask = (1 << P.lgT) - 1;
    const uint8_t *const ap[2] = {kg + page[0] * P.k.st[0] + (t0 & mask) * P.k.st[2],
                                  kg + page[1] * P.k.st[0] + ((t0 + 16) & mask) * P.k.st[2]};
    const uint8_t *const bp[2] = {vg + page[0] * P.v.st[0] + (t0 & mask) * P.v.st[2],
                                  vg + page[1] * P.v.st[0] + ((t0 + 16) & mask) * P.v.st[2]};
    if (whole && !bad) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int s = 0; s < NS; ++s)
          kr[hh][s] = *reinterpret_cast<const u4 *>(ap[hh] + 64 * s + ko);
#pragma unroll
      for (int i = 0; i < NU; ++i)
        vr8[i] = *reinterpret_cast<const u4 *>(bp[RPP * i / 16] + (RPP * i % 16) * P.v.st[2] + vo);
    } else {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int key = t0 + 16 * hh + n;
        const bool live = page[hh] >= 0 && key >= seen0 && key < seen1;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          kr[hh][s] = u4{0, 0, 0, 0};
          if (live && 64 * s + 16 * gq < P.D)
            kr[hh][s] = *reinterpret_cast<const u4 *>(ap[hh] + 64 * s + ko);
        }
      }
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int key = t0 + RPP * i + vr;
        vr8[i] = u4{0, 0, 0, 0};
        if (page[RPP * i / 16] >= 0 && key >= seen0 && key < seen1 && 16 * vc < P.D)
          vr8[i] = *reinterpret_cast<const u4 *>(bp[RPP * i / 16] + (RPP * i % 16) * P.v.st[2] + vo);
      }
    }
  };
  f32x4 o[NQ][NDB];
  float m[NQ], l[NQ];
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[qi][db] = zero4();
    m[qi] = -INFINITY;
    l[qi] = 0.f;
  }
  const float sl2 = P.sl2;
  const int tr_off = (4 * gq + (n >> 2)) * RS + 4 * (n & 3);
  const bool spans = P.Lq > 1;
  const int all0 = max(ka, w.lo_max), all1 = min(kb, w.hi_min);  // seen by every row
  auto run_tile = [&](int t0, auto edge_tile) {
    constexpr bool EDGE = decltype(edge_tile)::value;
    f32x4 s[NQ][2];
    float ksc[2], vsc[2];
    bool none[2] = {false, false};  // no page: keys that nothing sees
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int sc = win.scales_of(entry[hh]);
      ksc[hh] = scale_of(sc & 255);
      vsc[hh] = scale_of(sc >> 8);
      if (EDGE) none[hh] = win.page_of(entry[hh]) < 0;
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) s[qi][hh] = zero4();
#pragma unroll
      for (int t = 0; t < 2 * NS; ++t) {
        const bf8 kf = decode8(kr[hh][t / 2][2 * (t & 1)], kr[hh][t / 2][2 * (t & 1) + 1], ksc[hh]);
#pragma unroll
        for (int qi = 0; qi < NQ; ++qi)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) s[qi][hh] = M16::mma(kf, qf[qi][t][p], s[qi][hh]);
      }
    }
    __builtin_amdgcn_wave_barrier();  // the reads of the tile before are issued
    bool odd = false;
    if (EDGE && spans) {
      uint32_t mask[NU];
      bool some = false;
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        mask[i] = take_nans(vr8[i]);
        some |= mask[i] != 0;
      }
      odd = __builtin_amdgcn_ballot_w64(some) != 0;
      if (odd) {
#pragma unroll
        for (int i = 0; i < NU; ++i) nan[(RPP * i + vr) * UPR + vc] = (uint16_t)mask[i];
      }
    }
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      __bf16 *const d = vs + (RPP * i + vr) * RS + 16 * vc;
      const float sc = vsc[RPP * i / 16];
      *reinterpret_cast<bf8 *>(d) = decode8(vr8[i][0], vr8[i][1], sc);
      *reinterpret_cast<bf8 *>(d + 8) = decode8(vr8[i][2], vr8[i][3], sc);
    }
    if (t0 + NW * kTile < kb) load(t0 + NW * kTile);  // in flight during the rest
    float p[NQ][8];
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[qi][i] = s[qi][i / 4][i % 4];
        if (EDGE) {
          const int key = t0 + 16 * (i / 4) + 4 * gq + i % 4;
          if (none[i / 4] || key < ka || key >= kb || (unsigned)(key - lo[qi]) >= (unsigned)cnt[qi])
            p[qi][i] = -INFINITY;
        }
      }
      cache_softmax(p[qi], sl2, m[qi], l[qi], o[qi]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    bf8 bp[NQ][PP];
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) split8<PP>(p[qi], bp[qi]);
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const bf4 lo4 = M16::tr(vs + tr_off + 16 * db);
      const bf4 hi4 = M16::tr(vs + 16 * RS + tr_off + 16 * db);
      const bf8 va = __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi)
#pragma unroll
        for (int x = PP - 1; x >= 0; --x) o[qi][db] = M16::mma(va, bp[qi][x], o[qi][db]);
    }
    if (EDGE && odd) {
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi)
        put_nans<D>(nan, kTile, lo[qi] - t0, cnt[qi], gq, o[qi]);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  };
  int t0 = ka + wv * kTile;
  if (t0 < kb) load(t0);
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi)
#pragma unroll
    for (int s = 0; s < 2 * NS; ++s) qr[qi][s].template parts<NP>(qf[qi][s]);  // beside those loads
  for (; t0 < kb; t0 += NW * kTile) {
    if (t0 >= all0 && t0 + kTile <= all1 && !bad) run_tile(t0, std::false_type{});
    else run_tile(t0, std::true_type{});
  }
  // The waves' results meet in LDS, 16 rows at a time.
  constexpr int PS = D + 4;  // floats per row
  float *const po = reinterpret_cast<float *>(smem);
  float2 *const ml = reinterpret_cast<float2 *>(po + NW * 16 * PS);  // [NW][16]
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const float lt = quad_sum(l[qi]);
    __syncthreads();  // the tiles' LDS is free
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      *reinterpret_cast<f32x4 *>(po + (wv * 16 + n) * PS + 16 * db + 4 * gq) = o[qi][db];
    if (lane < 16) ml[wv * 16 + n] = make_float2(m[qi], lt);
    __syncthreads();
    constexpr int TPR = 4 * NW;  // threads per row
    const int r = tid / TPR;
    if (w.row0 + 16 * qi + r < w.row1) {
      float2 x[NW];
      float mt = -INFINITY, sum = 0.f;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        x[i] = ml[i * 16 + r];
        mt = fmaxf(mt, x[i].x);
      }
      float wt[NW];
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        wt[i] = x[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[i].x - mt);  // (NaN: a seen row)
        sum = x[i].y == 0.f ? sum : fmaf(wt[i], x[i].y, sum);
      }
      for (int c = 4 * (tid % TPR); c < D; c += 4 * TPR) {
        f32x4 a = zero4();
#pragma unroll
        for (int i = 0; i < NW; ++i)
          if (x[i].y != 0.f) a += wt[i] * *reinterpret_cast<const f32x4 *>(po + (i * 16 + r) * PS + c);
        cache_put<T>(P, A, w, g, part, 16 * qi + r, c, a, sum);
      }
      if (tid % TPR == 0) cache_put_ml(P, A, w, g, part, 16 * qi + r, mt, sum);
    }
  }
  __syncthreads();  // before the next item's tiles
}

template <int D>
constexpr int cache_tile() {
  return D > 128 ? 32 : 64;  // keys of a wide tile
}

// Wide: 16 NQ rows per wave; half of the waves stage the keys of a tile in LDS as
// bf16, half the values, for all of them, one barrier per tile.
template <typename T, int D, int NQ, int NW>
__device__ __forceinline__ void cache_wide(const CacheProb &P, const CacheArgs &A,
                                           const CacheItem &w, int g, int ka, int kb, int part,
                                           char *smem) {
  constexpr int NP = cache_parts<T>(), PP = cache_prob_parts<T>();
  constexpr int TK = cache_tile<D>(), CH = TK / 16;
  constexpr int NT = D / 32, NDB = D / 16, RSE = lds_row(D);
  constexpr int UPR = D / 16, RPW = 64 / UPR, RPP = RPW * NW / 2, NU = TK / RPP;
  static_assert(CH / 2 * NDB % NU == 0, "a unit is staged every so many products");
  __bf16 *const buf = reinterpret_cast<__bf16 *>(smem);
  const int tid = threadIdx.x, wv = uniform(tid >> 6), lane = tid & 63;
  const int n = lane & 15, gq = lane >> 4;

  // staging: the lane's unit and row of the wave's RPW; the wave's first row of a pass
  const bool isv = wv >= NW / 2;
  const CachePages &G = isv ? P.v : P.k;
  const int col = 16 * (lane % UPR), rl = lane / UPR, rw = (isv ? wv - NW / 2 : wv) * RPW;
  const int page_st = (int)G.st[0], slot_st = (int)G.st[2];
  const uint8_t *const code = G.code + g * G.st[1] + rl * slot_st + col;
  const int unit = (rw + rl) * RSE + (isv ? lds_y(D) : 0) + col;
  // the part's pages, kEntries at a time: page or -1, scale bytes
  int2 *const table = reinterpret_cast<int2 *>(buf + 2 * TK * RSE);
  // NaNs among the values of a tile that rows see differently: whether a wave found
  // some, and which
  int *const odds = reinterpret_cast<int *>(table + kEntries);      // [2][NW / 2]
  uint16_t *const nan = reinterpret_cast<uint16_t *>(odds + NW);    // [2][TK][UPR]

  const int row0 = w.row0 + wv * (16 * NQ);
  bf8 qf[NQ][NT][NP];
  int lo[NQ], cnt[NQ];  // keys that a row sees
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const CacheRow<T> r(P, A, w, g, row0 + 16 * qi + n);
    lo[qi] = r.lo;
    cnt[qi] = r.n;
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      Query8<T> x;
      x.load(r.q + 32 * s + 8 * gq, 32 * s + 8 * gq < P.D);
      x.template parts<NP>(qf[qi][s]);
    }
  }
  f32x4 o[NQ][NDB];
  float m[NQ], l[NQ];
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[qi][db] = zero4();
    m[qi] = -INFINITY;
    l[qi] = 0.f;
  }
  const float sl2 = P.sl2;
  const int ka_off = n * RSE + 8 * gq;
  const int tr_off = (4 * gq + (n >> 2)) * RSE + 4 * (n & 3);
  const bool spans = P.Lq > 1;  // rows may see different keys

  auto values = [&](const __bf16 *vs, int jj, int db) {  // V^T of 32 keys
    const __bf16 *ca = vs + 32 * jj * RSE + tr_off + 16 * db;
    const bf4 lo4 = M16::tr(ca), hi4 = M16::tr(ca + 16 * RSE);
    return (bf8)__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto product = [&](bf8 a, const auto &b, f32x4 c) {
#pragma unroll
    for (int p = (int)(sizeof(b) / sizeof(bf8)) - 1; p >= 0; --p) c = M16::mma(a, b[p], c);
    return c;
  };
  typedef f32x4 Scores[NQ][CH];
  Scores sa, sb;  // of the tile at hand and of the next
  float mx[NQ];   // the lane's largest score of the tile at hand
  auto largest = [&](const Scores &s, int qi, int ch) {
#pragma unroll
    for (int r = 0; r < 4; ++r) mx[qi] = fmaxf(mx[qi], s[qi][ch][r]);
  };
  const int per_chunk = kEntries << P.lgT;
  for (int ca = ka; ca < kb;) {
  const int e0 = ca >> P.lgT, cb = min(kb, (e0 << P.lgT) + per_chunk), e1 = (cb - 1) >> P.lgT;
  const int seen0 = max(ca, w.lo), seen1 = min(cb, w.hi);
  u4 pre[NU];
  float sc[NU];
  const int nkt = (cb - ca + TK - 1) / TK;
  // The tiles that every row sees in full are [ja, jb); they come first, then
  // those behind them, then those before.
  int ja = (max(w.lo_max - ca, 0) + TK - 1) / TK, jb = max(min(w.hi_min, cb) - ca, 0) / TK;
  if (jb <= ja) ja = jb = 0;
  auto first_key = [&](int i) {  // of the i-th tile
    const int j = ja + i;
    return ca + (j < nkt ? j : j - nkt) * TK;
  };
  // The table names a page that is none, among those that rows see.  (Pages in front of
  // every window may have been given back: 2048 tokens of 32 heads of 64, a window of
  // 4000, pages of 16: 209 us; 289 where those count.)
  bool bad = false;
  // The lane's units of a tile; entry(i): entry i of the table.
  auto load = [&](int mine, u4 (&x)[NU], float (&scale)[NU], auto entry) {
    const int t0 = first_key(max(min(mine, nkt - 1), 0));
    const bool some = mine >= 0 && mine < nkt;
    const bool whole = some && !bad && t0 >= seen0 && t0 + TK <= seen1 && P.D == D;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      const int key = t0 + rw + RPP * u;  // the wave's rows of a pass: one page's
      const int2 at = entry(min(key >> P.lgT, e1));
      scale[u] = scale_of(isv ? at.y >> 8 : at.y & 255);
      const uint8_t *const p = code + (int64_t)at.x * page_st + (key & ((1 << P.lgT) - 1)) * slot_st;
      if (whole) {
        x[u] = *reinterpret_cast<const u4 *>(p);
      } else {  // zeros for keys that no row sees and channels past the last: 0 times them is 0
        x[u] = u4{0, 0, 0, 0};
        if (some && at.x >= 0 && key + rl >= seen0 && key + rl < seen1 && col < P.D)
          x[u] = *reinterpret_cast<const u4 *>(p);
      }
    }
  };
  // V of the i-th tile and K of the next: the scores run one tile ahead.
  auto fetch = [&](int i) {
    load(isv ? i : i + 1, pre, sc, [&](int e) { return table[e - e0]; });
  };
  // The first tiles' loads go out beside the table's: K of two, V of one.
  u4 head[NU];
  float head_sc[NU];
  __syncthreads();  // the chunk before is done with the table
  {
    auto direct = [&](int e) { return cache_entry(P, w.b, g, e); };
    bool none = false;
    for (int e = (seen0 >> P.lgT) + lane; e <= (seen1 - 1) >> P.lgT; e += 64)
      none |= (uint32_t)(e < P.M ? P.tables[w.b * P.ts + e] : -1) >= (uint32_t)P.pages;
    bad = __builtin_amdgcn_ballot_w64(none) != 0;
    load(0, head, head_sc, direct);
    if (!isv) load(1, pre, sc, direct);
    for (int e = e0 + tid; e <= e1; e += 64 * NW) table[e - e0] = direct(e);
  }
  const int full = bad ? 0 : (jb - ja) & ~1;  // tiles that run as seen by every row
  auto put_unit = [&](int tile, int u, const u4 &x, float scale) {
    __bf16 *const d = buf + (tile & 1) * (TK * RSE) + unit + RPP * u * RSE;
    *reinterpret_cast<bf8 *>(d) = decode8(x[0], x[1], scale);
    *reinterpret_cast<bf8 *>(d + 8) = decode8(x[2], x[3], scale);
  };
  auto note_nans = [&](int tile, u4 (&x)[NU]) {
    if (isv && spans && tile >= full) {
      bool some = false;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const uint32_t mask = take_nans(x[u]);
        nan[(tile & 1) * (TK * UPR) + (rw + RPP * u + rl) * UPR + lane % UPR] = (uint16_t)mask;
        some |= mask != 0;
      }
      some = __builtin_amdgcn_ballot_w64(some) != 0;
      if (lane == 0) odds[(tile & 1) * (NW / 2) + wv - NW / 2] = some;
    }
  };
  // The i-th tile, its scores in `s`; the next tile's go to `next`.  EDGE: some
  // row does not see some of its keys.  Matrix products are issued between the vector
  // ALU's work, which fills the matrix unit's time: the next tile's scores beside the
  // first half of the exponentials, O beside the second.
  auto run_tile = [&](int i, Scores &s, Scores &next, auto edge_tile) {
    constexpr bool EDGE = decltype(edge_tile)::value;
    const __bf16 *vs = buf + (i & 1) * (TK * RSE) + lds_y(D);
    const __bf16 *ks = buf + ((i + 1) & 1) * (TK * RSE) + ka_off;
    const int t0 = first_key(i);
    int none = 0;  // groups of 16 keys of no page, one a bit
    if (EDGE && bad) {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch)
        none |= table[min((t0 + 16 * ch) >> P.lgT, e1) - e0].x < 0 ? 1 << ch : 0;
    }
    fetch(i + 1);  // in flight during this tile
    bool moves = false;
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      if (EDGE) {
        mx[qi] = -INFINITY;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = t0 + 16 * ch + 4 * gq + r;
            if ((none >> ch & 1) || key < ca || key >= cb || (unsigned)(key - lo[qi]) >= (unsigned)cnt[qi])
              s[qi][ch][r] = -INFINITY;
          }
          largest(s, qi, ch);
        }
      }
      moves |= mx[qi] * sl2 > m[qi] + 8.f;
    }
    // the reference point may trail the maximum by 8 (a factor 2^8 in p): exact after
    // the division by l
    if (__builtin_amdgcn_ballot_w64(moves) != 0) {
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        const float mn = fmaxf(m[qi], quad_max(mx[qi]) * sl2);
        const float alpha = __builtin_amdgcn_exp2f(m[qi] - (mn == -INFINITY ? 0.f : mn));
        l[qi] *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[qi][db] *= alpha;
        m[qi] = mn;
      }
    }
    float mu[NQ];
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) mu[qi] = m[qi] == -INFINITY ? 0.f : m[qi];
    auto expo = [&](int qi, int x) {  // the x-th of the lane's CH * 4 probabilities
      float &p = reinterpret_cast<float (&)[CH][4]>(s[qi])[x / 4][x % 4];
      p = __builtin_amdgcn_exp2f(fmaf(p, sl2, -mu[qi]));
      l[qi] += p;
    };
    auto rounded = [&](int qi, int jj, bf8 (&b)[PP]) {
      float p[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) p[x] = s[qi][2 * jj + x / 4][x % 4];
      split8<PP>(p, b);
    };
    constexpr int ALL = CH * 4, FIRST = CH > 2 ? ALL / 2 : ALL;  // a lane's scores, beside QK
    constexpr int QS = CH * NT, OS = CH / 2 * NDB;  // steps of the two products
    constexpr int RING = 3;
    bf8 kf[RING];  // of the next steps
    auto key = [&](int st) {
      return *reinterpret_cast<const bf8 *>(ks + 16 * (st / NT) * RSE + 32 * (st % NT));
    };
#pragma unroll
    for (int st = 0; st < RING - 1; ++st) kf[st] = key(st);
#pragma unroll
    for (int st = 0; st < QS; ++st) {
      const int ch = st / NT, t = st % NT;
      if (st + RING - 1 < QS) kf[(st + RING - 1) % RING] = key(st + RING - 1);
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        next[qi][ch] = product(kf[st % RING], qf[qi][t], t == 0 ? zero4() : next[qi][ch]);
#pragma unroll
        for (int x = st * FIRST / QS; x < (st + 1) * FIRST / QS; ++x) expo(qi, x);
      }
      __builtin_amdgcn_sched_barrier(0x124);
    }
    bf8 bp[NQ][PP];
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) rounded(qi, 0, bp[qi]);
    bf8 va[2];
    va[0] = values(vs, 0, 0);
#pragma unroll
    for (int st = 0; st < OS; ++st) {
      const int jj = st / NDB, db = st % NDB;
      if (jj > 0 && db == 0) {
#pragma unroll
        for (int qi = 0; qi < NQ; ++qi) rounded(qi, jj, bp[qi]);
      }
      if (st + 1 < OS) va[(st + 1) & 1] = values(vs, (st + 1) / NDB, (st + 1) % NDB);
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        o[qi][db] = product(va[st & 1], bp[qi], o[qi][db]);
        if (jj == 0) {
#pragma unroll
          for (int x = FIRST + db * (ALL - FIRST) / NDB; x < FIRST + (db + 1) * (ALL - FIRST) / NDB; ++x)
            expo(qi, x);
        }
      }
      // the next tiles' units between the products, which go on meanwhile
      if (st == 0) note_nans(i + 1, pre);
      if ((st + 1) % (OS / NU) == 0) {
        constexpr int EVERY = OS / NU;
        put_unit(isv ? i + 1 : i + 2, st / EVERY, pre[st / EVERY], sc[st / EVERY]);
      }
      __builtin_amdgcn_sched_barrier(0x124);
    }
    if (EDGE && spans) {
      int odd = 0;
#pragma unroll
      for (int x = 0; x < NW / 2; ++x) odd |= odds[(i & 1) * (NW / 2) + x];
      if (uniform(odd) != 0) {
#pragma unroll
        for (int qi = 0; qi < NQ; ++qi)
          put_nans<D>(nan + (i & 1) * (TK * UPR), TK, lo[qi] - t0, cnt[qi], gq, o[qi]);
      }
    }
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      mx[qi] = -INFINITY;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) largest(next, qi, ch);
    }
    __syncthreads();
  };
  note_nans(0, head);
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    put_unit(0, u, head[u], head_sc[u]);
    if (!isv) put_unit(1, u, pre[u], sc[u]);
  }
  __syncthreads();
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) mx[qi] = -INFINITY;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    bf8 kf[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      kf[t] = *reinterpret_cast<const bf8 *>(buf + ka_off + 16 * ch * RSE + 32 * t);
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      sa[qi][ch] = zero4();
#pragma unroll
      for (int t = 0; t < NT; ++t) sa[qi][ch] = product(kf[t], qf[qi][t], sa[qi][ch]);
      largest(sa, qi, ch);
    }
  }
  __syncthreads();  // these keys' place is the tile's after next
  int i = 0;
  for (; i < full; i += 2) {
    run_tile(i, sa, sb, std::false_type{});
    run_tile(i + 1, sb, sa, std::false_type{});
  }
  for (; i < nkt; ++i) {
    run_tile(i, sa, sb, std::true_type{});
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi)
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) sa[qi][ch] = sb[qi][ch];
  }
  ca = cb;
  }
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const float lt = quad_sum(l[qi]);
    const int r = wv * (16 * NQ) + 16 * qi + n;
    if (w.row0 + r >= w.row1) continue;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      cache_put<T>(P, A, w, g, part, r, 16 * db + 4 * gq, o[qi][db], lt);
    if (gq == 0) cache_put_ml(P, A, w, g, part, r, m[qi], lt);
  }
}

// This workgroup's part of the keys.  All units are shared out evenly, in order, so
// that a workgroup may end one item and begin others; or, where its even share is at
// most kAligned units and the items are fewer than the workgroups, each takes one chunk
// of one item, as beginning an item costs the time of several units.
template <typename F>
__device__ __forceinline__ void cache_parts_of(const CacheProb &P, const CacheArgs &A, F &&run) {
  CacheScan scan;
  int per_head = scan.total(P, 1), all = per_head * P.Hkv;  // (below 2^31: the host's check)
  if (all == 0) return;
  const int share = uniform(max((all - 1) / P.wgs + 1, P.least));
  int chunk = 1, n;
  if (share <= kAligned && P.items * P.Hkv <= P.wgs) {
    for (chunk = share; (per_head = scan.total(P, chunk)) * P.Hkv > P.wgs;) chunk += (chunk + 7) / 8;
    n = all = per_head * P.Hkv;
  } else {
    n = uniform(min((all - 1) / P.least + 1, P.wgs));
  }
  chunk = uniform(chunk);
  per_head = uniform(per_head);
  all = uniform(all);
  n = uniform(n);
  // tiles next to each other read the same keys: through one XCD's L2
  const int me = P.rt > 1 && n == P.wgs ? xcd_tile(blockIdx.x, P.wgs) : blockIdx.x;
  if (me >= n) return;
  int u = uniform((int)((int64_t)all * me / n));
  const int end = uniform((int)((int64_t)all * (me + 1) / n));
  int g = uniform(u / per_head);
  int off = u - g * per_head;
  int i = uniform(scan.find(P, off, chunk));
  off = uniform(off);
  while (u < end) {
    CacheItem w = scan.item(P, i);
    cache_uniform(w);
    if (w.units > 0) {
      const int chunks = uniform((w.units + chunk - 1) / chunk);
      const int take = min(chunks - off, end - u);
      const bool begins = off == 0, whole = begins && take == chunks;
      if (begins && threadIdx.x == 0) {
        // the workgroup that chunk x lies in is the largest whose part begins at x or before
        const int64_t x = u + chunks;
        A.span[(int64_t)g * P.items + i] = make_int2(me, (int)((x * n + all - 1) / all) - 1);
      }
      // (a chunk of several units: no more than kAligned a workgroup, the products are small)
      const int ua = chunk == 1 ? off : uniform(w.units * off / chunks);
      const int ub = chunk == 1 ? off + take : uniform(w.units * (off + take) / chunks);
      run(w, g, w.k0 + ua * kUnit, min(w.k0 + ub * kUnit, w.hi), whole ? -1 : 2 * me + (begins ? 1 : 0));
      u += take;
    }
    off = 0;
    if (++i == P.items) {
      i = 0;
      ++g;
    }
  }
}

// (float32 of 128 channels spills 3 registers: 16 x 8 heads, 5.2 TB/s all the same)
template <typename T, int D, int NQ, int NW>
__global__ void __launch_bounds__(64 * NW, D > 128 ? 1 : 2) k_cache_narrow(CacheProb P, CacheArgs A) {
  extern __shared__ __align__(16) char smem[];
  cache_parts_of(P, A, [&](const CacheItem &w, int g, int ka, int kb, int part) {
    cache_narrow<T, D, NQ, NW>(P, A, w, g, ka, kb, part, smem);
  });
}

// An item a workgroup.  Two of 64 bf16 channels share a CU (64 x 8 heads, 2048 keys: 24.4
// us, one 26.9).
template <typename T, int D>
__global__ void __launch_bounds__(64 * cache_whole(D).waves, (std::is_same<T, bf16_t>::value && D <= 64 ? 4 : 1))
    k_cache_whole(CacheProb P, CacheArgs A) {
  extern __shared__ __align__(16) char smem[];
  const int g = (int)(blockIdx.x / (uint32_t)P.items);
  const int i = (int)blockIdx.x - g * P.items;
  CacheItem w = cache_item(P, i, cache_len(P, i));
  cache_uniform(w);
  cache_narrow<T, D, 1, cache_whole(D).waves>(P, A, w, uniform(g), w.k0, w.hi, -1, smem);
}

// Waves that a SIMD holds of a wide workgroup's.  Eight waves of 16 bf16 rows of 64
// channels run as four, which spills 5 registers (8 x 8 heads, 512 rows: 138 us, as three
// 167, as two 164; 128 rows: 50, 60 and 61).  Of 128 channels eight waves of 32 rows spill
// 22, and are faster than 16 rows, which spill none (cache_shape's figures).
template <typename T, int D, int NW>
constexpr int cache_wide_waves() {
  return D > 128 ? 1 : std::is_same<T, bf16_t>::value && D <= 64 && NW == 8 ? 4 : 2;
}

template <typename T, int D, int NQ, int NW>
__global__ void __launch_bounds__(64 * NW, (cache_wide_waves<T, D, NW>())) k_cache_wide(CacheProb P, CacheArgs A) {
  extern __shared__ __align__(16) char smem[];
  cache_parts_of(P, A, [&](const CacheItem &w, int g, int ka, int kb, int part) {
    cache_wide<T, D, NQ, NW>(P, A, w, g, ka, kb, part, smem);
  });
}

// The parts of a row added: lanes take four channels each, 2^lgG of them a row, and
// 2^lgS such groups share the row's parts, each kJoin at a time.
template <typename T>
__global__ void __launch_bounds__(256) k_cache_join(CacheProb P, CacheArgs A, int lgG, int lgS) {
  __shared__ f32x4 so[256];
  __shared__ float2 sml[256];
  const int tid = threadIdx.x, c = 4 * (tid & ((1 << lgG) - 1));
  const int share = (tid >> lgG) & ((1 << lgS) - 1);
  const int64_t rows = (int64_t)P.B * P.Hkv * P.Mo;
  const int64_t mine = ((int64_t)blockIdx.x * 256 + tid) >> (lgG + lgS);
  const int64_t at = min(mine, rows - 1), bg = at / P.Mo;
  const int row = (int)(at - bg * P.Mo), b = (int)(bg / P.Hkv), g = (int)(bg - (int64_t)b * P.Hkv);
  const int tile = row / P.rows, item = b * P.rt + tile, r = row - tile * P.rows;
  int2 span = A.span[(int64_t)g * P.items + item];  // beside the length
  if (cache_item(P, item, cache_len(P, item)).units == 0) span = make_int2(0, -1);  // (not written)
  float m = -INFINITY, l = 0.f;
  f32x4 acc = zero4();
  if (span.x != span.y) {  // (else its workgroup has written it)
    for (int i0 = span.x + share; i0 <= span.y; i0 += kJoin << lgS) {  // a batch's loads together
      float2 x[kJoin];
      f32x4 o[kJoin];
#pragma unroll
      for (int u = 0; u < kJoin; ++u) {
        const int i = i0 + (u << lgS);
        x[u] = make_float2(-INFINITY, 0.f);
        o[u] = zero4();
        if (i <= span.y) {
          const int64_t part = (int64_t)(2 * i + (i == span.x ? 1 : 0)) * P.rows + r;
          x[u] = A.pml[part];
          if (c < P.D) o[u] = *reinterpret_cast<const f32x4 *>(A.po + part * P.D + c);
        }
      }
      float mn = m;
#pragma unroll
      for (int u = 0; u < kJoin; ++u) mn = fmaxf(mn, x[u].x);
      if (l != 0.f) {
        const float wt = __builtin_amdgcn_exp2f(m - mn);
        l *= wt;
        acc *= wt;
      }
      m = mn;
#pragma unroll
      for (int u = 0; u < kJoin; ++u)
        if (x[u].y != 0.f) {  // (0: a row that sees nothing of the part)
          const float wt = __builtin_amdgcn_exp2f(x[u].x - m);
          l = fmaf(wt, x[u].y, l);
          acc += wt * o[u];
        }
    }
  }
  if (lgS > 0) {
    so[tid] = acc;
    sml[tid] = make_float2(m, l);
    __syncthreads();
    if (share != 0) return;
    for (int i = 1; i < 1 << lgS; ++i) m = fmaxf(m, sml[tid + (i << lgG)].x);
    l = 0.f;
    acc = zero4();
    for (int i = 0; i < 1 << lgS; ++i) {
      const float2 x = sml[tid + (i << lgG)];
      if (x.y != 0.f) {
        const float wt = __builtin_amdgcn_exp2f(x.x - m);
        l = fmaf(wt, x.y, l);
        acc += wt * so[tid + (i << lgG)];
      }
    }
  }
  if (mine >= rows || span.x == span.y) return;
  const int64_t out = cache_out_row(P, b, g, row);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (c < P.D) cache_store4(static_cast<T *>(A.out) + out * P.D + c, acc * inv);
  if (c == 0 && A.lse != nullptr) A.lse[out] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// The instance's channels.  Widths between them run as the next, with guarded loads (a
// token, 32 x 8 heads, us: 32 channels 64 and 64 52, 80 105 and 128 104, 208 281 and 256 190).
int cache_width(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// Rows of a tile, the workgroup's waves, workgroups that the chip holds at once, and
// units that one takes at least (of 64 keys; a part costs its rows * D floats).
struct CacheShape {
  int rows, waves, wgs, least;
};
// Times in us, 8192 keys, bf16 but where said; heads: samples x key/value heads.
CacheShape cache_shape(int dtype, int D, int64_t rows) {
  // Float32's three parts leave registers for 16 rows; so do more than 64 channels (16 x 8
  // heads, 32 rows of 128: 72 to 75, a wide tile of 64 84 to 86; 8 x 4 heads, 24 of 256: 49
  // and the wide one 52).  More than 128 channels: one workgroup a CU (16 x 1 heads, 16
  // rows: 26, two of them 35).
  if (dtype == NA_F32 || rows <= (D > 64 ? 32 : 16)) return {16, 4, D > 128 ? 256 : 512, 2};
  if (rows <= 32) return {32, 4, 512, 2};  // (8 x 4 heads: 21; 16 rows 23, a wide tile 27)
  // fp16's two parts leave registers for one workgroup a CU (2 x 8 heads, 2048 rows: 735,
  // grids of two 750; bf16 481, of one 690)
  if (D > 128) return {64, 4, dtype == NA_F16 ? 256 : 512, 1};
  // (16 x 8 heads, 48 rows of 128: 86, three narrow tiles 125; 64 rows: 87, in a tile of
  // 128 118; of 64 channels 59 and 80)
  if (rows <= 64) return {64, 4, 512, 1};
  // (8 x 8 heads, 256 rows of 128: fp16 135, in tiles of 64 156; bf16 114, in tiles of 64
  // 142, of 128 119; 2 x 8 heads, 4096 rows: 352, 503 and 410; 16 x 8 heads, 128 rows: in a
  // tile of 256 194, of 128 122)
  if (dtype == NA_F16 || (D > 64 && rows <= 128)) return {128, 8, 256, 1};
  if (D > 64) return {256, 8, 256, 1};
  return {128, 8, 512, 1};  // (8 x 8 heads, 512 rows: 138, in tiles of 64 170)
}

// The most keys that an item's rows see, where tables are full.
int64_t cache_keys(const CacheProb &P) {
  return std::min((int64_t)P.M << P.lgT, (int64_t)P.W + P.rows);
}

CacheProb cache_prob(const na_cache_params *p, const na_cache *c) {
  CacheProb P{};
  P.B = p->batch;
  P.Lq = p->tokens;
  P.H = p->heads;
  P.Hkv = p->kv_heads;
  P.rep = p->heads / p->kv_heads;
  P.D = p->head_dim;
  P.Mo = P.Lq * P.rep;
  const CacheShape shape = cache_shape(p->dtype, P.D, P.Mo);
  P.rows = shape.rows;
  P.rt = (P.Mo + P.rows - 1) / P.rows;
  P.items = P.B * P.rt;
  P.pages = p->pages;
  P.lgT = lg_page(p->page_size);
  P.M = p->table_pages;
  P.W = p->window > 0 ? std::min(p->window, 1 << 30) : 1 << 30;
  P.least = shape.least;
  const CacheWhole whole = cache_whole(cache_width(P.D));
  const int64_t items = (int64_t)P.items * P.Hkv;
  const bool is_whole = P.rows == 16 && cache_keys(P) <= (items < 128 ? whole.keys : whole.many) &&
                        items * 64 * whole.waves < ((int64_t)1 << 32);
  P.wgs = is_whole ? 0 : shape.wgs;
  P.sl2 = p->scale * kLog2e;
  P.frep = make_fastdiv((uint32_t)P.rep);
  P.frt = make_fastdiv((uint32_t)P.rt);
  for (int i = 0; i < 3; ++i) P.qs[i] = p->q_stride[i];
  P.ts = p->table_stride;
  if (c != nullptr) {
    P.k = {static_cast<uint8_t *>(c->key), static_cast<uint8_t *>(c->key_scale),
           {c->key_stride[0], c->key_stride[1], c->key_stride[2]},
           {c->key_scale_stride[0], c->key_scale_stride[1]}};
    P.v = {static_cast<uint8_t *>(c->value), static_cast<uint8_t *>(c->value_scale),
           {c->value_stride[0], c->value_stride[1], c->value_stride[2]},
           {c->value_scale_stride[0], c->value_scale_stride[1]}};
  }
  return P;
}

struct CacheSizes {
  size_t po, pml, span;
  explicit CacheSizes(const CacheProb &P) {
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    po = up((size_t)2 * P.wgs * P.rows * P.D * sizeof(float));
    pml = up((size_t)2 * P.wgs * P.rows * sizeof(float2));
    span = up((size_t)P.Hkv * P.items * sizeof(int2));  // (never nothing: a caller may count on it)
  }
  size_t total() const { return po + pml + span; }
};

// Logs of the join's lanes per row and of the groups that share a row's parts: kJoin
// of them each where the workgroups are shared evenly by the items.
struct CacheJoinLanes {
  int lgG = 0, lgS = 0;
  explicit CacheJoinLanes(const CacheProb &P) {
    while ((4 << lgG) < P.D) ++lgG;
    const int64_t parts = P.wgs / std::max<int64_t>((int64_t)P.items * P.Hkv, 1) + 2;
    while (lgG + lgS < 8 && ((int64_t)kJoin << lgS) < parts) ++lgS;
  }
  int total() const { return lgG + lgS; }
};

size_t cache_narrow_lds(int D, int waves) {
  const size_t meet = waves * (sizeof(float) * 16 * (D + 4) + sizeof(float2) * 16);
  const size_t tiles = waves * kTile * (sizeof(__bf16) * (D + 8) + sizeof(uint16_t) * (D / 16));
  return std::max(meet, tiles);
}

template <typename T, int D, int NQ, int NW, bool WIDE>
void cache_launch(const CacheProb &P, const CacheArgs &A, hipStream_t st) {
  if constexpr (WIDE) {
    const size_t lds = sizeof(__bf16) * 2 * cache_tile<D>() * lds_row(D) +
                       sizeof(int2) * kEntries + sizeof(int) * NW +
                       sizeof(uint16_t) * 2 * cache_tile<D>() * (D / 16);
    hipLaunchKernelGGL((k_cache_wide<T, D, NQ, NW>), dim3(P.wgs), dim3(64 * NW), lds, st, P, A);
  } else {
    hipLaunchKernelGGL((k_cache_narrow<T, D, NQ, NW>), dim3(P.wgs), dim3(64 * NW),
                       cache_narrow_lds(D, NW), st, P, A);
  }
}

template <typename T, int D>
void cache_launch_whole(const CacheProb &P, const CacheArgs &A, hipStream_t st) {
  hipLaunchKernelGGL((k_cache_whole<T, D>), dim3((unsigned)(P.items * P.Hkv)), dim3(64 * cache_whole(D).waves),
                     cache_narrow_lds(D, cache_whole(D).waves), st, P, A);
}

template <typename T>
void cache_run(const CacheProb &P, const CacheArgs &A, hipStream_t st) {
  auto by_rows = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (P.wgs == 0) return cache_launch_whole<T, D>(P, A, st);
    if constexpr (sizeof(T) == 2) {
      if (P.rows == 64) return cache_launch<T, D, 1, 4, true>(P, A, st);
      if constexpr (D <= 64) {
        if (P.rows == 32) return cache_launch<T, D, 2, 4, false>(P, A, st);
      }
      if constexpr (D <= 128) {
        if constexpr (std::is_same<T, bf16_t>::value && D > 64) {
          if (P.rows == 256) return cache_launch<T, D, 2, 8, true>(P, A, st);
        }
        if (P.rows == 128) return cache_launch<T, D, 1, 8, true>(P, A, st);
      }
    }
    cache_launch<T, D, 1, 4, false>(P, A, st);
  };
  const int width = cache_width(P.D);
  if (width == 256) by_rows(std::integral_constant<int, 256>{});
  else if (width == 128) by_rows(std::integral_constant<int, 128>{});
  else by_rows(std::integral_constant<int, 64>{});
  if (P.wgs == 0) return;
  const CacheJoinLanes n(P);
  const int64_t threads = ((int64_t)P.B * P.Hkv * P.Mo) << n.total();
  hipLaunchKernelGGL((k_cache_join<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, P, A,
                     n.lgG, n.lgS);
}

}  // namespace

// A launch has fewer than 2^32 threads.
bool cache_attend_fits(const na_cache_params *p, size_t *workspace_bytes) {
  const CacheProb P = cache_prob(p, nullptr);
  *workspace_bytes = CacheSizes(P).total();
  const int64_t threads = ((int64_t)P.B * P.Hkv * P.Mo) << CacheJoinLanes(P).total();
  // all units, as the kernels count them, of full tables
  const int64_t units = (int64_t)P.items * P.Hkv * (cache_keys(P) / kUnit + 2);
  return threads < ((int64_t)1 << 32) - 256 && units < ((int64_t)1 << 31);
}

void cache_attend(const na_cache_params *p, const na_cache *c, const void *q, const int32_t *tables,
                  const int32_t *lens, void *out, float *lse, void *workspace, hipStream_t st) {
  CacheProb P = cache_prob(p, c);
  P.tables = tables;
  P.lens = lens;
  const CacheSizes s(P);
  char *const ws = static_cast<char *>(workspace);
  const CacheArgs A{q, out, lse, reinterpret_cast<float *>(ws),
                    reinterpret_cast<float2 *>(ws + s.po),
                    reinterpret_cast<int2 *>(ws + s.po + s.pml)};
  if (p->dtype == NA_F32) cache_run<float>(P, A, st);
  else if (p->dtype == NA_F16) cache_run<f16_t>(P, A, st);
  else cache_run<bf16_t>(P, A, st);
}

}  // namespace na
