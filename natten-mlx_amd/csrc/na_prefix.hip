// na_prefix.hip — attention of new tokens against a cache whose prefix the whole
// batch shares (serving).
//
// Query token j of sample b is token t = len_b - Lq + j of the sample's own
// sequence.  It sees all N prefix tokens, of which there is one copy, and its own
// tokens max(0, t - W + 1) .. t:
//   out = softmax(scale q k^T) v over both, lse the log of the softmax's sum.
//
// The prefix's keys are one product for the batch: the rows of a key/value head
// are all its query heads of all tokens of all samples, so every prefix tile is
// read once per tile of rows instead of once per sample: 128 or 256 rows in 16-bit
// types, 64 of them in heads past 128 channels or where there are no more, 16 in
// float32 or where there are no more.  A sample's own keys meet its own rows only.
// Both are cut into chunks of keys; a workgroup takes a chunk against a tile of rows
// and leaves (m, l, o) -- reference point, sum and unnormalised output of an online
// softmax, float32 -- and k_pfx_join adds the chunks of a row.  One launch holds the
// prefix's workgroups and the samples'.
//
// Two shapes of workgroup (NW waves, four or eight):
//  * wide: 16 NQ rows per wave, the waves share K / V tiles staged in LDS, one
//    barrier per tile;
//  * narrow: 16 rows, the waves take different tiles of 32 keys: K goes
//    from memory straight into the matrix operand, V through the wave's own LDS
//    (its transposing read), no barrier until the waves' results meet.
// float32 runs narrow on the float32 matrix cores, without LDS tiles.
//
// Scores, m, l and o are float32.  16-bit types round each probability to their
// own type before the product with V, as the matrix cores take it (off by at most
// half a step each, in fp16 at least 2^-32 of the row's largest; l adds them
// unrounded); out is rounded once.
//
// Bound, each on its own: narrow workgroups by memory (32 samples of 8 heads and up
// to 2048 own tokens of 128 bf16 channels against a prefix of 16384: k_pfx 43 us for
// 219 MB read, 5.0 TB/s; the join 6); wide ones by the exponentials beside the products:
// a score costs a quarter-rate exp2 and four more vector instructions, as much as
// its matrix work at 128 channels and twice it at 64 (1100 TFLOP/s with eight waves
// at 128 channels, 720 at 64; a large product of the library reaches 1183).  Both
// wait for the last workgroups where those in use are no whole rounds of the chip's
// 512 places: about 700 in the call above.
// Counters of 64 samples against 65536 prefix keys (161 us under the profiler, 147
// without): 551 MB read, matrix unit busy 30%, waves waiting for memory 35%.
//
// The wide instances of 128 channels use all 256 registers and spill 135 (four
// waves) or 151 (eight), those of 64 spill 12: in the loop over tiles of which some
// row sees a part, which causal diagonals and windows take (8 samples of 128 tokens,
// 16 heads of 128 channels, window 255 over 640, prefix 8192: 126 us, 60 by
// operations).  float32, whose workgroups hold 16 rows, takes 2.6 times its floor for
// one token (32 samples of 8 heads, up to 2048 own tokens of 128 channels, prefix
// 16384: 213 us, 83 by bytes) and 1.9 times for a prompt (8 samples of 128 tokens, 16
// heads of 64 channels, prefix 8192: 433 us, 230 by operations at the 154 TFLOP/s of
// a large product).
#include "na_launch.h"
#include "na_lean.h"

#include <algorithm>

namespace na {
namespace {

constexpr int kPfxNarrowKeys = 32;  // keys of a wave's tile
constexpr int kPfxJoin = 8;         // slots that a thread of the join loads at once

struct PfxProb {
  int32_t Lq, H, Hkv, rep, D;
  int32_t M, Mo;            // rows per key/value head: of the batch, of a sample
  int32_t N, S, W;          // prefix tokens, cached tokens a sample can hold, window
  int32_t n_prefix, n_own;  // workgroups
  int32_t prefix_launch;    // n_prefix up to a multiple of 8
  int32_t own_launch;
  int32_t rt_p, rt_o;       // row tiles
  int32_t rows_p, rows_o;   // rows per tile: 16 narrow, more wide
  int32_t waves;            // of a workgroup: 4 or 8
  int32_t chunk_p, chunk_o, SP, SO, NS;  // keys per chunk; chunks; slots per row
  float sl2;                // scale * log2(e)
  FastDiv frep, fLq, frt_p, fSP, frt_o, fSO, fHkv;
  int64_t qs[3];            // element strides: sample, token, head
  int64_t pks[2], pvs[2];   // prefix: token, head
  int64_t ks[3], vs[3];     // own: sample, token, head
  const int32_t *lens;      // own tokens per sample, or null: S
};

struct PfxArgs {
  const void *q, *pk, *pv, *k, *v;
  void *out;
  float *lse;
  float *po;    // [Hkv][M][NS][D] partial outputs, or null: one slot, written to out
  float2 *pml;  // [Hkv][M][NS] reference points and sums
};

__device__ __forceinline__ int pfx_len(const PfxProb &P, int b) {
  return P.lens == nullptr ? P.S : min(max(P.lens[b], 0), P.S);
}

// Own tokens [lo, hi) that token j of a sample of `len` tokens sees.
struct PfxSpan {
  int lo, hi;
};
__device__ __forceinline__ PfxSpan pfx_span(const PfxProb &P, int len, int j) {
  const int t = len - P.Lq + j;
  PfxSpan s;
  s.hi = max(t + 1, 0);
  s.lo = max(t - P.W + 1, 0);
  return s;
}

// What a workgroup does: keys [k0, k1) of one head against rows [row0, row1).
struct PfxItem {
  const char *k, *v;    // of key 0
  int64_t kst, vst;     // bytes from key to key
  int g, b, len;        // b < 0: the prefix
  int k0, k1, row0, row1, slot;
  int lo_max, hi_min;   // keys that every row sees: [lo_max, hi_min)
};

// False where there is nothing to do.
template <typename T>
__device__ __forceinline__ bool pfx_item(const PfxProb &P, const PfxArgs &A, int bid, PfxItem &w) {
  if (bid < P.prefix_launch) {
    const int item = xcd_tile(bid, P.prefix_launch);  // a chunk's row tiles share an L2
    if (item >= P.n_prefix) return false;
    const int c = (int)fdiv((uint32_t)item, P.frt_p), rt = item - c * P.rt_p;
    w.g = (int)fdiv((uint32_t)c, P.fSP);
    w.slot = c - w.g * P.SP;
    w.b = -1;
    w.len = 0;
    w.k0 = w.slot * P.chunk_p;
    w.k1 = min(w.k0 + P.chunk_p, P.N);
    w.row0 = rt * P.rows_p;
    w.row1 = min(w.row0 + P.rows_p, P.M);
    w.k = reinterpret_cast<const char *>(static_cast<const T *>(A.pk) + w.g * P.pks[1]);
    w.v = reinterpret_cast<const char *>(static_cast<const T *>(A.pv) + w.g * P.pvs[1]);
    w.kst = P.pks[0] * (int64_t)sizeof(T);
    w.vst = P.pvs[0] * (int64_t)sizeof(T);
    w.lo_max = 0;
    w.hi_min = P.N;
    return w.k0 < w.k1;
  }
  const int item = xcd_tile(bid - P.prefix_launch, P.own_launch);
  if (item >= P.n_own) return false;
  const int c = (int)fdiv((uint32_t)item, P.frt_o), rt = item - c * P.rt_o;
  const int bg = (int)fdiv((uint32_t)c, P.fSO), cc = c - bg * P.SO;
  w.b = (int)fdiv((uint32_t)bg, P.fHkv);
  w.g = bg - w.b * P.Hkv;
  w.slot = P.SP + cc;
  w.len = pfx_len(P, w.b);
  w.row0 = w.b * P.Mo + rt * P.rows_o;
  w.row1 = min(w.row0 + P.rows_o, (w.b + 1) * P.Mo);
  const int j0 = (int)fdiv((uint32_t)(w.row0 - w.b * P.Mo), P.frep);
  const int j1 = (int)fdiv((uint32_t)(w.row1 - 1 - w.b * P.Mo), P.frep);
  const PfxSpan first = pfx_span(P, w.len, j0), last = pfx_span(P, w.len, j1);
  const int lo = pfx_span(P, w.len, 0).lo;  // the sample's chunks start here
  w.k0 = max(lo + cc * P.chunk_o, first.lo);
  w.k1 = min(lo + (cc + 1) * P.chunk_o, last.hi);
  w.k = reinterpret_cast<const char *>(static_cast<const T *>(A.k) + w.b * P.ks[0] + w.g * P.ks[2]);
  w.v = reinterpret_cast<const char *>(static_cast<const T *>(A.v) + w.b * P.vs[0] + w.g * P.vs[2]);
  w.kst = P.ks[1] * (int64_t)sizeof(T);
  w.vst = P.vs[1] * (int64_t)sizeof(T);
  w.lo_max = last.lo;
  w.hi_min = min(first.hi, w.k1);
  return w.k0 < w.k1;
}

// A row of a workgroup's tile: its queries, and the keys of [k0, k1) it sees.
template <typename T>
struct PfxRow {
  const T *q;
  int lo, n;  // [lo, lo + n)
  __device__ __forceinline__ PfxRow(const PfxProb &P, const PfxArgs &A, const PfxItem &w, int row) {
    const int r = min(row, w.row1 - 1);
    const int tt = (int)fdiv((uint32_t)r, P.frep), i = r - tt * P.rep;
    const int b = (int)fdiv((uint32_t)tt, P.fLq), j = tt - b * P.Lq;
    q = static_cast<const T *>(A.q) + b * P.qs[0] + j * P.qs[1] + (int64_t)(w.g * P.rep + i) * P.qs[2];
    lo = w.k0;
    int hi = w.k1;
    if (w.b >= 0) {
      const PfxSpan s = pfx_span(P, w.len, j);
      lo = max(lo, s.lo);
      hi = min(hi, s.hi);
    }
    n = max(hi - lo, 0);
  }
};

// Row's element offset in out (its D channels) and index in lse.
__device__ __forceinline__ int64_t pfx_out_row(const PfxProb &P, int g, int row) {
  const int tt = (int)fdiv((uint32_t)row, P.frep);
  return (int64_t)tt * P.H + g * P.rep + (row - tt * P.rep);
}

template <typename T>
struct PfxStore;  // four results of a row, rounded
template <>
struct PfxStore<float> {
  static __device__ __forceinline__ void put(float *p, f32x4 x) { *reinterpret_cast<f32x4 *>(p) = x; }
};
template <typename T>
struct PfxStore16 {
  static __device__ __forceinline__ void put(T *p, f32x4 x) {
    typename L16<T>::v4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = (typename L16<T>::e)x[r];
    *reinterpret_cast<typename L16<T>::v4 *>(p) = o;
  }
};
template <>
struct PfxStore<bf16_t> : PfxStore16<bf16_t> {};
template <>
struct PfxStore<f16_t> : PfxStore16<f16_t> {};

// A row's slot: four channels from c, or the row's (m, l).
template <typename T>
__device__ __forceinline__ void pfx_put(const PfxProb &P, const PfxArgs &A, const PfxItem &w, int row,
                                        int c, f32x4 o, float l) {
  if (c >= P.D) return;
  if (A.po != nullptr) {
    const int64_t r = ((int64_t)w.g * P.M + row) * P.NS + w.slot;
    *reinterpret_cast<f32x4 *>(A.po + r * P.D + c) = o;
  } else {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    PfxStore<T>::put(static_cast<T *>(A.out) + pfx_out_row(P, w.g, row) * P.D + c, o * inv);
  }
}
__device__ __forceinline__ void pfx_put_ml(const PfxProb &P, const PfxArgs &A, const PfxItem &w,
                                           int row, float m, float l) {
  if (A.po != nullptr)
    A.pml[((int64_t)w.g * P.M + row) * P.NS + w.slot] = make_float2(m, l);
  else if (A.lse != nullptr)
    A.lse[pfx_out_row(P, w.g, row)] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// Any alignment of the elements.
template <typename T>
__device__ __forceinline__ typename L16<T>::v8 pfx_ld8(const char *p) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));
  typedef uint32_t r4 __attribute__((ext_vector_type(4)));
  const r4 x = *reinterpret_cast<const u4 *>(p);
  return __builtin_bit_cast(typename L16<T>::v8, x);
}
template <typename T>
__device__ __forceinline__ typename L16<T>::v8 pfx_zero8() {
  typename L16<T>::v8 z;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = (typename L16<T>::e)0.f;
  return z;
}

// How far below a row's largest score its reference point m is put: a power of two
// in every probability, which the division by l takes out.  In fp16, whose smallest
// step is 2^-24, probabilities of an m at the maximum vanish below 2^-25 of the
// largest, while l keeps them; from 2^7 up (with the factor 2^8 by which m may
// trail, below 2^15) the products lose 2^-32 of the largest at most.
template <typename T>
__host__ __device__ constexpr float pfx_lead() {
  return std::is_same<T, f16_t>::value ? 7.f : 0.f;
}

// Online softmax step of a lane's CH * 4 scores of one row (the four lanes of a
// row hold the others): scores to probabilities in place, m, l and o rescaled
// where the reference point m moves.  It may trail the maximum by 8 (a factor
// 2^8 in p) beside its lead: exact after the division by l.
template <typename T, int CH, int NDB>
__device__ __forceinline__ void pfx_softmax(float (&p)[CH][4], float sl2, float &m, float &l,
                                            f32x4 (&o)[NDB]) {
  float mx = -INFINITY;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, p[ch][r]);
  mx = quad_max(mx) * sl2;
  if (__builtin_amdgcn_ballot_w64(mx > m + (8.f + pfx_lead<T>())) != 0) {
    const float mn = fmaxf(m, mx - pfx_lead<T>());
    const float alpha = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.f : mn));
    l *= alpha;
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] *= alpha;
    m = mn;
  }
  const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      p[ch][r] = __builtin_amdgcn_exp2f(fmaf(p[ch][r], sl2, -mu));
      l += p[ch][r];
    }
}

// Whether 16-bit element x is an infinity or NaN.
template <typename T>
__device__ __forceinline__ bool pfx_odd16(uint32_t x) {
  const uint32_t e = sizeof(T) == 2 && std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
  return (x & e) == e;
}

// V rows [0, rows) of a tile in LDS hold an infinity or NaN (all lanes look).
template <typename T, int D>
__device__ __forceinline__ bool pfx_odd_tile(const typename L16<T>::e *vs, int stride, int rows,
                                             int lane) {
  bool odd = false;
  for (int u = lane; u < rows * (D / 8); u += 64) {
    const uint4 x = *reinterpret_cast<const uint4 *>(vs + u / (D / 8) * stride + u % (D / 8) * 8);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= pfx_odd16<T>(w[i]) | pfx_odd16<T>(w[i] >> 16);
  }
  return __builtin_amdgcn_ballot_w64(odd) != 0;
}

// o += P V key by key, only over the keys that the lane's row sees: for tiles
// where rows see different keys and V is not finite everywhere, where a product
// with a probability of zero would not be zero.
template <typename T, int CH, int NDB>
__device__ __forceinline__ void pfx_odd_pv(const float (&p)[CH][4],
                                                     const typename L16<T>::e *vs, int stride,
                                                     int lane, int lo, int n, f32x4 (&o)[NDB]) {
  const int row = lane & 15, gq = lane >> 4;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll 1
      for (int g2 = 0; g2 < 4; ++g2) {
        const int key = 16 * ch + 4 * g2 + r;
        const float pk = __shfl(p[ch][r], row + 16 * g2, 64);
        if ((unsigned)(key - lo) >= (unsigned)n) continue;
        const typename L16<T>::e *v = vs + key * stride + 4 * gq;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[db][c] = fmaf(pk, (float)v[16 * db + c], o[db][c]);
      }
}

template <int D>
constexpr int pfx_tile() {
  return D > 128 ? 32 : 64;  // keys of a wide tile
}

template <typename T, int D, int NQ, int NW>
__device__ __forceinline__ void pfx_wide(const PfxProb &P, const PfxArgs &A, const PfxItem &w,
                                         char *smem) {
  typedef L16<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v4 v4;
  typedef typename M::e E;
  constexpr int TK = pfx_tile<D>(), CH = TK / 16;
  constexpr int NT = D / 32, NDB = D / 16, RSE = lds_row(D);
  constexpr int UPR = D / 4, RPP = 64 * NW / UPR, NU = TK / RPP;
  E *const buf = reinterpret_cast<E *>(smem);
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
  const int n = lane & 15, gq = lane >> 4;

  // staging: the thread's column unit c and rows r0 + RPP i
  const int c = tid % UPR, r0 = tid / UPR;
  const bool isv = c >= D / 8;
  const int col = 8 * (isv ? c - D / 8 : c);
  const bool colok = col < P.D;
  const int64_t st = isv ? w.vst : w.kst;
  const char *const src = (isv ? w.v : w.k) + 2 * col + (int64_t)(w.k0 + r0) * st;
  const int unit = r0 * RSE + 8 * c + (isv ? 8 : 0);
  v8 pre[NU];
  const int total = w.k1 - w.k0, nkt = (total + TK - 1) / TK;
  // The tiles that every row sees in full are [ja, jb); they come first, then
  // those behind them, then those before.
  int ja = (max(w.lo_max - w.k0, 0) + TK - 1) / TK, jb = max(min(w.hi_min, w.k1) - w.k0, 0) / TK;
  if (jb <= ja) ja = jb = 0;
  auto first_key = [&](int i) {  // of the i-th tile, behind k0
    const int j = ja + i;
    return (j < nkt ? j : j - nkt) * TK;
  };
  // V of the i-th tile and K of the next: the scores run one tile ahead.
  auto fetch = [&](int i) {
    const int mine = isv ? i : i + 1;
    const int t = first_key(max(min(mine, nkt - 1), 0));
    const char *p = src + (int64_t)t * st;
    // (eight waves have registers left to hold the zeros of channels past D)
    if (i >= 0 && i + 1 < nkt && max(first_key(i), first_key(i + 1)) + TK <= total &&
        (NW > 4 || P.D == D)) {
      if (NW == 4 || colok) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          pre[u] = pfx_ld8<T>(p);
          p += RPP * st;
        }
      }
    } else {  // zeros behind the last key and channel: 0 times them is 0
      const int left = mine >= 0 && mine < nkt && colok ? total - t - r0 : 0;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        pre[u] = pfx_zero8<T>();
        if (RPP * u < left) pre[u] = pfx_ld8<T>(p);
        p += RPP * st;
      }
    }
  };
  auto put = [&](int i) {
    E *const d = buf + ((isv ? i : i + 1) & 1) * (TK * RSE) + unit;
#pragma unroll
    for (int u = 0; u < NU; ++u) *reinterpret_cast<v8 *>(d + RPP * u * RSE) = pre[u];
  };
  fetch(-1);

  const int row0 = w.row0 + wv * (16 * NQ);
  v8 qf[NQ][NT];
  int lo[NQ], cnt[NQ];  // keys that a row sees
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const PfxRow<T> r(P, A, w, row0 + 16 * qi + n);
    lo[qi] = r.lo - w.k0;
    cnt[qi] = r.n;
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      const int cq = 32 * s + 8 * gq;
      qf[qi][s] = cq < P.D ? pfx_ld8<T>(reinterpret_cast<const char *>(r.q + cq)) : pfx_zero8<T>();
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
  const bool spans = w.b >= 0 && P.Lq > 1;  // rows may see different keys

  auto values = [&](const E *vs, int jj, int db) {  // V^T of 32 keys
    const E *ca = vs + 32 * jj * RSE + tr_off + 16 * db;
    const v4 lo4 = M::tr(ca), hi4 = M::tr(ca + 16 * RSE);
    return (v8)__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  typedef f32x4 Scores[NQ][CH];
  Scores sa, sb;  // of the tile at hand and of the next
  float mx[NQ];   // the lane's largest score of the tile at hand
  auto keys = [&](const E *ks, int ch, v8 (&ka)[NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      ka[t] = *reinterpret_cast<const v8 *>(ks + 16 * ch * RSE + 32 * t);
  };
  auto largest = [&](const Scores &s, int qi, int ch) {
#pragma unroll
    for (int r = 0; r < 4; ++r) mx[qi] = fmaxf(mx[qi], s[qi][ch][r]);
  };
  // The i-th tile, its scores in `s`; the next tile's go to `next`.  EDGE: some
  // row does not see some of its keys.  Matrix products are issued two at a time
  // between the vector ALU's work, which fills the matrix unit's time: the next
  // tile's scores beside the first half of the exponentials, O beside the second.
  auto run_tile = [&](int i, Scores &s, Scores &next, auto edge_tile) {
    constexpr bool EDGE = decltype(edge_tile)::value;
    const E *vs = buf + (i & 1) * (TK * RSE) + lds_y(D);
    const E *ks = buf + ((i + 1) & 1) * (TK * RSE) + ka_off;
    fetch(i + 1);  // in flight during this tile
    const int t0 = first_key(i);
    bool moves = false;
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      if (EDGE) {
        mx[qi] = -INFINITY;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((unsigned)(t0 + 16 * ch + 4 * gq + r - lo[qi]) >= (unsigned)cnt[qi])
              s[qi][ch][r] = -INFINITY;
          largest(s, qi, ch);
        }
      }
      moves |= mx[qi] * sl2 > m[qi] + (8.f + pfx_lead<T>());
    }
    // the reference point may trail the maximum by 8 (a factor 2^8 in p) beside its
    // lead: exact after the division by l
    if (__builtin_amdgcn_ballot_w64(moves) != 0) {
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        const float mn = fmaxf(m[qi], quad_max(mx[qi]) * sl2 - pfx_lead<T>());
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
    auto rounded = [&](int qi, int jj) {
      v8 bp;
#pragma unroll
      for (int x = 0; x < 8; ++x) bp[x] = (E)s[qi][2 * jj + x / 4][x % 4];
      return bp;
    };
    constexpr int ALL = CH * 4, FIRST = CH > 2 ? ALL / 2 : ALL;  // a lane's scores, beside QK
    constexpr int QS = CH * NT, OS = CH / 2 * NDB;  // steps of the two products
    constexpr int RING = 4;
    v8 ka[RING];  // of the next steps
    auto key = [&](int st) {
      return *reinterpret_cast<const v8 *>(ks + 16 * (st / NT) * RSE + 32 * (st % NT));
    };
#pragma unroll
    for (int st = 0; st < RING - 1; ++st) ka[st] = key(st);
#pragma unroll
    for (int st = 0; st < QS; ++st) {
      const int ch = st / NT, t = st % NT;
      if (st + RING - 1 < QS) ka[(st + RING - 1) % RING] = key(st + RING - 1);
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        next[qi][ch] = M::mma(ka[st % RING], qf[qi][t], t == 0 ? zero4() : next[qi][ch]);
#pragma unroll
        for (int x = st * FIRST / QS; x < (st + 1) * FIRST / QS; ++x) expo(qi, x);
      }
      __builtin_amdgcn_sched_barrier(0x124);
    }
    bool odd = false;
    if (EDGE) odd = spans && pfx_odd_tile<T, D>(vs, RSE, TK, lane);
    if (EDGE && odd) {
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        float p[CH][4];
#pragma unroll
        for (int x = FIRST; x < ALL; ++x) expo(qi, x);
#pragma unroll
        for (int x = 0; x < ALL; ++x) p[x / 4][x % 4] = s[qi][x / 4][x % 4];
        pfx_odd_pv<T, CH, NDB>(p, vs, RSE, lane, lo[qi] - t0, cnt[qi], o[qi]);
      }
    } else {
      v8 bp[NQ];
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) bp[qi] = rounded(qi, 0);
      v8 va[2];
      va[0] = values(vs, 0, 0);
#pragma unroll
      for (int st = 0; st < OS; ++st) {
        const int jj = st / NDB, db = st % NDB;
        if (jj > 0 && db == 0) {
#pragma unroll
          for (int qi = 0; qi < NQ; ++qi) bp[qi] = rounded(qi, jj);
        }
        if (st + 1 < OS) va[(st + 1) & 1] = values(vs, (st + 1) / NDB, (st + 1) % NDB);
#pragma unroll
        for (int qi = 0; qi < NQ; ++qi) {
          o[qi][db] = M::mma(va[st & 1], bp[qi], o[qi][db]);
          if (jj == 0) {
#pragma unroll
            for (int x = FIRST + db * (ALL - FIRST) / NDB; x < FIRST + (db + 1) * (ALL - FIRST) / NDB; ++x)
              expo(qi, x);
          }
        }
        __builtin_amdgcn_sched_barrier(0x124);
      }
    }
    put(i + 1);
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      mx[qi] = -INFINITY;
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) largest(next, qi, ch);
    }
    __syncthreads();
  };
  put(-1);
  __syncthreads();
  fetch(0);
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) mx[qi] = -INFINITY;
#pragma unroll
  for (int ch = 0; ch < CH; ++ch) {
    v8 ka[NT];
    keys(buf + ka_off, ch, ka);
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) {
      sa[qi][ch] = zero4();
#pragma unroll
      for (int t = 0; t < NT; ++t) sa[qi][ch] = M::mma(ka[t], qf[qi][t], sa[qi][ch]);
      largest(sa, qi, ch);
    }
  }
  put(0);
  __syncthreads();
  auto follow = [&]() {
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi)
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) sa[qi][ch] = sb[qi][ch];
  };
  int i = 0;
  for (; i + 2 <= jb - ja; i += 2) {
    run_tile(i, sa, sb, std::false_type{});
    run_tile(i + 1, sb, sa, std::false_type{});
  }
  for (; i < nkt; ++i) {
    run_tile(i, sa, sb, std::true_type{});
    follow();
  }
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const float lt = quad_sum(l[qi]);
    const int row = row0 + 16 * qi + n;
    if (row >= w.row1) continue;
#pragma unroll
    for (int db = 0; db < NDB; ++db) pfx_put<T>(P, A, w, row, 16 * db + 4 * gq, o[qi][db], lt);
    if (gq == 0) pfx_put_ml(P, A, w, row, m[qi], lt);
  }
}

// The waves' results of up to 16 rows meet in LDS.  o: channel chan(db) ..
// + 3 of row lane & 15.
template <typename T, int D, int NW, int NDB, typename C>
__device__ __forceinline__ void pfx_meet(const PfxProb &P, const PfxArgs &A, const PfxItem &w,
                                         char *smem, float m, float l, const f32x4 (&o)[NDB], C chan) {
  constexpr int RS = D + 4;  // floats per row
  float *const po = reinterpret_cast<float *>(smem);
  float2 *const ml = reinterpret_cast<float2 *>(po + NW * 16 * RS);  // [NW][16]
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63, n = lane & 15;
  l = quad_sum(l);
  __syncthreads();  // the tiles' LDS is free
#pragma unroll
  for (int db = 0; db < NDB; ++db)
    *reinterpret_cast<f32x4 *>(po + (wv * 16 + n) * RS + chan(db)) = o[db];
  if (lane < 16) ml[wv * 16 + n] = make_float2(m, l);
  __syncthreads();
  constexpr int TPR = 4 * NW;  // threads per row
  const int r = tid / TPR, row = w.row0 + r;
  if (row >= w.row1) return;
  float2 x[NW];
  float mt = -INFINITY, lt = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    x[i] = ml[i * 16 + r];
    mt = fmaxf(mt, x[i].x);
  }
  float wt[NW];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    wt[i] = x[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x[i].x - mt);  // (NaN: a seen row)
    lt = x[i].y == 0.f ? lt : fmaf(wt[i], x[i].y, lt);
  }
  for (int c = 4 * (tid % TPR); c < D; c += 4 * TPR) {
    f32x4 s = zero4();
#pragma unroll
    for (int i = 0; i < NW; ++i)
      if (x[i].y != 0.f) s += wt[i] * *reinterpret_cast<const f32x4 *>(po + (i * 16 + r) * RS + c);
    pfx_put<T>(P, A, w, row, c, s, lt);
  }
  if (tid % TPR == 0) pfx_put_ml(P, A, w, row, mt, lt);
}

template <typename T, int D, int NW>
__device__ __forceinline__ void pfx_narrow(const PfxProb &P, const PfxArgs &A, const PfxItem &w,
                                           char *smem) {
  typedef L16<T> M;
  typedef typename M::v8 v8;
  typedef typename M::v4 v4;
  typedef typename M::e E;
  constexpr int TK = kPfxNarrowKeys, NT = D / 32, NDB = D / 16, RS = D + 8;
  constexpr int UPR = D / 8, RPP = 64 / UPR, NU = TK / RPP;  // V: units per row, rows per pass
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
  const int n = lane & 15, gq = lane >> 4;
  E *const vs = reinterpret_cast<E *>(smem) + wv * (TK * RS);  // the wave's own
  const PfxRow<T> row(P, A, w, w.row0 + n);
  const int lo = row.lo - w.k0, cnt = row.n;
  v8 qf[NT];
#pragma unroll
  for (int s = 0; s < NT; ++s) {
    const int cq = 32 * s + 8 * gq;
    qf[s] = cq < P.D ? pfx_ld8<T>(reinterpret_cast<const char *>(row.q + cq)) : pfx_zero8<T>();
  }
  const int vc = lane % UPR, vr = lane / UPR;
  const int total = w.k1 - w.k0;
  const char *const kp = w.k + (int64_t)(w.k0 + n) * w.kst + 16 * gq;
  const char *const vp = w.v + (int64_t)(w.k0 + vr) * w.vst + 16 * vc;
  v8 kr[2][NT], vr8[NU];
  auto load = [&](int t0) {
    const char *a = kp + (int64_t)t0 * w.kst, *b = vp + (int64_t)t0 * w.vst;
    if (t0 + TK <= total && P.D == D) {
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int s = 0; s < NT; ++s) kr[hh][s] = pfx_ld8<T>(a + 16 * hh * w.kst + 64 * s);
#pragma unroll
      for (int i = 0; i < NU; ++i) vr8[i] = pfx_ld8<T>(b + RPP * i * w.vst);
    } else {  // zeros behind the last key and channel: 0 times them is 0
      const int left = total - t0;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int s = 0; s < NT; ++s) {
          kr[hh][s] = pfx_zero8<T>();
          if (16 * hh + n < left && 32 * s + 8 * gq < P.D)
            kr[hh][s] = pfx_ld8<T>(a + 16 * hh * w.kst + 64 * s);
        }
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        vr8[i] = pfx_zero8<T>();
        if (RPP * i + vr < left && 8 * vc < P.D) vr8[i] = pfx_ld8<T>(b + RPP * i * w.vst);
      }
    }
  };
  f32x4 o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = zero4();
  float m = -INFINITY, l = 0.f;
  const float sl2 = P.sl2;
  const int tr_off = (4 * gq + (n >> 2)) * RS + 4 * (n & 3);
  const bool spans = w.b >= 0 && P.Lq > 1;
  const int all0 = w.lo_max - w.k0, all1 = min(w.hi_min, w.k1) - w.k0;  // seen by every row
  auto run_tile = [&](int t0, auto edge_tile) {
    constexpr bool EDGE = decltype(edge_tile)::value;
    f32x4 s[2] = {zero4(), zero4()};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) s[hh] = M::mma(kr[hh][t], qf[t], s[hh]);
    __builtin_amdgcn_wave_barrier();  // the reads of the tile before are issued
#pragma unroll
    for (int i = 0; i < NU; ++i)
      *reinterpret_cast<v8 *>(vs + (RPP * i + vr) * RS + 8 * vc) = vr8[i];
    if (t0 + NW * TK < total) load(t0 + NW * TK);  // in flight during the rest
    float p[2][4];
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[hh][r] = s[hh][r];
        if (EDGE && (unsigned)(t0 + 16 * hh + 4 * gq + r - lo) >= (unsigned)cnt) p[hh][r] = -INFINITY;
      }
    pfx_softmax<T, 2, NDB>(p, sl2, m, l, o);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (EDGE && spans && pfx_odd_tile<T, D>(vs, RS, TK, lane)) {
      pfx_odd_pv<T, 2, NDB>(p, vs, RS, lane, lo - t0, cnt, o);
    } else {
      v8 bp;
#pragma unroll
      for (int hh = 0; hh < 2; ++hh)
#pragma unroll
        for (int r = 0; r < 4; ++r) bp[4 * hh + r] = (E)p[hh][r];
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const v4 lo4 = M::tr(vs + tr_off + 16 * db);
        const v4 hi4 = M::tr(vs + 16 * RS + tr_off + 16 * db);
        o[db] = M::mma(__builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7), bp, o[db]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  };
  int t0 = wv * TK;
  if (t0 < total) load(t0);
  for (; t0 < total; t0 += NW * TK) {
    if (t0 >= all0 && t0 + TK <= all1) run_tile(t0, std::false_type{});
    else run_tile(t0, std::true_type{});
  }
  pfx_meet<T, D, NW, NDB>(P, A, w, smem, m, l, o, [&](int db) { return 16 * db + 4 * gq; });
}

// NW waves; a segment's rows per tile say how its workgroups are shaped.
template <typename T, int D, int NW>
__global__ void __launch_bounds__(64 * NW, D > 128 ? 1 : 2) k_pfx(PfxProb P, PfxArgs A) {
  extern __shared__ __align__(16) char smem[];
  PfxItem w;
  if (!pfx_item<T>(P, A, blockIdx.x, w)) return;
  const int rows = w.b < 0 ? P.rows_p : P.rows_o;
  if (rows == 16) {
    pfx_narrow<T, D, NW>(P, A, w, smem);
  } else if (rows == 16 * NW) {
    pfx_wide<T, D, 1, NW>(P, A, w, smem);
  } else {
    if constexpr (D <= 128) pfx_wide<T, D, 2, NW>(P, A, w, smem);
  }
}

// float32: 16 rows per workgroup, tiles of 16 keys per wave on 16x16x4 products.
// Contraction slots are dealt so that every operand is a 16-byte load: a lane's
// four channels 16 s + 4 gq .. of K feed four products, and its four channels
// 64 u + 4 n .. of a V row four blocks of O^T, whose row i is then channel
// 64 u + 4 i + e.
template <int D>
__global__ void __launch_bounds__(256) k_pfx32(PfxProb P, PfxArgs A) {
  constexpr int TK = 16, NS = D / 16, NU = D / 64;
  typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
  extern __shared__ __align__(16) char smem[];
  PfxItem w;
  if (!pfx_item<float>(P, A, blockIdx.x, w)) return;
  const int tid = threadIdx.x, wv = tid >> 6, lane = tid & 63;
  const int n = lane & 15, gq = lane >> 4;
  const PfxRow<float> row(P, A, w, w.row0 + n);
  const int lo = row.lo - w.k0, cnt = row.n;
  auto ld = [&](const char *p, bool ok) {
    f32x4 x = zero4();
    if (ok) x = *reinterpret_cast<const f4u *>(p);
    return x;
  };
  f32x4 qf[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s)
    qf[s] = ld(reinterpret_cast<const char *>(row.q + 16 * s + 4 * gq), 16 * s + 4 * gq < P.D);
  const int total = w.k1 - w.k0;
  const char *const kp = w.k + (int64_t)(w.k0 + n) * w.kst + 16 * gq;
  const char *const vp = w.v + (int64_t)(w.k0 + 4 * gq) * w.vst + 16 * n;
  f32x4 o[4 * NU];
#pragma unroll
  for (int i = 0; i < 4 * NU; ++i) o[i] = zero4();
  float m = -INFINITY, l = 0.f;
  const bool spans = w.b >= 0 && P.Lq > 1;
  f32x4 kr[NS], vr[4][NU];
  auto load_k = [&](int t0) {
    const char *const a = kp + (int64_t)t0 * w.kst;
    const bool ok = t0 + n < total;
#pragma unroll
    for (int s = 0; s < NS; ++s) kr[s] = ld(a + 64 * s, ok && 16 * s + 4 * gq < P.D);
  };
  auto load_v = [&](int t0) {
    const char *const b = vp + (int64_t)t0 * w.vst;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int u = 0; u < NU; ++u)
        vr[r][u] = ld(b + r * w.vst + 256 * u, t0 + 4 * gq + r < total && 64 * u + 4 * n < P.D);
  };
  load_k(wv * TK);  // (past the last key: zeros)
  load_v(wv * TK);
  for (int t0 = wv * TK; t0 < total; t0 += 4 * TK) {
    f32x4 s4 = zero4();
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s4 = __builtin_amdgcn_mfma_f32_16x16x4f32(kr[s][e], qf[s][e], s4, 0, 0, 0);
    load_k(t0 + 4 * TK);  // in flight during the softmax and the second product
    const bool all = w.k0 + t0 >= w.lo_max && w.k0 + t0 + TK <= min(w.hi_min, w.k1);
    float p[1][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      p[0][r] = all || (unsigned)(t0 + 4 * gq + r - lo) < (unsigned)cnt ? s4[r] : -INFINITY;
    pfx_softmax<float, 1, 4 * NU>(p, P.sl2, m, l, o);
    bool odd = false;
    if (!all && spans) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            odd |= (__float_as_uint(vr[r][u][e]) & 0x7f800000u) == 0x7f800000u;
    }
    if (__builtin_amdgcn_ballot_w64(odd) == 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[4 * u + e] =
                __builtin_amdgcn_mfma_f32_16x16x4f32(vr[r][u][e], p[0][r], o[4 * u + e], 0, 0, 0);
    } else {  // as pfx_odd_pv: V's elements come from the lanes that hold them
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll 1
        for (int g2 = 0; g2 < 4; ++g2) {
          const float pk = __shfl(p[0][r], n + 16 * g2, 64);
          const bool sees = (unsigned)(t0 + 4 * g2 + r - lo) < (unsigned)cnt;
#pragma unroll
          for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = __shfl(vr[r][u][e], 4 * gq + i + 16 * g2, 64);
                if (sees) o[4 * u + e][i] = fmaf(pk, v, o[4 * u + e][i]);
              }
        }
    }
    load_v(t0 + 4 * TK);
  }
  // block e of group u, element i: channel 64 u + 4 (4 gq + i) + e; dealt to
  // blocks of four adjacent channels
  f32x4 q4[4 * NU];
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) q4[4 * u + i][e] = o[4 * u + e][i];
  pfx_meet<float, D, 4, 4 * NU>(P, A, w, smem, m, l, q4,
                             [&](int x) { return 64 * (x >> 2) + 16 * gq + 4 * (x & 3); });
}

// The slots of a row added: lanes take four channels each, 2^lgG of them a row,
// and 2^lgS such groups share the row's slots.
template <typename T>
__global__ void __launch_bounds__(256) k_pfx_join(PfxProb P, PfxArgs A, int lgG, int lgS) {
  __shared__ f32x4 so[256];
  __shared__ float2 sml[256];
  const int tid = threadIdx.x, lane = tid & ((1 << lgG) - 1);
  const int group = tid >> lgG, share = group & ((1 << lgS) - 1);
  const int64_t rows = (int64_t)P.Hkv * P.M;
  const int64_t mine = ((int64_t)blockIdx.x * 256 + tid) >> (lgG + lgS);
  const int64_t r = min(mine, rows - 1);
  const int g = (int)(r / P.M), row = (int)(r - (int64_t)g * P.M);
  // the slots that were written: the prefix's, and the own chunks the row sees
  const int tt = (int)fdiv((uint32_t)row, P.frep);
  const int b = (int)fdiv((uint32_t)tt, P.fLq), j = tt - b * P.Lq;
  int c0 = 0, c1 = 0;
  if (P.SO > 0) {
    const int len = pfx_len(P, b), base = pfx_span(P, len, 0).lo;
    const PfxSpan s = pfx_span(P, len, j);
    if (s.hi > s.lo) {
      c0 = (s.lo - base) / P.chunk_o;
      c1 = (s.hi - 1 - base) / P.chunk_o + 1;
    }
  }
  const int count = P.SP + c1 - c0;
  auto slot = [&](int i) { return i < P.SP ? i : i + c0; };
  const float2 *const ml = A.pml + r * P.NS;
  const float *const po = A.po + r * P.NS * P.D;
  float m = -INFINITY, l = 0.f;
  f32x4 acc = zero4();
  const int c = 4 * lane;
  for (int i0 = share; i0 < count; i0 += kPfxJoin << lgS) {  // a batch's loads together
    float2 x[kPfxJoin];
    f32x4 o[kPfxJoin];
#pragma unroll
    for (int u = 0; u < kPfxJoin; ++u) {
      const int i = i0 + (u << lgS);
      x[u] = make_float2(-INFINITY, 0.f);
      o[u] = zero4();
      if (i < count) {
        x[u] = ml[slot(i)];
        if (c < P.D) o[u] = *reinterpret_cast<const f32x4 *>(po + (int64_t)slot(i) * P.D + c);
      }
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < kPfxJoin; ++u) mn = fmaxf(mn, x[u].x);
    if (l != 0.f) {
      const float wt = __builtin_amdgcn_exp2f(m - mn);
      l *= wt;
      acc *= wt;
    }
    m = mn;
#pragma unroll
    for (int u = 0; u < kPfxJoin; ++u)
      if (x[u].y != 0.f) {  // (0: a row that sees nothing of the chunk)
        const float wt = __builtin_amdgcn_exp2f(x[u].x - m);
        l = fmaf(wt, x[u].y, l);
        acc += wt * o[u];
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
  if (mine >= rows) return;
  const int64_t out = pfx_out_row(P, g, row);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (c < P.D) PfxStore<T>::put(static_cast<T *>(A.out) + out * P.D + c, acc * inv);
  if (lane == 0 && A.lse != nullptr) A.lse[out] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

int pfx_width(int dtype, int D) {  // the kernels' head dim
  if (dtype == NA_F32) return D <= 64 ? 64 : D <= 128 ? 128 : 256;
  return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256;
}

// Waves of the call's workgroups.  Eight where the batch's rows fill more than
// half of 256 against a prefix that is most of the keys' work: every K / V tile is
// then staged once for 256 rows, half the loads of four waves with 128 (256 rows
// of 128 channels, 8 heads, 65536 prefix keys: 119 -> 100 us; of 80 channels: 94 ->
// 77).  Where the samples' own keys are most of it, or a head fits 64 channels,
// four are as good or better (80 channels, 16384 prefix keys and 64 samples of up
// to 1024: 50.8 and 55.8 us; 64 channels, 65536 and up to 2048: 86 and 96).
int pfx_waves(const na_prefix_params *p, int64_t span) {
  const int64_t rows = (int64_t)p->batch * p->tokens * (p->heads / p->kv_heads);
  return p->dtype != NA_F32 && p->head_dim > 64 && p->head_dim <= 128 && rows > 128 &&
                 (rows + 255) / 256 * p->prefix >= p->batch * span / 2 ? 8 : 4;
}

// Rows of a tile: 16 narrow, above that 16 or, where there are more, 32 per wave.
// A sample's own rows are narrow up to two tiles, which read its keys one behind
// the other through an L2 (64 samples of 32 heads over one key/value head of 128
// channels: 49.6 us, 62.0 wide; 32 samples of 5 tokens, 8 groups of 64 channels and
// up to 4096 tokens: 54.7 and 61.7), but not in heads of 256 (152 us, 117 wide); a
// prefix is read once by wide tiles (32 rows, 65536 keys: 35.7 us, 40.7 narrow).
int pfx_rows(int dtype, int D, int64_t rows, int waves, int narrow) {
  if (dtype == NA_F32 || rows <= narrow) return 16;
  return rows <= 16 * waves || D > 128 ? 16 * waves : 32 * waves;
}

// Keys per chunk.  kPfxItems workgroups are on the chip at once (two on a CU): a
// chunk is a workgroup's part of all keys and row tiles, the samples' lengths
// taken as half their capacity.  Wide chunks are at least 512 keys (each leaves
// rows * D floats for the join; 8 heads x 16384 keys x 128 rows of 128 channels:
// 33.3 us in chunks of 256, 29.4 of 512, 32.7 of 768); a sample's are at most
// 1024, which evens out ragged lengths (64 samples of up to 2048, 8 heads: 56.6
// us, 69.2 in chunks of 2048) -- or an eighth of a workgroup's part, where there are
// that many rounds of them anyway and slots would fill the memory (8192 tokens of 32
// heads over 65536 own: 7.9 ms and 0.7 GB, 11.7 ms and 8.9 GB in chunks of 1024).
PfxProb pfx_prob(const na_prefix_params *p) {
  PfxProb P{};
  P.Lq = p->tokens;
  P.H = p->heads;
  P.Hkv = p->kv_heads;
  P.rep = p->heads / p->kv_heads;
  P.D = p->head_dim;
  P.Mo = P.Lq * P.rep;
  P.M = (int32_t)(p->batch * P.Mo);
  P.N = p->prefix;
  P.S = p->capacity;
  // No cache is longer than 2^30: a wider window is none, and a token's place less
  // the window (at least -2^30 - 2^30) stays in 32 bits.
  P.W = p->window > 0 ? std::min(p->window, 1 << 30) : 1 << 30;
  const int64_t span = std::min<int64_t>(P.S, (int64_t)P.W + P.Lq - 1);
  P.waves = pfx_waves(p, span);
  P.rows_p = pfx_rows(p->dtype, P.D, P.M, P.waves, 16);
  P.rows_o = pfx_rows(p->dtype, P.D, P.Mo, P.waves, P.D > 128 ? 16 : 32);
  P.rt_p = (P.M + P.rows_p - 1) / P.rows_p;
  P.rt_o = (P.Mo + P.rows_o - 1) / P.rows_o;
  const int64_t tp = (int64_t)P.Hkv * P.rt_p, to = (int64_t)p->batch * P.Hkv * P.rt_o;
  const int64_t want = (tp * P.N + to * span / 2) / (4 * kPfxItems / P.waves);
  auto chunk = [](int64_t keys, int64_t size) {  // even parts, whole tiles
    const int64_t parts = (keys + size - 1) / size;
    return (int32_t)(((keys + parts - 1) / parts + 63) / 64 * 64);
  };
  if (P.N > 0) {
    P.chunk_p = chunk(P.N, std::max<int64_t>(want, P.rows_p > 16 ? 512 : 128));
    P.SP = (P.N + P.chunk_p - 1) / P.chunk_p;
  }
  if (span > 0) {
    const int64_t least = P.rows_o > 16 ? 256 : 128;
    P.chunk_o = chunk(span, std::min(std::max(want, least), std::max<int64_t>(want / 8, 1024)));
    P.SO = (int32_t)((span + P.chunk_o - 1) / P.chunk_o);
  }
  P.NS = P.SP + P.SO;
  P.n_prefix = (int32_t)(tp * P.SP);
  P.n_own = (int32_t)(to * P.SO);
  P.prefix_launch = (P.n_prefix + 7) & ~7;
  P.own_launch = (P.n_own + 7) & ~7;
  P.sl2 = p->scale * kLog2e;
  P.frep = make_fastdiv((uint32_t)P.rep);
  P.fLq = make_fastdiv((uint32_t)P.Lq);
  P.frt_p = make_fastdiv((uint32_t)P.rt_p);
  P.frt_o = make_fastdiv((uint32_t)P.rt_o);
  P.fSP = make_fastdiv((uint32_t)std::max(P.SP, 1));
  P.fSO = make_fastdiv((uint32_t)std::max(P.SO, 1));
  P.fHkv = make_fastdiv((uint32_t)P.Hkv);
  for (int i = 0; i < 3; ++i) {
    P.qs[i] = p->q_stride[i];
    P.ks[i] = p->k_stride[i];
    P.vs[i] = p->v_stride[i];
  }
  for (int i = 0; i < 2; ++i) {
    P.pks[i] = p->prefix_k_stride[i];
    P.pvs[i] = p->prefix_v_stride[i];
  }
  P.lens = p->seq_lens;
  return P;
}

// One slot that every row fills needs no join.
bool pfx_direct(const PfxProb &P) { return P.SP == 1 && P.SO == 0; }

// Logs of the join's lanes per row and of the groups that share a row's slots.
struct PfxJoinLanes {
  int lgG = 0, lgS = 0;
  int total() const { return lgG + lgS; }
};
PfxJoinLanes pfx_join_lanes(const PfxProb &P) {
  PfxJoinLanes n;
  while ((4 << n.lgG) < P.D) ++n.lgG;
  while (n.total() < 8 && (kPfxJoin << n.lgS) < P.NS) ++n.lgS;
  return n;
}

size_t pfx_part_bytes(const PfxProb &P) {
  return ((size_t)P.Hkv * P.M * P.NS * P.D * sizeof(float) + 255) & ~(size_t)255;
}

template <typename T, int D, int NW>
void pfx_launch(const PfxProb &P, const PfxArgs &A, hipStream_t st) {
  auto lds = [&](int rows) -> size_t {
    if (rows > 16) return sizeof(T) * 2 * pfx_tile<D>() * lds_row(D);
    const size_t meet = NW * (sizeof(float) * 16 * (D + 4) + sizeof(float2) * 16);
    const size_t tiles = sizeof(T) == 2 ? sizeof(T) * NW * kPfxNarrowKeys * (D + 8) : 0;
    return std::max(meet, tiles);
  };
  const size_t bytes = std::max(P.SP > 0 ? lds(P.rows_p) : 0, P.SO > 0 ? lds(P.rows_o) : 0);
  const dim3 grid((unsigned)(P.prefix_launch + P.own_launch));
  if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((k_pfx32<D>), grid, dim3(256), bytes, st, P, A);
  else
    hipLaunchKernelGGL((k_pfx<T, D, NW>), grid, dim3(64 * NW), bytes, st, P, A);
}

template <typename T, int D>
void pfx_by_waves(const PfxProb &P, const PfxArgs &A, hipStream_t st) {
  if constexpr (sizeof(T) == 2 && D == 128)
    if (P.waves == 8) return pfx_launch<T, D, 8>(P, A, st);
  pfx_launch<T, D, 4>(P, A, st);
}

template <typename T>
void pfx_run(const PfxProb &P, const PfxArgs &A, hipStream_t st) {
  if (P.NS > 0) {
    const int width = pfx_width(sizeof(T) == 4 ? NA_F32 : NA_BF16, P.D);
    if (width == 256) pfx_by_waves<T, 256>(P, A, st);
    else if (width == 128) pfx_by_waves<T, 128>(P, A, st);
    else if (sizeof(T) == 4 || width == 64) pfx_by_waves<T, 64>(P, A, st);
    else if constexpr (sizeof(T) == 2) pfx_by_waves<T, 32>(P, A, st);
  }
  if (A.po == nullptr && P.NS > 0) return;
  const PfxJoinLanes n = pfx_join_lanes(P);
  const int64_t threads = ((int64_t)P.Hkv * P.M) << n.total();
  hipLaunchKernelGGL((k_pfx_join<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, P, A,
                     n.lgG, n.lgS);
}

}  // namespace

// A launch has fewer than 2^32 threads.
bool prefix_fits(const na_prefix_params *p, size_t *workspace_bytes) {
  const PfxProb P = pfx_prob(p);
  *workspace_bytes = P.NS == 0 || pfx_direct(P)
                         ? 0
                         : pfx_part_bytes(P) + sizeof(float2) * (size_t)P.Hkv * P.M * P.NS;
  const int64_t items =
      (int64_t)P.Hkv * P.rt_p * P.SP + (int64_t)p->batch * P.Hkv * P.rt_o * P.SO + 16;
  const int64_t rows = (int64_t)P.Hkv * P.M, lim = ((int64_t)1 << 32) - 256;
  return items * (64 * P.waves) < lim && rows << pfx_join_lanes(P).total() < lim;
}

void prefix_attention(const na_prefix_params *p, const void *q, const void *pk, const void *pv,
                      const void *k, const void *v, void *out, float *lse, void *workspace,
                      hipStream_t st) {
  const PfxProb P = pfx_prob(p);
  PfxArgs A{q, pk, pv, k, v, out, lse, nullptr, nullptr};
  if (P.NS > 0 && !pfx_direct(P)) {
    A.po = static_cast<float *>(workspace);
    A.pml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + pfx_part_bytes(P));
  }
  if (p->dtype == NA_F32) pfx_run<float>(P, A, st);
  else if (p->dtype == NA_F16) pfx_run<f16_t>(P, A, st);
  else pfx_run<bf16_t>(P, A, st);
}

}  // namespace na
