// na_norm_rotary.hip — layer norm of each head of queries and keys and their rotary
// positions in one pass, forward and backward, with the gradients of the norms'
// weights and biases.
//
//   xh = (x - mean x) rstd, rstd = 1 / sqrt(mean (x - mean x)^2 + eps),
//   y = R (xh w + b), R the rotation of the row's token (na_rotary.hip);
//   g' = R^T g, gw = g' w, dx = rstd (gw - mean gw - xh mean(gw xh)),
//   dw = sum over rows of g' xh, db = sum over rows of g',
// one w and b for the heads of q, one for those of k.
//
// A group of 1 to 64 lanes takes a row, which stays in registers from its load to
// its store: lanes hold the chunks that rotate together (two half an axis apart, or
// one of adjacent pairs), so the rotation needs no other lane; where half an axis
// is no number of chunks, each lane holds one chunk and takes the partners from a
// copy of the wave's rows in LDS, laid out by element and lane, which no two banks
// share.  A workgroup takes a run of tokens and fills the run's table of (cos, sin)
// once for all heads, from float64 angles as na_rotary.hip does.
//
// The backward computes a row's mean and deviation again, which costs two sums over
// registers where kept statistics would cost 8 bytes a row each way.  Its workgroups
// take the rows of q or those of k (one pair of column sums in registers) over runs
// of tokens; each leaves one row of partial sums, added in a fixed order by
// k_nr_wsum, so results do not depend on the run.
//
// Sums are float32; y, dx, dw and db are rounded once.  Bound: memory: 131072 tokens of
// 8 + 8 bf16 heads of 64, forward 537 MB in 124 us, backward 805 MB in 189, both 4.3 TB/s
// where a large copy reaches 4.7; 64 tokens of 32 + 8 heads of 128 take 5.8 us.
#include "na_rotary.h"

// Sums and products are fused where it says so and nowhere else: the kernels of rows
// that lie as one and of others give the same bits.
#pragma clang fp contract(off)

namespace na {
namespace {

// Most workgroups of a backward, four on a CU, and units per thread of a run: 25088
// tokens of 8 + 8 heads of 32 bf16 channels, backward: 27 us, 34 with 2048 workgroups;
// 131072 of 8 + 8 heads of 64, forward: 126, 135 with 8 units and 162 with 4.
constexpr int kNrBlocks = 1024;
constexpr int kNrUnits = 16;
constexpr int kNrTable = 2048;  // entries of a run's table, 16 KB

struct NrProb {
  RotProb R;  // per_block: tokens of a run; backward: of q's, qs / ks the rows of x
  int32_t lgG, wide;      // lanes per row; weights are float32
  int32_t fast;           // no chunk is cut off by a row's end, and a run's rows lie within
                          // 2^31 bytes of its first token's, samples behind each other
  int32_t per_k, bq, bk;  // backward: tokens of a run of k, workgroups of q and of k
  float eps, inv_d;
  FastDiv fH, fHk;
  int64_t gqs[3], gks[3];
};

// The lane's place in a row: first channels and channels left of its chunks.
template <typename T, int MODE>
struct NrLane {
  static constexpr int N = Chunk<T>::N, NT = MODE == kRotHalves ? 2 : 1;
  int c[NT], n[NT];
  int j, c0;  // unit, its first channel (halves: pair)
  bool turn;  // halves: its channels are rotated
  __device__ __forceinline__ NrLane(const RotProb &P, int unit) : j(unit), c0(unit * N) {
    int first = c0, second = P.D;
    turn = false;
    if (MODE == kRotHalves) {
      turn = c0 < P.pairs;
      const int a = rot_axis(P, c0);
      first = turn ? c0 + P.first[a] : 2 * c0;
      second = turn ? first + P.first[a + 1] - P.first[a] : first + N;
    }
    const bool live = j < P.upr;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int at = t == 0 ? first : second;
      n[t] = live ? max(P.D - at, 0) : 0;
      c[t] = n[t] > 0 ? at : 0;
    }
  }
};

// A chunk of which n elements belong to the row.
template <bool FAST, typename T>
__device__ __forceinline__ typename Chunk<T>::raw nr_load(const T *p, int n) {
  if (!FAST) return Chunk<T>::load(p, n);
  typename Chunk<T>::raw r = {0, 0, 0, 0};
  if (n > 0) r = *reinterpret_cast<const typename Chunk<T>::mem *>(p);
  return r;
}
template <bool FAST, typename T>
__device__ __forceinline__ void nr_store(T *p, const float *x, int n) {
  if (n > 0) Chunk<T>::store(p, x, FAST ? Chunk<T>::N : n);
}

// The lane's partners in the wave's copy of its rows: channel c of the row whose
// first lane is `base` lies at (c % N) * 64 + base + c / N.
template <int N>
struct NrPartner {
  int16_t at[N];
  __device__ __forceinline__ NrPartner(const RotProb &P, int c0, int base) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int ch = c0 + e, a = rot_axis(P, ch / 2);
      const int half = P.first[a + 1] - P.first[a];
      int o = ch - 2 * P.first[a] < half ? ch + half : ch - half;
      o = ch < 2 * P.pairs ? o : ch;
      at[e] = (int16_t)(o % N * 64 + base + o / N);
    }
  }
};

// The table of a token: entry (e, j) is what element e of unit j turns by -- its
// pair's (cos, sin), staged with the sign that its place in the pair takes -- so that
// the lanes of a row read next to each other.
template <typename T, int MODE>
struct NrTable {
  static constexpr int N = Chunk<T>::N, E = MODE == kRotAdjacent ? N / 2 : N;
  static __host__ __device__ __forceinline__ int units(const RotProb &P) {
    return MODE == kRotHalves ? P.pairs / N : P.upr;
  }
  static __host__ __device__ __forceinline__ int size(const RotProb &P) { return E * units(P); }
  static __device__ __forceinline__ int at(const RotProb &P, int i) {  // i: pair, or channel
    return i % E * units(P) + i / E;
  }
  // Of tokens t0 .. t0 + nt.  A barrier before they are read.
  static __device__ __forceinline__ void fill(const RotProb &P, const void *pos, const double *rate,
                                              int t0, int nt, float2 *cs) {
    const int n = size(P);
    for (int i = threadIdx.x; i < nt * P.pairs; i += kRotThreads) {
      const uint32_t t = fdiv((uint32_t)i, P.fpairs), p = (uint32_t)i - t * P.fpairs.d;
      const int a = rot_axis(P, (int)p);
      const float2 z = rot_cos_sin(P, pos, rate, (uint32_t)t0 + t, (int)p, a);
      float2 *const c = cs + (int)t * n;
      if (MODE == kRotStaged) {
        const int ch = (int)p + P.first[a];
        c[at(P, ch)] = make_float2(z.x, -z.y);
        c[at(P, ch + P.first[a + 1] - P.first[a])] = z;
      } else {
        c[at(P, (int)p)] = z;
      }
    }
  }
};

// x turned by the table `cs` of its token.
template <typename T, int MODE, int NT, int N>
__device__ __forceinline__ void nr_turn(const RotProb &P, const NrLane<T, MODE> &L,
                                        const NrPartner<N> &other, float *rows, const float2 *cs,
                                        float (&x)[NT][N]) {
  typedef NrTable<T, MODE> Table;
  const int units = Table::units(P);
  if constexpr (MODE == kRotHalves) {
    if (!L.turn) return;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 z = cs[e * units + L.j];
      const float u = x[0][e], v = x[1][e];
      x[0][e] = fmaf(u, z.x, -(v * z.y));
      x[1][e] = fmaf(v, z.x, u * z.y);
    }
  } else if constexpr (MODE == kRotAdjacent) {
#pragma unroll
    for (int e = 0; e < N; e += 2)
      if (L.c0 + e < 2 * P.pairs) {
        const float2 z = cs[e / 2 * units + L.j];
        const float u = x[0][e], v = x[0][e + 1];
        x[0][e] = fmaf(u, z.x, -(v * z.y));
        x[0][e + 1] = fmaf(v, z.x, u * z.y);
      }
  } else {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int e = 0; e < N; ++e) rows[e * 64 + lane] = x[0][e];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (L.c0 + e < 2 * P.pairs) {
        const float2 z = cs[e * units + L.j];
        x[0][e] = fmaf(x[0][e], z.x, rows[other.at[e]] * z.y);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // the next row's copy comes behind these reads
  }
}

// A weight vector's values at the lane's channels.
template <typename T, int MODE, int NT, int N>
__device__ __forceinline__ void nr_weights(const NrLane<T, MODE> &L, const void *w, int wide,
                                           float none, float (&x)[NT][N]) {
#pragma unroll
  for (int t = 0; t < NT; ++t) {
#pragma unroll
    for (int e = 0; e < N; ++e) x[t][e] = none;
    if (w == nullptr) continue;
    if (wide) {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const auto r = Chunk<float>::load(static_cast<const float *>(w) + L.c[t] + min(e, L.n[t]),
                                          L.n[t] - e);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[t][e + i] = Chunk<float>::get(r, i);
      }
    } else {
      const auto r = Chunk<T>::load(static_cast<const T *>(w) + L.c[t], L.n[t]);
#pragma unroll
      for (int e = 0; e < N; ++e) x[t][e] = Chunk<T>::get(r, e);
    }
  }
}

// 1 / sqrt(x): the hardware's estimate and one step of Newton's, off by less than two
// steps; outside the range where the step's products are normal, the exact quotient.
__device__ __forceinline__ float nr_rsqrt(float x) {
  float y = __builtin_amdgcn_rsqf(x);
  y = fmaf(0.5f * y, fmaf(-x * y, y, 1.f), y);
  if (!(x > 0x1p-60f && x < 0x1p+60f)) y = 1.f / sqrtf(x);
  return y;
}

// The row less its mean in place; 1 / std.
template <bool FAST, int NT, int N>
__device__ __forceinline__ float nr_center(float (&x)[NT][N], const int (&n)[NT], const NrProb &Q,
                                           int lgG) {
  float s = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < N; ++e) s += x[t][e];  // (zeros behind the last channel)
  // the quotient by D, to its last place: equal channels, where their sums are exact,
  // have their value for a mean
  s = lanes_sum(s, lgG);
  float mean = s * Q.inv_d;
  mean = fmaf(fmaf(-mean, (float)Q.R.D, s), Q.inv_d, mean);
  s = 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[t][e] -= mean;
      part = fmaf(FAST || e < n[t] ? x[t][e] : 0.f, x[t][e], part);
    }
    s += n[t] > 0 ? part : 0.f;
  }
  return nr_rsqrt(fmaf(lanes_sum(s, lgG), Q.inv_d, Q.eps));
}

// Rows of a tensor [.., heads, D] by token and head, from a run's first token.
template <bool FAST, typename T>
struct NrRows {
  const T *p, *run;
  const int64_t *st;
  int t0;
  __device__ __forceinline__ NrRows(const T *tensor, const int64_t *stride, int first)
      : p(tensor), run(tensor + (int64_t)first * stride[1]), st(stride), t0(first) {}
  // Row of head h of the run's token t.
  __device__ __forceinline__ const T *at(const NrProb &Q, int t, int h) const {
    if (FAST)
      return reinterpret_cast<const T *>(reinterpret_cast<const char *>(run) +
                                         (uint32_t)((t * (int)st[1] + h * (int)st[2]) * (int)sizeof(T)));
    const uint32_t tok = (uint32_t)(t0 + t), b = fdiv(tok, Q.R.fS), s = tok - b * Q.R.fS.d;
    return p + b * st[0] + s * st[1] + h * st[2];
  }
};

// LDS: the table, the rates, staged: the waves' copies of their rows.
template <typename T, int MODE>
struct NrSmem {
  float2 *cs;
  double *rate;
  float *rows;
  __device__ __forceinline__ NrSmem(char *smem, const RotProb &P) {
    rate = reinterpret_cast<double *>(smem);
    rows = reinterpret_cast<float *>(rate + rot_rates(P.pairs));
    cs = reinterpret_cast<float2 *>(rows + (MODE == kRotStaged ? kRotThreads * Chunk<T>::N : 0));
    rows += (threadIdx.x >> 6) * (64 * Chunk<T>::N);
  }
  static size_t bytes(const RotProb &P, int per) {
    return sizeof(double) * rot_rates(P.pairs) +
           (MODE == kRotStaged ? sizeof(float) * kRotThreads * Chunk<T>::N : 0) +
           sizeof(float2) * per * NrTable<T, MODE>::size(P);
  }
};

// LG: the log of the lanes per row, or negative: Q.lgG.
template <typename T, int MODE, bool FAST, int LG>
__global__ void __launch_bounds__(kRotThreads)
    k_nr_fwd(NrProb Q, const T *__restrict__ q, const T *__restrict__ k,
             const void *__restrict__ pos, const void *__restrict__ wq, const void *__restrict__ bq,
             const void *__restrict__ wk, const void *__restrict__ bk, T *__restrict__ oq,
             T *__restrict__ ok) {
  typedef Chunk<T> K;
  typedef NrLane<T, MODE> Lane;
  constexpr int N = K::N, NT = Lane::NT;
  extern __shared__ __align__(16) char smem[];
  const RotProb &P = Q.R;
  const NrSmem<T, MODE> S(smem, P);
  const int tid = threadIdx.x, lgG = LG >= 0 ? LG : Q.lgG, G = 1 << lgG;
  const int t0 = blockIdx.x * P.per_block, nt = min(P.per_block, P.tokens - t0);
  const int h0 = blockIdx.y * P.heads_per, nh = min(P.heads_per, P.H + P.Hk - h0);
  const Lane L(P, tid & (G - 1));
  const NrPartner<N> other(P, L.c0, tid & 63 & ~(G - 1));
  const int per_step = kRotThreads >> lgG, table = NrTable<T, MODE>::size(P);
  rot_rate(P, S.rate);
  bool ready = false;  // the table is there
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    // heads [ha, ha + hn) of q and k taken together; more than one token: all of them
    const int ha = part == 0 ? h0 : max(h0, P.H);
    const int hn = (part == 0 ? min(h0 + nh, P.H) : h0 + nh) - ha;
    if (hn <= 0) continue;
    const int rows = nt * hn;
    const int first = part == 0 ? ha : ha - P.H;  // head of the first row
    const NrRows<FAST, T> in(part == 0 ? q : k, part == 0 ? P.qs : P.ks, t0);
    // (the heads of a token lie behind each other, so do the rows of a run)
    T *const out = (part == 0 ? oq : ok) +
                   ((int64_t)t0 * (part == 0 ? P.H : P.Hk) + first) * P.D;
    auto token = [&](int r) {
      return nt == 1 ? 0 : (int)fdiv((uint32_t)r, part == 0 ? Q.fH : Q.fHk);
    };
    typename K::raw next[NT];
    auto fetch = [&](int r) {
      r = min(r, rows - 1);
      const int t = token(r);
      const T *const x = in.at(Q, t, first + r - t * hn);
#pragma unroll
      for (int i = 0; i < NT; ++i) next[i] = nr_load<FAST>(x + L.c[i], L.n[i]);
    };
    int r = tid >> lgG;
    fetch(r);
    float w[NT][N], b[NT][N];
    nr_weights(L, part == 0 ? wq : wk, Q.wide, 1.f, w);
    nr_weights(L, part == 0 ? bq : bk, Q.wide, 0.f, b);
    if (!ready) {
      __syncthreads();  // the rates are there
      NrTable<T, MODE>::fill(P, pos, S.rate, t0, nt, S.cs);
      __syncthreads();
      ready = true;
    }
    for (int r0 = 0; r0 < rows; r0 += per_step, r += per_step) {  // the same steps for every lane
      float x[NT][N];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) x[i][e] = K::get(next[i], e);
      if (r0 + per_step < rows) fetch(r + per_step);
      const float rstd = nr_center<FAST>(x, L.n, Q, lgG);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) x[i][e] = fmaf(x[i][e] * rstd, w[i][e], b[i][e]);
      nr_turn<T, MODE>(P, L, other, S.rows, S.cs + token(min(r, rows - 1)) * table, x);
      if (r >= rows) continue;
      T *const y = out + r * P.D;
#pragma unroll
      for (int i = 0; i < NT; ++i) nr_store<FAST>(y + L.c[i], x[i], L.n[i]);
    }
  }
}

struct NrGrads {
  const void *q, *k, *wq, *wk, *gq, *gk;
  void *dq, *dk;
  float *part;  // [bq + bk][2][D], or null: no sums wanted
};

// LG: the log of the lanes per row, or negative: Q.lgG.
template <typename T, int MODE, bool FAST, int LG>
__global__ void __launch_bounds__(kRotThreads)
    k_nr_bwd(NrProb Q, NrGrads A, const void *__restrict__ pos) {
  typedef Chunk<T> K;
  typedef NrLane<T, MODE> Lane;
  constexpr int N = K::N, NT = Lane::NT;
  extern __shared__ __align__(16) char smem[];
  const RotProb &P = Q.R;
  const bool isq = (int)blockIdx.x < Q.bq;
  const int per = isq ? P.per_block : Q.per_k, heads = isq ? P.H : P.Hk;
  const int block = isq ? blockIdx.x : blockIdx.x - Q.bq, blocks = isq ? Q.bq : Q.bk;
  const NrSmem<T, MODE> S(smem, P);
  const int table = NrTable<T, MODE>::size(P);
  const int tid = threadIdx.x, lgG = LG >= 0 ? LG : Q.lgG, G = 1 << lgG;
  const Lane L(P, tid & (G - 1));
  const NrPartner<N> other(P, L.c0, tid & 63 & ~(G - 1));
  const T *const x = static_cast<const T *>(isq ? A.q : A.k);
  const T *const g = static_cast<const T *>(isq ? A.gq : A.gk);
  T *const dx = static_cast<T *>(isq ? A.dq : A.dk);
  const int64_t *const xs = isq ? P.qs : P.ks, *const gs = isq ? Q.gqs : Q.gks;
  float w[NT][N];
  nr_weights(L, isq ? A.wq : A.wk, Q.wide, 1.f, w);
  float aw[NT][N], ab[NT][N];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) aw[i][e] = ab[i][e] = 0.f;
  rot_rate(P, S.rate);
  const int per_step = kRotThreads >> lgG;
  for (int64_t first = (int64_t)block * per; first < P.tokens; first += (int64_t)blocks * per) {
    const int t0 = (int)first, nt = min(per, P.tokens - t0), rows = nt * heads;
    const NrRows<FAST, T> xin(x, xs, t0), gin(g, gs, t0);
    T *const out = dx == nullptr ? nullptr : dx + (int64_t)t0 * heads * P.D;
    auto token = [&](int r) { return nt == 1 ? 0 : (int)fdiv((uint32_t)r, isq ? Q.fH : Q.fHk); };
    typename K::raw nx[NT], ng[NT];
    auto fetch = [&](int r) {
      const int in = min(r, rows - 1), t = token(in), h = in - t * heads;
      const T *const px = xin.at(Q, t, h), *const pg = gin.at(Q, t, h);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        nx[i] = nr_load<FAST>(px + L.c[i], L.n[i]);
        // rows past the last add nothing
        ng[i] = nr_load<FAST>(pg + L.c[i], r < rows ? L.n[i] : 0);
      }
    };
    int r = tid >> lgG;
    fetch(r);
    __syncthreads();  // the rates are there; the run before is done with its table
    NrTable<T, MODE>::fill(P, pos, S.rate, t0, nt, S.cs);
    __syncthreads();
    for (int r0 = 0; r0 < rows; r0 += per_step, r += per_step) {  // the same steps for every lane
      float h[NT][N], d[NT][N];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          h[i][e] = K::get(nx[i], e);
          d[i][e] = K::get(ng[i], e);
        }
      if (r0 + per_step < rows) fetch(r + per_step);
      nr_turn<T, MODE>(P, L, other, S.rows, S.cs + token(min(r, rows - 1)) * table, d);
      const float rstd = nr_center<FAST>(h, L.n, Q, lgG);
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          h[i][e] *= rstd;
          aw[i][e] = fmaf(d[i][e], h[i][e], aw[i][e]);
          ab[i][e] += d[i][e];
          d[i][e] *= w[i][e];
          s0 += d[i][e];  // (zeros behind the last channel)
          s1 = fmaf(d[i][e], h[i][e], s1);
        }
      if (out == nullptr) continue;
      s0 = lanes_sum(s0, lgG) * Q.inv_d;
      s1 = lanes_sum(s1, lgG) * Q.inv_d;
      if (r >= rows) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int e = 0; e < N; ++e) d[i][e] = rstd * fmaf(-h[i][e], s1, d[i][e] - s0);
        nr_store<FAST>(out + r * P.D + L.c[i], d[i], L.n[i]);
      }
    }
  }
  if (A.part == nullptr) return;
  // the wave's groups, then the workgroup's four waves
  for (int off = G; off < 64; off <<= 1)
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        aw[i][e] += __shfl_xor(aw[i][e], off, 64);
        ab[i][e] += __shfl_xor(ab[i][e], off, 64);
      }
  __syncthreads();  // the table's LDS is free
  float *const sums = reinterpret_cast<float *>(smem);  // [4][2][D]
  if ((tid & 63) < G) {
    float *const d = sums + (tid >> 6) * 2 * P.D;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < L.n[i]) {
          d[L.c[i] + e] = aw[i][e];
          d[P.D + L.c[i] + e] = ab[i][e];
        }
  }
  __syncthreads();
  for (int c = tid; c < 2 * P.D; c += kRotThreads)
    A.part[(int64_t)blockIdx.x * 2 * P.D + c] =
        (sums[c] + sums[2 * P.D + c]) + (sums[4 * P.D + c] + sums[6 * P.D + c]);
}

// Column sums of the partials of q's (blockIdx.y 0) or k's workgroups: 32 columns
// per workgroup, 32 threads to a column, always added in the same order.
template <typename T>
__global__ void __launch_bounds__(1024)
    k_nr_wsum(const float *__restrict__ part, void *dwq, void *dbq, void *dwk, void *dbk, int D,
              int bq, int bk, int wide) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, j = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c, first = blockIdx.y == 0 ? 0 : bq;
  const int n = blockIdx.y == 0 ? bq : bk;
  float s = 0.f;
  if (col < 2 * D) {
#pragma unroll 8
    for (int i = j; i < n; i += 32) s += part[(int64_t)(first + i) * 2 * D + col];
  }
  sums[j][c] = s;
  __syncthreads();
  s = sums[c][j];  // transposed: thread row j adds column j
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor(s, off, 32);
  const int o = blockIdx.x * 32 + j;
  if (c != 0 || o >= 2 * D) return;
  void *const d = blockIdx.y == 0 ? (o < D ? dwq : dbq) : (o < D ? dwk : dbk);
  if (d == nullptr) return;
  const int at = o < D ? o : o - D;
  if (wide) static_cast<float *>(d)[at] = s;
  else static_cast<T *>(d)[at] = from_f32<T>(s);
}

NrProb nr_prob(const na_norm_rotary_params *p, RotMode *mode) {
  NrProb Q{};
  *mode = rot_prob(&p->rotary, Q.R);
  Q.wide = p->weight_dtype == NA_F32;
  Q.eps = p->eps;
  Q.inv_d = 1.f / (float)Q.R.D;
  while ((1 << Q.lgG) < Q.R.upr) ++Q.lgG;
  Q.fH = make_fastdiv((uint32_t)std::max(Q.R.H, 1));
  Q.fHk = make_fastdiv((uint32_t)std::max(Q.R.Hk, 1));
  for (int i = 0; i < 3; ++i) {
    Q.gqs[i] = p->dq_stride[i];
    Q.gks[i] = p->dk_stride[i];
  }
  if (Q.R.fS.d == 1)  // one token a sample: the next one is the next sample's
    for (int64_t *st : {Q.R.qs, Q.R.ks, Q.gqs, Q.gks}) st[1] = st[0];
  return Q;
}

template <typename F>
void nr_by_type(int dtype, RotMode mode, F &&f) {
  auto by_mode = [&](auto t) {
    if (mode == kRotHalves) f(t, std::integral_constant<int, kRotHalves>{});
    else if (mode == kRotAdjacent) f(t, std::integral_constant<int, kRotAdjacent>{});
    else f(t, std::integral_constant<int, kRotStaged>{});
  };
  if (dtype == NA_F32) by_mode(float{});
  else if (dtype == NA_F16) by_mode(f16_t{});
  else by_mode(bf16_t{});
}

// The kernel's instance: the lanes per row are known to it for rows of 2 to 16 units,
// whose sums then take no branches (25088 tokens of 8 + 8 heads of 32 bf16 channels:
// forward 17.2 -> 16.2 us, backward 30.5 -> 26.5; 131072 of 8 + 8 heads of 64: 130 -> 124
// and 202 -> 189).
template <typename F>
void nr_by_lanes(const NrProb &Q, F &&f) {
#define I_(FAST, LG) f(std::integral_constant<bool, FAST>{}, std::integral_constant<int, LG>{})
  if (!Q.fast) I_(false, -1);
  else if (Q.lgG == 1) I_(true, 1);
  else if (Q.lgG == 2) I_(true, 2);
  else if (Q.lgG == 3) I_(true, 3);
  else if (Q.lgG == 4) I_(true, 4);
  else I_(true, -1);
#undef I_
}

// Entries of a token's table.
int nr_entries(const RotProb &P, int dtype, RotMode mode) {
  int n = 0;
  nr_by_type(dtype, mode, [&](auto t, auto m) {
    n = NrTable<decltype(t), decltype(m)::value>::size(P);
  });
  return n;
}

// Whether rows of runs of up to `per` tokens are and lie as NrProb::fast says.  (A slice in
// time of 131072 tokens of 8 + 8 heads of 64, whose samples lie apart: bf16 119 -> 130 us,
// backward 173 -> 202; float32 220 -> 221 and 330 -> 333.)
bool nr_fast(const RotProb &P, int dtype, const int64_t *st, int heads, int per) {
  if (P.D % (dtype == NA_F32 ? 4 : 8) != 0) return false;
  if (P.fS.d > 1 && (uint32_t)P.tokens > P.fS.d && st[0] != st[1] * (int64_t)P.fS.d) return false;
  if (st[1] < 0 || st[2] < 0 || st[1] >= (1 << 30) || st[2] >= (1 << 30)) return false;
  return (per * st[1] + heads * st[2]) * (dtype == NA_F32 ? 4 : 2) < ((int64_t)1 << 31);
}

// Tokens of a run: kNrUnits units per thread, as many as the table holds; fewer
// where the runs would not be `blocks`.
int nr_run(const RotProb &P, int entries, int heads, int blocks) {
  const int64_t row_units = std::max<int64_t>((int64_t)heads * P.upr, 1);
  int64_t per = std::max<int64_t>(1, kNrUnits * kRotThreads / row_units);
  per = std::min<int64_t>(per, std::max(1, kNrTable / entries));
  return (int)std::min<int64_t>(per, std::max<int64_t>(1, P.tokens / blocks));
}

// The backward's runs and workgroups, shared out by the heads of q and k.
void nr_bwd_plan(NrProb &Q, int dtype, RotMode mode) {
  RotProb &P = Q.R;
  const int entries = nr_entries(P, dtype, mode);
  auto part = [&](int heads, int32_t *per, int32_t *blocks) {
    const int most = std::max(1, (int)((int64_t)kNrBlocks * heads / std::max(P.H + P.Hk, 1)));
    *per = nr_run(P, entries, heads, most);
    *blocks = heads == 0 ? 0 : (int)std::min<int64_t>(most, ((int64_t)P.tokens + *per - 1) / *per);
  };
  part(P.H, &P.per_block, &Q.bq);
  part(P.Hk, &Q.per_k, &Q.bk);
  Q.fast = nr_fast(P, dtype, P.qs, P.H, P.per_block) && nr_fast(P, dtype, Q.gqs, P.H, P.per_block) &&
           nr_fast(P, dtype, P.ks, P.Hk, Q.per_k) && nr_fast(P, dtype, Q.gks, P.Hk, Q.per_k);
}

}  // namespace

bool norm_rotary_fwd(const na_norm_rotary_params *p, const void *q, const void *k, const void *pos,
                     const void *wq, const void *bq, const void *wk, const void *bk, void *oq,
                     void *ok, hipStream_t st) {
  RotMode mode;
  NrProb Q = nr_prob(p, &mode);
  RotProb &P = Q.R;
  // the heads of a token are shared out where there are few tokens
  const int heads = P.H + P.Hk;
  P.per_block = nr_run(P, nr_entries(P, p->rotary.dtype, mode), heads, kRotBlocks);
  P.heads_per = heads;
  if (P.per_block == 1 && P.tokens < kRotBlocks)
    P.heads_per = std::min(heads, kRotThreads >> Q.lgG);
  Q.fast = nr_fast(P, p->rotary.dtype, P.qs, P.H, P.per_block) &&
           nr_fast(P, p->rotary.dtype, P.ks, P.Hk, P.per_block);
  const dim3 grid((unsigned)(((int64_t)P.tokens + P.per_block - 1) / P.per_block),
                  (unsigned)((heads + P.heads_per - 1) / P.heads_per));
  if (grid.x >= ((int64_t)1 << 32) / kRotThreads || grid.y > 65535) return false;  // a launch ends there
  nr_by_type(p->rotary.dtype, mode, [&](auto t, auto m) {
    using T = decltype(t);
    const size_t lds = NrSmem<T, decltype(m)::value>::bytes(P, P.per_block);
    nr_by_lanes(Q, [&](auto fast, auto lg) {
      hipLaunchKernelGGL(
          (k_nr_fwd<T, decltype(m)::value, decltype(fast)::value, decltype(lg)::value>), grid,
          dim3(kRotThreads), lds, st, Q, (const T *)q, (const T *)k, pos, wq, bq, wk, bk, (T *)oq,
          (T *)ok);
    });
  });
  return true;
}

size_t norm_rotary_workspace(const na_norm_rotary_params *p) {
  RotMode mode;
  NrProb Q = nr_prob(p, &mode);
  nr_bwd_plan(Q, p->rotary.dtype, mode);
  return sizeof(float) * 2 * (size_t)Q.R.D * (size_t)(Q.bq + Q.bk);
}

void norm_rotary_bwd(const na_norm_rotary_params *p, const void *q, const void *k, const void *pos,
                     const void *wq, const void *wk, const void *gq, const void *gk, void *dq,
                     void *dk, void *dwq, void *dbq, void *dwk, void *dbk, void *workspace,
                     hipStream_t st) {
  RotMode mode;
  NrProb Q = nr_prob(p, &mode);
  Q.R.sign = -1.f;  // the gradients turn back
  nr_bwd_plan(Q, p->rotary.dtype, mode);
  const bool sums = dwq != nullptr || dbq != nullptr || dwk != nullptr || dbk != nullptr;
  const NrGrads A{q, k, wq, wk, gq, gk, dq, dk, sums ? static_cast<float *>(workspace) : nullptr};
  nr_by_type(p->rotary.dtype, mode, [&](auto t, auto m) {
    using T = decltype(t);
    const size_t lds = std::max(
        NrSmem<T, decltype(m)::value>::bytes(Q.R, std::max(Q.R.per_block, Q.per_k)),
        sizeof(float) * 8 * Q.R.D);
    if (Q.bq + Q.bk > 0)
      nr_by_lanes(Q, [&](auto fast, auto lg) {
        hipLaunchKernelGGL(
            (k_nr_bwd<T, decltype(m)::value, decltype(fast)::value, decltype(lg)::value>),
            dim3(Q.bq + Q.bk), dim3(kRotThreads), lds, st, Q, A, pos);
      });
    if (sums)  // (no rows: zeros)
      hipLaunchKernelGGL((k_nr_wsum<T>), dim3((2 * Q.R.D + 31) / 32, 2), dim3(1024), 0, st, A.part,
                         dwq, dbq, dwk, dbk, Q.R.D, Q.bq, Q.bk, Q.wide);
  });
}

}  // namespace na
