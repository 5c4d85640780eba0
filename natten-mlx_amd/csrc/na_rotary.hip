// na_rotary.hip — rotary positions by axis, of queries and keys in one launch.
//
// A token at (p_0, p_1, ...) rotates each pair (u, v) of axis a's channels:
//   angle = p_a theta^(-2 i / d_a), i the pair's place among the axis's d_a / 2,
//   (u, v) -> (u cos - v sin, u sin + v cos).
// The pairs of an axis whose channels start at c are (c + i, c + d_a / 2 + i), or
// (c + 2 i, c + 2 i + 1) interleaved; channels behind the last axis pass through.
// The backward is the same kernel with the angle negated.
//
// The angle is formed in float64, in turns, and reduced to half a turn before it
// is rounded: a float32 product of position and frequency is off by an eighth of
// a radian at a million tokens.  A workgroup takes a run of tokens: its threads
// first fill a table of (cos, sin) per token and pair in LDS, once for all heads,
// then stream the rows of all heads of q and k past it in 16-byte chunks.
//
// The reduced angle, the table and the products are float32 (float32 rows are off by
// 4.2e-8 of their norm, 3.3e-8 with sines of the float64 angle), the result is
// rounded once.  Bound: memory.  131072 tokens of 16 heads of 64 bf16 channels on
// three axes, whose halves are no number of chunks: 125 us, reading and writing 268
// MB each (4.3 TB/s; a large copy moves 4.9), 295 us where pairs are read and written
// singly instead of through LDS.
#include "na_chunk.h"
#include "na_launch.h"

#include <algorithm>
#include <cmath>

namespace na {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTable = 4096;  // (cos, sin) entries of a workgroup, 32 KB
constexpr int kRotUnits = 4;     // units per thread of a full launch

// How a row splits into the units that threads take: two chunks half an axis
// apart, or two of the channels behind the axes (16384 tokens of 40 heads, 64 of
// 128 channels rotated: 77 us, 85 where those took one each); a chunk of adjacent
// pairs; or, where half an axis is no number of chunks, any chunk, whose channels
// find their partners in a copy of the rows in LDS (the table then holds an entry
// per channel).
enum RotMode { kRotHalves, kRotAdjacent, kRotStaged };

struct RotProb {
  int32_t tokens, per_block;    // tokens, tokens per workgroup
  int32_t H, Hk, D, heads_per;  // query heads, key heads, channels, heads per workgroup
  int32_t pairs, upr;           // rotated pairs, units per row
  int32_t axes, interleaved, pos_type, pos_batched;
  int32_t first[kRotaryMaxAxes + 1];  // first pair of each axis, then `pairs`
  double scale[kRotaryMaxAxes];       // -2 log2(theta) / d_a
  float sign;                         // of the sines
  FastDiv fS, fE1, fE2, fupr, fheads, fpairs;
  int64_t qs[3], ks[3];               // element strides: sample, token, head
};

// Position of token s (of sample b) on axis a.
__device__ __forceinline__ double rot_position(const RotProb &P, const void *pos, uint32_t b,
                                               uint32_t s, int a) {
  if (P.pos_type == NA_POS_GRID) {
    const uint32_t r = fdiv(s, P.fE2), x2 = s - r * P.fE2.d;
    const uint32_t x0 = fdiv(r, P.fE1), x1 = r - x0 * P.fE1.d;
    const int k = a + 3 - P.axes;  // the last axis is the innermost
    return (double)(k == 2 ? x2 : k == 1 ? x1 : x0);
  }
  const int64_t i = ((P.pos_batched ? (int64_t)b * P.fS.d : 0) + s) * P.axes + a;
  switch (P.pos_type) {
    case NA_POS_I32:
      return (double)static_cast<const int32_t *>(pos)[i];
    case NA_POS_I64:
      return (double)static_cast<const int64_t *>(pos)[i];
    case NA_POS_F64:
      return static_cast<const double *>(pos)[i];
    default:
      return (double)static_cast<const float *>(pos)[i];
  }
}

// Places for the pairs' rates in LDS, a multiple of 16 bytes.
__host__ __device__ constexpr int rot_rates(int pairs) { return (pairs + 1) & ~1; }

// Rows of head h (of q, then of k) of a token.
template <typename T>
struct RotRow {
  const T *src;
  T *dst;
  __device__ __forceinline__ RotRow(const RotProb &P, const T *q, const T *k, T *oq, T *ok,
                                    uint32_t tok, int h) {
    const uint32_t b = fdiv(tok, P.fS), s = tok - b * P.fS.d;
    const bool isq = h < P.H;
    const int64_t *st = isq ? P.qs : P.ks;
    const int hh = isq ? h : h - P.H;
    src = (isq ? q : k) + b * st[0] + s * st[1] + hh * st[2];
    dst = isq ? oq + ((int64_t)tok * P.H + hh) * P.D : ok + ((int64_t)tok * P.Hk + hh) * P.D;
  }
};

// The rows of a workgroup, kRotUnits chunks per thread: kept in registers and
// copied to LDS, from where each channel takes its partner.
template <typename T>
__device__ __forceinline__ void rotate_staged(const RotProb &P, char *smem, const T *q, const T *k,
                                              T *oq, T *ok, int t0, int nt, int h0, int nh) {
  typedef Chunk<T> K;
  constexpr int N = K::N;
  const int width = 2 * P.pairs;
  const float2 *const cs = reinterpret_cast<const float2 *>(smem);
  // behind the rates: partner channel of each rotated one, then the rows, each
  // region from a 16-byte boundary
  uint16_t *const partner = reinterpret_cast<uint16_t *>(
      smem + sizeof(float2) * P.per_block * width + sizeof(double) * rot_rates(P.pairs));
  T *const rows = reinterpret_cast<T *>(partner + (width + 7) / 8 * 8);
  for (int c = threadIdx.x; c < width; c += kRotThreads) {
    int a = 0;
#pragma unroll
    for (int x = 1; x < kRotaryMaxAxes; ++x) a += x < P.axes && c >= 2 * P.first[x] ? 1 : 0;
    const int half = P.first[a + 1] - P.first[a];
    partner[c] = (uint16_t)(c - 2 * P.first[a] < half ? c + half : c - half);
  }
  const int units = nt * nh * P.upr;
  typename K::raw raw[kRotUnits];
  int tok[kRotUnits], c0[kRotUnits];
  T *dst[kRotUnits];
#pragma unroll
  for (int u = 0; u < kRotUnits; ++u) {
    const int i = threadIdx.x + u * kRotThreads;
    if (i >= units) break;
    const uint32_t row = fdiv((uint32_t)i, P.fupr), t = fdiv(row, P.fheads);
    const RotRow<T> r(P, q, k, oq, ok, (uint32_t)t0 + t, h0 + (int)(row - t * P.fheads.d));
    tok[u] = (int)t;
    c0[u] = (i - (int)(row * P.fupr.d)) * N;
    dst[u] = r.dst + c0[u];
    raw[u] = K::load(r.src + c0[u], P.D - c0[u]);
    *reinterpret_cast<typename K::raw *>(rows + i * N) = raw[u];
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kRotUnits; ++u) {
    const int i = threadIdx.x + u * kRotThreads;
    if (i >= units) break;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = K::get(raw[u], e);
    const float2 *const c = cs + tok[u] * width + c0[u];
    const T *const other = rows + i * N - c0[u];
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c0[u] + e < width) {
        const float2 z = c[e];
        x[e] = fmaf(x[e], z.x, to_f32(other[partner[c0[u] + e]]) * z.y);
      }
    K::store(dst[u], x, P.D - c0[u]);
  }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kRotThreads)
    k_rotary(RotProb P, const T *__restrict__ q, const T *__restrict__ k,
             const void *__restrict__ pos, T *__restrict__ oq, T *__restrict__ ok) {
  typedef Chunk<T> K;
  constexpr int N = K::N;
  extern __shared__ __align__(16) char smem[];
  constexpr int E = MODE == kRotStaged ? 2 : 1;  // table entries per pair
  float2 *const cs = reinterpret_cast<float2 *>(smem);  // [per_block][E pairs]
  double *const rate = reinterpret_cast<double *>(cs + P.per_block * E * P.pairs);  // [pairs]
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * P.per_block, nt = min(P.per_block, P.tokens - t0);
  const int h0 = blockIdx.y * P.heads_per, nh = min(P.heads_per, P.H + P.Hk - h0);

  for (int i = tid; i < P.pairs; i += kRotThreads) {
    int a = 0;
#pragma unroll
    for (int x = 1; x < kRotaryMaxAxes; ++x) a += x < P.axes && i >= P.first[x] ? 1 : 0;
    rate[i] = exp2((double)(i - P.first[a]) * P.scale[a]) * 0.15915494309189533577;
  }
  __syncthreads();
  for (int i = tid; i < nt * P.pairs; i += kRotThreads) {
    const uint32_t t = fdiv((uint32_t)i, P.fpairs), p = (uint32_t)i - t * P.fpairs.d;
    int a = 0;
#pragma unroll
    for (int x = 1; x < kRotaryMaxAxes; ++x) a += x < P.axes && (int)p >= P.first[x] ? 1 : 0;
    const uint32_t tok = (uint32_t)t0 + t, b = fdiv(tok, P.fS);
    const double turns = rot_position(P, pos, b, tok - b * P.fS.d, a) * rate[p];
    float sn, cn;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
    sn *= P.sign;
    if (MODE == kRotStaged) {
      float2 *const c = cs + 2 * ((int)t * P.pairs + P.first[a]) + ((int)p - P.first[a]);
      c[0] = make_float2(cn, -sn);
      c[P.first[a + 1] - P.first[a]] = make_float2(cn, sn);
    } else {
      cs[i] = make_float2(cn, sn);
    }
  }
  if (MODE == kRotStaged) {
    rotate_staged<T>(P, smem, q, k, oq, ok, t0, nt, h0, nh);
    return;
  }
  __syncthreads();

  const int units = nt * nh * P.upr;
#pragma unroll 2
  for (int i = tid; i < units; i += kRotThreads) {
    const uint32_t row = fdiv((uint32_t)i, P.fupr);
    const int j = i - (int)(row * P.fupr.d);
    const uint32_t t = fdiv(row, P.fheads);
    const int h = h0 + (int)(row - t * P.fheads.d);
    const RotRow<T> at(P, q, k, oq, ok, (uint32_t)t0 + t, h);
    const T *const src = at.src;
    T *const dst = at.dst;
    const float2 *c = cs + t * P.pairs;
    if (MODE == kRotHalves) {
      const int p0 = j * N;
      if (p0 < P.pairs) {
        int a = 0;
#pragma unroll
        for (int x = 1; x < kRotaryMaxAxes; ++x) a += x < P.axes && p0 >= P.first[x] ? 1 : 0;
        const int c0 = p0 + P.first[a], c1 = c0 + P.first[a + 1] - P.first[a];
        const typename K::raw ru = K::load(src + c0, N), rv = K::load(src + c1, N);
        float xu[N], xv[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 z = c[p0 + e];
          const float u = K::get(ru, e), v = K::get(rv, e);
          xu[e] = u * z.x - v * z.y;
          xv[e] = fmaf(v, z.x, u * z.y);
        }
        K::store(dst + c0, xu, N);
        K::store(dst + c1, xv, N);
      } else {  // channels that pass through, as many to a unit
        const int c0 = 2 * p0, c1 = c0 + N;
        const typename K::raw ru = K::load(src + c0, P.D - c0);
        typename K::raw rv{};
        if (c1 < P.D) rv = K::load(src + c1, P.D - c1);
        float xu[N], xv[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          xu[e] = K::get(ru, e);
          xv[e] = K::get(rv, e);
        }
        K::store(dst + c0, xu, P.D - c0);
        if (c1 < P.D) K::store(dst + c1, xv, P.D - c1);
      }
    } else if (MODE == kRotAdjacent) {
      const int c0 = j * N, n = P.D - c0;
      const typename K::raw r = K::load(src + c0, n);
      float x[N];
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        const float u = K::get(r, e), v = K::get(r, e + 1);
        const int p = (c0 + e) / 2;
        const float2 z = p < P.pairs ? c[p] : make_float2(1.f, 0.f);
        x[e] = p < P.pairs ? u * z.x - v * z.y : u;
        x[e + 1] = p < P.pairs ? fmaf(v, z.x, u * z.y) : v;
      }
      K::store(dst + c0, x, n);
    }
  }
}

}  // namespace

bool rotary(const na_rotary_params *p, const void *q, const void *k, const void *pos, void *oq,
            void *ok, hipStream_t st) {
  RotProb P{};
  const int n = p->dtype == NA_F32 ? 4 : 8;
  int64_t per_sample = 1;
  for (int a = 0; a < 3; ++a) per_sample *= p->extent[a];
  P.tokens = (int32_t)(p->batch * per_sample);
  P.H = p->heads;
  P.Hk = p->kv_heads;
  P.D = p->head_dim;
  P.axes = p->n_axes;
  P.interleaved = p->interleaved;
  P.pos_type = p->pos_type;
  P.pos_batched = p->pos_batched;
  P.sign = p->inverse ? -1.f : 1.f;
  bool whole = true;  // every half axis is a number of chunks
  for (int a = 0; a < p->n_axes; ++a) {
    P.first[a] = P.pairs;
    P.pairs += p->axis_dim[a] / 2;
    P.scale[a] = -2.0 * std::log2(p->theta) / p->axis_dim[a];
    whole = whole && p->axis_dim[a] / 2 % n == 0;
  }
  for (int a = p->n_axes; a <= kRotaryMaxAxes; ++a) P.first[a] = P.pairs;
  const int mode = p->interleaved ? kRotAdjacent : whole ? kRotHalves : kRotStaged;
  const int rest = P.D - 2 * P.pairs;
  P.upr = mode == kRotHalves ? P.pairs / n + (rest + 2 * n - 1) / (2 * n) : (P.D + n - 1) / n;
  for (int i = 0; i < 3; ++i) {
    P.qs[i] = p->q_stride[i];
    P.ks[i] = p->k_stride[i];
  }
  // kRotUnits units per thread; fewer where the launch would not fill the chip,
  // and the heads of a token shared out where one token is too many or too few
  const int heads = P.H + P.Hk, entries = P.pairs * (mode == kRotStaged ? 2 : 1);
  const int64_t row_units = (int64_t)heads * P.upr;
  int64_t per = std::max<int64_t>(1, kRotUnits * kRotThreads / row_units);
  per = std::min<int64_t>(per, std::max(1, kRotTable / entries));
  per = std::min<int64_t>(per, std::max<int64_t>(1, P.tokens / kRotBlocks));
  P.per_block = (int32_t)per;
  const bool few = per == 1 && P.tokens < kRotBlocks;
  P.heads_per = (int32_t)std::min<int64_t>(
      heads, std::max(1, (few ? 1 : kRotUnits) * kRotThreads / P.upr));
  if (per > 1) P.heads_per = heads;
  P.fS = make_fastdiv((uint32_t)per_sample);
  P.fE1 = make_fastdiv((uint32_t)p->extent[1]);
  P.fE2 = make_fastdiv((uint32_t)p->extent[2]);
  P.fupr = make_fastdiv((uint32_t)P.upr);
  P.fheads = make_fastdiv((uint32_t)P.heads_per);
  P.fpairs = make_fastdiv((uint32_t)P.pairs);
  const dim3 grid((unsigned)((P.tokens + per - 1) / per),
                  (unsigned)((heads + P.heads_per - 1) / P.heads_per));
  if (grid.x >= ((int64_t)1 << 32) / kRotThreads || grid.y > 65535) return false;  // a launch ends there
  size_t lds = sizeof(float2) * per * entries + sizeof(double) * rot_rates(P.pairs);
  if (mode == kRotStaged)
    lds += sizeof(uint16_t) * ((entries + 7) / 8 * 8) + 16 * (size_t)per * P.heads_per * P.upr;
  auto run = [&](auto tag) {
    using T = decltype(tag);
#define R_(M)                                                                                   \
  hipLaunchKernelGGL((k_rotary<T, M>), grid, dim3(kRotThreads), lds, st, P, (const T *)q,       \
                     (const T *)k, pos, (T *)oq, (T *)ok)
    if (mode == kRotHalves) R_(kRotHalves);
    else if (mode == kRotAdjacent) R_(kRotAdjacent);
    else R_(kRotStaged);
#undef R_
  };
  if (p->dtype == NA_F32) run(float{});
  else if (p->dtype == NA_F16) run(f16_t{});
  else run(bf16_t{});
  return true;
}

}  // namespace na
