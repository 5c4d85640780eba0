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
#include "na_rotary.h"

namespace na {
namespace {

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

  rot_rate(P, rate);
  __syncthreads();
  rot_table<MODE == kRotStaged>(P, pos, rate, t0, nt, cs);
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
  const int mode = rot_prob(p, P);
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
  P.fheads = make_fastdiv((uint32_t)P.heads_per);
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
