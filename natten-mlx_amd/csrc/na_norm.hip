// na_norm.hip — layer norm over the last dimension, forward and backward, with
// the weight's and bias's gradient.
//
//   mu = mean_c x, rstd = 1 / sqrt(mean_c (x - mu)^2 + eps),
//   xh = (x - mu) rstd, y = xh w + b;
//   dx = rstd (gw - mean_c gw - xh mean_c(gw xh)), gw = dy w,
//   dw = sum over rows of dy xh, db = sum over rows of dy.
//
// A row stays in registers between its sums (the squares are taken about the
// mean, not as a difference of moments), so each pass reads its inputs once.
// Lanes hold 16-byte chunks of a row: a group of 1..64 lanes for narrow rows
// (several rows per wave), a wave with two chunks per lane, or 4 or 16 waves for
// wide ones.  A group walks over rows with a fixed step, the next row's loads in
// flight, and keeps its columns' weights -- and in the backward its columns' sums
// -- in registers; a workgroup's sums leave as one row of partials, added in a
// fixed order by k_norm_wsum, so results do not depend on the run.
//
// Sums are float32; y, dx, dw and db are rounded once.  Bound: memory.  65536 rows
// of 2048 bf16 channels: forward 89 us, reading 268 and writing 270 MB (6.0 TB/s,
// the input partly from the last-level cache), backward 183 us for 545 and 277 MB
// (4.5; a large copy moves 4.9), the partials' sum 5.  25088 rows of 256: 8.7, 12.6
// and 3.9 us.  A call of few rows takes a launch's 2 us.
#include "na_chunk.h"
#include "na_launch.h"

#include <algorithm>
#include <type_traits>

namespace na {
namespace {

// A lane's columns of a weight vector, in the storage type.
template <typename T, typename W, int NT>
struct Cols {
  static constexpr int N = Chunk<T>::N, S = N * (int)sizeof(W) / 16;  // chunks of W per chunk of T
  typename Chunk<W>::raw r[NT][S];
  __device__ __forceinline__ void load(const W *w, int lane, int G, int C) {
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int d0 = (t * G + lane) * N + s * Chunk<W>::N;
        r[t][s] = Chunk<W>::load(w + min(d0, C), C - d0);
      }
  }
  __device__ __forceinline__ float get(int t, int e) const {
    return Chunk<W>::get(r[t][e / Chunk<W>::N], e % Chunk<W>::N);
  }
};

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// Sum over an aligned group of 2^lg lanes (wave-uniform lg), in every lane.
__device__ __forceinline__ float lanes_sum(float x, int lg) {
  if (lg > 0) x = dpp_add<0xB1>(x);   // lane ^ 1
  if (lg > 1) x = dpp_add<0x4E>(x);   // lane ^ 2
  if (lg > 2) x = dpp_add<0x141>(x);  // mirror within 8 lanes
  if (lg > 3) x = dpp_add<0x140>(x);  // mirror within 16 lanes
  if (lg > 4) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (lg > 5) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return x;
}

struct NormProb {
  int32_t rows, C, lgG;
  int32_t per_iter;          // rows of all workgroups in one step
  FastDiv inner;             // rows per outer step of the views
  int64_t xo, xi, go, gi;    // element strides of x's and dy's rows
  float eps, inv_c;
};

__device__ __forceinline__ int64_t view_off(const NormProb &P, uint32_t r, int64_t so, int64_t si) {
  const uint32_t o = fdiv(r, P.inner);
  return (int64_t)o * so + (int64_t)(r - o * P.inner.d) * si;
}

// Sums over a row of WPR waves: LDS slots alternate, so one barrier a call.
template <int WPR, int M>
struct RowSum {
  float *slots;  // [2][M][WPR]
  int turn = 0, lg, w, lane;
  __device__ __forceinline__ RowSum(float *s, int lgG) : slots(s), lg(lgG) {
    w = threadIdx.x >> 6;
    lane = threadIdx.x & 63;
  }
  __device__ __forceinline__ void operator()(float (&x)[M]) {
#pragma unroll
    for (int m = 0; m < M; ++m) x[m] = lanes_sum(x[m], WPR > 1 ? 6 : lg);
    if (WPR > 1) {
      float *s = slots + turn * M * WPR;
      turn ^= 1;
      if (lane == 0)
#pragma unroll
        for (int m = 0; m < M; ++m) s[m * WPR + w] = x[m];
      __syncthreads();
#pragma unroll
      for (int m = 0; m < M; ++m) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < WPR; ++i) t += s[m * WPR + i];
        x[m] = t;
      }
    }
  }
};

template <int WPR>
constexpr int norm_threads() {
  return WPR == 16 ? 1024 : 256;
}

// The thread's place: its lane in the row, lanes per row, first row.
template <int WPR>
struct Place {
  int lane, G, row;
  __device__ __forceinline__ Place(int lgG) {
    if (WPR > 1) {
      lane = threadIdx.x;
      G = 64 * WPR;
      row = blockIdx.x;
    } else {
      G = 1 << lgG;
      lane = threadIdx.x & (G - 1);
      row = (int)((blockIdx.x * 256u + threadIdx.x) >> lgG);
    }
  }
};

template <typename T, typename W, int NT, int WPR>
__global__ void __launch_bounds__(norm_threads<WPR>())
    k_norm_fwd(NormProb P, const T *__restrict__ x, const W *__restrict__ w,
               const W *__restrict__ b, T *__restrict__ y, float2 *__restrict__ stats) {
  typedef Chunk<T> K;
  constexpr int N = K::N;
  __shared__ float slots[2 * WPR];
  RowSum<WPR, 1> total(slots, P.lgG);
  const Place<WPR> at(P.lgG);
  typename K::raw nx[NT];
  auto fetch = [&](int row) {
    const T *p = x + view_off(P, (uint32_t)min(row, P.rows - 1), P.xo, P.xi);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d0 = (t * at.G + at.lane) * N;
      nx[t] = K::load(p + min(d0, P.C), P.C - d0);
    }
  };
  fetch(at.row);
  Cols<T, W, NT> wc, bc;
  if (w != nullptr) wc.load(w, at.lane, at.G, P.C);
  if (b != nullptr) bc.load(b, at.lane, at.G, P.C);
  for (int r0 = 0; r0 < P.rows; r0 += P.per_iter) {  // the same steps for every lane
    const int row = r0 + at.row;
    float v[NT][N], s[1] = {0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[t][e] = K::get(nx[t], e);
        s[0] += v[t][e];
      }
    if (r0 + P.per_iter < P.rows) fetch(row + P.per_iter);
    total(s);
    const float mean = s[0] / (float)P.C;  // equal channels: their value, where its sums are exact
    s[0] = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int n = P.C - (t * at.G + at.lane) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[t][e] -= mean;
        s[0] = fmaf(e < n ? v[t][e] : 0.f, v[t][e], s[0]);
      }
    }
    total(s);
    const float rstd = 1.f / sqrtf(fmaf(s[0], P.inv_c, P.eps));
    if (row >= P.rows) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d0 = (t * at.G + at.lane) * N;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float h = v[t][e] * rstd;
        v[t][e] = fmaf(h, w != nullptr ? wc.get(t, e) : 1.f, b != nullptr ? bc.get(t, e) : 0.f);
      }
      if (d0 < P.C) K::store(y + (int64_t)row * P.C + d0, v[t], P.C - d0);
    }
    if (stats != nullptr && at.lane == 0) stats[row] = make_float2(mean, rstd);
  }
}

// part: [gridDim.x][2][C] sums of dy xh and dy, or null; a single workgroup has
// none and writes dw and db (nullable) itself.
template <typename T, typename W, int NT, int WPR>
__global__ void __launch_bounds__(norm_threads<WPR>())
    k_norm_bwd(NormProb P, const T *__restrict__ x, const W *__restrict__ w,
               const T *__restrict__ dy, const float2 *__restrict__ stats, T *__restrict__ dx,
               float *__restrict__ part, W *__restrict__ dw, W *__restrict__ db) {
  typedef Chunk<T> K;
  constexpr int N = K::N;
  extern __shared__ float smem[];  // one wave per row: [4][2][NT G N] column sums; else slots
  RowSum<WPR, 2> total(smem, P.lgG);
  const Place<WPR> at(P.lgG);
  typename K::raw nx[NT], ng[NT];
  float2 nst;
  auto fetch = [&](int row) {
    const uint32_t r = (uint32_t)min(row, P.rows - 1);
    const T *p = x + view_off(P, r, P.xo, P.xi), *q = dy + view_off(P, r, P.go, P.gi);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d0 = (t * at.G + at.lane) * N;
      // rows past the last one add nothing
      nx[t] = K::load(p + min(d0, P.C), P.C - d0);
      ng[t] = K::load(q + min(d0, P.C), row < P.rows ? P.C - d0 : 0);
    }
    nst = stats[r];
  };
  fetch(at.row);
  Cols<T, W, NT> wc;
  if (w != nullptr) wc.load(w, at.lane, at.G, P.C);
  float aw[NT][N], ab[NT][N];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < N; ++e) aw[t][e] = ab[t][e] = 0.f;
  for (int r0 = 0; r0 < P.rows; r0 += P.per_iter) {
    const int row = r0 + at.row;
    const float mean = nst.x, rstd = nst.y;
    typename K::raw cx[NT], cg[NT];
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      cx[t] = nx[t];
      cg[t] = ng[t];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float g = K::get(cg[t], e), h = (K::get(cx[t], e) - mean) * rstd;
        const float gw = w != nullptr ? g * wc.get(t, e) : g;
        aw[t][e] = fmaf(g, h, aw[t][e]);
        ab[t][e] += g;
        s[0] += gw;
        s[1] = fmaf(gw, h, s[1]);
      }
    }
    if (r0 + P.per_iter < P.rows) fetch(row + P.per_iter);
    if (dx == nullptr) continue;
    total(s);
    const float m0 = s[0] * P.inv_c, m1 = s[1] * P.inv_c;
    if (row >= P.rows) continue;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d0 = (t * at.G + at.lane) * N;
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float g = K::get(cg[t], e), h = (K::get(cx[t], e) - mean) * rstd;
        const float gw = w != nullptr ? g * wc.get(t, e) : g;
        o[e] = rstd * (gw - m0 - h * m1);
      }
      if (d0 < P.C) K::store(dx + (int64_t)row * P.C + d0, o, P.C - d0);
    }
  }
  if (part == nullptr && dw == nullptr && db == nullptr) return;
  float *const pw = part + (int64_t)blockIdx.x * 2 * P.C, *const pb = pw + P.C;
  if (WPR > 1) {  // a thread's columns are its own
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int d0 = (t * at.G + at.lane) * N;
      if (d0 >= P.C) continue;
      if (part != nullptr) {
#pragma unroll
        for (int e = 0; e < N; e += 4) {
          Chunk<float>::store(pw + min(d0 + e, P.C), aw[t] + e, P.C - d0 - e);
          Chunk<float>::store(pb + min(d0 + e, P.C), ab[t] + e, P.C - d0 - e);
        }
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (d0 + e >= P.C) continue;
          if (dw != nullptr) dw[d0 + e] = from_f32<W>(aw[t][e]);
          if (db != nullptr) db[d0 + e] = from_f32<W>(ab[t][e]);
        }
      }
    }
    return;
  }
  // the wave's groups, then the workgroup's four waves
  for (int off = at.G; off < 64; off <<= 1)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        aw[t][e] += __shfl_xor(aw[t][e], off, 64);
        ab[t][e] += __shfl_xor(ab[t][e], off, 64);
      }
  const int width = NT * at.G * N;
  if ((int)(threadIdx.x & 63) < at.G) {
    float *const d = smem + (threadIdx.x >> 6) * 2 * width + at.lane * N;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const int c = t * at.G * N + e;
        *reinterpret_cast<float4 *>(d + c) =
            make_float4(aw[t][e], aw[t][e + 1], aw[t][e + 2], aw[t][e + 3]);
        *reinterpret_cast<float4 *>(d + width + c) =
            make_float4(ab[t][e], ab[t][e + 1], ab[t][e + 2], ab[t][e + 3]);
      }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < P.C; c += 256) {
    float sw = 0.f, sb = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sw += smem[k * 2 * width + c];
      sb += smem[k * 2 * width + width + c];
    }
    if (part != nullptr) {
      pw[c] = sw;
      pb[c] = sb;
    } else {
      if (dw != nullptr) dw[c] = from_f32<W>(sw);
      if (db != nullptr) db[c] = from_f32<W>(sb);
    }
  }
}

// Column sums of n rows of partials [n][2][C]: 32 columns per workgroup, 32
// threads to a column, always added in the same order.
template <typename W>
__global__ void __launch_bounds__(1024)
    k_norm_wsum(const float *__restrict__ part, W *__restrict__ dw, W *__restrict__ db, int C, int n) {
  __shared__ float sums[32][33];
  const int c = threadIdx.x & 31, j = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + c;
  float s = 0.f;
  if (col < 2 * C) {
#pragma unroll 8
    for (int k = j; k < n; k += 32) s += part[(int64_t)k * 2 * C + col];
  }
  sums[j][c] = s;
  __syncthreads();
  // transposed: thread row j adds column j
  s = sums[c][j];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor(s, off, 32);
  const int o = blockIdx.x * 32 + j;
  if (c != 0 || o >= 2 * C) return;
  W *const d = o < C ? dw : db;
  if (d != nullptr) d[o < C ? o : o - C] = from_f32<W>(s);
}

struct NormShape {
  int nt, wpr, lgG, per_block;  // chunks per lane, waves per row, lanes per row, rows per workgroup
};

// Lanes for a row of C channels.  Two chunks per lane where a wave takes a row,
// as the backward's column sums fill the registers beyond (2048 bf16 channels over
// 4096 rows: four chunks per lane 38.9 us, four waves per row 16.7); the backward
// of few rows spreads them over more lanes (768 channels over 2000 rows: 14.7 and
// 11.0 us; the forward takes 4.0 and 5.0).  16-bit rows past 4096 channels take four
// chunks per lane of four waves all the same, whose backward holds 255 registers, one
// wave on a SIMD (8192 rows of 8192 bf16 channels: forward 58 us, backward 83, 4.7 and
// 4.9 TB/s; of 5120, which leave 3 of 8 chunks empty: 47 and 73, 3.6 and 3.4; sixteen
// waves of one chunk were not measured).  Past 8192 channels the backward spills 8 to
// 14 registers in 16-bit types, 85 in float32.
NormShape norm_shape(int dtype, int64_t rows, int C, bool backward) {
  const int n = dtype == NA_F32 ? 4 : 8;
  const int chunks = (C + n - 1) / n;
  NormShape s{};
  if (chunks > 1024) {
    s.wpr = 16;
    s.nt = chunks > 2048 ? 4 : 2;
  } else if (chunks > 128 || (chunks > 64 && backward && rows <= 2048)) {
    s.wpr = 4;
    s.nt = chunks > 512 ? 4 : chunks > 256 ? 2 : 1;
  } else {
    s.wpr = 1;
    s.nt = chunks > 64 ? 2 : 1;
    while ((s.nt << s.lgG) < chunks) ++s.lgG;
  }
  s.per_block = s.wpr > 1 ? 1 : 256 >> s.lgG;
  return s;
}

// The backward's workgroups each leave 2 C partial sums, so they take eight steps
// over the rows at least, once they fill the chip (2048 rows of 16384 channels:
// 256 workgroups 53 us, 512 72; 65536 of 2048: 240 and 159).
int norm_blocks(const NormShape &s, int64_t rows, bool backward) {
  const int64_t steps = (rows + s.per_block - 1) / s.per_block;
  if (!backward) return (int)std::min<int64_t>(steps, s.wpr == 16 ? 1024 : 8192);
  return (int)std::min(steps, std::min<int64_t>(std::max<int64_t>(steps / 8, 256), 512));
}

NormProb norm_prob(const NormArgs &A, const NormShape &s, int blocks) {
  NormProb P{};
  P.rows = (int32_t)A.rows;
  P.C = A.C;
  P.lgG = s.lgG;
  P.per_iter = s.per_block * blocks;
  P.inner = make_fastdiv((uint32_t)A.inner);
  P.xo = A.x_outer;
  P.xi = A.x_inner;
  P.go = A.g_outer;
  P.gi = A.g_inner;
  P.eps = A.eps;
  P.inv_c = 1.f / (float)A.C;
  return P;
}

// WIDE: rows of four-byte elements, the only ones beyond 2048 chunks.
template <bool WIDE, typename F>
void norm_by_shape(const NormShape &s, F &&f) {
#define S_(NT, WPR) f(std::integral_constant<int, NT>{}, std::integral_constant<int, WPR>{})
  if (s.wpr == 16) {
    if (s.nt == 2) S_(2, 16);
    else if constexpr (WIDE) S_(4, 16);
  } else if (s.wpr == 4) {
    if (s.nt == 1) S_(1, 4);
    else if (s.nt == 2) S_(2, 4);
    else S_(4, 4);
  } else {
    if (s.nt == 1) S_(1, 1);
    else S_(2, 1);
  }
#undef S_
}

template <typename F>
void norm_by_type(int dtype, int wdtype, F &&f) {
  if (dtype == NA_F32) f(float{}, float{});
  else if (dtype == NA_F16 && wdtype == NA_F32) f(f16_t{}, float{});
  else if (dtype == NA_F16) f(f16_t{}, f16_t{});
  else if (wdtype == NA_F32) f(bf16_t{}, float{});
  else f(bf16_t{}, bf16_t{});
}

}  // namespace

size_t norm_workspace(int dtype, int64_t rows, int C) {
  const int blocks = norm_blocks(norm_shape(dtype, rows, C, true), rows, true);
  return blocks > 1 ? sizeof(float) * 2 * (size_t)C * (size_t)blocks : 0;
}

void norm_fwd(const NormArgs &A, const void *x, const void *w, const void *b, void *y, float *stats,
              hipStream_t st) {
  const NormShape s = norm_shape(A.dtype, A.rows, A.C, false);
  const int blocks = norm_blocks(s, A.rows, false);
  const NormProb P = norm_prob(A, s, blocks);
  norm_by_type(A.dtype, A.wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    norm_by_shape<sizeof(T) == 4>(s, [&](auto nt, auto wpr) {
      constexpr int NT = decltype(nt)::value, WPR = decltype(wpr)::value;
      hipLaunchKernelGGL((k_norm_fwd<T, W, NT, WPR>), dim3(blocks), dim3(norm_threads<WPR>()), 0, st,
                         P, (const T *)x, (const W *)w, (const W *)b, (T *)y, (float2 *)stats);
    });
  });
}

void norm_bwd(const NormArgs &A, const void *x, const void *w, const void *dy, const float *stats,
              void *dx, void *dw, void *db, void *workspace, hipStream_t st) {
  const NormShape s = norm_shape(A.dtype, A.rows, A.C, true);
  const int blocks = norm_blocks(s, A.rows, true);
  const NormProb P = norm_prob(A, s, blocks);
  const bool sums = dw != nullptr || db != nullptr;
  float *const part = sums && blocks > 1 ? static_cast<float *>(workspace) : nullptr;
  norm_by_type(A.dtype, A.wdtype, [&](auto t, auto wt) {
    using T = decltype(t);
    using W = decltype(wt);
    if (blocks > 0)
      norm_by_shape<sizeof(T) == 4>(s, [&](auto nt, auto wpr) {
        constexpr int NT = decltype(nt)::value, WPR = decltype(wpr)::value;
        const size_t lds = sizeof(float) * (WPR > 1 ? 4 * WPR : 8 * NT * (16 / sizeof(T)) << s.lgG);
        hipLaunchKernelGGL((k_norm_bwd<T, W, NT, WPR>), dim3(blocks), dim3(norm_threads<WPR>()), lds,
                           st, P, (const T *)x, (const W *)w, (const T *)dy, (const float2 *)stats,
                           (T *)dx, part, (W *)dw, (W *)db);
      });
    if (sums && blocks != 1)  // no rows: no partials, zeros
      hipLaunchKernelGGL((k_norm_wsum<W>), dim3((2 * A.C + 31) / 32), dim3(1024), 0, st, part,
                         (W *)dw, (W *)db, A.C, blocks);
  });
}

}  // namespace na
