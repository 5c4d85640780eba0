// na_rotary.h — positions, angles and rows of the kernels that rotate queries and
// keys (na_rotary.hip, na_norm_rotary.hip).
#pragma once

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

// Axis of a pair.
__device__ __forceinline__ int rot_axis(const RotProb &P, int pair) {
  int a = 0;
#pragma unroll
  for (int x = 1; x < kRotaryMaxAxes; ++x) a += x < P.axes && pair >= P.first[x] ? 1 : 0;
  return a;
}

// Turns of each pair per unit of position; a barrier before rot_table.
__device__ __forceinline__ void rot_rate(const RotProb &P, double *rate) {
  for (int i = threadIdx.x; i < P.pairs; i += kRotThreads)
    rate[i] = exp2((double)(i - P.first[rot_axis(P, i)]) * P.scale[rot_axis(P, i)]) *
              0.15915494309189533577;
}

// (cos, sin) of the angle by which token `tok` turns pair p of axis a.
__device__ __forceinline__ float2 rot_cos_sin(const RotProb &P, const void *pos, const double *rate,
                                              uint32_t tok, int p, int a) {
  const uint32_t b = fdiv(tok, P.fS);
  const double turns = rot_position(P, pos, b, tok - b * P.fS.d, a) * rate[p];
  float sn, cn;
  sincospif(2.f * (float)(turns - rint(turns)), &sn, &cn);
  return make_float2(cn, sn * P.sign);
}

// Those of tokens t0 .. t0 + nt: [nt][pairs], or [nt][2 pairs] by channel with the
// sine's sign in it.  A barrier before they are read.
template <bool BY_CHANNEL>
__device__ __forceinline__ void rot_table(const RotProb &P, const void *pos, const double *rate,
                                          int t0, int nt, float2 *cs) {
  for (int i = threadIdx.x; i < nt * P.pairs; i += kRotThreads) {
    const uint32_t t = fdiv((uint32_t)i, P.fpairs), p = (uint32_t)i - t * P.fpairs.d;
    const int a = rot_axis(P, (int)p);
    const float2 z = rot_cos_sin(P, pos, rate, (uint32_t)t0 + t, (int)p, a);
    if (BY_CHANNEL) {
      float2 *const c = cs + 2 * ((int)t * P.pairs + P.first[a]) + ((int)p - P.first[a]);
      c[0] = make_float2(z.x, -z.y);
      c[P.first[a + 1] - P.first[a]] = z;
    } else {
      cs[i] = z;
    }
  }
}

// What a call's sizes and axes say; returns how its rows split into units.
inline RotMode rot_prob(const na_rotary_params *p, RotProb &P) {
  const int n = p->dtype == NA_F32 ? 4 : 8;
  int64_t per_sample = p->batch > 0 ? 1 : 0;  // (without samples extents are not bounded)
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
  const RotMode mode = p->interleaved ? kRotAdjacent : whole ? kRotHalves : kRotStaged;
  const int rest = P.D - 2 * P.pairs;
  P.upr = mode == kRotHalves ? P.pairs / n + (rest + 2 * n - 1) / (2 * n) : (P.D + n - 1) / n;
  for (int i = 0; i < 3; ++i) {
    P.qs[i] = p->q_stride[i];
    P.ks[i] = p->k_stride[i];
  }
  // (an extent may be 0: a backward without tokens still writes the weights' gradients)
  P.fS = make_fastdiv((uint32_t)std::max<int64_t>(per_sample, 1));
  P.fE1 = make_fastdiv((uint32_t)std::max<int64_t>(p->extent[1], 1));
  P.fE2 = make_fastdiv((uint32_t)std::max<int64_t>(p->extent[2], 1));
  P.fupr = make_fastdiv((uint32_t)P.upr);
  P.fpairs = make_fastdiv((uint32_t)P.pairs);
  return mode;
}

}  // namespace
}  // namespace na
