// na_cache.hip — new keys and values written into the pages of an 8-bit cache.
//
// Token j of sample b's L is token t = len_b - L + j of its sequence, slot t mod T of
// page tables[b][t / T].  Per page and head, of keys and of values,
//   e = smallest exponent with max |x| <= 448 2^e over the page's new tokens,
//   at least the held exponent where the page holds tokens in front of them,
//   code = x 2^-e rounded to e4m3 (half to even).
// Where e grows, the codes in front are divided by 2^growth: exact but for what falls
// below e4m3's normal range.  Scales are powers of two so that growing them rounds
// nothing else, and because e4m3 loses nothing by it: its steps are relative.  What is
// not finite is stored as NaN and does not count for e.
//
// A workgroup takes a page of a sample, a head, and keys or values: it holds the new
// rows in registers, so they are read once; a wave where they are 64 units of 16
// elements at most, four waves otherwise.  No two workgroups write to one page and
// head.  Bound: memory (prompts: 4 x 16384 bf16 tokens of 8 heads of 128, 403 MB, in
// 80 us, 5.0 TB/s; a large copy reaches 4.7), the launch (64 single tokens: 4.1 us).
#include "na_cache.h"
#include "na_chunk.h"
#include "na_launch.h"

#include <algorithm>
#include <type_traits>

namespace na {
namespace {

struct AppendProb {
  int32_t B, L, Hk, pages, lgT, M, D;
  int32_t np;   // pages that a sample's new tokens can touch
  int32_t upr;  // units of 16 elements per row
  FastDiv fupr, fHk, fnp;
  int64_t xs[2][3];  // new keys and values: sample, token, head
  int64_t ts;
  const int32_t *tables, *lens, *fresh;
  CachePages pg[2];
};

// 16 elements of a row as floats, from raw words.
template <typename T>
struct Row16 {
  static constexpr int NC = 16 / Chunk<T>::N;
  typename Chunk<T>::raw r[NC];
  __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int i = 0; i < NC; ++i) r[i] = Chunk<T>::load(p + i * Chunk<T>::N, Chunk<T>::N);
  }
  __device__ __forceinline__ float get(int e) const {
    return Chunk<T>::get(r[e / Chunk<T>::N], e % Chunk<T>::N);
  }
};

__device__ __forceinline__ float exp2i(int e) {  // 2^e, -126 .. 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

template <typename T, int NU, int NT>
__global__ void __launch_bounds__(NT)
    k_cache_append(AppendProb P, const T *__restrict__ key, const T *__restrict__ value) {
  __shared__ uint32_t tops[4];
  const int tid = threadIdx.x;
  const uint32_t bpk = fdiv(blockIdx.x, P.fHk);
  const int h = (int)(blockIdx.x - bpk * P.fHk.d), kv = (int)(bpk & 1);
  const uint32_t b = fdiv(bpk >> 1, P.fnp);
  const int len = min(max(P.lens[b], 0), P.M << P.lgT);
  const int count = P.fresh == nullptr ? P.L : min(max(P.fresh[b], 0), P.L);
  const int lo = max(len - count, 0);  // new tokens [lo, len)
  const int pi = (lo >> P.lgT) + (int)((bpk >> 1) - b * P.fnp.d);
  const int at = pi << P.lgT;
  const int s0 = max(lo - at, 0), rows = min(len - at, 1 << P.lgT) - s0;
  if (rows <= 0) return;
  const int page = P.tables[b * P.ts + pi];
  if ((uint32_t)page >= (uint32_t)P.pages) return;  // holds nothing
  const CachePages &G = P.pg[kv];
  uint8_t *const code = G.code + page * G.st[0] + h * G.st[1];
  uint8_t *const scale = G.scale + page * G.sc[0] + h * G.sc[1];
  const int64_t *const xs = P.xs[kv];
  // (token `at + s0` is number at + s0 - (len - L) of the new ones)
  const T *const x = (kv ? value : key) + b * xs[0] + (at + s0 - len + P.L) * xs[1] + h * xs[2];
  const int units = rows * P.upr;
  Row16<T> v[NU];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = tid + i * NT;
    if (u >= units) break;
    const uint32_t r = fdiv((uint32_t)u, P.fupr);
    v[i].load(x + r * xs[1] + 16 * (u - (int)(r * P.fupr.d)));
  }
  const int held = s0 > 0 ? min(max((int)*scale - kScaleBias, kScaleLow), kScaleHigh) : kScaleLow;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (tid + i * NT >= units) break;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t a = __float_as_uint(v[i].get(e)) & 0x7fffffffu;
      top = max(top, a < 0x7f800000u ? a : 0u);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off, 64));
  if (NT > 64) {
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = max(max(tops[0], tops[1]), max(tops[2], tops[3]));
  }
  // 448 = 1.75 2^8
  const int need = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  const int e = min(max(need, held), kScaleHigh);
  if (s0 > 0 && e > held) {
    const float f = exp2i(max(held - e, -40));  // (every code is 0 from 2^-20 on)
    for (int u = tid; u < s0 * P.upr; u += NT) {
      const uint32_t r = fdiv((uint32_t)u, P.fupr);
      uint4 *const p =
          reinterpret_cast<uint4 *>(code + r * G.st[2] + 16 * (u - (int)(r * P.fupr.d)));
      uint4 c = *p;
      uint32_t *const w = reinterpret_cast<uint32_t *>(&c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false);
        const auto d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
        int o = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(d[0] * f, d[1] * f, o, true);
      }
      *p = c;
    }
  }
  const float inv = exp2i(-e);
  auto scaled = [&](float t) {
    const float y = fminf(fmaxf(t * inv, -448.f), 448.f);
    return (__float_as_uint(t) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : y;
  };
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = tid + i * NT;
    if (u >= units) break;
    const uint32_t r = fdiv((uint32_t)u, P.fupr);
    uint4 c;
    uint32_t *const w = reinterpret_cast<uint32_t *>(&c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      int o = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(v[i].get(4 * j)), scaled(v[i].get(4 * j + 1)), 0,
                                              false);
      w[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(v[i].get(4 * j + 2)),
                                                       scaled(v[i].get(4 * j + 3)), o, true);
    }
    *reinterpret_cast<uint4 *>(code + (s0 + r) * G.st[2] + 16 * (u - (int)(r * P.fupr.d))) = c;
  }
  if (tid == 0) *scale = (uint8_t)(e + kScaleBias);
}

}  // namespace

bool cache_append(const na_cache_params *p, const na_cache *c, const void *key, const void *value,
                  const int32_t *tables, const int32_t *lens, const int32_t *fresh,
                  hipStream_t st) {
  AppendProb P{};
  P.B = p->batch;
  P.L = p->tokens;
  P.Hk = p->kv_heads;
  P.pages = p->pages;
  P.lgT = lg_page(p->page_size);
  P.M = p->table_pages;
  P.D = p->head_dim;
  const int T = p->page_size;
  P.np = (int32_t)std::min<int64_t>(((int64_t)P.L + T - 2) / T + 1, std::max(P.M, 1));
  P.upr = P.D / 16;
  P.fupr = make_fastdiv((uint32_t)P.upr);
  P.fHk = make_fastdiv((uint32_t)P.Hk);
  P.fnp = make_fastdiv((uint32_t)P.np);
  for (int i = 0; i < 3; ++i) {
    P.xs[0][i] = p->k_stride[i];
    P.xs[1][i] = p->v_stride[i];
  }
  P.ts = p->table_stride;
  P.tables = tables;
  P.lens = lens;
  P.fresh = fresh;
  P.pg[0] = {static_cast<uint8_t *>(c->key), static_cast<uint8_t *>(c->key_scale),
             {c->key_stride[0], c->key_stride[1], c->key_stride[2]},
             {c->key_scale_stride[0], c->key_scale_stride[1]}};
  P.pg[1] = {static_cast<uint8_t *>(c->value), static_cast<uint8_t *>(c->value_scale),
             {c->value_stride[0], c->value_stride[1], c->value_stride[2]},
             {c->value_scale_stride[0], c->value_scale_stride[1]}};
  const int64_t blocks = (int64_t)P.B * P.np * 2 * P.Hk;
  const int units = std::min(P.L, T) * P.upr;  // of a workgroup
  if (blocks >= ((int64_t)1 << 32) / 256 || blocks >= ((int64_t)1 << 31)) return false;
  auto run = [&](auto tag) {
    using E = decltype(tag);
    auto launch = [&](auto nu, auto nt) {
      constexpr int NU = decltype(nu)::value, NT = decltype(nt)::value;
      hipLaunchKernelGGL((k_cache_append<E, NU, NT>), dim3((unsigned)blocks), dim3(NT), 0, st, P,
                         (const E *)key, (const E *)value);
    };
#define U_(NU, NT) launch(std::integral_constant<int, NU>{}, std::integral_constant<int, NT>{})
    // (512 single tokens of 8 heads of 128: 7.0 us, with four waves 11.7; 8 x 2048 of 8
    // heads of 64, pages of 16: 10.9 and 20.1.  Registers for no more than the units:
    // 8 x 4096 of 8 heads of 128, pages of 64: 27.5, with those for 2048 units 30.7)
    if (units <= 64) U_(1, 64);
    else if (units <= 256) U_(1, 256);
    else if (units <= 512) U_(2, 256);
    else if (units <= 1024) U_(4, 256);
    else U_(8, 256);
#undef U_
  };
  if (p->dtype == NA_F32) run(float{});
  else if (p->dtype == NA_F16) run(f16_t{});
  else run(bf16_t{});
  return true;
}

}  // namespace na
