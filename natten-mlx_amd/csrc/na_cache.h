// na_cache.h — the paged cache of keys and values in 8 bits: pages of
// 2^lgT tokens, elements e4m3, one scale 2^(s - 127) per page and head, its byte s
// as e8m0 holds it (na_cache.hip, na_cache_attend.hip).
#pragma once

#include "na_common.h"

namespace na {
namespace {

constexpr int kScaleBias = 127;
constexpr int kScaleLow = -117, kScaleHigh = 119;  // exponents: every value is a normal bf16

struct CachePages {  // keys or values
  uint8_t *code;
  uint8_t *scale;
  int64_t st[3];  // bytes from page to page, head to head, token to token
  int64_t sc[2];  // of the scales: page, head
};

inline int lg_page(int page_size) {
  int lg = 0;
  while ((1 << lg) < page_size) ++lg;
  return lg;
}

}  // namespace
}  // namespace na
