// The key/value cache in pages of 8-bit numbers: its layout, the limits of its
// sizes, and a sequence's tokens.
//
// A page holds `page` tokens of one sequence.  For every key/value head it has the
// tokens' keys, then their values, a byte a number: number + 128, numbers -127 to
// 127, which times the scale of the page, the head and keys or values stand for the
// elements.  With dp = d rounded up to 16 (the columns past d hold 0):
//   key c of token j at      j dp + c
//   value c of token j at    page dp + (j / 32) 32 dp + 32 c + 4 r(j / 4 % 8) + j % 4,
// r the reversal of three bits.  Rows of keys and, 32 tokens at a time, columns of
// values then are what a lane of the matrix unit takes, without a transposition: the
// attention's P has tokens 4 g .. 4 g + 3 and 4 g + 16 .. 4 g + 19 in lane group g, and
// these are 8 consecutive bytes of a column.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.hpp"

namespace aar {

struct KvPages {
  uint8_t* bytes;        // [n_pages][Hkv][2][page * dp]
  float* scales;         // [n_pages][Hkv][2]
  float* open;           // [B][Hkv][2][page][d]
  const int64_t* table;  // [B][width]
  int64_t n_pages;
  int B, width, Hkv, shift, d, dp;  // page = 1 << shift

  __device__ __forceinline__ int page() const { return 1 << shift; }
  // Bytes of one head's keys, or values, in a page.
  __device__ __forceinline__ int half() const { return dp << shift; }
  __device__ __forceinline__ uint8_t* head(int64_t id, int h, int kv) const {
    return bytes + ((id * Hkv + h) * 2 + kv) * (int64_t)half();
  }
  __device__ __forceinline__ float* scale(int64_t id, int h) const { return scales + (id * Hkv + h) * 2; }
  // Page `at` of sequence b, or -1 where the table names none.
  __device__ __forceinline__ int64_t id(int b, int at) const {
    const int64_t x = table[(int64_t)b * width + at];
    return x >= 0 && x < n_pages ? x : -1;
  }
};

// Where a group's four tokens from 4 q on stand among the 32 bytes of a value column.
__device__ __forceinline__ int value_quad(int q) { return 4 * ((q & 1) << 2 | (q & 2) | q >> 2); }

// A sequence's tokens: `len`, of which those from `first` on are the call's new
// ones.  Numbers that do not fit (a length below 0 or past the table, more new
// tokens than the call has or than there are) leave the sequence out.
struct KvSpan {
  int len, first;
  bool ok;
};
__device__ __forceinline__ KvSpan kv_span(const KvPages& c, const int64_t* lens, const int64_t* new_lens, int T, int b) {
  const int64_t len = lens[b], n = new_lens ? new_lens[b] : T;
  const bool ok = len >= 0 && len <= ((int64_t)c.width << c.shift) && n >= 0 && n <= T && n <= len;
  return {ok ? (int)len : 0, ok ? (int)(len - n) : 0, ok};
}

constexpr int64_t kKvMost = int64_t(1) << 30;  // tokens of a sequence

// The cache's sizes: AAR_OK, or what is wrong with them.
inline int kv_check(const aar_kv_cache* c) {
  if (!c || c->sequences < 0 || c->table_width < 0 || c->n_pages < 0 || c->kv_heads <= 0 || c->d <= 0 || c->d > 128) {
    return AAR_EINVAL;
  }
  if (c->page != 32 && c->page != 64 && c->page != 128) return AAR_EINVAL;
  if (c->table_width > kKvMost / c->page || c->kv_heads > (1 << 16) || c->n_pages > (int64_t(1) << 40)) return AAR_EUNSUPPORTED;
  if (c->sequences > (1 << 22) || c->sequences * c->kv_heads > (1 << 22)) return AAR_EUNSUPPORTED;
  return AAR_OK;
}

inline KvPages kv_pages(const aar_kv_cache* c) {
  KvPages p{};
  p.bytes = c->pages;
  p.scales = c->scales;
  p.open = c->open;
  p.table = c->table;
  p.n_pages = c->n_pages;
  p.B = (int)c->sequences;
  p.width = (int)c->table_width;
  p.Hkv = (int)c->kv_heads;
  p.shift = c->page == 32 ? 5 : (c->page == 64 ? 6 : 7);
  p.d = (int)c->d;
  p.dp = (int)ceil_div(c->d, 16) * 16;
  return p;
}

}  // namespace aar
