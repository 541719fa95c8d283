// The paged 8-bit key/value cache: new tokens into it, and its tokens back as rows.
//
// A page, head and keys or values has one scale, s = max |x| / 127 over the rows that
// the page holds, rounded to fp32, and the numbers are x / s rounded to nearest (ties
// to even).  The rows of a sequence's last page, until it is full, are kept in fp32 as
// well: every append rounds the whole page from them, so what a page holds does not
// depend on how its tokens came, and no number is rounded twice.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.hpp"
#include "flash_tile.hpp"
#include "kv_page.hpp"

namespace aar {
namespace {

struct KvRows {
  FaIn k, v;    // append: the new rows
  FaOut ko, vo;  // read: where rows go
  const int64_t* lens;
  const int64_t* new_lens;
  const int64_t* from;
  int* err;
  int T, stride;
};

// A thread's share of a page: 4 tokens by 4 columns.  Eight quads of tokens are
// neighbours, then the columns: a wave reads eight rows' 128 bytes at once and writes
// whole 32-byte sectors of both layouts without a transposition through LDS.
constexpr int kKvThreads = 256;
struct Unit {
  int q, j, c;  // quad in its group of 32 tokens, first token, first column
  __device__ __forceinline__ Unit(int u, int dp) {
    const int cols = dp / 4;
    q = u & 7;
    j = (u >> 3) / cols * 32 + 4 * q;
    c = (u >> 3) % cols * 4;
  }
};

__device__ __forceinline__ uint32_t* value_word(uint8_t* half, const Unit& w, int e, int dp) {
  return reinterpret_cast<uint32_t*>(half + (w.j >> 5) * 32 * dp + (w.c + e) * 32 + value_quad(w.q));
}

// x / s to the nearest whole number, ties to even, plus 128, from inv, nearly 1 / s: the
// remainder of x after q steps is exact, and more than half a step of it (or just that,
// q odd) is one step further.
__device__ __forceinline__ uint32_t kv_byte(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), over = fabsf(r) - 0.5f * s;
  if (over > 0.f || (over == 0.f && ((int)q & 1))) q += copysignf(1.f, r);
  return (uint32_t)((int)fminf(fmaxf(q, -127.f), 127.f) + 128);
}

// The same for all but about one in 50 000: 2^23 and a half of it take the fraction off,
// and the low byte is the number + 128; near enough to a border to be wrong sets `near`.
// For steps above 2^-100, whose largest quotient rounds to 127.
__device__ __forceinline__ uint32_t kv_byte_fast(float x, float s, float inv, bool& near) {
  const float y = fmaf(x, inv, 12582912.f + 128.f), q = y - (12582912.f + 128.f);
  near = near || fabsf(fmaf(-q, s, x)) >= 0.5f * s;
  return __float_as_uint(y);
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return lo | hi;
#else
  return a;
#endif
}

// Largest of the workgroup's values.
__device__ __forceinline__ uint32_t group_max(uint32_t v, uint32_t* s) {
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, o, kWave));
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < (int)blockDim.x / kWave; ++w) v = max(v, s[w]);
  __syncthreads();  // s may be written again, and every thread has the rows that it read
  return v;
}

// A workgroup takes every stride-th page that the new tokens touch, of a sequence,
// head, and keys or values; the rows of a page that was begun before come from the
// open rows, which the workgroup of the first page alone may replace (by those of the
// last page, after it has read them).
// Bound by the bytes of the rows and of the pages: 128 heads' 1000 rows of d 128 33 us for
// 164 MB, and 30 for those of the read; a single token's page 6.
template <int UNITS, bool VEC>
__global__ void __launch_bounds__(kKvThreads)
kv_append_kernel(const KvPages c, const KvRows a) {
  __shared__ uint32_t smax[kKvThreads / kWave];
  const int BH = c.B * c.Hkv, bh = blockIdx.x % BH, b = bh / c.Hkv, h = bh % c.Hkv;
  const int kv = blockIdx.x / BH & 1, z = blockIdx.x / BH / 2;
  const KvSpan span = kv_span(c, a.lens, a.new_lens, a.T, b);
  if (!span.ok && a.err) *a.err = 1;
  const int s = span.first, e = span.len;
  if (s == e) return;
  const int page = c.page(), p0 = s >> c.shift, p1 = (e - 1) >> c.shift;
  const bool begun = (s & (page - 1)) != 0, left = (e & (page - 1)) != 0;
  // the last page is the first one's workgroup's where both may want the open rows
  const bool both = begun && left && p1 > p0;

  const FaIn& x = kv ? a.v : a.k;
  const float* rows = x.p + (int64_t)b * x.sb + (int64_t)h * x.sh;
  float* open = c.open + ((int64_t)bh * 2 + kv) * page * c.d;
  const int units = (c.dp / 4) << (c.shift - 2);
  auto take = [&](int p) {
    const int base = p << c.shift, lo = max(s, base) - base, hi = min(e - base, page);
    const int64_t id = c.id(b, p);
    f32x4 v[UNITS][4];
    // no branches: all of a thread's loads in flight
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const Unit w(min((int)(threadIdx.x + i * blockDim.x), units - 1), c.dp);
      const int col = min(w.c, (c.d - 1) & ~3);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int j = min(w.j + t, hi - 1);
        const float* row = j < lo ? open + (int64_t)j * c.d : rows + (int64_t)(base + j - s) * x.st;
        v[i][t] = load4<VEC>(row + col, c.d - col);
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const Unit w(threadIdx.x + i * blockDim.x, c.dp);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (w.j + t >= hi || w.c >= c.d) v[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 4; ++n) top = max(top, __float_as_uint(fabsf(v[i][t][n])));
      }
    }
    top = group_max(top, smax);  // as bits: a NaN is the largest
    const float scale = __uint_as_float(top) / 127.0f;
    // of steps below 2^-100 the inverse may be infinite: both sides times 2^64
    const bool tiny = scale < 0x1p-100f;
    const float f = tiny ? 0x1p64f : 1.f, step = scale * f, inv = 1.0f / step;
    const bool flat = !(scale > 0.f && scale < INFINITY);  // all 0, or not finite: numbers of 0
    if (id < 0 && a.err) *a.err = 1;
    if (id >= 0 && threadIdx.x == 0) c.scale(id, h)[kv] = scale;
    uint8_t* half = id < 0 ? nullptr : c.head(id, h, kv);
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
      const int u = threadIdx.x + i * blockDim.x;
      if (u >= units) continue;
      const Unit w(u, c.dp);
      if (id >= 0) {
        uint32_t n[4][4];
        bool near = tiny || flat;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
          for (int k = 0; k < 4; ++k) n[t][k] = kv_byte_fast(v[i][t][k], step, inv, near);
        }
        if (near) {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int k = 0; k < 4; ++k) n[t][k] = flat ? 128u : kv_byte(v[i][t][k] * f, step, inv);
          }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          if (kv) *value_word(half, w, t, c.dp) = low_bytes(n[0][t], n[1][t], n[2][t], n[3][t]);
          else *reinterpret_cast<uint32_t*>(half + (w.j + t) * c.dp + w.c) = low_bytes(n[t][0], n[t][1], n[t][2], n[t][3]);
        }
      }
      if (p != p1 || !left || w.c >= c.d) continue;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int j = w.j + t;
        if (j >= lo && j < hi) store4<VEC>(open + (int64_t)j * c.d + w.c, v[i][t], c.d - w.c);
      }
    }
  };
  for (int p = p0 + z; p < (both ? p1 : p1 + 1); p += a.stride) take(p);
  if (both && z == 0) take(p1);
}

// The same of the pages that rows [from, from + T) touch.  Tokens that the sequence
// does not hold are rows of zeros.
template <bool VEC>
__global__ void __launch_bounds__(kKvThreads)
kv_read_kernel(const KvPages c, const KvRows a) {
  const int BH = c.B * c.Hkv, bh = blockIdx.x % BH, b = bh / c.Hkv, h = bh % c.Hkv;
  const int kv = blockIdx.x / BH & 1;
  const KvSpan span = kv_span(c, a.lens, nullptr, 0, b);
  const int64_t far = int64_t(1) << 40;
  const int64_t from = a.from ? min(max(a.from[b], -far), far) : 0;
  if (!span.ok && a.err) *a.err = 1;
  const FaOut& y = kv ? a.vo : a.ko;
  float* rows = y.p + (int64_t)b * y.sb + (int64_t)h * y.sh;
  const int units = (c.dp / 4) << (c.shift - 2);
  for (int64_t p = (from >> c.shift) + blockIdx.x / BH / 2; p << c.shift < from + a.T; p += a.stride) {
    const int64_t base = p << c.shift;
    const bool held = base >= 0 && base < span.len;
    const int64_t id = held ? c.id(b, (int)p) : -1;
    if (held && id < 0 && a.err) *a.err = 1;
    uint8_t* half = id < 0 ? nullptr : c.head(id, h, kv);
    const float scale = id < 0 ? 0.f : c.scale(id, h)[kv];
    for (int u = threadIdx.x; u < units; u += blockDim.x) {
      const Unit w(u, c.dp);
      if (w.c >= c.d) continue;
      uint32_t n[4] = {0, 0, 0, 0};
      if (id >= 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          n[t] = kv ? *value_word(half, w, t, c.dp) : *reinterpret_cast<uint32_t*>(half + (w.j + t) * c.dp + w.c);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t pos = base + w.j + t, row = pos - from;
        if (row < 0 || row >= a.T) continue;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (id >= 0 && pos < span.len) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t byte = (kv ? n[k] >> (8 * t) : n[t] >> (8 * k)) & 255u;
            v[k] = (float)((int)byte - 128) * scale;
          }
        }
        store4<VEC>(rows + row * y.st + w.c, v, c.d - w.c);
      }
    }
  }
}

// A page's units, and the threads that take them.
int kv_units(const KvPages& c) { return (c.dp / 4) << (c.shift - 2); }
unsigned kv_threads(const KvPages& c) { return (unsigned)std::min(kKvThreads, (int)ceil_div(kv_units(c), kWave) * kWave); }

// The call's grid (a dispatch holds its work items in 32 bits), and the pages that a
// workgroup's are apart.
dim3 kv_grid(const KvPages& c, int64_t T, KvRows* a) {
  const int64_t bh = 2 * (int64_t)c.B * c.Hkv, pages = ceil_div(T, int64_t(1) << c.shift) + 1;
  a->stride = (int)std::min(pages, (int64_t)UINT32_MAX / kKvThreads / bh);
  return dim3((unsigned)(bh * a->stride));
}

bool kv_vec(const KvPages& c, const void* x, const void* y, const void* open, const int64_t* strides) {
  if (c.d % 4 != 0 || !aligned16(x) || !aligned16(y) || !aligned16(open)) return false;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % 4 != 0) return false;
  return true;
}

template <bool VEC>
int launch_append(const KvPages& c, const KvRows& a, dim3 grid, hipStream_t st) {
  const unsigned threads = kv_threads(c);
  const int units = (int)ceil_div(kv_units(c), threads);
  if (units == 1) kv_append_kernel<1, VEC><<<grid, dim3(threads), 0, st>>>(c, a);
  else if (units == 2) kv_append_kernel<2, VEC><<<grid, dim3(threads), 0, st>>>(c, a);
  else kv_append_kernel<4, VEC><<<grid, dim3(threads), 0, st>>>(c, a);
  return launch_status();
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

size_t aar_kv_cache_page_bytes(int64_t kv_heads, int64_t page, int64_t d) {
  const aar_kv_cache c{nullptr, nullptr, nullptr, nullptr, 0, 0, 0, kv_heads, page, d};
  if (kv_check(&c) != AAR_OK) return 0;
  return (size_t)(kv_heads * 2 * page * (ceil_div(d, 16) * 16));
}

int aar_kv_cache_append_f32(const aar_kv_cache* cache, const float* k, const float* v, const int64_t* strides,
                            const int64_t* lens, const int64_t* new_lens, int64_t T, int* err, void* stream) {
  const int rc = kv_check(cache);
  if (rc != AAR_OK) return rc;
  if (T < 0) return AAR_EINVAL;
  if (T > kKvMost) return AAR_EUNSUPPORTED;
  if (cache->sequences == 0 || T == 0) return AAR_OK;
  const bool pages = cache->n_pages > 0;
  if (!k || !v || !strides || !lens || !cache->open || (cache->table_width > 0 && !cache->table) ||
      (pages && (!cache->pages || !cache->scales))) {
    return AAR_EINVAL;
  }
  if (!aligned16(cache->pages)) return AAR_EINVAL;
  const KvPages c = kv_pages(cache);
  KvRows a{};
  a.k = FaIn{k, strides[0], strides[1], strides[2]};
  a.v = FaIn{v, strides[3], strides[4], strides[5]};
  a.lens = lens;
  a.new_lens = new_lens;
  a.err = err;
  a.T = (int)T;
  const dim3 grid = kv_grid(c, std::min(T, (int64_t)c.width << c.shift), &a);
  if (kv_vec(c, k, v, cache->open, strides)) return launch_append<true>(c, a, grid, as_stream(stream));
  return launch_append<false>(c, a, grid, as_stream(stream));
}

int aar_kv_cache_read_f32(const aar_kv_cache* cache, const int64_t* from, const int64_t* lens, float* k, float* v,
                          const int64_t* strides, int64_t T, int* err, void* stream) {
  const int rc = kv_check(cache);
  if (rc != AAR_OK) return rc;
  if (T < 0) return AAR_EINVAL;
  if (T > kKvMost) return AAR_EUNSUPPORTED;
  if (cache->sequences == 0 || T == 0) return AAR_OK;
  if (!k || !v || !strides || !lens || (cache->table_width > 0 && !cache->table) ||
      (cache->n_pages > 0 && (!cache->pages || !cache->scales))) {
    return AAR_EINVAL;
  }
  if (!aligned16(cache->pages)) return AAR_EINVAL;
  const KvPages c = kv_pages(cache);
  KvRows a{};
  a.ko = FaOut{k, strides[0], strides[1], strides[2]};
  a.vo = FaOut{v, strides[3], strides[4], strides[5]};
  a.lens = lens;
  a.from = from;
  a.err = err;
  a.T = (int)T;
  const dim3 grid = kv_grid(c, T, &a), block(kv_threads(c));
  if (kv_vec(c, k, v, nullptr, strides)) kv_read_kernel<true><<<grid, block, 0, as_stream(stream)>>>(c, a);
  else kv_read_kernel<false><<<grid, block, 0, as_stream(stream)>>>(c, a);
  return launch_status();
}

}  // extern "C"
