// Attention of new tokens over the paged 8-bit key/value cache (kv_page.hpp), with an
// optional window and sinks.
//
// The queries of sequence b are its last n tokens; the query at position i sees the
// keys j <= i with i - j < window or j < sinks.  With kq, vq the numbers of a page and
// sk, sv its scales,
//   s_ij = scale sk (q_i . kq_j),  O_i = sum_j P_ij sv vq_j,  P = softmax(s).
//
// Numbers of 8 bits are exact in fp16, so a product over them needs the other operand
// alone in two fp16 parts: q, its row scaled such that its largest element is in
// [2^13, 2^14), is off by at most 2^-22 of an element or 2^-38 of the row's largest;
// P, at most 2^4 times 2^11, by 2^-22 of itself or 2^-36 of the row's largest.  Sums are
// in fp32 and take the pages' scales after the matrix op.
//
// Single tokens are bound by the cache's bytes: 384 heads, 4096 tokens, d 64: 30.4 + 4.0 us for
// 150 MB; 16 x 4 heads, 32768 tokens, d 128: 85 + 4.3 us for 402 MB, 4.7 TB/s.  Chunks of a
// prompt are bound by the vector unit, which makes the numbers fp16 for every 16 rows anew: 48
// heads' 250 rows over 4096 tokens 41 us, 17 at the matrix unit's rate.  Two and four groups of
// rows that share a wave's tiles were slower: their registers cost the second wave of a SIMD.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "common.hpp"
#include "flash_tile.hpp"
#include "kv_page.hpp"

namespace aar {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct KvAttn {
  FaIn q;
  FaOut o;
  const int64_t* lens;
  const int64_t* new_lens;
  int* err;
  float* part_o;  // [blocks of rows][splits][rows of a block][DT] normalised partial O
  float* part_l;  // [blocks of rows][splits][rows of a block] m + log2(l) of it
  int T, G, R;    // R = G * T query rows of each key/value head
  int window, sinks, blocks, splits;
  float scale_log2;
};

constexpr int kKeys = 32;  // of a tile
constexpr int kRows = 16;  // of a workgroup
// Waves that a SIMD holds, by their registers: of workgroups of 4 waves, and of one that
// fills a CU.  Four of the small ones a SIMD, which would fit for dt = 64 but for two
// registers, take 36.0 us where three take 34.7 (32 x 12 heads' single rows, 4096 tokens).
constexpr int kv_resident(int dt) { return dt <= 64 ? 3 : 2; }
constexpr int kv_wide(int dt) { return dt <= 64 ? 4 : 2; }

// D = A B + C for 16 x 16 over 32: lane (r = lane % 16, g = lane / 16) holds A[r][8g ..
// 8g+7] and B[8g .. 8g+7][r], and C[4g .. 4g+3][r].
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
#else
  return c;
#endif
}

// Bytes lo .. lo + 1 of x, numbers + 128, as fp16: 1024 + byte by its bits, less 1152.
template <int LO>
__device__ __forceinline__ uint32_t halves_of(uint32_t x) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t v = __builtin_amdgcn_perm(x, 0x64646464u, LO == 0 ? 0x00050004u : 0x00070006u);
#else
  const uint32_t v = x;
#endif
  const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, v) - off);
}
__device__ __forceinline__ u32x4 halves_of(uint32_t x, uint32_t y) {
  return u32x4{halves_of<0>(x), halves_of<2>(x), halves_of<0>(y), halves_of<2>(y)};
}

// (a, b) in two fp16 parts, a pair a word.  one: 1, unknown to the compiler, so that a
// difference is one mixed multiply-add and not a conversion and a subtraction.
__device__ __forceinline__ void split_pair(float a, float b, float one, uint32_t& hi, uint32_t& lo) {
  const f16x2 x = __builtin_convertvector(f32x2{a, b}, f16x2);
  hi = __builtin_bit_cast(uint32_t, x);
  const f32x2 rest = {fmaf(a, one, -(float)x[0]), fmaf(b, one, -(float)x[1])};
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
}

// Over the four lanes that hold a query row.
__device__ __forceinline__ float row_max(float v) { return half_swap_max(fmaxf(v, swizzle_xor16(v))); }
__device__ __forceinline__ float row_sum(float v) { return half_swap_sum(v + swizzle_xor16(v)); }

// The tiles of keys that any of the tokens [t0, t1] sees: sinks' tiles, then the
// window's.
struct Tiles {
  int sinks, near, count;
  __device__ __forceinline__ Tiles(const KvAttn& a, int first, int t0, int t1) {
    const int end = first + t1, low = max(0, first + t0 - a.window + 1);
    near = low / kKeys;
    sinks = min((min(a.sinks, end + 1) + kKeys - 1) / kKeys, near);
    count = t1 < t0 ? 0 : sinks + end / kKeys + 1 - near;
  }
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : near + i - sinks; }
};

// Bytes on the device: a pointer put together from a lane's words has to say so, or its
// loads are flat ones, which wait for LDS too.
typedef const __attribute__((address_space(1))) uint8_t* DeviceBytes;

// What a wave reads of a tile: rows of keys 16 bytes a lane, columns of values 8.
template <int DT>
struct Tile {
  static constexpr int NK = (DT + 63) / 64, NB = DT / 16;
  u32x4 k[2][NK];
  u32x2 v[NB];
  __device__ __forceinline__ void load_keys(DeviceBytes keys, int dp, int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        k[n][c] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
        if (64 * c + 16 * g < dp) k[n][c] = *(const __attribute__((address_space(1))) u32x4*)(keys + (16 * n + r) * dp + 64 * c + 16 * g);
      }
    }
  }
  __device__ __forceinline__ void load_values(DeviceBytes values, int dp, int lane) {
    const int r = lane & 15, g = lane >> 4, at = 8 * ((g & 1) << 1 | g >> 1);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      v[b] = u32x2{0x80808080u, 0x80808080u};
      if (16 * b < dp) v[b] = *(const __attribute__((address_space(1))) u32x2*)(values + (16 * b + r) * 32 + at);
    }
  }
};

// A workgroup takes 16 query rows of a key/value head (the rows of the G query
// heads that share it, one list) and a range of their tiles; its W waves take every
// W-th tile, each with an online softmax of its own, and meet at the end.
template <int DT, int W, bool VEC>
__global__ void __launch_bounds__(W * kWave, W == 4 ? kv_resident(DT) : kv_wide(DT))
kv_attn_kernel(const KvPages c, const KvAttn a) {
  constexpr int NK = Tile<DT>::NK, NB = Tile<DT>::NB, NP = 2 * NK;  // NP: 32-column steps of a score
  __shared__ f32x4 so[W][NB][kWave];
  __shared__ float sm[W][kWave], sl[W][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int BH = c.B * c.Hkv, bh = blockIdx.x % BH, b = bh / c.Hkv, hk = bh % c.Hkv;
  const int part = blockIdx.x / BH % a.splits, block = blockIdx.x / BH / a.splits;
  const int row0 = block * kRows, row1 = min(a.R, row0 + kRows) - 1;
  const int row = row0 + r, head = row / a.T, t = row - head * a.T;  // the lane's

  // the row of q, on its way before the numbers that say whether it counts
  f32x4 x[NP][2];
  const float* q = a.q.p + (int64_t)b * a.q.sb + ((int64_t)hk * a.G + head) * a.q.sh + (int64_t)t * a.q.st;
#pragma unroll
  for (int s = 0; s < NP; ++s) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int col = 64 * (s >> 1) + 16 * g + 8 * (s & 1) + 4 * p;
      x[s][p] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (row < a.R && col < c.d) x[s][p] = load4<VEC>(q + col, c.d - col);
    }
  }
  const KvSpan span = kv_span(c, a.lens, a.new_lens, a.T, b);
  if (!span.ok && a.err) *a.err = 1;

  // the tokens that the block's rows belong to
  const int n = span.len - span.first;
  int t0 = 0, t1 = a.T - 1;
  if (row0 / a.T == row1 / a.T) {
    t0 = row0 % a.T;
    t1 = row1 % a.T;
  }
  t1 = min(t1, n - 1);
  const int pos = row < a.R && t < n ? span.first + t : -1;  // -1: a row that is none
  const Tiles tiles(a, span.first, t0, t1);
  const int i0 = (int)((int64_t)tiles.count * part / a.splits), i1 = (int)((int64_t)tiles.count * (part + 1) / a.splits);

  // 64 of the wave's tiles at a time: a lane looks one up
  int key = 0;
  float sk = 0.f, sv = 0.f;
  const uint8_t* at = nullptr;
  uint64_t rest = 0;  // the lanes of the tiles to come
  auto keys_at = [&](int i) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)(uintptr_t)at, i);
    const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uintptr_t)at >> 32), i);
    return (DeviceBytes)((uint64_t)hi << 32 | lo);
  };
  Tile<DT> tile;
  int i = -1;  // the present tile's lane
  auto look_up = [&](int base) {
    const int mine = base + W * lane;
    int64_t id = -1;
    if (mine < i1) {
      key = tiles.at(mine) * kKeys;
      id = c.id(b, key >> c.shift);
      if (id < 0 && a.err) *a.err = 1;
    }
    if (id >= 0) {
      at = c.head(id, hk, 0) + (key & (c.page() - 1)) * c.dp;
      const float* s = c.scale(id, hk);
      sk = s[0];
      sv = s[1];
    }
    rest = __ballot(id >= 0);
    i = rest != 0 ? __ffsll((unsigned long long)rest) - 1 : -1;
    if (i < 0) return;
    tile.load_keys(keys_at(i), c.dp, lane);
    tile.load_values(keys_at(i) + c.half(), c.dp, lane);
  };
  look_up(i0 + wave);

  // q in parts, its row's factor 2^-ex
  u32x4 qp[NP][2];
  float top = 0.f;
#pragma unroll
  for (int s = 0; s < NP; ++s) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][p][e]));
    }
  }
  top = row_max(top);
  const int ex = top > 0.f ? 13 - ilogbf(top) : 0;
  const float sign = copysignf(1.f, a.scale_log2);
  float one = 1.f;
  asm("" : "+v"(one));
#pragma unroll
  for (int s = 0; s < NP; ++s) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      uint32_t hi, lo;
      split_pair(ldexpf(x[s][p >> 1][2 * (p & 1)] * sign, ex), ldexpf(x[s][p >> 1][2 * (p & 1) + 1] * sign, ex), one, hi,
                 lo);
      qp[s][0][p] = hi;
      qp[s][1][p] = lo;
    }
  }

  f32x4 o[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  // `next_keys` and `next_values` send for the next tile's as soon as this one's are used
  auto compute = [&](int key0, float sk, float sv, auto next_keys, auto next_values) {
    f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      u32x4 k[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) k[h] = halves_of(tile.k[h][p >> 1][2 * (p & 1)], tile.k[h][p >> 1][2 * (p & 1) + 1]);
#pragma unroll
      for (int part = 1; part >= 0; --part) {
#pragma unroll
        for (int h = 0; h < 2; ++h) s[h] = mfma16(k[h], qp[p][part], s[h]);
      }
    }
    next_keys();

    // positive, so that the largest product is the largest score; a scale that is not finite
    // times its page's numbers, which are 0, is NaN
    const float f = sk < INFINITY ? fmaxf(ldexpf(sk * fabsf(a.scale_log2), -ex), 0x1p-126f) : INFINITY;
    const bool all = key0 + kKeys - 1 <= span.first + t0 && (key0 > span.first + t1 - a.window || key0 + kKeys <= a.sinks);
    float mx = -INFINITY, sum = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!all) {
          const int key = key0 + 16 * h + 4 * g + e;
          const bool sees = key <= pos && (key > pos - a.window || key < a.sinks);
          s[h][e] = sees ? s[h][e] : -INFINITY;
        }
        mx = fmaxf(mx, s[h][e]);
      }
    }
    mx *= f;
    // a scale that is not finite reaches the rows that see it alone
    const float weight = all || row_max(mx) != -INFINITY ? sv : 0.f;
    if (__any(mx > m + 4.f)) {  // the maximum follows only where P would pass 2^4
      mx = fmaxf(row_max(mx), m);
      const float alpha = mx > m ? exp2f(m - mx) : 1.f;
      m = mx;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NB; ++d) o[d] *= alpha;
    }
    const float mu = m == -INFINITY ? 11.f : 11.f - m;
    u32x4 pp[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[h][e] = fast_exp2(fmaf(s[h][e], f, mu));
        sum += s[h][e];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t hi, lo;
        split_pair(s[h][2 * e], s[h][2 * e + 1], one, hi, lo);
        pp[0][2 * h + e] = hi;
        pp[1][2 * h + e] = lo;
      }
    }
    l += sum;
#pragma unroll
    for (int d = 0; d < NB; d += 2) {
      if (16 * d >= c.dp) continue;
      u32x4 v[2];
      f32x4 y[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) v[n] = halves_of(tile.v[d + n][0], tile.v[d + n][1]);
      // a matrix op waits for the one whose sum it continues: two sums take turns
#pragma unroll
      for (int n = 0; n < 2; ++n) y[n] = mfma16(v[n], pp[1], f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int n = 0; n < 2; ++n) y[n] = mfma16(v[n], pp[0], y[n]);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d + n][e] = fmaf(weight, y[n][e], o[d + n][e]);
      }
    }
    next_values();
  };

  for (int base = i0 + wave; base < i1;) {
    while (i >= 0) {
      rest &= rest - 1;
      const int next = rest != 0 ? __ffsll((unsigned long long)rest) - 1 : -1;
      const DeviceBytes p = keys_at(next < 0 ? i : next);
      compute(__builtin_amdgcn_readlane(key, i), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sk), i)),
              __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sv), i)),
              [&] { tile.load_keys(p, c.dp, lane); }, [&] { tile.load_values(p + c.half(), c.dp, lane); });
      i = next;
    }
    base += W * kWave;
    if (base < i1) look_up(base);
  }

  // the waves' sums meet: a thread takes every W-th block of columns of its lane's row
  sm[wave][lane] = m;
  sl[wave][lane] = row_sum(l);
#pragma unroll
  for (int d = 0; d < NB; ++d) so[wave][d][lane] = o[d];
  __syncthreads();
  if (row >= a.R) return;
  float f[W], mx = sm[0][lane], sum = 0.f;
#pragma unroll
  for (int v = 1; v < W; ++v) mx = fmaxf(mx, sm[v][lane]);
  const float mu = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int v = 0; v < W; ++v) {
    f[v] = exp2f(sm[v][lane] - mu);
    sum += sl[v][lane] * f[v];
  }
  const bool none = pos < 0 || sum == 0.f;  // a row that sees nothing, or is none
  const float inv = 1.0f / sum;
  const int64_t prow = (((int64_t)block * BH + bh) * a.splits + part) * kRows + r;
  float* orow = a.splits > 1 ? a.part_o + prow * DT
                             : a.o.p + (int64_t)b * a.o.sb + ((int64_t)hk * a.G + head) * a.o.sh + (int64_t)t * a.o.st;
  for (int d = wave; d < NB; d += W) {
    const int col = 16 * d + 4 * g;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const f32x4 z = so[v][d][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += z[e] * f[v];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = none ? 0.f : y[e] * inv;
    if (a.splits > 1) *reinterpret_cast<f32x4*>(orow + col) = y;
    else if (col < c.d) store4<VEC>(orow + col, y, c.d - col);
  }
  if (a.splits > 1 && wave == 0 && g == 0) a.part_l[prow] = none ? -INFINITY : mx + log2f(sum);
}

// The parts of every query row, as cross attention's: with L_p = m_p + log2(l_p),
//   O = sum_p 2^(L_p - M) O_p / sum_p 2^(L_p - M),  M the largest L_p.
template <int DT, bool VEC>
__global__ void __launch_bounds__(256)
kv_attn_join_kernel(const KvPages c, const KvAttn a) {
  constexpr int kLanes = DT / 4;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, item = u / kLanes;
  const int BH = c.B * c.Hkv, bh = (int)(item / a.R), row = (int)(item % a.R), col = (int)(u % kLanes) * 4;
  if (bh >= BH) return;
  const int64_t at = ((int64_t)(row / kRows) * BH + bh) * a.splits * kRows + row % kRows;
  // eight parts' loads in flight
  constexpr int U = 8;
  float mx = -INFINITY, w = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < a.splits; p0 += U) {
    float l[U];
    f32x4 x[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int p = min(p0 + i, a.splits - 1);
      l[i] = a.part_l[at + (int64_t)p * kRows];
      x[i] = *reinterpret_cast<const f32x4*>(a.part_o + (at + (int64_t)p * kRows) * DT + col);
    }
    float top = mx;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (p0 + i >= a.splits) l[i] = -INFINITY;
      top = fmaxf(top, l[i]);
    }
    const float mu = top == -INFINITY ? 0.f : top, f = exp2f(mx - mu);
    w *= f;
    o *= f;
    mx = top;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float h = exp2f(l[i] - mu);
      w += h;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += h * x[i][e];
    }
  }
  const float inv = w == 0.f ? 0.f : 1.0f / w;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  const int head = row / a.T, t = row - head * a.T, b = bh / c.Hkv, hk = bh % c.Hkv;
  if (col < c.d) {
    store4<VEC>(a.o.p + (int64_t)b * a.o.sb + ((int64_t)hk * a.G + head) * a.o.sh + (int64_t)t * a.o.st + col, o, c.d - col);
  }
}

// ------------------------------------------------------------------ host side

int kv_tile_dim(int64_t d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

struct KvPlan {
  int splits, waves;
  int64_t blocks;
};

KvPlan kv_plan(const aar_kv_cache& c, int64_t H, int64_t T, int64_t window, int64_t sinks) {
  const int64_t R = H / c.kv_heads * T, cus = device_cu_count();
  KvPlan p;
  p.blocks = ceil_div(R, kRows);
  const int64_t grid = p.blocks * c.sequences * c.kv_heads;
  const int64_t most = std::min(c.table_width * c.page, std::min(window, kKvMost) + std::min(sinks, kKvMost) + T);
  const int64_t tiles = ceil_div(most, kKeys);
  const int dt = kv_tile_dim(c.d), wide = 4 * kv_wide(dt);
  p.waves = 4;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({kv_resident(dt) * cus / grid, tiles / (2 * p.waves), 64}));
  // A workgroup that fills a CU, and no join: where most CUs have one (256 heads' single rows,
  // d 64, 500 tokens: 10.2 us, in parts 10.8; 4000: 23.1 and 26.0; d 128, 16000: 184 and 187),
  // and for texts of two tiles a wave, where a second launch costs more (6 heads, 1000 tokens:
  // 10.1 us a call and 11.6, though 9.7 and 9.2 from a graph).  Else in parts (48 heads, d 128,
  // 4000 tokens: 17.4 us, whole 30.7).
  if (p.splits > 1 && grid <= cus && tiles <= (4 * grid >= 3 * cus ? 16 : 2) * wide) {
    p.waves = wide;
    p.splits = 1;
  }
  return p;
}

int kv_attn_check(const aar_kv_cache* c, int64_t H, int64_t T, int64_t window, int64_t sinks) {
  const int rc = kv_check(c);
  if (rc != AAR_OK) return rc;
  if (H <= 0 || H % c->kv_heads != 0 || T < 0 || window < 1 || sinks < 0) return AAR_EINVAL;
  if (T > (1 << 24) || H > (1 << 24) || H / c->kv_heads * T > (1 << 24)) return AAR_EUNSUPPORTED;
  // a dispatch holds its work items in 32 bits: 256 for a block of rows
  const int64_t blocks = ceil_div(H / c->kv_heads * T, kRows) * c->sequences * c->kv_heads;
  if (blocks >= (int64_t(1) << 22)) return AAR_EUNSUPPORTED;
  return AAR_OK;
}

size_t kv_part_rows(const aar_kv_cache& c, const KvPlan& p) {
  return (size_t)p.blocks * c.sequences * c.kv_heads * p.splits * kRows;
}

template <int DT, bool VEC>
int launch_attn(const KvPages& c, const KvAttn& a, int waves, hipStream_t st) {
  constexpr int kMost = 4 * kv_wide(DT);
  const int64_t BH = (int64_t)c.B * c.Hkv;
  const dim3 grid((unsigned)(BH * a.blocks * a.splits)), block(waves * kWave);
  if (waves == kMost) kv_attn_kernel<DT, kMost, VEC><<<grid, block, 0, st>>>(c, a);
  else kv_attn_kernel<DT, 4, VEC><<<grid, block, 0, st>>>(c, a);
  const int rc = launch_status();
  if (rc != AAR_OK || a.splits == 1) return rc;
  const int64_t units = BH * a.R * (DT / 4);
  kv_attn_join_kernel<DT, VEC><<<dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, st>>>(c, a);
  return launch_status();
}

template <bool VEC>
int kv_attn_dims(const KvPages& c, const KvAttn& a, int waves, hipStream_t st) {
  const int dt = kv_tile_dim(c.d);
  if (dt == 32) return launch_attn<32, VEC>(c, a, waves, st);
  if (dt == 64) return launch_attn<64, VEC>(c, a, waves, st);
  return launch_attn<128, VEC>(c, a, waves, st);
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

size_t aar_kv_cache_attn_workspace_bytes(const aar_kv_cache* cache, int64_t H, int64_t T, int64_t window,
                                         int64_t sinks) {
  if (kv_attn_check(cache, H, T, window, sinks) != AAR_OK || cache->sequences == 0 || T == 0) return 0;
  const KvPlan p = kv_plan(*cache, H, T, window, sinks);
  if (p.splits == 1) return 0;
  return kv_part_rows(*cache, p) * (kv_tile_dim(cache->d) + 1) * sizeof(float);
}

int aar_kv_cache_attn_f32(const aar_kv_cache* cache, const float* q, float* o, const int64_t* strides,
                          const int64_t* lens, const int64_t* new_lens, int64_t H, int64_t T, int64_t window,
                          int64_t sinks, float scale, void* workspace, size_t workspace_bytes, int* err, void* stream) {
  const int rc = kv_attn_check(cache, H, T, window, sinks);
  if (rc != AAR_OK) return rc;
  if (cache->sequences == 0 || T == 0) return AAR_OK;
  if (!q || !o || !strides || !lens || (cache->table_width > 0 && !cache->table) ||
      (cache->n_pages > 0 && (!cache->pages || !cache->scales))) {
    return AAR_EINVAL;
  }
  if (!aligned16(cache->pages)) return AAR_EINVAL;
  const KvPages c = kv_pages(cache);
  const KvPlan p = kv_plan(*cache, H, T, window, sinks);
  KvAttn a{};
  a.q = FaIn{q, strides[0], strides[1], strides[2]};
  a.o = FaOut{o, strides[3], strides[4], strides[5]};
  a.lens = lens;
  a.new_lens = new_lens;
  a.err = err;
  a.T = (int)T;
  a.G = (int)(H / cache->kv_heads);
  a.R = a.G * a.T;
  a.window = (int)std::min(window, kKvMost);
  a.sinks = (int)std::min(sinks, kKvMost);
  a.blocks = (int)p.blocks;
  a.splits = p.splits;
  a.scale_log2 = scale * kLog2e;
  if (p.splits > 1) {
    const size_t need = aar_kv_cache_attn_workspace_bytes(cache, H, T, window, sinks);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return AAR_EWORKSPACE;
    a.part_o = static_cast<float*>(workspace);
    a.part_l = a.part_o + kv_part_rows(*cache, p) * kv_tile_dim(cache->d);
  }
  bool vec = c.d % 4 == 0 && aligned16(q) && aligned16(o);
  for (int i = 0; i < 6; ++i) vec = vec && strides[i] % 4 == 0;
  return vec ? kv_attn_dims<true>(c, a, p.waves, as_stream(stream))
             : kv_attn_dims<false>(c, a, p.waves, as_stream(stream));
}

}  // extern "C"
