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
constexpr int kWaves = 4;

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

// (a, b) in two fp16 parts, a pair a word.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  const f16x2 x = __builtin_convertvector(f32x2{a, b}, f16x2);
  hi = __builtin_bit_cast(uint32_t, x);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a - (float)x[0], b - (float)x[1]}, f16x2));
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

// What a wave reads of a tile: rows of keys 16 bytes a lane, columns of values 8.
template <int DT>
struct Tile {
  static constexpr int NK = (DT + 63) / 64, NB = DT / 16;
  u32x4 k[2][NK];
  u32x2 v[NB];
  __device__ __forceinline__ void load(const uint8_t* keys, const uint8_t* values, int dp, int lane) {
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int c = 0; c < NK; ++c) {
        k[n][c] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
        if (64 * c + 16 * g < dp) k[n][c] = *reinterpret_cast<const u32x4*>(keys + (16 * n + r) * dp + 64 * c + 16 * g);
      }
    }
    const int at = 8 * ((g & 1) << 1 | g >> 1);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      if (16 * b < dp) v[b] = *reinterpret_cast<const u32x2*>(values + (16 * b + r) * 32 + at);
  }
};

// A workgroup takes 16 NC query rows of a key/value head (the rows of the G query
// heads that share it, one list) and a range of their tiles; its waves take every
// fourth tile, each with an online softmax of its own, and meet at the end.
template <int DT, int NC, bool VEC>
__global__ void __launch_bounds__(kWaves * kWave)
kv_attn_kernel(const KvPages c, const KvAttn a) {
  constexpr int NK = Tile<DT>::NK, NB = Tile<DT>::NB, NP = 2 * NK;  // NP: 32-column steps of a score
  __shared__ f32x4 so[kWaves / 2][NC][NB][kWave];
  __shared__ float sm[kWaves / 2][NC][kWave], sl[kWaves / 2][NC][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int BH = c.B * c.Hkv, bh = blockIdx.x % BH, b = bh / c.Hkv, hk = bh % c.Hkv;
  const int rest = blockIdx.x / BH, part = rest % a.splits, block = rest / a.splits;
  const KvSpan span = kv_span(c, a.lens, a.new_lens, a.T, b);
  if (!span.ok && a.err) *a.err = 1;
  const int n = span.len - span.first, row0 = block * 16 * NC, row1 = min(a.R, row0 + 16 * NC) - 1;

  // the tokens that the block's rows belong to
  int t0 = 0, t1 = a.T - 1;
  if (row0 / a.T == row1 / a.T) {
    t0 = row0 % a.T;
    t1 = row1 % a.T;
  }
  t1 = min(t1, n - 1);
  const Tiles tiles(a, span.first, t0, t1);
  const int i0 = (int)((int64_t)tiles.count * part / a.splits), i1 = (int)((int64_t)tiles.count * (part + 1) / a.splits);

  // q in parts, and each row's position (-1: a row that is none) and factor
  u32x4 qp[NC][NP][2];
  int pos[NC], ex[NC];
#pragma unroll
  for (int w = 0; w < NC; ++w) {
    const int row = row0 + 16 * w + r, head = row / a.T, t = row - head * a.T;
    const bool real = row < a.R && t < n;
    pos[w] = real ? span.first + t : -1;
    const float* q = a.q.p + (int64_t)b * a.q.sb + ((int64_t)hk * a.G + head) * a.q.sh + (int64_t)t * a.q.st;
    f32x4 x[NP][2];
    float top = 0.f;
#pragma unroll
    for (int s = 0; s < NP; ++s) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int col = 64 * (s >> 1) + 16 * g + 8 * (s & 1) + 4 * p;
        x[s][p] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (real && col < c.d) x[s][p] = load4<VEC>(q + col, c.d - col);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[s][p][e]));
      }
    }
    top = row_max(top);
    ex[w] = top > 0.f ? 14 - ilogbf(top) - 1 : 0;
#pragma unroll
    for (int s = 0; s < NP; ++s) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t hi, lo;
        split_pair(ldexpf(x[s][p >> 1][2 * (p & 1)], ex[w]), ldexpf(x[s][p >> 1][2 * (p & 1) + 1], ex[w]), hi, lo);
        qp[w][s][0][p] = hi;
        qp[w][s][1][p] = lo;
      }
    }
  }

  f32x4 o[NC][NB];
  float m[NC], l[NC];
#pragma unroll
  for (int w = 0; w < NC; ++w) {
    m[w] = -INFINITY;
    l[w] = 0.f;
#pragma unroll
    for (int d = 0; d < NB; ++d) o[w][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](const Tile<DT>& x, int key0, float sk, float sv) {
    f32x4 s[NC][2];
#pragma unroll
    for (int w = 0; w < NC; ++w) s[w][0] = s[w][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 k = halves_of(x.k[h][p >> 1][2 * (p & 1)], x.k[h][p >> 1][2 * (p & 1) + 1]);
#pragma unroll
        for (int w = 0; w < NC; ++w) {
          s[w][h] = mfma16(k, qp[w][p][1], s[w][h]);
          s[w][h] = mfma16(k, qp[w][p][0], s[w][h]);
        }
      }
    }
    u32x4 pp[NC][2];
    float weight[NC];  // of the values: 0 where the row sees none of the tile
    const bool all = key0 + kKeys - 1 <= span.first + t0 && (key0 > span.first + t1 - a.window || key0 + kKeys <= a.sinks);
#pragma unroll
    for (int w = 0; w < NC; ++w) {
      const float f = ldexpf(sk * a.scale_log2, -ex[w]);
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = s[w][h][e] * f;
          if (!all) {
            const int key = key0 + 16 * h + 4 * g + e;
            const bool sees = key <= pos[w] && (key > pos[w] - a.window || key < a.sinks);
            v = sees ? v : -INFINITY;
          }
          s[w][h][e] = v;
          mx = fmaxf(mx, v);
        }
      }
      // a scale that is not finite reaches the rows that see it alone
      weight[w] = all || row_max(mx) != -INFINITY ? sv : 0.f;
      if (__any(mx > m[w] + 4.f)) {  // the maximum follows only where P would pass 2^4
        mx = fmaxf(row_max(mx), m[w]);
        const float alpha = mx > m[w] ? exp2f(m[w] - mx) : 1.f;
        m[w] = mx;
        l[w] *= alpha;
#pragma unroll
        for (int d = 0; d < NB; ++d) o[w][d] *= alpha;
      }
      const float mu = m[w] == -INFINITY ? -11.f : m[w] - 11.f;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[w][h][e] = fast_exp2(s[w][h][e] - mu);
          sum += s[w][h][e];
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t hi, lo;
          split_pair(s[w][h][2 * e], s[w][h][2 * e + 1], hi, lo);
          pp[w][0][2 * h + e] = hi;
          pp[w][1][2 * h + e] = lo;
        }
      }
      l[w] += sum;
    }
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      if (16 * d >= c.dp) continue;
      const u32x4 v = halves_of(x.v[d][0], x.v[d][1]);
#pragma unroll
      for (int w = 0; w < NC; ++w) {
        f32x4 t = mfma16(v, pp[w][1], f32x4{0.f, 0.f, 0.f, 0.f});
        t = mfma16(v, pp[w][0], t);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[w][d][e] = fmaf(weight[w], t[e], o[w][d][e]);
      }
    }
  };

  // 64 of the wave's tiles at a time: a lane looks one up
  for (int base = i0 + wave; base < i1; base += kWaves * kWave) {
    const int mine = base + kWaves * lane;
    int key = 0;
    int64_t id = -1;
    float sk = 0.f, sv = 0.f;
    if (mine < i1) {
      key = tiles.at(mine) * kKeys;
      id = c.id(b, key >> c.shift);
      if (id < 0 && a.err) *a.err = 1;
      if (id >= 0) {
        const float* s = c.scale(id, hk);
        sk = s[0];
        sv = s[1];
      }
    }
    const uint8_t* at = id < 0 ? nullptr : c.head(id, hk, 0) + (key & (c.page() - 1)) * c.dp;
    const uint64_t live = __ballot(id >= 0);
    const int count = min(kWave, (i1 - base + kWaves - 1) / kWaves);
    Tile<DT> x[2];
    auto fetch = [&](int i, Tile<DT>& t) {
      if (i >= count || !(live >> i & 1)) return;
      const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)(uintptr_t)at, i);
      const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)((uintptr_t)at >> 32), i);
      const uint8_t* p = reinterpret_cast<const uint8_t*>((uint64_t)hi << 32 | lo);
      t.load(p, p + c.half(), c.dp, lane);
    };
    auto step = [&](int i, const Tile<DT>& t) {
      if (i >= count || !(live >> i & 1)) return;
      compute(t, __builtin_amdgcn_readlane(key, i), __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sk), i)),
              __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sv), i)));
    };
    fetch(0, x[0]);
    for (int i = 0; i < count; i += 2) {
      fetch(i + 1, x[1]);
      step(i, x[0]);
      fetch(i + 2, x[0]);
      step(i + 1, x[1]);
    }
  }

  // the waves' sums meet, half of them at a time
#pragma unroll
  for (int w = 0; w < NC; ++w) l[w] = row_sum(l[w]);
#pragma unroll
  for (int half = kWaves / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int w = 0; w < NC; ++w) {
        sm[wave - half][w][lane] = m[w];
        sl[wave - half][w][lane] = l[w];
#pragma unroll
        for (int d = 0; d < NB; ++d) so[wave - half][w][d][lane] = o[w][d];
      }
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int w = 0; w < NC; ++w) {
        const float other = sm[wave][w][lane], mx = fmaxf(m[w], other), mu = mx == -INFINITY ? 0.f : mx;
        const float f = exp2f(m[w] - mu), h = exp2f(other - mu);
        m[w] = mx;
        l[w] = l[w] * f + sl[wave][w][lane] * h;
#pragma unroll
        for (int d = 0; d < NB; ++d) {
          const f32x4 x = so[wave][w][d][lane];
#pragma unroll
          for (int e = 0; e < 4; ++e) o[w][d][e] = o[w][d][e] * f + x[e] * h;
        }
      }
    }
    __syncthreads();
  }
  if (wave != 0) return;
#pragma unroll
  for (int w = 0; w < NC; ++w) {
    const int in = 16 * w + r, row = row0 + in, head = row / a.T, t = row - head * a.T;
    if (row >= a.R) continue;
    const bool none = pos[w] < 0 || l[w] == 0.f;  // a row that sees nothing, or is none
    const float inv = 1.0f / l[w];
    const int64_t at = (((int64_t)block * BH + bh) * a.splits + part) * (16 * NC) + in;
    float* orow = a.splits > 1 ? a.part_o + at * DT
                               : a.o.p + (int64_t)b * a.o.sb + ((int64_t)hk * a.G + head) * a.o.sh + (int64_t)t * a.o.st;
#pragma unroll
    for (int d = 0; d < NB; ++d) {
      const int col = 16 * d + 4 * g;
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = none ? 0.f : o[w][d][e] * inv;
      if (a.splits > 1) *reinterpret_cast<f32x4*>(orow + col) = v;
      else if (col < c.d) store4<VEC>(orow + col, v, c.d - col);
    }
    if (a.splits > 1 && g == 0) a.part_l[at] = none ? -INFINITY : m[w] + log2f(l[w]);
  }
}

// The parts of every query row, as cross attention's: with L_p = m_p + log2(l_p),
//   O = sum_p 2^(L_p - M) O_p / sum_p 2^(L_p - M),  M the largest L_p.
template <int DT, int NC, bool VEC>
__global__ void __launch_bounds__(256)
kv_attn_join_kernel(const KvPages c, const KvAttn a) {
  constexpr int kLanes = DT / 4, kRows = 16 * NC;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, item = u / kLanes;
  const int BH = c.B * c.Hkv, bh = (int)(item / a.R), row = (int)(item % a.R), col = (int)(u % kLanes) * 4;
  if (bh >= BH) return;
  const int64_t at = ((int64_t)(row / kRows) * BH + bh) * a.splits * kRows + row % kRows;
  float mx = -INFINITY;
  for (int p = 0; p < a.splits; ++p) mx = fmaxf(mx, a.part_l[at + p * kRows]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float w = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    const float f = exp2f(a.part_l[at + p * kRows] - mu);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (at + p * kRows) * DT + col);
    w += f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += f * x[e];
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

// 16-row groups of a workgroup: as many as its rows fill.
int kv_groups(int64_t R, int64_t d) { return R <= 16 ? 1 : (R <= 32 || d > 64 ? 2 : 4); }

struct KvPlan {
  int groups, splits;
  int64_t blocks;
};

KvPlan kv_plan(const aar_kv_cache& c, int64_t H, int64_t T, int64_t window, int64_t sinks) {
  const int64_t R = H / c.kv_heads * T, cus = device_cu_count();
  KvPlan p;
  p.groups = kv_groups(R, c.d);
  p.blocks = ceil_div(R, 16 * p.groups);
  const int64_t grid = p.blocks * c.sequences * c.kv_heads;
  const int64_t most = std::min(c.table_width * c.page, std::min(window, kKvMost) + std::min(sinks, kKvMost) + T);
  const int64_t tiles = ceil_div(most, kKeys);
  const int64_t s = grid >= 2 * cus ? 1 : std::min(ceil_div(4 * cus, grid), tiles / (2 * kWaves));
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(s, 64));
  return p;
}

int kv_attn_check(const aar_kv_cache* c, int64_t H, int64_t T, int64_t window, int64_t sinks) {
  const int rc = kv_check(c);
  if (rc != AAR_OK) return rc;
  if (H <= 0 || H % c->kv_heads != 0 || T < 0 || window < 1 || sinks < 0) return AAR_EINVAL;
  if (T > (1 << 24) || H > (1 << 24) || H / c->kv_heads * T > (1 << 24)) return AAR_EUNSUPPORTED;
  // a dispatch holds its work items in 32 bits
  const int64_t blocks = ceil_div(H / c->kv_heads * T, 16) * c->sequences * c->kv_heads;
  if (blocks > (int64_t)UINT32_MAX / (64 * kWaves * kWave)) return AAR_EUNSUPPORTED;
  return AAR_OK;
}

size_t kv_part_rows(const aar_kv_cache& c, const KvPlan& p) {
  return (size_t)p.blocks * c.sequences * c.kv_heads * p.splits * 16 * p.groups;
}

template <int DT, int NC, bool VEC>
int launch_attn(const KvPages& c, const KvAttn& a, hipStream_t st) {
  const int64_t BH = (int64_t)c.B * c.Hkv;
  kv_attn_kernel<DT, NC, VEC><<<dim3((unsigned)(BH * a.blocks * a.splits)), dim3(kWaves * kWave), 0, st>>>(c, a);
  const int rc = launch_status();
  if (rc != AAR_OK || a.splits == 1) return rc;
  const int64_t units = BH * a.R * (DT / 4);
  kv_attn_join_kernel<DT, NC, VEC><<<dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, st>>>(c, a);
  return launch_status();
}

template <int DT, bool VEC>
int kv_attn_groups(const KvPages& c, const KvAttn& a, int groups, hipStream_t st) {
  if (groups == 1) return launch_attn<DT, 1, VEC>(c, a, st);
  if (groups == 2) return launch_attn<DT, 2, VEC>(c, a, st);
  if constexpr (DT <= 64) return launch_attn<DT, 4, VEC>(c, a, st);
  return AAR_EUNSUPPORTED;
}

template <bool VEC>
int kv_attn_dims(const KvPages& c, const KvAttn& a, int groups, hipStream_t st) {
  const int dt = kv_tile_dim(c.d);
  if (dt == 32) return kv_attn_groups<32, VEC>(c, a, groups, st);
  if (dt == 64) return kv_attn_groups<64, VEC>(c, a, groups, st);
  return kv_attn_groups<128, VEC>(c, a, groups, st);
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
  return vec ? kv_attn_dims<true>(c, a, p.groups, as_stream(stream)) : kv_attn_dims<false>(c, a, p.groups, as_stream(stream));
}

}  // extern "C"
