// Causal self attention with a sliding window and sinks, forward and backward, in fp32
// on the fp16 matrix cores (half_tile.hpp).
//
// Query i sees the keys j <= i with i - j < W or j < S; over these
//   s_ij = scale q_i . k_j,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),
//   O_i = sum_j exp(s_ij - m_i) v_j / l_i,      lse_i = m_i + ln l_i,
// and backward, with P = exp(s - lse), D_i = dO_i . O_i and dS = P (dO V^T - D):
//   dQ = scale dS K,  dV = P^T dO,  dK = scale dS^T Q, both summed over the query heads
// that share a key/value head.  Every query sees itself, so no row is empty.
//
// A block of 128 queries visits the tiles of 32 keys that any of its rows sees: the
// sinks' and the window's.  A block of 128 keys visits the queries up to W - 1 behind
// its last key, of all heads that share it; the later ones that see its sinks are visited
// for the sinks' tiles alone, in parts that are summed at the end.
//
// Bound by the matrix unit for long windows: 24 heads on 8, 16384 tokens, window 1024, d 64:
// forward 351 us (at 880 TFLOP/s of fp16 products; a large library product reaches 1095),
// dQ 567 (850), dK and dV 829 (840), where the chip's clock falls to 1.6-1.8 GHz.  Short
// texts are bound by the bytes and by a wave's chain of tiles (a tile some 1 us forward, 2 for
// dK and dV): 384 heads, 256 tokens, window 128: 36, 52 and 60 us for 100, 150 and 150 MB.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "common.hpp"
#include "flash_tile.hpp"
#include "half_tile.hpp"

namespace aar {
namespace {

struct WaArgs {
  FaIn q, k, v, o_in, dout;
  FaOut o, dq, dk, dv;
  float* lse;                // [B * H][T]
  char *kv_img, *qd_img;     // [B * Hkv][tiles] pairs of K's and V's planes, [B * H][tiles] of Q's and dO's
  float *l2, *D;             // [B * H][32 * tiles] lse in log2 (+inf past T) and dO . O of every query row
  float *dk_part, *dv_part;  // [B * Hkv][sink_tiles][far_parts][32][DP] sums of the sinks' far queries
  int T, d, H, G, Hkv, BH, BHkv;  // BH = B * H query heads, BHkv = B * Hkv
  int W, S, tiles;                // tiles of 32 rows
  bool whole;                     // a head's tiles fit in LDS
  int turns;                      // workgroups that take its waves in turn, of 4
  int sink_tiles, far_parts, far_chunk;  // dK/dV: key tiles that hold sinks, parts of their far queries (0: none), tiles of one
  float scale, scale_log2;
};

__device__ __forceinline__ bool wa_sees(const WaArgs& a, int i, int j) { return j <= i && (i - j < a.W || j < a.S); }

// Whether every, or any, of the queries [i, i + 32) sees all of the keys, or any, [j, j + 32).
__device__ __forceinline__ bool wa_all(const WaArgs& a, int i, int j) {
  return j + kTile - 1 <= i && (i + kTile - 1 - j < a.W || j + kTile <= a.S);
}
__device__ __forceinline__ bool wa_any(const WaArgs& a, int i, int j) {
  return j <= i + kTile - 1 && (i - (j + kTile - 1) < a.W || j < a.S);
}

// What a lane sees of a tile as bits, an accumulator's row (its offset without the lane's
// half) a bit: two instructions an element then hide what it does not see, where comparing
// takes five and as many on masks of lanes.
__device__ __forceinline__ uint32_t bits_below(int n) {
  n = min(max(n, 0), 32);
  return n == 32 ? 0xffffffffu : (1u << n) - 1;
}
__device__ __forceinline__ uint32_t keys_seen(const WaArgs& a, int i, int j0) {  // of keys from j0 on, by query i
  return bits_below(i + 1 - j0) & (~bits_below(i - a.W + 1 - j0) | bits_below(a.S - j0));
}
__device__ __forceinline__ uint32_t queries_that_see(const WaArgs& a, int i0, int j) {  // from i0 on, key j
  return ~bits_below(j - i0) & (j < a.S ? 0xffffffffu : bits_below(j + a.W - i0));
}
// All bits set where element r of an accumulator is seen.
__device__ __forceinline__ uint32_t seen(uint32_t bits, int r) { return (uint32_t)((int)(bits << (31 - acc_row(r, 0))) >> 31); }

// The key tiles of queries [q0, q1]: sinks' tiles, then the window's.
struct WaTiles {
  int sinks, near, count;
  __device__ __forceinline__ WaTiles(const WaArgs& a, int q0, int q1) {
    near = max(0, q0 - a.W + 1) / kTile;
    sinks = min((min(a.S, a.T) + kTile - 1) / kTile, near);
    count = sinks + q1 / kTile + 1 - near;
  }
  __device__ __forceinline__ int key(int i) const { return (i < sinks ? i : near + i - sinks) * kTile; }
};

template <typename T>
__device__ __forceinline__ auto wa_head(const T& x, const WaArgs& a, int bh) {  // query head bh
  return x.p + (int64_t)(bh / a.H) * x.sb + (int64_t)(bh % a.H) * x.sh;
}
template <typename T>
__device__ __forceinline__ auto wa_kv_head(const T& x, const WaArgs& a, int bhk) {
  return x.p + (int64_t)(bhk / a.Hkv) * x.sb + (int64_t)(bhk % a.Hkv) * x.sh;
}
// The key/value head of query head bh.
__device__ __forceinline__ int wa_kv(const WaArgs& a, int bh) { return bh / a.H * a.Hkv + bh % a.H / a.G; }

// A lane's row of accumulators times f.
template <int DP, bool VEC>
__device__ __forceinline__ void wa_store(float* row, const f32x16 (&x)[DP / 32], float f, int d, int h) {
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int dd = b * 32 + 8 * g + 4 * h;
      if (dd >= d) continue;
      const f32x4 v = {x[b][4 * g] * f, x[b][4 * g + 1] * f, x[b][4 * g + 2] * f, x[b][4 * g + 3] * f};
      store4<VEC>(row + dd, v, d - dd);
    }
  }
}

// A tile's exponent, by which its planes are scaled: half_exponent's of its largest element,
// the lowest bit set where the planes do not hold it (elements that are not finite or
// out of range, or rows whose largest elements are more than 2^16 apart: parts are off by up
// to 2^-38 of the tile's largest element, which is then no more than 2^-22 of a row's).
__device__ __forceinline__ uint32_t top_bits(uint32_t t) { return t & ~1u; }
// log2 of row_factor: 2^14 over the scale.
__device__ __forceinline__ int top_log(uint32_t t) { return (int)(t >> 23) - 126; }
// It travels with the planes, in the spare bytes of their first row: a load of its own
// would wait for the DMAs sent before it.
template <int DP>
__device__ __forceinline__ uint32_t top_of(const char* planes) {
  return __builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t*>(planes + 2 * DP));
}

// Scale of a tile's planes from the bits of its rows' largest elements: `hi` the most of
// them, `lo` the least of those that are not 0.  Sets the lowest bit where these do not
// hold the tile.
__device__ __forceinline__ uint32_t tile_top(uint32_t hi, uint32_t lo) {
  bool bad = false;
  const uint32_t ex = half_exponent(hi, bad);
  return ex | (bad || (hi != 0 && (lo >> 23) + 16 < (hi >> 23)) ? 1u : 0u);
}

// The planes of a tile's 32 rows of K or V, once for all the blocks that read them, as the
// matrix passes have them in LDS: these then move by DMA alone, and their factors are a
// tile's.  Bound by the bytes.
template <int DP, bool VEC>
__global__ void __launch_bounds__(kFaThreads)
window_split_kernel(const WaArgs a) {
  using Tile = HalfTile<DP>;
  __shared__ uint32_t most[4], least[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int second = blockIdx.x & 1, at = blockIdx.x >> 1, bhk = at / a.tiles, row0 = at % a.tiles * kTile;
  const FaIn& x = second ? a.v : a.k;
  Tile t;
  t.template load<VEC>(wa_kv_head(x, a, bhk) + (int64_t)row0 * x.st, x.st, a.T - row0, a.d,
                       typename Tile::Place(x.st, a.d, tid));

  // the largest element of the tile and the least of its rows' (as bits, NaN the largest)
  uint32_t hi = 0, lo = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < Tile::kPer; ++i) {
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = nan_max(top, fabsf(t.f[i][g][e]));
    const uint32_t row = row_top<Tile::kOcts>(__float_as_uint(top) & 0x7fffffffu);
    hi = max(hi, row);
    if (row != 0) lo = min(lo, row);
  }
#pragma unroll
  for (int o = 32; o >= 8; o /= 2) {
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, kWave));
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, kWave));
  }
  if (lane == 0) {
    most[wave] = hi;
    least[wave] = lo;
  }
  __syncthreads();
  const uint32_t top = tile_top(max(max(most[0], most[1]), max(most[2], most[3])),
                                min(min(least[0], least[1]), min(least[2], least[3])));
  char* img = a.kv_img + (int64_t)blockIdx.x * Tile::kBytes;
  if (tid == 0) *reinterpret_cast<uint32_t*>(img + 2 * DP) = top;
  const float m = half_scale(top_bits(top));
#pragma unroll
  for (int i = 0; i < Tile::kPer; ++i) {
    u32x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t y, z;
      half_split_pair(t.f[i][e >> 1][2 * (e & 1)], t.f[i][e >> 1][2 * (e & 1) + 1], m, y, z);
      h[e] = y;
      l[e] = z;
    }
    char* to = img + Tile::row(i, tid) * Tile::kRow + 2 * Tile::col(tid);
    *reinterpret_cast<u32x4*>(to) = h;
    *reinterpret_cast<u32x4*>(to + Tile::kPlane) = l;
  }
}

// A wave's 32 rows, a lane its row's octets of its half of each 16 columns (zeros past the
// text).  Its loads are all sent at once: a branch around each makes every one wait for
// the one before (8 of them 6 us).
template <int DP, bool VEC>
struct LaneRow {
  f32x4 x[DP / 16][2];
  // p: row `row0` of the head; rows from T on are not read
  __device__ __forceinline__ LaneRow(const float* p, int64_t st, int row0, int T, int d, int lr, int h) {
    const __amdgpu_buffer_rsrc_t b = row_buffer(p, kNowhere - 1);
    const uint32_t at = (uint32_t)lr * (uint32_t)st * 4u;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int dd = 16 * c + 8 * h + 4 * g;
        const uint32_t off = row0 + lr < T && dd < d ? at + 4u * dd : kNowhere;
        x[c][g] = VEC ? buffer_load4(b, off) : buffer_load1x4(b, off, d - dd);
      }
    }
  }
  __device__ __forceinline__ float half(float f, u32x4 (&out)[DP / 16][2], bool& bad) {  // half_row's, of f times the row
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
      for (int g = 0; g < 2; ++g) x[c][g] *= f;
    }
    return half_row<DP>(x, out, bad);
  }
  __device__ __forceinline__ float dot(const LaneRow& y) const {  // of the lane's octets
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(x[c][g][e], y.x[c][g][e], s);
      }
    }
    return s;
  }
};

// A wave's 32 rows in parts of a tile's scale: into registers, and as planes to `img` (HBM
// or LDS; null: not).  Returns the tile's exponent.
template <int DP, bool VEC>
__device__ __forceinline__ uint32_t split_rows(const LaneRow<DP, VEC>& rows, int lr, int h, u32x4 (&out)[DP / 16][2], char* img) {
  const auto& x = rows.x;
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int e = 0; e < 4; ++e) top = nan_max(top, fabsf(x[c][g][e]));
    }
  }
  uint32_t row = __float_as_uint(top) & 0x7fffffffu;
  row = max(row, (uint32_t)__shfl_xor((int)row, 32, kWave));
  uint32_t hi = row, lo = row != 0 ? row : 0xffffffffu;
#pragma unroll
  for (int o = 16; o > 0; o /= 2) {
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, kWave));
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, kWave));
  }
  const uint32_t t = tile_top(hi, lo);
  const float m = half_scale(top_bits(t));
  if (img && lr == 0 && h == 0) *reinterpret_cast<uint32_t*>(img + 2 * DP) = t;
  char* to = img + lr * HalfTile<DP>::kRow + 16 * h;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t y, z;
      half_split_pair(x[c][e >> 1][2 * (e & 1)], x[c][e >> 1][2 * (e & 1) + 1], m, y, z);
      out[c][0][e] = y;
      out[c][1][e] = z;
    }
    if (!img) continue;
    *reinterpret_cast<u32x4*>(to + 32 * c) = out[c][0];
    *reinterpret_cast<u32x4*>(to + 32 * c + HalfTile<DP>::kPlane) = out[c][1];
  }
  return t;
}

// A pair of planes from HBM into LDS: 1024 bytes a wave and DMA, as many DMAs for every
// wave (the last ones of some move the same bytes again).
template <int DP, int WAVES>
constexpr int kStageDmas = (2 * HalfTile<DP>::kBytes / 1024 + WAVES - 1) / WAVES;
template <int DP, int WAVES>
__device__ __forceinline__ void stage_pair(const char* src, char* lds, int wave, int lane) {
  constexpr int n = 2 * HalfTile<DP>::kBytes / 1024;
  static_assert(n * 1024 == 2 * HalfTile<DP>::kBytes, "whole DMAs");
#pragma unroll
  for (int k = 0; k < kStageDmas<DP, WAVES>; ++k) {
    const int i = min(wave + WAVES * k, n - 1);
    dma16_untracked_s(lane * 16 + i * 1024, src, (lds_void_t*)(lds + i * 1024));
  }
}

// Texts of up to TILES tiles are kept in LDS whole: a workgroup takes a head, a wave splits
// a tile of K and of V (of Q and of dO) straight into LDS, and then its own 32 rows need
// no barrier, no planes in HBM and no other workgroup's.  TILES = 0: longer texts.
// With gradients, 384 heads of d 64: 128 tokens 89 us from HBM's planes and 65 so, 256 tokens
// 179 and 146; d 128, 64 tokens 102 and 80, 128 tokens 167 and 153 (forward 33 and 34).  The
// other side are few key/value heads of many query heads each, which dK and dV take in turn
// (16 of 6, 256 tokens: 167 and 180).
// Where half the CUs would have no head, two workgroups take one: both have its tiles, the
// first the rows of waves 0 to 3 and the second those of waves 4 to 7, so that a SIMD has one
// (6 heads, 200 tokens: 54.5 and 52.0 us; 96 heads, 256 tokens: 70.1 and 68.4).
constexpr int wa_whole(int dp) { return dp == 64 ? 8 : 4; }
constexpr int wa_threads(int tiles) { return tiles ? tiles * kWave : kFaThreads; }

// Until the next of a longer text's tiles has arrived, in the other one of two buffers, and
// every wave is done with the tile before.  More buffers where a CU has one workgroup gave
// nothing (6 heads, 4096 tokens, window 1024, d 64, with gradients: 210 us with two, 217 with
// seven).
__device__ __forceinline__ void ring_next() {
  wait_vm_lgkm0<0>();
  ring_barrier();
}

// Forward.  P is formed as 2^(s + v - R + 11), with v the exponent of the tile's values and
// R, the row's, such that it stays below 2^15: the largest s + v so far, followed only when
// it is passed by 2^4, so O is rarely rescaled.  So O is sum P V 2^(25 - R), and l is kept
// as l 2^(-R - 29).
template <int DP, bool VEC, int TILES>
__global__ void __launch_bounds__(wa_threads(TILES), TILES ? (DP == 64 ? 2 : 1) : (DP == 64 ? 3 : 2))
window_fwd_kernel(const WaArgs a) {
  using Tile = HalfTile<DP>;
  constexpr int NB = DP / 32;
  __shared__ __attribute__((aligned(16))) char kv[TILES ? TILES : 2][2 * Tile::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, turn = blockIdx.x / a.BH, bhk = wa_kv(a, bh);
  // the text's end first: the first rows' lists are short, and fill the end of the grid (64
  // heads on 16, 1777 tokens, d 128, causal: 206 us in the text's order, 186 so)
  const int q0 = TILES ? 0 : (a.tiles - 1) / 4 * kBlock - turn * kBlock, w0 = q0 + wave * kTile, qi = w0 + lr;  // this lane's row
  const int wr = min(w0, a.T - 1);  // a row that is there
  auto rows_of = [&](const FaIn& x, const float* head) {
    return LaneRow<DP, VEC>(head + (int64_t)wr * x.st, x.st, w0, a.T, a.d, lr, h);
  };
  const WaTiles tiles(a, TILES ? w0 : q0, min(TILES ? w0 + kTile : q0 + kBlock, a.T) - 1);
  const char* img = a.kv_img + (int64_t)bhk * a.tiles * 2 * Tile::kBytes;
  auto stage = [&](int t, int buf) {
    stage_pair<DP, 4>(img + (int64_t)(tiles.key(t) / kTile) * 2 * Tile::kBytes, kv[buf], wave, lane);
  };
  if (!TILES) stage(0, 0);

  LaneRow<DP, VEC> row = rows_of(a.q, wa_head(a.q, a, bh));
  u32x4 qp[DP / 16][2];
  if (TILES) {
    const LaneRow<DP, VEC> k = rows_of(a.k, wa_kv_head(a.k, a, bhk)), v = rows_of(a.v, wa_kv_head(a.v, a, bhk));
    split_rows<DP, VEC>(k, lr, h, qp, kv[wave]);
    split_rows<DP, VEC>(v, lr, h, qp, kv[wave] + Tile::kBytes);
  }
  bool row_bad = false;
  uint32_t held = 0;  // the lowest bit: a tile that is not
  const float qf = row.half(a.scale_log2, qp, row_bad);
  if (TILES) {
    __syncthreads();
    if (a.turns > 1 && wave / 4 != turn) return;
  }
  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = zero16();
  float R = -INFINITY, l = 0.f, one = 1.f;
  asm("" : "+v"(one));

  auto follow = [&](float mx, float slack) {
    if (!__any(mx > R + slack)) return;
    mx = half_swap_max(mx);
    const bool move = mx > R + slack;
    const float alpha = move ? fast_exp2(R - mx) : 1.f;
    if (move) R = mx;
    l *= alpha;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
    }
  };
  auto hide = [&](f32x16& s, int kv0) {
    if (wa_all(a, w0, kv0)) return;
    const uint32_t bits = keys_seen(a, qi, kv0 + 4 * h), none = __float_as_uint(-INFINITY);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t m = seen(bits, r);
      s[r] = __uint_as_float((__float_as_uint(s[r]) & m) | (none & ~m));
    }
  };

  for (int t = 0, buf = 1; t < tiles.count; ++t) {
    const int kv0 = tiles.key(t);
    if (TILES) {
      buf = kv0 / kTile;
    } else {
      buf ^= 1;
      ring_next();
      if (t + 1 < tiles.count) stage(t + 1, buf ^ 1);
    }
    if (w0 >= a.T || !wa_any(a, w0, kv0)) continue;
    const uint32_t kt = top_of<DP>(kv[buf]), vt = top_of<DP>(kv[buf] + Tile::kBytes);
    held |= kt | vt;
    f32x16 s = half_rows<DP>(kv[buf], qp, lr, h);
    hide(s, kv0);
    const float cs = qf * row_factor(top_bits(kt)), vl = (float)top_log(vt);
    float mx = -INFINITY, ps = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    follow(fmaf(mx, cs, vl), 4.f);
    const float by = R == -INFINITY ? 0.f : vl - R + 11.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(fmaf(s[r], cs, by));
      ps += s[r];
    }
    l = fmaf(ps, pow2(-top_log(vt) - 40), l);
    half_cols<DP, true>(kv[buf] + Tile::kBytes, s, one, 0, lane, o);
    half_cols<DP, true>(kv[buf] + Tile::kBytes, s, one, 1, lane, o);
  }
  l = half_swap_sum(l);
  float f = 0x1p-54f / l, lse = log2f(l) + R + 29.f;

  if (w0 < a.T && __any(row_bad || (held & 1))) {
    const float* __restrict__ K = wa_kv_head(a.k, a, bhk);
    const float* __restrict__ V = wa_kv_head(a.v, a, bhk);
    const float* Q = qi < a.T ? wa_head(a.q, a, bh) + (int64_t)qi * a.q.st : nullptr;
    R = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = zero16();
    for (int t = 0; t < tiles.count; ++t) {
      const int kv0 = tiles.key(t);
      if (!wa_any(a, w0, kv0)) continue;
      f32x16 s = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d;
        s = mfma32(in && kv0 + lr < a.T ? K[(int64_t)(kv0 + lr) * a.k.st + c + h] : 0.f,
                   in && Q ? Q[c + h] * a.scale_log2 : 0.f, s);
      }
      hide(s, kv0);
      float mx = -INFINITY, ps = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
      follow(mx, 0.f);
      const float mu = R == -INFINITY ? 0.f : R;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = fast_exp2(s[r] - mu);
        ps += s[r];
      }
      l += half_swap_sum(ps);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int col = b * 32 + lr;
#pragma unroll
        for (int st = 0; st < 16; ++st) {
          const int row = kv0 + acc_row(st, h);
          o[b] = mfma32(row < a.T && col < a.d ? finite(V[(int64_t)row * a.v.st + col]) : 0.f, s[st], o[b]);
        }
      }
      add_not_finite(V, a.v.st, kv0, a.T, a.d, s, [&](int j) { return wa_sees(a, qi, j); }, o);
    }
    f = 1.0f / l;
    lse = log2f(l) + R;
  }
  if (qi >= a.T) return;
  wa_store<DP, VEC>(wa_head(a.o, a, bh) + (int64_t)qi * a.o.st, o, f, a.d, h);
  if (h == 0) a.lse[(int64_t)bh * a.T + qi] = lse * kLn2;
}

// dQ, and what dK's and dV's pass reads of a query row: the planes of Q and dO, D and lse.
template <int DP, bool VEC, int TILES>
__global__ void __launch_bounds__(wa_threads(TILES), DP == 64 ? 2 : 1)
window_bwd_dq_kernel(const WaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char kv[TILES ? TILES : 2][2 * Tile::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, turn = blockIdx.x / a.BH, bhk = wa_kv(a, bh);
  // the text's end first, as forward
  const int q0 = TILES ? 0 : (a.tiles - 1) / 4 * kBlock - turn * kBlock, w0 = q0 + wave * kTile, qi = w0 + lr;
  const bool row_ok = qi < a.T;
  const int wr = min(w0, a.T - 1);  // a row that is there
  auto rows_of = [&](const FaIn& x, const float* head) {
    return LaneRow<DP, VEC>(head + (int64_t)wr * x.st, x.st, w0, a.T, a.d, lr, h);
  };
  const WaTiles tiles(a, TILES ? w0 : q0, min(TILES ? w0 + kTile : q0 + kBlock, a.T) - 1);
  const char* img = a.kv_img + (int64_t)bhk * a.tiles * 2 * Tile::kBytes;
  auto stage = [&](int t, int buf) {
    stage_pair<DP, 4>(img + (int64_t)(tiles.key(t) / kTile) * 2 * Tile::kBytes, kv[buf], wave, lane);
  };
  if (!TILES) stage(0, 0);

  const LaneRow<DP, VEC> q = rows_of(a.q, wa_head(a.q, a, bh));
  if (!VEC) sched_fence();  // single floats' places fill the registers: one operand's at a time
  const LaneRow<DP, VEC> dO = rows_of(a.dout, wa_head(a.dout, a, bh));
  if (!VEC) sched_fence();
  const LaneRow<DP, VEC> O = rows_of(a.o_in, wa_head(a.o_in, a, bh));
  const float lse = a.lse[(int64_t)bh * a.T + min(qi, a.T - 1)];
  u32x4 qp[DP / 16][2], dop[DP / 16][2];
  if (TILES) {
    const LaneRow<DP, VEC> k = rows_of(a.k, wa_kv_head(a.k, a, bhk)), v = rows_of(a.v, wa_kv_head(a.v, a, bhk));
    split_rows<DP, VEC>(k, lr, h, qp, kv[wave]);
    split_rows<DP, VEC>(v, lr, h, qp, kv[wave] + Tile::kBytes);
  }
  const float l2 = row_ok ? lse * kLog2e : INFINITY, dsum = half_swap_sum(dO.dot(O));
  bool row_bad = false;
  uint32_t held = 0;
  float qf = 0.f, df = 0.f;
  const bool mine = !TILES || a.turns == 1 || wave / 4 == turn;
  if (w0 < a.T && mine) {
    const int64_t tile = (int64_t)bh * a.tiles + w0 / kTile;
    if (h == 0) {
      a.D[tile * kTile + lr] = dsum;
      a.l2[tile * kTile + lr] = l2;
    }
    char* to = a.qd_img + tile * 2 * Tile::kBytes;
    const uint32_t qt = split_rows<DP, VEC>(q, lr, h, qp, TILES ? nullptr : to);
    const uint32_t ot = split_rows<DP, VEC>(dO, lr, h, dop, TILES ? nullptr : to + Tile::kBytes);
    held = qt | ot;
    qf = lane_factor(top_bits(qt)) * a.scale_log2;
    df = lane_factor(top_bits(ot));
  }
  if (TILES) {
    __syncthreads();
    if (!mine) return;
  }
  f32x16 dq[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dq[b] = zero16();
  HalfScale<NB> fit;

  auto hide = [&](f32x16& x, int kv0) {
    if (wa_all(a, w0, kv0)) return;
    const uint32_t bits = keys_seen(a, qi, kv0 + 4 * h);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = __uint_as_float(__float_as_uint(x[r]) & seen(bits, r));
  };
  for (int t = 0, buf = 1; t < tiles.count; ++t) {
    const int kv0 = tiles.key(t);
    if (TILES) {
      buf = kv0 / kTile;
    } else {
      buf ^= 1;
      ring_next();
      if (t + 1 < tiles.count) stage(t + 1, buf ^ 1);
    }
    if (w0 >= a.T || !wa_any(a, w0, kv0)) continue;
    const uint32_t kt = top_of<DP>(kv[buf]), vt = top_of<DP>(kv[buf] + Tile::kBytes);
    held |= kt | vt;
    const f32x16 s = half_rows<DP>(kv[buf], qp, lr, h);
    f32x16 dp = half_rows<DP>(kv[buf] + Tile::kBytes, dop, lr, h);
    const float kfac = row_factor(top_bits(kt)), cs = qf * kfac, cd = df * row_factor(top_bits(vt));
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) dp[r] = fast_exp2(fmaf(s[r], cs, -l2)) * fmaf(dp[r], cd, -dsum);
    hide(dp, kv0);
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dp[r]));
    fit.follow(top * kfac, dq, row_bad);
    const float f = fminf(fit.f * kfac, 0x1p126f);
    half_cols<DP>(kv[buf], dp, f, 0, lane, dq);
    half_cols<DP>(kv[buf], dp, f, 1, lane, dq);
  }
  fit.undo(dq);

  if (w0 < a.T && __any(row_bad || (held & 1))) {
    const float* __restrict__ K = wa_kv_head(a.k, a, bhk);
    const float* __restrict__ V = wa_kv_head(a.v, a, bhk);
    const float* Q = row_ok ? wa_head(a.q, a, bh) + (int64_t)qi * a.q.st : nullptr;
    const float* dO = row_ok ? wa_head(a.dout, a, bh) + (int64_t)qi * a.dout.st : nullptr;
#pragma unroll
    for (int b = 0; b < NB; ++b) dq[b] = zero16();
    for (int t = 0; t < tiles.count; ++t) {
      const int kv0 = tiles.key(t);
      if (!wa_any(a, w0, kv0)) continue;
      f32x16 s = zero16(), dp = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d, key = in && kv0 + lr < a.T;
        s = mfma32(key ? K[(int64_t)(kv0 + lr) * a.k.st + c + h] : 0.f, in && Q ? Q[c + h] * a.scale_log2 : 0.f, s);
        dp = mfma32(key ? V[(int64_t)(kv0 + lr) * a.v.st + c + h] : 0.f, in && dO ? dO[c + h] : 0.f, dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = fast_exp2(s[r] - l2) * (dp[r] - dsum);
      hide(dp, kv0);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int col = b * 32 + lr;
#pragma unroll
        for (int st = 0; st < 16; ++st) {
          const int key = kv0 + acc_row(st, h);
          dq[b] = mfma32(key < a.T && col < a.d ? finite(K[(int64_t)key * a.k.st + col]) : 0.f, dp[st], dq[b]);
        }
      }
      add_not_finite(K, a.k.st, kv0, a.T, a.d, dp, [&](int j) { return wa_sees(a, qi, j); }, dq);
    }
  }
  if (row_ok) wa_store<DP, VEC>(wa_head(a.dq, a, bh) + (int64_t)qi * a.dq.st, dq, a.scale, a.d, h);
}

// The list of query tiles of 32 WAVES keys from k0 on: `count` tiles from `first` on of
// each of the G heads that share them, items [begin, end) of it.  Four waves: a key block
// with the queries up to the last that its window reaches (all later ones if it holds
// sinks and these have no parts of their own).  One: 32 keys that hold sinks with a part of
// the far queries, those behind their block's window.
template <int WAVES>
struct WaList {
  int k0, part, first, count, begin, end;
  // wave: of a workgroup that takes a whole head, a list for each
  __device__ __forceinline__ WaList(const WaArgs& a, int item, int wave) {
    const int tile = WAVES == 4 ? 4 * item + wave : item / a.far_parts;
    part = WAVES == 4 ? 0 : item % a.far_parts;
    k0 = tile * kTile;
    // the last query that the window of a key of the block reaches
    const int64_t most = (int64_t)k0 / kBlock * kBlock + kBlock - 1 + a.W - 1;
    int last = most >= a.T ? a.T - 1 : (int)most;
    if (WAVES == 4) {
      if (k0 < a.S && a.far_parts == 0) last = a.T - 1;
      first = tile;
      count = last / kTile + 1 - first;
      begin = 0;
      end = a.G * count;
    } else {
      first = last / kTile + 1;
      count = a.tiles - first;
      begin = min(part * a.far_chunk, a.G * count);
      end = min(begin + a.far_chunk, a.G * count);
    }
  }
};

// dK and dV: a wave takes 32 keys, a lane its key, and walks its workgroup's list.
template <int DP, bool VEC, int WAVES, int TILES>
__global__ void __launch_bounds__(TILES ? wa_threads(TILES) : WAVES * kWave, DP == 64 ? 2 : 1)
window_bwd_dkdv_kernel(const WaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char qd[TILES ? TILES : 2][2 * Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float stats[TILES ? TILES : 2][2 * kTile];  // lse in log2, D
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 31, h = lane >> 5;
  const int bhk = blockIdx.x % a.BHkv, item = blockIdx.x / a.BHkv;
  const WaList<WAVES> part(a, TILES ? 0 : item, TILES ? wave : 0);
  const bool mine = !TILES || a.turns == 1 || wave / 4 == item;
  const int kw = TILES ? wave * kTile : part.k0 + wave * kTile;  // the wave's first key
  const int kj = kw + lr;
  const bool key_ok = kj < a.T;
  const int wr = min(kw, a.T - 1);  // a row that is there
  auto rows_of = [&](const FaIn& x, const float* head) {
    return LaneRow<DP, VEC>(head + (int64_t)wr * x.st, x.st, kw, a.T, a.d, lr, h);
  };
  const int head0 = bhk / a.Hkv * a.H + bhk % a.Hkv * a.G;  // the first query head
  // where item t of the list stands among all heads' tiles
  struct Place {
    int head, tile;
  };
  // (the same in all lanes, which the compiler does not see through the loop)
  auto place = [&](int head, int tile) {
    return Place{__builtin_amdgcn_readfirstlane(head), __builtin_amdgcn_readfirstlane(tile)};
  };
  auto place_of = [&](int t) { return place(head0 + t / part.count, part.first + t % part.count); };
  auto next_of = [&](Place p) {
    const bool same = p.tile + 1 < part.first + part.count;
    return place(same ? p.head : p.head + 1, same ? p.tile + 1 : part.first);
  };
  auto stage = [&](Place p, int buf) {
    const int64_t at = (int64_t)p.head * a.tiles + p.tile;
    stage_pair<DP, WAVES>(a.qd_img + at * 2 * Tile::kBytes, qd[buf], wave, lane);
    dma4_untracked((lane < kTile ? a.l2 : a.D) + at * kTile + lr, (lds_void_t*)stats[buf]);
  };
  Place here = part.begin < part.end ? place_of(part.begin) : place(head0, part.first), ahead = here;
  if (!TILES && part.begin < part.end) {
    stage(ahead, 0);
    ahead = next_of(ahead);
  }

  u32x4 kp[DP / 16][2], vp[DP / 16][2];
  bool key_bad = false;
  uint32_t held = 0;
  float kf, vf;
  {
    LaneRow<DP, VEC> k = rows_of(a.k, wa_kv_head(a.k, a, bhk)), v = rows_of(a.v, wa_kv_head(a.v, a, bhk));
    kf = k.half(a.scale_log2, kp, key_bad);
    vf = v.half(1.f, vp, key_bad);
  }
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
  HalfScale<NB> fit_k, fit_v;

  // P or dS of the queries from i0 on that do not see the lane's key
  auto hide = [&](f32x16& p, int i0) {
    if (wa_all(a, i0, kw)) return;
    const uint32_t bits = queries_that_see(a, i0 + 4 * h, kj);
#pragma unroll
    for (int r = 0; r < 16; ++r) p[r] = __uint_as_float(__float_as_uint(p[r]) & seen(bits, r));
  };
  const int heads = TILES ? a.G : 1;  // lists one after the other
  for (int g = 0; g < heads; ++g) {
  if (TILES) {
    // the head's queries; every wave is done with the head before
    u32x4 parts[DP / 16][2];
    const int bh = head0 + g;
    if (g > 0) __syncthreads();
    const float stat = (h == 0 ? a.l2 : a.D)[((int64_t)bh * a.tiles + wave) * kTile + lr];
    const LaneRow<DP, VEC> q = rows_of(a.q, wa_head(a.q, a, bh));
    if (!VEC) {  // single floats' places fill the registers: one operand's at a time
      split_rows<DP, VEC>(q, lr, h, parts, qd[wave]);
      sched_fence();
    }
    const LaneRow<DP, VEC> dO = rows_of(a.dout, wa_head(a.dout, a, bh));
    if (VEC) split_rows<DP, VEC>(q, lr, h, parts, qd[wave]);
    split_rows<DP, VEC>(dO, lr, h, parts, qd[wave] + Tile::kBytes);
    stats[wave][lane] = stat;
    __syncthreads();
    if (!mine) continue;
    here = place(bh, part.first);
  }
  for (int t = part.begin, cur = 1; t < (TILES ? part.count : part.end); ++t) {
    const int i0 = here.tile * kTile;
    here = next_of(here);
    if (TILES) {
      cur = i0 / kTile;
    } else {
      cur ^= 1;
      ring_next();
      if (t + 1 < part.end) {
        stage(ahead, cur ^ 1);
        ahead = next_of(ahead);
      }
    }
    if (kw >= a.T || !wa_any(a, i0, kw)) continue;
    const uint32_t qt = top_of<DP>(qd[cur]), ot = top_of<DP>(qd[cur] + Tile::kBytes);
    held |= qt | ot;
    const char* dos = qd[cur] + Tile::kBytes;
    const float qfac = row_factor(top_bits(qt)), ofac = row_factor(top_bits(ot)), cs = kf * qfac, cd = vf * ofac;
    f32x16 s = half_rows<DP>(qd[cur], kp, lr, h);
    sched_fence();
    float top = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 l4 = row_values(stats[cur], g, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g + e] = fast_exp2(fmaf(s[4 * g + e], cs, -l4[e]));
    }
    hide(s, i0);
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    fit_v.follow(top * ofac, dv, key_bad);
    float f = fminf(fit_v.f * ofac, 0x1p126f);
    half_cols<DP>(dos, s, f, 0, lane, dv);
    half_cols<DP>(dos, s, f, 1, lane, dv);
    f32x16 x = half_rows<DP>(dos, vp, lr, h);
    sched_fence();
    top = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 d4 = row_values(stats[cur] + kTile, g, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g + e] = s[4 * g + e] * fmaf(x[4 * g + e], cd, -d4[e]);
    }
    hide(x, i0);  // where D is not finite
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
    fit_k.follow(top * qfac, dk, key_bad);
    f = fminf(fit_k.f * qfac, 0x1p126f);
    half_cols<DP>(qd[cur], x, f, 0, lane, dk);
    half_cols<DP>(qd[cur], x, f, 1, lane, dk);
  }
  }
  if (!mine) return;
  fit_v.undo(dv);
  fit_k.undo(dk);

  if (kw < a.T && part.begin < part.end && __any(key_bad || (held & 1))) {
    const float* K = key_ok ? wa_kv_head(a.k, a, bhk) + (int64_t)kj * a.k.st : nullptr;
    const float* V = key_ok ? wa_kv_head(a.v, a, bhk) + (int64_t)kj * a.v.st : nullptr;
#pragma unroll
    for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
    for (int t = part.begin; t < part.end; ++t) {
      const Place p = place_of(t);
      const int i0 = p.tile * kTile, bh = p.head;
      if (!wa_any(a, i0, kw)) continue;
      const float* Qh = wa_head(a.q, a, bh);
      const float* dOh = wa_head(a.dout, a, bh);
      const int64_t stat = (int64_t)bh * a.tiles * kTile;
      const bool mine = i0 + lr < a.T;
      f32x16 s = zero16(), dp = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d;
        s = mfma32(in && mine ? Qh[(int64_t)(i0 + lr) * a.q.st + c + h] : 0.f, in && K ? K[c + h] * a.scale_log2 : 0.f, s);
        dp = mfma32(in && mine ? dOh[(int64_t)(i0 + lr) * a.dout.st + c + h] : 0.f, in && V ? V[c + h] : 0.f, dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = i0 + acc_row(r, h);
        const bool sees = key_ok && i < a.T && wa_sees(a, i, kj);
        s[r] = sees ? fast_exp2(s[r] - a.l2[stat + i]) : 0.f;
        dp[r] = sees ? s[r] * (dp[r] - a.D[stat + i]) : 0.f;
      }
#pragma unroll
      for (int st = 0; st < 16; ++st) {
        const int i = i0 + acc_row(st, h);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int col = b * 32 + lr;
          const bool in = i < a.T && col < a.d;
          dv[b] = mfma32(in ? finite(dOh[(int64_t)i * a.dout.st + col]) : 0.f, s[st], dv[b]);
          dk[b] = mfma32(in ? finite(Qh[(int64_t)i * a.q.st + col]) : 0.f, dp[st], dk[b]);
        }
      }
      const auto sees = [&](int i) { return wa_sees(a, i, kj); };
      add_not_finite(dOh, a.dout.st, i0, a.T, a.d, s, sees, dv);
      add_not_finite(Qh, a.q.st, i0, a.T, a.d, dp, sees, dk);
    }
  }
  if (!key_ok) return;
  if (WAVES == 4) {
    wa_store<DP, VEC>(wa_kv_head(a.dk, a, bhk) + (int64_t)kj * a.dk.st, dk, a.scale, a.d, h);
    wa_store<DP, VEC>(wa_kv_head(a.dv, a, bhk) + (int64_t)kj * a.dv.st, dv, 1.0f, a.d, h);
  } else {
    const int64_t at = (((int64_t)bhk * a.sink_tiles * a.far_parts + item) * kTile + lr) * DP;
    wa_store<DP, true>(a.dk_part + at, dk, a.scale, DP, h);
    wa_store<DP, true>(a.dv_part + at, dv, 1.0f, DP, h);
  }
}

// The sinks' dK and dV: their far queries' parts, in an order of their own, on top of the
// near ones' sums.  A workgroup takes a key, 256 / (DP / 4) groups of its threads parts in
// turn.
template <int DP, bool VEC>
__global__ void __launch_bounds__(256)
window_bwd_sum_kernel(const WaArgs a) {
  constexpr int kLanes = DP / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 sk[kGroups][kLanes], sv[kGroups][kLanes];
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c = 4 * lane;
  const int bhk = blockIdx.x / a.S, key = blockIdx.x % a.S;
  const int64_t at = (((int64_t)bhk * a.sink_tiles + key / kTile) * a.far_parts * kTile + key % kTile) * DP + c;
  f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
#pragma unroll 4
  for (int p = group; p < a.far_parts; p += kGroups) {
    dk += *reinterpret_cast<const f32x4*>(a.dk_part + at + (int64_t)p * kTile * DP);
    dv += *reinterpret_cast<const f32x4*>(a.dv_part + at + (int64_t)p * kTile * DP);
  }
  sk[group][lane] = dk;
  sv[group][lane] = dv;
  __syncthreads();
  if (group != 0 || c >= a.d) return;
  float* ok = wa_kv_head(a.dk, a, bhk) + (int64_t)key * a.dk.st + c;
  float* ov = wa_kv_head(a.dv, a, bhk) + (int64_t)key * a.dv.st + c;
  dk = load4<VEC>(ok, a.d - c);
  dv = load4<VEC>(ov, a.d - c);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    dk += sk[g][lane];
    dv += sv[g][lane];
  }
  store4<VEC>(ok, dk, a.d - c);
  store4<VEC>(ov, dv, a.d - c);
}

// ------------------------------------------------------------------ host side

int wa_dim(int64_t d) { return d <= 64 ? 64 : 128; }

int wa_check(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window, int64_t sinks) {
  if (B < 0 || H < 0 || Hkv < 0 || T < 0 || d <= 0 || d > 128 || window < 1 || sinks < 0) return AAR_EINVAL;
  if ((H == 0) != (Hkv == 0) || (H > 0 && H % Hkv != 0)) return AAR_EINVAL;
  if (B > (1 << 20) || H > (1 << 20) || T > (1 << 24)) return AAR_EUNSUPPORTED;
  // a dispatch holds its work items in 32 bits: two tiles of 256 threads for 32 keys
  if (B * H * ceil_div(T, kBlock) >= (1 << 20) || B * H * T > (int64_t)UINT32_MAX / 64) return AAR_EUNSUPPORTED;
  return AAR_OK;
}

WaArgs wa_args(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window, int64_t sinks, float scale) {
  WaArgs a{};
  a.T = (int)T;
  a.d = (int)d;
  a.H = (int)H;
  a.G = (int)(H / Hkv);
  a.Hkv = (int)Hkv;
  a.BH = (int)(B * H);
  a.BHkv = (int)(B * Hkv);
  a.W = (int)std::min(window, T);
  a.S = (int)std::min(sinks, T);
  a.tiles = (int)ceil_div(T, kTile);
  a.whole = a.tiles <= wa_whole(wa_dim(d));
  a.turns = a.whole && a.tiles > 4 && 2 * a.BH <= device_cu_count() ? 2 : 1;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  return a;
}

// Parts of the sinks' far queries: where the block that holds the first sinks would have
// a list more than twice as long as the others', for up to 64 tiles of sinks (24 heads on 8,
// 16384 tokens, window 1024, 4 sinks, with the forward: 4558 us in one list, 1581 so; 6 heads,
// 2048 tokens, window 64: 193 and 94; 600 tokens, the shortest: 86 and 84).
void wa_bwd_plan(WaArgs& a) {
  const int64_t near = std::min<int64_t>(a.T - 1, kBlock - 1 + (int64_t)a.W - 1) / kTile + 1, far = a.tiles - near;
  a.sink_tiles = (int)ceil_div(a.S, kTile);
  a.far_parts = a.far_chunk = 0;
  if (a.whole || a.sink_tiles == 0 || a.sink_tiles > 64 || far <= near) return;
  if ((int64_t)a.BHkv * a.S > (1 << 23)) return;  // the summing dispatch's; such a grid has work enough
  // a wave a SIMD
  const int64_t waves = 4 * device_cu_count(), all = (int64_t)a.BHkv * a.sink_tiles * a.G * far;
  a.far_chunk = (int)std::max<int64_t>(8, ceil_div(all, waves));
  a.far_parts = (int)ceil_div(a.G * far, (int64_t)a.far_chunk);
}

// Where the workspace holds item i: K's and V's planes, then for the backward Q's and
// dO's, l2, D, and the parts of dK and dV.
size_t wa_bytes(const WaArgs& a, int i) {
  const size_t pair = a.whole ? 0 : 2 * (wa_dim(a.d) == 64 ? HalfTile<64>::kBytes : HalfTile<128>::kBytes);
  const size_t kv = (size_t)a.BHkv * a.tiles, q = (size_t)a.BH * a.tiles;
  const size_t part = (size_t)a.BHkv * a.sink_tiles * a.far_parts * kTile * wa_dim(a.d) * sizeof(float);
  const size_t size[6] = {kv * pair, q * pair, q * kTile * sizeof(float), q * kTile * sizeof(float), part, part};
  size_t at = 0;
  for (int k = 0; k < i; ++k) at += (size[k] + 15) / 16 * 16;
  return at;
}
constexpr int kWaFwd = 1, kWaBwd = 6;  // items of a forward and of a backward

bool wa_workspace(WaArgs& a, void* workspace, size_t bytes, int items) {
  if (wa_bytes(a, items) == 0) return true;
  if (!workspace || !aligned16(workspace) || bytes < wa_bytes(a, items)) return false;
  char* ws = static_cast<char*>(workspace);
  a.kv_img = ws;
  if (items == kWaFwd) return true;
  a.qd_img = ws + wa_bytes(a, 1);
  a.l2 = reinterpret_cast<float*>(ws + wa_bytes(a, 2));
  a.D = reinterpret_cast<float*>(ws + wa_bytes(a, 3));
  a.dk_part = reinterpret_cast<float*>(ws + wa_bytes(a, 4));
  a.dv_part = reinterpret_cast<float*>(ws + wa_bytes(a, 5));
  return true;
}

// Row strides whose tiles' offsets fit, and whose rows do not overlap.
bool wa_rows_ok(const int64_t* strides, std::initializer_list<int> operands, int64_t T, int64_t d) {
  for (int i : operands) {
    const int64_t st = strides[3 * i + 2];
    if (T > 1 && (st < d || st > (int64_t(1) << 23))) return false;
  }
  return true;
}

bool wa_vec_ok(int64_t d, std::initializer_list<const void*> ptrs, const int64_t* strides, int n) {
  if (d % 4 != 0) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % 4 != 0) return false;
  return true;
}

FaIn wa_in(const float* p, const int64_t* s, int64_t T, int64_t d) { return FaIn{p, s[0], s[1], T > 1 ? s[2] : d}; }
FaOut wa_out(float* p, const int64_t* s) { return FaOut{p, s[0], s[1], s[2]}; }

template <int DP, bool VEC>
int launch_split(const WaArgs& a, hipStream_t st) {
  window_split_kernel<DP, VEC><<<dim3((unsigned)(2 * a.BHkv * (int64_t)a.tiles)), dim3(kFaThreads), 0, st>>>(a);
  return launch_status();
}

// The forms for texts that LDS holds, by their tiles.
template <int DP, bool VEC, int TILES>
int launch_whole_fwd(const WaArgs& a, hipStream_t st) {
  window_fwd_kernel<DP, VEC, TILES><<<dim3((unsigned)(a.BH * a.turns)), dim3(wa_threads(a.tiles)), 0, st>>>(a);
  return launch_status();
}
template <int DP, bool VEC, int TILES>
int launch_whole_bwd(const WaArgs& a, hipStream_t st) {
  window_bwd_dq_kernel<DP, VEC, TILES><<<dim3((unsigned)(a.BH * a.turns)), dim3(wa_threads(a.tiles)), 0, st>>>(a);
  const int rc = launch_status();
  if (rc != AAR_OK) return rc;
  window_bwd_dkdv_kernel<DP, VEC, 4, TILES><<<dim3((unsigned)(a.BHkv * a.turns)), dim3(wa_threads(a.tiles)), 0, st>>>(a);
  return launch_status();
}

template <int DP, bool VEC>
int launch_fwd(const WaArgs& a, hipStream_t st) {
  if (a.whole) {
    if (a.tiles <= 2) return launch_whole_fwd<DP, VEC, 2>(a, st);
    if (a.tiles <= 4) return launch_whole_fwd<DP, VEC, 4>(a, st);
    if constexpr (wa_whole(DP) > 4) return launch_whole_fwd<DP, VEC, wa_whole(DP)>(a, st);
  }
  const int rc = launch_split<DP, VEC>(a, st);
  if (rc != AAR_OK) return rc;
  const dim3 grid((unsigned)(ceil_div(a.T, kBlock) * a.BH)), block(kFaThreads);
  window_fwd_kernel<DP, VEC, 0><<<grid, block, 0, st>>>(a);
  return launch_status();
}

template <int DP, bool VEC>
int launch_bwd(const WaArgs& a, hipStream_t st) {
  if (a.whole) {
    if (a.tiles <= 2) return launch_whole_bwd<DP, VEC, 2>(a, st);
    if (a.tiles <= 4) return launch_whole_bwd<DP, VEC, 4>(a, st);
    if constexpr (wa_whole(DP) > 4) return launch_whole_bwd<DP, VEC, wa_whole(DP)>(a, st);
  }
  int rc = launch_split<DP, VEC>(a, st);
  if (rc != AAR_OK) return rc;
  const int64_t blocks = ceil_div(a.T, kBlock);
  const dim3 rows((unsigned)(blocks * a.BH)), keys((unsigned)(blocks * a.BHkv)), block(kFaThreads);
  window_bwd_dq_kernel<DP, VEC, 0><<<rows, block, 0, st>>>(a);
  rc = launch_status();
  if (rc != AAR_OK) return rc;
  window_bwd_dkdv_kernel<DP, VEC, 4, 0><<<keys, block, 0, st>>>(a);
  rc = launch_status();
  if (rc != AAR_OK || a.far_parts == 0) return rc;
  const int64_t far = (int64_t)a.BHkv * a.sink_tiles * a.far_parts;
  window_bwd_dkdv_kernel<DP, VEC, 1, 0><<<dim3((unsigned)far), dim3(kWave), 0, st>>>(a);
  rc = launch_status();
  if (rc != AAR_OK) return rc;
  window_bwd_sum_kernel<DP, VEC><<<dim3((unsigned)((int64_t)a.BHkv * a.S)), dim3(256), 0, st>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

size_t aar_window_attn_fwd_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window,
                                           int64_t sinks) {
  if (wa_check(B, H, Hkv, T, d, window, sinks) != AAR_OK || B == 0 || H == 0 || T == 0) return 0;
  return wa_bytes(wa_args(B, H, Hkv, T, d, window, sinks, 1.0f), kWaFwd);
}

int aar_window_attn_fwd_f32(const float* q, const float* k, const float* v, float* o, float* lse, int64_t B, int64_t H,
                            int64_t Hkv, int64_t T, int64_t d, const int64_t* strides, int64_t window, int64_t sinks,
                            float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = wa_check(B, H, Hkv, T, d, window, sinks);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0 || T == 0) return AAR_OK;
  if (!q || !k || !v || !o || !lse || !strides) return AAR_EINVAL;
  if (!wa_rows_ok(strides, {0, 1, 2}, T, d)) return AAR_EUNSUPPORTED;
  WaArgs a = wa_args(B, H, Hkv, T, d, window, sinks, scale);
  if (!wa_workspace(a, workspace, workspace_bytes, kWaFwd)) return AAR_EWORKSPACE;
  a.lse = lse;
  a.q = wa_in(q, strides, T, d);
  a.k = wa_in(k, strides + 3, T, d);
  a.v = wa_in(v, strides + 6, T, d);
  a.o = wa_out(o, strides + 9);
  const bool vec = wa_vec_ok(d, {q, k, v, o}, strides, 12);
  hipStream_t st = as_stream(stream);
  if (wa_dim(d) == 64) return vec ? launch_fwd<64, true>(a, st) : launch_fwd<64, false>(a, st);
  return vec ? launch_fwd<128, true>(a, st) : launch_fwd<128, false>(a, st);
}

size_t aar_window_attn_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window,
                                           int64_t sinks) {
  if (wa_check(B, H, Hkv, T, d, window, sinks) != AAR_OK || B == 0 || H == 0 || T == 0) return 0;
  WaArgs a = wa_args(B, H, Hkv, T, d, window, sinks, 1.0f);
  wa_bwd_plan(a);
  return wa_bytes(a, kWaBwd);
}

int aar_window_attn_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* lse,
                            const float* dout, float* dq, float* dk, float* dv, int64_t B, int64_t H, int64_t Hkv,
                            int64_t T, int64_t d, const int64_t* strides, int64_t window, int64_t sinks, float scale,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = wa_check(B, H, Hkv, T, d, window, sinks);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0 || T == 0) return AAR_OK;
  if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv || !strides) return AAR_EINVAL;
  if (!wa_rows_ok(strides, {0, 1, 2, 3, 4}, T, d)) return AAR_EUNSUPPORTED;
  WaArgs a = wa_args(B, H, Hkv, T, d, window, sinks, scale);
  wa_bwd_plan(a);
  if (!wa_workspace(a, workspace, workspace_bytes, kWaBwd)) return AAR_EWORKSPACE;
  a.lse = const_cast<float*>(lse);
  a.q = wa_in(q, strides, T, d);
  a.k = wa_in(k, strides + 3, T, d);
  a.v = wa_in(v, strides + 6, T, d);
  a.o_in = wa_in(o, strides + 9, T, d);
  a.dout = wa_in(dout, strides + 12, T, d);
  a.dq = wa_out(dq, strides + 15);
  a.dk = wa_out(dk, strides + 18);
  a.dv = wa_out(dv, strides + 21);
  const bool vec = wa_vec_ok(d, {q, k, v, o, dout, dq, dk, dv}, strides, 24);
  hipStream_t st = as_stream(stream);
  if (wa_dim(d) == 64) return vec ? launch_bwd<64, true>(a, st) : launch_bwd<64, false>(a, st);
  return vec ? launch_bwd<128, true>(a, st) : launch_bwd<128, false>(a, st);
}

}  // extern "C"
