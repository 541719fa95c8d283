// fp32 products on the fp16 matrix cores: operands in two fp16 parts scaled row by row,
// tiles of them in LDS, and the scale of what is multiplied with a tile's columns.
//
// x 2^e = hi + lo, hi rounded from x 2^e and lo from what that leaves, so that three
// matrix ops (lo hi, hi lo, hi hi; 16 steps each at 16 times the fp32 instruction's
// rate) stand for one fp32 product.  An operand is off by at most 2^-22 of itself or,
// where that is more, 2^-38 of its row's largest element, lo lo is at most 2^-22 of a
// product and is left out; sums are in fp32.  e is a row's own (where a kernel says so, that of
// a tile of 32 rows), such that its largest element is in [2^13, 2^14).  Over the head dim a row's factor is one of the output's
// row or column.  Over a tile's rows it goes to the other operand, P or dS, which is
// scaled by the lane's own power of two that follows the largest |P| 2^-e (|dS| 2^-e)
// so far (HalfScale).  Rows whose largest element is not 0 and outside [2^-99, 2^60) are
// not held so; `bad` says that one was met, and the kernels do its rows again with the
// fp32 instruction.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "bf16x3.hpp"
#include "common.hpp"
#include "flash_tile.hpp"

namespace aar {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mfma_f16(const u32x4& a, const u32x4& b, const f32x16& c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
#else
  return c;
#endif
}

// The products, smallest first.
constexpr int kHalfProducts = 3;
__device__ constexpr int kHalfA[kHalfProducts] = {1, 0, 0};
__device__ constexpr int kHalfB[kHalfProducts] = {0, 1, 0};

// The two parts of (a, b) m, a pair a word; m is a power of two, so the fused
// product and difference are exact.
__device__ __forceinline__ void half_split_pair(float a, float b, float m, uint32_t& hi, uint32_t& lo) {
  const f32x2 v = {a * m, b * m};
  const f16x2 x = __builtin_convertvector(v, f16x2);
  const f32x2 rest = {fmaf(a, m, -(float)x[0]), fmaf(b, m, -(float)x[1])};
  hi = __builtin_bit_cast(uint32_t, x);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // |e| <= 126

// A row's scale from the bits u of its largest magnitude: their exponent, of which the
// factors below are made (the least for zeros), and whether the parts do not hold the
// row: below 2^-99 the scale would pass 2^112, and what undoes it leave fp32's normal
// range; sums of 128 products of 2^60 and 2^60 end at 2^127.
__device__ __forceinline__ uint32_t half_exponent(uint32_t u, bool& bad) {
  const uint32_t lo = (127 - 99) << 23, hi = (127 + 60) << 23;
  bad = bad || (u != 0 && u - lo >= hi - lo);
  return max(u, lo) & 0x7F800000u;
}

// The scale 2^e, and what undoes it: for a tile's row 2^(14 - e), which is 1 to 2 times
// the row's largest magnitude, so that P or dS times it is as large as its largest term
// and leaves fp32's range no sooner.  The 2^14 comes off with the factor of the lane's
// own row in a score or dP, with HalfScale's in a sum.
__device__ __forceinline__ float half_scale(uint32_t e) { return __uint_as_float((267u << 23) - e); }
__device__ __forceinline__ float row_factor(uint32_t e) { return __uint_as_float(e + (1u << 23)); }
__device__ __forceinline__ float lane_factor(uint32_t e) { return __uint_as_float(e - (27u << 23)); }

// Largest of the 8 or 16 lanes of a tile's row (magnitudes, as their bits).
template <int N>
__device__ __forceinline__ uint32_t row_top(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  if (N == 16) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  return v;
}

// Rows as a buffer: reads at or past `bytes` from p give zeros.
constexpr uint32_t kNowhere = 0x80000000u;  // an offset past every buffer's end

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const float* p, uint32_t bytes) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(p), 0, (int)bytes, 0x00027000);
#endif
}
__device__ __forceinline__ f32x4 buffer_load4(__amdgpu_buffer_rsrc_t rows, uint32_t at) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, (int)at, 0, 0));
#else
  return f32x4{0.f, 0.f, 0.f, 0.f};
#endif
}

// The first `valid` of four floats, one by one.
__device__ __forceinline__ f32x4 buffer_load1x4(__amdgpu_buffer_rsrc_t rows, uint32_t at, int valid) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#if defined(__HIP_DEVICE_COMPILE__)
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int off = e < valid ? (int)(at + 4 * e) : (int)kNowhere;
    v[e] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rows, off, 0, 0));
  }
#endif
  return v;
}

// The larger, or NaN where one is.
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A [32][DP] tile in two planes of 32 rows; a row's 16 spare bytes put 16
// consecutive rows' 128-bit reads on distinct banks.
template <int DP>
struct HalfTile {
  static constexpr int kRow = 2 * DP + 16;  // bytes
  static constexpr int kPlane = kTile * kRow;
  static constexpr int kBytes = 2 * kPlane;
  static constexpr int kOcts = DP / 8;
  static constexpr int kPer = kTile * kOcts / kFaThreads;  // 8-column units a thread stages
  static_assert(kPer * kFaThreads == kTile * kOcts && kOcts <= 16, "whole units, a row in 16 lanes");
  f32x4 f[kPer][2];
  uint32_t ex[kPer];  // of the rows that `store` has scaled: half_exponent's

  // Row of unit i of thread tid, and its first column.
  __device__ __forceinline__ static int row(int i, int tid) { return (tid + i * kFaThreads) / kOcts; }
  __device__ __forceinline__ static int col(int tid) { return 8 * (tid % kOcts); }
  // Where this thread's units stand in rows of `st` floats, in bytes from row 0.
  struct Place {
    uint32_t at[kPer][2];
    __device__ __forceinline__ Place(int64_t st, int d, int tid) {
#pragma unroll
      for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int g = 0; g < 2; ++g)
          at[i][g] = col(tid) + 4 * g < d ? (uint32_t)((row(i, tid) * st + col(tid) + 4 * g) * 4) : kNowhere;
    }
  };
  // The 32 rows from p on, of which `rows` are read, others are zeros.  VEC: rows are
  // 16-byte aligned and d is a multiple of 4.
  template <bool VEC = true>
  __device__ __forceinline__ void load(const float* p, int64_t st, int rows, int d, const Place& w) {
    const int last = min(rows, kTile) - 1;  // no branch: loads in flight stay countable
    const uint32_t bytes = (uint32_t)(last * (int)st + d) * 4u & ~(uint32_t)(last >> 31);
    const __amdgpu_buffer_rsrc_t b = row_buffer(p, bytes);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (VEC) f[i][g] = buffer_load4(b, w.at[i][g]);
        else f[i][g] = buffer_load1x4(b, w.at[i][g], d - (int)(threadIdx.x % kOcts) * 8 - 4 * g);
      }
  }
  // Rows [row0, row0 + 32) of a list of `n` that is Tq rows of each of several heads.
  __device__ __forceinline__ void load_heads(const float* p, int64_t sh, int64_t st, int Tq, int row0, int n, int d,
                                             int tid) {
    const __amdgpu_buffer_rsrc_t b = row_buffer(p, kNowhere - 1);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = row0 + row(i, tid), g = r / Tq, t = r - g * Tq;
      const uint32_t at = (uint32_t)((g * sh + t * st + col(tid)) * 4);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        f[i][k] = buffer_load4(b, r < n && col(tid) + 4 * k < d ? at + 16 * k : kNowhere);
    }
  }
  __device__ __forceinline__ void store(char* s, int tid, bool& bad) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int e = 0; e < 2; ++e) top = fmaxf(fmaxf(top, fabsf(f[i][g][2 * e])), fabsf(f[i][g][2 * e + 1]));
      ex[i] = half_exponent(row_top<kOcts>(__float_as_uint(top)), bad);
      const float m = half_scale(ex[i]);
      u32x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t x, y;
        half_split_pair(f[i][e >> 1][2 * (e & 1)], f[i][e >> 1][2 * (e & 1) + 1], m, x, y);
        hi[e] = x;
        lo[e] = y;
      }
      char* at = s + row(i, tid) * kRow + 2 * col(tid);
      *reinterpret_cast<u32x4*>(at) = hi;
      *reinterpret_cast<u32x4*>(at + kPlane) = lo;
    }
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: 16 lanes read four rows of 16 halves each (lane j the four
// from column 4 (j % 4) of row j / 4) and lane j receives column j of the rows.
__device__ __forceinline__ void read_columns(const char* p, uint32_t& lo, uint32_t& hi) {
#if defined(__HIP_DEVICE_COMPILE__)
  const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 w = __builtin_bit_cast(u32x2, v);
  lo = w[0];
  hi = w[1];
#endif
}

// tile . B over the head dim: the tile's 32 rows are the output's rows, B's columns
// (b[c][part], lane = column) the output's.
template <int DP>
__device__ __forceinline__ f32x16 half_rows(const char* s, const u32x4 (&b)[DP / 16][2], int lr, int h) {
  f32x16 acc = zero16();
  const char* p = s + lr * HalfTile<DP>::kRow + 16 * h;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    u32x4 x[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) x[i] = *reinterpret_cast<const u32x4*>(p + i * HalfTile<DP>::kPlane + 32 * c);
#pragma unroll
    for (int i = 0; i < kHalfProducts; ++i) acc = mfma_f16(x[kHalfA[i]], b[c][kHalfB[i]], acc);
  }
  return acc;
}

// The two parts of (a, b), a pair a word.  one: 1, unknown to the compiler, so that a
// difference is one mixed multiply-add and not a conversion and a subtraction.
__device__ __forceinline__ void half_split_plain(float a, float b, float one, uint32_t& hi, uint32_t& lo) {
  const f16x2 x = __builtin_convertvector(f32x2{a, b}, f16x2);
  const f32x2 rest = {fmaf(a, one, -(float)x[0]), fmaf(b, one, -(float)x[1])};
  hi = __builtin_bit_cast(uint32_t, x);
  lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
}

// acc[b] += tile^T . x over rows 16 k .. 16 k + 15 of the tile, x = accumulator
// registers 8 k .. 8 k + 7 of x times f (PLAIN: of x, f = 1): column 32 b + lr of the tile.
template <int DP, bool PLAIN = false>
__device__ __forceinline__ void half_cols(const char* s, const f32x16& x, float f, int k, int lane,
                                          f32x16 (&acc)[DP / 32]) {
  using T = HalfTile<DP>;
  const int h = lane >> 5, j = lane & 15;
  const char* p = s + (16 * k + 4 * h + (j >> 2)) * T::kRow + 2 * (16 * ((lane >> 4) & 1) + 4 * (j & 3));
  u32x4 pp[2];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    uint32_t hi, lo;
    if (PLAIN) half_split_plain(x[8 * k + 2 * e], x[8 * k + 2 * e + 1], f, hi, lo);
    else half_split_pair(x[8 * k + 2 * e], x[8 * k + 2 * e + 1], f, hi, lo);
    pp[0][e] = hi;
    pp[1][e] = lo;
  }
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
    u32x4 y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[4];
      read_columns(p + i * T::kPlane + 64 * b, w[0], w[1]);
      read_columns(p + i * T::kPlane + 64 * b + 8 * T::kRow, w[2], w[3]);
      y[i] = u32x4{w[0], w[1], w[2], w[3]};
    }
#pragma unroll
    for (int i = 0; i < kHalfProducts; ++i) acc[b] = mfma_f16(y[kHalfA[i]], pp[kHalfB[i]], acc[b]);
  }
}

// A lane's row (its half's octets of each 16 columns), or times f from p, in parts; returns its
// factor.
template <int DP>
__device__ __forceinline__ float half_row(const f32x4 (&x)[DP / 16][2], u32x4 (&out)[DP / 16][2], bool& bad) {
  float top = 0.f;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[c][g][e]));
    }
  }
  const uint32_t ex = half_exponent(__float_as_uint(half_swap_max(top)), bad);
  const float m = half_scale(ex);
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t hi, lo;
      half_split_pair(x[c][e >> 1][2 * (e & 1)], x[c][e >> 1][2 * (e & 1) + 1], m, hi, lo);
      out[c][0][e] = hi;
      out[c][1][e] = lo;
    }
  }
  return lane_factor(ex);
}
template <int DP, bool VEC = true>
__device__ __forceinline__ float half_row(const float* p, int d, float f, int h, u32x4 (&out)[DP / 16][2], bool& bad) {
  f32x4 x[DP / 16][2];
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int dd = 16 * c + 8 * h + 4 * g;
      x[c][g] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (p && dd < d) x[c][g] = load4<VEC>(p + dd, d - dd) * f;
    }
  }
  return half_row<DP>(x, out, bad);
}

// The power of two f = 2^log that a lane's P or dS, times the factors of the other
// operand's rows, is scaled by, from the magnitudes up to `top` of a tile's: the first tile
// sets it such that the largest is in [2^13, 2^14), a later one lowers it, with the sums
// so far, when it passes 2^15.  Magnitudes below 2^-112 would need more than the largest
// scale, 2^126; under that one what a part rounds is 2^-151, less than fp32 holds.
template <int NB>
struct HalfScale {
  int log = 0;
  float f = 1.f, most = -1.f, big = 0.f;  // `most`: what f holds; `big`: the largest so far
  __device__ __forceinline__ void follow(float top, f32x16 (&acc)[NB], bool& bad) {
    top = half_swap_max(top);
    big = fmaxf(big, top);
    if (!__any(top > most)) return;
    if (top > most) {
      const int to = 140 - (int)(__float_as_uint(big) >> 23);
      bad = bad || to < -114;  // infinite
      const int by = min(min(to, 126) - log, 126);
      log += by;
      f = pow2(log);
      most = ldexpf(32768.f, -log);
      const float g = ldexpf(1.f, by);
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[b][r] *= g;
      }
    }
  }
  // The sums themselves.
  __device__ __forceinline__ void undo(f32x16 (&acc)[NB]) const {
    const float by = pow2(-log);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[b][r] = acc[b][r] * 0x1p-14f * by;
    }
  }
};

// Rows 8 g + 4 h .. of a tile's row values.
__device__ __forceinline__ f32x4 row_values(const float* x, int g, int h) {
  return *reinterpret_cast<const f32x4*>(x + 8 * g + 4 * h);
}

// What a masked product over rows [row0, row0 + 32) of p gets from their elements that
// are not finite: columns c of row j add w_j x_jc to the lanes whose `sees(j)` is true, to
// no others (0 times an infinity is NaN).  w as a product's accumulators leave it, acc
// as half_cols has it; the product itself takes `finite` elements alone.
__device__ __forceinline__ float finite(float x) { return fabsf(x) < INFINITY ? x : 0.f; }

template <int NB, class Sees>
__device__ __forceinline__ void add_not_finite(const float* p, int64_t st, int row0, int end, int d, const f32x16& w,
                                               Sees sees, f32x16 (&acc)[NB]) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int j = 0; j < 2 * kTile; ++j) {  // halves of rows
    const int row = j >> 1, c0 = 64 * (j & 1), c = c0 + lane;
    if (row0 + row >= end) break;
    const float x = c < d ? p[(int64_t)(row0 + row) * st + c] : 0.f;
    uint64_t rest = __ballot(!(fabsf(x) < INFINITY));
#pragma unroll 1
    while (rest != 0) {
      const int at = __ffsll((unsigned long long)rest) - 1, col = c0 + at, r = (row >> 3) * 4 + (row & 3);
      rest &= rest - 1;
      float f = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i == r) f = w[i];
      f = __shfl(f, (lane & 31) | (row >> 2 & 1) << 5, kWave) * __shfl(x, at, kWave);
      if (!sees(row0 + row) || (lane >> 5) != (col >> 2 & 1)) continue;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i >> 2) + (i & 3) == (col & ~4)) acc[b][i] += f;
      }
    }
  }
}

}  // namespace aar
