// What the attention kernels' tiles are made of: the matrix op and the layout
// of its accumulators, row loads and stores, cooperative copies of [32][DP]
// tiles into LDS (plain, transposed, and split into bf16 parts), and strided
// [B, H, T, d] operands.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "bf16x3.hpp"
#include "common.hpp"
#include "flash_offsets.hpp"

namespace aar {

constexpr int kFaThreads = 256;  // 4 waves
constexpr int kTile = 32;        // keys (or queries) per inner tile
constexpr int kBlock = 128;      // queries (or keys) per workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ f32x16 mfma32(float a, float b, const f32x16& c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// 2^x on the transcendental unit (v_exp_f32): inputs are scaled logits minus
// a running max, so results below 2^-126 (flushed to zero) carry no weight.
// The builtin exists only for the device target; the host pass never runs it.
__device__ __forceinline__ float fast_exp2(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);
#else
  return x;
#endif
}

// Row index (within a 32-row tile) of accumulator register r for lane half h.
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// 4 consecutive floats p[0..3] of a row with `valid` leading entries (zeros
// past it).  VEC: the row is 16-byte aligned and valid is 0 or >= 4.
template <bool VEC>
__device__ __forceinline__ f32x4 load4(const float* __restrict__ p, int valid) {
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (VEC) {
    if (valid >= 4) v = *reinterpret_cast<const f32x4*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) v[e] = p[e];
  }
  return v;
}

template <bool VEC>
__device__ __forceinline__ void store4(float* __restrict__ p, f32x4 v, int valid) {
  if (VEC) {
    if (valid >= 4) *reinterpret_cast<f32x4*>(p) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) p[e] = v[e];
  }
}

// Column c's rows of a transposed tile stand at r ^ 4 ((c / 16) % 4) (SWZ): a
// copy's 16 consecutive columns then reach 16 banks instead of 4, and groups of 4
// consecutive rows stay together.
template <bool SWZ>
__device__ __forceinline__ int vt_swz(int c, int r) { return SWZ ? r ^ (((c >> 4) & 3) << 2) : r; }
// Cooperative copy of a [32][DP] tile (rows row0.., head dim padded to DP with
// zeros, rows past T zero) from global into registers, then into LDS with row
// stride LD.
template <int DP, bool VEC>
struct TileCopy {
  static constexpr int kUnits = kTile * DP / 4;
  static constexpr int kPer = (kUnits + kFaThreads - 1) / kFaThreads;
  f32x4 reg[kPer];

  __device__ __forceinline__ void load(const float* __restrict__ base, int64_t st, int row0, int T, int d,
                                       int tid) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = tid + i * kFaThreads;
      const int r = u / (DP / 4);
      const int c = (u % (DP / 4)) * 4;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (u < kUnits && row0 + r < T) v = load4<VEC>(base + (int64_t)(row0 + r) * st + c, d - c);
      reg[i] = v;
    }
  }

  template <int LD>
  __device__ __forceinline__ void store(float* __restrict__ s, int tid) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = tid + i * kFaThreads;
      if (u < kUnits) {
        const int r = u / (DP / 4);
        const int c = (u % (DP / 4)) * 4;
        *reinterpret_cast<f32x4*>(s + r * LD + c) = reg[i];
      }
    }
  }

  // Transposed: element (row r, column c) to s[c * LDT + vt_swz(c, r)], so
  // that 4 consecutive rows of one column are one 128-bit LDS read.
  template <int LDT, bool SWZ>
  __device__ __forceinline__ void store_t(float* __restrict__ s, int tid) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = tid + i * kFaThreads;
      if (u < kUnits) {
        const int r = u / (DP / 4);
        const int c = (u % (DP / 4)) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) s[(c + e) * LDT + vt_swz<SWZ>(c + e, r)] = reg[i][e];
      }
    }
  }
};

// A [B, H, T, d] operand with element (b, h, t, c) at p[b*sb + h*sh + t*st + c]
// (the head dim is contiguous).  Contiguous [B*H, T, d] tensors, the q/k/v
// views of a packed [B, T, 3, H, d] projection and outputs in [B, T, H, d]
// are all of this form.
struct FaIn {
  const float* p;
  int64_t sb, sh, st;
  __device__ __forceinline__ const float* head(int bh, int H) const {
    return p + (int64_t)(bh / H) * sb + (int64_t)(bh % H) * sh;
  }
};
struct FaOut {
  float* p;
  int64_t sb, sh, st;
  __device__ __forceinline__ float* head(int bh, int H) const {
    return p + (int64_t)(bh / H) * sb + (int64_t)(bh % H) * sh;
  }
};

// Row stride of a transposed [DP][32] tile: 36 keeps the 128-bit reads of 32
// consecutive columns (one per lane) bank-conflict free.
constexpr int kLdt = kTile + 4;

// A [32][DP] tile staged transposed for the split products whose reduced-over
// dimension is the tile's rows (V^T P^T): a thread takes 8 rows of one
// column, which is one lane's operand of the matrix op.  Planes are
// [part][octet][column] in 16-byte units.
template <int DP>
struct FaKtSplit {
  static constexpr int kUnits = DP * 4;  // (column, octet of rows)
  static constexpr int kPer = kUnits / kFaThreads;
  static_assert(kUnits % kFaThreads == 0, "whole units per thread");
  static constexpr int kPlanes = 3 * kUnits;  // 16-byte units of a stage
  float f[kPer][8];
  float top = 0.f;  // largest magnitude of this thread's elements

  // Key e of octet o = 2s + h within the tile: acc_row(8s + e, h).
  __device__ __forceinline__ static int key(int o, int e) {
    return 16 * (o >> 1) + 8 * (e >> 2) + 4 * (o & 1) + (e & 3);
  }
  // Rows past T are clamped onto row T - 1 (their P is 0; an infinite element
  // sends the wave to the fp32 instruction) and columns past d onto column d - 1 (they
  // feed outputs that are not stored), so no load is predicated.  Offsets
  // within a tile fit 32 bits (`small`) or take the clamped form, whose
  // addresses are 64-bit and signed.
  uint32_t off[kPer];
  int64_t row4;  // bytes per row
  bool small;
  __device__ __forceinline__ void init(int64_t st, int d, int tid) {
    row4 = st * 4;
    small = tile_offsets_fit(st);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = tid + i * kFaThreads;
      off[i] = tile_offset(key(u / DP, 0), st, min(u % DP, d - 1));
    }
  }
  __device__ __forceinline__ void load(const float* __restrict__ K, int64_t st, int row0, int T, int d, int tid) {
    if (row0 + kTile <= T && small) {
      const char* base = reinterpret_cast<const char*>(K + (int64_t)row0 * st);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e)  // key(o, e) = key(o, 0) + key(0, e)
          f[i][e] = *reinterpret_cast<const float*>(base + key(0, e) * row4 + off[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int u = tid + i * kFaThreads;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = min(row0 + key(u / DP, e), T - 1);
          f[i][e] = K[(int64_t)row * st + min(u % DP, d - 1)];
        }
      }
    }
  }
  // rem: what the splits left over (bf16_split_pair).
  __device__ __forceinline__ void store(u32x4* s, int tid, uint32_t& rem) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int u = tid + i * kFaThreads;
      u32x4 parts[3];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t w[3];
        top = fmaxf(fmaxf(top, fabsf(f[i][2 * e])), fabsf(f[i][2 * e + 1]));
        bf16_split_pair(f[i][2 * e], f[i][2 * e + 1], w, rem);
#pragma unroll
        for (int p = 0; p < 3; ++p) parts[p][e] = w[p];
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) s[p * kUnits + u] = parts[p];
    }
  }
};

// The same for products over the columns (K Q^T): a thread takes 8 columns of
// one row; planes are [part][octet of columns][row], the octets one unit
// further apart so that the eight threads of a row store to distinct banks.
template <int DP>
struct FaRowSplit {
  static constexpr int kOcts = DP / 8;
  static constexpr int kUnits = kTile * kOcts;
  static_assert(kUnits == kFaThreads, "one unit per thread");
  static constexpr int kOs = kTile + 1;
  static constexpr int kPlane = kOcts * kOs;
  f32x4 f[2];
  float top = 0.f;

  // Rows past T are clamped onto row T - 1 (the caller masks them), columns
  // past d onto earlier ones (Q is zero there).
  uint32_t off[2];
  bool small;
  __device__ __forceinline__ static int column(int tid, int g, int d) {
    return min(8 * (tid % kOcts) + 4 * g, d - 4);  // d is a multiple of 4
  }
  __device__ __forceinline__ void init(int64_t st, int d, int tid) {
    small = tile_offsets_fit(st);
#pragma unroll
    for (int g = 0; g < 2; ++g) off[g] = tile_offset(tid / kOcts, st, column(tid, g, d));
  }
  __device__ __forceinline__ void load(const float* __restrict__ K, int64_t st, int row0, int T, int d, int tid) {
    if (row0 + kTile <= T && small) {
      const char* base = reinterpret_cast<const char*>(K + (int64_t)row0 * st);
#pragma unroll
      for (int g = 0; g < 2; ++g) f[g] = *reinterpret_cast<const f32x4*>(base + off[g]);
    } else {
      const float* row = K + (int64_t)min(row0 + tid / kOcts, T - 1) * st;
#pragma unroll
      for (int g = 0; g < 2; ++g) f[g] = *reinterpret_cast<const f32x4*>(row + column(tid, g, d));
    }
  }
  __device__ __forceinline__ void store(u32x4* s, int tid, uint32_t& rem) {
    u32x4 parts[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = f[e >> 1][2 * (e & 1)], y = f[e >> 1][2 * (e & 1) + 1];
      uint32_t w[3];
      top = fmaxf(fmaxf(top, fabsf(x)), fabsf(y));
      bf16_split_pair(x, y, w, rem);
#pragma unroll
      for (int p = 0; p < 3; ++p) parts[p][e] = w[p];
    }
#pragma unroll
    for (int p = 0; p < 3; ++p) s[p * kPlane + (tid % kOcts) * kOs + tid / kOcts] = parts[p];
  }
};

}  // namespace aar
