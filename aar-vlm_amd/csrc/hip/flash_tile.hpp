// What the attention kernels' tiles are made of: the matrix op and the layout
// of its accumulators, row loads and stores, cooperative copies of [32][DP]
// tiles into LDS (plain and transposed), and strided [B, H, T, d] operands.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.hpp"

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

}  // namespace aar
