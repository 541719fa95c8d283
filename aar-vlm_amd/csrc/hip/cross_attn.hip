// Cross attention: queries against an encoder's keys and values of another
// length, forward and backward, in fp32.
//
// For every batch b and query head h, with the keys j < len[b] and the shared
// key/value head hk = h / G, G = H / Hkv:
//   s_ij = scale q_i . k_j,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),
//   O_i = sum_j exp(s_ij - m_i) v_j / l_i,      lse_i = m_i + ln l_i
// and a row without keys has O = 0, lse = -inf.  Backward, with P = exp(s - lse),
// D_i = dO_i . O_i and dS = P (dO V^T - D):
//   dQ = scale dS K,  dV = P^T dO,  dK = scale dS^T Q, both summed over the G
//   heads that share the key.
//
// The query heads of a shared key/value head are one list of G * Tq query rows, so
// a workgroup's K and V tiles serve whatever heads its rows belong to, and the
// sums over the group happen in the accumulators that dK and dV have anyway.
// Rows of K and V from len[b] on are never read; their gradients are zero.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "common.hpp"
#include "flash_offsets.hpp"
#include "flash_tile.hpp"
#include "half_tile.hpp"

namespace aar {
namespace {

struct CaArgs {
  FaIn q, k, v, o_in, dout;
  FaOut o, dq, dk, dv;
  const int64_t* lens;
  float* lse;     // [B * Hkv][R]
  float* D;       // [B * Hkv][R], backward
  float* part_o;  // [B * Hkv][splits][R][DP] normalised partial O
  float* part_l;  // [B * Hkv][splits][R] m + log2(l) of it
  int Tq, Tk, d, G, Hkv, R, BH;  // R = G * Tq rows of each of the BH = B * Hkv key/value heads
  int splits, chunk;             // key ranges of the forward or of dQ, and their keys
  float *dq_part, *dk_part, *dv_part;  // backward: [splits][BH][R][DP], [kv_splits][BH][Tk][DP] partial sums
  int kv_splits, kv_tiles;             // ranges of query rows of dK and dV, and their tiles
  float scale, scale_log2;
};

// Keys of batch b.
__device__ __forceinline__ int ca_len(const CaArgs& a, int bh) {
  if (!a.lens) return a.Tk;
  const int64_t n = a.lens[bh / a.Hkv];
  return n < 0 ? 0 : (n > a.Tk ? a.Tk : (int)n);
}

// Element offset of query row r of key/value head bh in a query-shaped operand.
template <typename T>
__device__ __forceinline__ int64_t ca_row(const T& x, const CaArgs& a, int bh, int r) {
  const int g = a.G == 1 ? 0 : r / a.Tq;
  const int t = a.G == 1 ? r : r - g * a.Tq;
  return (int64_t)(bh / a.Hkv) * x.sb + ((int64_t)(bh % a.Hkv) * a.G + g) * x.sh + (int64_t)t * x.st;
}

// The first head of key/value head bh's group in a query-shaped operand.
__device__ __forceinline__ const float* ca_group(const FaIn& x, const CaArgs& a, int bh) {
  return x.p + (int64_t)(bh / a.Hkv) * x.sb + (int64_t)(bh % a.Hkv) * a.G * x.sh;
}

template <typename T>
__device__ __forceinline__ auto ca_head(const T& x, const CaArgs& a, int bh) {
  return x.p + (int64_t)(bh / a.Hkv) * x.sb + (int64_t)(bh % a.Hkv) * x.sh;
}

// A lane's row of a forward: O and lse, or the normalised part and its log2 sum.
template <int DP, bool VEC>
__device__ __forceinline__ void ca_store_row(const CaArgs& a, int bh, int part, int qi, int h,
                                             const f32x16 (&o)[DP / 32], float m, float l) {
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const float l2 = m + log2f(l);
  const int64_t prow = ((int64_t)bh * a.splits + part) * a.R + qi;
  float* orow = a.splits > 1 ? a.part_o + prow * DP : a.o.p + ca_row(a.o, a, bh, qi);
#pragma unroll
  for (int b = 0; b < DP / 32; ++b) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int dd = b * 32 + 8 * g + 4 * h;
      const f32x4 v = {o[b][4 * g] * inv, o[b][4 * g + 1] * inv, o[b][4 * g + 2] * inv, o[b][4 * g + 3] * inv};
      if (a.splits > 1) *reinterpret_cast<f32x4*>(orow + dd) = v;
      else if (dd < a.d) store4<VEC>(orow + dd, v, a.d - dd);
    }
  }
  if (h == 0) {
    if (a.splits > 1) a.part_l[prow] = l2;
    else a.lse[(int64_t)bh * a.R + qi] = l2 * kLn2;
  }
}

// A lane's row of accumulators times f.
template <int DP, bool VEC>
__device__ __forceinline__ void ca_store_scaled(float* row, const f32x16 (&x)[DP / 32], float f, int d, int h) {
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

// A lane's row of dQ: to its place, or its part's.
template <int DP, bool VEC>
__device__ __forceinline__ void ca_store_dq(const CaArgs& a, int bh, int part, int qi, const f32x16 (&dq)[DP / 32],
                                            int h) {
  if (a.splits > 1) {
    ca_store_scaled<DP, true>(a.dq_part + (((int64_t)part * a.BH + bh) * a.R + qi) * DP, dq, a.scale, DP, h);
  } else {
    ca_store_scaled<DP, VEC>(a.dq.p + ca_row(a.dq, a, bh, qi), dq, a.scale, a.d, h);
  }
}

// A lane's key: dK and dV.  A masked key's zero is written as such (its sums may
// hold 0 * inf).
template <int DP, bool VEC>
__device__ __forceinline__ void ca_store_key(const CaArgs& a, int bh, int part, int kj, bool key_ok,
                                             f32x16 (&dk)[DP / 32], f32x16 (&dv)[DP / 32], int h) {
  if (!key_ok) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b) dk[b] = dv[b] = zero16();
  }
  if (a.kv_splits > 1) {
    const int64_t at = (((int64_t)part * a.BH + bh) * a.Tk + kj) * DP;
    ca_store_scaled<DP, true>(a.dk_part + at, dk, a.scale, DP, h);
    ca_store_scaled<DP, true>(a.dv_part + at, dv, 1.0f, DP, h);
    return;
  }
  ca_store_scaled<DP, VEC>(ca_head(a.dk, a, bh) + (int64_t)kj * a.dk.st, dk, a.scale, a.d, h);
  ca_store_scaled<DP, VEC>(ca_head(a.dv, a, bh) + (int64_t)kj * a.dv.st, dv, 1.0f, a.d, h);
}

// -------------------------------------------------------------- few query rows

// Sum over the LPK lanes that hold a key's row.
template <int LPK>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp_quad_xor1(x);
  x += dpp_quad_xor2(x);
  x += dpp_half_mirror(x);
  if (LPK >= 16) x += dpp_row_mirror(x);
  if (LPK >= 32) x += swizzle_xor16(x);
  return x;
}

// Up to RQ query rows a key/value head (single tokens): bound by the bytes of K
// and V.  LPK lanes hold a key's row, four floats each, and walk the keys with
// their own online softmax, U keys' loads in flight; the groups' and waves'
// states meet once at the end.  The key range is split over enough workgroups to
// fill the GPU, joined by cross_combine_kernel.  32 x 6 heads' single rows over up to
// 2048 keys, d 64 (151 MB): 29 us, 5.2 TB/s, and 4.7 us for the parts.
template <int RQ, int LPK, bool VEC>
__global__ void __launch_bounds__(256)
cross_rows_kernel(const CaArgs a) {
  constexpr int U = 4;
  constexpr int kGroups = kWave / LPK;
  constexpr int kWaves = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane / LPK, c = 4 * (lane % LPK);
  const int bh = blockIdx.x % a.BH, part = blockIdx.x / a.BH;
  const int len = ca_len(a, bh);
  const int k0 = part * a.chunk, k1 = min(len, k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);

  f32x4 q[RQ], acc[RQ];
  float m[RQ], l[RQ];
#pragma unroll
  for (int r = 0; r < RQ; ++r) {
    q[r] = acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r < a.R && c < a.d) q[r] = load4<VEC>(a.q.p + ca_row(a.q, a, bh, r) + c, a.d - c);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[r][e] *= a.scale_log2;
    m[r] = -INFINITY;
    l[r] = 0.f;
  }
  for (int b = k0 + wave * U * kGroups; b < k1; b += kWaves * U * kGroups) {
    f32x4 kf[U], vf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = b + u * kGroups + sub;
      kf[u] = vf[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (key < k1 && c < a.d) {
        kf[u] = load4<VEC>(K + (int64_t)key * a.k.st + c, a.d - c);
        vf[u] = load4<VEC>(V + (int64_t)key * a.v.st + c, a.d - c);
      }
    }
#pragma unroll
    for (int r = 0; r < RQ; ++r) {
      float s[U], mn = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float x = lanes_sum<LPK>(kf[u][0] * q[r][0] + kf[u][1] * q[r][1] + kf[u][2] * q[r][2] + kf[u][3] * q[r][3]);
        s[u] = b + u * kGroups + sub < k1 ? x : -INFINITY;
        mn = fmaxf(mn, s[u]);
      }
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2(m[r] - mu);
      l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = fast_exp2(s[u] - mu);
        l[r] += p;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] += p * vf[u][e];
      }
      m[r] = mn;
    }
  }

  // The wave's groups, then the waves.
  __shared__ f32x4 sacc[kWaves][RQ][LPK];
  __shared__ float sm[kWaves][RQ], sl[kWaves][RQ];
#pragma unroll
  for (int r = 0; r < RQ; ++r) {
    float mw = m[r];
#pragma unroll
    for (int o = LPK; o < kWave; o *= 2) mw = fmaxf(mw, __shfl_xor(mw, o, kWave));
    const float f = fast_exp2(m[r] - (mw == -INFINITY ? 0.f : mw));
    float lw = l[r] * f;
    f32x4 aw;
#pragma unroll
    for (int e = 0; e < 4; ++e) aw[e] = acc[r][e] * f;
#pragma unroll
    for (int o = LPK; o < kWave; o *= 2) {
      lw += __shfl_xor(lw, o, kWave);
#pragma unroll
      for (int e = 0; e < 4; ++e) aw[e] += __shfl_xor(aw[e], o, kWave);
    }
    if (sub == 0) sacc[wave][r][lane] = aw;
    if (lane == 0) {
      sm[wave][r] = mw;
      sl[wave][r] = lw;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < RQ * LPK; i += 256) {
    const int r = i / LPK, cc = 4 * (i % LPK);
    if (r >= a.R) continue;
    float mx = sm[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mx = fmaxf(mx, sm[w][r]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ls = 0.f;
    f32x4 os = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(sm[w][r] - mu);
      ls += sl[w][r] * f;
#pragma unroll
      for (int e = 0; e < 4; ++e) os[e] += sacc[w][r][i % LPK][e] * f;
    }
    const float inv = ls == 0.f ? 0.f : 1.0f / ls;
#pragma unroll
    for (int e = 0; e < 4; ++e) os[e] *= inv;
    if (a.splits > 1) {
      const int64_t row = ((int64_t)bh * a.splits + part) * a.R + r;
      *reinterpret_cast<f32x4*>(a.part_o + row * (4 * LPK) + cc) = os;
      if (cc == 0) a.part_l[row] = mx + log2f(ls);
    } else {
      if (cc < a.d) store4<VEC>(a.o.p + ca_row(a.o, a, bh, r) + cc, os, a.d - cc);
      if (cc == 0) a.lse[(int64_t)bh * a.R + r] = (mx + log2f(ls)) * kLn2;
    }
  }
}

// The gradients of up to RQ query rows a key/value head, bound by the bytes of K, V, dK
// and dV like the forward by K's and V's: a key's row gives its scores and dP, hence its
// dK and dV, and its share of dQ, in one pass.  dQ's sums meet as the forward's do.
// 17 x 4 heads' single rows over 4340 keys, d 128 (604 MB): 100 us, 6.0 TB/s, and 7 us
// for dQ's parts; the tiles' kernels, 31 of their 32 rows empty, take 420.
template <int RQ, int LPK, bool VEC>
__global__ void __launch_bounds__(256)
cross_bwd_rows_kernel(const CaArgs a) {
  constexpr int U = RQ >= 8 ? 2 : 4;
  constexpr int kGroups = kWave / LPK;
  constexpr int kWaves = 4;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane / LPK, c = 4 * (lane % LPK);
  const int bh = blockIdx.x % a.BH, part = blockIdx.x / a.BH;
  const int len = ca_len(a, bh);
  const int k0 = part * a.chunk, k1 = min(len, k0 + a.chunk), end = min(a.Tk, k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);
  float* __restrict__ dK = ca_head(a.dk, a, bh);
  float* __restrict__ dV = ca_head(a.dv, a, bh);

  f32x4 q[RQ], g[RQ], dq[RQ];
  float l2[RQ], D[RQ];
#pragma unroll
  for (int r = 0; r < RQ; ++r) {
    q[r] = g[r] = dq[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    f32x4 o = q[r];
    l2[r] = INFINITY;
    if (r < a.R) {
      if (c < a.d) {
        q[r] = load4<VEC>(a.q.p + ca_row(a.q, a, bh, r) + c, a.d - c);
        g[r] = load4<VEC>(a.dout.p + ca_row(a.dout, a, bh, r) + c, a.d - c);
        o = load4<VEC>(a.o_in.p + ca_row(a.o_in, a, bh, r) + c, a.d - c);
      }
      l2[r] = a.lse[(int64_t)bh * a.R + r] * kLog2e;
      if (l2[r] == -INFINITY) l2[r] = INFINITY;  // a row without keys has P = 0
    }
    D[r] = lanes_sum<LPK>(g[r][0] * o[0] + g[r][1] * o[1] + g[r][2] * o[2] + g[r][3] * o[3]);
  }
  for (int b = k0 + wave * U * kGroups; b < end; b += kWaves * U * kGroups) {
    f32x4 kf[U], vf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = b + u * kGroups + sub;
      kf[u] = vf[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (key < k1 && c < a.d) {
        kf[u] = load4<VEC>(K + (int64_t)key * a.k.st + c, a.d - c);
        vf[u] = load4<VEC>(V + (int64_t)key * a.v.st + c, a.d - c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = b + u * kGroups + sub;
      f32x4 dk = {0.f, 0.f, 0.f, 0.f}, dv = dk;
#pragma unroll
      for (int r = 0; r < RQ; ++r) {
        const float s = lanes_sum<LPK>(kf[u][0] * q[r][0] + kf[u][1] * q[r][1] + kf[u][2] * q[r][2] + kf[u][3] * q[r][3]);
        const float dp = lanes_sum<LPK>(vf[u][0] * g[r][0] + vf[u][1] * g[r][1] + vf[u][2] * g[r][2] + vf[u][3] * g[r][3]);
        if (r >= a.R || key >= k1) continue;
        const float p = fast_exp2(s * a.scale_log2 - l2[r]), ds = p * (dp - D[r]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dk[e] += ds * q[r][e];
          dv[e] += p * g[r][e];
          dq[r][e] += ds * kf[u][e];
        }
      }
      if (key < end && c < a.d) {
        store4<VEC>(dK + (int64_t)key * a.dk.st + c, dk * a.scale, a.d - c);
        store4<VEC>(dV + (int64_t)key * a.dv.st + c, dv, a.d - c);
      }
    }
  }

  // The wave's groups, then the waves.
  __shared__ f32x4 sdq[kWaves][RQ][LPK];
#pragma unroll
  for (int r = 0; r < RQ; ++r) {
#pragma unroll
    for (int o = LPK; o < kWave; o *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) dq[r][e] += __shfl_xor(dq[r][e], o, kWave);
    if (sub == 0) sdq[wave][r][lane] = dq[r];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < RQ * LPK; i += 256) {
    const int r = i / LPK, cc = 4 * (i % LPK);
    if (r >= a.R) continue;
    f32x4 x = sdq[0][r][i % LPK];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x += sdq[w][r][i % LPK];
    x *= a.scale;
    if (a.splits > 1) {
      *reinterpret_cast<f32x4*>(a.dq_part + (((int64_t)part * a.BH + bh) * a.R + r) * (4 * LPK) + cc) = x;
    } else if (cc < a.d) {
      store4<VEC>(a.dq.p + ca_row(a.dq, a, bh, r) + cc, x, a.d - cc);
    }
  }
}

// The parts of every query row: with L_p = m_p + log2(l_p) and M their largest,
//   O = sum_p 2^(L_p - M) O_p / W,  lse = (M + log2 W) ln 2,  W = sum_p 2^(L_p - M);
// a row without keys has M = -inf.  DP / 4 lanes a row.
template <int DP, bool VEC>
__global__ void __launch_bounds__(256)
cross_combine_kernel(const CaArgs a) {
  constexpr int kLanes = DP / 4;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = u / kLanes;
  if (row >= (int64_t)a.BH * a.R) return;
  const int c = (int)(u % kLanes) * 4;
  const int bh = (int)(row / a.R), r = (int)(row % a.R);
  const float* L = a.part_l + (int64_t)bh * a.splits * a.R + r;
  const float* O = a.part_o + ((int64_t)bh * a.splits * a.R + r) * DP + c;
  float mx = -INFINITY;
  for (int p = 0; p < a.splits; ++p) mx = fmaxf(mx, L[(int64_t)p * a.R]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float w = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {
    const float f = fast_exp2(L[(int64_t)p * a.R] - mu);
    const f32x4 x = *reinterpret_cast<const f32x4*>(O + (int64_t)p * a.R * DP);
    w += f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += f * x[e];
  }
  const float inv = w == 0.f ? 0.f : 1.0f / w;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  if (c < a.d) store4<VEC>(a.o.p + ca_row(a.o, a, bh, r) + c, o, a.d - c);
  if (c == 0) a.lse[row] = (mx + log2f(w)) * kLn2;
}

// ------------------------------------------------------------------- forward

// A workgroup takes 128 query rows (32 a wave, a lane its row) and its key range,
// 32 keys at a time: S^T = K Q^T leaves a lane 16 keys of its row, whose online
// softmax is in registers but for one exchange with lane ^ 32, and P feeds
// O^T += V^T P^T from the registers it is left in.  This form and its gradients run
// for unaligned rows (and those further apart than a tile's reads below allow), bound by
// the fp32 matrix instruction: 8 x 12 heads, 1024 x 4096, d 64, aligned, took 934 us,
// 110 TFLOP/s of the 153 that a large fp32 product reaches.
template <int DP>
__global__ void __launch_bounds__(kFaThreads)
cross_fwd_kernel(const CaArgs a) {
  constexpr int NC = DP / 8;
  constexpr int NB = DP / 32;
  constexpr int LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float ks[2][kTile * LD];
  __shared__ __attribute__((aligned(16))) float vts[2][DP * kLdt];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH;
  const int rest = blockIdx.x / a.BH;
  const int part = rest % a.splits, qb = rest / a.splits;
  const int len = ca_len(a, bh);
  const int k0 = part * a.chunk, k1 = min(len, k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);
  const int qi = qb * kBlock + wave * kTile + lr;  // this lane's row

  f32x4 qr[NC];
  const float* Q = a.q.p + (qi < a.R ? ca_row(a.q, a, bh, qi) : 0);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int dd = 8 * c + 4 * h;
    qr[c] = qi < a.R ? load4<false>(Q + dd, a.d - dd) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = zero16();
  float m = -INFINITY, l = 0.f;
  const int ntiles = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  const bool work = qb * kBlock + wave * kTile < a.R;

  TileCopy<DP, false> kc, vc;
  if (ntiles > 0) {
    kc.load(K, a.k.st, k0, k1, a.d, tid);
    vc.load(V, a.v.st, k0, k1, a.d, tid);
    kc.template store<LD>(ks[0], tid);
    vc.template store_t<kLdt, true>(vts[0], tid);
  }
  __syncthreads();
  for (int t = 0; t < ntiles; ++t) {
    const int kv0 = k0 + t * kTile;
    const bool has_next = t + 1 < ntiles;
    if (has_next) {
      kc.load(K, a.k.st, kv0 + kTile, k1, a.d, tid);
      vc.load(V, a.v.st, kv0 + kTile, k1, a.d, tid);
    }
    if (work) {
      const float* kt = ks[t & 1];
      const float* vt = vts[t & 1];
      f32x16 s = zero16();
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const f32x4 kf = *reinterpret_cast<const f32x4*>(kt + lr * LD + 8 * c + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = mfma32(kf[e], qr[c][e], s);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = kv0 + acc_row(r, h) < k1 ? s[r] * a.scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[r]);
      }
      mx = half_swap_max(mx);
      const float mn = fmaxf(m, mx);
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2(m - mu);
      float ps = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = fast_exp2(s[r] - mu);
        ps += s[r];
      }
      l = l * alpha + half_swap_sum(ps);
      m = mn;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int col = b * 32 + lr;
          const f32x4 vf = *reinterpret_cast<const f32x4*>(vt + col * kLdt + vt_swz<true>(col, 8 * g + 4 * h));
#pragma unroll
          for (int e = 0; e < 4; ++e) o[b] = mfma32(vf[e], s[4 * g + e], o[b]);
        }
      }
    }
    if (has_next) {
      kc.template store<LD>(ks[(t + 1) & 1], tid);
      vc.template store_t<kLdt, true>(vts[(t + 1) & 1], tid);
    }
    __syncthreads();
  }
  if (qi < a.R) ca_store_row<DP, false>(a, bh, part, qi, h, o, m, l);
}

// ------------------------------------------------------------------ backward

// dQ, and D of the rows for the dK/dV pass: a workgroup takes 128 query rows with
// q and dO in registers and walks the keys: S^T, dP^T (lane = row), dS, dQ^T +=
// K^T dS^T.
template <int DP>
__global__ void __launch_bounds__(kFaThreads)
cross_bwd_dq_kernel(const CaArgs a) {
  constexpr int NC = DP / 8;
  constexpr int NB = DP / 32;
  constexpr int LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float ks[2][kTile * LD];
  __shared__ __attribute__((aligned(16))) float vs[2][kTile * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, rest = blockIdx.x / a.BH;
  const int part = rest % a.splits, qb = rest / a.splits;
  const int k0 = part * a.chunk, k1 = min(ca_len(a, bh), k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);
  const int qi = qb * kBlock + wave * kTile + lr;
  const bool row_ok = qi < a.R;

  f32x4 qr[NC], dor[NC];
  float dsum = 0.f;
  {
    const float* Q = a.q.p + (row_ok ? ca_row(a.q, a, bh, qi) : 0);
    const float* dO = a.dout.p + (row_ok ? ca_row(a.dout, a, bh, qi) : 0);
    const float* O = a.o_in.p + (row_ok ? ca_row(a.o_in, a, bh, qi) : 0);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int dd = 8 * c + 4 * h;
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      qr[c] = row_ok ? load4<false>(Q + dd, a.d - dd) : z;
      dor[c] = row_ok ? load4<false>(dO + dd, a.d - dd) : z;
      const f32x4 of = row_ok ? load4<false>(O + dd, a.d - dd) : z;
#pragma unroll
      for (int e = 0; e < 4; ++e) dsum += dor[c][e] * of[e];
    }
  }
  dsum = half_swap_sum(dsum);
  // A row without keys, or past the end, has P = 0.
  float l2 = row_ok ? a.lse[(int64_t)bh * a.R + qi] * kLog2e : INFINITY;
  if (l2 == -INFINITY) l2 = INFINITY;
  if (row_ok && h == 0 && part == 0) a.D[(int64_t)bh * a.R + qi] = dsum;
  f32x16 dq[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dq[b] = zero16();
  const int ntiles = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  const bool work = qb * kBlock + wave * kTile < a.R;

  TileCopy<DP, false> kc, vc;
  if (ntiles > 0) {
    kc.load(K, a.k.st, k0, k1, a.d, tid);
    vc.load(V, a.v.st, k0, k1, a.d, tid);
    kc.template store<LD>(ks[0], tid);
    vc.template store<LD>(vs[0], tid);
  }
  __syncthreads();
  for (int t = 0; t < ntiles; ++t) {
    const int kv0 = k0 + t * kTile;
    const bool has_next = t + 1 < ntiles;
    if (has_next) {
      kc.load(K, a.k.st, kv0 + kTile, k1, a.d, tid);
      vc.load(V, a.v.st, kv0 + kTile, k1, a.d, tid);
    }
    if (work) {
      const float* kt = ks[t & 1];
      const float* vt = vs[t & 1];
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const f32x4 kf = *reinterpret_cast<const f32x4*>(kt + lr * LD + 8 * c + 4 * h);
        const f32x4 vf = *reinterpret_cast<const f32x4*>(vt + lr * LD + 8 * c + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s = mfma32(kf[e], qr[c][e], s);
          dp = mfma32(vf[e], dor[c][e], dp);
        }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool in = kv0 + acc_row(r, h) < k1;
        const float p = fast_exp2(s[r] * a.scale_log2 - l2);
        dp[r] = in ? p * (dp[r] - dsum) : 0.f;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int st = 0; st < 16; ++st) dq[b] = mfma32(kt[acc_row(st, h) * LD + b * 32 + lr], dp[st], dq[b]);
      }
    }
    if (has_next) {
      kc.template store<LD>(ks[(t + 1) & 1], tid);
      vc.template store<LD>(vs[(t + 1) & 1], tid);
    }
    __syncthreads();
  }
  if (row_ok) ca_store_dq<DP, false>(a, bh, part, qi, dq, h);
}

// A [32][DP] tile of query rows (TileCopy over rows that may cross heads).
template <int DP>
struct CaRowTile : TileCopy<DP, false> {
  using Base = TileCopy<DP, false>;
  __device__ __forceinline__ void load_rows(const FaIn& x, const CaArgs& a, int bh, int row0, int tid) {
#pragma unroll
    for (int i = 0; i < Base::kPer; ++i) {
      const int u = tid + i * kFaThreads;
      const int r = row0 + u / (DP / 4);
      const int c = (u % (DP / 4)) * 4;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (u < Base::kUnits && r < a.R) v = load4<false>(x.p + ca_row(x, a, bh, r) + c, a.d - c);
      Base::reg[i] = v;
    }
  }
};

// dK and dV: a workgroup takes 128 keys (32 a wave, a lane its key, k and v in
// registers) and walks the query rows: S, dP (lane = key), P, dS, dV^T += dO^T P,
// dK^T += Q^T dS.
template <int DP>
__global__ void __launch_bounds__(kFaThreads, DP <= 64 ? 2 : 1)
cross_bwd_dkdv_kernel(const CaArgs a) {
  constexpr int NC = DP / 8;
  constexpr int NB = DP / 32;
  constexpr int LD = DP + 4;
  __shared__ __attribute__((aligned(16))) float qs[2][kTile * LD];
  __shared__ __attribute__((aligned(16))) float dos[2][kTile * LD];
  __shared__ __attribute__((aligned(16))) float ls[2][kTile];
  __shared__ __attribute__((aligned(16))) float ds[2][kTile];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, rest = blockIdx.x / a.BH;
  const int part = rest % a.kv_splits, kb = rest / a.kv_splits;
  const int len = ca_len(a, bh);
  const int kw = kb * kBlock + wave * kTile;  // the wave's first key
  const int kj = kw + lr;
  const bool key_ok = kj < len;
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);

  f32x4 kr[NC], vr[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int dd = 8 * c + 4 * h;
    kr[c] = key_ok ? load4<false>(K + (int64_t)kj * a.k.st + dd, a.d - dd) : f32x4{0.f, 0.f, 0.f, 0.f};
    vr[c] = key_ok ? load4<false>(V + (int64_t)kj * a.v.st + dd, a.d - dd) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
  // a workgroup whose keys are all masked only writes zeros
  const int t0 = part * a.kv_tiles;
  const int t1 = kb * kBlock < len ? min((a.R + kTile - 1) / kTile, t0 + a.kv_tiles) : t0;

  CaRowTile<DP> qc, dc;
  float lreg = 0.f, dreg = 0.f;
  auto load_tile = [&](int t) {
    qc.load_rows(a.q, a, bh, t * kTile, tid);
    dc.load_rows(a.dout, a, bh, t * kTile, tid);
    if (tid < kTile) {
      const int r = t * kTile + tid;
      lreg = r < a.R ? a.lse[(int64_t)bh * a.R + r] * kLog2e : INFINITY;
      if (lreg == -INFINITY) lreg = INFINITY;
      dreg = r < a.R ? a.D[(int64_t)bh * a.R + r] : 0.f;
    }
  };
  auto store_tile = [&](int buf) {
    qc.template store<LD>(qs[buf], tid);
    dc.template store<LD>(dos[buf], tid);
    if (tid < kTile) {
      ls[buf][tid] = lreg;
      ds[buf][tid] = dreg;
    }
  };
  if (t0 < t1) {
    load_tile(t0);
    store_tile(0);
  }
  __syncthreads();
  for (int t = t0; t < t1; ++t) {
    const int cur = (t - t0) & 1;
    const bool has_next = t + 1 < t1;
    if (has_next) load_tile(t + 1);
    if (kw < len) {
      const float* qt = qs[cur];
      const float* dot = dos[cur];
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const f32x4 qf = *reinterpret_cast<const f32x4*>(qt + lr * LD + 8 * c + 4 * h);
        const f32x4 df = *reinterpret_cast<const f32x4*>(dot + lr * LD + 8 * c + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s = mfma32(qf[e], kr[c][e], s);
          dp = mfma32(df[e], vr[c][e], dp);
        }
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(&ls[cur][8 * g + 4 * h]);
        const f32x4 d4 = *reinterpret_cast<const f32x4*>(&ds[cur][8 * g + 4 * h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          const float p = key_ok ? fast_exp2(s[r] * a.scale_log2 - l4[e]) : 0.f;
          s[r] = p;
          dp[r] = key_ok ? p * (dp[r] - d4[e]) : 0.f;
        }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int st = 0; st < 16; ++st) {
          const int q = acc_row(st, h);
          dv[b] = mfma32(dot[q * LD + b * 32 + lr], s[st], dv[b]);
          dk[b] = mfma32(qt[q * LD + b * 32 + lr], dp[st], dk[b]);
        }
      }
    }
    if (has_next) store_tile(cur ^ 1);
    __syncthreads();
  }
  if (kj < a.Tk) ca_store_key<DP, false>(a, bh, part, kj, key_ok, dk, dv, h);
}

// ---------------------------------------------------- on the fp16 matrix cores
// The same passes with every operand in two fp16 parts: x 2^e = hi + lo, hi rounded
// from x 2^e and lo from what that leaves, so that three matrix ops (lo hi, hi lo,
// hi hi; 16 steps each at 16 times the fp32 instruction's rate) stand for one
// fp32 product.  An operand is off by at most 2^-22 of itself or, where that is more,
// 2^-38 of its row's largest element, lo lo is at most 2^-22 of a product and is left
// out; sums are in fp32, with fewer roundings than the fp32 instruction's, which
// leaves the results nearer to the exact ones.  8 x 12 heads, 1024 x 4096, d 64 (in
// brackets with the fp32 instruction): forward 392 us (934), dQ 575 (1276), dK/dV 820
// (1730), off by 0.76e-6 (1.2e-6) in O's norm, 1.0e-6 (1.3e-6) in dQ's, 0.80e-6
// (0.88e-6) in dK's and dV's.  That is 263 TFLOP/s of the forward's products, 789 on the
// cores.  Three bf16 parts and six products hold all 24 bits, but took 590, 806 and 1125
// us.  What bounds these is that a wave's matrix ops and its vector instructions (scales,
// exponentials, splits) wait for each other: the forward's matrix units are busy for 40 %
// of the cycles and its vector units for 64 %, dQ's for 39 and 45, dK/dV's for 37 and 49,
// at 1.9 to 2.0 GHz.
//
// e is a row's own, such that its largest element is in [2^13, 2^14).  Over the head
// dim a row's factor is one of the output's row or column.  Over a tile's rows it
// goes to the other operand, P or dS, which is scaled by the lane's own power of two
// that follows the largest |P| 2^-e (|dS| 2^-e) so far: what is rounded there is at
// most 2^-38 of the largest term of the lane's sum, or 2^-150 where that is more.
//
// What a wave keeps in registers for all tiles (q; q and dO; k and v) is split once; a
// tile is split on its way into LDS, once a workgroup, as two row-major planes.
// Products over the head dim read rows of them; products over the tile's rows (V^T
// P^T, K^T dS^T, dO^T P, Q^T dS) read columns through the transposing LDS read, so a
// tile that serves both is split and stored once.  P and dS are split in the
// registers the softmax leaves them in.  Rows whose largest element is outside
// [2^-99, 2^60) (infinities too) are not held so: the waves that meet one do their
// rows again with the fp32 instruction, from HBM, at a tenth of the speed.  8 x 12 heads,
// 512 x 1024, forward + backward 293 us, with a row of dO of 2^-110 in every head 1773,
// with an infinite value in every head 2826.

// Forward.  The running maximum m of a row follows its scores only when they pass it
// by 2^4, so O is rarely rescaled; when it moves, the scale of P is found again.
template <int DP>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 3 : 2)
cross_fwd_split_kernel(const CaArgs a) {
  using Tile = HalfTile<DP>;
  constexpr int NB = DP / 32;
  __shared__ __attribute__((aligned(16))) char ks[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char vs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float kf[2][kTile], vf[2][kTile];  // the rows' factors
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH;
  const int rest = blockIdx.x / a.BH;
  const int part = rest % a.splits, qb = rest / a.splits;
  const int len = ca_len(a, bh);
  const int k0 = part * a.chunk, k1 = min(len, k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);
  const int qi = qb * kBlock + wave * kTile + lr;  // this lane's row
  const bool work = qb * kBlock + wave * kTile < a.R;
  const float* Q = qi < a.R ? a.q.p + ca_row(a.q, a, bh, qi) : nullptr;
  if (tid == 0) not_held = 0;

  u32x4 qp[DP / 16][2];
  bool row_bad = false, bad = false;
  const float qf = half_row<DP>(Q, a.d, a.scale_log2, h, qp, row_bad);
  f32x16 o[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) o[b] = zero16();
  float m = -INFINITY, l = 0.f;
  HalfScale<NB> fit;

  auto follow = [&](float mx, float slack) {
    mx = half_swap_max(mx);
    const bool move = mx > m + slack;
    if (!__any(move)) return;
    const float alpha = move ? fast_exp2(m - mx) : 1.f;
    if (move) {
      m = mx;
      fit.most = -1.f;
    }
    l *= alpha;
    fit.big *= alpha;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int r = 0; r < 16; ++r) o[b][r] *= alpha;
    }
  };
  auto compute = [&](int buf, int kv0) {
    f32x16 s = half_rows<DP>(ks[buf], qp, lr, h);
    float mx = -INFINITY, ps = 0.f, top = 0.f;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 k4 = row_values(kf[buf], g, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * g + e] *= k4[e];
    }
    if (kv0 + kTile > k1) {
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (kv0 + acc_row(r, h) >= k1) s[r] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
    follow(mx * qf, 4.f);
    const float mu = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v4 = row_values(vf[buf], g, h);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = fast_exp2(s[4 * g + e] * qf - mu);
        ps += p;
        s[4 * g + e] = p * v4[e];
        top = fmaxf(top, s[4 * g + e]);
      }
    }
    l += half_swap_sum(ps);
    fit.follow(top, o, row_bad);
    half_cols<DP>(vs[buf], s, fit.f, 0, lane, o);
    half_cols<DP>(vs[buf], s, fit.f, 1, lane, o);
  };

  const int ntiles = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  Tile kc[2], vc[2];
  const typename Tile::Place kat(a.k.st, a.d, tid), vat(a.v.st, a.d, tid);
  auto load = [&](int i, int t) {
    const int row0 = k0 + t * kTile;
    kc[i].load(K + (int64_t)row0 * a.k.st, a.k.st, k1 - row0, a.d, kat);
    vc[i].load(V + (int64_t)row0 * a.v.st, a.v.st, k1 - row0, a.d, vat);
  };
  auto store = [&](int i, int buf) {
    kc[i].store(ks[buf], tid, bad);
    vc[i].store(vs[buf], tid, bad);
    if (Tile::col(tid) != 0) return;
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      const int r = Tile::row(n, tid);
      kf[buf][r] = row_factor(kc[i].ex[n]);
      vf[buf][r] = row_factor(vc[i].ex[n]);
    }
  };
  if (ntiles > 0) {
    load(0, 0);
    load(1, 1);
    store(0, 0);
    load(0, 2);
  }
  lds_barrier();
  // Iteration t: tile t in LDS, t + 1 in registers, t + 2 on its way, t + 3 sent for.
  for (int t = 0; t < ntiles; t += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u >= ntiles) break;
      if (work) compute(u, k0 + (t + u) * kTile);
      store(1 - u, 1 - u);
      load(1 - u, t + u + 3);
      lds_barrier();
    }
  }
  fit.undo(o);

  if (bad) not_held = 1;
  __syncthreads();
  if (work && ntiles > 0 && __any(row_bad || not_held)) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = zero16();
    for (int t = 0; t < ntiles; ++t) {
      const int kv0 = k0 + t * kTile;
      f32x16 s = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d;
        s = mfma32(in && kv0 + lr < k1 ? K[(int64_t)(kv0 + lr) * a.k.st + c + h] : 0.f,
                   in && Q ? Q[c + h] * a.scale_log2 : 0.f, s);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (kv0 + acc_row(r, h) >= k1) s[r] = -INFINITY;
        mx = fmaxf(mx, s[r]);
      }
      follow(mx, 0.f);
      const float mu = m == -INFINITY ? 0.f : m;
      float ps = 0.f;
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
          o[b] = mfma32(row < k1 && col < a.d ? V[(int64_t)row * a.v.st + col] : 0.f, s[st], o[b]);
        }
      }
    }
  }
  if (qi < a.R) ca_store_row<DP, true>(a, bh, part, qi, h, o, m, l);
}

// dQ (and D).
template <int DP>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 3 : 1)
cross_bwd_dq_split_kernel(const CaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char ks[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char vs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float kf[2][kTile], vf[2][kTile];  // the rows' factors
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, rest = blockIdx.x / a.BH;
  const int part = rest % a.splits, qb = rest / a.splits;
  const int k0 = part * a.chunk, k1 = min(ca_len(a, bh), k0 + a.chunk);
  const float* __restrict__ K = ca_head(a.k, a, bh);
  const float* __restrict__ V = ca_head(a.v, a, bh);
  const int qi = qb * kBlock + wave * kTile + lr;
  const bool row_ok = qi < a.R, work = qb * kBlock + wave * kTile < a.R;
  const float* Q = row_ok ? a.q.p + ca_row(a.q, a, bh, qi) : nullptr;
  const float* dO = row_ok ? a.dout.p + ca_row(a.dout, a, bh, qi) : nullptr;
  if (tid == 0) not_held = 0;

  float dsum = 0.f;
  if (row_ok) {
    const float* O = a.o_in.p + ca_row(a.o_in, a, bh, qi);
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      const int dd = 8 * c + 4 * h;
      if (dd < a.d) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(dO + dd), y = *reinterpret_cast<const f32x4*>(O + dd);
        dsum += x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3];
      }
    }
  }
  dsum = half_swap_sum(dsum);
  float l2 = row_ok ? a.lse[(int64_t)bh * a.R + qi] * kLog2e : INFINITY;
  if (l2 == -INFINITY) l2 = INFINITY;  // a row without keys has P = 0
  if (row_ok && h == 0 && part == 0) a.D[(int64_t)bh * a.R + qi] = dsum;

  u32x4 qp[DP / 16][2], dop[DP / 16][2];
  bool row_bad = false, bad = false;
  const float qf = half_row<DP>(Q, a.d, a.scale_log2, h, qp, row_bad);
  const float df = half_row<DP>(dO, a.d, 1.f, h, dop, row_bad);
  f32x16 dq[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dq[b] = zero16();
  HalfScale<NB> fit;

  const int ntiles = k1 > k0 ? (k1 - k0 + kTile - 1) / kTile : 0;
  Tile kc, vc;
  const typename Tile::Place kat(a.k.st, a.d, tid), vat(a.v.st, a.d, tid);
  auto load = [&](int t) {
    const int row0 = k0 + t * kTile;
    kc.load(K + (int64_t)row0 * a.k.st, a.k.st, k1 - row0, a.d, kat);
    vc.load(V + (int64_t)row0 * a.v.st, a.v.st, k1 - row0, a.d, vat);
  };
  auto store = [&](int buf) {
    kc.store(ks[buf], tid, bad);
    vc.store(vs[buf], tid, bad);
    if (Tile::col(tid) != 0) return;
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      const int r = Tile::row(n, tid);
      kf[buf][r] = row_factor(kc.ex[n]);
      vf[buf][r] = row_factor(vc.ex[n]);
    }
  };
  if (ntiles > 0) {
    load(0);
    store(0);
  }
  lds_barrier();
  for (int t = 0; t < ntiles; ++t) {
    const int buf = t & 1, kv0 = k0 + t * kTile;
    const bool has_next = t + 1 < ntiles;
    if (has_next) load(t + 1);
    if (work) {
      const f32x16 s = half_rows<DP>(ks[buf], qp, lr, h);
      f32x16 dp = half_rows<DP>(vs[buf], dop, lr, h);
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 k4 = row_values(kf[buf], g, h), v4 = row_values(vf[buf], g, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          const float p = fast_exp2(s[r] * k4[e] * qf - l2);
          dp[r] = p * (dp[r] * v4[e] * df - dsum) * k4[e];
        }
      }
      if (kv0 + kTile > k1) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kv0 + acc_row(r, h) >= k1) dp[r] = 0.f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(dp[r]));
      fit.follow(top, dq, row_bad);
      half_cols<DP>(ks[buf], dp, fit.f, 0, lane, dq);
      half_cols<DP>(ks[buf], dp, fit.f, 1, lane, dq);
    }
    if (has_next) store(buf ^ 1);
    lds_barrier();
  }
  fit.undo(dq);

  if (bad) not_held = 1;
  __syncthreads();
  if (work && ntiles > 0 && __any(row_bad || not_held)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) dq[b] = zero16();
    for (int t = 0; t < ntiles; ++t) {
      const int kv0 = k0 + t * kTile;
      f32x16 s = zero16(), dp = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d, key = in && kv0 + lr < k1;
        s = mfma32(key ? K[(int64_t)(kv0 + lr) * a.k.st + c + h] : 0.f, in && Q ? Q[c + h] * a.scale_log2 : 0.f, s);
        dp = mfma32(key ? V[(int64_t)(kv0 + lr) * a.v.st + c + h] : 0.f, in && dO ? dO[c + h] : 0.f, dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = fast_exp2(s[r] - l2) * (dp[r] - dsum);
        dp[r] = kv0 + acc_row(r, h) < k1 ? x : 0.f;
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int col = b * 32 + lr;
#pragma unroll
        for (int st = 0; st < 16; ++st) {
          const int row = kv0 + acc_row(st, h);
          dq[b] = mfma32(row < k1 && col < a.d ? K[(int64_t)row * a.k.st + col] : 0.f, dp[st], dq[b]);
        }
      }
    }
  }
  if (row_ok) ca_store_dq<DP, true>(a, bh, part, qi, dq, h);
}

// dK and dV.
template <int DP>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 2 : 1)
cross_bwd_dkdv_split_kernel(const CaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char qs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char dos[2][Tile::kBytes];
  // factors of Q's rows and of dO's; lse in log2 and D
  __shared__ __attribute__((aligned(16))) float qf[2][kTile], df[2][kTile], ls[2][kTile], ds[2][kTile];
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, rest = blockIdx.x / a.BH;
  const int part = rest % a.kv_splits, kb = rest / a.kv_splits;
  const int len = ca_len(a, bh);
  const int kw = kb * kBlock + wave * kTile;
  const int kj = kw + lr;
  const bool key_ok = kj < len, work = kw < len;
  const float* K = key_ok ? ca_head(a.k, a, bh) + (int64_t)kj * a.k.st : nullptr;
  const float* V = key_ok ? ca_head(a.v, a, bh) + (int64_t)kj * a.v.st : nullptr;
  if (tid == 0) not_held = 0;

  u32x4 kp[DP / 16][2], vp[DP / 16][2];
  bool key_bad = false, bad = false;
  const float kf = half_row<DP>(K, a.d, a.scale_log2, h, kp, key_bad);
  const float vf = half_row<DP>(V, a.d, 1.f, h, vp, key_bad);
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
  HalfScale<NB> fit_k, fit_v;
  const int t0 = part * a.kv_tiles;
  const int t1 = kb * kBlock < len ? min((a.R + kTile - 1) / kTile, t0 + a.kv_tiles) : t0;

  Tile qc, dc;
  const float* Q = ca_group(a.q, a, bh);
  const float* dO = ca_group(a.dout, a, bh);
  const typename Tile::Place qat(a.q.st, a.d, tid), oat(a.dout.st, a.d, tid);
  float lreg[Tile::kPer], dreg[Tile::kPer];
  auto lse_of = [&](int r) {
    const float x = r < a.R ? a.lse[(int64_t)bh * a.R + r] * kLog2e : INFINITY;
    return x == -INFINITY ? INFINITY : x;  // a row without keys, or past the end, has P = 0
  };
  auto d_of = [&](int r) { return r < a.R ? a.D[(int64_t)bh * a.R + r] : 0.f; };
  auto load = [&](int t) {
    const int row0 = t * kTile;
    if (a.G == 1) {
      qc.load(Q + (int64_t)row0 * a.q.st, a.q.st, a.R - row0, a.d, qat);
      dc.load(dO + (int64_t)row0 * a.dout.st, a.dout.st, a.R - row0, a.d, oat);
    } else {
      qc.load_heads(Q, a.q.sh, a.q.st, a.Tq, row0, a.R, a.d, tid);
      dc.load_heads(dO, a.dout.sh, a.dout.st, a.Tq, row0, a.R, a.d, tid);
    }
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      lreg[n] = dreg[n] = 0.f;
      if (Tile::col(tid) != 0) continue;
      lreg[n] = lse_of(row0 + Tile::row(n, tid));
      dreg[n] = d_of(row0 + Tile::row(n, tid));
    }
  };
  auto store = [&](int buf) {
    qc.store(qs[buf], tid, bad);
    dc.store(dos[buf], tid, bad);
    if (Tile::col(tid) != 0) return;
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      const int r = Tile::row(n, tid);
      qf[buf][r] = row_factor(qc.ex[n]);
      df[buf][r] = row_factor(dc.ex[n]);
      ls[buf][r] = lreg[n];
      ds[buf][r] = dreg[n];
    }
  };
  if (t0 < t1) {
    load(t0);
    store(0);
  }
  lds_barrier();
  for (int t = t0; t < t1; ++t) {
    const int cur = (t - t0) & 1;
    const bool has_next = t + 1 < t1;
    if (has_next) load(t + 1);
    if (work) {
      f32x16 s = half_rows<DP>(qs[cur], kp, lr, h);
      sched_fence();
      f32x16 x;
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 q4 = row_values(qf[cur], g, h), l4 = row_values(ls[cur], g, h), o4 = row_values(df[cur], g, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          s[r] = key_ok ? fast_exp2(s[r] * q4[e] * kf - l4[e]) : 0.f;
          x[r] = s[r] * o4[e];
          top = fmaxf(top, x[r]);
        }
      }
      fit_v.follow(top, dv, key_bad);
      half_cols<DP>(dos[cur], x, fit_v.f, 0, lane, dv);
      half_cols<DP>(dos[cur], x, fit_v.f, 1, lane, dv);
      x = half_rows<DP>(dos[cur], vp, lr, h);
      sched_fence();
      top = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 q4 = row_values(qf[cur], g, h), o4 = row_values(df[cur], g, h), d4 = row_values(ds[cur], g, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          // P before Q's scale: dP - D is finite for all rows that are held, its product with that need not be
          x[r] = s[r] * (x[r] * o4[e] * vf - d4[e]) * q4[e];
          top = fmaxf(top, fabsf(x[r]));
        }
      }
      fit_k.follow(top, dk, key_bad);
      half_cols<DP>(qs[cur], x, fit_k.f, 0, lane, dk);
      half_cols<DP>(qs[cur], x, fit_k.f, 1, lane, dk);
    }
    if (has_next) store(cur ^ 1);
    lds_barrier();
  }
  fit_v.undo(dv);
  fit_k.undo(dk);

  if (bad) not_held = 1;
  __syncthreads();
  if (work && t0 < t1 && __any(key_bad || not_held)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
    for (int t = t0; t < t1; ++t) {
      const int row0 = t * kTile;
      const bool mine = row0 + lr < a.R;
      const float* Q = mine ? a.q.p + ca_row(a.q, a, bh, row0 + lr) : nullptr;
      const float* dO = mine ? a.dout.p + ca_row(a.dout, a, bh, row0 + lr) : nullptr;
      f32x16 s = zero16(), dp = zero16();
      for (int c = 0; c < a.d; c += 2) {
        const bool in = c + h < a.d;
        s = mfma32(in && Q ? Q[c + h] : 0.f, in && K ? K[c + h] * a.scale_log2 : 0.f, s);
        dp = mfma32(in && dO ? dO[c + h] : 0.f, in && V ? V[c + h] : 0.f, dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = row0 + acc_row(r, h);
        s[r] = key_ok ? fast_exp2(s[r] - lse_of(i)) : 0.f;
        dp[r] = key_ok ? s[r] * (dp[r] - d_of(i)) : 0.f;
      }
#pragma unroll
      for (int st = 0; st < 16; ++st) {
        const int r = row0 + acc_row(st, h);
        const int64_t qo = r < a.R ? ca_row(a.q, a, bh, r) : 0, oo = r < a.R ? ca_row(a.dout, a, bh, r) : 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const int col = b * 32 + lr;
          const bool in = r < a.R && col < a.d;
          dv[b] = mfma32(in ? a.dout.p[oo + col] : 0.f, s[st], dv[b]);
          dk[b] = mfma32(in ? a.q.p[qo + col] : 0.f, dp[st], dk[b]);
        }
      }
    }
  }
  if (kj < a.Tk) ca_store_key<DP, true>(a, bh, part, kj, key_ok, dk, dv, h);
}

// The parts of dQ (rows [0, n_q) of DP / 4 lanes), then of dK and dV, summed in order.
template <int DP, bool VEC>
__global__ void __launch_bounds__(256)
cross_bwd_sum_kernel(const CaArgs a) {
  constexpr int kLanes = DP / 4;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row = u / kLanes;
  const int c = (int)(u % kLanes) * 4;
  const int64_t nq = a.splits > 1 ? (int64_t)a.BH * a.R : 0, nk = a.kv_splits > 1 ? (int64_t)a.BH * a.Tk : 0;
  const float* part = a.dq_part;
  float* out;
  int64_t n = nq;
  int splits = a.splits;
  if (row < nq) {
    out = a.dq.p + ca_row(a.dq, a, (int)(row / a.R), (int)(row % a.R));
  } else {
    row -= nq;
    n = nk;
    splits = a.kv_splits;
    if (row >= 2 * nk) return;
    const bool v = row >= nk;
    if (v) row -= nk;
    part = v ? a.dv_part : a.dk_part;
    const FaOut& x = v ? a.dv : a.dk;
    out = ca_head(x, a, (int)(row / a.Tk)) + row % a.Tk * x.st;
  }
  if (c >= a.d) return;
  f32x4 s = *reinterpret_cast<const f32x4*>(part + row * DP + c);
  for (int p = 1; p < splits; ++p) s += *reinterpret_cast<const f32x4*>(part + (p * n + row) * DP + c);
  store4<VEC>(out + c, s, a.d - c);
}

// ------------------------------------------------------------------ host side

// Query rows a key/value head up to which cross_rows_kernel runs: 192 heads' 4 rows of
// 577 keys in 18 us against the tiles' 24; 8 rows would take 23 against 24 (of 4096
// keys 98 against 90).  And cross_bwd_rows_kernel, forward + backward: 4 rows of 577 keys
// 45 us against 80, 8 rows 58 against 81 (of 4096 keys 281 against 466).
constexpr int kFewRows = 4, kFewBwd = 8;
constexpr int kMaxSplits = 64;

int pad_dim(int64_t d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

// Ranges a pass's loop of `tiles` is split into, for grids that do not fill the
// GPU's `slots` workgroups.  A tile takes about `us` microseconds and a workgroup
// another two of its own, and parts cost a launch and their bytes twice; the fewest
// microseconds win.  Forward + backward of 2 x 8 heads' 512 x 4096, d 64, 188 us, unsplit
// 508; 36 x 6 heads' 1865 rows over 31 keys 346, 386; the forward of 4 x 16 heads on 4,
// 301 x 1111, d 128, 64, 91.  Full grids are not split: 64 x 6 heads, 256 x 577, 331 us,
// its 768 and 1920 workgroups as two parts each 489.  Two slots a CU, although the 64-wide
// forward and dQ fit three: with three 2 x 8 heads' 512 x 4096 takes 51 us forward against
// 48, 8 x 12 heads' 512 x 2048 and others the same.
int ca_splits(int64_t grid, int64_t slots, int64_t tiles, int64_t least, double us, double part_bytes) {
  int best = 1;
  double cost = 0;
  if (grid >= slots) return 1;
  for (int s = 1; s <= kMaxSplits && (s == 1 || tiles / s >= least); ++s) {
    const double t = std::max(1.0, (double)(grid * s) / slots) * ((double)ceil_div(tiles, s) * us + 2.0) +
                     (s > 1 ? 4.0 + s * part_bytes / 2.0e6 : 0.0);
    if (s == 1 || t < 0.97 * cost) {
      best = s;
      cost = t;
    }
  }
  return best;
}

// Key ranges of the few-row kernels, which live on loads in flight: four workgroups to
// a CU, in ranges of at least 64 keys.
int64_t few_splits(int64_t bh, int64_t Tk) {
  const int64_t cus = device_cu_count(), s = bh * 3 / 2 >= 4 * cus ? 1 : ceil_div(4 * cus, bh);
  return std::max<int64_t>(1, std::min<int64_t>({s, Tk / 64, (int64_t)kMaxSplits}));
}

// Key ranges of a forward, and their keys.
void ca_plan(int64_t bh, int64_t R, int64_t Tk, int64_t d, int* splits, int* chunk) {
  const int64_t cus = device_cu_count(), tiles = ceil_div(Tk, kTile);
  int64_t s;
  if (R <= kFewRows) {
    s = few_splits(bh, Tk);
  } else {
    s = ca_splits(bh * ceil_div(R, kBlock), 2 * cus, tiles, 4, d > 64 ? 4.0 : 2.0, (double)bh * R * pad_dim(d) * 4);
  }
  const int64_t c = ceil_div(std::max<int64_t>(tiles, 1), s);
  *chunk = (int)(c * kTile);
  *splits = (int)std::max<int64_t>(1, ceil_div(tiles, c));
}

// Whether the gradients are cross_bwd_rows_kernel's.
bool few_rows(const CaArgs& a) { return a.R > 0 && a.R <= kFewBwd && a.Tk > 0; }

// Key ranges of dQ and ranges of query rows of dK and dV.
void ca_bwd_plan(CaArgs& a) {
  const int64_t cus = device_cu_count(), kt = ceil_div((int64_t)a.Tk, kTile), qt = ceil_div((int64_t)a.R, kTile);
  const int64_t slots = (a.d > 64 ? 1 : 2) * cus, dp = pad_dim(a.d);
  int64_t s = few_rows(a) ? few_splits(a.BH, a.Tk)
                          : ca_splits(a.BH * ceil_div((int64_t)a.R, kBlock), slots, kt, 4, a.d > 64 ? 6.0 : 3.0,
                                      (double)a.BH * a.R * dp * 4);
  int64_t c = ceil_div(std::max<int64_t>(kt, 1), s);
  a.chunk = (int)(c * kTile);
  a.splits = (int)std::max<int64_t>(1, ceil_div(kt, c));
  s = few_rows(a) ? 1
                  : ca_splits(a.BH * ceil_div((int64_t)a.Tk, kBlock), slots, qt, 4, a.d > 64 ? 10.0 : 5.0,
                              (double)a.BH * a.Tk * dp * 8);
  c = ceil_div(std::max<int64_t>(qt, 1), s);
  a.kv_tiles = (int)c;
  a.kv_splits = (int)std::max<int64_t>(1, ceil_div(qt, c));
}

// The head dim that the tiled passes are built for.  They run on the fp16 matrix cores
// where rows are 16-byte aligned, with up to 64 floats padded to that.  Forward +
// backward of 384 heads' 256 x 300, d 64: 212 us against 391 with the fp32 instruction,
// 256 x 7: 86 against 102; 16 x 7 alone loses (27 against 24).  96 heads' 512 x 2048,
// d 32: 409 us against 527.
template <int DP, bool VEC>
constexpr int kTileDim = VEC && DP < 64 ? 64 : DP;

bool ca_shape_ok(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk) {
  const int64_t most = int64_t(1) << 24;
  if (B > most || H > most || Tq > most || Tk > most) return false;
  if (H / Hkv * Tq > most || B * Hkv > most) return false;
  // a dispatch holds its work items in 32 bits
  const int64_t q = B * Hkv * ceil_div(H / Hkv * Tq, kBlock), k = B * Hkv * ceil_div(Tk, kBlock);
  return q * kFaThreads <= (int64_t)UINT32_MAX && k * kFaThreads <= (int64_t)UINT32_MAX &&
         B * H * Tq <= (int64_t)UINT32_MAX / 32;
}

// Whether the offsets of the fp16 passes' tiles fit in 31 bits of bytes, and no two
// of their rows overlap: rows of K and V, and of Q and dO within a tile (one head a
// key/value head) or within the heads that share a key.
bool ca_rows_ok(const FaIn& x, int64_t d, int64_t heads, int64_t rows) {
  const int64_t most = int64_t(1) << 28;
  if (x.st < d || x.st > most / kTile || x.sh < 0) return false;
  return heads == 1 || rows == 0 || (x.sh <= most / heads && x.st <= most / rows && heads * x.sh + rows * x.st <= most);
}

bool ca_vec_ok(int64_t d, std::initializer_list<const void*> ptrs, const int64_t* strides, int n) {
  if (d % 4 != 0) return false;
  for (const void* p : ptrs)
    if (!aligned16(p)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % 4 != 0) return false;
  return true;
}

FaIn ca_in(const float* p, const int64_t* s) { return FaIn{p, s[0], s[1], s[2]}; }
FaOut ca_out(float* p, const int64_t* s) { return FaOut{p, s[0], s[1], s[2]}; }

template <int DP, bool VEC, bool FWD>
void launch_few(const CaArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.BH * a.splits)), block(256);
  if constexpr (FWD) {
    if (a.R == 1) cross_rows_kernel<1, DP / 4, VEC><<<grid, block, 0, st>>>(a);
    else if (a.R == 2) cross_rows_kernel<2, DP / 4, VEC><<<grid, block, 0, st>>>(a);
    else cross_rows_kernel<4, DP / 4, VEC><<<grid, block, 0, st>>>(a);
  } else {
    if (a.R == 1) cross_bwd_rows_kernel<1, DP / 4, VEC><<<grid, block, 0, st>>>(a);
    else if (a.R == 2) cross_bwd_rows_kernel<2, DP / 4, VEC><<<grid, block, 0, st>>>(a);
    else if (a.R <= 4) cross_bwd_rows_kernel<4, DP / 4, VEC><<<grid, block, 0, st>>>(a);
    else cross_bwd_rows_kernel<8, DP / 4, VEC><<<grid, block, 0, st>>>(a);
  }
}

template <int DP, bool VEC>
int launch_fwd(const CaArgs& a, hipStream_t st) {
  constexpr int TP = kTileDim<DP, VEC>;
  const bool few = a.R <= kFewRows;
  if (few) {
    launch_few<DP, VEC, true>(a, st);
  } else {
    const dim3 grid((unsigned)(ceil_div(a.R, kBlock) * a.BH * a.splits));
    if constexpr (VEC) cross_fwd_split_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
    else cross_fwd_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
  }
  const int rc = launch_status();
  if (rc != AAR_OK || a.splits == 1) return rc;
  const int64_t rows = (int64_t)a.BH * a.R;
  auto blocks = [&](int dim) { return dim3((unsigned)ceil_div(rows * (dim / 4), (int64_t)256)); };
  if (few) cross_combine_kernel<DP, VEC><<<blocks(DP), dim3(256), 0, st>>>(a);
  else cross_combine_kernel<TP, VEC><<<blocks(TP), dim3(256), 0, st>>>(a);
  return launch_status();
}

template <int DP, bool VEC>
int launch_bwd(const CaArgs& a, hipStream_t st) {
  constexpr int TP = kTileDim<DP, VEC>;
  const bool few = few_rows(a);
  int rc = AAR_OK;
  if (few) {
    launch_few<DP, VEC, false>(a, st);
    rc = launch_status();
  } else {
    if (a.R > 0) {
      const dim3 grid((unsigned)(ceil_div(a.R, kBlock) * a.BH * a.splits));
      if constexpr (VEC) cross_bwd_dq_split_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
      else cross_bwd_dq_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
      rc = launch_status();
    }
    if (rc != AAR_OK || a.Tk == 0) return rc;
    const dim3 grid((unsigned)(ceil_div(a.Tk, kBlock) * a.BH * a.kv_splits));
    if constexpr (VEC) cross_bwd_dkdv_split_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
    else cross_bwd_dkdv_kernel<TP><<<grid, dim3(kFaThreads), 0, st>>>(a);
    rc = launch_status();
  }
  const int64_t rows = (a.splits > 1 ? (int64_t)a.BH * a.R : 0) + (a.kv_splits > 1 ? 2 * (int64_t)a.BH * a.Tk : 0);
  if (rc != AAR_OK || rows == 0) return rc;
  auto blocks = [&](int dim) { return dim3((unsigned)ceil_div(rows * (dim / 4), (int64_t)256)); };
  if (few) cross_bwd_sum_kernel<DP, VEC><<<blocks(DP), dim3(256), 0, st>>>(a);
  else cross_bwd_sum_kernel<TP, VEC><<<blocks(TP), dim3(256), 0, st>>>(a);
  return launch_status();
}

template <bool FWD>
int ca_dispatch(const CaArgs& a, bool vec, hipStream_t st) {
  const int dp = pad_dim(a.d);
  if constexpr (FWD) {
    if (dp == 32) return vec ? launch_fwd<32, true>(a, st) : launch_fwd<32, false>(a, st);
    if (dp == 64) return vec ? launch_fwd<64, true>(a, st) : launch_fwd<64, false>(a, st);
    return vec ? launch_fwd<128, true>(a, st) : launch_fwd<128, false>(a, st);
  } else {
    if (dp == 32) return vec ? launch_bwd<32, true>(a, st) : launch_bwd<32, false>(a, st);
    if (dp == 64) return vec ? launch_bwd<64, true>(a, st) : launch_bwd<64, false>(a, st);
    return vec ? launch_bwd<128, true>(a, st) : launch_bwd<128, false>(a, st);
  }
}

int ca_check(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d) {
  if (B < 0 || H < 0 || Hkv < 0 || Tq < 0 || Tk < 0 || d <= 0 || d > 128) return AAR_EINVAL;
  if ((H == 0) != (Hkv == 0) || (H > 0 && H % Hkv != 0)) return AAR_EINVAL;
  if (H > 0 && !ca_shape_ok(B, H, Hkv, Tq, Tk)) return AAR_EUNSUPPORTED;
  return AAR_OK;
}

// Floats of a part's row, at most.
int part_dim(int64_t d) { return std::max(pad_dim(d), 64); }

size_t part_o_bytes(int64_t bh, int64_t R, int64_t d, int splits) {
  return (size_t)bh * splits * (size_t)R * part_dim(d) * sizeof(float);
}

// Where the backward's workspace holds item i (D, dQ's parts, dK's, dV's); 4: its end.
size_t bwd_bytes(const CaArgs& a, int i) {
  const size_t dp = part_dim(a.d), bh = a.BH;
  const size_t size[4] = {(bh * a.R * sizeof(float) + 15) / 16 * 16,
                          a.splits > 1 ? a.splits * bh * a.R * dp * sizeof(float) : 0,
                          a.kv_splits > 1 ? a.kv_splits * bh * a.Tk * dp * sizeof(float) : 0,
                          a.kv_splits > 1 ? a.kv_splits * bh * a.Tk * dp * sizeof(float) : 0};
  size_t at = 0;
  for (int k = 0; k < i; ++k) at += size[k];
  return at;
}

CaArgs ca_args(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d, const int64_t* lens, float* lse,
               float scale) {
  CaArgs a{};
  a.lens = lens;
  a.lse = lse;
  a.Tq = (int)Tq;
  a.Tk = (int)Tk;
  a.d = (int)d;
  a.G = (int)(H / Hkv);
  a.Hkv = (int)Hkv;
  a.R = (int)(H / Hkv * Tq);
  a.BH = (int)(B * Hkv);
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  return a;
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

size_t aar_cross_attn_fwd_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d) {
  if (ca_check(B, H, Hkv, Tq, Tk, d) != AAR_OK || B == 0 || H == 0 || Tq == 0 || Tk == 0) return 0;
  int splits, chunk;
  ca_plan(B * Hkv, H / Hkv * Tq, Tk, d, &splits, &chunk);
  if (splits == 1) return 0;
  return part_o_bytes(B * Hkv, H / Hkv * Tq, d, splits) + (size_t)B * H * Tq * splits * sizeof(float);
}

int aar_cross_attn_fwd_f32(const float* q, const float* k, const float* v, const int64_t* kv_lens, float* o, float* lse,
                           int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d,
                           const int64_t* strides, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = ca_check(B, H, Hkv, Tq, Tk, d);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0 || Tq == 0) return AAR_OK;
  if (!q || !o || !lse || !strides || (Tk > 0 && (!k || !v))) return AAR_EINVAL;
  CaArgs a = ca_args(B, H, Hkv, Tq, Tk, d, kv_lens, lse, scale);
  a.q = ca_in(q, strides);
  a.k = ca_in(k, strides + 3);
  a.v = ca_in(v, strides + 6);
  a.o = ca_out(o, strides + 9);
  ca_plan(a.BH, a.R, Tk, d, &a.splits, &a.chunk);
  if (a.splits > 1) {
    const size_t need = aar_cross_attn_fwd_workspace_bytes(B, H, Hkv, Tq, Tk, d);
    if (!workspace || !aligned16(workspace) || workspace_bytes < need) return AAR_EWORKSPACE;
    a.part_o = static_cast<float*>(workspace);
    a.part_l = reinterpret_cast<float*>(static_cast<char*>(workspace) + part_o_bytes(a.BH, a.R, d, a.splits));
  }
  const bool near = a.R <= kFewRows || (ca_rows_ok(a.k, d, 1, Tk) && ca_rows_ok(a.v, d, 1, Tk));
  return ca_dispatch<true>(a, near && ca_vec_ok(d, {q, k, v, o}, strides, 12), as_stream(stream));
}

// D of every query row, then the parts of dQ, dK and dV
size_t aar_cross_attn_bwd_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d) {
  if (ca_check(B, H, Hkv, Tq, Tk, d) != AAR_OK || B == 0 || H == 0 || Tq == 0) return 0;
  CaArgs a = ca_args(B, H, Hkv, Tq, Tk, d, nullptr, nullptr, 1.0f);
  ca_bwd_plan(a);
  return bwd_bytes(a, 4);
}

int aar_cross_attn_bwd_f32(const float* q, const float* k, const float* v, const int64_t* kv_lens, const float* o,
                           const float* lse, const float* dout, float* dq, float* dk, float* dv, int64_t B, int64_t H,
                           int64_t Hkv, int64_t Tq, int64_t Tk, int64_t d, const int64_t* strides, float scale,
                           void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = ca_check(B, H, Hkv, Tq, Tk, d);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0) return AAR_OK;
  if (!strides) return AAR_EINVAL;
  if (Tq > 0 && (!q || !o || !lse || !dout || !dq)) return AAR_EINVAL;
  if (Tk > 0 && (!k || !v || !dk || !dv)) return AAR_EINVAL;
  if (Tq == 0 && Tk == 0) return AAR_OK;
  CaArgs a = ca_args(B, H, Hkv, Tq, Tk, d, kv_lens, const_cast<float*>(lse), scale);
  ca_bwd_plan(a);
  if (Tq > 0) {
    if (!workspace || !aligned16(workspace) || workspace_bytes < bwd_bytes(a, 4)) return AAR_EWORKSPACE;
    char* ws = static_cast<char*>(workspace);
    a.D = reinterpret_cast<float*>(ws);
    a.dq_part = reinterpret_cast<float*>(ws + bwd_bytes(a, 1));
    a.dk_part = reinterpret_cast<float*>(ws + bwd_bytes(a, 2));
    a.dv_part = reinterpret_cast<float*>(ws + bwd_bytes(a, 3));
  }
  a.q = ca_in(q, strides);
  a.k = ca_in(k, strides + 3);
  a.v = ca_in(v, strides + 6);
  a.o_in = ca_in(o, strides + 9);
  a.dout = ca_in(dout, strides + 12);
  a.dq = ca_out(dq, strides + 15);
  a.dk = ca_out(dk, strides + 18);
  a.dv = ca_out(dv, strides + 21);
  const bool near = few_rows(a) || (ca_rows_ok(a.k, d, 1, Tk) && ca_rows_ok(a.v, d, 1, Tk) &&
                                    ca_rows_ok(a.q, d, a.G, Tq) && ca_rows_ok(a.dout, d, a.G, Tq));
  return ca_dispatch<false>(a, near && ca_vec_ok(d, {q, k, v, o, dout, dq, dk, dv}, strides, 24), as_stream(stream));
}

}  // extern "C"
