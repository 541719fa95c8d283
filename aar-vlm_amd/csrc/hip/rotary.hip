// Norms of queries and keys for each head with the rotary position embedding
// in the same pass, forward and backward.
//
// Per head x[0, d): rstd = rsqrt(mean x^2 + eps), xh = x rstd, u = xh w, and the
// pairs (c, c + r/2) of u turned by a = position base^(-2c/r).  Backward, with g
// the gradient turned back by -a:
//   dw = sum over rows and heads of g xh,   dx = rstd (w g - xh mean(w g xh)).
//
// Bound by HBM: the forward reads and writes each head once, the backward reads
// x and dy and writes dx (rstd is recomputed from x, which it needs anyway).
// A head takes d/8 lanes with 4 + 4 elements each, the halves of its pairs, so
// norm and rotation stay inside a lane but for one sum over the head's lanes; a
// wave walks a row's heads and forms the row's angles once, beside the first
// heads' loads.  The angle in turns is position * base^(-2c/r) / (2 pi) in fp64
// (frequencies from the host, in the kernel's arguments), whose fraction alone, in
// [-1/2, 1/2], goes to fp32: an angle is off by up to 2 pi 2^-26 = 1e-7, at a position of
// 10^6 as at the first, which is of the order of the turned values' own roundings.  dw
// accumulates in registers over a persistent grid, one partial row per workgroup, joined
// in a fixed order: no atomics.  32768 rows of 40 heads, d 128: forward 257 us, 5.2 TB/s, backward 378 us,
// 5.3 TB/s; 16384 rows of 12 heads, d 64: 17.8 us (100 MB, from the caches in part)
// and 28.9 us, and 4.2 us to join dw.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "common.hpp"

namespace aar {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 256;

struct RopeFreq {
  double turn[kMaxDim / 2];  // base^(-2c/r) / (2 pi)
};

struct RopeArgs {
  const float *gy, *x, *wq, *wk;
  const int64_t* pos;
  float* y;     // forward's y, backward's dx
  float* part;  // backward: [workgroups][2 d] partial dwq, dwk
  int64_t gy_row, x_row, y_row, n_pos, rows;
  int hq, heads, d, r, split;  // split: waves that share a row's heads
  float eps;
};

__device__ __forceinline__ void turn_sincos(double t, float& sn, float& cs) {
  t -= rint(t);
  sincospif(2.0f * (float)t, &sn, &cs);
}

// Sum over the LPH consecutive lanes of a head.
template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
  if (LPH >= 2) v += dpp_quad_xor1(v);
  if (LPH >= 4) v += dpp_quad_xor2(v);
  if (LPH >= 8) v += dpp_half_mirror(v);
  if (LPH >= 16) v += dpp_row_mirror(v);
  if (LPH >= 32) v += swizzle_xor16(v);
  return v;
}

// d = r = 8 * (lanes in use of LPH): a head in LPH lanes, 64 / LPH heads a wave
// step.  BWD also accumulates dwq and dwk.
template <int LPH, bool BWD>
__global__ void __launch_bounds__(kThreads)
rope_vec_kernel(const RopeArgs a, const RopeFreq fr) {
  constexpr int kHeads = kWave / LPH;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = a.d / 2;
  const int c = 4 * (lane % LPH);
  const bool on = c < half;
  const float inv_d = 1.0f / (float)a.d;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 wq1 = zero, wq2 = zero, wk1 = zero, wk2 = zero;
  double turn[4] = {0., 0., 0., 0.};
  if (on) {
    if (a.hq > 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wq1[e] = a.wq[c + e];
        wq2[e] = a.wq[c + half + e];
      }
    }
    if (a.heads > a.hq) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        wk1[e] = a.wk[c + e];
        wk2[e] = a.wk[c + half + e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) turn[e] = fr.turn[c + e];
  }
  f32x4 dq1 = zero, dq2 = zero, dk1 = zero, dk2 = zero;
  // One head of each lane's group: its output and, in the backward, its share of dw.
  auto head = [&](int64_t row, int h, bool act, const f32x4& x1, const f32x4& x2, const f32x4& g1, const f32x4& g2,
                  const f32x4& sn, const f32x4& cs) {
    const bool is_q = h < a.hq;
    const f32x4 w1 = is_q ? wq1 : wk1, w2 = is_q ? wq2 : wk2;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += x1[e] * x1[e] + x2[e] * x2[e];
    const float rstd = 1.0f / sqrtf(head_sum<LPH>(ss) * inv_d + a.eps);
    f32x4 o1, o2;
    if (!BWD) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u1 = x1[e] * rstd * w1[e], u2 = x2[e] * rstd * w2[e];
        o1[e] = u1 * cs[e] - u2 * sn[e];
        o2[e] = u2 * cs[e] + u1 * sn[e];
      }
    } else {
      f32x4 h1, h2, r1, r2;
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        r1[e] = g1[e] * cs[e] + g2[e] * sn[e];
        r2[e] = g2[e] * cs[e] - g1[e] * sn[e];
        h1[e] = x1[e] * rstd;
        h2[e] = x2[e] * rstd;
        dot += r1[e] * w1[e] * h1[e] + r2[e] * w2[e] * h2[e];
      }
      const float mean = head_sum<LPH>(dot) * inv_d;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o1[e] = rstd * (r1[e] * w1[e] - h1[e] * mean);
        o2[e] = rstd * (r2[e] * w2[e] - h2[e] * mean);
      }
      if (act) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p1 = r1[e] * h1[e], p2 = r2[e] * h2[e];
          dq1[e] += is_q ? p1 : 0.f;
          dq2[e] += is_q ? p2 : 0.f;
          dk1[e] += is_q ? 0.f : p1;
          dk2[e] += is_q ? 0.f : p2;
        }
      }
    }
    if (act) {
      float* yp = a.y + row * a.y_row + (int64_t)h * a.d + c;
      __builtin_nontemporal_store(o1, reinterpret_cast<f32x4*>(yp));
      __builtin_nontemporal_store(o2, reinterpret_cast<f32x4*>(yp + half));
    }
  };
  const int64_t units = a.rows * a.split;
  const int64_t step = (int64_t)gridDim.x * (kThreads / kWave);
  for (int64_t u = (int64_t)blockIdx.x * (kThreads / kWave) + wave; u < units; u += step) {
    const int64_t row = u / a.split;
    const int part = (int)(u - row * a.split);
    // the first heads' loads run beside the angles
    f32x4 x1, x2, g1, g2;
    int h;
    auto load = [&](int h0) {
      h = h0 + lane / LPH;
      x1 = x2 = g1 = g2 = zero;
      if (on && h < a.heads) {
        const float* xp = a.x + row * a.x_row + (int64_t)h * a.d + c;
        x1 = *reinterpret_cast<const f32x4*>(xp);
        x2 = *reinterpret_cast<const f32x4*>(xp + half);
        if (BWD) {
          const float* gp = a.gy + row * a.gy_row + (int64_t)h * a.d + c;
          g1 = *reinterpret_cast<const f32x4*>(gp);
          g2 = *reinterpret_cast<const f32x4*>(gp + half);
        }
      }
    };
    int h0 = part * kHeads;
    load(h0);
    const double p = (double)a.pos[row % a.n_pos];
    f32x4 sn, cs;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float s1, c1;
      turn_sincos(p * turn[e], s1, c1);
      sn[e] = s1;
      cs[e] = c1;
    }
    for (;;) {
      head(row, h, on && h < a.heads, x1, x2, g1, g2, sn, cs);
      h0 += a.split * kHeads;
      if (h0 >= a.heads) break;
      load(h0);
    }
  }
  if (!BWD) return;
  // The wave's heads, then the workgroup's waves, in a fixed order.
  __shared__ float red[kThreads / kWave][4][4 * LPH];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float v[4] = {dq1[e], dq2[e], dk1[e], dk2[e]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = LPH; o < kWave; o *= 2) v[i] += __shfl_xor(v[i], o, kWave);
      if (lane < LPH) red[wave][i][c + e] = v[i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
    // column i of dwq | dwk
    const int which = i / a.d, col = i - which * a.d;
    const int slot = 2 * which + (col >= half ? 1 : 0), cc = col >= half ? col - half : col;
    float s = red[0][slot][cc];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) s += red[w][slot][cc];
    a.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
  }
}

// Any even rotary width, any d up to 64 kN, any alignment: lane l of a wave has a head's
// elements l, l + 64, ...; the partner of a pair is read again.  As above a wave walks
// a row's heads and forms the row's angles once, beside the first head's loads.
// 16384 rows of 12 heads, d 30, forward + backward 100 us (32, 64 and 4 to join dw; 94 MB),
// with the angles formed for every head and four slots a lane whatever d 200.
template <int kN, bool BWD>
__global__ void __launch_bounds__(kThreads)
rope_any_kernel(const RopeArgs a, const RopeFreq fr) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int half = a.r / 2;
  const float inv_d = 1.0f / (float)a.d;
  float dq[kN] = {}, dk[kN] = {};
  int other[kN];  // the pair's other element, the own one past the rotation
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int e = lane + i * kWave;
    other[i] = e >= a.r ? e : (e < half ? e + half : e - half);
  }
  const int64_t units = a.rows * a.split;
  const int64_t step = (int64_t)gridDim.x * (kThreads / kWave);
  for (int64_t u = (int64_t)blockIdx.x * (kThreads / kWave) + wave; u < units; u += step) {
    const int64_t row = u / a.split;
    int h = (int)(u - row * a.split);
    float x[kN], xo[kN], g[kN], go[kN], ww[kN], wo[kN];  // own element and the pair's other one
    auto load = [&]() {
      const float* w = h < a.hq ? a.wq : a.wk;
      const float* xp = a.x + row * a.x_row + (int64_t)h * a.d;
      const float* gp = BWD ? a.gy + row * a.gy_row + (int64_t)h * a.d : nullptr;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = lane + i * kWave;
        x[i] = xo[i] = g[i] = go[i] = ww[i] = wo[i] = 0.f;
        if (e >= a.d) continue;
        x[i] = xp[e];
        ww[i] = w[e];
        if (BWD) {
          g[i] = gp[e];
          go[i] = gp[other[i]];
        } else {
          xo[i] = xp[other[i]];
          wo[i] = w[other[i]];
        }
      }
    };
    load();
    const double p = a.r > 0 ? (double)a.pos[row % a.n_pos] : 0.0;
    float sn[kN], cs[kN];
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int e = lane + i * kWave;
      sn[i] = 0.f;
      cs[i] = 1.f;
      if (e >= a.r) continue;
      float s1, c1;
      turn_sincos(p * fr.turn[e < half ? e : other[i]], s1, c1);
      // own' = own cos + other * sn in the forward
      sn[i] = e < half ? -s1 : s1;
      cs[i] = c1;
    }
    for (;;) {
      const bool is_q = h < a.hq;
      float* yp = a.y + row * a.y_row + (int64_t)h * a.d;
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < kN; ++i) ss += x[i] * x[i];
      const float rstd = 1.0f / sqrtf(wave_sum(ss) * inv_d + a.eps);
      float dot = 0.f;
      if (BWD) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          if (lane + i * kWave < a.r) g[i] = g[i] * cs[i] - go[i] * sn[i];
          dot += g[i] * ww[i] * (x[i] * rstd);
        }
        dot = wave_sum(dot) * inv_d;
      }
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int e = lane + i * kWave;
        if (e >= a.d) continue;
        const float xh = x[i] * rstd;
        if (BWD) {
          yp[e] = rstd * (g[i] * ww[i] - xh * dot);
          if (is_q) dq[i] += g[i] * xh;
          else dk[i] += g[i] * xh;
        } else {
          yp[e] = e < a.r ? xh * ww[i] * cs[i] + xo[i] * rstd * wo[i] * sn[i] : xh * ww[i];
        }
      }
      h += a.split;
      if (h >= a.heads) break;
      load();
    }
  }
  if (!BWD) return;
  __shared__ float red[kThreads / kWave][2][kMaxDim];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    red[wave][0][lane + i * kWave] = dq[i];
    red[wave][1][lane + i * kWave] = dk[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.d; i += kThreads) {
    const int which = i / a.d, col = i - which * a.d;
    float s = red[0][which][col];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) s += red[w][which][col];
    a.part[(int64_t)blockIdx.x * 2 * a.d + i] = s;
  }
}

// dwq | dwk: column sums of the partial rows.  A workgroup takes 8 columns, 128
// slices of the rows each in order, then a fixed tree over the slices.
constexpr int kFinCols = 8, kFinSlices = 128;

__global__ void __launch_bounds__(kFinCols* kFinSlices)
rope_finish_kernel(const float* __restrict__ part, int parts, int d, float* __restrict__ dwq, float* __restrict__ dwk) {
  __shared__ float acc[kFinSlices][kFinCols];
  const int cl = threadIdx.x % kFinCols, sl = threadIdx.x / kFinCols;
  const int col = blockIdx.x * kFinCols + cl;
  const int per = (parts + kFinSlices - 1) / kFinSlices;
  float s = 0.f;
  if (col < 2 * d)
    for (int p = sl * per; p < min(parts, (sl + 1) * per); ++p) s += part[(int64_t)p * 2 * d + col];
  acc[sl][cl] = s;
  __syncthreads();
  for (int h = kFinSlices / 2; h >= 1; h /= 2) {
    if (sl < h) acc[sl][cl] += acc[sl + h][cl];
    __syncthreads();
  }
  if (sl == 0 && col < 2 * d) (col < d ? dwq[col] : dwk[col - d]) = acc[0][cl];
}

// The vector kernel takes whole-width rotations of heads in 4 + 4 element
// lanes, with 16-byte rows.
int lanes_per_head(const RopeArgs& a) {
  if (a.r != a.d || a.d % 8 != 0 || a.x_row % 4 != 0 || a.y_row % 4 != 0 || a.gy_row % 4 != 0) return 0;
  if (!aligned16(a.x) || !aligned16(a.y) || !aligned16(a.gy)) return 0;
  int l = 4;
  while (l < a.d / 8) l *= 2;
  return l;
}

// Workgroups of the backward, and its dw partial rows.  Persistent, two to a CU:
// forward + backward of 32768 x 40 heads, d 128, in 636 us (one to a CU 654, four 648,
// eight 650), of 4096 x 12, d 64, in 19.1 (21.5, 19.9, 25.0).
int64_t bwd_groups(int64_t rows, int64_t heads) {
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows * heads, 4), 2 * (int64_t)device_cu_count()));
}

template <bool BWD>
int launch(RopeArgs a, const RopeFreq& fr, int64_t groups, hipStream_t st) {
  const int lph = lanes_per_head(a);
  // A row's heads are spread over waves where there are too few rows to fill
  // the GPU with one wave each (16 a CU: 512 rows of 40 heads, d 128, forward 8.4 us,
  // with 4 a CU 8.7, with 32 8.4 but 4096 x 12 heads forward + backward 22 against 20).
  const int steps = (int)ceil_div(a.heads, lph == 0 ? 1 : kWave / lph);
  const int64_t want = ceil_div(16 * (int64_t)device_cu_count(), a.rows);
  a.split = (int)std::max<int64_t>(1, std::min<int64_t>(steps, want));
  const int64_t g = BWD ? groups : std::min<int64_t>(ceil_div(a.rows * a.split, 4), 1 << 20);
  if (lph == 0) {
    auto kernel = a.d <= 64 ? rope_any_kernel<1, BWD> : a.d <= 128 ? rope_any_kernel<2, BWD> : rope_any_kernel<4, BWD>;
    kernel<<<dim3((unsigned)g), dim3(kThreads), 0, st>>>(a, fr);
    return launch_status();
  }
  auto kernel = lph == 4 ? rope_vec_kernel<4, BWD>
                : lph == 8 ? rope_vec_kernel<8, BWD>
                : lph == 16 ? rope_vec_kernel<16, BWD> : rope_vec_kernel<32, BWD>;
  kernel<<<dim3((unsigned)g), dim3(kThreads), 0, st>>>(a, fr);
  return launch_status();
}

int rope_check(int64_t rows, int64_t q_heads, int64_t k_heads, int64_t d, int64_t r, const int64_t* positions,
               int64_t n_positions, double base, float eps) {
  if (rows < 0 || q_heads < 0 || k_heads < 0 || d < 2 || r < 0 || r > d || r % 2 != 0) return AAR_EINVAL;
  if (!(base > 0.0) || !(base < INFINITY) || !(eps >= 0.f) || !(eps < INFINITY)) return AAR_EINVAL;
  if (d > kMaxDim || q_heads + k_heads > (1 << 20) || rows > (int64_t(1) << 40)) return AAR_EUNSUPPORTED;
  if (r > 0 && rows > 0 && (n_positions <= 0 || rows % n_positions != 0 || !positions)) return AAR_EINVAL;
  return AAR_OK;
}

// base^(-2c/r) / (2 pi): every eighth by pow, those between by a product (a
// call's 64 pow would cost more than its launch).
void rope_freq(RopeFreq& fr, int64_t r, double base) {
  const double ratio = r > 0 ? pow(base, -2.0 / (double)r) : 1.0;
  for (int64_t c = 0; c < r / 2; ++c)
    fr.turn[c] = c % 8 == 0 ? pow(base, -2.0 * (double)c / (double)r) / (2.0 * M_PI) : fr.turn[c - 1] * ratio;
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

int aar_qk_norm_rope_fwd_f32(const float* x, int64_t x_row, const float* wq, const float* wk, const int64_t* positions,
                             int64_t n_positions, float* y, int64_t y_row, int64_t rows, int64_t q_heads,
                             int64_t k_heads, int64_t d, int64_t rotary_dim, double base, float eps, void* stream) {
  const int rc = rope_check(rows, q_heads, k_heads, d, rotary_dim, positions, n_positions, base, eps);
  if (rc != AAR_OK) return rc;
  const int64_t heads = q_heads + k_heads;
  if (rows == 0 || heads == 0) return AAR_OK;
  if (!x || !y || (q_heads > 0 && !wq) || (k_heads > 0 && !wk)) return AAR_EINVAL;
  if (rows > 1 && (x_row < heads * d || y_row < heads * d)) return AAR_EINVAL;
  if (x == y && x_row != y_row && rows > 1) return AAR_EINVAL;
  RopeFreq fr;
  rope_freq(fr, rotary_dim, base);
  RopeArgs a{nullptr, x, wq, wk, positions, y, nullptr, 0, x_row, y_row, std::max<int64_t>(n_positions, 1), rows,
             (int)q_heads, (int)heads, (int)d, (int)rotary_dim, 1, eps};
  return launch<false>(a, fr, 0, as_stream(stream));
}

size_t aar_qk_norm_rope_bwd_workspace_bytes(int64_t rows, int64_t q_heads, int64_t k_heads, int64_t d) {
  if (rows <= 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads <= 0 || d < 2 || d > kMaxDim) return 0;
  return (size_t)bwd_groups(rows, q_heads + k_heads) * 2 * (size_t)d * sizeof(float);
}

int aar_qk_norm_rope_bwd_f32(const float* gy, int64_t gy_row, const float* x, int64_t x_row, const float* wq,
                             const float* wk, const int64_t* positions, int64_t n_positions, float* dx, int64_t dx_row,
                             float* dwq, float* dwk, int64_t rows, int64_t q_heads, int64_t k_heads, int64_t d,
                             int64_t rotary_dim, double base, float eps, void* workspace, size_t workspace_bytes,
                             void* stream) {
  int rc = rope_check(rows, q_heads, k_heads, d, rotary_dim, positions, n_positions, base, eps);
  if (rc != AAR_OK) return rc;
  const int64_t heads = q_heads + k_heads;
  if (!dwq || !dwk) return AAR_EINVAL;
  hipStream_t st = as_stream(stream);
  if (rows == 0 || heads == 0) {
    rc = aar_memset_zero(dwq, (size_t)d * sizeof(float), stream);
    return rc != AAR_OK ? rc : aar_memset_zero(dwk, (size_t)d * sizeof(float), stream);
  }
  if (!x || !gy || !dx || (q_heads > 0 && !wq) || (k_heads > 0 && !wk)) return AAR_EINVAL;
  if (rows > 1 && (x_row < heads * d || gy_row < heads * d || dx_row < heads * d)) return AAR_EINVAL;
  if (dx == gy && dx_row != gy_row && rows > 1) return AAR_EINVAL;
  if (!workspace || workspace_bytes < aar_qk_norm_rope_bwd_workspace_bytes(rows, q_heads, k_heads, d))
    return AAR_EWORKSPACE;
  RopeFreq fr;
  rope_freq(fr, rotary_dim, base);
  const int64_t groups = bwd_groups(rows, heads);
  float* part = static_cast<float*>(workspace);
  RopeArgs a{gy, x, wq, wk, positions, dx, part, gy_row, x_row, dx_row, std::max<int64_t>(n_positions, 1), rows,
             (int)q_heads, (int)heads, (int)d, (int)rotary_dim, 1, eps};
  rc = launch<true>(a, fr, groups, st);
  if (rc != AAR_OK) return rc;
  rope_finish_kernel<<<dim3((unsigned)ceil_div(2 * d, kFinCols)), dim3(kFinCols * kFinSlices), 0, st>>>(
      part, (int)groups, (int)d, dwq, dwk);
  return launch_status();
}

}  // extern "C"
