// Distillation from a teacher's top logits, forward and backward.
//
// With tau the temperature, p = softmax(t / tau) over a row's teacher entries
// and q = softmax(z / tau) over the vocabulary:
//   row loss = tau^2 sum_k p_k (ln p_k - ln q[id_k]),
//   dz       = grad tau / counted (q - sum_{k: id_k = v} p_k).
//
// Bound by HBM: z is read once for the row's maximum and sum (online, one
// rescale per 16 elements of a lane) and once more with dz written.  A row takes
// W waves: one up to 2048 columns, then a workgroup of 4, or of 16 where the rows
// are too few to fill the GPU.  Rows of any alignment take 128-bit accesses: up
// to three leading elements bring a row's pointer onto 16 bytes.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "common.hpp"

namespace aar {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxTop = 1024;

// 2^x on the transcendental unit; results below 2^-126 are flushed to zero.
__device__ __forceinline__ float fast_exp2(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_exp2f(x);
#else
  return x;
#endif
}

// A running maximum and sum of 2^(k (x - max)).
struct MaxSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void merge(float m2, float s2, float k) {
    const float mn = fmaxf(m, m2);
    const float mu = mn == -INFINITY ? 0.f : mn;
    // (a NaN sum stays: its maximum, which fmaxf skips, does not matter)
    s = s * fast_exp2((m - mu) * k) + s2 * fast_exp2((m2 - mu) * k);
    m = mn;
  }
  template <int N>
  __device__ __forceinline__ void take(const float (&x)[N], float k) {
    float mn = m;
#pragma unroll
    for (int i = 0; i < N; ++i) mn = fmaxf(mn, x[i]);
    const float mu = mn == -INFINITY ? 0.f : mn;
    s *= fast_exp2((m - mu) * k);
#pragma unroll
    for (int i = 0; i < N; ++i) s += fast_exp2((x[i] - mu) * k);
    m = mn;
  }
};

// Elements before a row's first 16-byte boundary.
__device__ __forceinline__ int row_lead(const float* p, int V) {
  return min(V, (int)((16u - ((unsigned)(uintptr_t)p & 15u)) & 15u) / 4);
}

// The teacher's entries of a row as a wave sees them: how many there are, and
// whether one is out of range.
__device__ __forceinline__ void scan_ids(const int64_t* ids, int top, int64_t V, int lane, bool& any, bool& bad) {
  bool a = false, b = false;
  for (int k = lane; k < top; k += kWave) {
    const int64_t id = ids[k];
    a = a || id >= 0;
    b = b || id < -1 || id >= V;
  }
  any = __any(a) != 0;
  bad = __any(b) != 0;
}

// Largest entry and sum of a row's teacher distribution (a wave; every lane
// returns both).  sum = 0 where every entry is -inf.
__device__ __forceinline__ void teacher_sum(const float* t, const int64_t* ids, int top, float k, int lane, float& tm,
                                            float& ts) {
  tm = -INFINITY;
  for (int i = lane; i < top; i += kWave)
    if (ids[i] >= 0) tm = fmaxf(tm, t[i]);
  tm = wave_max(tm);
  const float mu = tm == -INFINITY ? 0.f : tm;
  ts = 0.f;
  for (int i = lane; i < top; i += kWave)
    if (ids[i] >= 0) ts += fast_exp2((t[i] - mu) * k);
  ts = wave_sum(ts);
  tm = mu;
}

// A row that is left out (no loss is -inf).
__device__ __forceinline__ void leave_out(float* row_loss, float* stats, int64_t row) {
  row_loss[row] = -INFINITY;
  stats[2 * row] = 0.f;
  stats[2 * row + 1] = INFINITY;
}

// One row per W waves; row_loss and stats.
template <int W>
__global__ void __launch_bounds__(W > 4 ? W * kWave : 256)
distill_row_kernel(const float* __restrict__ Z, const float* __restrict__ Tl, const int64_t* __restrict__ Ti,
                   float* __restrict__ row_loss, float* __restrict__ stats, int64_t n, int V, int top, float k,
                   float inv_tau, float tau2, int* __restrict__ err) {
  constexpr int kWaves = (W > 4 ? W : 4);
  constexpr int kRows = kWaves / W;
  __shared__ float pm[kWaves], ps[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = wave % W, rt = wr * kWave + lane;
  const int64_t row = (int64_t)blockIdx.x * kRows + wave / W;
  bool any = false, bad = false;
  if (row < n) scan_ids(Ti + row * top, top, V, lane, any, bad);
  const bool on = any && !bad;
  MaxSum a;
  const float* z = Z + row * V;
  if (on) {
    const int lead = row_lead(z, V), body = (V - lead) / 4, tail = V - lead - 4 * body;
    if (rt < lead) a.take<1>({z[rt]}, k);
    if (rt < tail) a.take<1>({z[V - tail + rt]}, k);
    const f32x4* zv = reinterpret_cast<const f32x4*>(z + lead);
    int i = rt;
    for (; i + 3 * W * kWave < body; i += 4 * W * kWave) {
      f32x4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = zv[i + u * W * kWave];
      float x[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) x[u] = v[u / 4][u % 4];
      a.take<16>(x, k);
    }
    for (; i < body; i += W * kWave) {
      const f32x4 v = zv[i];
      a.take<4>({v[0], v[1], v[2], v[3]}, k);
    }
  }
  // The lanes' and waves' pairs in a fixed tree.
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) a.merge(__shfl_xor(a.m, o, kWave), __shfl_xor(a.s, o, kWave), k);
  if (W > 1) {
    if (lane == 0) {
      pm[wave] = a.m;
      ps[wave] = a.s;
    }
    __syncthreads();
    a = MaxSum{};
#pragma unroll
    for (int w = 0; w < W; ++w) a.merge(pm[wave / W * W + w], ps[wave / W * W + w], k);
  }
  if (row >= n || wr != 0) return;
  if (!on) {
    if (lane == 0) {
      leave_out(row_loss, stats, row);
      if (bad && err) *err = 1;
    }
    return;
  }
  const float* t = Tl + row * top;
  const int64_t* ids = Ti + row * top;
  float tm, ts;
  teacher_sum(t, ids, top, k, lane, tm, ts);
  if (ts == 0.f) {  // nothing above -inf: left out like a row without entries
    if (lane == 0) leave_out(row_loss, stats, row);
    return;
  }
  const float ln_s = logf(a.s);
  // sum_k p_k (ln p_k - ln q_k) = sum_k e_k ((t_k - tm) / tau - ln q_k) / ts - ln ts
  float acc = 0.f;
  for (int i = lane; i < top; i += kWave) {
    const int64_t id = ids[i];
    if (id < 0) continue;
    const float e = fast_exp2((t[i] - tm) * k);
    const float lnq = (z[id] - a.m) * inv_tau - ln_s;
    if (!(e == 0.f)) acc += e * ((t[i] - tm) * inv_tau - lnq);
  }
  acc = wave_sum(acc);
  if (lane == 0) {
    row_loss[row] = tau2 * (acc / ts - logf(ts));
    stats[2 * row] = a.m;
    stats[2 * row + 1] = a.s;
  }
}

// The mean of the counted rows' losses and their number: one workgroup, each
// thread its rows in order (in double), then a fixed tree.
constexpr int kMeanThreads = 1024;
constexpr int kMeanChunk = 16;

__global__ void __launch_bounds__(kMeanThreads)
distill_mean_kernel(const float* __restrict__ row_loss, float* __restrict__ stats, float* __restrict__ loss, int64_t n) {
  __shared__ double ds[kMeanThreads / kWave];
  __shared__ long long cs[kMeanThreads / kWave];
  double s = 0.0;
  long long c = 0;
  for (int64_t base = 0; base < n; base += (int64_t)kMeanThreads * kMeanChunk) {
    float l[kMeanChunk];
#pragma unroll
    for (int u = 0; u < kMeanChunk; ++u) {
      const int64_t i = base + (int64_t)u * kMeanThreads + threadIdx.x;
      l[u] = i < n ? row_loss[i] : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kMeanChunk; ++u) {
      if (l[u] == -INFINITY) continue;
      s += (double)l[u];
      ++c;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o, kWave);
    c += __shfl_xor(c, o, kWave);
  }
  if ((threadIdx.x & 63) == 0) {
    ds[threadIdx.x >> 6] = s;
    cs[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kMeanThreads / kWave; ++w) {
      s += ds[w];
      c += cs[w];
    }
    loss[0] = c > 0 ? (float)(s / (double)c) : 0.f;
    stats[2 * n] = (float)c;
  }
}

// dz of one row per W waves: grad tau / counted q everywhere, then the
// teacher's entries over it (after every wave's stores of the row).
template <int W, bool VEC>
__global__ void __launch_bounds__(W > 4 ? W * kWave : 256)
distill_bwd_kernel(const float* __restrict__ grad, const float* __restrict__ Z, const float* __restrict__ Tl,
                   const int64_t* __restrict__ Ti, const float* __restrict__ stats, float* __restrict__ dZ, int64_t n,
                   int V, int top, float k, float tau) {
  constexpr int kWaves = (W > 4 ? W : 4);
  constexpr int kRows = kWaves / W;
  extern __shared__ int sh[];  // ids and p of the rows' entries
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wr = wave % W, rt = wr * kWave + lane;
  // the forward's last rows first: they may still be in the caches
  const int64_t row = n - 1 - ((int64_t)blockIdx.x * kRows + wave / W);
  int* sid = sh + (wave / W) * 2 * top;
  float* sp = reinterpret_cast<float*>(sid + top);
  const bool here = row >= 0;
  const float m = here ? stats[2 * row] : 0.f, s = here ? stats[2 * row + 1] : INFINITY;
  const bool on = s != INFINITY;
  const float* z = Z + row * V;
  float* dz = dZ + row * V;
  const float c = grad[0] * tau / stats[2 * n];
  const float f = c / s;
  if (on && wr == 0) {
    const float* t = Tl + row * top;
    const int64_t* ids = Ti + row * top;
    float tm, ts;
    teacher_sum(t, ids, top, k, lane, tm, ts);
    const float inv = 1.0f / ts;
    for (int i = lane; i < top; i += kWave) {
      const int id = (int)ids[i];
      sid[i] = id;
      sp[i] = id < 0 ? 0.f : fast_exp2((t[i] - tm) * k) * inv;
    }
  }
  if (here) {
    auto one = [&](float x) { return on ? f * fast_exp2((x - m) * k) : 0.f; };
    if (VEC) {
      const int lead = row_lead(z, V), body = (V - lead) / 4, tail = V - lead - 4 * body;
      if (rt < lead) dz[rt] = on ? one(z[rt]) : 0.f;
      if (rt < tail) dz[V - tail + rt] = on ? one(z[V - tail + rt]) : 0.f;
      const f32x4* zv = reinterpret_cast<const f32x4*>(z + lead);
      f32x4* dv = reinterpret_cast<f32x4*>(dz + lead);
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      int i = rt;
      for (; i + 3 * W * kWave < body; i += 4 * W * kWave) {
        f32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = on ? zv[i + u * W * kWave] : zero;
#pragma unroll
        for (int u = 0; u < 4; ++u)
          dv[i + u * W * kWave] = f32x4{one(v[u][0]), one(v[u][1]), one(v[u][2]), one(v[u][3])};
      }
      for (; i < body; i += W * kWave) {
        const f32x4 v = on ? zv[i] : zero;
        dv[i] = f32x4{one(v[0]), one(v[1]), one(v[2]), one(v[3])};
      }
    } else {
      for (int i = rt; i < V; i += W * kWave) dz[i] = on ? one(z[i]) : 0.f;
    }
  }
  // This wave's stores have reached memory before any wave overwrites some.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (!on) return;
  for (int i = rt; i < top; i += W * kWave) {
    const int id = sid[i];
    if (id < 0) continue;
    // the first entry of an id writes the sum over all of them
    float p = 0.f;
    bool first = true;
    for (int j = 0; j < top; ++j) {
      if (sid[j] != id) continue;
      if (j < i) first = false;
      p += sp[j];
    }
    if (first) dz[id] = f * fast_exp2((z[id] - m) * k) - c * p;
  }
}

// Short rows (V <= 80, up to 16 entries): 16 lanes a row, four rows a wave, the
// row in registers.  With a wave a row, most lanes of a character vocabulary's
// rows are idle: 16384 x 65 forward + backward 14.5 us against 29.9, x 80 14.3 against
// 28.1 (1000 rows the same either way).  With 8 columns a lane 16384 x 96 and x 128 would
// take 14 against 28 too, 4096 x 256 with 8 entries 14.8 against 14.2, with 64 entries 28
// against 18.
constexpr int kShortVocab = 80, kShortTop = 16, kShortLanes = 16;
constexpr int kShortRows = 256 / kShortLanes;       // of a workgroup
constexpr int kShortCols = kShortVocab / kShortLanes;  // columns of a lane

__device__ __forceinline__ float sum16(float v) {
  v += dpp_quad_xor1(v);
  v += dpp_quad_xor2(v);
  v += dpp_half_mirror(v);
  v += dpp_row_mirror(v);
  return v;
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_quad_xor1(v));
  v = fmaxf(v, dpp_quad_xor2(v));
  v = fmaxf(v, dpp_half_mirror(v));
  v = fmaxf(v, dpp_row_mirror(v));
  return v;
}

// A row's teacher entries, one to each of its 16 lanes: its weight e = 2^(k (t - max))
// and their sum.
struct ShortTeacher {
  int id;
  float t, e;  // t - max, and its exponential
  float sum;
  bool on, bad;
  __device__ __forceinline__ void load(const float* Tl, const int64_t* Ti, bool here, int top, int V, float k, int l) {
    const int64_t v = here && l < top ? Ti[l] : -1;
    t = v >= 0 ? Tl[l] : -INFINITY;
    id = v >= 0 && v < V ? (int)v : -1;
    // across the row's 16 lanes
    const bool any = sum16(v >= 0 ? 1.f : 0.f) > 0.f;
    bad = sum16(v < -1 || v >= V ? 1.f : 0.f) > 0.f;
    const float tm = max16(t);
    t -= tm == -INFINITY ? 0.f : tm;
    e = id >= 0 ? fast_exp2(t * k) : 0.f;
    sum = sum16(e);
    on = any && !bad && sum != 0.f;
  }
};

// A short row's logits: column l + 16 i in slot i (-inf past the row's end).
__device__ __forceinline__ void short_row(const float* z, bool on, int V, int l, float (&x)[kShortCols]) {
#pragma unroll
  for (int i = 0; i < kShortCols; ++i) {
    const int v = l + i * kShortLanes;
    x[i] = on && v < V ? z[v] : -INFINITY;
  }
}

__global__ void __launch_bounds__(256)
distill_short_row_kernel(const float* __restrict__ Z, const float* __restrict__ Tl, const int64_t* __restrict__ Ti,
                         float* __restrict__ row_loss, float* __restrict__ stats, int64_t n, int V, int top, float k,
                         float inv_tau, float tau2, int* __restrict__ err) {
  const int l = threadIdx.x % kShortLanes;
  const int64_t row = (int64_t)blockIdx.x * kShortRows + threadIdx.x / kShortLanes;
  const bool here = row < n;
  const float* z = Z + row * V;
  ShortTeacher te;
  te.load(Tl + row * top, Ti + row * top, here, top, V, k, l);
  float x[kShortCols];
  short_row(z, te.on, V, l, x);
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kShortCols; ++i) m = fmaxf(m, x[i]);
  m = max16(m);
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < kShortCols; ++i)
    if (l + i * kShortLanes < V) s += fast_exp2((x[i] - m) * k);
  s = sum16(s);
  const float ln_s = logf(s);
  float acc = 0.f;
  if (te.on && te.id >= 0 && !(te.e == 0.f)) acc = te.e * (te.t * inv_tau - ((z[te.id] - m) * inv_tau - ln_s));
  acc = sum16(acc);
  if (!here || l != 0) return;
  if (te.bad && err) *err = 1;
  if (!te.on) {
    leave_out(row_loss, stats, row);
  } else {
    row_loss[row] = tau2 * (acc / te.sum - logf(te.sum));
    stats[2 * row] = m;
    stats[2 * row + 1] = s;
  }
}

__global__ void __launch_bounds__(256)
distill_short_bwd_kernel(const float* __restrict__ grad, const float* __restrict__ Z, const float* __restrict__ Tl,
                         const int64_t* __restrict__ Ti, const float* __restrict__ stats, float* __restrict__ dZ,
                         int64_t n, int V, int top, float k, float tau) {
  __shared__ float ps[kShortRows][kShortVocab];  // each column's p
  __shared__ int sid[kShortRows][kShortTop];
  __shared__ float sp[kShortRows][kShortTop];
  const int l = threadIdx.x % kShortLanes, r = threadIdx.x / kShortLanes;
  const int64_t row = (int64_t)blockIdx.x * kShortRows + r;
  const bool here = row < n;
  const float m = here ? stats[2 * row] : 0.f, s = here ? stats[2 * row + 1] : INFINITY;
  const bool on = s != INFINITY;
  ShortTeacher te;
  te.load(Tl + row * top, Ti + row * top, here, top, V, k, l);
  float x[kShortCols];
  short_row(Z + row * V, on, V, l, x);
#pragma unroll
  for (int i = 0; i < kShortCols; ++i) ps[r][l + i * kShortLanes] = 0.f;
  sid[r][l] = te.id;
  sp[r][l] = te.e / te.sum;
  __syncthreads();
  if (on && te.id >= 0) {
    // the first entry of an id writes the sum over all of them
    float p = 0.f;
    bool first = true;
#pragma unroll
    for (int j = 0; j < kShortTop; ++j) {
      if (sid[r][j] != te.id) continue;
      if (j < l) first = false;
      p += sp[r][j];
    }
    if (first) ps[r][te.id] = p;
  }
  __syncthreads();
  if (!here) return;
  const float c = grad[0] * tau / stats[2 * n];
  const float f = c / s;
#pragma unroll
  for (int i = 0; i < kShortCols; ++i) {
    const int v = l + i * kShortLanes;
    if (v < V) dZ[row * V + v] = on ? f * fast_exp2((x[i] - m) * k) - c * ps[r][v] : 0.f;
  }
}

// Waves per row, forward + backward in us with 1, 4 and 16: 4096 x 2048 26.9, 30.6,
// 72.8; 4096 x 4096 42.5, 40.5, 78.0; 64 x 50000 69.5, 30.6, 24.3; 500 x 50000 78.7,
// 57.2, 58.1.  So one up to 2048 columns, then a workgroup of 4, of 16 where there are
// no more rows than CUs.
int waves_per_row(int64_t n, int64_t vocab) {
  if (vocab <= 2048) return 1;
  return vocab >= 16384 && n <= (int64_t)device_cu_count() ? 16 : 4;
}

template <int W>
int launch_rows(const float* z, const float* tl, const int64_t* ti, float* row_loss, float* stats, int64_t n, int V,
                int top, float tau, int* err, hipStream_t st) {
  constexpr int kThreads = W > 4 ? W * kWave : 256;
  const int64_t blocks = ceil_div(n, kThreads / (W * kWave));
  distill_row_kernel<W><<<dim3((unsigned)blocks), dim3(kThreads), 0, st>>>(z, tl, ti, row_loss, stats, n, V, top,
                                                                          kLog2e / tau, 1.0f / tau, tau * tau, err);
  return launch_status();
}

template <int W>
int launch_bwd(const float* grad, const float* z, const float* tl, const int64_t* ti, const float* stats, float* dz,
               int64_t n, int V, int top, float tau, hipStream_t st) {
  constexpr int kThreads = W > 4 ? W * kWave : 256;
  constexpr int kRows = kThreads / (W * kWave);
  const dim3 blocks((unsigned)ceil_div(n, kRows));
  const size_t lds = (size_t)kRows * top * 2 * sizeof(int);
  // the rows of both reach 16 bytes at the same columns, or the stores do not vectorise
  if (((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15u) == 0) {
    distill_bwd_kernel<W, true><<<blocks, dim3(kThreads), lds, st>>>(grad, z, tl, ti, stats, dz, n, V, top,
                                                                     kLog2e / tau, tau);
  } else {
    distill_bwd_kernel<W, false><<<blocks, dim3(kThreads), lds, st>>>(grad, z, tl, ti, stats, dz, n, V, top,
                                                                      kLog2e / tau, tau);
  }
  return launch_status();
}

bool short_rows(int64_t vocab, int64_t top) { return vocab <= kShortVocab && top <= kShortTop; }

int launch_short(const float* z, const float* tl, const int64_t* ti, float* row_loss, float* stats, int64_t n, int V,
                 int top, float tau, int* err, hipStream_t st) {
  distill_short_row_kernel<<<dim3((unsigned)ceil_div(n, kShortRows)), dim3(256), 0, st>>>(
      z, tl, ti, row_loss, stats, n, V, top, kLog2e / tau, 1.0f / tau, tau * tau, err);
  return launch_status();
}

int launch_short_bwd(const float* grad, const float* z, const float* tl, const int64_t* ti, const float* stats,
                     float* dz, int64_t n, int V, int top, float tau, hipStream_t st) {
  distill_short_bwd_kernel<<<dim3((unsigned)ceil_div(n, kShortRows)), dim3(256), 0, st>>>(
      grad, z, tl, ti, stats, dz, n, V, top, kLog2e / tau, tau);
  return launch_status();
}

// A launch's work items are counted in 32 bits: 2^28 - 16 short rows, 2^26 - 4 of a wave,
// 2^24 - 1 of a workgroup (of 16 waves: no more than CUs).
int distill_check(int64_t n, int64_t vocab, int64_t top, float tau) {
  // (tau^2 ln(vocab) and log2(e) / tau stay in fp32's range)
  if (n < 0 || vocab <= 0 || top <= 0 || !(tau >= 0x1p-61f) || !(tau <= 0x1p61f)) return AAR_EINVAL;
  if (top > kMaxTop || vocab > INT32_MAX - 4096) return AAR_EUNSUPPORTED;
  const int64_t rows = short_rows(vocab, top) ? kShortRows : (waves_per_row(n, vocab) == 1 ? 4 : 1);  // of a workgroup
  return ceil_div(n, rows) * 256 > (int64_t)UINT32_MAX ? AAR_EUNSUPPORTED : AAR_OK;
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

// the rows' losses
size_t aar_distill_workspace_bytes(int64_t n) { return n > 0 ? (size_t)n * sizeof(float) : 0; }

int aar_distill_fwd_f32(const float* logits, const float* t_logits, const int64_t* t_ids, float* loss, float* stats,
                        int64_t n, int64_t vocab, int64_t top, float temperature, int* err, void* workspace,
                        size_t workspace_bytes, void* stream) {
  int rc = distill_check(n, vocab, top, temperature);
  if (rc != AAR_OK) return rc;
  if (!loss || !stats || (n > 0 && (!logits || !t_logits || !t_ids))) return AAR_EINVAL;
  if (n > 0 && (!workspace || workspace_bytes < aar_distill_workspace_bytes(n))) return AAR_EWORKSPACE;
  hipStream_t st = as_stream(stream);
  float* row_loss = static_cast<float*>(workspace);
  if (n > 0) {
    const int w = waves_per_row(n, vocab);
    auto launch = w == 1 ? launch_rows<1> : (w == 4 ? launch_rows<4> : launch_rows<16>);
    if (short_rows(vocab, top)) launch = launch_short;
    rc = launch(logits, t_logits, t_ids, row_loss, stats, n, (int)vocab, (int)top, temperature, err, st);
    if (rc != AAR_OK) return rc;
  }
  distill_mean_kernel<<<dim3(1), dim3(kMeanThreads), 0, st>>>(row_loss, stats, loss, n);
  return launch_status();
}

int aar_distill_bwd_f32(const float* grad, const float* logits, const float* t_logits, const int64_t* t_ids,
                        const float* stats, float* dlogits, int64_t n, int64_t vocab, int64_t top, float temperature,
                        void* stream) {
  const int rc = distill_check(n, vocab, top, temperature);
  if (rc != AAR_OK) return rc;
  if (n == 0) return AAR_OK;
  if (!grad || !logits || !t_logits || !t_ids || !stats || !dlogits) return AAR_EINVAL;
  const int w = waves_per_row(n, vocab);
  auto launch = w == 1 ? launch_bwd<1> : (w == 4 ? launch_bwd<4> : launch_bwd<16>);
  if (short_rows(vocab, top)) launch = launch_short_bwd;
  return launch(grad, logits, t_logits, t_ids, stats, dlogits, n, (int)vocab, (int)top, temperature,
                as_stream(stream));
}

}  // extern "C"
