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
// its last key, of all heads that share it; a block that holds sinks visits all later
// ones, in parts of a common length that are summed at the end.
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
  float* lse;      // [B * H][T]
  float* D;        // [B * H][T], backward
  float *dk_part, *dv_part;  // [B * Hkv][items][128][DP] partial sums
  int T, d, H, G, Hkv, BH, BHkv;  // BH = B * H query heads, BHkv = B * Hkv
  int W, S;
  int chunk, sink_blocks, sink_parts, parts;  // dK/dV: tiles of a part, blocks that hold sinks, their parts, others'
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

// Forward.  The running maximum of a row follows its scores only when they pass it by
// 2^4, so O is rarely rescaled; when it moves, the scale of P is found again.
template <int DP, bool VEC>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 3 : 2)
window_fwd_kernel(const WaArgs a) {
  using Tile = HalfTile<DP>;
  constexpr int NB = DP / 32;
  __shared__ __attribute__((aligned(16))) char ks[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char vs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float kf[2][kTile], vf[2][kTile];  // the rows' factors
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, qb = blockIdx.x / a.BH;
  const float* __restrict__ K = wa_kv_head(a.k, a, wa_kv(a, bh));
  const float* __restrict__ V = wa_kv_head(a.v, a, wa_kv(a, bh));
  const int q0 = qb * kBlock, w0 = q0 + wave * kTile, qi = w0 + lr;  // this lane's row
  const float* Q = qi < a.T ? wa_head(a.q, a, bh) + (int64_t)qi * a.q.st : nullptr;
  const WaTiles tiles(a, q0, min(q0 + kBlock, a.T) - 1);
  if (tid == 0) not_held = 0;

  u32x4 qp[DP / 16][2];
  bool row_bad = false, bad = false;
  const float qf = half_row<DP, VEC>(Q, a.d, a.scale_log2, h, qp, row_bad);
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
  auto hide = [&](f32x16& s, int kv0) {
    if (wa_all(a, w0, kv0)) return;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!wa_sees(a, qi, kv0 + acc_row(r, h))) s[r] = -INFINITY;
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
    hide(s, kv0);
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

  Tile kc[2], vc[2];
  const typename Tile::Place kat(a.k.st, a.d, tid), vat(a.v.st, a.d, tid);
  auto load = [&](int i, int t) {
    const int row0 = tiles.key(min(t, tiles.count - 1));
    kc[i].template load<VEC>(K + (int64_t)row0 * a.k.st, a.k.st, a.T - row0, a.d, kat);
    vc[i].template load<VEC>(V + (int64_t)row0 * a.v.st, a.v.st, a.T - row0, a.d, vat);
  };
  auto store = [&](int i, int buf) {
    kc[i].template store<true>(ks[buf], tid, bad);
    vc[i].template store<true>(vs[buf], tid, bad);
    if (Tile::col(tid) != 0) return;
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      const int r = Tile::row(n, tid);
      kf[buf][r] = row_factor(kc[i].ex[n]);
      vf[buf][r] = row_factor(vc[i].ex[n]);
    }
  };
  load(0, 0);
  load(1, 1);
  store(0, 0);
  load(0, 2);
  lds_barrier();
  // Iteration t: tile t in LDS, t + 1 in registers, t + 2 on its way, t + 3 sent for.
  for (int t = 0; t < tiles.count; t += 2) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u >= tiles.count) break;
      const int kv0 = tiles.key(t + u);
      if (w0 < a.T && wa_any(a, w0, kv0)) compute(u, kv0);
      store(1 - u, 1 - u);
      load(1 - u, t + u + 3);
      lds_barrier();
    }
  }
  fit.undo(o);

  if (bad) not_held = 1;
  __syncthreads();
  if (w0 < a.T && __any(row_bad || not_held)) {
    m = -INFINITY;
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
      float mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[r]);
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
          o[b] = mfma32(row < a.T && col < a.d ? finite(V[(int64_t)row * a.v.st + col]) : 0.f, s[st], o[b]);
        }
      }
      add_not_finite(V, a.v.st, kv0, a.T, a.d, s, [&](int j) { return wa_sees(a, qi, j); }, o);
    }
  }
  if (qi >= a.T) return;
  wa_store<DP, VEC>(wa_head(a.o, a, bh) + (int64_t)qi * a.o.st, o, 1.0f / l, a.d, h);
  if (h == 0) a.lse[(int64_t)bh * a.T + qi] = (m + log2f(l)) * kLn2;
}

// dQ (and D).
template <int DP, bool VEC>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 3 : 1)
window_bwd_dq_kernel(const WaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char ks[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char vs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) float kf[2][kTile], vf[2][kTile];  // the rows' factors
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bh = blockIdx.x % a.BH, qb = blockIdx.x / a.BH;
  const float* __restrict__ K = wa_kv_head(a.k, a, wa_kv(a, bh));
  const float* __restrict__ V = wa_kv_head(a.v, a, wa_kv(a, bh));
  const int q0 = qb * kBlock, w0 = q0 + wave * kTile, qi = w0 + lr;
  const bool row_ok = qi < a.T;
  const float* Q = row_ok ? wa_head(a.q, a, bh) + (int64_t)qi * a.q.st : nullptr;
  const float* dO = row_ok ? wa_head(a.dout, a, bh) + (int64_t)qi * a.dout.st : nullptr;
  const WaTiles tiles(a, q0, min(q0 + kBlock, a.T) - 1);
  if (tid == 0) not_held = 0;

  float dsum = 0.f;
  if (row_ok) {
    const float* O = wa_head(a.o_in, a, bh) + (int64_t)qi * a.o_in.st;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c) {
      const int dd = 8 * c + 4 * h;
      if (dd < a.d) {
        const f32x4 x = load4<VEC>(dO + dd, a.d - dd), y = load4<VEC>(O + dd, a.d - dd);
        dsum += x[0] * y[0] + x[1] * y[1] + x[2] * y[2] + x[3] * y[3];
      }
    }
  }
  dsum = half_swap_sum(dsum);
  const float l2 = row_ok ? a.lse[(int64_t)bh * a.T + qi] * kLog2e : INFINITY;
  if (row_ok && h == 0) a.D[(int64_t)bh * a.T + qi] = dsum;

  u32x4 qp[DP / 16][2], dop[DP / 16][2];
  bool row_bad = false, bad = false;
  const float qf = half_row<DP, VEC>(Q, a.d, a.scale_log2, h, qp, row_bad);
  const float df = half_row<DP, VEC>(dO, a.d, 1.f, h, dop, row_bad);
  f32x16 dq[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dq[b] = zero16();
  HalfScale<NB> fit;

  auto hide = [&](f32x16& x, int kv0) {
    if (wa_all(a, w0, kv0)) return;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!wa_sees(a, qi, kv0 + acc_row(r, h))) x[r] = 0.f;
  };
  Tile kc, vc;
  const typename Tile::Place kat(a.k.st, a.d, tid), vat(a.v.st, a.d, tid);
  auto load = [&](int t) {
    const int row0 = tiles.key(t);
    kc.template load<VEC>(K + (int64_t)row0 * a.k.st, a.k.st, a.T - row0, a.d, kat);
    vc.template load<VEC>(V + (int64_t)row0 * a.v.st, a.v.st, a.T - row0, a.d, vat);
  };
  auto store = [&](int buf) {
    kc.template store<true>(ks[buf], tid, bad);
    vc.template store<true>(vs[buf], tid, bad);
    if (Tile::col(tid) != 0) return;
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      const int r = Tile::row(n, tid);
      kf[buf][r] = row_factor(kc.ex[n]);
      vf[buf][r] = row_factor(vc.ex[n]);
    }
  };
  load(0);
  store(0);
  lds_barrier();
  for (int t = 0; t < tiles.count; ++t) {
    const int buf = t & 1, kv0 = tiles.key(t);
    const bool has_next = t + 1 < tiles.count;
    if (has_next) load(t + 1);
    if (w0 < a.T && wa_any(a, w0, kv0)) {
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
      hide(dp, kv0);
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
  if (w0 < a.T && __any(row_bad || not_held)) {
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
          const int row = kv0 + acc_row(st, h);
          dq[b] = mfma32(row < a.T && col < a.d ? finite(K[(int64_t)row * a.k.st + col]) : 0.f, dp[st], dq[b]);
        }
      }
      add_not_finite(K, a.k.st, kv0, a.T, a.d, dp, [&](int j) { return wa_sees(a, qi, j); }, dq);
    }
  }
  if (row_ok) wa_store<DP, VEC>(wa_head(a.dq, a, bh) + (int64_t)qi * a.dq.st, dq, a.scale, a.d, h);
}

// A part of a key block's list of query tiles: `heads` lists of `count` tiles from the
// block's first key on.
struct WaPart {
  int kb, part, parts, first, count, begin, end;
  int64_t slot;  // of its partial sums
  // Item i of a key/value head: the parts of the blocks that hold sinks, then the others'.
  __device__ __forceinline__ WaPart(const WaArgs& a, int bhk, int item) {
    const int sinks = a.sink_blocks * a.sink_parts, blocks = (a.T + kBlock - 1) / kBlock;
    const bool sink = item < sinks;
    const int i = sink ? item : item - sinks;
    parts = sink ? a.sink_parts : a.parts;
    kb = (sink ? 0 : a.sink_blocks) + i / parts;
    part = i % parts;
    first = kb * (kBlock / kTile);
    // the last query that sees a key of the block
    const int64_t most = (int64_t)kb * kBlock + kBlock - 1 + a.W - 1;
    const int last = sink || most >= a.T ? a.T - 1 : (int)most;
    count = last / kTile + 1 - first;
    begin = min(part * a.chunk, a.G * count);
    end = min(begin + a.chunk, a.G * count);
    slot = (int64_t)bhk * (sinks + (int64_t)(blocks - a.sink_blocks) * a.parts) + item;
  }
};

// dK and dV: a workgroup takes 128 keys, 32 a wave, a lane its key, and a part of the
// query tiles that see them.
template <int DP, bool VEC>
__global__ void __launch_bounds__(kFaThreads, DP == 64 ? 2 : 1)
window_bwd_dkdv_kernel(const WaArgs a) {
  constexpr int NB = DP / 32;
  using Tile = HalfTile<DP>;
  __shared__ __attribute__((aligned(16))) char qs[2][Tile::kBytes];
  __shared__ __attribute__((aligned(16))) char dos[2][Tile::kBytes];
  // factors of Q's rows and of dO's; lse in log2 and D
  __shared__ __attribute__((aligned(16))) float qf[2][kTile], df[2][kTile], ls[2][kTile], ds[2][kTile];
  __shared__ int not_held;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lr = lane & 31, h = lane >> 5;
  const int bhk = blockIdx.x % a.BHkv;
  const WaPart part(a, bhk, blockIdx.x / a.BHkv);
  const int kw = part.kb * kBlock + wave * kTile;  // the wave's first key
  const int kj = kw + lr;
  const bool key_ok = kj < a.T;
  const float* K = key_ok ? wa_kv_head(a.k, a, bhk) + (int64_t)kj * a.k.st : nullptr;
  const float* V = key_ok ? wa_kv_head(a.v, a, bhk) + (int64_t)kj * a.v.st : nullptr;
  const int head0 = bhk / a.Hkv * a.H + bhk % a.Hkv * a.G;  // the first query head
  if (tid == 0) not_held = 0;

  u32x4 kp[DP / 16][2], vp[DP / 16][2];
  bool key_bad = false, bad = false;
  const float kf = half_row<DP, VEC>(K, a.d, a.scale_log2, h, kp, key_bad);
  const float vf = half_row<DP, VEC>(V, a.d, 1.f, h, vp, key_bad);
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
  HalfScale<NB> fit_k, fit_v;

  Tile qc, dc;
  const typename Tile::Place qat(a.q.st, a.d, tid), oat(a.dout.st, a.d, tid);
  float lreg[Tile::kPer], dreg[Tile::kPer];
  auto row_of = [&](int t) { return (part.first + t % part.count) * kTile; };
  auto load = [&](int t) {
    const int bh = head0 + t / part.count, row0 = row_of(t);
    qc.template load<VEC>(wa_head(a.q, a, bh) + (int64_t)row0 * a.q.st, a.q.st, a.T - row0, a.d, qat);
    dc.template load<VEC>(wa_head(a.dout, a, bh) + (int64_t)row0 * a.dout.st, a.dout.st, a.T - row0, a.d, oat);
#pragma unroll
    for (int n = 0; n < Tile::kPer; ++n) {
      lreg[n] = dreg[n] = 0.f;
      const int r = row0 + Tile::row(n, tid);
      if (Tile::col(tid) != 0) continue;
      lreg[n] = r < a.T ? a.lse[(int64_t)bh * a.T + r] * kLog2e : INFINITY;
      dreg[n] = r < a.T ? a.D[(int64_t)bh * a.T + r] : 0.f;
    }
  };
  auto store = [&](int buf) {
    qc.template store<true>(qs[buf], tid, bad);
    dc.template store<true>(dos[buf], tid, bad);
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
  // P or dS of the queries from i0 on that do not see the lane's key
  auto hide = [&](f32x16& p, int i0) {
    if (wa_all(a, i0, kw)) return;
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (!wa_sees(a, i0 + acc_row(r, h), kj)) p[r] = 0.f;
  };
  if (part.begin < part.end) {
    load(part.begin);
    store(0);
  }
  lds_barrier();
  for (int t = part.begin; t < part.end; ++t) {
    const int cur = (t - part.begin) & 1, i0 = row_of(t);
    const bool has_next = t + 1 < part.end;
    if (has_next) load(t + 1);
    if (kw < a.T && wa_any(a, i0, kw)) {
      f32x16 s = half_rows<DP>(qs[cur], kp, lr, h);
      sched_fence();
      f32x16 x;
      float top = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 q4 = row_values(qf[cur], g, h), l4 = row_values(ls[cur], g, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          s[r] = key_ok ? fast_exp2(s[r] * q4[e] * kf - l4[e]) : 0.f;
        }
      }
      hide(s, i0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 o4 = row_values(df[cur], g, h);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
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
        }
      }
      hide(x, i0);  // where D is not finite
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
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
  if (kw < a.T && part.begin < part.end && __any(key_bad || not_held)) {
#pragma unroll
    for (int b = 0; b < NB; ++b) dk[b] = dv[b] = zero16();
    for (int t = part.begin; t < part.end; ++t) {
      const int i0 = row_of(t), bh = head0 + t / part.count;
      if (!wa_any(a, i0, kw)) continue;
      const float* Qh = wa_head(a.q, a, bh);
      const float* dOh = wa_head(a.dout, a, bh);
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
        const int64_t at = (int64_t)bh * a.T + (i < a.T ? i : 0);
        s[r] = sees ? fast_exp2(s[r] - a.lse[at] * kLog2e) : 0.f;
        dp[r] = sees ? s[r] * (dp[r] - a.D[at]) : 0.f;
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
  if (part.parts > 1) {
    const int64_t at = (part.slot * kBlock + wave * kTile + lr) * DP;
    wa_store<DP, true>(a.dk_part + at, dk, a.scale, DP, h);
    wa_store<DP, true>(a.dv_part + at, dv, 1.0f, DP, h);
  } else {
    wa_store<DP, VEC>(wa_kv_head(a.dk, a, bhk) + (int64_t)kj * a.dk.st, dk, a.scale, a.d, h);
    wa_store<DP, VEC>(wa_kv_head(a.dv, a, bhk) + (int64_t)kj * a.dv.st, dv, 1.0f, a.d, h);
  }
}

// The parts of dK and dV of the first `rows` keys of every head, summed in order.
template <int DP, bool VEC>
__global__ void __launch_bounds__(256)
window_bwd_sum_kernel(const WaArgs a, int first, int rows) {
  constexpr int kLanes = DP / 4;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, item = u / kLanes;
  const int c = (int)(u % kLanes) * 4, bhk = (int)(item / rows), key = first + (int)(item % rows);
  if (bhk >= a.BHkv || c >= a.d) return;
  const int kb = key / kBlock;
  const bool sink = kb < a.sink_blocks;
  const WaPart part(a, bhk, sink ? kb * a.sink_parts : a.sink_blocks * a.sink_parts + (kb - a.sink_blocks) * a.parts);
  const int parts = (a.G * part.count + a.chunk - 1) / a.chunk;
  const int64_t at = (part.slot * kBlock + key % kBlock) * DP + c;
  f32x4 dk = *reinterpret_cast<const f32x4*>(a.dk_part + at), dv = *reinterpret_cast<const f32x4*>(a.dv_part + at);
#pragma unroll 4
  for (int p = 1; p < parts; ++p) {
    dk += *reinterpret_cast<const f32x4*>(a.dk_part + at + (int64_t)p * kBlock * DP);
    dv += *reinterpret_cast<const f32x4*>(a.dv_part + at + (int64_t)p * kBlock * DP);
  }
  store4<VEC>(wa_kv_head(a.dk, a, bhk) + (int64_t)key * a.dk.st + c, dk, a.d - c);
  store4<VEC>(wa_kv_head(a.dv, a, bhk) + (int64_t)key * a.dv.st + c, dv, a.d - c);
}

// ------------------------------------------------------------------ host side

int wa_dim(int64_t d) { return d <= 64 ? 64 : 128; }

int wa_check(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window, int64_t sinks) {
  if (B < 0 || H < 0 || Hkv < 0 || T < 0 || d <= 0 || d > 128 || window < 1 || sinks < 0) return AAR_EINVAL;
  if ((H == 0) != (Hkv == 0) || (H > 0 && H % Hkv != 0)) return AAR_EINVAL;
  if (B > (1 << 20) || H > (1 << 20) || T > (1 << 24)) return AAR_EUNSUPPORTED;
  // a dispatch holds its work items in 32 bits
  if (B * H * ceil_div(T, kBlock) >= (1 << 24) || B * H * T > (int64_t)UINT32_MAX / 32) return AAR_EUNSUPPORTED;
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
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  return a;
}

// Parts of dK's and dV's query tiles.
void wa_bwd_plan(WaArgs& a) {
  const int blocks = (int)ceil_div(a.T, kBlock), all = (int)ceil_div(a.T, kTile);
  const int near = (int)std::min<int64_t>(all, ceil_div(kBlock + (int64_t)a.W - 1, kTile) + 1);
  a.sink_blocks = (int)std::min<int64_t>(ceil_div(a.S, kBlock), blocks);
  // at most 64 parts of the sinks' blocks in all, each as long as another block's list at least
  a.chunk = std::max(a.G * near, (int)ceil_div((int64_t)a.G * all, std::max(1, 64 / std::max(1, a.sink_blocks))));
  a.parts = 1;
  a.sink_parts = (int)ceil_div((int64_t)a.G * all, a.chunk);
}

int64_t wa_items(const WaArgs& a) {
  return (int64_t)a.sink_blocks * a.sink_parts + (ceil_div(a.T, kBlock) - a.sink_blocks) * a.parts;
}
bool wa_split(const WaArgs& a) { return a.parts > 1 || (a.sink_blocks > 0 && a.sink_parts > 1); }

// D, then the parts of dK and of dV.
size_t wa_part_bytes(const WaArgs& a) {
  return wa_split(a) ? (size_t)a.BHkv * wa_items(a) * kBlock * wa_dim(a.d) * sizeof(float) : 0;
}
size_t wa_d_bytes(const WaArgs& a) { return ((size_t)a.BH * a.T * sizeof(float) + 15) / 16 * 16; }

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
int launch_fwd(const WaArgs& a, hipStream_t st) {
  window_fwd_kernel<DP, VEC><<<dim3((unsigned)(ceil_div(a.T, kBlock) * a.BH)), dim3(kFaThreads), 0, st>>>(a);
  return launch_status();
}

template <int DP, bool VEC>
int launch_bwd(const WaArgs& a, hipStream_t st) {
  window_bwd_dq_kernel<DP, VEC><<<dim3((unsigned)(ceil_div(a.T, kBlock) * a.BH)), dim3(kFaThreads), 0, st>>>(a);
  int rc = launch_status();
  if (rc != AAR_OK) return rc;
  window_bwd_dkdv_kernel<DP, VEC><<<dim3((unsigned)(wa_items(a) * a.BHkv)), dim3(kFaThreads), 0, st>>>(a);
  rc = launch_status();
  if (rc != AAR_OK || !wa_split(a)) return rc;
  const int first = a.sink_blocks > 0 && a.sink_parts > 1 ? 0 : a.sink_blocks * kBlock;
  const int last = a.parts > 1 ? a.T : std::min(a.T, a.sink_blocks * kBlock), rows = last - first;
  const int64_t units = (int64_t)a.BHkv * rows * (DP / 4);
  window_bwd_sum_kernel<DP, VEC><<<dim3((unsigned)ceil_div(units, 256)), dim3(256), 0, st>>>(a, first, rows);
  return launch_status();
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

size_t aar_window_attn_fwd_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t d, int64_t window,
                                           int64_t sinks) {
  (void)B, (void)H, (void)Hkv, (void)T, (void)d, (void)window, (void)sinks;
  return 0;
}

int aar_window_attn_fwd_f32(const float* q, const float* k, const float* v, float* o, float* lse, int64_t B, int64_t H,
                            int64_t Hkv, int64_t T, int64_t d, const int64_t* strides, int64_t window, int64_t sinks,
                            float scale, void* workspace, size_t workspace_bytes, void* stream) {
  (void)workspace, (void)workspace_bytes;
  const int rc = wa_check(B, H, Hkv, T, d, window, sinks);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0 || T == 0) return AAR_OK;
  if (!q || !k || !v || !o || !lse || !strides) return AAR_EINVAL;
  if (!wa_rows_ok(strides, {0, 1, 2}, T, d)) return AAR_EUNSUPPORTED;
  WaArgs a = wa_args(B, H, Hkv, T, d, window, sinks, scale);
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
  return wa_d_bytes(a) + 2 * wa_part_bytes(a);
}

int aar_window_attn_bwd_f32(const float* q, const float* k, const float* v, const float* o, const float* lse,
                            const float* dout, float* dq, float* dk, float* dv, int64_t B, int64_t H, int64_t Hkv,
                            int64_t T, int64_t d, const int64_t* strides, int64_t window, int64_t sinks, float scale,
                            void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = wa_check(B, H, Hkv, T, d, window, sinks);
  if (rc != AAR_OK) return rc;
  if (B == 0 || H == 0 || T == 0) return AAR_OK;
  if (!q || !k || !v || !o || !lse || !dout || !dq || !dk || !dv || !strides) return AAR_EINVAL;
  if (!wa_rows_ok(strides, {0, 1, 2, 4}, T, d)) return AAR_EUNSUPPORTED;
  WaArgs a = wa_args(B, H, Hkv, T, d, window, sinks, scale);
  wa_bwd_plan(a);
  if (!workspace || !aligned16(workspace) || workspace_bytes < wa_d_bytes(a) + 2 * wa_part_bytes(a)) return AAR_EWORKSPACE;
  char* ws = static_cast<char*>(workspace);
  a.D = reinterpret_cast<float*>(ws);
  a.dk_part = reinterpret_cast<float*>(ws + wa_d_bytes(a));
  a.dv_part = reinterpret_cast<float*>(ws + wa_d_bytes(a) + wa_part_bytes(a));
  a.lse = const_cast<float*>(lse);
  a.q = wa_in(q, strides, T, d);
  a.k = wa_in(k, strides + 3, T, d);
  a.v = wa_in(v, strides + 6, T, d);
  a.o_in = FaIn{o, strides[9], strides[10], strides[11]};
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
