// Scaled embedding lookup and its gradient by sorted tokens.
//
//   out[i] = scale w[ids[i]],     dw[v] = scale sum_{i: ids[i] = v} g[i].
//
// Bound by HBM: the lookup reads and writes n rows; the gradient reads n rows
// and writes every row of the table, most of them zeros in a subword vocabulary.
// Three launches, no float atomics, so the same bits on every run:
//  1 sort    each workgroup owns a slice of the vocabulary and reads all ids (a
//            few hundred KB that stay in the caches): counts per id, the number
//            of ids below its slice, hence where each of its ids' runs begins,
//            and on a second reading the tokens of every run in their order.  No
//            workgroup waits for another, where a radix sort needs seven launches.
//  2 sum     a wave per chunk of sorted tokens and 256 columns adds up runs; a run
//            inside the chunk goes to its row, one that crosses chunks leaves a
//            partial row per chunk.  Chunks are equally long, so a token that
//            takes a tenth of the batch is spread like any other.  Further waves
//            zero the rows that no token names.
//  3 join    the workgroup of the chunk where a crossing run begins adds its
//            partial rows, a quarter of them a wave, in a fixed order.
// 32768 tokens of 50000 ids, 768 columns: lookup 30 us, sort 16, sum 49 (254 MB at 5.2
// TB/s), join 8.  16384 tokens of 65 ids, 384 columns: 6, 12, 7 and 6, the launches'
// and the ids' latencies.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "common.hpp"

namespace aar {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kMaxSlice = 1024;  // ids of a workgroup: one scan of its threads; 64 KB of counts

__global__ void __launch_bounds__(256)
embed_scaled_vec_kernel(const f32x4* __restrict__ w, const int64_t* __restrict__ ids, f32x4* __restrict__ out,
                        int64_t n, int64_t vocab, int64_t dim4, float scale, int* __restrict__ err) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= n) return;
  const int64_t id = ids[i];
  const bool ok = id >= 0 && id < vocab;
  if (!ok && lane == 0 && err) *err = 1;
  const f32x4* src = w + (ok ? id : 0) * dim4;
  f32x4* dst = out + i * dim4;
  const float f = ok ? scale : 0.f;
  constexpr int kU = 4;  // loads in flight
  for (int64_t k = lane; k < dim4; k += kU * kWave) {
    f32x4 v[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      v[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (ok && k + u * kWave < dim4) v[u] = src[k + u * kWave];
    }
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (k + u * kWave < dim4) __builtin_nontemporal_store(v[u] * f, dst + k + u * kWave);
  }
}

__global__ void __launch_bounds__(256)
embed_scaled_kernel(const float* __restrict__ w, const int64_t* __restrict__ ids, float* __restrict__ out, int64_t n,
                    int64_t vocab, int64_t dim, float scale, int* __restrict__ err) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (i >= n) return;
  const int64_t id = ids[i];
  const bool ok = id >= 0 && id < vocab;
  if (!ok && lane == 0 && err) *err = 1;
  for (int64_t k = lane; k < dim; k += kWave) out[i * dim + k] = ok ? w[id * dim + k] * scale : 0.f;
}

// Sorted tokens and run starts: start[v] for v <= vocab, token[] in runs of
// equal ids, each in the tokens' order, and sid[] their ids.  Bound by the latency
// of the ids' loads, so a wave has 32 groups of 64 in flight, and those of up to
// 32768 tokens stay in registers for the second reading.
__global__ void __launch_bounds__(kSortThreads)
embed_sort_kernel(const int64_t* __restrict__ ids, int n, int vocab, int slice, int* __restrict__ token,
                  int* __restrict__ sid, int* __restrict__ start) {
  __shared__ int cnt[kSortWaves * kMaxSlice];  // [wave][id]: counts, then where the wave's next token goes
  __shared__ int sums[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int v0 = blockIdx.x * slice, nv = min(slice, vocab - v0);
  for (int i = tid; i < kSortWaves * slice; i += kSortThreads) cnt[i] = 0;
  __syncthreads();

  // A wave's part of the tokens, whole groups of 64.
  const int per = ((n + kSortWaves - 1) / kSortWaves + kWave - 1) / kWave * kWave;
  const int t0 = min(n, wave * per), t1 = min(n, t0 + per);
  int* mine = cnt + wave * slice;
  int below = 0;
  constexpr int kU = 32;
  int r[kU];  // the groups' ids within the slice, -1 for the others
  auto read = [&](int b) {
    int64_t id[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int i = b + u * kWave + lane;
      id[u] = i < t1 ? ids[i] : -1;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      below += id[u] >= 0 && id[u] < v0 ? 1 : 0;
      r[u] = id[u] >= v0 && id[u] < v0 + nv ? (int)(id[u] - v0) : -1;
    }
  };
  for (int b = t0; b < t1; b += kU * kWave) {
    read(b);
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (r[u] >= 0) atomicAdd(&mine[r[u]], 1);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o, kWave);
  if (lane == 0) sums[wave] = below;
  __syncthreads();
  int base = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) base += sums[w];
  __syncthreads();

  // Exclusive scan of the ids' counts (thread = id), then of each id's waves.
  int total = 0;
  if (tid < nv)
    for (int w = 0; w < kSortWaves; ++w) total += cnt[w * slice + tid];
  int inc = total;
#pragma unroll
  for (int o = 1; o < kWave; o *= 2) {
    const int up = __shfl_up(inc, o, kWave);
    if (lane >= o) inc += up;
  }
  if (lane == kWave - 1) sums[wave] = inc;
  __syncthreads();
  for (int w = 0; w < wave; ++w) base += sums[w];
  if (tid < nv) {
    int at = base + inc - total;
    start[v0 + tid] = at;
    if (v0 + tid == vocab - 1) start[vocab] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = cnt[w * slice + tid];
      cnt[w * slice + tid] = at;
      at += c;
    }
  }
  __syncthreads();

  // The tokens, group by group: the lanes that hold the same id take its next
  // places in lane order.
  for (int b = t0; b < t1; b += kU * kWave) {
    if (per > kU * kWave) read(b);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      unsigned long long todo = __ballot(r[u] >= 0);
      if (todo == 0) continue;
      const int at = r[u] >= 0 ? mine[r[u]] : 0;
      int rank = 0, count = 0;  // among the group's lanes of the same id
      while (todo) {
        const int rr = __builtin_amdgcn_readlane(r[u], __builtin_ctzll(todo));
        const unsigned long long same = __ballot(r[u] == rr);
        if (r[u] == rr) {
          rank = __builtin_popcountll(same & ((1ull << lane) - 1));
          count = __builtin_popcountll(same);
        }
        todo &= ~same;
      }
      if (r[u] >= 0) {
        token[at + rank] = b + u * kWave + lane;
        sid[at + rank] = v0 + r[u];
        if (rank == 0) mine[r[u]] = at + count;
      }
      // The next group's lanes read what these wrote: LDS keeps a wave's order, and this the compiler's.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

struct EmbedArgs {
  const float* g;
  const int* token;
  const int* sid;
  const int* start;
  float* part;  // [chunks][2][dim]: the run that began before the chunk, the one that goes on after it
  float* dw;
  int64_t dim;
  int n, vocab, chunk, chunks;
  int block0, blocks;  // the launch's part of a row's blocks of 64 lanes' columns
  int zero_waves;
  float scale;
};

template <bool VEC>
using EmbedVec = typename std::conditional<VEC, f32x4, float>::type;

__device__ __forceinline__ float embed_zero(float*) { return 0.f; }
__device__ __forceinline__ f32x4 embed_zero(f32x4*) { return f32x4{0.f, 0.f, 0.f, 0.f}; }

// Ids whose empty rows one wave zeroes (89139 rows of 896: 59 us, with 16 ids 63, 64 65).
constexpr int kZeroIds = 4;
constexpr int kRows = 8;      // rows whose loads a wave has in flight

template <bool VEC>
__global__ void __launch_bounds__(256)
embed_sum_kernel(const EmbedArgs a) {
  using V = EmbedVec<VEC>;
  constexpr int kE = VEC ? 4 : 1;
  const int lane = threadIdx.x & 63;
  int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t dimv = a.dim / kE;
  const V zero = embed_zero((V*)nullptr);
  if (unit >= (int64_t)a.chunks * a.blocks) {
    // rows without a token
    unit -= (int64_t)a.chunks * a.blocks;
    if (unit >= a.zero_waves) return;
    for (int64_t v0 = unit * kZeroIds; v0 < a.vocab; v0 += (int64_t)a.zero_waves * kZeroIds) {
      const int v = (int)v0 + lane;
      const bool empty = lane < kZeroIds && v < a.vocab && a.start[v] == a.start[v + 1];
      unsigned long long todo = __ballot(empty);
      while (todo) {
        const int l = __builtin_ctzll(todo);
        V* row = reinterpret_cast<V*>(a.dw + (v0 + l) * a.dim);
        for (int64_t c = lane; c < dimv; c += kWave) __builtin_nontemporal_store(zero, row + c);
        todo &= todo - 1;
      }
    }
    return;
  }
  const int chunk = (int)(unit / a.blocks);
  const int64_t col = (a.block0 + unit % a.blocks) * kWave + lane;
  const bool on = col < dimv;
  const int total = a.start[a.vocab];
  const int p0 = chunk * a.chunk, p1 = min(total, p0 + a.chunk);
  if (p0 >= p1) return;
  const V* g = reinterpret_cast<const V*>(a.g) + (on ? col : 0);
  V acc = zero;
  int cur = -1;
  // A run's sum: to its row, or where it crosses the chunk's ends to a partial row.
  auto flush = [&]() {
    if (cur < 0 || !on) return;
    if (a.start[cur] < p0) {
      reinterpret_cast<V*>(a.part + (int64_t)2 * chunk * a.dim)[col] = acc;
    } else if (a.start[cur + 1] > p1) {
      reinterpret_cast<V*>(a.part + ((int64_t)2 * chunk + 1) * a.dim)[col] = acc;
    } else {
      reinterpret_cast<V*>(a.dw + (int64_t)cur * a.dim)[col] = acc * a.scale;
    }
  };
  for (int b = p0; b < p1; b += kWave) {
    const int nb = min(kWave, p1 - b);
    const int tok = lane < nb ? a.token[b + lane] : 0;
    const int id = lane < nb ? a.sid[b + lane] : 0;
    for (int j = 0; j < nb; j += kRows) {
      V x[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        const int t = __builtin_amdgcn_readlane(tok, min(j + u, nb - 1));
        x[u] = on ? g[(int64_t)t * dimv] : zero;
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        if (j + u >= nb) break;
        const int v = __builtin_amdgcn_readlane(id, j + u);
        if (v != cur) {
          flush();
          cur = v;
          acc = zero;
        }
        acc += x[u];
      }
    }
  }
  flush();
}

template <bool VEC>
__global__ void __launch_bounds__(256)
embed_join_kernel(const EmbedArgs a) {
  using V = EmbedVec<VEC>;
  constexpr int kE = VEC ? 4 : 1;
  __shared__ V red[4][kWave];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chunk = (int)(blockIdx.x / (unsigned)a.blocks);
  const int64_t dimv = a.dim / kE;
  const int64_t col = (a.block0 + (int64_t)(blockIdx.x % (unsigned)a.blocks)) * kWave + lane;
  const int total = a.start[a.vocab];
  const int p0 = chunk * a.chunk, p1 = p0 + a.chunk;
  if (p1 >= total) return;  // the last chunk's runs end in it
  const int v = a.sid[p1 - 1];
  const int end = a.start[v + 1];
  if (a.start[v] < p0 || end <= p1) return;  // began before, or ends here
  const int last = (end - 1) / a.chunk;      // partial rows: chunk's second, then the first of chunk + 1 .. last
  const int count = last - chunk + 1;
  const int per = (count + 3) / 4;
  const int i0 = wave * per, i1 = min(count, i0 + per);
  const V zero = embed_zero((V*)nullptr);
  V acc = zero;
  if (col < dimv) {
    auto at = [&](int i) {
      const int64_t row = i == 0 ? 2 * (int64_t)chunk + 1 : 2 * ((int64_t)chunk + i);
      return reinterpret_cast<const V*>(a.part + row * a.dim)[col];
    };
    int i = i0;
    for (; i + kRows <= i1; i += kRows) {
      V x[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) x[u] = at(i + u);
#pragma unroll
      for (int u = 0; u < kRows; ++u) acc += x[u];
    }
    for (; i < i1; ++i) acc += at(i);
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && col < dimv)
    reinterpret_cast<V*>(a.dw + (int64_t)v * a.dim)[col] =
        ((red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane])) * a.scale;
}

// Ids per sorting workgroup: 256 slices of a vocabulary (lookup + gradient of 32768
// tokens of 50000 ids 104 us; 128 slices 106, 512 slices 113), more of a large one.
int64_t slice_ids(int64_t vocab) { return std::min<int64_t>(kMaxSlice, ceil_div(vocab, 256)); }

// Sorted tokens per chunk: about 2000 chunks of a large batch (so a run has at most
// that many partial rows), 16 tokens at least.  131072 tokens of 50000 ids, 256
// columns, lookup + gradient: 159 us, with 512 chunks 211, 1024 170, 4096 156.
int64_t chunk_tokens(int64_t n) { return std::max<int64_t>(16, ceil_div(ceil_div(n, 2048), kRows) * kRows); }

size_t round16(size_t b) { return (b + 15) / 16 * 16; }
size_t token_bytes(int64_t n) { return round16((size_t)n * sizeof(int)); }
size_t start_bytes(int64_t vocab) { return round16(((size_t)vocab + 1) * sizeof(int)); }

bool embed_shape_ok(int64_t n, int64_t vocab, int64_t dim) {
  return n <= INT32_MAX - 65536 && vocab <= INT32_MAX - 65536 && dim <= INT32_MAX;
}

// A launch's work items are counted in 32 bits, so tables of more than 2^26 ids are
// zeroed by waves that take several fours of them, and rows of more columns than 2^24
// waves (or the join's workgroups) cover go in several launches.
constexpr int64_t kMaxWaves = (int64_t(1) << 24) - 1;

template <bool VEC>
int launch_sum(EmbedArgs a, hipStream_t st) {
  const int64_t blocks = ceil_div(a.dim, (VEC ? 4 : 1) * kWave), most = std::max<int64_t>(1, kMaxWaves / a.chunks);
  for (int64_t b = 0; b < blocks; b += most) {
    a.block0 = (int)b;
    a.blocks = (int)std::min(most, blocks - b);
    a.zero_waves = b == 0 ? (int)std::min<int64_t>(ceil_div(a.vocab, kZeroIds), kMaxWaves) : 0;
    const int64_t sums = (int64_t)a.chunks * a.blocks;
    embed_sum_kernel<VEC><<<dim3((unsigned)ceil_div(sums + a.zero_waves, 4)), dim3(256), 0, st>>>(a);
    int rc = launch_status();
    if (rc != AAR_OK) return rc;
    if (a.chunks < 2) continue;
    embed_join_kernel<VEC><<<dim3((unsigned)sums), dim3(256), 0, st>>>(a);
    rc = launch_status();
    if (rc != AAR_OK) return rc;
  }
  return AAR_OK;
}

}  // namespace
}  // namespace aar

using namespace aar;

extern "C" {

int aar_embedding_scaled_fwd_f32(const float* w, const int64_t* ids, float* out, int64_t n, int64_t vocab, int64_t dim,
                                 float scale, int* err, void* stream) {
  if (n < 0 || vocab < 0 || dim < 0) return AAR_EINVAL;
  if (n == 0 || dim == 0) return AAR_OK;
  if (!ids || !out || (vocab > 0 && !w)) return AAR_EINVAL;
  if (ceil_div(n, 4) * 256 > (int64_t)UINT32_MAX) return AAR_EUNSUPPORTED;
  const dim3 grid((unsigned)ceil_div(n, 4));
  if (dim % 4 == 0 && (vocab == 0 || aligned16(w)) && aligned16(out)) {
    embed_scaled_vec_kernel<<<grid, dim3(256), 0, as_stream(stream)>>>(
        reinterpret_cast<const f32x4*>(w), ids, reinterpret_cast<f32x4*>(out), n, vocab, dim / 4, scale, err);
  } else {
    embed_scaled_kernel<<<grid, dim3(256), 0, as_stream(stream)>>>(w, ids, out, n, vocab, dim, scale, err);
  }
  return launch_status();
}

size_t aar_embedding_sorted_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t dim) {
  if (n <= 0 || vocab <= 0 || dim <= 0 || !embed_shape_ok(n, vocab, dim)) return 0;
  const int64_t chunks = ceil_div(n, chunk_tokens(n));
  return 2 * token_bytes(n) + start_bytes(vocab) + (size_t)chunks * 2 * (size_t)dim * sizeof(float);
}

int aar_embedding_sorted_bwd_f32(const float* g, const int64_t* ids, float* dw, int64_t n, int64_t vocab, int64_t dim,
                                 float scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (n < 0 || vocab < 0 || dim < 0) return AAR_EINVAL;
  if (vocab == 0 || dim == 0) return AAR_OK;
  if (!dw) return AAR_EINVAL;
  if (n == 0) return aar_memset_zero(dw, (size_t)vocab * dim * sizeof(float), stream);
  if (!g || !ids) return AAR_EINVAL;
  if (!embed_shape_ok(n, vocab, dim)) return AAR_EUNSUPPORTED;
  if (!workspace || !aligned16(workspace) || workspace_bytes < aar_embedding_sorted_bwd_workspace_bytes(n, vocab, dim))
    return AAR_EWORKSPACE;
  hipStream_t st = as_stream(stream);
  char* ws = static_cast<char*>(workspace);
  int* token = reinterpret_cast<int*>(ws);
  int* sid = reinterpret_cast<int*>(ws + token_bytes(n));
  int* start = reinterpret_cast<int*>(ws + 2 * token_bytes(n));
  const int64_t slice = slice_ids(vocab), chunk = chunk_tokens(n);
  EmbedArgs a{g, token, sid, start, reinterpret_cast<float*>(ws + 2 * token_bytes(n) + start_bytes(vocab)), dw, dim,
              (int)n, (int)vocab, (int)chunk, (int)ceil_div(n, chunk), 0, 0, 0, scale};
  const bool vec = dim % 4 == 0 && aligned16(g) && aligned16(dw);
  embed_sort_kernel<<<dim3((unsigned)ceil_div(vocab, slice)), dim3(kSortThreads), 0, st>>>(ids, (int)n, (int)vocab,
                                                                                          (int)slice, token, sid, start);
  const int rc = launch_status();
  if (rc != AAR_OK) return rc;
  return vec ? launch_sum<true>(a, st) : launch_sum<false>(a, st);
}

}  // extern "C"
