// Attention over part of a text, and a cache of its keys and values: window attention
// with sinks, and the paged 8-bit cache that generation reads.  The reference has no
// counterparts; checks, messages and autograd Functions follow those of
// flash_attention.  Device work runs in csrc/hip/{window_attn,kv_cache,kv_attn}.hip.
#include <algorithm>
#include <cmath>
#include <functional>
#include <string>

#include "aar_hip.h"
#include "kv_cache.hpp"
#include "ops.hpp"

namespace aar {

namespace {

const float* fp(const Tensor& t) { return static_cast<const float*>(t.data()); }
float* fp(Tensor& t) { return static_cast<float*>(t.data()); }
const int64_t* ip(const Tensor& t) { return static_cast<const int64_t*>(t.data()); }

Tensor as_contig(const Tensor& t) { return t.is_contiguous() ? t : contiguous(t); }

constexpr int64_t kRowMost = int64_t(1) << 23;  // floats between rows that the kernels take

// A [B, H, T, d] operand the kernels read in place: the head dim contiguous and rows
// apart by at least their length, else a dense copy.
Tensor head_view(const Tensor& t) {
  const bool unit = t.strides[3] == 1 || t.shape[3] == 1;
  const bool rows = t.shape[2] <= 1 || (t.strides[2] >= t.shape[3] && t.strides[2] <= kRowMost);
  return unit && rows ? t : contiguous(t);
}
void strides_of(int64_t* dst, const Tensor& t) {
  for (int i = 0; i < 3; ++i) dst[i] = t.strides[i];
}

struct WindowDims {
  int64_t B = 0, H = 0, Hkv = 0, T = 0, d = 0, window = 1, sinks = 0;
};

void check_window(int64_t window, int64_t sinks, const char* op) {
  if (window < 1) throw std::invalid_argument(std::string(op) + ": window must be at least 1");
  if (sinks < 0) throw std::invalid_argument(std::string(op) + ": sinks must not be negative");
}

void check_heads(const WindowDims& c) {
  if (c.H <= 0 || c.Hkv <= 0 || c.H % c.Hkv != 0) {
    throw std::invalid_argument("window_attention: query heads must be a multiple of key/value heads");
  }
  if (c.d <= 0 || c.d > 128) throw std::invalid_argument("window_attention: d_head must be in [1, 128]");
}

void window_forward(const WindowDims& c, const float* q, const float* k, const float* v, float* o, float* lse,
                    const int64_t* st) {
  const float s = 1.0f / std::sqrt(static_cast<float>(c.d));
  Workspace ws(aar_window_attn_fwd_workspace_bytes(c.B, c.H, c.Hkv, c.T, c.d, c.window, c.sinks));
  check_status(aar_window_attn_fwd_f32(q, k, v, o, lse, c.B, c.H, c.Hkv, c.T, c.d, st, c.window, c.sinks, s, ws.data(),
                                       ws.bytes(), current_stream()),
               "window_attention");
}

void window_backward(const WindowDims& c, const float* q, const float* k, const float* v, const float* o,
                     const float* lse, const float* go, float* dq, float* dk, float* dv, const int64_t* st) {
  const float s = 1.0f / std::sqrt(static_cast<float>(c.d));
  Workspace ws(aar_window_attn_bwd_workspace_bytes(c.B, c.H, c.Hkv, c.T, c.d, c.window, c.sinks));
  check_status(aar_window_attn_bwd_f32(q, k, v, o, lse, go, dq, dk, dv, c.B, c.H, c.Hkv, c.T, c.d, st, c.window,
                                       c.sinks, s, ws.data(), ws.bytes(), current_stream()),
               "window_attention backward");
}

class WindowAttentionFunction : public Function {
 public:
  Tensor q, k, v, saved_o, saved_lse;
  WindowDims dims;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor go = head_view(g);
    Tensor dq = Tensor::empty(q.shape, q.dtype, q.device);
    Tensor dk = Tensor::empty(k.shape, k.dtype, k.device);
    Tensor dv = Tensor::empty(v.shape, v.dtype, v.device);
    int64_t st[24];
    const Tensor* ops[8] = {&q, &k, &v, &saved_o, &go, &dq, &dk, &dv};
    for (int i = 0; i < 8; ++i) strides_of(st + 3 * i, *ops[i]);
    window_backward(dims, fp(q), fp(k), fp(v), fp(saved_o), fp(saved_lse), fp(go), fp(dq), fp(dk), fp(dv), st);
    return {dq, dk, dv};
  }
  const char* name() const override { return "WindowAttentionFunction"; }
};

// qkv [..., T, (H + 2 Hkv) d] (queries, keys, values) -> [..., T, H d].
class WindowQKVFunction : public Function {
 public:
  Tensor qkv, saved_o, saved_lse;
  WindowDims dims;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor go = as_contig(g);
    Tensor dqkv = Tensor::empty(qkv.shape, qkv.dtype, qkv.device);
    int64_t st[24];
    packed_strides(dims, st, 8);
    const int64_t kat = dims.H * dims.d, vat = kat + dims.Hkv * dims.d;
    const float* x = fp(qkv);
    float* y = fp(dqkv);
    if (qkv.numel() == 0) return {dqkv};
    window_backward(dims, x, x + kat, x + vat, fp(saved_o), fp(saved_lse), fp(go), y, y + kat, y + vat, st);
    return {dqkv};
  }
  const char* name() const override { return "WindowQKVFunction"; }

  // q, k, v, o, dout, dq, dk, dv
  static void packed_strides(const WindowDims& c, int64_t* st, int n) {
    const int64_t wide = (c.H + 2 * c.Hkv) * c.d, one = c.H * c.d;
    for (int i = 0; i < n; ++i) {
      const int64_t row = i == 3 || i == 4 ? one : wide;
      st[3 * i] = c.T * row;
      st[3 * i + 1] = c.d;
      st[3 * i + 2] = row;
    }
  }
};

}  // namespace

Tensor window_attention(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window, int64_t sinks) {
  if (q.dtype != DType::Fp32 || k.dtype != DType::Fp32 || v.dtype != DType::Fp32) {
    throw std::invalid_argument("window_attention: only Fp32 supported");
  }
  if (q.device != k.device || q.device != v.device) throw std::invalid_argument("window_attention: device mismatch");
  if (q.shape.size() != 4 || k.shape.size() != 4 || v.shape.size() != 4) {
    throw std::invalid_argument("window_attention: q, k, v must be 4D [B, H, T, d]");
  }
  if (k.shape != v.shape) throw std::invalid_argument("window_attention: k and v must share shape");
  if (k.shape[0] != q.shape[0] || k.shape[2] != q.shape[2] || k.shape[3] != q.shape[3]) {
    throw std::invalid_argument("window_attention: q and k must share batch, length and head dim");
  }
  WindowDims c{q.shape[0], q.shape[1], k.shape[1], q.shape[2], q.shape[3], window, sinks};
  check_heads(c);
  check_window(window, sinks, "window_attention");
  if (q.device == Device::CPU) throw_cpu_compute("window_attention");
  Tensor qv = head_view(q), kv = head_view(k), vv = head_view(v);
  Tensor out = Tensor::empty(q.shape, q.dtype, q.device);
  Tensor lse = Tensor::empty({c.B, c.H, c.T}, q.dtype, q.device);
  int64_t st[12];
  const Tensor* ops[4] = {&qv, &kv, &vv, &out};
  for (int i = 0; i < 4; ++i) strides_of(st + 3 * i, *ops[i]);
  window_forward(c, fp(qv), fp(kv), fp(vv), fp(out), fp(lse), st);
  if (!q.requires_grad && !k.requires_grad && !v.requires_grad) return out;
  auto fn = std::make_shared<WindowAttentionFunction>();
  fn->record_input(q);
  fn->record_input(k);
  fn->record_input(v);
  fn->q = qv;
  fn->k = kv;
  fn->v = vv;
  fn->saved_o = out;
  fn->saved_lse = lse;
  fn->dims = c;
  out.requires_grad = true;
  out.grad_fn = fn;
  return out;
}

Tensor window_attention_qkv(const Tensor& qkv, int64_t n_heads, int64_t n_kv_heads, int64_t window, int64_t sinks) {
  if (qkv.dtype != DType::Fp32) throw std::invalid_argument("window_attention: only Fp32 supported");
  if (qkv.shape.size() < 2) throw std::invalid_argument("window_attention: need [..., T, (H + 2 * Hkv) * d]");
  if (n_heads <= 0 || n_kv_heads <= 0 || qkv.shape.back() % (n_heads + 2 * n_kv_heads) != 0) {
    throw std::invalid_argument("window_attention: last dim must be (n_heads + 2 * n_kv_heads) * d_head");
  }
  WindowDims c{1, n_heads, n_kv_heads, qkv.shape[qkv.shape.size() - 2], qkv.shape.back() / (n_heads + 2 * n_kv_heads),
               window, sinks};
  check_heads(c);
  check_window(window, sinks, "window_attention");
  if (qkv.device == Device::CPU) throw_cpu_compute("window_attention");
  Tensor x = as_contig(qkv);
  for (size_t i = 0; i + 2 < x.shape.size(); ++i) c.B *= x.shape[i];
  std::vector<int64_t> shape(x.shape);
  shape.back() = c.H * c.d;
  Tensor out = Tensor::empty(shape, x.dtype, x.device);
  Tensor lse = Tensor::empty({c.B, c.H, c.T}, x.dtype, x.device);
  int64_t st[12];
  WindowQKVFunction::packed_strides(c, st, 4);
  if (x.numel() > 0) {
    const float* p = fp(x);
    window_forward(c, p, p + c.H * c.d, p + (c.H + c.Hkv) * c.d, fp(out), fp(lse), st);
  }
  if (!qkv.requires_grad) return out;
  auto fn = std::make_shared<WindowQKVFunction>();
  fn->record_input(qkv);
  fn->qkv = x;
  fn->saved_o = out;
  fn->saved_lse = lse;
  fn->dims = c;
  out.requires_grad = true;
  out.grad_fn = fn;
  return out;
}

// ------------------------------------------------------------------------ cache

KVCache::KVCache(int64_t layers, int64_t sequences, int64_t kv_heads, int64_t d_head, int64_t max_tokens, int64_t page,
                 int64_t pages, int64_t window, int64_t sinks)
    : B_(sequences), Hkv_(kv_heads), d_(d_head), P_(page), window_(window), sinks_(sinks) {
  const int64_t most = int64_t(1) << 30;
  if (layers < 1 || sequences < 1 || kv_heads < 1) {
    throw std::invalid_argument("KVCache: layers, sequences and kv_heads must be positive");
  }
  if (d_head < 1 || d_head > 128) throw std::invalid_argument("KVCache: d_head must be in [1, 128]");
  if (page != 32 && page != 64 && page != 128) throw std::invalid_argument("KVCache: page must be 32, 64 or 128");
  if (max_tokens < 1 || max_tokens > most - page) throw std::invalid_argument("KVCache: max_tokens must be in [1, 2^30 - page]");
  if (pages < 0 || pages > most) throw std::invalid_argument("KVCache: pages must be in [0, 2^30]");
  if (window < 0 || sinks < 0) throw std::invalid_argument("KVCache: window and sinks must not be negative");
  if (kv_heads > (1 << 16) || sequences > (1 << 22) || sequences * kv_heads > (1 << 22)) {
    throw std::invalid_argument("KVCache: sequences * kv_heads must be at most 2^22, kv_heads 2^16");
  }
  width_ = (max_tokens + page - 1) / page;
  n_pages_ = pages > 0 ? pages : sequences * width_;
  page_bytes_ = aar_kv_cache_page_bytes(kv_heads, page, d_head);
  for (int64_t i = 0; i < layers; ++i) {
    pools_.push_back({std::make_shared<Storage>(n_pages_ * page_bytes_, device_allocator()),
                      std::make_shared<Storage>(n_pages_ * kv_heads * 2 * sizeof(float), device_allocator()),
                      std::make_shared<Storage>(sequences * kv_heads * 2 * page * d_head * sizeof(float), device_allocator())});
  }
  state_.assign(layers, kAppended);
  table_.assign(sequences * width_, -1);
  lens_.assign(sequences, 0);
  new_.assign(sequences, 0);
  refs_.assign(n_pages_, 0);
  for (int64_t i = n_pages_; i-- > 0;) free_.push_back(i);
  table_dev_ = Tensor::empty({B_, width_}, DType::Int64, Device::CUDA);
  lens_dev_ = Tensor::empty({B_}, DType::Int64, Device::CUDA);
  new_dev_ = Tensor::empty({B_}, DType::Int64, Device::CUDA);
  upload();
}

size_t KVCache::nbytes() const {
  size_t n = 0;
  for (const Pool& p : pools_) n += p.pages->nbytes() + p.scales->nbytes() + p.open->nbytes();
  return n;
}

// In stream order: what is enqueued already reads the numbers before.
void KVCache::upload() {
  copy_bytes(table_dev_.data(), Device::CUDA, table_.data(), Device::CPU, table_.size() * sizeof(int64_t));
  copy_bytes(lens_dev_.data(), Device::CUDA, lens_.data(), Device::CPU, lens_.size() * sizeof(int64_t));
  copy_bytes(new_dev_.data(), Device::CUDA, new_.data(), Device::CPU, new_.size() * sizeof(int64_t));
}

void KVCache::drop(int64_t page) {
  if (page < 0 || --refs_[page] > 0) return;
  free_.insert(std::upper_bound(free_.begin(), free_.end(), page, std::greater<int64_t>()), page);
}

void KVCache::clear(int64_t sequence) {
  for (int64_t at = 0; at < width_; ++at) {
    drop(entry(sequence, at));
    entry(sequence, at) = -1;
  }
  lens_[sequence] = new_[sequence] = 0;
  if (std::count(lens_.begin(), lens_.end(), 0) == B_) std::fill(state_.begin(), state_.end(), kAppended);
}

void KVCache::check_sequence(int64_t sequence, const char* op) const {
  if (sequence < 0 || sequence >= B_) throw std::out_of_range(std::string("KVCache.") + op + ": no such sequence");
}

void KVCache::extend(const std::vector<int64_t>& counts) {
  std::lock_guard<std::mutex> lock(mu_);
  if (static_cast<int64_t>(counts.size()) != B_) throw std::invalid_argument("KVCache.extend: one count per sequence");
  int64_t most = 0, need = 0, returned = 0;
  auto pages = [&](int64_t tokens) { return (tokens + P_ - 1) / P_; };
  // the pages [first, last) that neither this step's first token nor a later one sees
  auto first_left = [&](int64_t b) { return pages(std::min(sinks_, lens_[b])); };
  auto last_left = [&](int64_t b) { return window_ > 0 ? std::max<int64_t>(0, lens_[b] - window_ + 1) / P_ : 0; };
  for (int64_t b = 0; b < B_; ++b) {
    if (counts[b] < 0 || counts[b] > width_ * P_ - lens_[b]) {
      throw std::invalid_argument("KVCache.extend: a sequence would pass max_tokens");
    }
    most = std::max(most, counts[b]);
    need += pages(lens_[b] + counts[b]) - pages(lens_[b]);
    for (int64_t at = first_left(b); at < last_left(b); ++at) {
      const int64_t page = entry(b, at);
      if (page >= 0 && refs_[page] == 1) ++returned;
    }
  }
  if (need > free_pages() + returned) throw std::runtime_error("KVCache.extend: out of pages");
  T_ = most;
  for (int64_t b = 0; b < B_; ++b) {
    for (int64_t at = first_left(b); at < last_left(b); ++at) {
      drop(entry(b, at));
      entry(b, at) = -1;
    }
  }
  for (int64_t b = 0; b < B_; ++b) {
    for (int64_t at = pages(lens_[b]); at < pages(lens_[b] + counts[b]); ++at) {
      entry(b, at) = free_.back();
      refs_[free_.back()] = 1;
      free_.pop_back();
    }
    lens_[b] += counts[b];
    new_[b] = counts[b];
  }
  if (T_ > 0) {
    for (State& s : state_) s = s == kAppended ? kOpen : kMissed;
  }
  upload();
}

const KVCache::Pool& KVCache::pool(int64_t layer) const {
  if (layer < 0 || layer >= layers()) throw std::out_of_range("KVCache: no such layer");
  return pools_[layer];
}

aar_kv_cache KVCache::view(int64_t layer) const {
  const Pool& p = pool(layer);
  return {static_cast<uint8_t*>(p.pages->data()), static_cast<float*>(p.scales->data()),
          static_cast<float*>(p.open->data()), ip(table_dev_), B_, width_, n_pages_, Hkv_, P_, d_};
}

void KVCache::check_rows(const Tensor& t, int64_t heads, const char* op) const {
  const std::string name = std::string("KVCache.") + op;
  if (t.dtype != DType::Fp32) throw std::invalid_argument(name + ": only Fp32 supported");
  if (t.shape.size() != 4 || t.shape[0] != B_ || t.shape[2] != T_ || t.shape[3] != d_ ||
      (heads ? t.shape[1] != heads : t.shape[1] <= 0 || t.shape[1] % Hkv_ != 0)) {
    throw std::invalid_argument(name + ": need [sequences, heads, T, d_head] of the last extend");
  }
  if (t.device == Device::CPU) throw_cpu_compute(name.c_str());
}

void KVCache::check_whole(int64_t layer, const char* op) const {
  if (state_[layer] == kMissed) throw std::runtime_error(std::string("KVCache.") + op + ": the layer has missed tokens");
}

void KVCache::append(int64_t layer, const Tensor& k, const Tensor& v) {
  std::lock_guard<std::mutex> lock(mu_);
  const aar_kv_cache c = view(layer);
  check_rows(k, Hkv_, "append");
  check_rows(v, Hkv_, "append");
  check_whole(layer, "append");
  // twice, a page that the step has filled would take its first rows from the next page's
  if (T_ > 0 && state_[layer] == kAppended) throw std::runtime_error("KVCache.append: the layer has this step's tokens");
  Tensor kv = head_view(k), vv = head_view(v);
  int64_t st[6];
  strides_of(st, kv);
  strides_of(st + 3, vv);
  check_status(aar_kv_cache_append_f32(&c, fp(kv), fp(vv), st, ip(lens_dev_), ip(new_dev_), T_,
                                       device_error_word(kErrCachePage), current_stream()),
               "KVCache.append");
  state_[layer] = kAppended;
}

Tensor KVCache::attend(int64_t layer, const Tensor& q) {
  std::lock_guard<std::mutex> lock(mu_);
  const aar_kv_cache c = view(layer);
  check_rows(q, 0, "attend");
  check_whole(layer, "attend");
  if (state_[layer] == kOpen) throw std::runtime_error("KVCache.attend: append the layer's keys and values first");
  const int64_t H = q.shape[1], window = window_ > 0 ? window_ : int64_t(1) << 30;
  Tensor qv = head_view(q);
  // rows of all heads beside each other, as the next projection reads them
  Tensor rows = Tensor::empty({B_, T_, H, d_}, q.dtype, q.device);
  Tensor out = make_view(rows, {B_, H, T_, d_}, {T_ * H * d_, d_, H * d_, 1}, 0);
  int64_t st[6];
  strides_of(st, qv);
  strides_of(st + 3, out);
  Workspace ws(aar_kv_cache_attn_workspace_bytes(&c, H, T_, window, sinks_));
  check_status(aar_kv_cache_attn_f32(&c, fp(qv), fp(out), st, ip(lens_dev_), ip(new_dev_), H, T_, window, sinks_,
                                     1.0f / std::sqrt(static_cast<float>(d_)), ws.data(), ws.bytes(),
                                     device_error_word(kErrCachePage), current_stream()),
               "KVCache.attend");
  return out;
}

Tensor KVCache::positions() const {
  std::lock_guard<std::mutex> lock(mu_);
  Tensor host = Tensor::empty({B_, T_}, DType::Int64, Device::CPU);
  int64_t* p = static_cast<int64_t*>(host.data());
  for (int64_t b = 0; b < B_; ++b)
    for (int64_t t = 0; t < T_; ++t) p[b * T_ + t] = lens_[b] - new_[b] + t;
  return host.to(Device::CUDA);
}

std::pair<Tensor, Tensor> KVCache::read(int64_t layer, int64_t first, int64_t n) {
  std::lock_guard<std::mutex> lock(mu_);
  const aar_kv_cache c = view(layer);
  check_whole(layer, "read");
  if (state_[layer] == kOpen) throw std::runtime_error("KVCache.read: append the layer's keys and values first");
  if (first < 0 || n < 0 || n > width_ * P_) throw std::invalid_argument("KVCache.read: need first >= 0, 0 <= n <= max_tokens");
  Tensor from = Tensor::empty({B_}, DType::Int64, Device::CPU);
  std::fill_n(static_cast<int64_t*>(from.data()), B_, first);
  from = from.to(Device::CUDA);
  Tensor k = Tensor::empty({B_, Hkv_, n, d_}, DType::Fp32, Device::CUDA);
  Tensor v = Tensor::empty({B_, Hkv_, n, d_}, DType::Fp32, Device::CUDA);
  int64_t st[6];
  strides_of(st, k);
  strides_of(st + 3, v);
  if (n > 0) {
    // pages that the window has left have no id: zeros, and no error
    check_status(aar_kv_cache_read_f32(&c, ip(from), ip(lens_dev_), fp(k), fp(v), st, n, nullptr, current_stream()),
                 "KVCache.read");
  }
  return {k, v};
}

void KVCache::fork(int64_t src, int64_t dst) {
  std::lock_guard<std::mutex> lock(mu_);
  check_sequence(src, "fork");
  check_sequence(dst, "fork");
  if (src == dst) return;
  if (new_[src] > 0 && std::count(state_.begin(), state_.end(), kOpen) > 0) {
    throw std::runtime_error("KVCache.fork: a layer has not appended this step's tokens");
  }
  const int64_t full = lens_[src] / P_, rest = lens_[src] % P_;
  int64_t returned = 0;  // pages that dst holds alone
  for (int64_t at = 0; at < width_; ++at) {
    const int64_t page = entry(dst, at);
    if (page >= 0 && refs_[page] == 1) ++returned;
  }
  if (rest > 0 && free_pages() + returned == 0) throw std::runtime_error("KVCache.fork: out of pages");
  clear(dst);
  for (int64_t at = 0; at < full; ++at) {
    entry(dst, at) = entry(src, at);
    if (entry(src, at) >= 0) ++refs_[entry(src, at)];
  }
  if (rest > 0) {  // a page that is not full has rows to come: a copy of it, and of its open rows
    const int64_t from = entry(src, full), to = free_.back();
    free_.pop_back();
    refs_[to] = 1;
    entry(dst, full) = to;
    auto copy = [](Storage& s, int64_t to, int64_t from, size_t bytes) {
      char* p = static_cast<char*>(s.data());
      copy_bytes(p + to * bytes, Device::CUDA, p + from * bytes, Device::CUDA, bytes);
    };
    for (const Pool& p : pools_) {
      copy(*p.pages, to, from, page_bytes_);
      copy(*p.scales, to, from, Hkv_ * 2 * sizeof(float));
      copy(*p.open, dst, src, Hkv_ * 2 * P_ * d_ * sizeof(float));
    }
  }
  lens_[dst] = lens_[src];
  new_[dst] = 0;
  upload();
}

void KVCache::free(int64_t sequence) {
  std::lock_guard<std::mutex> lock(mu_);
  check_sequence(sequence, "free");
  clear(sequence);
  upload();
}

}  // namespace aar
