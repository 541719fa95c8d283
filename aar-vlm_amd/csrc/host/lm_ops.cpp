// Operators of a decoder that reads an encoder's states and learns from a larger
// teacher: cross attention, per-head norms of queries and keys with the position
// rotation, the scaled embedding with its gradient by sorted tokens, and
// distillation from a teacher's top logits.  The reference has no counterparts;
// checks, messages and autograd Functions follow those of its neighbouring ops
// (flash_attention, layernorm, embedding, cross_entropy).  Device work runs in
// csrc/hip/{cross_attn,rotary,embed_sorted,distill}.hip.
#include <cmath>

#include "aar_hip.h"
#include "ops.hpp"

namespace aar {

namespace {

const float* fp(const Tensor& t) { return static_cast<const float*>(t.data()); }
float* fp(Tensor& t) { return static_cast<float*>(t.data()); }
const int64_t* ip(const Tensor& t) { return static_cast<const int64_t*>(t.data()); }

Tensor as_contig(const Tensor& t) { return t.is_contiguous() ? t : contiguous(t); }
int64_t n_of(const Tensor& t) { return static_cast<int64_t>(t.numel()); }

template <class Fn>
Tensor attach(std::shared_ptr<Fn> fn, Tensor out) {
  out.requires_grad = true;
  out.grad_fn = std::move(fn);
  return out;
}

// ------------------------------------------------------------ cross attention

// The dims and element strides of one call: q-shaped and k-shaped operands as
// (sb, sh, st).
struct CrossDims {
  int64_t B = 0, H = 0, Hkv = 0, Tq = 0, Tk = 0, d = 0;
};

void put3(int64_t* dst, int64_t sb, int64_t sh, int64_t st) {
  dst[0] = sb;
  dst[1] = sh;
  dst[2] = st;
}

void check_lens(const std::shared_ptr<Tensor>& lens, int64_t B, Device device, const char* op) {
  if (!lens) return;
  const std::string name(op);
  if (lens->dtype != DType::Int64) throw std::invalid_argument(name + ": kv_lens must be Int64");
  if (lens->shape.size() != 1 || lens->shape[0] != B) {
    throw std::invalid_argument(name + ": kv_lens must be 1D, one length per batch");
  }
  if (lens->device != device) throw std::invalid_argument(name + ": device mismatch");
}

void cross_forward(const CrossDims& c, const float* q, const float* k, const float* v, const int64_t* lens, float* o,
                   float* lse, const int64_t* st, const char* op) {
  const float s = 1.0f / std::sqrt(static_cast<float>(c.d));
  Workspace ws(aar_cross_attn_fwd_workspace_bytes(c.B, c.H, c.Hkv, c.Tq, c.Tk, c.d));
  check_status(aar_cross_attn_fwd_f32(q, k, v, lens, o, lse, c.B, c.H, c.Hkv, c.Tq, c.Tk, c.d, st, s, ws.data(),
                                      ws.bytes(), current_stream()),
               op);
}

void cross_backward(const CrossDims& c, const float* q, const float* k, const float* v, const int64_t* lens,
                    const float* o, const float* lse, const float* go, float* dq, float* dk, float* dv,
                    const int64_t* st, const char* op) {
  const float s = 1.0f / std::sqrt(static_cast<float>(c.d));
  Workspace ws(aar_cross_attn_bwd_workspace_bytes(c.B, c.H, c.Hkv, c.Tq, c.Tk, c.d));
  check_status(aar_cross_attn_bwd_f32(q, k, v, lens, o, lse, go, dq, dk, dv, c.B, c.H, c.Hkv, c.Tq, c.Tk, c.d, st, s,
                                      ws.data(), ws.bytes(), current_stream()),
               op);
}

// A [B, H, T, d] operand the kernels read in place: any strides with the head
// dim contiguous, else a dense copy.
Tensor head_view(const Tensor& t) { return t.strides[3] == 1 || t.shape[3] == 1 ? t : contiguous(t); }
void strides_of(int64_t* dst, const Tensor& t) { put3(dst, t.strides[0], t.strides[1], t.strides[2]); }

class CrossAttentionFunction : public Function {
 public:
  Tensor q, k, v, saved_o, saved_lse;
  std::shared_ptr<Tensor> lens;
  CrossDims dims;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor go = head_view(g);
    Tensor dq = Tensor::empty(q.shape, q.dtype, q.device);
    Tensor dk = Tensor::empty(k.shape, k.dtype, k.device);
    Tensor dv = Tensor::empty(v.shape, v.dtype, v.device);
    int64_t st[24];
    const Tensor* ops[8] = {&q, &k, &v, &saved_o, &go, &dq, &dk, &dv};
    for (int i = 0; i < 8; ++i) strides_of(st + 3 * i, *ops[i]);
    cross_backward(dims, fp(q), fp(k), fp(v), lens ? ip(*lens) : nullptr, fp(saved_o), fp(saved_lse), fp(go), fp(dq),
                   fp(dk), fp(dv), st, "cross_attention backward");
    return {dq, dk, dv};
  }
  const char* name() const override { return "CrossAttentionFunction"; }
};

// q [B, Tq, H*d], kv [B, Tk, 2*Hkv*d] (keys, then values) -> [B, Tq, H*d].
class CrossPackedFunction : public Function {
 public:
  Tensor q, kv, saved_o, saved_lse;
  std::shared_ptr<Tensor> lens;
  CrossDims dims;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor go = as_contig(g);
    Tensor dq = Tensor::empty(q.shape, q.dtype, q.device);
    Tensor dkv = Tensor::empty(kv.shape, kv.dtype, kv.device);
    int64_t st[24];
    packed_strides(dims, st, true);
    const int64_t half = dims.Hkv * dims.d;
    const float* x = fp(kv);
    float* y = fp(dkv);
    cross_backward(dims, fp(q), x, x ? x + half : x, lens ? ip(*lens) : nullptr, fp(saved_o), fp(saved_lse), fp(go),
                   fp(dq), y, y ? y + half : y, st, "cross_attention backward");
    return {dq, dkv};
  }
  const char* name() const override { return "CrossPackedFunction"; }

  static void packed_strides(const CrossDims& c, int64_t* st, bool backward) {
    const int64_t q = c.H * c.d, kv = 2 * c.Hkv * c.d;
    auto q3 = [&](int i) { put3(st + 3 * i, c.Tq * q, c.d, q); };
    auto kv3 = [&](int i) { put3(st + 3 * i, c.Tk * kv, c.d, kv); };
    q3(0);
    kv3(1);
    kv3(2);
    q3(3);
    if (!backward) return;
    q3(4);
    q3(5);
    kv3(6);
    kv3(7);
  }
};

// -------------------------------------------------------------- norm + rotation

class QkNormRopeFunction : public Function {
 public:
  Tensor x, wq, wk, positions;
  int64_t hq = 0, hk = 0, d = 0, rotary = 0;
  double base = 0;
  float eps = 0;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor gc = as_contig(g);
    Tensor dx = Tensor::empty(x.shape, x.dtype, x.device);
    Tensor dwq = Tensor::empty({d}, x.dtype, x.device), dwk = Tensor::empty({d}, x.dtype, x.device);
    const int64_t row = (hq + hk) * d, rows = n_of(x) / row;
    Workspace ws(aar_qk_norm_rope_bwd_workspace_bytes(rows, hq, hk, d));
    check_status(aar_qk_norm_rope_bwd_f32(fp(gc), row, fp(x), row, fp(wq), fp(wk), rotary ? ip(positions) : nullptr,
                                          rotary ? n_of(positions) : 0, fp(dx), row, fp(dwq), fp(dwk), rows, hq, hk, d,
                                          rotary, base, eps, ws.data(), ws.bytes(), current_stream()),
                 "qk_norm_rope backward");
    return {dx, dwq, dwk};
  }
  const char* name() const override { return "QkNormRopeFunction"; }
};

// ------------------------------------------------------------------- embedding

class EmbeddingScaledFunction : public Function {
 public:
  Tensor saved_ids;
  int64_t vocab = 0;
  float scale = 1.0f;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor gc = as_contig(g);
    return {embedding_sorted_grad(gc, saved_ids, vocab, scale)};
  }
  const char* name() const override { return "EmbeddingScaledFunction"; }
};

// ----------------------------------------------------------------- distillation

class DistillFunction : public Function {
 public:
  Tensor logits, t_logits, t_ids, stats;
  float temperature = 1.0f;
  std::vector<Tensor> backward(const Tensor& g) override {
    Tensor gc = as_contig(g);
    Tensor dz = Tensor::empty(logits.shape, logits.dtype, logits.device);
    check_status(aar_distill_bwd_f32(fp(gc), fp(logits), fp(t_logits), ip(t_ids), fp(stats), fp(dz), logits.shape[0],
                                     logits.shape[1], t_ids.shape[1], temperature, current_stream()),
                 "distill_loss backward");
    return {dz};
  }
  const char* name() const override { return "DistillFunction"; }
};

}  // namespace

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::shared_ptr<Tensor>& kv_lens) {
  const char* op = "cross_attention";
  if (q.dtype != DType::Fp32 || k.dtype != DType::Fp32 || v.dtype != DType::Fp32) {
    throw std::invalid_argument("cross_attention: only Fp32 supported");
  }
  if (q.device != k.device || q.device != v.device) throw std::invalid_argument("cross_attention: device mismatch");
  if (q.shape.size() != 4 || k.shape.size() != 4 || v.shape.size() != 4) {
    throw std::invalid_argument("cross_attention: q, k, v must be 4D [B, H, T, d]");
  }
  if (k.shape != v.shape) throw std::invalid_argument("cross_attention: k and v must share shape");
  CrossDims c{q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3]};
  if (k.shape[0] != c.B || k.shape[3] != c.d) {
    throw std::invalid_argument("cross_attention: q and k must share batch and head dim");
  }
  if (c.H <= 0 || c.Hkv <= 0 || c.H % c.Hkv != 0) {
    throw std::invalid_argument("cross_attention: query heads must be a multiple of key/value heads");
  }
  if (c.d <= 0 || c.d > 128) throw std::invalid_argument("cross_attention: d_head must be in [1, 128]");
  check_lens(kv_lens, c.B, q.device, op);
  if (q.device == Device::CPU) throw_cpu_compute(op);
  Tensor qv = head_view(q), kv = head_view(k), vv = head_view(v);
  std::shared_ptr<Tensor> lens = kv_lens ? std::make_shared<Tensor>(as_contig(*kv_lens)) : nullptr;
  Tensor out = Tensor::empty(q.shape, q.dtype, q.device);
  Tensor lse = Tensor::empty({c.B, c.H, c.Tq}, q.dtype, q.device);
  int64_t st[12];
  strides_of(st, qv);
  strides_of(st + 3, kv);
  strides_of(st + 6, vv);
  strides_of(st + 9, out);
  cross_forward(c, fp(qv), fp(kv), fp(vv), lens ? ip(*lens) : nullptr, fp(out), fp(lse), st, op);
  if (!q.requires_grad && !k.requires_grad && !v.requires_grad) return out;
  auto fn = std::make_shared<CrossAttentionFunction>();
  fn->record_input(q);
  fn->record_input(k);
  fn->record_input(v);
  fn->q = qv;
  fn->k = kv;
  fn->v = vv;
  fn->saved_o = out;
  fn->saved_lse = lse;
  fn->lens = lens;
  fn->dims = c;
  return attach(fn, out);
}

Tensor cross_attention_packed(const Tensor& q, const Tensor& kv, int64_t n_heads, int64_t n_kv_heads,
                              const std::shared_ptr<Tensor>& kv_lens) {
  const char* op = "cross_attention";
  if (q.dtype != DType::Fp32 || kv.dtype != DType::Fp32) {
    throw std::invalid_argument("cross_attention: only Fp32 supported");
  }
  if (q.device != kv.device) throw std::invalid_argument("cross_attention: device mismatch");
  if (q.shape.size() != 3 || kv.shape.size() != 3 || q.shape[0] != kv.shape[0]) {
    throw std::invalid_argument("cross_attention: need q [B, Tq, H*d] and kv [B, Tk, 2*Hkv*d]");
  }
  if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) {
    throw std::invalid_argument("cross_attention: query heads must be a multiple of key/value heads");
  }
  if (q.shape[2] % n_heads != 0 || kv.shape[2] != 2 * n_kv_heads * (q.shape[2] / n_heads)) {
    throw std::invalid_argument("cross_attention: last dims must be n_heads * d and 2 * n_kv_heads * d");
  }
  CrossDims c{q.shape[0], n_heads, n_kv_heads, q.shape[1], kv.shape[1], q.shape[2] / n_heads};
  if (c.d <= 0 || c.d > 128) throw std::invalid_argument("cross_attention: d_head must be in [1, 128]");
  check_lens(kv_lens, c.B, q.device, op);
  if (q.device == Device::CPU) throw_cpu_compute(op);
  Tensor qc = as_contig(q), kvc = as_contig(kv);
  std::shared_ptr<Tensor> lens = kv_lens ? std::make_shared<Tensor>(as_contig(*kv_lens)) : nullptr;
  Tensor out = Tensor::empty(qc.shape, q.dtype, q.device);
  Tensor lse = Tensor::empty({c.B, c.H, c.Tq}, q.dtype, q.device);
  int64_t st[12];
  CrossPackedFunction::packed_strides(c, st, false);
  const float* x = fp(kvc);
  cross_forward(c, fp(qc), x, x ? x + c.Hkv * c.d : x, lens ? ip(*lens) : nullptr, fp(out), fp(lse), st, op);
  if (!qc.requires_grad && !kvc.requires_grad) return out;
  auto fn = std::make_shared<CrossPackedFunction>();
  fn->record_input(qc);
  fn->record_input(kvc);
  fn->q = qc;
  fn->kv = kvc;
  fn->saved_o = out;
  fn->saved_lse = lse;
  fn->lens = lens;
  fn->dims = c;
  return attach(fn, out);
}

int64_t check_rope(const Tensor& x, const Tensor& q_weight, const Tensor& k_weight,
                   const std::shared_ptr<Tensor>& positions, int64_t heads, int64_t& rotary_dim, double base, float eps,
                   const char* op) {
  const std::string name(op);
  if (x.dtype != DType::Fp32 || q_weight.dtype != DType::Fp32 || k_weight.dtype != DType::Fp32) {
    throw std::invalid_argument(name + ": only Fp32 supported");
  }
  if (x.device != q_weight.device || x.device != k_weight.device) {
    throw std::invalid_argument(name + ": device mismatch");
  }
  if (x.shape.size() < 2) throw std::invalid_argument(name + ": need [..., T, heads * d_head]");
  if (heads <= 0 || x.shape.back() % heads != 0 || x.shape.back() == 0) {
    throw std::invalid_argument(name + ": last dim must be heads * d_head");
  }
  const int64_t d = x.shape.back() / heads;
  if (d < 2 || d > 256) throw std::invalid_argument(name + ": d_head must be in [2, 256]");
  if (q_weight.shape != std::vector<int64_t>{d} || k_weight.shape != std::vector<int64_t>{d}) {
    throw std::invalid_argument(name + ": weights must be 1D of d_head");
  }
  if (rotary_dim < 0) rotary_dim = d;
  if (rotary_dim > d || rotary_dim % 2 != 0) {
    throw std::invalid_argument(name + ": rotary_dim must be even and at most d_head");
  }
  if (!(base > 0.0) || !std::isfinite(base)) throw std::invalid_argument(name + ": base must be positive");
  if (!(eps >= 0.0f) || !std::isfinite(eps)) throw std::invalid_argument(name + ": eps must not be negative");
  if (rotary_dim > 0) {
    if (!positions) throw std::invalid_argument(name + ": positions are needed for a rotation");
    if (positions->dtype != DType::Int64) throw std::invalid_argument(name + ": positions must be Int64");
    if (positions->device != x.device) throw std::invalid_argument(name + ": device mismatch");
    std::vector<int64_t> rows(x.shape.begin(), x.shape.end() - 1);
    if (positions->shape != rows && positions->shape != std::vector<int64_t>{rows.back()}) {
      throw std::invalid_argument(name + ": positions must be [T] or one per row");
    }
  }
  return d;
}

Tensor qk_norm_rope(const Tensor& x, const Tensor& q_weight, const Tensor& k_weight,
                    const std::shared_ptr<Tensor>& positions, int64_t n_q_heads, int64_t n_k_heads, int64_t rotary_dim,
                    double base, float eps) {
  const char* op = "qk_norm_rope";
  if (n_q_heads < 0 || n_k_heads < 0) throw std::invalid_argument("qk_norm_rope: negative head count");
  const int64_t d = check_rope(x, q_weight, k_weight, positions, n_q_heads + n_k_heads, rotary_dim, base, eps, op);
  if (x.device == Device::CPU) throw_cpu_compute(op);
  Tensor xc = as_contig(x), wq = as_contig(q_weight), wk = as_contig(k_weight);
  Tensor pos;
  if (rotary_dim > 0) pos = as_contig(*positions);
  Tensor out = Tensor::empty(xc.shape, xc.dtype, xc.device);
  const int64_t row = (n_q_heads + n_k_heads) * d, rows = n_of(xc) / row;
  check_status(aar_qk_norm_rope_fwd_f32(fp(xc), row, fp(wq), fp(wk), rotary_dim ? ip(pos) : nullptr,
                                        rotary_dim ? n_of(pos) : 0, fp(out), row, rows, n_q_heads, n_k_heads, d,
                                        rotary_dim, base, eps, current_stream()),
               op);
  if (!xc.requires_grad && !wq.requires_grad && !wk.requires_grad) return out;
  auto fn = std::make_shared<QkNormRopeFunction>();
  fn->record_input(xc);
  fn->record_input(wq);
  fn->record_input(wk);
  fn->x = xc;
  fn->wq = wq;
  fn->wk = wk;
  fn->positions = pos;
  fn->hq = n_q_heads;
  fn->hk = n_k_heads;
  fn->d = d;
  fn->rotary = rotary_dim;
  fn->base = base;
  fn->eps = eps;
  return attach(fn, out);
}

Tensor embedding_sorted_grad(const Tensor& g, const Tensor& ids, int64_t vocab, float scale) {
  const int64_t D = g.shape.back(), n = n_of(ids);
  Tensor dW = Tensor::empty({vocab, D}, DType::Fp32, Device::CUDA);
  Workspace ws(aar_embedding_sorted_bwd_workspace_bytes(n, vocab, D));
  check_status(aar_embedding_sorted_bwd_f32(fp(g), ip(ids), fp(dW), n, vocab, D, scale, ws.data(), ws.bytes(),
                                            current_stream()),
               "embedding backward");
  return dW;
}

Tensor embedding_scaled(const Tensor& weight, const Tensor& ids, float scale) {
  const char* op = "embedding_scaled";
  if (weight.dtype != DType::Fp32) throw std::invalid_argument("embedding_scaled: weight must be Fp32");
  if (ids.dtype != DType::Int64) throw std::invalid_argument("embedding_scaled: ids must be Int64");
  if (weight.shape.size() != 2) {
    throw std::invalid_argument("embedding_scaled: weight must be 2D (vocab_size, embed_dim)");
  }
  if (weight.device != ids.device) throw std::invalid_argument("embedding_scaled: device mismatch");
  if (weight.device == Device::CPU) throw_cpu_compute(op);
  Tensor wc = as_contig(weight), ic = as_contig(ids);
  const int64_t V = wc.shape[0], D = wc.shape[1];
  std::vector<int64_t> out_shape = ic.shape;
  out_shape.push_back(D);
  Tensor out = Tensor::empty(out_shape, DType::Fp32, Device::CUDA);
  check_status(aar_embedding_scaled_fwd_f32(fp(wc), ip(ic), fp(out), n_of(ic), V, D, scale,
                                            device_error_word(kErrEmbeddingId), current_stream()),
               op);
  if (!wc.requires_grad) return out;
  auto fn = std::make_shared<EmbeddingScaledFunction>();
  fn->record_input(wc);
  fn->saved_ids = ic;
  fn->vocab = V;
  fn->scale = scale;
  return attach(fn, out);
}

Tensor distill_loss(const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_ids, float temperature) {
  const char* op = "distill_loss";
  if (logits.dtype != DType::Fp32 || teacher_logits.dtype != DType::Fp32) {
    throw std::invalid_argument("distill_loss: logits must be Fp32");
  }
  if (teacher_ids.dtype != DType::Int64) throw std::invalid_argument("distill_loss: teacher_ids must be Int64");
  if (logits.shape.size() != 2) throw std::invalid_argument("distill_loss: logits must be 2D (N, V)");
  if (teacher_ids.shape.size() != 2 || teacher_ids.shape[0] != logits.shape[0] ||
      teacher_logits.shape != teacher_ids.shape) {
    throw std::invalid_argument("distill_loss: teacher logits and ids must be 2D (N, K)");
  }
  if (logits.device != teacher_logits.device || logits.device != teacher_ids.device) {
    throw std::invalid_argument("distill_loss: device mismatch");
  }
  const int64_t N = logits.shape[0], V = logits.shape[1], K = teacher_ids.shape[1];
  if (V == 0) throw std::invalid_argument("distill_loss: empty vocabulary");
  if (K < 1 || K > 1024) throw std::invalid_argument("distill_loss: K must be in [1, 1024]");
  if (!(temperature >= 0x1p-61f) || !(temperature <= 0x1p61f)) {
    throw std::invalid_argument("distill_loss: temperature must be positive, in [2^-61, 2^61]");
  }
  if (logits.device == Device::CPU) throw_cpu_compute(op);
  Tensor lc = as_contig(logits), tc = as_contig(teacher_logits), ic = as_contig(teacher_ids);
  Tensor out = Tensor::empty({}, DType::Fp32, Device::CUDA);
  Tensor stats = Tensor::empty({2 * N + 1}, DType::Fp32, Device::CUDA);
  Workspace ws(aar_distill_workspace_bytes(N));
  check_status(aar_distill_fwd_f32(fp(lc), fp(tc), ip(ic), fp(out), fp(stats), N, V, K, temperature,
                                   device_error_word(kErrDistillId), ws.data(), ws.bytes(), current_stream()),
               op);
  if (!lc.requires_grad) return out;
  auto fn = std::make_shared<DistillFunction>();
  fn->record_input(lc);
  fn->logits = lc;
  fn->t_logits = tc;
  fn->t_ids = ic;
  fn->stats = stats;
  fn->temperature = temperature;
  return attach(fn, out);
}

}  // namespace aar
