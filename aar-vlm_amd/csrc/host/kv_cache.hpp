// The key/value cache of a decoder's layers (no counterpart in the reference): pages
// of 8-bit numbers for each layer, one table of pages and one length per sequence for
// all of them.
#pragma once

#include <cstdint>
#include <memory>
#include <mutex>
#include <utility>
#include <vector>

#include "aar_hip.h"
#include "tensor.hpp"

namespace aar {

// Sequences are the rows of a batch.  A step of the model is `extend` (how many tokens
// each sequence gets; pages are taken for them), then for every layer `append` with the
// new tokens' keys and values, once, and `attend` with their queries, as often as wanted;
// what breaks that order throws std::runtime_error and changes nothing.  A layer that has
// missed tokens is not used again until all sequences are empty.  The page numbers are the
// same in all layers.  A full page never changes, so a fork shares its parent's; the
// pages a window has left are given back.
class KVCache {
 public:
  // max_tokens: of a sequence; pages 0: enough for every sequence's max_tokens.
  // window 0: every token stays visible.
  KVCache(int64_t layers, int64_t sequences, int64_t kv_heads, int64_t d_head, int64_t max_tokens, int64_t page,
          int64_t pages, int64_t window, int64_t sinks);

  // counts[b] new tokens of sequence b; none at all leaves the cache as it is.
  // Throws std::runtime_error, nothing changed, where there are too few free pages.
  void extend(const std::vector<int64_t>& counts);
  // The new tokens' keys and values [sequences, kv_heads, T, d], T the largest count
  // (rows from counts[b] on are not read).  Constants: no gradient passes.
  void append(int64_t layer, const Tensor& k, const Tensor& v);
  // Their attention: q [sequences, H, T, d] -> the same shape, rows from counts[b] on 0.
  Tensor attend(int64_t layer, const Tensor& q);
  // Positions of the new tokens, Int64 [sequences, T].
  Tensor positions() const;
  // Tokens [first, first + n) of every sequence as rows (keys, values), [sequences,
  // kv_heads, n, d]; zeros where a sequence holds none.
  std::pair<Tensor, Tensor> read(int64_t layer, int64_t first, int64_t n);

  // Sequence dst, which is emptied first, continues from what src holds: not between src's
  // extend and the last layer's append.
  void fork(int64_t src, int64_t dst);
  // Empties a sequence.
  void free(int64_t sequence);

  const std::vector<int64_t>& lengths() const { return lens_; }
  int64_t free_pages() const { return static_cast<int64_t>(free_.size()); }
  int64_t layers() const { return static_cast<int64_t>(pools_.size()); }
  int64_t window() const { return window_; }
  int64_t sinks() const { return sinks_; }
  size_t nbytes() const;

 private:
  struct Pool {
    std::shared_ptr<Storage> pages, scales, open;
  };
  aar_kv_cache view(int64_t layer) const;
  const Pool& pool(int64_t layer) const;
  int64_t& entry(int64_t sequence, int64_t at) { return table_[sequence * width_ + at]; }
  void check_sequence(int64_t sequence, const char* op) const;
  void check_rows(const Tensor& t, int64_t heads, const char* op) const;
  void check_whole(int64_t layer, const char* op) const;
  void drop(int64_t page);
  void clear(int64_t sequence);
  void upload();

  mutable std::mutex mu_;
  int64_t B_, Hkv_, d_, P_, width_, n_pages_, window_, sinks_, T_ = 0;
  size_t page_bytes_ = 0;
  std::vector<Pool> pools_;
  enum State : char { kMissed, kOpen, kAppended };  // a step's tokens, or some step's: not there; of this step not yet; there
  std::vector<State> state_;  // of each layer
  std::vector<int64_t> table_, lens_, new_, refs_, free_;  // free_: the lowest last
  Tensor table_dev_, lens_dev_, new_dev_;
};

}  // namespace aar
