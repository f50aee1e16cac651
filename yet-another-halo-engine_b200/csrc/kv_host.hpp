// Host side of the cache: the page allocator, the per-sequence block tables, per-layer lengths, validation, and the
// planners that turn a batch of sequences into the work lists the kernels read. No CUDA in this header.
//
// The reference keeps one sequence with an identity page table (engine/model/loom_decoder.hpp:175-179) and validates
// every table entry before upload (engine/model/loom_prefill.hpp:1314-1316); batching, the free list and the split-K
// planner are this library's own. Errors are reported as codes plus a message, never thrown across the C ABI, and
// every check runs before anything is queued (engine/model/loom_decoder.hpp:186-209).
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <string>
#include <utility>
#include <vector>

#include "../../include/yahkv.h"
#include "kernels.cuh"

namespace yahkv {

struct HostError {
  int code = YAHKV_OK;
  std::string message;
};

// The layers that a plan has served since it was made. The layers of a decode step have equal lengths and share one plan; a
// layer that comes again is another step and plans again, also where no length has changed since. (A yahkv_batch is the form
// that keeps its work lists from step to step.)
struct StepLayers {
  std::vector<char> served;
  bool Comes(int layer) const { return layer >= 0 && static_cast<std::size_t>(layer) < served.size() && served[static_cast<std::size_t>(layer)] != 0; }
  void Serve(int layer, int n_layers, bool new_plan) {
    if (new_plan || served.empty()) served.assign(static_cast<std::size_t>(n_layers), 0);
    served[static_cast<std::size_t>(layer)] = 1;
  }
};

class KvHost {
 public:
  explicit KvHost(const yahkv_config& cfg) : cfg_(cfg) {
    const std::size_t ns = static_cast<std::size_t>(cfg.max_seqs);
    table_.assign(ns * static_cast<std::size_t>(cfg.max_pages_per_seq), 0);
    n_pages_.assign(ns, 0);
    live_.assign(ns, 0);
    len_.assign(ns * static_cast<std::size_t>(cfg.n_layers), 0);
    dirty_lo_.assign(ns, 0);
    dirty_hi_.assign(ns, 0);
    refs_.assign(static_cast<std::size_t>(cfg.num_pages), 0);
    evicted_.assign(ns, 0);
    generation_.assign(ns, 0);
    // LIFO free list: page 0 is handed out first.
    free_pages_.reserve(static_cast<std::size_t>(cfg.num_pages));
    for (int p = cfg.num_pages - 1; p >= 0; --p) free_pages_.push_back(p);
    free_seqs_.reserve(ns);
    for (int s = cfg.max_seqs - 1; s >= 0; --s) free_seqs_.push_back(s);
  }

  static int ValidateConfig(const yahkv_config& c, std::string* why) {
    auto bad = [&](const char* m) {
      *why = m;
      return YAHKV_ERR_INVALID;
    };
    if (c.n_q_heads != kQHeads || c.n_kv_heads != kKvHeads || c.head_dim != kHeadDim)
      return bad("geometry must be 24 query heads, 4 kv heads, head_dim 256");
    if (c.page_tokens != kPageTokens) return bad("page_tokens must be 64");
    if (c.fmt != YAHKV_FMT_Q8_0 && c.fmt != YAHKV_FMT_Q4_0 && c.fmt != YAHKV_FMT_KV8A16 && c.fmt != YAHKV_FMT_KV4A16 &&
        c.fmt != YAHKV_FMT_F16)
      return bad("fmt must be YAHKV_FMT_Q8_0, YAHKV_FMT_Q4_0, YAHKV_FMT_KV8A16, YAHKV_FMT_KV4A16 or YAHKV_FMT_F16");
    if ((c.fmt == YAHKV_FMT_KV8A16 || c.fmt == YAHKV_FMT_KV4A16) && c.kv_head_count != 0 && c.kv_head_count != kKvHeads)
      return bad("YAHKV_FMT_KV8A16 / YAHKV_FMT_KV4A16 contexts hold all four kv heads");
    if (c.n_layers < 1 || c.n_layers > 1024) return bad("n_layers out of range");
    if (c.num_pages < 1) return bad("num_pages must be positive");
    if (c.max_seqs < 1 || c.max_pages_per_seq < 1) return bad("max_seqs and max_pages_per_seq must be positive");
    if (c.max_splits < 0 || c.max_batch_tokens < 0) return bad("max_splits and max_batch_tokens must not be negative");
    static_assert(kCombineMaxUnits == 1024, "the message below names the limit");
    if (c.max_prefill_keys < 0 || 1LL * c.max_prefill_keys * kKvHeads >= (1LL << 31))
      return bad("max_prefill_keys out of range");
    if (c.max_splits > kCombineMaxUnits) return bad("max_splits must not exceed 1024 (the combine kernel's unit limit)");
    if (c.kv_head_begin < 0 || c.kv_head_count < 0 || c.kv_head_begin + c.kv_head_count > kKvHeads ||
        (c.kv_head_count == 0 && c.kv_head_begin != 0))
      return bad("kv_head_begin / kv_head_count must describe a range inside the 4 kv heads (count 0 = all)");
    // Token rows of all layers are addressed by a signed 32-bit tensor-map coordinate.
    const long long rows = 1LL * c.n_layers * c.num_pages * kKvHeads * kPageTokens;
    if (rows >= (1LL << 31)) return bad("n_layers * num_pages too large for the pool's row index");
    return YAHKV_OK;
  }

  const yahkv_config& cfg() const { return cfg_; }
  int kv_head_begin() const { return cfg_.kv_head_begin; }
  int kv_head_count() const { return cfg_.kv_head_count == 0 ? kKvHeads : cfg_.kv_head_count; }
  int pages_free() const { return static_cast<int>(free_pages_.size()); }
  bool live(int seq) const { return seq >= 0 && seq < cfg_.max_seqs && live_[static_cast<std::size_t>(seq)] != 0; }
  // Tells a sequence from the ones that had its id before.
  std::uint32_t generation(int seq) const { return generation_[static_cast<std::size_t>(seq)]; }
  int n_pages(int seq) const { return n_pages_[static_cast<std::size_t>(seq)]; }
  std::int64_t PagesHold(int seq) const { return static_cast<std::int64_t>(n_pages(seq)) * kPageTokens; }   // tokens
  const std::int32_t* table_row(int seq) const {
    return table_.data() + static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.max_pages_per_seq);
  }
  std::int64_t len(int seq, int layer) const {
    return len_[static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.n_layers) + static_cast<std::size_t>(layer)];
  }

  HostError SeqCreate(std::int32_t* seq) {
    if (free_seqs_.empty()) return {YAHKV_ERR_CAPACITY, "no free sequence slot (max_seqs reached)"};
    const int s = free_seqs_.back();
    free_seqs_.pop_back();
    live_[static_cast<std::size_t>(s)] = 1;
    generation_[static_cast<std::size_t>(s)] += 1;
    n_pages_[static_cast<std::size_t>(s)] = 0;
    evicted_[static_cast<std::size_t>(s)] = 0;
    SetLenAll(s, 0);
    *seq = s;
    return {};
  }

  HostError SeqFree(int seq) {
    if (!live(seq)) return {YAHKV_ERR_INVALID, "seq_free: not a live sequence: " + std::to_string(seq)};
    ReleasePages(seq);
    live_[static_cast<std::size_t>(seq)] = 0;
    SetLenAll(seq, 0);
    free_seqs_.push_back(seq);
    return {};
  }

  HostError SeqReserve(int seq, std::int64_t n_tokens) {
    if (!live(seq)) return {YAHKV_ERR_INVALID, "seq_reserve: not a live sequence: " + std::to_string(seq)};
    if (n_tokens < 0) return {YAHKV_ERR_INVALID, "seq_reserve: negative token count"};
    const std::int64_t need = (n_tokens + kPageTokens - 1) / kPageTokens;
    const int have = n_pages_[static_cast<std::size_t>(seq)];
    if (need <= have) return {};
    if (need > cfg_.max_pages_per_seq)
      return {YAHKV_ERR_CAPACITY, "seq_reserve: " + std::to_string(n_tokens) + " tokens need more than max_pages_per_seq pages"};
    if (need - have > static_cast<std::int64_t>(free_pages_.size()))
      return {YAHKV_ERR_NO_PAGES, "seq_reserve: page pool exhausted (" + std::to_string(free_pages_.size()) +
                                      " free, " + std::to_string(need - have) + " needed)"};
    std::int32_t* row = mutable_row(seq);
    for (int i = have; i < need; ++i) {
      const std::int32_t p = free_pages_.back();
      free_pages_.pop_back();
      refs_[static_cast<std::size_t>(p)] = 1;
      row[i] = p;
    }
    n_pages_[static_cast<std::size_t>(seq)] = static_cast<int>(need);
    MarkDirty(seq, have, static_cast<int>(need));
    return {};
  }

  HostError SeqSetTable(int seq, const std::int32_t* pages, int n) {
    if (!live(seq)) return {YAHKV_ERR_INVALID, "seq_set_table: not a live sequence: " + std::to_string(seq)};
    if (n < 0 || (n > 0 && pages == nullptr)) return {YAHKV_ERR_INVALID, "seq_set_table: bad page list"};
    if (n > cfg_.max_pages_per_seq) return {YAHKV_ERR_CAPACITY, "seq_set_table: more pages than max_pages_per_seq"};
    // Validate everything before changing anything.
    std::vector<std::int32_t> sorted(pages, pages + n);
    std::sort(sorted.begin(), sorted.end());
    std::vector<char> mine(static_cast<std::size_t>(cfg_.num_pages), 0);
    for (int i = 0; i < n_pages(seq); ++i) mine[static_cast<std::size_t>(table_row(seq)[i])] = 1;
    for (int i = 0; i < n; ++i) {
      const std::int32_t p = sorted[static_cast<std::size_t>(i)];
      if (p < 0 || p >= cfg_.num_pages)
        return {YAHKV_ERR_INVALID, "page table entry out of range: " + std::to_string(p)};
      if (i > 0 && sorted[static_cast<std::size_t>(i - 1)] == p)
        return {YAHKV_ERR_INVALID, "page table names page " + std::to_string(p) + " twice"};
      // free, or held by this sequence alone
      if (refs_[static_cast<std::size_t>(p)] > mine[static_cast<std::size_t>(p)])
        return {YAHKV_ERR_INVALID, "page " + std::to_string(p) + " belongs to sequence " + std::to_string(OtherHolder(p, seq))};
    }
    ReleasePages(seq);
    // Take the named pages out of the free list.
    std::vector<char> take(static_cast<std::size_t>(cfg_.num_pages), 0);
    for (int i = 0; i < n; ++i) take[static_cast<std::size_t>(pages[i])] = 1;
    free_pages_.erase(std::remove_if(free_pages_.begin(), free_pages_.end(),
                                     [&](std::int32_t p) { return take[static_cast<std::size_t>(p)] != 0; }),
                      free_pages_.end());
    std::int32_t* row = mutable_row(seq);
    for (int i = 0; i < n; ++i) {
      row[i] = pages[i];
      refs_[static_cast<std::size_t>(pages[i])] = 1;
    }
    n_pages_[static_cast<std::size_t>(seq)] = n;
    MarkDirty(seq, 0, n);
    return {};
  }

  HostError SeqSetLen(int seq, int layer, std::int64_t len) {
    if (!live(seq)) return {YAHKV_ERR_INVALID, "seq_set_len: not a live sequence: " + std::to_string(seq)};
    if (layer < -1 || layer >= cfg_.n_layers) return {YAHKV_ERR_INVALID, "seq_set_len: layer out of range"};
    if (len < 0 || len > static_cast<std::int64_t>(n_pages_[static_cast<std::size_t>(seq)]) * kPageTokens)
      return {YAHKV_ERR_INVALID, "seq_set_len: length beyond the reserved pages"};
    if (layer == -1)
      SetLenAll(seq, len);
    else
      len_ref(seq, layer) = len;
    if (layer == -1 && len == 0) evicted_[static_cast<std::size_t>(seq)] = 0;   // starts over: slots are positions again
    return {};
  }

  HostError CheckFork(int seq, std::int64_t n_tokens) const {
    if (!live(seq)) return {YAHKV_ERR_INVALID, "seq_fork: not a live sequence: " + std::to_string(seq)};
    if (n_tokens < 0) return {YAHKV_ERR_INVALID, "seq_fork: negative token count"};
    for (int l = 0; l < cfg_.n_layers; ++l)
      if (len(seq, l) < n_tokens)
        return {YAHKV_ERR_ORDER, "seq_fork: sequence " + std::to_string(seq) + " holds " + std::to_string(len(seq, l)) +
                                     " tokens in layer " + std::to_string(l) + ", " + std::to_string(n_tokens) + " asked for"};
    if (n_tokens > PagesHold(seq))   // its table was set by hand and the length not yet
      return {YAHKV_ERR_ORDER, "seq_fork: the table of sequence " + std::to_string(seq) + " has fewer pages than " + std::to_string(n_tokens) + " tokens need"};
    return {};
  }
  // A new sequence whose first n_tokens / 64 pages are seq's own (counted references, never written while shared) and
  // whose length is n_tokens in every layer. A prefix that ends inside a page takes a page of its own for the rest:
  // *copy_src / *copy_dst then name the page to copy (-1: nothing to copy). Nothing changes on error.
  HostError SeqFork(int seq, std::int64_t n_tokens, std::int32_t* out, std::int32_t* copy_src, std::int32_t* copy_dst) {
    if (HostError bad = CheckFork(seq, n_tokens); bad.code != YAHKV_OK) return bad;
    const int whole = static_cast<int>(n_tokens / kPageTokens);
    const bool rest = n_tokens % kPageTokens != 0;
    if (rest && free_pages_.empty()) return {YAHKV_ERR_NO_PAGES, "seq_fork: no free page for the prefix's last, partly filled page"};
    std::int32_t s = -1;
    HostError e = SeqCreate(&s);
    if (e.code != YAHKV_OK) return e;
    std::int32_t* row = mutable_row(s);
    const std::int32_t* from = table_row(seq);
    for (int i = 0; i < whole; ++i) {
      row[i] = from[i];
      refs_[static_cast<std::size_t>(from[i])] += 1;
    }
    *copy_src = *copy_dst = -1;
    if (rest) {
      row[whole] = free_pages_.back();
      free_pages_.pop_back();
      refs_[static_cast<std::size_t>(row[whole])] = 1;
      *copy_src = from[whole], *copy_dst = row[whole];
    }
    n_pages_[static_cast<std::size_t>(s)] = whole + (rest ? 1 : 0);
    evicted_[static_cast<std::size_t>(s)] = n_tokens > 0 ? evicted_[static_cast<std::size_t>(seq)] : 0;
    MarkDirty(s, 0, n_pages_[static_cast<std::size_t>(s)]);
    SetLenAll(s, n_tokens);
    *out = s;
    return {};
  }

  // Eviction of every listed sequence longer than n_keep (all layers equally long) down to n_keep slots: the pages it
  // will have. A page it holds alone is kept and overwritten; a page that another sequence holds too at the time of the
  // call is replaced by a free one, also when that other sequence is evicted by the same call and lets go of it.
  // Changes no sequence; CommitEvict with the same lists then moves the tables over. The keys have been moved on the device
  // by then, so it may not fail: what it needs room for is reserved here.
  HostError PlanEvict(int n_seqs, const std::int32_t* seq_ids, std::int64_t n_keep, std::vector<EvictSeq>* seqs,
                      std::vector<std::int32_t>* dst_pages, bool* any) {
    seqs->clear();
    dst_pages->clear();
    *any = false;
    std::vector<char> seen(static_cast<std::size_t>(cfg_.max_seqs), 0);
    const int np = static_cast<int>((n_keep + kPageTokens - 1) / kPageTokens);
    std::size_t fresh = 0;
    for (int b = 0; b < n_seqs; ++b) {
      const int s = seq_ids[b];
      if (!live(s)) return {YAHKV_ERR_INVALID, "evict: not a live sequence: " + std::to_string(s)};
      if (seen[static_cast<std::size_t>(s)]++) return {YAHKV_ERR_INVALID, "evict: sequence " + std::to_string(s) + " is listed twice"};
      const std::int64_t n = len(s, 0);
      for (int l = 1; l < cfg_.n_layers; ++l)
        if (len(s, l) != n)
          return {YAHKV_ERR_ORDER, "evict: sequence " + std::to_string(s) + " has different lengths in its layers"};
      if (n > PagesHold(s))
        return {YAHKV_ERR_ORDER, "evict: the table of sequence " + std::to_string(s) + " has fewer pages than its length needs"};
      EvictSeq e{};
      e.seq = s, e.n_keys = static_cast<std::int32_t>(n), e.first_dst = static_cast<std::int32_t>(dst_pages->size());
      seqs->push_back(e);
      if (n <= n_keep) continue;
      *any = true;
      for (int i = 0; i < np; ++i) {
        std::int32_t page = table_row(s)[i];
        if (refs_[static_cast<std::size_t>(page)] > 1) {
          if (fresh == free_pages_.size())
            return {YAHKV_ERR_NO_PAGES, "evict: no free page to take the place of a shared one"};
          page = free_pages_[free_pages_.size() - 1 - fresh++];
        }
        dst_pages->push_back(page);
      }
    }
    std::size_t held = 0;
    for (const EvictSeq& e : *seqs) held += static_cast<std::size_t>(n_pages(e.seq));
    evict_dropped_.clear();
    evict_dropped_.reserve(held);
    dirty_list_.reserve(dirty_list_.size() + seqs->size());
    return {};
  }
  void CommitEvict(std::int64_t n_keep, const std::vector<EvictSeq>& seqs, const std::vector<std::int32_t>& dst_pages) noexcept {
    const int np = static_cast<int>((n_keep + kPageTokens - 1) / kPageTokens);
    for (const EvictSeq& e : seqs) {
      if (e.n_keys <= n_keep) continue;
      std::int32_t* row = mutable_row(e.seq);
      for (int i = 0; i < n_pages(e.seq); ++i) {
        const std::int32_t to = i < np ? dst_pages[static_cast<std::size_t>(e.first_dst + i)] : -1;
        if (to == row[i]) continue;
        evict_dropped_.push_back(row[i]);
        if (to < 0) continue;
        free_pages_.pop_back();   // in PlanEvict's order
        refs_[static_cast<std::size_t>(to)] = 1;
        row[i] = to;
      }
      n_pages_[static_cast<std::size_t>(e.seq)] = np;
      SetLenAll(e.seq, n_keep);
      SetEvicted(e.seq);
      MarkDirty(e.seq, 0, np);
    }
    for (std::int32_t p : evict_dropped_) Unref(p);   // only now: a page let go of here was nobody's fresh page
    evict_dropped_.clear();
    InvalidateDecodePlan(), InvalidateSharedPlan();   // made for other sequences, even where a length comes again
  }
  int page_refs(std::int32_t page) const { return refs_[static_cast<std::size_t>(page)]; }
  // Keys of the sequence have been evicted: its slots no longer count positions.
  bool evicted(int seq) const { return evicted_[static_cast<std::size_t>(seq)] != 0; }
  void SetEvicted(int seq) { evicted_[static_cast<std::size_t>(seq)] = 1; }
  // The first page of [position lo, hi) that another sequence holds too; -1: none. Such a page may not be written.
  std::int32_t SharedPageIn(int seq, std::int64_t lo, std::int64_t hi) const {
    for (std::int64_t i = lo / kPageTokens; i < (hi + kPageTokens - 1) / kPageTokens && i < n_pages(seq); ++i)
      if (refs_[static_cast<std::size_t>(table_row(seq)[i])] > 1) return table_row(seq)[i];
    return -1;
  }

  // Checks one append call and computes its slots; on success also advances the lengths. Nothing changes on error.
  HostError PlanAppend(int layer, int n_tokens, const std::int32_t* seq_ids, const std::int64_t* positions,
                       std::int64_t* slots_out) {
    if (layer < 0 || layer >= cfg_.n_layers) return {YAHKV_ERR_INVALID, "append: layer out of range"};
    if (n_tokens < 0) return {YAHKV_ERR_INVALID, "append: negative token count"};
    if (n_tokens > 0 && (seq_ids == nullptr || positions == nullptr)) return {YAHKV_ERR_INVALID, "append: null id or position array"};
    scratch_len_.clear();
    for (int t = 0; t < n_tokens; ++t) {
      const int s = seq_ids[t];
      if (!live(s)) return {YAHKV_ERR_INVALID, "append: not a live sequence: " + std::to_string(s)};
      std::int64_t cur = -1;
      for (auto& e : scratch_len_)
        if (e.first == s) cur = e.second;
      if (cur < 0) cur = len(s, layer);
      const std::int64_t pos = positions[t];
      if (pos != cur)
        return {YAHKV_ERR_ORDER, "append: sequence " + std::to_string(s) + " layer " + std::to_string(layer) +
                                     " expects position " + std::to_string(cur) + ", got " + std::to_string(pos)};
      if (pos >= static_cast<std::int64_t>(n_pages_[static_cast<std::size_t>(s)]) * kPageTokens)
        return {YAHKV_ERR_INVALID, "append: position " + std::to_string(pos) + " of sequence " + std::to_string(s) +
                                       " is past its reserved pages"};
      const std::int32_t page = table_row(s)[pos / kPageTokens];
      if (refs_[static_cast<std::size_t>(page)] > 1)   // a prefix rolled back below a fork
        return {YAHKV_ERR_INVALID, "append: position " + std::to_string(pos) + " of sequence " + std::to_string(s) +
                                       " lies in page " + std::to_string(page) + ", which another sequence shares"};
      slots_out[t] = static_cast<std::int64_t>(page) * kPageTokens + pos % kPageTokens;
      bool found = false;
      for (auto& e : scratch_len_)
        if (e.first == s) e.second = pos + 1, found = true;
      if (!found) scratch_len_.emplace_back(s, pos + 1);
    }
    for (auto& e : scratch_len_) len_ref(e.first, layer) = e.second;
    return {};
  }

  // Split-K plan of one decode call. units / items are rebuilt only when the (sequence, length) list or the split
  // request differs from the cached one; *changed says whether they must be uploaded again.
  HostError PlanDecode(int layer, int n_seqs, const std::int32_t* seq_ids, int n_splits, int max_splits,
                       int max_units, bool* changed) {
    if (layer < 0 || layer >= cfg_.n_layers) return {YAHKV_ERR_INVALID, "attend_decode: layer out of range"};
    if (n_seqs < 0 || (n_seqs > 0 && seq_ids == nullptr)) return {YAHKV_ERR_INVALID, "attend_decode: bad sequence list"};
    if (n_seqs > cfg_.max_seqs) return {YAHKV_ERR_CAPACITY, "attend_decode: more rows than max_seqs"};
    if (n_splits < 0) return {YAHKV_ERR_INVALID, "attend_decode: negative n_splits"};
    if (n_splits > max_splits) return {YAHKV_ERR_CAPACITY, "attend_decode: n_splits above max_splits"};
    key_scratch_.clear();
    key_scratch_.push_back(n_splits);
    long long total_pages = 0;
    for (int b = 0; b < n_seqs; ++b) {
      const int s = seq_ids[b];
      if (!live(s)) return {YAHKV_ERR_INVALID, "attend_decode: not a live sequence: " + std::to_string(s)};
      const std::int64_t n = len(s, layer);
      if (n <= 0)
        return {YAHKV_ERR_ORDER, "attend_decode: sequence " + std::to_string(s) + " has no keys in layer " +
                                     std::to_string(layer) + " (append first)"};
      key_scratch_.push_back(s);
      key_scratch_.push_back(n);
      total_pages += (n + kPageTokens - 1) / kPageTokens;
    }
    if (key_scratch_ == plan_key_) {
      *changed = false;
      return {};
    }
    // Automatic unit size: about five units per resident CTA slot (148 SMs x 2), at most 24 pages each. Measured on
    // the batch-32 benchmark: 10 pages 237 us, 16: 226, 24: 222, 32: 224, 48: 227 per layer; smaller units pay the
    // per-CTA prologue and partial write-back more often, larger ones leave a longer tail.
    const int hb = kv_head_begin(), hc = kv_head_count();
    int auto_pages = static_cast<int>((total_pages * hc + 1479) / 1480);
    auto_pages = std::min(std::max(auto_pages, 1), 24);
    // Built beside the present plan, in memory that is kept: fresh pages for the lists cost more than the planning.
    std::vector<DecodeUnit>& units = next_units_;
    std::vector<CombineItem>& items = next_items_;
    units.clear();
    items.assign(static_cast<std::size_t>(n_seqs) * kKvHeads, CombineItem{});
    std::int32_t slot = 0;   // pages of the units so far
    for (int b = 0; b < n_seqs; ++b) {
      const int s = seq_ids[b];
      const std::int64_t n = len(s, layer);
      const int pages = static_cast<int>((n + kPageTokens - 1) / kPageTokens);
      CutUnits(pages, n_splits, max_splits, auto_pages);
      const int nu = static_cast<int>(bounds_.size());
      for (int h = hb; h < hb + hc; ++h) {   // heads outside the context's range keep n_partials = 0
        items[static_cast<std::size_t>(b) * kKvHeads + h] = {static_cast<std::int32_t>(units.size()), nu};
        AddUnits(b, s, h, n, 0, &slot, &units);
      }
    }
    if (static_cast<long long>(units.size()) > max_units)
      return {YAHKV_ERR_CAPACITY, "attend_decode: split-K plan needs " + std::to_string(units.size()) +
                                      " units, workspace holds " + std::to_string(max_units)};
    LongestFirst(&units);
    unit_pages_ = slot;
    units_.swap(units);
    items_.swap(items);
    plan_key_ = key_scratch_;
    *changed = true;
    return {};
  }
  void InvalidateDecodePlan() { plan_key_.clear(); }

  // ---- decode attention over shared prefixes -------------------------------------------------------------------
  // Rows of the call whose tables start with the same page share a prefix: the longest run of pages common to all of
  // them that every one of them has filled. A group of two rows or more gets prefix tiles (all its rows at once,
  // csrc/shared_attn.cu); what a row has behind its group's prefix, or the whole of a row without one, becomes
  // ordinary split-K units. n_pairs: CTA pairs the device runs at once; max_part_rows: rows of the prefix workspace.
  HostError PlanDecodeShared(int layer, int n_seqs, const std::int32_t* seq_ids, int n_splits, int max_splits,
                             int max_units, int n_pairs, std::int64_t max_part_rows, bool* changed) {
    if (layer < 0 || layer >= cfg_.n_layers) return {YAHKV_ERR_INVALID, "attend_decode_shared: layer out of range"};
    if (n_seqs < 0 || (n_seqs > 0 && seq_ids == nullptr)) return {YAHKV_ERR_INVALID, "attend_decode_shared: bad sequence list"};
    if (n_seqs > cfg_.max_seqs) return {YAHKV_ERR_CAPACITY, "attend_decode_shared: more rows than max_seqs"};
    if (n_splits < 0) return {YAHKV_ERR_INVALID, "attend_decode_shared: negative n_splits"};
    if (n_splits > max_splits) return {YAHKV_ERR_CAPACITY, "attend_decode_shared: n_splits above max_splits"};
    key_scratch_.clear();
    key_scratch_.push_back(n_splits);
    key_scratch_.push_back(table_epoch_);
    for (int b = 0; b < n_seqs; ++b) {
      const int s = seq_ids[b];
      if (!live(s)) return {YAHKV_ERR_INVALID, "attend_decode_shared: not a live sequence: " + std::to_string(s)};
      const std::int64_t n = len(s, layer);
      if (n <= 0)
        return {YAHKV_ERR_ORDER, "attend_decode_shared: sequence " + std::to_string(s) + " has no keys in layer " +
                                     std::to_string(layer) + " (append first)"};
      key_scratch_.push_back(s);
      key_scratch_.push_back(n);
    }
    if (key_scratch_ == shared_.key) {
      *changed = false;
      return {};
    }
    SharedPlan& plan = next_shared_;   // beside the present one, in memory that is kept
    plan.key = key_scratch_;
    plan.tiles.clear(), plan.rows.clear(), plan.units.clear();
    std::vector<std::int64_t> lens(static_cast<std::size_t>(n_seqs));
    for (int b = 0; b < n_seqs; ++b) lens[static_cast<std::size_t>(b)] = len(seq_ids[b], layer);
    const std::vector<PrefixGroup> groups = FindPrefixes(n_seqs, seq_ids, lens.data());
    plan.first_page.assign(static_cast<std::size_t>(n_seqs), 0);
    for (const PrefixGroup& g : groups)
      for (std::int32_t b : g.rows) plan.first_page[static_cast<std::size_t>(b)] = g.pages;
    std::vector<int> suffix(static_cast<std::size_t>(n_seqs));
    for (int b = 0; b < n_seqs; ++b)
      suffix[static_cast<std::size_t>(b)] = static_cast<int>((lens[static_cast<std::size_t>(b)] + kPageTokens - 1) / kPageTokens) -
                                            plan.first_page[static_cast<std::size_t>(b)];
    const SharedShape shape = ChooseSharedShape(groups, suffix, n_pairs, n_splits, max_part_rows);
    BuildPrefixTiles(n_seqs, seq_ids, groups, shape.part_pages, &plan);
    const int hb = kv_head_begin(), hc = kv_head_count(), auto_pages = shape.unit_pages;
    std::int32_t slot = 0;
    plan.items.assign(static_cast<std::size_t>(n_seqs) * kKvHeads, CombineItem{});
    for (int b = 0; b < n_seqs; ++b) {
      const int first = plan.first_page[static_cast<std::size_t>(b)];
      const std::int64_t n = lens[static_cast<std::size_t>(b)];
      const int pages = static_cast<int>((n + kPageTokens - 1) / kPageTokens) - first;
      bounds_.clear();
      if (pages > 0) CutUnits(pages, n_splits, max_splits, auto_pages);
      const int nu = static_cast<int>(bounds_.size());
      for (int h = hb; h < hb + hc; ++h) {
        plan.items[static_cast<std::size_t>(b) * kKvHeads + h] = {static_cast<std::int32_t>(plan.units.size()), nu};
        AddUnits(b, seq_ids[b], h, n, first, &slot, &plan.units);
      }
    }
    if (static_cast<long long>(plan.units.size()) > max_units)
      return {YAHKV_ERR_CAPACITY, "attend_decode_shared: split-K plan needs " + std::to_string(plan.units.size()) +
                                      " units, workspace holds " + std::to_string(max_units)};
    LongestFirst(&plan.units);
    std::swap(shared_, next_shared_);
    *changed = true;
    return {};
  }
  struct SharedPlan {
    std::vector<std::int64_t> key;
    std::vector<int> first_page;            // per row: pages its group's prefix covers (0: no group)
    std::vector<PrefixTile> tiles;          // neighbouring pairs: the two CTAs of a cluster
    std::vector<std::int32_t> rows;         // batch rows of the groups, one list after the other
    std::vector<PrefixItem> prefix_items;   // per (row, kv head): where its prefix partials lie
    std::vector<DecodeUnit> units;
    std::vector<CombineItem> items;
  };
  const SharedPlan& shared_plan() const { return shared_; }
  void InvalidateSharedPlan() { shared_.key.clear(); }

  struct PrefixGroup {
    std::vector<std::int32_t> rows;   // rows of the call
    int pages = 0;                    // the prefix they share
    int n_mt = 0;                     // CTA pairs of 256 (row, query head) pairs
  };
  // Which rows compute a prefix together. The rows' full pages form a tree (forks of forks branch where their tables
  // differ); a group is rows below one node, with the pages down to it, and saves (rows - 1) x pages page reads. Every
  // row is in at most one group. A node's rows are one group, or groups further down with the rows that are in none of
  // those as a group of their own, whichever saves most in all: a short row does not cut the prefix of the long ones, and
  // a few long rows do not take the common prefix from the others.
  // A prefix that does not pay (PrefixPays) is left to its rows.
  std::vector<PrefixGroup> FindPrefixes(int n_seqs, const std::int32_t* seq_ids, const std::int64_t* lens) const {
    std::vector<PrefixGroup> groups;
    std::vector<std::int32_t> rows;
    for (int b = 0; b < n_seqs; ++b)
      if (lens[b] >= kPageTokens) rows.push_back(b);
    std::vector<PrefixNode> tree;
    ForEachBranch(rows, 0, seq_ids, [&](std::vector<std::int32_t>& together) {
      if (together.size() < 2) return;
      tree.clear();
      BuildPrefixTree(together, 0, seq_ids, lens, &tree);
      std::vector<int> above{0};
      SolvePrefixes(&tree, 0, &above);
      std::vector<std::int32_t> alone;
      EmitPrefixes(tree, 0, 0, &alone, &groups);
    });
    for (PrefixGroup& g : groups)
      g.n_mt = (static_cast<int>(g.rows.size()) * kGroup + 2 * kPrefillTileRows - 1) / (2 * kPrefillTileRows);
    return groups;
  }
  // Whether computing `pages` pages once for `rows` rows is faster than leaving them to the rows' own units: it costs two
  // launches' time and CTA pairs that work on half-empty tiles. It pays from a number of saved page reads on, and from a
  // number of pages on that falls once the rows' units alone (four per row at least) no longer fit the device at once (f16
  // one CTA per SM, q8_0 two). Measured in 483 cases of 2 .. 96 rows and 1 .. 256 pages with suffixes of up to 64 tokens, us
  // per call with / without the pass:
  //   f16   2 x 64 13.6 / 13.3   2 x 128 16.2 / 23.7    8 x 4 10.3 / 9.2    8 x 8 10.8 / 13.1   32 x 4 13.5 / 12.1   32 x 6 13.2 / 17.7
  //         43 x 1 14.5 / 14.1   43 x 2 14.7 / 16.7    64 x 1 14.7 / 15.8
  //   q8_0  2 x 16 12.8 / 11.7   2 x 32 13.4 / 13.5     8 x 1 10.7 / 10.7   8 x 4 11.0 / 11.3   24 x 2 13.5 / 13.0   24 x 4 13.7 / 15.4
  //         48 x 4 17.8 / 15.9   48 x 6 16.5 / 18.2    96 x 3 23.5 / 22.6   96 x 4 21.7 / 24.8
  //   q4_0  2 x 16 12.2 / 11.2   2 x 32 13.0 / 14.1     8 x 2 10.7 / 10.3   8 x 4 10.9 / 11.1   32 x 1 13.2 / 12.8   32 x 2 13.3 / 15.1
  // The rule takes the faster side, or one at most 12 % slower; by mean 0.2, 0.4 and 0.1 % are lost.
  bool PrefixPaysMeasured(int rows, int pages) const {
    const std::int64_t saved = static_cast<std::int64_t>(rows - 1) * pages * kv_head_count() / kKvHeads;   // measured with all heads
    switch (cfg_.fmt) {
      case YAHKV_FMT_F16: return saved >= 54 && pages >= (rows < 40 ? 6 : rows < 60 ? 2 : 1);
      case YAHKV_FMT_Q8_0: return saved >= 20 && pages >= (rows < 16 ? 1 : rows < 32 ? 4 : rows < 72 ? 6 : 4);
      default: return saved >= 27 && pages >= (rows < 20 ? 3 : 2);
    }
  }
  bool PrefixPays(int rows, int pages) const {
    if (shared_min_saved_ > 0) return static_cast<std::int64_t>(rows - 1) * pages >= shared_min_saved_;
    return PrefixPaysMeasured(rows, pages);
  }
  // The page reads a prefix must save instead of the measured rule.
  void SetSharedMinSaved(int pages) {
    shared_min_saved_ = pages;
    InvalidateSharedPlan();
  }

  // How a shared plan is cut: pages per prefix part and pages per suffix unit.
  //
  // Every (group, kv head, 256 rows) is cut along its pages into parts, one CTA pair each; the pairs of a wave take as
  // long as the largest part. The suffix units run beside the prefix pass on the SMs it leaves free, and on all of them
  // once it is done, so the wave need not be the whole device: for every wave size the suffixes' end is estimated from
  // the measured times of a pair (6 us and 0.75 us per fp16 page, 0.95 us where pages are dequantized) and of a unit
  // (f16 three CTAs per SM, 7 us and 2 us per page; q8_0 two, 4 and 0.9; q4_0 four, 4 and 1.6), and the cheapest pair of
  // sizes is taken. 96 rows x 16421 fp16: 83 us with the whole device and units of two pages, 76 as chosen here, 69 with the
  // units' present form of three CTAs per SM.
  struct SharedShape {
    int part_pages = 1, unit_pages = 1;
  };
  SharedShape ChooseSharedShape(const std::vector<PrefixGroup>& groups, const std::vector<int>& suffix, int n_pairs, int n_splits,
                                std::int64_t max_part_rows) const {
    const int hc = kv_head_count();
    const bool f16 = cfg_.fmt == YAHKV_FMT_F16, q8 = cfg_.fmt == YAHKV_FMT_Q8_0;
    const double pair_fixed = 6.0, pair_page = f16 ? 0.75 : 0.95;
    const double unit_fixed = f16 ? 7.0 : 4.0, unit_page = f16 ? 2.0 : q8 ? 0.9 : 1.6;
    const int ctas = f16 ? 3 : q8 ? 2 : 4;
    auto pairs_at = [&](int per) {
      long long n = 0;
      for (const PrefixGroup& g : groups) n += static_cast<long long>(g.n_mt) * hc * ((g.pages + per - 1) / per);
      return n;
    };
    auto rows_at = [&](int per) {
      long long n = 0;
      for (const PrefixGroup& g : groups) n += static_cast<long long>(g.rows.size()) * kGroup * hc * ((g.pages + per - 1) / per);
      return n;
    };
    int most = 1, longest = 0;
    for (const PrefixGroup& g : groups) most = std::max(most, g.pages);
    for (int n : suffix) longest = std::max(longest, n);
    // units of p pages (or the asked-for number of them per row): how many, their mean time and the longest one's
    struct Units {
      int pages;
      long long count;
      double mean, longest;
    };
    std::vector<Units> cuts;
    for (int p : {1, 2, 4, 6, 8, 12, 16, 24}) {
      Units u{p, 0, unit_fixed, unit_fixed};
      int largest = 0;
      long long pages = 0;
      for (int n : suffix) {
        const int per = n_splits > 0 ? std::max((n + n_splits - 1) / n_splits, 1) : p;
        u.count += static_cast<long long>(hc) * ((n + per - 1) / per);
        largest = std::max(largest, std::min(n, per));
        pages += static_cast<long long>(hc) * n;
      }
      u.longest += unit_page * largest;
      if (u.count > 0) u.mean += unit_page * static_cast<double>(pages) / static_cast<double>(u.count);
      cuts.push_back(u);
      if (n_splits > 0 || p >= longest) break;
    }
    SharedShape best;
    double least = -1.0;
    const int waves_max = groups.empty() ? 1 : 4;
    for (int step = 0; step <= 10; ++step) {   // the wave: all pairs down to half of them
      const int wave = groups.empty() ? 0 : std::max(n_pairs - n_pairs * step / 20, 1);
      for (int waves = 1; waves <= waves_max; ++waves) {
        int per = 1;
        double prefix = 0.0;
        if (!groups.empty()) {   // the smallest part that fits the waves
          int lo = 1, hi = most;
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (pairs_at(mid) <= static_cast<long long>(waves) * wave) hi = mid;
            else lo = mid + 1;
          }
          per = lo;
          while (per < most && rows_at(per) > max_part_rows) ++per;   // one part per tile always fits (24 rows per batch row)
          prefix = static_cast<double>((pairs_at(per) + wave - 1) / wave) * (pair_fixed + pair_page * per);
        }
        const int busy = static_cast<int>(std::min<long long>(groups.empty() ? 0 : pairs_at(per), n_pairs));
        const long long beside = 2LL * (n_pairs - busy) * ctas, all = 2LL * n_pairs * ctas;
        for (const Units& u : cuts) {
          const double left = static_cast<double>(u.count) - static_cast<double>(beside) * prefix / u.mean;
          double end = prefix;
          if (u.count > 0)
            end = std::max(end, left > 0.0 ? prefix + left / static_cast<double>(all) * u.mean + 0.5 * u.longest
                                           : static_cast<double>(u.count) / static_cast<double>(beside) * u.mean + 0.5 * u.longest);
          end += 0.005 * static_cast<double>(u.count + pairs_at(per));   // the partials: written, read, joined
          if (least < 0.0 || end < least - 1e-9) least = end, best.part_pages = per, best.unit_pages = u.pages;
        }
      }
      if (groups.empty()) break;
    }
    return best;
  }

  // The tiles of the prefix pass and where every row finds its partials.
  void BuildPrefixTiles(int n_seqs, const std::int32_t* seq_ids, const std::vector<PrefixGroup>& groups, int per, SharedPlan* plan) const {
    const int hb = kv_head_begin(), hc = kv_head_count();
    plan->prefix_items.assign(static_cast<std::size_t>(n_seqs) * kKvHeads, PrefixItem{});
    std::int64_t part_row = 0;
    for (const PrefixGroup& g : groups) {
      const std::int32_t list = static_cast<std::int32_t>(plan->rows.size());
      const int n_rows = static_cast<int>(g.rows.size()) * kGroup;
      const int n_parts = (g.pages + per - 1) / per;
      plan->rows.insert(plan->rows.end(), g.rows.begin(), g.rows.end());
      for (int h = hb; h < hb + hc; ++h) {
        for (std::size_t i = 0; i < g.rows.size(); ++i)
          plan->prefix_items[static_cast<std::size_t>(g.rows[i]) * kKvHeads + h] = {
              static_cast<std::int32_t>(part_row + static_cast<std::int64_t>(i) * kGroup), n_parts, n_rows, 0};
        for (int k = 0; k < n_parts; ++k) {
          for (int r = 0; r < g.n_mt * 2 * kPrefillTileRows; r += kPrefillTileRows) {   // two CTAs per pair, the last may be empty
            PrefixTile t{};
            t.row_list = list, t.row0 = r, t.n_rows = std::min(std::max(n_rows - r, 0), kPrefillTileRows);
            t.kvh = h, t.seq = seq_ids[g.rows[0]];
            t.page_begin = g.pages * k / n_parts, t.page_end = g.pages * (k + 1) / n_parts;
            t.part_row0 = static_cast<std::int32_t>(part_row + r);
            plan->tiles.push_back(t);
          }
          part_row += n_rows;
        }
      }
    }
    // longest parts first; the two CTAs of a pair have equal keys and stay neighbours
    std::stable_sort(plan->tiles.begin(), plan->tiles.end(), [](const PrefixTile& a, const PrefixTile& b) {
      return a.page_end - a.page_begin > b.page_end - b.page_begin;
    });
  }

  // ---- kv8a16: which of a (sequence, layer)'s two open-tile buffers is current, and the V tile work of an append --
  int open_cur(int seq, int layer) const {
    return open_cur_.empty() ? 0 : open_cur_[static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.n_layers) + static_cast<std::size_t>(layer)];
  }
  // Called after a successful PlanAppend of the same call: the tokens of every sequence are consecutive positions
  // starting at its previous length, so the first position seen is that length. Builds one work item per 16-key tile
  // the call touches and flips the open buffer of sequences whose newest tile changed.
  void PlanKv8Tiles(int layer, int n_tokens, const std::int32_t* seq_ids, const std::int64_t* positions,
                    std::vector<VTileWork>* work) {
    if (open_cur_.empty()) open_cur_.assign(static_cast<std::size_t>(cfg_.max_seqs) * static_cast<std::size_t>(cfg_.n_layers), 0);
    work->clear();
    struct Span {
      int seq;
      std::int64_t p0, p1;
    };
    std::vector<Span> spans;
    for (int t = 0; t < n_tokens; ++t) {
      bool found = false;
      for (auto& sp : spans)
        if (sp.seq == seq_ids[t]) sp.p1 = positions[t] + 1, found = true;
      if (!found) spans.push_back({seq_ids[t], positions[t], positions[t] + 1});
    }
    for (const Span& sp : spans) {
      const std::size_t si = static_cast<std::size_t>(sp.seq) * static_cast<std::size_t>(cfg_.n_layers) + static_cast<std::size_t>(layer);
      const int cur = open_cur_[si];
      const std::int64_t t0 = sp.p0 / kTileKeys, t1 = (sp.p1 - 1) / kTileKeys;
      for (std::int64_t tile = t0; tile <= t1; ++tile) {
        VTileWork w{};
        w.state_row = static_cast<std::int32_t>(si);
        w.phys_tile = table_row(sp.seq)[tile * kTileKeys / kPageTokens] * kTilesPerPage + static_cast<std::int32_t>(tile % kTilesPerPage);
        w.n_old = tile == t0 ? static_cast<std::int32_t>(sp.p0 - tile * kTileKeys) : 0;
        w.n_keys = static_cast<std::int32_t>(std::min<std::int64_t>(kTileKeys, sp.p1 - tile * kTileKeys));
        w.read_buf = cur;
        w.write_buf = tile != t1 ? -1 : (t0 == t1 ? cur : cur ^ 1);
        w.complete = w.n_keys == kTileKeys ? 1 : 0;
        for (int j = 0; j < kTileKeys; ++j) w.src[j] = -1;
        work->push_back(w);
      }
      if (t0 != t1) open_cur_[si] = cur ^ 1;
    }
    // input token index of every new key
    for (int t = 0; t < n_tokens; ++t) {
      const std::int64_t tile = positions[t] / kTileKeys;
      std::size_t base = 0;
      for (const Span& sp : spans) {
        const std::int64_t t0 = sp.p0 / kTileKeys, t1 = (sp.p1 - 1) / kTileKeys;
        if (sp.seq == seq_ids[t]) {
          (*work)[base + static_cast<std::size_t>(tile - t0)].src[positions[t] % kTileKeys] = t;
          break;
        }
        base += static_cast<std::size_t>(t1 - t0 + 1);
      }
    }
  }
  void ResetOpenState(int seq) {
    if (open_cur_.empty()) return;
    for (int l = 0; l < cfg_.n_layers; ++l) open_cur_[static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.n_layers) + static_cast<std::size_t>(l)] = 0;
  }
  std::int64_t unit_pages() const { return unit_pages_; }   // pages of all units of the plan: slots of their scores
  const std::vector<DecodeUnit>& units() const { return units_; }
  const std::vector<CombineItem>& items() const { return items_; }

  // Work lists of one prefill call: per sequence the span of the fp16 scratch it is dequantized into, and tiles of
  // 128 query rows x one query head, the ones with the most keys first so that the short ones fill the tail.
  // n_sm > 0: the tiles of the last, partly filled wave (one CTA per SM and wave, all tiles cost about the same) are
  // split along their keys into parts that fill the wave's idle SMs; `merges` lists them for the merge kernel, one
  // entry per head.
  HostError PlanPrefill(int layer, int n_seqs, const std::int32_t* seq_ids, const std::int32_t* chunk_lens,
                        int max_rows, int n_sm, std::vector<PrefillSeq>* seqs, std::vector<PrefillTile>* tiles,
                        std::vector<PrefillMerge>* merges, int* n_parts, std::int64_t* total_rows,
                        std::int64_t* scratch_rows, int* max_pages) {
    if (layer < 0 || layer >= cfg_.n_layers) return {YAHKV_ERR_INVALID, "attend_prefill: layer out of range"};
    if (n_seqs < 0 || (n_seqs > 0 && (seq_ids == nullptr || chunk_lens == nullptr)))
      return {YAHKV_ERR_INVALID, "attend_prefill: bad sequence list"};
    seqs->clear();
    tiles->clear();
    std::int64_t row = 0, kv_row = 0;
    *max_pages = 0;
    for (int i = 0; i < n_seqs; ++i) {
      const int s = seq_ids[i];
      if (!live(s)) return {YAHKV_ERR_INVALID, "attend_prefill: not a live sequence: " + std::to_string(s)};
      const std::int64_t n = len(s, layer);
      const int c = chunk_lens[i];
      if (c <= 0) return {YAHKV_ERR_INVALID, "attend_prefill: chunk length must be positive"};
      if (c > n)
        return {YAHKV_ERR_ORDER, "attend_prefill: chunk of " + std::to_string(c) + " rows but sequence " +
                                     std::to_string(s) + " holds " + std::to_string(n) + " keys (append first)"};
      PrefillSeq ps{};
      ps.seq = s;
      ps.n_pages = static_cast<std::int32_t>((n + kPageTokens - 1) / kPageTokens);
      ps.kv_len = static_cast<std::int32_t>(n);
      ps.kv_rows = ps.n_pages * kPageTokens;
      ps.kv_row0 = static_cast<std::int32_t>(kv_row);
      seqs->push_back(ps);
      *max_pages = std::max(*max_pages, static_cast<int>(ps.n_pages));
      for (int r = 0; r < c; r += kPrefillTileRows)
        for (int h = kv_head_begin() * kGroup; h < (kv_head_begin() + kv_head_count()) * kGroup; ++h) {
          PrefillTile t{};
          t.kv_row0 = static_cast<std::int32_t>(kv_row + static_cast<std::int64_t>(h / kGroup) * ps.kv_rows);
          t.head = h;
          t.q_row0 = static_cast<std::int32_t>(row + r);
          t.n_rows = std::min(kPrefillTileRows, c - r);
          t.pos0 = static_cast<std::int32_t>(n - c + r);
          t.jt_begin = 0, t.jt_end = (t.pos0 + t.n_rows + 63) / 64, t.part = -1;
          tiles->push_back(t);
        }
      row += c;
      kv_row += static_cast<std::int64_t>(kKvHeads) * ps.kv_rows;
      if (kv_row >= (1LL << 31)) return {YAHKV_ERR_CAPACITY, "attend_prefill: too many cached keys in one call"};
    }
    if (row > max_rows) return {YAHKV_ERR_CAPACITY, "attend_prefill: more query rows than max_batch_tokens"};
    std::stable_sort(tiles->begin(), tiles->end(),
                     [](const PrefillTile& a, const PrefillTile& b) { return a.pos0 + a.n_rows > b.pos0 + b.n_rows; });
    merges->clear();
    *n_parts = 0;
    // The kernel runs the two heads of a pair (entries 2 i and 2 i + 1: equal sort keys keep the neighbours of the loop
    // above together) as one CTA pair on two SMs, so the wave is counted in pairs.
    const int n_pairs = static_cast<int>(tiles->size()) / 2;
    const int wave = n_sm / 2;
    const int tail = wave > 0 ? n_pairs % wave : 0;   // a call of fewer pairs than the wave is all tail
    // Split factor: the tail's pairs cut into f key ranges take ceil(tail f / wave) waves of 1 / f tile time each.
    int f = 1;
    double best = 1.0;
    for (int c = 2; c <= kPrefillMaxParts && tail > 0; ++c) {
      const double cost = static_cast<double>((tail * c + wave - 1) / wave) / c;
      if (cost < best - 1e-9) best = cost, f = c;
    }
    if (f > 1) {
      const std::vector<PrefillTile> last(tiles->end() - 2 * tail, tiles->end());
      tiles->resize(static_cast<std::size_t>(2 * (n_pairs - tail)));
      for (std::size_t i = 0; i + 1 < last.size(); i += 2) {
        const PrefillTile& t = last[i];
        const int ff = std::min(f, t.jt_end / 2);   // a part covers at least two key tiles
        if (ff < 2) {
          tiles->push_back(last[i]);
          tiles->push_back(last[i + 1]);
          continue;
        }
        // part k of the two heads sits at entries first + 2 k, first + 2 k + 1 and takes the part slots of the same
        // parity: the merge kernel steps by two
        merges->push_back({static_cast<std::int32_t>(tiles->size()), ff});
        merges->push_back({static_cast<std::int32_t>(tiles->size()) + 1, ff});
        for (int k = 0; k < ff; ++k)
          for (int h = 0; h < 2; ++h) {
            PrefillTile p = last[i + static_cast<std::size_t>(h)];
            p.jt_begin = t.jt_end * k / ff, p.jt_end = t.jt_end * (k + 1) / ff, p.part = (*n_parts)++;
            tiles->push_back(p);
          }
      }
    }
    *total_rows = row;
    *scratch_rows = kv_row;
    return {};
  }

  // Puts a range back that ForEachDirty handed out but the caller could not upload.
  void MarkDirtyAgain(int seq, int lo, int hi) { MarkDirty(seq, lo, hi); }

  // Rows of the block table changed since the last call: [lo, hi) per sequence. The caller uploads and clears.
  template <class F>
  void ForEachDirty(F&& fn) {
    for (int s : dirty_list_) {
      const std::size_t i = static_cast<std::size_t>(s);
      if (dirty_hi_[i] > dirty_lo_[i]) fn(s, dirty_lo_[i], dirty_hi_[i]);
      dirty_lo_[i] = dirty_hi_[i] = 0;
    }
    dirty_list_.clear();
  }

 private:
  // ---- the tree of shared prefixes (FindPrefixes) ----
  // Rows that agree in their first `pages` pages. What is best below a node depends on the nearest group above it, which
  // its rows may join instead: with D pages in that group (0: there is none) a row that joins it counts D. Entry k of the
  // three lists is for the k-th of the possible groups above, from none to the parent.
  struct PrefixNode {
    int pages = 0, count = 0;             // the agreed pages; rows at and below the node
    std::vector<std::int32_t> rows;       // rows that end here or go on alone
    std::vector<int> children;
    enum Choice : char { kJoin, kWhole, kSplit };
    std::vector<std::int64_t> value;      // page reads saved below, plus D for every row that joins the group above
    std::vector<int> up;                  // rows that join it
    std::vector<Choice> choice;           // no group here; all rows one group; a group of the rows that are in none below
  };
  // Calls fn with the rows that have the same page `at`, page by page.
  template <class F>
  void ForEachBranch(const std::vector<std::int32_t>& rows, int at, const std::int32_t* seq_ids, F&& fn) const {
    std::vector<std::pair<std::int32_t, std::int32_t>> by_page;   // (page, row)
    by_page.reserve(rows.size());
    for (std::int32_t b : rows) by_page.emplace_back(table_row(seq_ids[b])[at], b);
    std::sort(by_page.begin(), by_page.end());
    std::vector<std::int32_t> branch;
    for (std::size_t i = 0; i < by_page.size();) {
      branch.clear();
      const std::int32_t page = by_page[i].first;
      for (; i < by_page.size() && by_page[i].first == page; ++i) branch.push_back(by_page[i].second);
      fn(branch);
    }
  }
  // The node of two rows or more that agree in their first `from` pages; its children behind it. Returns its index.
  int BuildPrefixTree(const std::vector<std::int32_t>& rows, int from, const std::int32_t* seq_ids, const std::int64_t* lens,
                      std::vector<PrefixNode>* tree) const {
    const std::int32_t* first = table_row(seq_ids[rows[0]]);
    int common = static_cast<int>(lens[rows[0]] / kPageTokens);
    for (std::size_t i = 1; i < rows.size(); ++i) {
      common = std::min(common, static_cast<int>(lens[rows[i]] / kPageTokens));
      const int known = std::min(from, common);
      const std::int32_t* row = table_row(seq_ids[rows[i]]);
      if (std::memcmp(first + known, row + known, static_cast<std::size_t>(common - known) * sizeof(*row)) != 0)
        common = static_cast<int>(std::mismatch(first + known, first + common, row + known).first - first);
    }
    const int at = static_cast<int>(tree->size());
    tree->emplace_back();
    (*tree)[static_cast<std::size_t>(at)].pages = common;
    (*tree)[static_cast<std::size_t>(at)].count = static_cast<int>(rows.size());
    std::vector<std::int32_t> longer;
    for (std::int32_t b : rows)
      if (lens[b] / kPageTokens <= common) (*tree)[static_cast<std::size_t>(at)].rows.push_back(b);
      else longer.push_back(b);
    ForEachBranch(longer, common, seq_ids, [&](const std::vector<std::int32_t>& branch) {
      if (branch.size() == 1) {
        (*tree)[static_cast<std::size_t>(at)].rows.push_back(branch[0]);
      } else {
        const int child = BuildPrefixTree(branch, common, seq_ids, lens, tree);
        (*tree)[static_cast<std::size_t>(at)].children.push_back(child);
      }
    });
    return at;
  }
  // Fills value, up and choice of a node and of what is below it; above: the pages of the groups that may lie above.
  void SolvePrefixes(std::vector<PrefixNode>* tree, int at, std::vector<int>* above) const {
    PrefixNode& v = (*tree)[static_cast<std::size_t>(at)];
    above->push_back(v.pages);
    for (int c : v.children) SolvePrefixes(tree, c, above);
    above->pop_back();
    const std::size_t self = above->size();
    const std::int64_t own = static_cast<std::int64_t>(v.rows.size());
    std::int64_t split = v.pages * (own - 1);
    int left = static_cast<int>(own);
    for (int c : v.children) split += (*tree)[static_cast<std::size_t>(c)].value[self], left += (*tree)[static_cast<std::size_t>(c)].up[self];
    const std::int64_t whole = static_cast<std::int64_t>(v.pages) * (v.count - 1);
    const bool may_whole = PrefixPays(v.count, v.pages);
    // beside groups below, a group must be worth its own tiles
    const bool may_split = left >= 2 && left < v.count && PrefixPays(left, v.pages) && PrefixPaysMeasured(left, v.pages);
    v.value.resize(self), v.up.resize(self), v.choice.resize(self);
    for (std::size_t k = 0; k < self; ++k) {
      v.value[k] = (*above)[k] * own, v.up[k] = static_cast<int>(own), v.choice[k] = PrefixNode::kJoin;
      for (int c : v.children) v.value[k] += (*tree)[static_cast<std::size_t>(c)].value[k], v.up[k] += (*tree)[static_cast<std::size_t>(c)].up[k];
      if (may_whole && (whole > v.value[k] || (k == 0 && whole == v.value[k]))) v.value[k] = whole, v.up[k] = 0, v.choice[k] = PrefixNode::kWhole;
      if (may_split && split > v.value[k]) v.value[k] = split, v.up[k] = 0, v.choice[k] = PrefixNode::kSplit;
    }
  }
  void RowsBelow(const std::vector<PrefixNode>& tree, int at, std::vector<std::int32_t>* rows) const {
    const PrefixNode& v = tree[static_cast<std::size_t>(at)];
    rows->insert(rows->end(), v.rows.begin(), v.rows.end());
    for (int c : v.children) RowsBelow(tree, c, rows);
  }
  // The groups that were chosen at and below a node, given the k-th possible group above; `up` receives the rows that join it.
  void EmitPrefixes(const std::vector<PrefixNode>& tree, int at, std::size_t k, std::vector<std::int32_t>* up,
                    std::vector<PrefixGroup>* groups, std::size_t depth = 1) const {
    const PrefixNode& v = tree[static_cast<std::size_t>(at)];
    if (v.choice[k] == PrefixNode::kJoin) {
      up->insert(up->end(), v.rows.begin(), v.rows.end());
      for (int c : v.children) EmitPrefixes(tree, c, k, up, groups, depth + 1);
      return;
    }
    PrefixGroup g;
    g.pages = v.pages;
    if (v.choice[k] == PrefixNode::kWhole) {
      RowsBelow(tree, at, &g.rows);
    } else {
      g.rows = v.rows;
      for (int c : v.children) EmitPrefixes(tree, c, depth, &g.rows, groups, depth + 1);
    }
    std::sort(g.rows.begin(), g.rows.end());
    groups->push_back(std::move(g));
  }

  // The units that CutUnits has cut (bounds_), for one batch row and kv head, behind the row's first `first` pages. *slot counts
  // the pages of all units.
  void AddUnits(int b, int seq, int h, std::int64_t n_keys, int first, std::int32_t* slot, std::vector<DecodeUnit>* units) const {
    const std::size_t at = units->size(), n = bounds_.size();
    units->resize(at + n);
    DecodeUnit* u = units->data() + at;
    int page = 0;
    for (std::size_t k = 0; k < n; ++k, ++u) {
      u->batch = b, u->seq = seq, u->kvh = h;
      u->page_begin = first + page, u->page_end = first + bounds_[k];
      u->n_keys = static_cast<std::int32_t>(n_keys);
      u->partial = static_cast<std::int32_t>(at + k);
      u->pad = *slot;
      *slot += bounds_[k] - page;
      page = bounds_[k];
    }
  }
  // Longest units first, equal ones in their order: CTAs are handed out in index order, so the short tail units fill the
  // last wave. Counted by length: every call with changed lengths does this (1280 units: 5 us, a comparison sort 30).
  void LongestFirst(std::vector<DecodeUnit>* units) {
    int longest = 0;
    for (const DecodeUnit& u : *units) longest = std::max(longest, u.page_end - u.page_begin);
    sort_at_.assign(static_cast<std::size_t>(longest) + 2, 0);
    for (const DecodeUnit& u : *units) ++sort_at_[static_cast<std::size_t>(longest - (u.page_end - u.page_begin)) + 1];
    for (std::size_t i = 1; i < sort_at_.size(); ++i) sort_at_[i] += sort_at_[i - 1];
    sort_scratch_.resize(units->size());
    for (const DecodeUnit& u : *units) sort_scratch_[static_cast<std::size_t>(sort_at_[static_cast<std::size_t>(longest - (u.page_end - u.page_begin))]++)] = u;
    units->swap(sort_scratch_);
  }
  // Page boundaries of one sequence's split-K units over `pages` pages, into bounds_.
  void CutUnits(int pages, int n_splits, int max_splits, int auto_pages) {
    int per = n_splits > 0 ? (pages + n_splits - 1) / n_splits : auto_pages;
    per = std::max(per, (pages + max_splits - 1) / max_splits);
    // The part kernel's two page sets take alternate pages of a unit: an odd count leaves one set idle for a page,
    // so a unit costs as much as the next even count. Rounding up never raises the number of units.
    if (per > 1) per += per & 1;
    const int nu = (pages + per - 1) / per;
    // Graded sizes: with eight or more units the last quarter of them is half as long (and the others a little
    // longer, the count stays). CTAs take units longest first, so the short ones of all sequences run last and fill
    // the gaps of the final wave: equal units on a grid that is not a multiple of the resident CTAs leave a last
    // wave that is mostly idle (8 x 131072 tokens in 64 splits: 1952 equal units on 592 CTA slots).
    bounds_.clear();
    if (nu >= 8) {
      const int n_small = nu / 4, n_big = nu - n_small;
      int big = (2 * pages + 2 * n_big + n_small - 1) / (2 * n_big + n_small);
      big += big & 1;
      const int small = std::max(((big / 2) + 1) & ~1, 2);
      int p = 0;
      for (int k = 0; k < n_big && p < pages; ++k) bounds_.push_back(p = std::min(p + big, pages));
      while (p < pages) bounds_.push_back(p = std::min(p + small, pages));
    } else {
      for (int k = 0; k < nu; ++k) bounds_.push_back(std::min(pages, (k + 1) * per));
    }
  }
  std::int32_t* mutable_row(int seq) {
    return table_.data() + static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.max_pages_per_seq);
  }
  std::int64_t& len_ref(int seq, int layer) {
    return len_[static_cast<std::size_t>(seq) * static_cast<std::size_t>(cfg_.n_layers) + static_cast<std::size_t>(layer)];
  }
  void SetLenAll(int seq, std::int64_t v) {
    for (int l = 0; l < cfg_.n_layers; ++l) len_ref(seq, l) = v;
  }
  void ReleasePages(int seq) {
    const std::int32_t* row = table_row(seq);
    // Pushed in table order, so the most recently added page is reused first.
    for (int i = 0; i < n_pages_[static_cast<std::size_t>(seq)]; ++i) Unref(row[i]);
    n_pages_[static_cast<std::size_t>(seq)] = 0;
    ++table_epoch_;
  }
  void Unref(std::int32_t page) {
    if (--refs_[static_cast<std::size_t>(page)] == 0) free_pages_.push_back(page);
  }
  // A live sequence other than `seq` whose table names page p; -1: there is none.
  int OtherHolder(std::int32_t p, int seq) const {
    for (int s = 0; s < cfg_.max_seqs; ++s) {
      if (s == seq || !live(s)) continue;
      for (int i = 0; i < n_pages(s); ++i)
        if (table_row(s)[i] == p) return s;
    }
    return -1;
  }
  void MarkDirty(int seq, int lo, int hi) {
    ++table_epoch_;
    const std::size_t i = static_cast<std::size_t>(seq);
    if (dirty_hi_[i] == dirty_lo_[i]) {
      dirty_lo_[i] = lo, dirty_hi_[i] = hi;
      dirty_list_.push_back(seq);
    } else {
      dirty_lo_[i] = std::min(dirty_lo_[i], lo), dirty_hi_[i] = std::max(dirty_hi_[i], hi);
    }
  }

  yahkv_config cfg_;
  std::vector<std::int32_t> table_;
  std::vector<int> n_pages_;
  std::vector<char> live_;
  std::vector<std::int64_t> len_;
  std::vector<int> dirty_lo_, dirty_hi_, dirty_list_;
  std::vector<int> refs_;       // sequences whose table names the page
  std::vector<std::uint32_t> generation_;   // sequences created under the id so far
  std::vector<char> evicted_;   // per sequence: keys were evicted, slots are not positions
  std::int64_t table_epoch_ = 0;   // counts table changes: what a cached prefix grouping depends on
  std::vector<std::int32_t> free_pages_;     // room for every page from the start: giving one back does not fail
  std::vector<std::int32_t> evict_dropped_;
  std::vector<int> free_seqs_;
  std::vector<std::pair<int, std::int64_t>> scratch_len_;
  std::vector<std::int64_t> key_scratch_, plan_key_;
  std::vector<int> sort_at_;
  std::vector<DecodeUnit> sort_scratch_;
  std::vector<DecodeUnit> units_;
  std::int64_t unit_pages_ = 0;
  std::vector<CombineItem> items_;
  std::vector<DecodeUnit> next_units_;
  std::vector<CombineItem> next_items_;
  SharedPlan shared_, next_shared_;   // the plan of attend_decode_shared, and the memory of the one before
  int shared_min_saved_ = 0;    // 0: PrefixPaysMeasured decides
  std::vector<int> open_cur_;   // kv8a16: current open-tile buffer per (sequence, layer)
  std::vector<int> bounds_;     // PlanDecode: page boundaries of one sequence's units
};

}  // namespace yahkv
