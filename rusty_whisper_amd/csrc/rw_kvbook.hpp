// rw_kvbook.hpp -- which sequence holds which pages of a paged key/value
// cache, and when: adding, extending, forking, truncating, releasing and
// compacting sequences.
//
// A page holds page_rows rows of every layer and is counted once per sequence
// that lists it.  A fork lists its parent's pages, so rows are shared until
// one of the two grows into a shared page; that page is then replaced by a
// copy (copy on write).  The book moves no data: it says which pages to copy,
// and the caller queues that copy before anything that writes the rows.
//
// The lowest free page id is handed out first (as is the lowest sequence id),
// so equal histories give equal tables.  Every function either does all that
// it was asked or changes nothing.
//
// Host-only C++ (no HIP types), so the logic is tested on the CPU under
// AddressSanitizer.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include <vector>

namespace rw {

enum class BookError { none, seq, twice, length, pages, seqs, room };

class KvBook {
 public:
  KvBook(size_t n_pages, size_t page_rows, size_t max_seqs)
      : rows_(page_rows), refs_(n_pages, 0), free_(n_pages), free_bits_((n_pages + 63) / 64, 0), max_seqs_(max_seqs) {
    for (size_t p = 0; p < n_pages; ++p) free_bits_[p >> 6] |= (uint64_t)1 << (p & 63);
  }

  size_t n_pages() const { return refs_.size(); }
  size_t free_pages() const { return free_; }
  size_t n_seqs() const { return live_; }
  bool live(int32_t s) const { return s >= 0 && (size_t)s < seqs_.size() && seqs_[s].live; }
  size_t len(int32_t s) const { return seqs_[s].len; }
  const std::vector<int32_t> &pages(int32_t s) const { return seqs_[s].pages; }

  // n new sequences without rows
  BookError add(size_t n, int32_t *out) {
    if (n > max_seqs_ - live_) return BookError::seqs;
    make_room(n);
    for (size_t i = 0; i < n; ++i) out[i] = take_seq();
    return BookError::none;
  }

  // n new sequences, the i-th with the rows of from[i]
  BookError fork(const int32_t *from, size_t n, int32_t *out) {
    for (size_t i = 0; i < n; ++i)
      if (!live(from[i])) return BookError::seq;
    if (n > max_seqs_ - live_) return BookError::seqs;
    std::vector<std::vector<int32_t>> lists(n);
    for (size_t i = 0; i < n; ++i) lists[i] = seqs_[from[i]].pages;
    std::vector<size_t> lens(n);
    for (size_t i = 0; i < n; ++i) lens[i] = seqs_[from[i]].len;
    make_room(n);
    for (size_t i = 0; i < n; ++i) {
      out[i] = take_seq();
      Seq &s = seqs_[out[i]];
      for (int32_t p : lists[i]) ++refs_[p];
      s.pages.swap(lists[i]);
      s.len = lens[i];
    }
    return BookError::none;
  }

  // more[i] further rows for seqs[i] (no sequence twice).  src/dst (n entries
  // each) and *n_copies get the pages to copy.
  BookError extend(const int32_t *seqs, size_t n, const size_t *more, int32_t *src, int32_t *dst, size_t *n_copies) {
    *n_copies = 0;
    const BookError e = distinct(seqs, n);
    if (e != BookError::none) return e;
    for (size_t i = 0; i < n; ++i)
      if (more[i] > (size_t)INT32_MAX || seqs_[seqs[i]].len > (size_t)INT32_MAX - more[i]) return BookError::length;
    // The pages needed.  Of the k sequences of this call that share a last
    // page which nobody else holds, the last one to be extended keeps it.
    size_t need = 0;
    for (size_t i = 0; i < n; ++i) {
      Seq &s = seqs_[seqs[i]];
      if (shares_tail(s, more[i])) --refs_[s.pages.back()], s.counted = true, ++need;
      need += pages_of(s.len + more[i]) - s.pages.size();
    }
    for (size_t i = 0; i < n; ++i) {
      Seq &s = seqs_[seqs[i]];
      if (s.counted) ++refs_[s.pages.back()], s.counted = false;
    }
    if (need > free_) return BookError::pages;
    for (size_t i = 0; i < n; ++i) seqs_[seqs[i]].pages.reserve(pages_of(seqs_[seqs[i]].len + more[i]));
    for (size_t i = 0; i < n; ++i) {
      Seq &s = seqs_[seqs[i]];
      if (shares_tail(s, more[i])) {
        const int32_t p = take_page();
        src[*n_copies] = s.pages.back(), dst[*n_copies] = p;
        ++*n_copies;
        --refs_[s.pages.back()];
        s.pages.back() = p;
      }
      s.len += more[i];
      while (s.pages.size() < pages_of(s.len)) s.pages.push_back(take_page());
    }
    return BookError::none;
  }

  // drops the rows from `len` on
  BookError truncate(int32_t seq, size_t len) {
    if (!live(seq)) return BookError::seq;
    Seq &s = seqs_[seq];
    if (len > s.len) return BookError::length;
    s.len = len;
    while (s.pages.size() > pages_of(len)) drop_page(s.pages.back()), s.pages.pop_back();
    return BookError::none;
  }

  // ends sequences (none twice)
  BookError release(const int32_t *seqs, size_t n) {
    const BookError e = distinct(seqs, n);
    if (e != BookError::none) return e;
    for (size_t i = 0; i < n; ++i) {
      Seq &s = seqs_[seqs[i]];
      for (int32_t p : s.pages) drop_page(p);
      s.pages.clear();
      s.live = false;
      --live_;
      if ((size_t)seqs[i] < seq_hint_) seq_hint_ = (size_t)seqs[i];
    }
    return BookError::none;
  }

  // Moves pages so that the u used ones have the ids 0 .. u - 1: src/dst get
  // the moves, in order of dst.  With fewer than the needed `cap` entries
  // nothing changes; *n is the number needed either way.
  BookError compact(int32_t *src, int32_t *dst, size_t cap, size_t *n) {
    const size_t used = refs_.size() - free_;
    size_t moves = 0;
    for (size_t p = used; p < refs_.size(); ++p) moves += refs_[p] != 0;
    *n = moves;
    if (moves > cap) return BookError::room;
    if (!moves) return BookError::none;
    std::vector<int32_t> to(refs_.size() - used, -1);
    size_t hole = 0, i = 0;
    for (size_t p = used; p < refs_.size(); ++p) {
      if (!refs_[p]) continue;
      while (refs_[hole]) ++hole;
      src[i] = (int32_t)p, dst[i] = (int32_t)hole, ++i;
      to[p - used] = (int32_t)hole;
      refs_[hole] = refs_[p], refs_[p] = 0;
      free_bits_[hole >> 6] &= ~((uint64_t)1 << (hole & 63));
      free_bits_[p >> 6] |= (uint64_t)1 << (p & 63);
    }
    hint_ = used >> 6;
    for (Seq &s : seqs_)
      for (int32_t &p : s.pages)
        if ((size_t)p >= used) p = to[p - used];
    return BookError::none;
  }

 private:
  struct Seq {
    size_t len = 0;
    std::vector<int32_t> pages;
    bool live = false;
    bool counted = false;  // scratch of distinct() and extend(); false between calls
  };

  size_t pages_of(size_t len) const { return (len + rows_ - 1) / rows_; }
  // growing s by `more` rows writes into a page that another sequence lists
  bool shares_tail(const Seq &s, size_t more) const { return more && s.len % rows_ && refs_[s.pages.back()] > 1; }

  BookError distinct(const int32_t *seqs, size_t n) {
    size_t i = 0;
    BookError e = BookError::none;
    for (; i < n; ++i) {
      if (!live(seqs[i])) {
        e = BookError::seq;
        break;
      }
      if (seqs_[seqs[i]].counted) {
        e = BookError::twice;
        break;
      }
      seqs_[seqs[i]].counted = true;
    }
    for (size_t j = 0; j < i; ++j) seqs_[seqs[j]].counted = false;
    return e;
  }

  // entries for n more sequences, so that taking them cannot fail
  void make_room(size_t n) {
    size_t dead = 0;
    for (size_t s = seq_hint_; s < seqs_.size() && dead < n; ++s) dead += !seqs_[s].live;
    if (dead < n) seqs_.resize(seqs_.size() + (n - dead));
  }
  int32_t take_seq() {
    while (seqs_[seq_hint_].live) ++seq_hint_;
    Seq &s = seqs_[seq_hint_];
    s.live = true;
    s.len = 0;
    ++live_;
    return (int32_t)seq_hint_++;
  }

  int32_t take_page() {  // free_ > 0
    while (!free_bits_[hint_]) ++hint_;
    const int b = __builtin_ctzll(free_bits_[hint_]);
    free_bits_[hint_] &= free_bits_[hint_] - 1;
    const size_t p = hint_ * 64 + b;
    refs_[p] = 1;
    --free_;
    return (int32_t)p;
  }
  void drop_page(int32_t p) {
    if (--refs_[p]) return;
    free_bits_[p >> 6] |= (uint64_t)1 << (p & 63);
    if ((size_t)(p >> 6) < hint_) hint_ = p >> 6;
    ++free_;
  }

  size_t rows_;
  std::vector<uint32_t> refs_;  // per page: the sequences that list it
  size_t free_;                 // pages nobody lists
  std::vector<uint64_t> free_bits_;
  size_t hint_ = 0;             // no free page below word hint_
  std::vector<Seq> seqs_;
  size_t live_ = 0, max_seqs_, seq_hint_ = 0;  // no dead sequence below seq_hint_
};

}  // namespace rw
