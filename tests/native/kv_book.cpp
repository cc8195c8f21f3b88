// Random histories of rw::KvBook (rusty_whisper_amd/csrc/rw_kvbook.hpp) on the
// CPU: after every call each page's holders are counted from the sequences'
// lists, and a page is free exactly if nobody lists it.  Built with
// AddressSanitizer and UBSan by tests/test_kv_book_cpu.py.
#include <cstdio>
#include <random>
#include <set>
#include <vector>

#include "rw_kvbook.hpp"

using rw::BookError;
using rw::KvBook;

int main() {
  long bad = 0, done = 0;
  for (unsigned seed = 0; seed < 20; ++seed) {
    std::mt19937 rng(seed);
    const size_t P = 16 << (seed % 3), pages = 1 + rng() % 300, max_seqs = 1 + rng() % 40;
    KvBook b(pages, P, max_seqs);
    for (int it = 0; it < 3000; ++it) {
      std::vector<int32_t> live;
      for (int32_t s = 0; s < (int32_t)max_seqs; ++s)
        if (b.live(s)) live.push_back(s);
      std::vector<int32_t> pick;
      for (int32_t s : live)
        if (rng() % 3 == 0) pick.push_back(s);
      std::vector<int32_t> out(max_seqs + 4), src(pages + 4), dst(pages + 4);
      std::vector<size_t> more(pick.size());
      for (size_t &m : more) m = rng() % 4 ? rng() % 3 : rng() % (4 * P);
      size_t n = 0;
      BookError e = BookError::none;
      switch (rng() % 7) {
        case 0: e = b.add(rng() % 4, out.data()); break;
        case 1: e = b.fork(pick.data(), pick.size(), out.data()); break;
        case 2: case 3: e = b.extend(pick.data(), pick.size(), more.data(), src.data(), dst.data(), &n); break;
        case 4: if (!live.empty()) e = b.truncate(live[0], b.len(live[0]) / 2); break;
        case 5: if (rng() % 4 == 0) e = b.release(pick.data(), pick.size()); break;
        default: e = b.compact(src.data(), dst.data(), src.size(), &n); break;
      }
      done += e == BookError::none;
      std::vector<int> held(pages, 0);
      size_t used = 0, count = 0;
      for (int32_t s = 0; s < (int32_t)max_seqs; ++s) {
        if (!b.live(s)) continue;
        ++count;
        if (b.pages(s).size() != (b.len(s) + P - 1) / P) ++bad;
        std::set<int32_t> seen;
        for (int32_t p : b.pages(s)) {
          if (p < 0 || (size_t)p >= pages || !seen.insert(p).second) ++bad;
          else if (!held[p]++) ++used;
        }
      }
      if (used + b.free_pages() != pages || count != b.n_seqs()) ++bad;
    }
  }
  printf("done=%ld bad=%ld\n", done, bad);
  return bad != 0;
}
