// rw::ThreadNumber and rw::WorkspacePool::collect (rusty_whisper_amd/csrc/rw_pool.hpp)
// on the CPU, as the library keys the workspace of a stream handle that means
// another stream in every thread: threads at once have buffers of their own,
// a later thread never that of an ended one before it was freed, and the
// buffers of ended threads do not add up.  Built with ThreadSanitizer and with
// AddressSanitizer by tests/test_stream_keys_cpu.py.
#include <algorithm>
#include <atomic>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <set>
#include <thread>
#include <vector>

#include "rw_pool.hpp"

static std::atomic<long> g_live{0};
static int a_alloc(size_t bytes, void **out) {
  *out = malloc(bytes);
  ++g_live;
  return *out ? 0 : -4;
}
static void a_free(void *p) {
  --g_live;
  free(p);
}
using Pool = rw::WorkspacePool<uint64_t>;

// the library's steps for such a handle
static Pool::Slot *take(Pool &pool, size_t bytes) {
  const uint64_t me = rw::ThreadNumber::mine();
  const std::vector<uint64_t> ended = rw::ThreadNumber::take_ended();
  if (!ended.empty())
    pool.collect([&](uint64_t k) { return std::find(ended.begin(), ended.end(), k) != ended.end(); });
  Pool::Slot *s = nullptr;
  return pool.acquire(me, bytes, &s) ? nullptr : s;
}

int main() {
  constexpr int THREADS = 8, ROUNDS = 40;
  std::atomic<int> bad{0};
  auto *pool = new Pool(a_alloc, a_free, 256);
  std::set<uint64_t> numbers;
  std::mutex mu;
  Pool::Slot *mine = take(*pool, 1000);  // this thread's is kept all along
  memset(mine->p, 77, 1000);
  pool->release(mine);
  for (int round = 0; round < ROUNDS; ++round) {
    std::atomic<int> here{0};
    std::vector<std::thread> ts;
    for (int t = 0; t < THREADS; ++t)
      ts.emplace_back([&, t] {
        {
          std::lock_guard<std::mutex> lk(mu);
          if (!numbers.insert(rw::ThreadNumber::mine()).second) ++bad;  // a number given twice
        }
        if (rw::ThreadNumber::mine() != rw::ThreadNumber::mine()) ++bad;
        // all threads have queued their work (let go of their slots) before anyone's is looked at:
        // what is written stands for work that is still to run
        Pool::Slot *s = take(*pool, 500 + 700 * t);
        unsigned char *p = (unsigned char *)s->p;
        memset(p, t + 1, 500);
        pool->release(s);
        ++here;
        while (here < THREADS) std::this_thread::yield();
        for (int i = 0; i < 500; ++i)
          if (p[i] != t + 1) {
            ++bad;
            break;
          }
        s = take(*pool, 100);  // again: the same buffer
        if (s->p != p) ++bad;
        pool->release(s);
      });
    for (auto &th : ts) th.join();
    // this round's, perhaps (their threads have ended since), and this thread's
    if (g_live > 2 * THREADS + 1) ++bad;
  }
  mine = take(*pool, 1000);
  if (g_live != 1) ++bad;
  for (int i = 0; i < 1000; ++i) bad += ((unsigned char *)mine->p)[i] != 77;
  pool->release(mine);
  delete pool;
  printf("bad=%d live=%ld numbers=%zu\n", bad.load(), g_live.load(), numbers.size());
  return bad.load() != 0 || g_live.load() != 0;
}
