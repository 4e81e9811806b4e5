// Buffers of threads' streams (csrc/scratch.h): free for other streams when the thread has ended, never before.
#include "scratch.h"

#include <cstdio>
#include <cstdlib>
#include <memory>
#include <set>

using tinyoai::ScratchPool;

#define CHECK(x)                                           \
  do {                                                     \
    if (!(x)) {                                            \
      std::printf("line %d: %s\n", __LINE__, #x);          \
      std::exit(1);                                        \
    }                                                      \
  } while (0)

static std::set<void *> live;
static void *alloc(size_t) {
  void *p = std::malloc(16);
  live.insert(p);
  return p;
}
static void give(void *p) {
  CHECK(live.erase(p) == 1);
  std::free(p);
}

int main() {
  const void *own = reinterpret_cast<const void *>(uintptr_t(2));  // one handle for each thread's stream
  auto stream = [](int i) { return reinterpret_cast<const void *>(uintptr_t(64 * (i + 1))); };
  {
    ScratchPool p;
    // threads one after another, more of them than there are buffers: one buffer
    std::set<void *> used;
    for (uint64_t i = 1; i <= 40; i++) {
      const auto thread = std::make_shared<int>();
      const std::weak_ptr<const void> life = thread;
      const ScratchPool::Lease a = p.eager(own, i, 100, alloc, &life), b = p.eager(own, i, 90, alloc, &life);
      CHECK(a.ptr == b.ptr && !a.shared && !b.shared);
      used.insert(a.ptr);
    }
    CHECK(used.size() == 1 && live.size() == 1);
    // eight that live: each its own; the ninth shares, and so does a stream
    std::shared_ptr<int> threads[9];
    std::weak_ptr<const void> lives[9];
    void *ptr[9];
    used.clear();
    for (int i = 0; i < 9; i++) {
      threads[i] = std::make_shared<int>();
      lives[i] = threads[i];
      const ScratchPool::Lease l = p.eager(own, 100 + i, 100, alloc, &lives[i]);
      CHECK(l.shared == (i == 8));
      used.insert(ptr[i] = l.ptr);
    }
    CHECK(used.size() == 9 && p.eager(stream(0), 0, 100, alloc).shared);
    // one ends: a stream takes its buffer, also for a larger call, and keeps it; the others keep theirs
    threads[3].reset();
    const ScratchPool::Lease s = p.eager(stream(0), 0, 100, alloc);
    CHECK(!s.shared && s.ptr == ptr[3] && p.eager(stream(1), 0, 100, alloc).shared);
    threads[5].reset();
    const ScratchPool::Lease t = p.eager(stream(1), 0, 500, alloc);
    CHECK(!t.shared && !used.count(t.ptr) && live.count(ptr[5]));
    for (int i : {0, 1, 2, 4, 6, 7}) CHECK(p.eager(own, 100 + i, 100, alloc, &lives[i]).ptr == ptr[i]);
    CHECK(p.eager(stream(0), 0, 100, alloc).ptr == s.ptr && p.eager(stream(1), 0, 400, alloc).ptr == t.ptr);
    // a stream's buffer is nobody else's, however long it is not used
    CHECK(p.eager(own, 108, 100, alloc, &lives[8]).shared);
    p.clear(give);
    CHECK(live.empty());
  }
  std::printf("ok\n");
  return 0;
}
