// Device memory that a context replaces as its calls need more of it.  `A`
// gives the memory: void* alloc(size_t), which throws where there is none.
#pragma once
#include <cstddef>

namespace rdet {

// A workspace: nothing in it outlives the call that uses it.
struct GrowBuf {
  void* p = nullptr;
  size_t bytes = 0;
  // At least `need` bytes, doubled so that growing calls replace it rarely, or
  // just `need` where twice that is not to be had.  After a failure the buffer
  // is the old one with its own size.
  template <class A>
  void reserve(A& a, size_t need) {
    if (bytes >= need) return;
    size_t want = 2 * need;
    void* n = nullptr;
    try {
      n = a.alloc(want);
    } catch (...) {
      n = a.alloc(want = need);
    }
    p = n;
    bytes = want;
  }
};

}  // namespace rdet
