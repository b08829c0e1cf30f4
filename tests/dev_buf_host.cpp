// The growing buffers of a context over a host allocator that fails on demand.
#include <cstdint>
#include <map>
#include <stdexcept>

#include "dev_buf.h"

namespace {
struct FakeAlloc {
  std::map<void*, size_t> live;
  uintptr_t next = 4096;
  uint64_t fail = 0;  // bit i: the i-th call from now on fails
  int calls = 0;
  size_t most = 0, held = 0;
  void* alloc(size_t bytes) {
    const bool bad = fail >> calls & 1;
    ++calls;
    if (bad) throw std::runtime_error("no memory");
    void* p = reinterpret_cast<void*>(next);
    next += (bytes + 4095) / 4096 * 4096 + 4096;
    live[p] = bytes;
    held += bytes;
    if (held > most) most = held;
    return p;
  }
  void release(void* p) {
    held -= live.at(p);
    live.erase(p);
  }
  void arm(uint64_t f) {
    fail = f;
    calls = 0;
  }
  // the buffer lies in live memory of at least the size that it claims
  bool holds(const void* p, size_t bytes) const {
    const auto it = live.find(const_cast<void*>(p));
    return bytes == 0 ? true : it != live.end() && it->second >= bytes;
  }
};
}  // namespace

extern "C" {
// 0: after every request of a workspace, failed ones among them, it holds what it claims
int workspace(uint64_t fail_first, uint64_t fail_second) {
  FakeAlloc a;
  rdet::GrowBuf b;
  const size_t needs[] = {1000, 900, 5000, 5000, 5000};
  const uint64_t fails[] = {fail_first, 0, fail_second, 3, 0};
  for (int i = 0; i < 5; ++i) {
    const rdet::GrowBuf before = b;
    a.arm(fails[i]);
    bool failed = false;
    try {
      b.reserve(a, needs[i]);
    } catch (const std::exception&) {
      failed = true;
    }
    if (!a.holds(b.p, b.bytes)) return 1 + i;
    if (failed ? b.p != before.p || b.bytes != before.bytes : b.bytes < needs[i]) return 11 + i;
    if (i == 4 && failed) return 21;
  }
  return 0;
}

// Passes of growing and falling row counts; in the one numbered `victim` the
// allocations of `fail` fail.  0: a failed pass leaves the trees' rows and the
// epoch as they were, and everything holds what it claims.
int passes(int victim, uint64_t fail) {
  FakeAlloc a;
  rdet::GrowRows tables, tree;
  rdet::GrowBuf ws;
  uint64_t epoch = 7;
  const int rows[] = {1, 40, 200, 30, 900, 900, 2000};
  for (int i = 0; i < 7; ++i) {
    const rdet::GrowRows tree0 = tree;
    const uint64_t epoch0 = epoch;
    const rdet::PassNeed n{rows[i], 4096, 4000, 256, (size_t)rows[i] * 3000, 9000, 768};
    a.arm(i == victim ? fail : 0);
    bool failed = false;
    try {
      rdet::reserve_pass(a, n, tables, ws, tree, epoch);
    } catch (const std::exception&) {
      failed = true;
    }
    if (failed && (i != victim || tree.p != tree0.p || tree.rows != tree0.rows || epoch != epoch0)) return 1 + i;
    if (!failed && (epoch != epoch0 + 1 || tree.rows < rows[i] || tables.rows < rows[i] || ws.bytes < n.workspace)) return 11 + i;
    if (!a.holds(tree.p, tree.rows ? (size_t)tree.rows * n.tree_row + n.tree_extra : 0)) return 21 + i;
    if (!a.holds(tables.p, tables.rows ? (size_t)tables.rows * n.table_row + n.table_extra : 0)) return 31 + i;
    if (!a.holds(ws.p, ws.bytes)) return 41 + i;
    if (a.live.size() > 3) return 51 + i;  // nothing superseded stays
  }
  return 0;
}

// Passes that need one row more each time: allocations in all (their number
// grows with the logarithm), or -1 where more than the buffers in use and one
// beside them was ever held.
int growing(int passes, int most) {
  FakeAlloc a;
  rdet::GrowRows tables, tree;
  rdet::GrowBuf ws;
  uint64_t epoch = 0;
  int calls = 0;
  for (int i = 1; i <= passes; ++i) {
    const rdet::PassNeed n{i, most, 4000, 256, (size_t)i * 3000, 9000, 768};
    a.arm(0);
    rdet::reserve_pass(a, n, tables, ws, tree, epoch);
    calls += a.calls;
    if (tree.rows > most || tables.rows > most || a.live.size() != 3) return -1;
  }
  const size_t last = (size_t)tree.rows * 9000 + 768 + (size_t)tables.rows * 4000 + 256 + ws.bytes;
  return a.held == last && a.most <= 2 * last ? calls : -1;
}
}
