// Device memory that a context replaces as its calls need more of it.  `A`
// gives and takes the memory: void* alloc(size_t), which throws where there is
// none, and void release(void*), which waits until nothing uses it any more.
#pragma once
#include <cstddef>
#include <cstdint>

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
    if (p) a.release(p);
    p = n;
    bytes = want;
  }
};

// Rows of one size, `extra` bytes for all of them together: at least `least`
// rows, and twice as many as before when they grow, but not more than `most`
// (which every need is within) for either reason.
struct GrowRows {
  void* p = nullptr;
  int rows = 0;
  template <class A>
  void reserve(A& a, int need, int least, int most, size_t row_bytes, size_t extra) {
    if (rows >= need) return;
    int want = rows > 0 ? 2 * rows : least;
    if (want > most) want = most;
    if (want < need) want = need;
    void* n = nullptr;
    try {
      n = a.alloc((size_t)want * row_bytes + extra);
    } catch (...) {
      if (want == need) throw;
      n = a.alloc((size_t)(want = need) * row_bytes + extra);
    }
    if (p) a.release(p);
    p = n;
    rows = want;
  }
};

// What a pass over drafted trees needs: the batch tables, a workspace, and the
// rows that hold the trees' outputs until a path is accepted.  Those come last
// and the epoch, which ends earlier trees, after them: a call that fails here
// leaves every tree of an earlier one as it was.
struct PassNeed {
  int rows, most;
  size_t table_row, table_extra, workspace, tree_row, tree_extra;
};
template <class A>
void reserve_pass(A& a, const PassNeed& n, GrowRows& tables, GrowBuf& ws, GrowRows& tree, uint64_t& epoch) {
  tables.reserve(a, n.rows, 8, n.most, n.table_row, n.table_extra);
  ws.reserve(a, n.workspace);
  tree.reserve(a, n.rows, 64, n.most, n.tree_row, n.tree_extra);
  epoch += 1;
}

}  // namespace rdet
