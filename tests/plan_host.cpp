// The tree attention's launch plan of a group, from the library itself.
#include "kernels.h"

extern "C" long long plan(int nseq, const int* ctx, const int* nodes, int heads, int kv, int d, int window, int* out) {
  static rdet::TreeGroup g;
  g = rdet::TreeGroup{};
  for (int i = 0; i < nseq; ++i) {
    g.seq[i].ctx = ctx[i];
    g.seq[i].n = nodes[i];
    g.seq[i].node0 = g.nnode;
    g.nnode += nodes[i];
  }
  g.nseq = nseq;
  g.Hq = heads;
  g.Hkv = kv;
  g.d = d;
  g.window = window;
  const size_t bytes = rdet::tree_attn_plan(g);
  int splits = 0;
  for (int i = 0; i < nseq; ++i) splits = g.seq[i].splits > splits ? g.seq[i].splits : splits;
  const int v[] = {g.nr, g.qk_tiles, splits, g.ex_chunks, g.qk_items, g.pv_items};
  for (int i = 0; i < 6; ++i) out[i] = v[i];
  return (long long)bytes;
}
