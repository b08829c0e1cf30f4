// Attention of a tree of drafted tokens over a KV cache, exact: for every
// node, attention_output_into (det_kernels.rs:340-367) over the rows it sees,
// in the order of their positions: the cache rows of its window, its
// ancestors and itself.
//
//   s[j] = requantize(sum_i q[i] k[j][i])              (wrapping i64)
//   m = max s (the first of equal ones), e[j] = exp_term(s[j], m)
//   w[j] = softmax_weight(e[j], sum e); w[first max] += 1 - sum w
//   out[i] = requantize(sum_j w[j] v[j][i])            (wrapping i64)
//
// The weights are rounded against the row's complete maximum and sum, so the
// scores of all keys come before the first weight: three kernels over a
// scratch of scores.  A key is an index into the sequence's [lo, lo + len):
// cache rows lo .. ctx - 1, then the nodes (key ctx + i).  The order of keys
// is the order of positions along every node's path, because parents come
// before their children.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "det_dev.cuh"
#include "kernels.h"

namespace rdet {
namespace {

__device__ __forceinline__ void ta_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void ta_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... KArgs, typename... Args>
inline void ta_launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

// the sequence of node `node` (nodes of the sequences in order)
__device__ __forceinline__ int seq_of_node(const TreeGroup& g, int node) {
  int s = 0;
  while (s + 1 < g.nseq && g.seq[s + 1].node0 <= node) ++s;
  return s;
}
__device__ __forceinline__ const int32_t* key_row(const TreeSeq& t, int kvh, int key, int d) {
  return key < t.ctx ? t.k + (int64_t)kvh * t.kstride + (int64_t)key * d
                     : t.kt + (int64_t)kvh * t.tstride + (int64_t)(key - t.ctx) * d;
}
__device__ __forceinline__ const int32_t* value_row(const TreeSeq& t, int kvh, int key, int d) {
  return key < t.ctx ? t.v + (int64_t)kvh * t.kstride + (int64_t)key * d
                     : t.vt + (int64_t)kvh * t.tstride + (int64_t)(key - t.ctx) * d;
}
// the lowest position node `mask` (its depth is the number of its ancestors) attends
__device__ __forceinline__ int first_pos(const TreeGroup& g, const TreeSeq& t, uint64_t mask) {
  const int p = t.ctx + __popcll(mask);  // position + 1
  return g.window > 0 && p > g.window ? p - g.window : 0;
}
// whether a node with ancestor mask `mask` and first position `start` attends key `key`
__device__ __forceinline__ bool sees(const TreeGroup& g, const TreeSeq& t, uint64_t mask, int start, int key) {
  if (key < t.ctx) return key >= start;
  const int i = key - t.ctx;
  if (!((mask >> i) & 1)) return false;
  return t.ctx + __popcll(g.mask[t.node0 + i]) - 1 >= start;
}

// scores: one warp per (row, key), lanes over the head's dims
__global__ void __launch_bounds__(256) tree_scores(const __grid_constant__ TreeGroup g) {
  ta_wait();
  ta_go();
  const int row = blockIdx.y, node = row / g.Hq, head = row % g.Hq;
  const TreeSeq& t = g.seq[seq_of_node(g, node)];
  const int kvh = head / (g.Hq / g.Hkv), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int32_t* q = g.q + (int64_t)row * g.d;
  int32_t* sc = static_cast<int32_t*>(g.ws) + t.soff + ((int64_t)(node - t.node0) * g.Hq + head) * t.pad;
  for (int j = blockIdx.x * 8 + warp; j < t.len; j += gridDim.x * 8) {
    const int32_t* k = key_row(t, kvh, t.lo + j, g.d);
    int64_t acc = 0;
    for (int i = lane; i < g.d; i += 32) acc = mac_wide(acc, q[i], k[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) sc[j] = requantize(acc);
  }
}

__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t t = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

// weights in the place of the scores (0 for keys the node does not attend)
__global__ void __launch_bounds__(256) tree_softmax(const __grid_constant__ TreeGroup g) {
  ta_wait();
  ta_go();
  __shared__ int64_t red[8];
  __shared__ uint64_t best[8];
  const int row = blockIdx.x, node = row / g.Hq, head = row % g.Hq, tid = threadIdx.x;
  const TreeSeq& t = g.seq[seq_of_node(g, node)];
  int32_t* sc = static_cast<int32_t*>(g.ws) + t.soff + ((int64_t)(node - t.node0) * g.Hq + head) * t.pad;
  const uint64_t mask = g.mask[node];
  const int start = first_pos(g, t, mask);
  // (value, lowest index first): the node itself is always attended, so the key is never 0
  uint64_t b = 0;
  for (int j = tid; j < t.len; j += blockDim.x)
    if (sees(g, t, mask, start, t.lo + j))
      b = max(b, (uint64_t)((uint32_t)sc[j] ^ 0x80000000u) << 32 | (uint32_t)~j);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
  if ((tid & 31) == 0) best[tid >> 5] = b;
  __syncthreads();
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) b = max(b, best[w]);
  const int32_t m = (int32_t)((uint32_t)(b >> 32) ^ 0x80000000u);
  const int mi = (int)~(uint32_t)b;
  int64_t sum = 0;
  for (int j = tid; j < t.len; j += blockDim.x)
    if (sees(g, t, mask, start, t.lo + j)) sum += exp_term(sc[j], m);
  sum = block_sum(sum, red);
  int64_t wsum = 0;
  for (int j = tid; j < t.len; j += blockDim.x) {
    const int32_t w = sees(g, t, mask, start, t.lo + j) ? softmax_weight(exp_term(sc[j], m), sum) : 0;
    sc[j] = w;
    wsum += w;
  }
  wsum = block_sum(wsum, red);
  __syncthreads();
  if (tid == 0) sc[mi] = add_sat(sc[mi], sub_sat(kOneAct, (int32_t)wsum));
}

// weighted values: one block per row, threads over the head's dims
__global__ void __launch_bounds__(256) tree_values(const __grid_constant__ TreeGroup g) {
  ta_wait();
  ta_go();
  const int row = blockIdx.x, node = row / g.Hq, head = row % g.Hq;
  const TreeSeq& t = g.seq[seq_of_node(g, node)];
  const int kvh = head / (g.Hq / g.Hkv);
  const int32_t* w = static_cast<int32_t*>(g.ws) + t.soff + ((int64_t)(node - t.node0) * g.Hq + head) * t.pad;
  for (int i = threadIdx.x; i < g.d; i += blockDim.x) {
    int64_t acc = 0;
    for (int j = 0; j < t.len; ++j) acc = mac_wide(acc, w[j], value_row(t, kvh, t.lo + j, g.d)[i]);
    g.out[(int64_t)row * g.d + i] = requantize(acc);
  }
}

}  // namespace

size_t tree_attn_plan(TreeGroup& g) {
  int64_t off = 0;
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    // the shallowest node's window is the lowest of the tree
    t.lo = g.window > 0 && t.ctx + 1 > g.window ? std::min(t.ctx, t.ctx + 1 - g.window) : 0;
    t.len = t.ctx - t.lo + t.n;
    t.pad = (t.len + 63) & ~63;
    t.soff = off;
    off += (int64_t)t.pad * t.n * g.Hq;
  }
  return (size_t)off * 4;
}

void launch_tree_attn(const TreeGroup& g, cudaStream_t s) {
  int maxlen = 0;
  for (int i = 0; i < g.nseq; ++i) maxlen = std::max(maxlen, g.seq[i].len);
  const int rows = g.nnode * g.Hq;
  ta_launch(tree_scores, dim3(std::min(64, (maxlen + 7) / 8), rows), dim3(256), 0, s, g);
  ta_launch(tree_softmax, dim3(rows), dim3(256), 0, s, g);
  ta_launch(tree_values, dim3(rows), dim3(256), 0, s, g);
}

}  // namespace rdet
