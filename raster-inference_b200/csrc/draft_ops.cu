// The other operators that verify drafted tokens: rules on logits rows with
// the greedy token under them, and the move of an accepted path's K/V rows
// into the caches.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "det_dev.cuh"
#include "kernels.h"

namespace rdet {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ void do_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void do_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------
// Rules on a logits row.  One thread-block cluster per row: CTA r takes the
// tiles r, r + CL, ... of the vocabulary and the row's best (value, token) is
// reduced through distributed shared memory, so a call needs no workspace.
// A tile's tokens with a history count or a bias ("special" ones, few) are
// marked in a bit set while the counts are taken; the stream over the tile
// passes the others through, and the special ones are then computed one per
// thread, so that the division's long sequence runs on dense warps only.
// ---------------------------------------------------------------------------
constexpr int kRuleThreads = 512;
constexpr int kRuleTile = 16384;  // tokens of one tile: a 64 KB count table

__device__ __forceinline__ int32_t clamp_i32(int64_t v) {
  return v > INT32_MAX ? INT32_MAX : (v < INT32_MIN ? INT32_MIN : (int32_t)v);
}
// larger value wins, ties keep the lower token; 0 stands for no token
__device__ __forceinline__ uint64_t rule_key(int32_t v, uint32_t t) {
  return (uint64_t)((uint32_t)v ^ 0x80000000u) << 32 | (uint32_t)~t;
}

struct RuleSmem {
  uint32_t count[kRuleTile];
  uint32_t special[kRuleTile / 32];  // tokens with a count or a bias
  uint32_t biased[kRuleTile / 32];
  uint16_t list[kRuleTile];          // the special tokens, in any order
};

__global__ void __launch_bounds__(kRuleThreads) logit_rules_kernel(const __grid_constant__ RuleRows rs, uint32_t vocab,
                                                                  uint32_t* tokens) {
  extern __shared__ __align__(16) unsigned char rule_raw[];
  RuleSmem& sm = *reinterpret_cast<RuleSmem*>(rule_raw);
  __shared__ uint64_t best[kRuleThreads / 32], cta_best;
  __shared__ uint32_t nspecial;
  cg::cluster_group cl = cg::this_cluster();
  const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int tid = threadIdx.x, row = blockIdx.y;
  const RuleRow& r = rs.row[row];
  do_wait();
  do_go();
  const bool hist = r.history_len > 0 || r.token != 0xffffffffu || r.parent >= 0;
  const bool any = hist || r.n_bias > 0;
  uint64_t b = 0;
  for (uint32_t t0 = (uint32_t)rank * kRuleTile; t0 < vocab; t0 += (uint32_t)CL * kRuleTile) {
    const uint32_t nt = min((uint32_t)kRuleTile, vocab - t0);
    if (any) {
      __syncthreads();  // the previous tile's tables are no longer read
      for (int i = tid; i < kRuleTile / 4; i += kRuleThreads)
        reinterpret_cast<uint4*>(sm.count)[i] = make_uint4(0, 0, 0, 0);
      for (int i = tid; i < kRuleTile / 32; i += kRuleThreads) sm.special[i] = sm.biased[i] = 0;
      if (tid == 0) nspecial = 0;
      __syncthreads();
      auto mark = [&](uint32_t i) {
        if (!(atomicOr(&sm.special[i >> 5], 1u << (i & 31)) & (1u << (i & 31))))
          sm.list[atomicAdd(&nspecial, 1u)] = (uint16_t)i;
      };
      for (uint32_t k = tid; k < r.history_len; k += kRuleThreads) {
        const uint32_t i = r.history[k] - t0;
        if (i < nt) {
          atomicAdd(&sm.count[i], 1u);
          mark(i);
        }
      }
      if (tid == 0)  // the row's own token and its ancestors'
        for (int p = row; p >= 0; p = rs.row[p].parent) {
          const uint32_t tok = rs.row[p].token;
          if (tok != 0xffffffffu && tok - t0 < nt) {
            atomicAdd(&sm.count[tok - t0], 1u);
            mark(tok - t0);
          }
        }
      for (uint32_t k = tid; k < r.n_bias; k += kRuleThreads) {
        const uint32_t i = r.bias_ids[k] - t0;
        if (i < nt) {
          atomicOr(&sm.biased[i >> 5], 1u << (i & 31));
          mark(i);
        }
      }
      __syncthreads();
    }
    for (uint32_t i = tid; i < nt; i += kRuleThreads) {
      int32_t v = r.logits[t0 + i];
      const bool ok = !r.allow || ((r.allow[(t0 + i) >> 5] >> ((t0 + i) & 31)) & 1);
      if (!ok) v = INT32_MIN;
      else if (!any || !((sm.special[i >> 5] >> (i & 31)) & 1)) b = max(b, rule_key(v, t0 + i));
      if (r.out) r.out[t0 + i] = v;
    }
    if (any) {
      __syncthreads();  // the special tokens' values replace what the stream wrote
      for (uint32_t k = tid; k < nspecial; k += kRuleThreads) {
        const uint32_t i = sm.list[k], t = t0 + i;
        if (r.allow && !((r.allow[t >> 5] >> (t & 31)) & 1)) continue;
        int32_t v = r.logits[t];
        const uint32_t c = sm.count[i];
        if (c) {
          v = v > 0 ? div_act(v, r.repetition) : mul_sat(v, r.repetition);
          v = sub_sat(sub_sat(v, clamp_i32((int64_t)r.frequency * (int64_t)c)), r.presence);
        }
        if ((sm.biased[i >> 5] >> (i & 31)) & 1) {
          int64_t s = 0;
          for (uint32_t j = 0; j < r.n_bias; ++j)
            if (r.bias_ids[j] == t) s += r.bias_values[j];
          v = add_sat(v, clamp_i32(s));
        }
        b = max(b, rule_key(v, t));
        if (r.out) r.out[t] = v;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
  if ((tid & 31) == 0) best[tid >> 5] = b;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kRuleThreads / 32; ++w) b = max(b, best[w]);
    cta_best = b;
  }
  cl.sync();
  if (rank == 0 && tid == 0) {
    for (int c = 1; c < CL; ++c) b = max(b, *cl.map_shared_rank(&cta_best, c));
    tokens[row] = b ? ~(uint32_t)b : 0xffffffffu;
  }
  cl.sync();  // every CTA's shared memory stays until it has been read
}

// ---------------------------------------------------------------------------
// Accepted rows.  A thread moves one column (16 bytes, or one value where
// head_dim or an address is not a multiple of 16 bytes) of every row of the
// path, in order.  A draft that lies in the cache itself is safe: path[i] >= i
// and the path increases, so row i is written after it was read and after
// every row before it.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void move_rows(const CommitMoves& m, const CommitMove& v, int cols) {
  T* dst = reinterpret_cast<T*>(v.cache);
  const T* src = reinterpret_cast<const T*>(v.draft);
  const int n = m.len[v.path];
  for (int64_t c = threadIdx.x + (int64_t)blockIdx.x * blockDim.x; c < (int64_t)v.kv_heads * cols;
       c += (int64_t)gridDim.x * blockDim.x) {
    const int64_t h = c / cols, x = c % cols;
    for (int i = 0; i < n; ++i)
      dst[(h * v.cap + v.context + i) * cols + x] = src[(h * v.draft_cap + m.node[v.path][i]) * cols + x];
  }
}
__global__ void __launch_bounds__(256) tree_commit_kernel(const __grid_constant__ CommitMoves m) {
  do_wait();
  do_go();
  const CommitMove& v = m.mv[blockIdx.y];
  const bool wide = v.head_dim % 4 == 0 && ((reinterpret_cast<uintptr_t>(v.cache) | reinterpret_cast<uintptr_t>(v.draft)) & 15) == 0;
  if (wide) move_rows<int4>(m, v, v.head_dim / 4);
  else move_rows<int32_t>(m, v, v.head_dim);
}

}  // namespace

void draft_ops_init() {
  cudaFuncSetAttribute(logit_rules_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(RuleSmem));
}

void launch_logit_rules(const RuleRows& r, int rows, uint32_t vocab, uint32_t* tokens, cudaStream_t s) {
  const int tiles = (int)((vocab + kRuleTile - 1) / kRuleTile);
  int CL = 1;
  while (CL < 8 && CL < tiles) CL *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CL, rows, 1);
  cfg.blockDim = dim3(kRuleThreads, 1, 1);
  cfg.dynamicSmemBytes = sizeof(RuleSmem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CL;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, logit_rules_kernel, r, vocab, tokens);
}

void launch_tree_commit(const CommitMoves& m, int moves, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1, moves, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, tree_commit_kernel, m);
}

}  // namespace rdet
