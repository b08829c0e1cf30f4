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
// Rules on a logits row.  One thread-block cluster per row: its CTAs take
// parts of the vocabulary, and the row's best (value, token) is reduced
// through distributed shared memory, so a call needs no workspace.  A CTA
//   gathers   the history's ids and the biases that fall into its part in a
//             hash table (counts, sums of biases) and marks their tokens in a
//             bit set, reading the history once;
//   computes  the marked tokens (few), one listed slot per thread, so that their
//             loads and the division's long sequence are waited for once, on
//             dense warps;
//   streams   its part without a barrier: every token is copied, masked ones
//             as the lowest value, and the maximum of the unmarked ones found;
//             then the marked tokens' values replace what the stream wrote.
// Bound by memory: a row streams once.  61 rows of 262144 logits under all rules
// and a history of 4096, written out (130 MB): 41 us, 3.2 TB/s, of which the
// stream takes 26; gathering and computing, on every CTA at once, leave the
// memory idle.  (Bringing the CTA's part into L2 meanwhile: 43; half of the
// warps gathering while the others stream: 44.)
// The time goes by the different ids of a history rather than by its length: one
// row of 262144 takes 17 us under 32768 ids of 8000 different ones, 40 under
// 131072 of 8000, 12 under 8192 ids all over the vocabulary, but 102 under 16384
// of those and 790 under 131072, where the CTAs' tables overflow (61 rows: 84, 224, 52, 541 and 3412).
// ---------------------------------------------------------------------------

__device__ __forceinline__ int32_t clamp_i32(int64_t v) {
  return v > INT32_MAX ? INT32_MAX : (v < INT32_MIN ? INT32_MIN : (int32_t)v);
}
// larger value wins, ties keep the lower token; 0 stands for no token
__device__ __forceinline__ uint64_t rule_key(int32_t v, uint32_t t) {
  return (uint64_t)((uint32_t)v ^ 0x80000000u) << 32 | (uint32_t)~t;
}

// The CTAs of a row take its chunks of 512 tokens in turn, so that the low ids,
// which tokenizers give the frequent tokens, spread over all of them, in
// batches of 65536 tokens (li: a token's number within its CTA's batch).  The
// stream takes four 16-byte pieces per thread and step.  Where a batch marks
// more tokens than the table holds, it is computed after the stream, block by
// block of as many tokens as there are slots, each of which reads the history again.
constexpr int kRuleVec = 4;
constexpr uint32_t kRuleChunk = 512;
constexpr uint32_t kRuleBatch = 65536, kRuleSlots = 2048, kRuleProbes = 32, kRuleEmpty = 0xffffffffu;
struct RuleSmem {
  unsigned long long bias[kRuleSlots];  // sums of the biases, exact
  uint32_t key[kRuleSlots];             // li, or empty
  uint32_t count[kRuleSlots];
  uint32_t marked[kRuleBatch / 32];
  uint16_t list[kRuleSlots];            // the slots in use, in any order
};

// Loads of rows that are touched once, and of the words of rules.  None is .nc:
// this grid may be resident already while the grid before it writes what it
// reads, so only coherent loads behind the wait see it.
__device__ __forceinline__ void ld_stream(int4& v, const int32_t* p, bool on) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p ld.global.L1::no_allocate.v4.s32 {%0, %1, %2, %3}, [%4];\n}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"((int)on));
}
__device__ __forceinline__ void ld_word(uint32_t& v, const uint32_t* p, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p ld.global.u32 %0, [%1];\n}"
               : "+r"(v)
               : "l"(p), "r"((int)on));
}

template <int THREADS, int ROWS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logit_rules_kernel(const __grid_constant__ RuleRowsOf<ROWS> rs,
                                                                             uint32_t vocab, uint32_t* tokens) {
  constexpr uint32_t kStep = THREADS * 4 * kRuleVec;
  extern __shared__ __align__(16) unsigned char rule_raw[];
  RuleSmem& sm = *reinterpret_cast<RuleSmem*>(rule_raw);
  __shared__ uint64_t best[THREADS / 32], cta_best;
  __shared__ uint32_t s_over, s_used;
  cg::cluster_group cl = cg::this_cluster();
  const uint32_t CL = cl.num_blocks(), rank = cl.block_rank();  // CL: a power of two
  const int tid = threadIdx.x, row = blockIdx.y;
  const int32_t* const logits = rs.row[row].logits;
  int32_t* const out = rs.row[row].out;
  const uint32_t* const allow = rs.row[row].allow;
  const uint32_t* const history = rs.row[row].history;
  const uint32_t* const bias_ids = rs.row[row].bias_ids;
  const uint32_t hlen = rs.row[row].history_len, nbias = rs.row[row].n_bias;
  do_wait();
  do_go();
  const bool any = hlen > 0 || nbias > 0 || rs.row[row].has_path;
  const bool wide = ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  auto allowed = [&](uint32_t w) {
    uint32_t v = 0xffffffffu;
    ld_word(v, allow + w, allow != nullptr);
    return v;
  };
  uint64_t b = 0;
  // the thread's first maximum of unmarked tokens (they come in ascending
  // order), and the first of them where all are at the lowest value
  int32_t bv = INT32_MIN;
  uint32_t bt = 0xffffffffu, lowest = 0xffffffffu;
  const uint32_t share = 31 - __clz((int)CL);  // log2 of the row's CTAs
  const uint32_t chunks = (vocab + kRuleChunk - 1) / kRuleChunk;
  for (uint32_t c0 = 0; (c0 << share) + rank < chunks; c0 += kRuleBatch / kRuleChunk) {  // the batch's first chunk
    auto token = [&](uint32_t li) { return (((c0 + li / kRuleChunk) << share) + rank) * kRuleChunk + li % kRuleChunk; };
    // f(li) for the ids of the row's history and path, g(li, value) for its biases
    auto each = [&](auto&& f, auto&& g) {
      auto local = [&](uint32_t id, auto&& h) {
        const uint32_t c = id / kRuleChunk, li = ((c >> share) - c0) * kRuleChunk + id % kRuleChunk;
        if (id < vocab && (c & (CL - 1)) == rank && (c >> share) >= c0 && li < kRuleBatch) h(li);
      };
      // a thread's biases and eight of its ids in flight together
      uint32_t bi[2] = {kRuleEmpty, kRuleEmpty}, bw[2] = {0, 0};  // (empty: past every vocabulary)
      const uint32_t* const bias_values = reinterpret_cast<const uint32_t*>(rs.row[row].bias_values);
      for (uint32_t k0 = 0; k0 < max(hlen, nbias); k0 += 8 * THREADS) {
        uint32_t id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          id[k] = kRuleEmpty;
          ld_word(id[k], history + k0 + tid + k * THREADS, k0 + tid + k * THREADS < hlen);
        }
        if (k0 == 0) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            ld_word(bi[k], bias_ids + tid + k * THREADS, tid + k * THREADS < nbias);
            ld_word(bw[k], bias_values + tid + k * THREADS, tid + k * THREADS < nbias);
          }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) local(id[k], f);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) local(bi[k], [&](uint32_t li) { g(li, (int32_t)bw[k]); });
      for (uint32_t k = tid + 2 * THREADS; k < nbias; k += THREADS)
        local(bias_ids[k], [&](uint32_t li) { g(li, (int32_t)bias_values[k]); });
      if (tid < ROWS && (rs.row[row].path[tid >> 6] >> (tid & 63) & 1)) local(rs.row[tid].token, f);
    };
    // the slot of li; the table's load is low, so few probes reach it
    auto slot = [&](uint32_t li) {
      uint32_t h = (li * 40503u >> 5) % kRuleSlots;
      for (uint32_t n = 0; n < kRuleProbes; ++n, h = (h + 1) % kRuleSlots) {
        const uint32_t old = atomicCAS(&sm.key[h], kRuleEmpty, li);
        if (old == kRuleEmpty) sm.list[atomicAdd(&s_used, 1u)] = (uint16_t)h;
        if (old == kRuleEmpty || old == li) return h;
      }
      s_over = 1;
      return kRuleSlots;
    };
    auto clear = [&] {
      for (uint32_t i = tid; i < kRuleSlots; i += THREADS) {
        sm.bias[i] = 0;
        sm.key[i] = kRuleEmpty;
        sm.count[i] = 0;
      }
    };
    // token t with the rules that slot h holds; false where it is masked
    auto compute = [&](uint32_t t, uint32_t h, int32_t& x) {
      x = logits[t];
      const uint32_t ok = allowed(t >> 5) >> (t & 31), c = sm.count[h];
      const int64_t bias = (int64_t)sm.bias[h];
      if (!(ok & 1)) return false;
      if (c) {
        const int32_t rep = rs.row[row].repetition;
        x = x > 0 ? div_act(x, rep) : mul_sat(x, rep);
        x = sub_sat(sub_sat(x, clamp_i32((int64_t)rs.row[row].frequency * (int64_t)c)), rs.row[row].presence);
      }
      x = add_sat(x, clamp_i32(bias));
      b = max(b, rule_key(x, t));
      return true;
    };
    if (any) {
      clear();
      for (uint32_t i = tid; i < kRuleBatch / 32; i += THREADS) sm.marked[i] = 0;
      if (tid == 0) s_over = s_used = 0;
      __syncthreads();
      auto mark = [&](uint32_t li) { atomicOr(&sm.marked[li >> 5], 1u << (li & 31)); };
      each(
          [&](uint32_t li) {
            mark(li);
            const uint32_t h = slot(li);
            if (h < kRuleSlots) atomicAdd(&sm.count[h], 1u);
          },
          [&](uint32_t li, int32_t value) {
            mark(li);
            const uint32_t h = slot(li);
            if (h < kRuleSlots) atomicAdd(&sm.bias[h], (unsigned long long)(long long)value);
          });
      __syncthreads();
    }
    int4 v[kRuleVec] = {};
    auto load = [&](uint32_t l0) {
#pragma unroll
      for (int k = 0; k < kRuleVec; ++k) {
        const uint32_t li = l0 + 4 * (tid + k * THREADS), t = token(li);
        ld_stream(v[k], logits + t, wide && li < kRuleBatch && t + 4 <= vocab && t < vocab);
      }
    };
    load(0);
    if (any && !s_over)
      for (uint32_t k = tid; k < s_used; k += THREADS) {
        const uint32_t h = sm.list[k];
        int32_t x;
        if (compute(token(sm.key[h]), h, x)) sm.count[h] = (uint32_t)x;
        else sm.key[h] = kRuleEmpty;  // masked: stays what the stream writes
      }
    auto unmarked = [&](uint32_t li) { return any ? ~sm.marked[li >> 5] : 0xffffffffu; };
    for (uint32_t l0 = 0; l0 < kRuleBatch && token(l0) < vocab; l0 += kStep) {
#pragma unroll
      for (int k = 0; k < kRuleVec; ++k) {
        const uint32_t li = l0 + 4 * (tid + k * THREADS), t = token(li);
        if (wide && t < vocab && t + 4 <= vocab) {
          const uint32_t s = t & 31, ok = allowed(t >> 5) >> s, plain = ok & (unmarked(li) >> s) & 15u;
          if (!(ok & 1)) v[k].x = INT32_MIN;
          if (!(ok & 2)) v[k].y = INT32_MIN;
          if (!(ok & 4)) v[k].z = INT32_MIN;
          if (!(ok & 8)) v[k].w = INT32_MIN;
          if (out) __stcs(reinterpret_cast<int4*>(out + t), v[k]);
          const int32_t x = plain & 1 ? v[k].x : INT32_MIN, y = plain & 2 ? v[k].y : INT32_MIN,
                        z = plain & 4 ? v[k].z : INT32_MIN, u = plain & 8 ? v[k].w : INT32_MIN;
          const int32_t m = max(max(x, y), max(z, u));
          if (m > bv) {
            bv = m;
            bt = t + (x == m ? 0 : y == m ? 1 : z == m ? 2 : 3);
          }
          if (plain && lowest == 0xffffffffu) lowest = t + __ffs(plain) - 1;
        } else if (t < vocab) {  // the row's last tokens, or a row that is not 16-byte aligned
          for (uint32_t e = 0; e < 4 && t + e < vocab; ++e) {
            int32_t x = logits[t + e];
            const uint32_t s = (t + e) & 31;
            if (!(allowed((t + e) >> 5) >> s & 1)) x = INT32_MIN;
            else if (unmarked(li) >> s & 1) b = max(b, rule_key(x, t + e));
            if (out) out[t + e] = x;
          }
        }
      }
      load(l0 + kStep);
    }
    if (any) {
      __syncthreads();  // the marked tokens' values replace what the stream wrote
      if (!s_over) {
        for (uint32_t k = tid; out && k < s_used; k += THREADS) {
          const uint32_t h = sm.list[k];
          if (sm.key[h] != kRuleEmpty) out[token(sm.key[h])] = (int32_t)sm.count[h];
        }
        __syncthreads();
      } else {
        for (uint32_t block = 0; block < kRuleBatch; block += kRuleSlots) {
          __syncthreads();
          clear();
          __syncthreads();
          each(
              [&](uint32_t li) {
                if (li - block < kRuleSlots) atomicAdd(&sm.count[li - block], 1u);
              },
              [&](uint32_t li, int32_t value) {
                if (li - block < kRuleSlots) atomicAdd(&sm.bias[li - block], (unsigned long long)(long long)value);
              });
          __syncthreads();
          for (uint32_t h = tid; h < kRuleSlots; h += THREADS)
            if ((sm.marked[(block + h) >> 5] >> (h & 31)) & 1) {
              int32_t x;
              const uint32_t t = token(block + h);
              if (compute(t, h, x) && out) out[t] = x;
            }
        }
        __syncthreads();
      }
    }
  }
  if (bt != 0xffffffffu) b = max(b, rule_key(bv, bt));
  else if (lowest != 0xffffffffu) b = max(b, rule_key(INT32_MIN, lowest));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
  if ((tid & 31) == 0) best[tid >> 5] = b;
  __syncthreads();
  if (tid < 32) {
    b = tid < THREADS / 32 ? best[tid] : 0;
#pragma unroll
    for (int o = THREADS / 64; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    if (tid == 0) cta_best = b;
  }
  cl.sync();
  if (rank == 0 && tid < 32) {
    b = tid < (int)CL ? *cl.map_shared_rank(&cta_best, tid) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) b = max(b, __shfl_xor_sync(0xffffffffu, b, o));
    if (tid == 0) tokens[row] = b ? ~(uint32_t)b : 0xffffffffu;
  }
  cl.sync();  // every CTA's shared memory stays until it has been read
}

// ---------------------------------------------------------------------------
// Accepted rows.  A thread moves one column (16 bytes, or one value where
// head_dim or an address is not a multiple of 16 bytes) of every row of the
// path, in order; one CTA a move.  A draft that lies in the cache itself is
// safe: path[i] >= i and the path increases, so row i is written after it was
// read and after every row before it.  Bound by its start and one chain of
// loads: 768 moves of about seven rows (25.7 MB both ways) take 5.1 us, 48
// moves 1.9.
// ---------------------------------------------------------------------------
template <typename T, typename M>
__device__ __forceinline__ void move_rows(const M& m, const CommitMove& v, int cols) {
  T* dst = reinterpret_cast<T*>(v.cache);
  const T* src = reinterpret_cast<const T*>(v.draft);
  const int n = m.len[v.path];
  for (int c = threadIdx.x; c < (int)(v.kv_heads_1 + 1) * cols; c += blockDim.x) {
    const int64_t h = c / cols, x = c % cols;
    for (int i = 0; i < n; ++i)
      dst[(h * v.cap + v.context + i) * cols + x] = src[(h * v.draft_cap + m.node[v.path][i]) * cols + x];
  }
}
template <int M, int P>
__global__ void __launch_bounds__(256) tree_commit_kernel(const __grid_constant__ CommitMovesOf<M, P> m) {
  do_wait();
  do_go();
  const CommitMove& v = m.mv[blockIdx.x];
  const int d = v.head_dim_1 + 1;
  const bool wide = d % 4 == 0 && ((reinterpret_cast<uintptr_t>(v.cache) | reinterpret_cast<uintptr_t>(v.draft)) & 15) == 0;
  if (wide) move_rows<int4>(m, v, d / 4);
  else move_rows<int32_t>(m, v, d);
}

}  // namespace

template <int THREADS, int ROWS>
static void rules_attr() {
  cudaFuncSetAttribute(logit_rules_kernel<THREADS, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                       (int)sizeof(RuleSmem));
  cudaFuncSetAttribute(logit_rules_kernel<THREADS, ROWS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
}
void draft_ops_init() {
  rules_attr<256, kRuleRows>();
  rules_attr<1024, kRuleFew>();
}

template <int THREADS, int ROWS>
static void rules_launch(const RuleRowsOf<ROWS>& r, int rows, uint32_t vocab, uint32_t* tokens, int most, cudaStream_t s) {
  const int tiles = (int)((vocab + THREADS * 16 - 1) / (THREADS * 16));
  int CL = 1;
  while (CL < most && CL < tiles) CL *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CL, rows, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
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
  cudaLaunchKernelEx(&cfg, logit_rules_kernel<THREADS, ROWS>, r, vocab, tokens);
}

// Few rows (16 CTAs each at most one an SM) take the largest clusters (sixteen
// CTAs) of large CTAs: one row of 262144 logits under a history of 513 takes
// 7.7 us (512 threads and eight CTAs a row: 9.7).  Many rows fill the GPU with
// small CTAs, four of them an SM.
void launch_logit_rules(const RuleRows& r, int rows, uint32_t vocab, uint32_t* tokens, cudaStream_t s) {
  static_assert(kRuleFew == 148 / 16, "one CTA an SM");
  if (rows <= kRuleFew) {
    RuleRowsOf<kRuleFew> few;
    std::copy(r.row, r.row + rows, few.row);
    rules_launch<1024, kRuleFew>(few, rows, vocab, tokens, 16, s);
  } else {
    rules_launch<256, kRuleRows>(r, rows, vocab, tokens, 8, s);
  }
}

template <int M, int P>
static void commit_launch(const CommitMovesOf<M, P>& m, int moves, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(moves, 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, tree_commit_kernel<M, P>, m);
}
void launch_tree_commit(const CommitMoves& m, int moves, int paths, cudaStream_t s) {
  if (moves <= kCommitFewMoves && paths <= kCommitFewPaths) {
    CommitMovesOf<kCommitFewMoves, kCommitFewPaths> few;
    std::copy(m.mv, m.mv + moves, few.mv);
    std::copy(m.len, m.len + paths, few.len);
    memcpy(few.node, m.node, sizeof(m.node[0]) * (size_t)paths);
    commit_launch(few, moves, s);
  } else {
    commit_launch(m, moves, s);
  }
}

}  // namespace rdet
