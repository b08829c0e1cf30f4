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
// A weight is rounded against the row's complete maximum and sum, so no
// running softmax is exact: the scores of all keys come before the first exp
// term, and all terms before the first weight.  Three kernels over a scratch,
// coupled by programmatic dependent launch: scores with each block's row
// maxima (tensor cores), softmax (CUDA cores), weighted values (tensor cores).
// The residual 1 - sum w is a term of its own, added with the first maximum's
// value where the sums are rounded.  A key is an index into the sequence's [lo, lo + len): cache rows lo .. ctx - 1,
// then the nodes (key ctx + i).  The order of keys is the order of positions
// along every node's path, because parents come before their children.
//
// Digits.  The tensor cores multiply signed bytes.  Queries and weights are
// split into balanced base-256 digits, x = sum_a 256^a x_a with x_a in
// [-128, 127]: the bytes of (x + 0x80808080) ^ 0x80808080, for every i32 up to
// 0x7f7f7f7f (a block with a larger query value takes the direct wrapping i64
// sums).  Keys and values, of which there are far more, take the cheapest
// split: their bytes as they are, the three lower ones with the top bit
// flipped, so that k = sum_b 256^b k_b + 0x808080 for every i32.  Then
//   sum_i q k = sum_{a,b} 256^(a+b) sum_i q_a k_b + 0x808080 sum_i q
//   sum_j w v = sum_{a,b} 256^(a+b) sum_j w_a v_b + 0x808080 sum_j w,
// each correction one number a query row.
//
// Scores.  The keys of a 128-key tile are the MMA's M rows, one operand A per
// key byte b; operand B stacks the digits of NR query rows (rows a * NR + r).
// The MMA of key byte b accumulates at TMEM column b * NR, so column block g
// (columns [g NR, (g + 1) NR)) sums exactly the products of shift 8 g: seven
// blocks, each at most 4 * 2^14 * 512 = 2^25 in magnitude, exact in s32.
// A query row is a (node, head of the KV head's group); all of them read a
// key tile at once, so the cache streams once per NR rows.  Keys rather than
// query rows are the MMA's M: seven column blocks of NR leave TMEM room for
// operand A, and a lane is a key, so that scores store coalesced.
//
// Weighted values.  M rows are 128 dims of the transposed value tile, B the
// three digits of the weights (a weight lies in [0, 2^16]): six column
// blocks, each at most 3 * 2^14 per key, exact in s32 up to 2^15 keys.
//
// Measured (eight heads of two KV heads, head_dim 512; warm passes in a graph).
// 64 nodes at context 32768, 256 query rows a KV head: 303 us, of which scores
// 119 (tensor pipe active 50%, its products alone take 62), softmax 83, values
// 101 (58%, 46).  16 nodes at context 4096: 35 us (13.6, 8.5, 13), most of it
// the start and the end of three dependent kernels of one CTA an SM.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "det_dev.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace rdet {

// set when a bounded wait gives up (read by launch_error_words)
__device__ int g_tree_err = 0;

namespace {

using namespace tcx;

constexpr int kTrKeys = 128;           // keys of a score tile (MMA M)
constexpr int kTrSlot = 128 * 64 * 4;  // a stage's rows: 128 keys of 64 dims, or 64 keys of 128
constexpr int kTrConv = 512;           // converter threads (warps 0-15)
constexpr int kTrConvWarps = kTrConv / 32;
constexpr int kQkThreads = 800;        // + warps 16-19 drain, warp 20 issues the MMAs, warps 21-24 load
constexpr int kQkDrainWarps = 20;      // warps 0-19
constexpr int kTrLoaders = 128;        // loading threads (64 took as long to issue a stage's copies as its MMAs take)
constexpr int kPvThreads = 672;        // + warp 16 issues the MMAs, warps 17-20 load
constexpr int kTrMaxDigit = 0x7f7f7f7f;
constexpr int kTrSplitKeys = 32704;    // keys of one value CTA at most: 3 * 2^14 each in s32

__device__ __forceinline__ void ta_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void ta_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void ta_fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// byte offset of (row r, 16-byte chunk c) in a [rows][64 B] tile in the
// 64-byte swizzle (16-byte chunk index XOR bits 1-2 of the row)
__device__ __forceinline__ int ta_sw(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); }

// kind::i8 instruction descriptor: s32 accumulator, s8 A and B, both K-major,
// M = 128, N = n (a multiple of 16)
__device__ __forceinline__ uint32_t ta_idesc(int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void ta_ld4(uint32_t taddr, int32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr));
}
template <int COLS>
__device__ __forceinline__ void ta_alloc(uint32_t* holder) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(holder)), "n"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void ta_dealloc(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS) : "memory");
}

// Bounded wait on a phase parity (about a second): false when it gave up.
// Every barrier's waiter follows all of its phases in order.
__device__ __forceinline__ bool ta_mbar_wait(uint64_t* b, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 18); ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(su32(b)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

// smem_desc_sw64 of an address `bytes` further on (shared addresses stay below
// 2^18, so the address field does not carry)
__device__ __forceinline__ uint64_t ta_adv(uint64_t desc, int bytes) { return desc + (uint64_t)(bytes >> 4); }

// balanced digits of x as four signed bytes
__device__ __forceinline__ uint32_t ta_digits(int32_t x) { return ((uint32_t)x + 0x80808080u) ^ 0x80808080u; }
// 4 x 4 byte transpose: o[b] = byte b of w0..w3 (w0 in the low byte)
__device__ __forceinline__ void ta_t4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&o)[4]) {
  const uint32_t t0 = __byte_perm(w0, w1, 0x5140), t1 = __byte_perm(w2, w3, 0x5140);
  const uint32_t t2 = __byte_perm(w0, w1, 0x7362), t3 = __byte_perm(w2, w3, 0x7362);
  o[0] = __byte_perm(t0, t1, 0x5410);
  o[1] = __byte_perm(t0, t1, 0x7632);
  o[2] = __byte_perm(t2, t3, 0x5410);
  o[3] = __byte_perm(t2, t3, 0x7632);
}

template <typename... KArgs, typename... Args>
inline void ta_launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, cudaStream_t s,
                      Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// ---- sequences, keys, rows -----------------------------------------------------
// the lowest position a node with ancestor mask `mask` attends
__device__ __forceinline__ int first_pos(const TreeGroup& g, const TreeSeq& t, uint64_t mask) {
  const int p = t.ctx + __popcll(mask);  // position + 1
  return g.window > 0 && p > g.window ? p - g.window : 0;
}
// whether a node with ancestor mask `mask` and first position `start` attends key `key`
__device__ __forceinline__ bool sees(const TreeGroup& g, const TreeSeq& t, uint64_t mask, int start, int key) {
  if (key < t.ctx) return key >= start;
  const int i = key - t.ctx;
  if (i >= t.n || !((mask >> i) & 1)) return false;
  return t.ctx + __popcll(g.mask[t.node0 + i]) - 1 >= start;
}
// the sequence whose items [first, next first) hold item `it` (a warp's lanes
// hold one sequence each; at most 32 sequences)
__device__ __forceinline__ int seq_of(const int32_t* first, int nseq, int it) {
  const int lane = threadIdx.x & 31;
  const unsigned m = __ballot_sync(0xffffffffu, lane < nseq && first[lane] <= it);
  return 31 - __clz((int)m);
}

// Loads into registers that keep their values where `on` is false.  Written
// as predicated instructions: a load under a branch or a select makes the
// compiler wait for it where the paths meet, which costs the prefetch its
// point (a stage took a memory latency longer).  Not .nc: a grid may be
// resident already while the grid before it writes what it reads.
__device__ __forceinline__ void ld16(uint4& v, const void* p, bool on) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %5, 0;\n @p ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n}"
      : "+r"(v.x), "+r"(v.y), "+r"(v.z), "+r"(v.w)
      : "l"(p), "r"((int)on));
}
__device__ __forceinline__ void ld4(uint32_t& v, const void* p, bool on) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %2, 0;\n @p ld.global.L1::no_allocate.u32 %0, [%1];\n}"
               : "+r"(v)
               : "l"(p), "r"((int)on));
}
// the warp's number, known to be the same in all lanes
__device__ __forceinline__ int ta_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }
__device__ __forceinline__ bool ta_elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
// kind::i8 MMA with operand A in TMEM (128 lanes, four K bytes a column)
__device__ __forceinline__ void ta_mma(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void ta_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ void ta_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// thread-block cluster: barrier, and the word at the same place in CTA `rank`
__device__ __forceinline__ void ta_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void ta_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint64_t ta_ld_cluster(const uint64_t* p, int rank) {
  uint64_t v;
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.u64 %0, [a];\n}"
      : "=l"(v)
      : "r"(su32(p)), "r"(rank)
      : "memory");
  return v;
}

// asynchronous copies into shared memory, zeros where `on` is false, and their
// arrival on a barrier once all of the thread's copies so far are there
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(on ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// four dims from `dim` on of a row of d: 16 bytes where every row is 16-byte
// aligned, else one value at a time; what lies past the head is left alone
template <bool VEC>
__device__ __forceinline__ void load4(uint4& v, const int32_t* row, int dim, int d, bool on) {
  if (VEC) {
    ld16(v, row + dim, on && dim < d);
  } else {
    ld4(v.x, row + dim, on && dim < d);
    ld4(v.y, row + dim + 1, on && dim + 1 < d);
    ld4(v.z, row + dim + 2, on && dim + 2 < d);
    ld4(v.w, row + dim + 3, on && dim + 3 < d);
  }
}
__device__ __forceinline__ int32_t max4(int32_t m, const uint4& v) {
  return max(max(max(m, (int32_t)v.x), max((int32_t)v.y, (int32_t)v.z)), (int32_t)v.w);
}

// the bytes of four keys' or values' words as four operand words
__device__ __forceinline__ void ta_bytes(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&o)[4]) {
  ta_t4(w0, w1, w2, w3, o);
  o[0] ^= 0x80808080u;
  o[1] ^= 0x80808080u;
  o[2] ^= 0x80808080u;
}
constexpr int64_t kTrBias = 0x808080;

// the rare weights that the reciprocal leaves open, out of line
__device__ __noinline__ int32_t ta_weight_exact(uint32_t e, uint64_t sum) {
  return softmax_weight(e == 0xffffffffu ? kOneAcc : (int64_t)e, (int64_t)sum);
}
__device__ __forceinline__ int32_t ta_weight(uint32_t e, uint32_t inv, uint64_t sum) {
  int32_t w;
  return softmax_weight_near(e, inv, &w) ? w : ta_weight_exact(e, sum);
}

// add + sum over g of 256^g c_g, wrapping: widening multiply-adds below 2^32,
// the rest in the high word
__device__ __forceinline__ int64_t shift_sum(int64_t add, int32_t c0, int32_t c1, int32_t c2, int32_t c3, int32_t c4,
                                             int32_t c5, int32_t c6) {
  int64_t v = mac_wide(add, c0, 1);
  v = mac_wide(v, c1, 1 << 8);
  v = mac_wide(v, c2, 1 << 16);
  v = mac_wide(v, c3, 1 << 24);
  const uint32_t hi = (uint32_t)((uint64_t)v >> 32) + (uint32_t)c4 + ((uint32_t)c5 << 8) + ((uint32_t)c6 << 16);
  return (int64_t)((uint64_t)hi << 32 | (uint32_t)v);
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
// A stage is 64 dims of a tile's 128 keys, 32 KB as they are in a ring of slots
// in shared memory (16-byte piece c of key k at c ^ (k & 7), so that 32 keys'
// pieces are read without bank conflicts).  The key bytes go to the MMAs
// through TMEM, operand A lying there: written to shared memory and read back
// by the MMAs they made its bandwidth the bound (1550 cycles a stage at 64 rows,
// of which the MMAs take 1024).  A unit of operand A is half the stage's dims of
// the four key bytes, eight columns each; one refills while the other is
// multiplied.  (Eight units beside smaller accumulators, or four of two bytes,
// measured the same or slower.)
constexpr int kQkMaxStages = 6;
constexpr int kSmemMost = 232448;  // a CTA's shared memory
template <int NR>
struct QkRows;
template <int NR>
__host__ __device__ constexpr int qk_stages(int ns);
template <int NR>
__host__ __device__ constexpr int qk_smem(int ns) { return qk_stages<NR>(ns) * kTrSlot + ns * 4 * NR * 64 + 512; }

// what draining a tile needs, per row of the block
template <int NR>
struct QkRows {
  int4 corr[NR];           // 0x808080 times the sum of the query row: 16 bits, 16 bits, high word
  uint64_t mask[NR];       // the node's ancestors and itself
  int32_t start[NR];       // the first position it attends
  uint32_t top[NR];        // its largest score so far, order-preserving as u32
  int32_t npos[kTreeNodes];  // positions of the tree's nodes
  int32_t* sc;             // scores of the block's row 0
  int32_t pad, nr, ctx, lo, len, maxstart;
};
template <int NR>
struct QkShared {
  uint64_t raw_full[kQkMaxStages], raw_empty[kQkMaxStages], a_full[2], a_empty[2], acc_full, acc_empty;
  uint32_t tmem;
  int fail;
  QkRows<NR> rows;
};
template <int NR>
__host__ __device__ constexpr int qk_stages(int ns) {
  const int n = (kSmemMost - 512 - (int)sizeof(QkShared<NR>) - ns * 4 * NR * 64) / kTrSlot;
  return n < kQkMaxStages ? n : kQkMaxStages;
}
// Scores of the row quads quad, quad + step, .. of a tile from TMEM (this
// lane's key is j, the tile's first one j0), and each row's largest one.  At 64
// rows the accumulator fills TMEM, so the MMAs stand still meanwhile: 4500 of a
// tile's 13700 cycles at head_dim 512, spread over all twenty warps, bound by
// the instructions that join and round seven sums (in 32-bit pieces; in 64 bits
// the call above took 4 us more).
template <int NR>
__device__ __noinline__ void qk_drain(QkRows<NR>& c, uint32_t taddr, int j0, int quad, int step) {
  const int lane = threadIdx.x & 31, j = j0 + 32 * ((threadIdx.x >> 5) & 3) + lane, key = c.lo + j;
  const bool in = j < c.len, all = c.lo + j0 >= c.maxstart && c.lo + j0 + kTrKeys <= c.ctx;  // every row attends every key
  const int nr = c.nr;
  int32_t* out = c.sc + (int64_t)(4 * quad) * c.pad + j;
  for (int r = 4 * quad; r < nr; r += 4 * step, out += 4 * (int64_t)step * c.pad) {
    int32_t v[7][4];
#pragma unroll
    for (int b = 0; b < 7; ++b) ta_ld4(taddr + b * NR + r, v[b]);
    tmem_wait_ld();
    uint32_t top[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int4 k = c.corr[r + i];
      const int32_t s = requantize_digits(v[0][i], v[1][i], v[2][i], v[3][i], v[4][i], v[5][i], v[6][i], k.x, k.y, k.z);
      if (in && r + i < nr) out[(int64_t)i * c.pad] = s;
      top[i] = (uint32_t)s ^ 0x80000000u;
    }
    if (!all) {
      const int n = key - c.ctx;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool vis = in && (n < 0 ? key >= c.start[r + i] : (c.mask[r + i] >> n & 1) && c.npos[n] >= c.start[r + i]);
        if (!vis) top[i] = 0;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = __reduce_max_sync(0xffffffffu, top[i]);
    if (lane < 4) atomicMax(&c.top[r + lane], lane < 2 ? (lane == 0 ? top[0] : top[1]) : (lane == 2 ? top[2] : top[3]));
  }
}
// The same by direct wrapping sums, for a block with a query value outside
// the digits' range.
template <int NR>
__device__ __noinline__ void qk_drain_direct(QkRows<NR>& c, const int32_t* k, const int32_t* qb, int r0, int G, int Hq,
                                             int d, int j0, int quad, int step) {
  const int lane = threadIdx.x & 31, j = j0 + 32 * ((threadIdx.x >> 5) & 3) + lane, key = c.lo + j;
  for (int r4 = 4 * quad; r4 < c.nr; r4 += 4 * step)
    for (int r = r4; r < min(c.nr, r4 + 4); ++r) {
      const int node = (r0 + r) / G;
      const int32_t* q = qb + ((int64_t)node * Hq + (r0 + r - node * G)) * d;
      int64_t acc = 0;
      bool vis = j < c.len;
      if (vis) {
        for (int e = 0; e < d; ++e) acc = mac_wide(acc, q[e], k[e]);
        c.sc[(int64_t)r * c.pad + j] = requantize(acc);
        const int n = key - c.ctx;
        vis = n < 0 ? key >= c.start[r] : (c.mask[r] >> n & 1) && c.npos[n] >= c.start[r];
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, vis ? (uint32_t)requantize(acc) ^ 0x80000000u : 0u);
      if (lane == 0) atomicMax(&c.top[r], top);
    }
}

// Scores.  Bound by the MMAs and shared memory about equally: a stage of 64
// rows takes some 1150 cycles, the MMAs 1024, the rows' way in and out with the
// MMAs' reads of the query digits the bandwidth of 1024.
template <int NR, bool VEC>
__global__ void __launch_bounds__(kQkThreads, 1) tree_qk(const __grid_constant__ TreeGroup g) {
  constexpr int na = 4;                         // query digits
  constexpr int kA = 448;                       // TMEM column of operand A's two units
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 511) & ~(uintptr_t)511);
  __shared__ __align__(16) QkShared<NR> sh;
  const int tid = threadIdx.x, warp = ta_warp(), lane = tid & 31;

  // item -> sequence, KV head, row block, key tiles [t0, t1)
  const int si = seq_of(g.qk_first, g.nseq, blockIdx.x);
  const TreeSeq t = g.seq[si];
  const int d = g.d, ns = (d + 63) / 64, G = g.G, Hq = g.Hq, nst = qk_stages<NR>(ns);
  unsigned char* const slots = sm;                    // [nst][128 keys]
  unsigned char* const qpl = sm + nst * kTrSlot;    // [chunk][4 NR rows][64 B]
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, tiles = (t.len + kTrKeys - 1) / kTrKeys, qt = g.qk_tiles;
  const int it = blockIdx.x - g.qk_first[si];
  const int blk = it / t.qk_per, part = it - blk * t.qk_per, t0 = part * qt, t1 = min(tiles, t0 + qt);
  const int kvh = blk / nrb, rb = blk - kvh * nrb;
  const int r0 = rb * NR, nr = min(NR, rows - r0);
  const int total = (t1 - t0) * ns;
  const int32_t* const kc = t.k + (int64_t)kvh * t.kstride;
  const int32_t* const kt = t.kt + (int64_t)kvh * t.tstride;
  const int32_t* const qb = g.q + ((int64_t)t.node0 * Hq + kvh * G) * d;
  const int last_key = t.lo + t.len - 1, last_tile = t1 - t0 - 1;
  if (tid == 0) {
    for (int i = 0; i < nst; ++i) {
      mbar_init(&sh.raw_full[i], kTrLoaders);
      mbar_init(&sh.raw_empty[i], kTrConvWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.a_full[i], kTrConvWarps / 2);
      mbar_init(&sh.a_empty[i], 1);
    }
    mbar_init(&sh.acc_full, 1);
    mbar_init(&sh.acc_empty, kQkDrainWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.fail = 0;
    sh.rows.sc = static_cast<int32_t*>(g.ws) + t.soff + ((int64_t)kvh * rows + r0) * t.pad;
    sh.rows.pad = t.pad;
    sh.rows.nr = nr;
    sh.rows.ctx = t.ctx;
    sh.rows.lo = t.lo;
    sh.rows.len = t.len;
    // (no row's window begins later than that of a node at the tree's greatest possible depth)
    sh.rows.maxstart = g.window > 0 ? max(0, t.ctx + t.n - g.window) : 0;
  }
  if (tid < t.n) sh.rows.npos[tid] = t.ctx + __popcll(g.mask[t.node0 + tid]) - 1;
  if (warp == 20) ta_alloc<512>(&sh.tmem);
  if (tid < NR) {
    const uint64_t m = tid < nr ? g.mask[t.node0 + (r0 + tid) / G] : 0;
    sh.rows.mask[tid] = m;
    sh.rows.start[tid] = tid < nr ? first_pos(g, t, m) : 0;
    sh.rows.top[tid] = 0;
  }
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!ta_mbar_wait(bar, parity)) sh.fail = 1;
  };

  // Stage u into its slot.  Keys past the sequence and dims past the head are zero.
  const int lp = tid - (kQkThreads - kTrLoaders);
  int lt = t0, ls = 0, lb = 0, lph = 1;  // next stage's tile, chunk, slot and the parity of the slot's last use
  auto load = [&]() {
    const uint32_t slot = su32(slots) + lb * kTrSlot;
    const int key0 = t.lo + lt * kTrKeys;
    if (VEC) {  // 16 bytes of keys p / 16, p / 16 + 8, ..
      const int p = lp, dim = ls * 64 + 4 * (p & 15), row0 = p >> 4;
      const bool on = dim < d;
      const uint32_t dst = slot + row0 * 256 + 16 * ((p & 15) ^ row0);
      const int od = on ? dim : 0;
      if (key0 + kTrKeys <= t.ctx) {  // cache rows only
        const int32_t* src = kc + (int64_t)(key0 + row0) * d + od;
#pragma unroll
        for (int i = 0; i < 16; ++i) cp16(dst + i * 2048, src + (int64_t)i * (8 * d), on);
      } else {
        for (int i = 0; i < 16; ++i) {
          const int key = min(key0 + row0 + 8 * i, last_key);
          cp16(dst + i * 2048, (key < t.ctx ? kc + (int64_t)key * d : kt + (int64_t)(key - t.ctx) * d) + od,
               on && key0 + row0 + 8 * i <= last_key);
        }
      }
    } else {  // one dim of every other key
      const int p = lp & 63, dim = ls * 64 + p, od = min(dim, d - 1);
      for (int i = lp >> 6; i < kTrKeys; i += 2) {
        const int key = min(key0 + i, last_key);
        cp4(slot + i * 256 + 16 * ((p >> 2) ^ (i & 7)) + 4 * (p & 3),
            (key < t.ctx ? kc + (int64_t)key * d : kt + (int64_t)(key - t.ctx) * d) + od, dim < d && key0 + i <= last_key);
      }
    }
    cp_arrive(&sh.raw_full[lb]);
    if (++ls == ns) { ls = 0; ++lt; }
    if (++lb == nst) { lb = 0; lph ^= 1; }
  };
  __syncthreads();  // the barriers are there
  ta_wait();
  ta_go();
  // Query digits: chunk s holds dims [64 s, 64 s + 64) of rows a * NR + r; a
  // half warp takes a row, 16 bytes a lane and chunk.
  const int half = lane >> 4, l16 = lane & 15;
  uint4 v[8];
  auto load_q = [&](int r) {
#pragma unroll
    for (int s = 0; s < 8; ++s) v[s] = make_uint4(0, 0, 0, 0);
    const int rr = r0 + min(r, nr - 1), node = rr / G;
    const int32_t* q = qb + ((int64_t)node * Hq + (rr - node * G)) * d;
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (s < ns) load4<VEC>(v[s], q, 64 * s + 4 * l16, d, r < nr);
  };
  int32_t qmax = INT32_MIN;
  if (warp > 20) {
    for (int u = 0; u < min(nst, total); ++u) load();
  } else {
#pragma unroll 1
    for (int r = 2 * warp + half; r < NR; r += 42) {
      load_q(r);
      int64_t sum = 0;
      unsigned char* const dst = qpl + ta_sw(r, l16 >> 2) + 4 * (l16 & 3);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        if (s < ns) {
          sum += (int64_t)(int32_t)v[s].x + (int32_t)v[s].y + (int32_t)v[s].z + (int32_t)v[s].w;
          qmax = max4(qmax, v[s]);
          uint32_t o[4];
          ta_t4(ta_digits((int32_t)v[s].x), ta_digits((int32_t)v[s].y), ta_digits((int32_t)v[s].z),
                ta_digits((int32_t)v[s].w), o);
#pragma unroll
          for (int a = 0; a < 4; ++a) *reinterpret_cast<uint32_t*>(dst + s * (4 * NR * 64) + a * (NR * 64)) = o[a];
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (l16 == 0) {
        const int64_t k = sum * kTrBias;
        sh.rows.corr[r] = make_int4((int32_t)(k & 0xffff), (int32_t)((k >> 16) & 0xffff), (int32_t)(k >> 32), 0);
      }
    }
    ta_fence_async();
  }
  fence_before();
  // a query value outside the digits' range: the block's scores are taken directly
  const bool qover = __syncthreads_or(qmax > kTrMaxDigit);
  fence_after();
  // All 512 columns are this CTA's: they begin at 0 (a constant address keeps
  // the MMA warp's operands uniform).
  constexpr uint32_t tmem = 0;
  if (tid == 0 && sh.tmem != 0) sh.fail = 1;
  // a fifth of the tile's rows by each of the five groups of four warps
  auto drain = [&](int tile) {
    const int j0 = (t0 + tile) * kTrKeys, quad = warp < kTrConvWarps ? 1 + (warp >> 2) : 0;
    wait(&sh.acc_full, tile & 1);
    fence_after();
    if (!qover) {
      qk_drain<NR>(sh.rows, tmem + ((uint32_t)(32 * (warp & 3)) << 16), j0, quad, 5);
    } else {
      const int key = t.lo + j0 + 32 * (warp & 3) + lane;
      qk_drain_direct<NR>(sh.rows, key < t.ctx ? kc + (int64_t)key * d : kt + (int64_t)(key - t.ctx) * d, qb, r0, G, Hq, d,
                          j0, quad, 5);
    }
    fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.acc_empty);
  };

  if (warp < kTrConvWarps) {
    // Key 32 (warp % 4) + lane, dims 16 (warp / 4) .. + 16 of the stage.  A tile
    // is drained once the next one's first stage is converted (which waits
    // for no MMA of that next tile).
    const int key = 32 * (warp & 3) + lane, grp = warp >> 2, h = grp >> 1;
    const uint32_t at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kA + 32 * h + 4 * (grp & 1);
    const unsigned char* const row = slots + key * 256;
    int dt = 0, due = ns + 1, pb = 0, ph = 0;
    for (int u = 0; u < total; ++u) {
      wait(&sh.raw_full[pb], ph);
      uint4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = *reinterpret_cast<const uint4*>(row + pb * kTrSlot + 16 * ((4 * grp + i) ^ (key & 7)));
      uint32_t o[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ta_bytes(x[i].x, x[i].y, x[i].z, x[i].w, o[i]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.raw_empty[pb]);
      if (++pb == nst) { pb = 0; ph ^= 1; }
      if (u > 0) wait(&sh.a_empty[h], (u - 1) & 1);
      fence_after();
#pragma unroll
      for (int b = 0; b < 4; ++b) ta_st4(at + 8 * b, o[0][b], o[1][b], o[2][b], o[3][b]);
      ta_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.a_full[h]);
      if (u + 1 == due) {
        drain(dt++);
        due += ns;
      }
    }
    while (dt <= last_tile) drain(dt++);
  } else if (warp < 20) {
    for (int tile = 0; tile <= last_tile; ++tile) drain(tile);
  } else if (warp == 20) {
    // The whole warp follows the loop and one lane issues: a loop in a branch of
    // one lane moves every operand to a uniform register by itself, about 80
    // cycles an MMA, which made the issue the bound (132 us instead of 121 for
    // 64 nodes at context 32768).
    const bool leader = ta_elect();
    const uint32_t full = ta_idesc(na * NR), low = ta_idesc((na - 1) * NR), one = ta_idesc(NR);
    const uint64_t qdesc = smem_desc_sw64(su32(qpl));
    int tile = 0, s = 0;
    for (int u = 0; u < total; ++u) {
      if (s == 0 && tile >= 1) wait(&sh.acc_empty, (tile - 1) & 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t qd = ta_adv(qdesc, s * (4 * NR * 64) + 32 * h);
        const uint32_t a = tmem + kA + 32 * h;
        wait(&sh.a_full[h], u & 1);
        fence_after();
        if (leader) {
          if (h == 0 && s == 0) {
            // the first products of a tile open its column blocks: byte b adds
            // to the blocks that the bytes before it opened and opens block
            // b + na - 1
            ta_mma(tmem, a, qd, full, 0);
#pragma unroll
            for (int b = 1; b < 4; ++b) {
              ta_mma(tmem + b * NR, a + 8 * b, qd, low, 1);
              ta_mma(tmem + (b + na - 1) * NR, a + 8 * b, ta_adv(qd, (na - 1) * NR * 64), one, 0);
            }
          } else {
#pragma unroll
            for (int b = 0; b < 4; ++b) ta_mma(tmem + b * NR, a + 8 * b, qd, full, 1);
          }
          mma_commit(&sh.a_empty[h]);
          if (h == 1 && s == ns - 1) mma_commit(&sh.acc_full);
        }
        __syncwarp();
      }
      if (++s == ns) {
        s = 0;
        ++tile;
      }
    }
  } else {
    for (int u = nst; u < total; ++u) {
      wait(&sh.raw_empty[lb], lph);
      load();
    }
    cp_wait_all();
  }
  fence_before();
  __syncthreads();
  if (tid < nr) {
    uint32_t* tmax = reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(g.ws) + g.max_off) + t.moff;
    tmax[((int64_t)kvh * rows + r0 + tid) * t.qk_per + part] = sh.rows.top[tid];
  }
  if (sh.fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == 20) ta_dealloc<512>(tmem);
}

// ---------------------------------------------------------------------------
// Softmax: a cluster takes a row, a CTA one chunk of its keys.  The chunk's exp
// terms stay in shared memory while the cluster adds up its sums; the weights'
// digits then replace the scores, as the value kernel's operand tiles want them
// (three planes of 64 bytes per 64 keys, at every 256 bytes of the row).  A
// term is held as u32: the one value of 2^32 (a score equal to the maximum) is
// coded 2^32 - 1, which no other score gives (the next lower score's term is
// below 2^32 - 2^15).  Bound by the instructions of the exp terms where there
// are many rows (16.8 million scores in 83 us, 2.7 instructions a cycle and SM),
// by its chain of loads, barriers and sums where there are few.  One CTA for
// 128 rows of 4112 keys each took 8 us longer than clusters of five, weights
// made in the value kernel, once per 128 dims, 14 us more at 64 nodes.
// ---------------------------------------------------------------------------
constexpr int kExThreads = 256;
constexpr int kExMostKeys = 32768;  // of a CTA: 128 KB of terms

__device__ __forceinline__ uint64_t ta_warp_sum(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kExThreads) tree_softmax(const __grid_constant__ TreeGroup g) {
  extern __shared__ __align__(16) unsigned char tr_raw[];
  uint4* const terms = reinterpret_cast<uint4*>(tr_raw);  // four keys each
  __shared__ uint64_t red[kExThreads / 32], s_part;
  __shared__ int32_t redi[kExThreads / 32], redw[kExThreads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // row of the group: (sequence, KV head, node, head of the KV head's group)
  const int C = g.ex_chunks, grow = blockIdx.x / C, chunk = blockIdx.x - grow * C;
  const int si = seq_of(g.row_first, g.nseq, grow);
  const TreeSeq t = g.seq[si];
  const int rows = t.n * g.G, lrow = grow - g.row_first[si], rr = lrow % rows;
  const uint64_t mask = g.mask[t.node0 + rr / g.G];
  const int start = first_pos(g, t, mask);
  unsigned char* const ws = static_cast<unsigned char*>(g.ws);
  int32_t* const sc = reinterpret_cast<int32_t*>(ws) + t.soff + (int64_t)lrow * t.pad;
  const uint32_t* tmax = reinterpret_cast<const uint32_t*>(ws + g.max_off) + t.moff + (int64_t)lrow * t.qk_per;
  ta_wait();
  ta_go();
  if (chunk == 0 && t.splits > 1) {  // the value kernel's sums and counters
    uint64_t* acc = reinterpret_cast<uint64_t*>(ws + g.acc_off) + (int64_t)grow * g.d;
    for (int i = tid; i < g.d; i += kExThreads) acc[i] = 0;
    const int items = t.cfirst + (lrow / rows * ((rows + g.nr - 1) / g.nr) + rr / g.nr) * ((g.d + 127) / 128);
    if (rr % g.nr == 0 && tid < (g.d + 127) / 128) reinterpret_cast<uint32_t*>(ws + g.cnt_off)[items + tid] = 0;
  }
  const int k0 = chunk * g.ex_keys, k1 = min(t.pad, k0 + g.ex_keys);  // (k0 >= k1: no keys)
  uint4 next;
  ld16(next, sc + k0 + 4 * tid, k0 + 4 * tid < k1);
  uint32_t top = 0;
  for (int i = lane; i < t.qk_per; i += 32) top = max(top, tmax[i]);
  const uint32_t m = __reduce_max_sync(0xffffffffu, top) ^ 0x80000000u;
  uint64_t sum = 0;
  int32_t first = INT32_MAX;  // the thread's first key at the maximum
  for (int j = k0 + 4 * tid; j < k1; j += 4 * kExThreads) {
    const uint4 v = next;
    ld16(next, sc + j + 4 * kExThreads, j + 4 * kExThreads < k1);
    const int key = t.lo + j;
    uint32_t vis = 15u;
    if (!(key >= start && key + 3 < t.ctx)) {
      vis = 0;
      for (int i = 0; i < 4; ++i) vis |= sees(g, t, mask, start, key + i) ? 1u << i : 0u;
    }
    auto term = [&](uint32_t x, int i) -> uint32_t {
      const uint32_t D = m - x;  // below the maximum by D
      const bool on = vis >> i & 1;
      uint32_t e = on && D < (16u << 16) ? exp_term_below(D) : 0;
      if (on && D == 0) {
        e = 0xffffffffu;
        first = min(first, j + i);
        sum += 1;
      }
      sum += e;
      return e;
    };
    terms[(j - k0) >> 2] = make_uint4(term(v.x, 0), term(v.y, 1), term(v.z, 2), term(v.w, 3));
  }
  sum = ta_warp_sum(sum);
  first = __reduce_min_sync(0xffffffffu, first);
  if (lane == 0) {
    red[warp] = sum;
    redi[warp] = first;
  }
  __syncthreads();
  sum = ta_warp_sum(lane < kExThreads / 32 ? red[lane] : 0);
  first = __reduce_min_sync(0xffffffffu, lane < kExThreads / 32 ? redi[lane] : INT32_MAX);
  if (C > 1) {
    if (tid == 0) s_part = sum;
    ta_cluster_arrive();
    ta_cluster_wait();
    sum = ta_warp_sum(lane < C ? ta_ld_cluster(&s_part, lane) : 0);
    ta_cluster_arrive();  // (waited for before the CTA ends: its part is read by the others)
  }
  const uint32_t inv = softmax_inverse(sum);
  int32_t wsum = 0;
  for (int j = k0 + 4 * tid; j < k1; j += 4 * kExThreads) {
    const uint4 e = terms[(j - k0) >> 2];
    const int32_t w0 = ta_weight(e.x, inv, sum), w1 = ta_weight(e.y, inv, sum), w2 = ta_weight(e.z, inv, sum),
                  w3 = ta_weight(e.w, inv, sum);
    wsum += w0 + w1 + w2 + w3;
    uint32_t o[4];
    ta_t4(ta_digits(w0), ta_digits(w1), ta_digits(w2), ta_digits(w3), o);
    // (a chunk of 64 keys lies with 16 neighbouring threads, whose scores it replaces)
    uint32_t* const out = reinterpret_cast<uint32_t*>(sc) + (j & ~63) + ((j & 63) >> 2);
#pragma unroll
    for (int a = 0; a < 3; ++a) out[16 * a] = o[a];
  }
  wsum = __reduce_add_sync(0xffffffffu, wsum);
  if (lane == 0) redw[warp] = wsum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kExThreads / 32; ++w) wsum += redw[w];
    reinterpret_cast<int32_t*>(ws + g.sum_off)[(int64_t)grow * C + chunk] = wsum;
    reinterpret_cast<int32_t*>(ws + g.idx_off)[(int64_t)grow * C + chunk] = first;
  }
  if (C > 1) ta_cluster_wait();
}

// ---------------------------------------------------------------------------
// weighted values: an item is a (sequence, KV head, row block, block of 128
// dims); its keys are split over `splits` CTAs in chunks of 64.  The partial
// i64 sums meet in global memory (wrapping integer adds: any order gives the
// same sum) and the item's last CTA to arrive rounds them.  (Clusters with the
// sums in distributed shared memory measured worse: only about 13 clusters of
// eight large CTAs fit the GPU at once, so 16 took two waves.)
// ---------------------------------------------------------------------------
// A stage is 64 keys of the 128 dims, 32 KB as they are in a ring of slots; the
// value bytes go to the MMAs through TMEM like the key bytes above (a thread
// holds one dim of 16 keys); the weights' digits, operand B, lie behind them.
// Bound by shared memory: a stage of 64 rows takes some 1230 cycles, its
// traffic 1000 of them, its MMAs 768.
constexpr int kPvStages = 6;
template <int NR>
__host__ __device__ constexpr int pv_slot() { return kTrSlot + 3 * NR * 64; }
template <int NR>
__host__ __device__ constexpr int pv_stages() { return NR == 16 ? kPvStages : 5; }
template <int NR>
__host__ __device__ constexpr int pv_smem() { return pv_stages<NR>() * pv_slot<NR>() + 512; }

template <int NR, bool VEC>
__global__ void __launch_bounds__(kPvThreads, 1) tree_pv(const __grid_constant__ TreeGroup g) {
  constexpr int kA = 448;                       // TMEM column of operand A's two units
  constexpr int kSt = pv_stages<NR>(), kSlot = pv_slot<NR>();
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 511) & ~(uintptr_t)511);
  unsigned char* slots = sm;                    // [slot][64 keys][128 dims], [3 NR rows][64 keys]
  __shared__ __align__(8) uint64_t raw_full[kPvStages], raw_empty[kPvStages], a_full[2], a_empty[2], acc_full;
  __shared__ uint32_t tmem_holder;
  __shared__ int s_fail;
  __shared__ int32_t s_first[NR];               // each row's first maximum
  __shared__ int32_t s_wsum[NR];                // its sum of weights
  __shared__ uint32_t s_last;
  const int tid = threadIdx.x, warp = ta_warp(), lane = tid & 31;

  const int si = seq_of(g.pv_first, g.nseq, blockIdx.x);
  const TreeSeq t = g.seq[si];
  const int d = g.d, nd = (d + 127) / 128, G = g.G, Hq = g.Hq;
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, chunks = t.pad / 64;
  const int S = t.splits, ic = blockIdx.x - g.pv_first[si], it = ic / S, sp = ic - it * S;
  const int blk = it / nd, db = it - blk * nd, kvh = blk / nrb, rb = blk - kvh * nrb;
  const int c0 = (int)((int64_t)chunks * sp / S), c1 = (int)((int64_t)chunks * (sp + 1) / S);
  const int r0 = rb * NR, nr = min(NR, rows - r0), total = c1 - c0;
  const int lrow0 = kvh * rows + r0, grow0 = g.row_first[si] + lrow0;
  unsigned char* const ws = static_cast<unsigned char*>(g.ws);
  const unsigned char* const wts = ws + 4 * (t.soff + (int64_t)lrow0 * t.pad + c0 * 64);  // 256 bytes per row and stage
  const int32_t* const vc = t.v + (int64_t)kvh * t.kstride;
  const int32_t* const vt = t.vt + (int64_t)kvh * t.tstride;
  const int last_key = t.lo + t.len - 1;

  // Stage lu into its slot.  Keys past the sequence (their weights are zero) and
  // dims past the head (their sums are not stored) are zero.
  const int lp = tid - (kPvThreads - kTrLoaders);
  int lu = 0, lb = 0, lph = 1;  // next stage, its slot and the parity of the slot's last use
  auto load = [&]() {
    const uint32_t slot = su32(slots) + lb * kSlot;
    const int key0 = t.lo + (c0 + lu) * 64;
    if (VEC) {  // 16 bytes of keys p / 32, p / 32 + 4, ..
      const int p = lp, dim = db * 128 + 4 * (p & 31), row0 = p >> 5;
      const bool on = dim < d;
      const uint32_t dst = slot + row0 * 512 + 16 * (p & 31);
      const int od = on ? dim : 0;
      if (key0 + 64 <= t.ctx) {  // cache rows only
        const int32_t* src = vc + (int64_t)(key0 + row0) * d + od;
#pragma unroll
        for (int i = 0; i < 16; ++i) cp16(dst + i * 2048, src + (int64_t)i * (4 * d), on);
      } else {
        for (int i = 0; i < 16; ++i) {
          const int key = min(key0 + row0 + 4 * i, last_key);
          cp16(dst + i * 2048, (key < t.ctx ? vc + (int64_t)key * d : vt + (int64_t)(key - t.ctx) * d) + od,
               on && key0 + row0 + 4 * i <= last_key);
        }
      }
    } else {  // one dim of every key
      const int dim = db * 128 + lp, od = min(dim, d - 1);
      for (int i = 0; i < 64; ++i) {
        const int key = min(key0 + i, last_key);
        cp4(slot + i * 512 + 4 * lp, (key < t.ctx ? vc + (int64_t)key * d : vt + (int64_t)(key - t.ctx) * d) + od,
            dim < d && key0 + i <= last_key);
      }
    }
    ++lu;
    if (++lb == kSt) { lb = 0; lph ^= 1; }
  };
  // Stage u's weights into slot b, and the stage's arrival: 16 bytes of rows
  // p / 4, p / 4 + 32, .. (rows past the block are zero)
  auto load_w = [&](int u, int b) {
    const int c = lp & 3;
    const uint32_t dst = su32(slots) + b * kSlot + kTrSlot;
#pragma unroll
    for (int i = 0; i < (NR + 31) / 32; ++i) {
      const int r = (lp >> 2) + 32 * i;
      const unsigned char* src = wts + (int64_t)min(r, nr - 1) * t.pad * 4 + u * 256 + 16 * c;
#pragma unroll
      for (int a = 0; a < 3; ++a)
        if (r < NR) cp16(dst + ta_sw(a * NR + r, c), src + 64 * a, r < nr);
    }
    cp_arrive(&raw_full[b]);
  };
  if (tid == 0) {
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&raw_full[i], kTrLoaders);
      mbar_init(&raw_empty[i], kTrConvWarps + 1);  // the converters have read the values, the MMAs the weights
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&a_full[i], kTrConvWarps / 2);
      mbar_init(&a_empty[i], 1);
    }
    mbar_init(&acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_fail = 0;
  }
  if (warp == kTrConvWarps) ta_alloc<512>(&tmem_holder);
  fence_before();
  __syncthreads();  // the barriers and TMEM are there
  fence_after();
  // The values do not depend on the terms: their first stages load before the
  // wait (this grid starts only after the score kernel has completed, and with
  // it everything before it).
  if (warp > kTrConvWarps)
    for (int u = 0; u < min(kSt, total); ++u) load();
  ta_wait();
  ta_go();
  if (warp > kTrConvWarps) {
    for (int u = 0; u < min(kSt, total); ++u) load_w(u, u);
  }
  constexpr uint32_t tmem = 0;  // all 512 columns, as above
  if (tid == 0 && tmem_holder != 0) s_fail = 1;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!ta_mbar_wait(bar, parity)) s_fail = 1;
  };

  if (warp < kTrConvWarps) {
    // dim 32 (warp % 4) + lane, keys 16 (warp / 4) .. + 16 of the stage
    const int grp = warp >> 2, h = grp >> 1;
    const uint32_t at = ((uint32_t)(32 * (warp & 3)) << 16) + kA + 32 * h + 4 * (grp & 1);
    const unsigned char* const col = slots + 16 * grp * 512 + 4 * (32 * (warp & 3) + lane);
    int pb = 0, ph = 0;
    for (int u = 0; u < total; ++u) {
      wait(&raw_full[pb], ph);
      uint32_t x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = *reinterpret_cast<const uint32_t*>(col + pb * kSlot + 512 * i);
      uint32_t o[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ta_bytes(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3], o[i]);
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty[pb]);
      if (++pb == kSt) { pb = 0; ph ^= 1; }
      if (u > 0) wait(&a_empty[h], (u - 1) & 1);
      fence_after();
#pragma unroll
      for (int b = 0; b < 4; ++b) ta_st4(at + 8 * b, o[0][b], o[1][b], o[2][b], o[3][b]);
      ta_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[h]);
    }
  } else if (warp == kTrConvWarps) {
    const bool leader = ta_elect();
    const uint32_t full = ta_idesc(3 * NR), low = ta_idesc(2 * NR), one = ta_idesc(NR);
    const uint64_t wdesc = smem_desc_sw64(su32(slots) + kTrSlot);
    int pb = 0;
    for (int u = 0; u < total; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint64_t wd = ta_adv(wdesc, pb * kSlot + 32 * h);
        const uint32_t a = tmem + kA + 32 * h;
        wait(&a_full[h], u & 1);
        if (h == 0) ta_fence_async();  // the weights' tile: the converters saw its arrival before theirs
        fence_after();
        if (leader) {
          if (h == 0 && u == 0) {  // opens the column blocks, as in the score kernel
            ta_mma(tmem, a, wd, full, 0);
#pragma unroll
            for (int b = 1; b < 4; ++b) {
              ta_mma(tmem + b * NR, a + 8 * b, wd, low, 1);
              ta_mma(tmem + (b + 2) * NR, a + 8 * b, ta_adv(wd, 2 * NR * 64), one, 0);
            }
          } else {
#pragma unroll
            for (int b = 0; b < 4; ++b) ta_mma(tmem + b * NR, a + 8 * b, wd, full, 1);
          }
          mma_commit(&a_empty[h]);
          if (h == 1) mma_commit(&raw_empty[pb]);
          if (h == 1 && u == total - 1) mma_commit(&acc_full);
        }
        __syncwarp();
      }
      if (++pb == kSt) pb = 0;
    }
    if (total > 0) wait(&acc_full, 0);
  } else {
    for (int u = kSt; u < total; ++u) {
      wait(&raw_empty[lb], lph);
      const int b = lb;
      load();
      load_w(u, b);
    }
    // the rows' first maxima and sums of weights, wanted at the end
    constexpr int kT = kTrLoaders / NR;  // threads a row
    const int r = lp / kT;
    const int64_t at = (int64_t)(grow0 + min(r, nr - 1)) * g.ex_chunks;
    const int32_t* pw = reinterpret_cast<const int32_t*>(ws + g.sum_off) + at;
    const int32_t* pidx = reinterpret_cast<const int32_t*>(ws + g.idx_off) + at;
    int32_t v = 0, f = INT32_MAX;
    for (int i = lp % kT; i < g.ex_chunks; i += kT) {
      v += pw[i];
      f = min(f, pidx[i]);
    }
#pragma unroll
    for (int o = kT / 2; o > 0; o >>= 1) {
      v += __shfl_xor_sync(0xffffffffu, v, o);
      f = min(f, __shfl_xor_sync(0xffffffffu, f, o));
    }
    if (lp % kT == 0) {
      s_first[r] = f;
      s_wsum[r] = v;
    }
    cp_wait_all();
  }
  __syncthreads();
  fence_after();
  // ---- the block's partial sums: lane dl, rows split over the four quarters
  const int dl = tid & 127, quarter = (tid >> 7) & 3, dim = db * 128 + dl;
  auto orow = [&](int r) {
    const int rr = r0 + r, node = rr / G;
    return g.out + ((int64_t)(t.node0 + node) * Hq + kvh * G + (rr - node * G)) * d;
  };
  // Row r's sum v of digit products to the output: the bytes'
  // bias, and what the weights' roundings left times the first maximum's value.
  unsigned long long* const acc = reinterpret_cast<unsigned long long*>(ws + g.acc_off) + (int64_t)grow0 * d;
  auto first_value = [&](int r) {  // the first maximum's value
    const int key = t.lo + s_first[r];
    return (key < t.ctx ? vc + (int64_t)key * d : vt + (int64_t)(key - t.ctx) * d)[dim];
  };
  auto finish = [&](int r, uint64_t v, int32_t value) {
    const int32_t wt = s_wsum[r];
    v += (uint64_t)(kTrBias * wt) + (uint64_t)mul_wide(sub_sat(kOneAct, wt), value);
    orow(r)[dim] = requantize_flat((int64_t)v);
  };
  if (warp < kTrConvWarps && total > 0) {
    constexpr int kQ = NR / 4;
    const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
    for (int r = quarter * kQ; r < min(nr, (quarter + 1) * kQ); r += 4) {
      int32_t c[6][4];
#pragma unroll
      for (int b = 0; b < 6; ++b) ta_ld4(taddr + b * NR + r, c[b]);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t v = shift_sum(0, c[0][i], c[1][i], c[2][i], c[3][i], c[4][i], c[5][i], 0);
        if (r + i < nr && dim < d) {
          if (S > 1) atomicAdd(acc + (int64_t)(r + i) * d + dim, (unsigned long long)v);
          else finish(r + i, (uint64_t)v, first_value(r + i));
        }
      }
    }
  }
  if (S > 1) {
    uint32_t* const cnt = reinterpret_cast<uint32_t*>(ws + g.cnt_off) + t.cfirst + it;
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(cnt, 1u) == (uint32_t)S - 1;
    __syncthreads();
    if (s_last && warp < kTrConvWarps && dim < d) {
      __threadfence();
      // a thread's rows in flight together (one after the other the sixteen of a
      // 64-row block took the last CTA 11000 cycles)
      constexpr int kF = NR == 16 ? 1 : 8;
      for (int q = quarter; q < nr; q += 4 * kF) {
        uint64_t v[kF];
        int32_t value[kF];
#pragma unroll
        for (int i = 0; i < kF; ++i) {
          const int r = min(q + 4 * i, nr - 1);
          v[i] = __ldcg(acc + (int64_t)r * d + dim);
          value[i] = first_value(r);
        }
#pragma unroll
        for (int i = 0; i < kF; ++i)
          if (q + 4 * i < nr) finish(q + 4 * i, v[i], value[i]);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (s_fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == kTrConvWarps) ta_dealloc<512>(tmem);
}

template <int NR, bool VEC>
void qk_attr() {
  int most = 0;
  for (int ns = 1; ns <= 8; ++ns) most = std::max(most, qk_smem<NR>(ns));
  cudaFuncSetAttribute(tree_qk<NR, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}
template <int NR, bool VEC>
void pv_attr() {
  cudaFuncSetAttribute(tree_pv<NR, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, pv_smem<NR>());
}

}  // namespace

void tree_attn_init() {
  qk_attr<16, true>();
  qk_attr<16, false>();
  qk_attr<32, true>();
  qk_attr<32, false>();
  qk_attr<64, true>();
  qk_attr<64, false>();
  cudaFuncSetAttribute(tree_softmax, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kExMostKeys);
  cudaFuncSetAttribute(tree_softmax, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  pv_attr<16, true>();
  pv_attr<16, false>();
  pv_attr<32, true>();
  pv_attr<32, false>();
  pv_attr<64, true>();
  pv_attr<64, false>();
}

int32_t* tree_attn_error_word() {
  void* p = nullptr;
  cudaGetSymbolAddress(&p, g_tree_err);
  return static_cast<int32_t*>(p);
}

size_t tree_attn_plan(TreeGroup& g) {
  constexpr int kSms = 148;
  const int G = g.G = g.Hq / g.Hkv, nd = (g.d + 127) / 128;
  int maxrows = 0, maxpad = 0;
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    // the shallowest node's window is the lowest of the tree
    t.lo = g.window > 0 && t.ctx + 1 > g.window ? std::min(t.ctx, t.ctx + 1 - g.window) : 0;
    t.len = t.ctx - t.lo + t.n;
    t.pad = (t.len + 63) & ~63;
    maxrows = std::max(maxrows, t.n * G);
    maxpad = std::max(maxpad, t.pad);
  }
  // Rows of a block.  64 rows read each key and value half as often as 32, but
  // leave half as many items: taken where those still make a wave of score
  // tiles.  Eight heads of two KV heads, head_dim 512, 32 against 64 rows: 16
  // nodes at context 4096 (66 tiles of 64 rows) 35.9 / 41.4 us, at 8192 (130)
  // 46.4 / 46.7, at 16384 (258) 71.6 / 66.8; 64 nodes at 32768 389 / 282.
  int64_t wide = 0;  // score tiles of 64-row blocks
  for (int i = 0; i < g.nseq; ++i)
    wide += (int64_t)g.Hkv * ((g.seq[i].n * G + 63) / 64) * ((g.seq[i].len + kTrKeys - 1) / kTrKeys);
  g.nr = maxrows <= 16 ? 16 : maxrows <= 32 || wide < kSms ? 32 : 64;
  int64_t soff = 0, moff = 0;
  int rows = 0, pv = 0, qk = 0, counters = 0;
  auto blocks = [&](const TreeSeq& t) { return (int64_t)g.Hkv * ((t.n * G + g.nr - 1) / g.nr); };
  auto ceil_div = [](int x, int y) { return (x + y - 1) / y; };
  // Key tiles of a score CTA and 64-key chunks of a value CTA: the size with
  // the shortest run of work on one SM, from the least size of each number of
  // waves (one CTA an SM; a CTA's fixed work is counted in stages of its loop).
  auto pick = [&](int most, auto&& ctas, auto&& stages) {
    int size = most;
    int64_t best = INT64_MAX;
    for (int waves = 1; waves <= 4; ++waves) {
      int lo = 1, hi = most;  // the least size whose CTAs take `waves` waves
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (ctas(mid) <= (int64_t)waves * kSms) hi = mid;
        else lo = mid + 1;
      }
      const int64_t cost = (ctas(lo) + kSms - 1) / kSms * stages(lo);
      if (cost < best) {
        best = cost;
        size = lo;
      }
    }
    return size;
  };
  const int ns = (g.d + 63) / 64;
  g.qk_tiles = pick(
      ceil_div(maxpad, kTrKeys),
      [&](int k) {
        int64_t n = 0;
        for (int i = 0; i < g.nseq; ++i) n += blocks(g.seq[i]) * ceil_div(ceil_div(g.seq[i].len, kTrKeys), k);
        return n;
      },
      [&](int k) { return k * (ns + (g.nr == 64 ? 4 : 2)) + 8; });
  const int per = pick(
      std::min(kTrSplitKeys, maxpad) / 64,
      [&](int k) {
        int64_t n = 0;
        for (int i = 0; i < g.nseq; ++i) n += blocks(g.seq[i]) * nd * ceil_div(g.seq[i].pad / 64, k);
        return n;
      },
      [&](int k) { return k + 10; });
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    t.soff = soff;
    soff += (int64_t)t.pad * t.n * g.Hq;
    g.row_first[i] = rows;
    rows += t.n * g.Hq;
    t.splits = ceil_div(t.pad / 64, per);
    g.pv_first[i] = pv;
    pv += (int)blocks(t) * nd * t.splits;
    t.cfirst = counters;
    counters += (int)blocks(t) * nd;
    t.qk_per = ceil_div(ceil_div(t.len, kTrKeys), g.qk_tiles);
    g.qk_first[i] = qk;
    qk += (int)blocks(t) * t.qk_per;
    t.moff = moff;
    moff += (int64_t)t.n * g.Hq * t.qk_per;
  }
  g.rows = rows;
  g.pv_items = pv;
  g.qk_items = qk;
  // Keys of a softmax CTA: four per thread, more where the CTAs would not be
  // resident at once (a CTA is mostly latency: 1288 rows of up to 4108 keys take
  // 46 us in clusters of three CTAs, 25 with one CTA a row; 128 rows of 4112 keys
  // 8.5 us in clusters of five, 17 with one), and so many that a row's cluster
  // has at most eight CTAs (sixteen for the longest).
  g.ex_keys = 4 * kExThreads;
  while ((g.ex_keys < 32 * kExThreads && (int64_t)rows * ceil_div(maxpad, g.ex_keys) > 8 * kSms) ||
         ceil_div(maxpad, g.ex_keys) > (g.ex_keys < kExMostKeys ? 8 : 16))
    g.ex_keys *= 2;
  g.ex_chunks = ceil_div(maxpad, g.ex_keys);
  g.ex_keys = (ceil_div(maxpad, g.ex_chunks) + 63) & ~63;
  auto up = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  g.max_off = up(soff * 4);
  g.sum_off = up(g.max_off + moff * 4);
  g.idx_off = up(g.sum_off + (int64_t)rows * g.ex_chunks * 4);
  g.acc_off = up(g.idx_off + (int64_t)rows * g.ex_chunks * 4);
  g.cnt_off = up(g.acc_off + (int64_t)rows * g.d * 8);
  return g.ws_bytes = (size_t)up(g.cnt_off + (int64_t)counters * 4);
}

template <int NR, bool VEC>
static void tree_launch(const TreeGroup& g, cudaStream_t s) {
  const int ns = (g.d + 63) / 64;
  ta_launch(tree_qk<NR, VEC>, dim3(g.qk_items), dim3(kQkThreads), qk_smem<NR>(ns), 1, s, g);
  ta_launch(tree_softmax, dim3((unsigned)g.rows * g.ex_chunks), dim3(kExThreads), 4 * (size_t)g.ex_keys, g.ex_chunks, s, g);
  ta_launch(tree_pv<NR, VEC>, dim3(g.pv_items), dim3(kPvThreads), pv_smem<NR>(), 1, s, g);
}

void launch_tree_attn(const TreeGroup& g, cudaStream_t s) {
  // 16-byte copies where every row is 16-byte aligned
  uintptr_t bits = reinterpret_cast<uintptr_t>(g.q);
  for (int i = 0; i < g.nseq; ++i) {
    const TreeSeq& t = g.seq[i];
    bits |= reinterpret_cast<uintptr_t>(t.k) | reinterpret_cast<uintptr_t>(t.kt);
    bits |= reinterpret_cast<uintptr_t>(t.v) | reinterpret_cast<uintptr_t>(t.vt);
  }
  const bool vec = g.d % 4 == 0 && (bits & 15) == 0;
  if (g.nr == 16) vec ? tree_launch<16, true>(g, s) : tree_launch<16, false>(g, s);
  else if (g.nr == 32) vec ? tree_launch<32, true>(g, s) : tree_launch<32, false>(g, s);
  else vec ? tree_launch<64, true>(g, s) : tree_launch<64, false>(g, s);
}

}  // namespace rdet
