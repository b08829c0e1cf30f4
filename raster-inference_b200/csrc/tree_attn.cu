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
// running softmax is exact: the scores of all keys come before the first
// weight.  Three kernels over a scratch, coupled by programmatic dependent
// launch: scores and weighted values on the tensor cores, the softmax on the
// CUDA cores between them.  A key is an index into the sequence's
// [lo, lo + len): cache rows lo .. ctx - 1, then the nodes (key ctx + i).  The
// order of keys is the order of positions along every node's path, because
// parents come before their children.
//
// Digits.  x = sum_b 256^b x_b with x_b in [-128, 127] (balanced base-256
// digits) holds for every i32 up to 0x7f7f7f7f: the digits are the bytes of
// (x + 0x80808080) ^ 0x80808080.  Then sum x y = sum_{a,b} 256^(a+b) sum x_b
// y_a, signed int8 products that need no offset corrections, and digits that
// are zero throughout (activations after a norm rarely reach 2^23) cost
// nothing.  A tile that holds a larger value takes the direct wrapping i64
// sums instead.
//
// Scores.  The keys of a 128-key tile are the MMA's M rows, one operand A per
// key digit b; operand B stacks the digits of NR query rows (rows a * NR + r).
// The MMA of key digit b accumulates at TMEM column b * NR, so column block g
// (columns [g NR, (g + 1) NR)) sums exactly the products of shift 8 g: seven
// blocks, each at most 4 * 2^14 * 512 = 2^25 in magnitude, exact in s32.
// A query row is a (node, head of the KV head's group); all of them read a
// key tile at once, so the cache streams once per NR rows.
//
// Weighted values.  M rows are 128 dims of the transposed value tile, B the
// three digits of the weights (a weight lies in [-2^23, 2^16]): six column
// blocks, each at most 3 * 2^14 per key, exact in s32 up to 2^15 keys.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "det_dev.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace rdet {

// set when a bounded wait gives up (read by tree_attn_error_flag)
__device__ int g_tree_err = 0;

namespace {

namespace cg = cooperative_groups;
using namespace tcx;

constexpr int kTrKeys = 128;           // keys of a score tile (MMA M)
constexpr int kTrPlane = 128 * 64;     // one digit plane of a stage: 128 rows of 64 bytes
constexpr int kTrPlanes = 4 * kTrPlane;
constexpr int kTrConv = 256;           // converter threads (warps 0-7)
constexpr int kQkThreads = 416;        // + warps 8-11 drain the accumulators, warp 12 issues the MMAs
constexpr int kPvThreads = 288;        // + warp 8 issues the MMAs
constexpr int kTrMaxDigit = 0x7f7f7f7f;
constexpr int kTrSplitKeys = 16384;    // keys of one value split at most (s32 accumulators)

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

// digits of x as four signed bytes
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
__device__ __forceinline__ const int32_t* key_row(const TreeSeq& t, int kvh, int key, int d) {
  return key < t.ctx ? t.k + (int64_t)kvh * t.kstride + (int64_t)key * d
                     : t.kt + (int64_t)kvh * t.tstride + (int64_t)(key - t.ctx) * d;
}
__device__ __forceinline__ const int32_t* value_row(const TreeSeq& t, int kvh, int key, int d) {
  return key < t.ctx ? t.v + (int64_t)kvh * t.kstride + (int64_t)key * d
                     : t.vt + (int64_t)kvh * t.tstride + (int64_t)(key - t.ctx) * d;
}
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

// four dims from `dim` on of a row (zero past the head): 16-byte loads where
// every row is 16-byte aligned, else one value at a time
template <bool VEC>
__device__ __forceinline__ uint4 load4(const int32_t* row, int dim, int d) {
  if (VEC) return dim < d ? __ldg(reinterpret_cast<const uint4*>(row + dim)) : make_uint4(0, 0, 0, 0);
  uint4 v = make_uint4(0, 0, 0, 0);
  if (dim < d) v.x = (uint32_t)row[dim];
  if (dim + 1 < d) v.y = (uint32_t)row[dim + 1];
  if (dim + 2 < d) v.z = (uint32_t)row[dim + 2];
  if (dim + 3 < d) v.w = (uint32_t)row[dim + 3];
  return v;
}
__device__ __forceinline__ bool over(const uint4& v) {
  return max(max((int32_t)v.x, (int32_t)v.y), max((int32_t)v.z, (int32_t)v.w)) > kTrMaxDigit;
}

// sum of seven column blocks: sum_g 256^g c[g], wrapping
__device__ __forceinline__ int64_t shift_sum(const int32_t (&c)[7]) {
  const int64_t p0 = mac_wide(c[0], c[1], 256), p1 = mac_wide(c[2], c[3], 256), p2 = mac_wide(c[4], c[5], 256);
  return (int64_t)((uint64_t)p0 + ((uint64_t)p1 << 16) + ((uint64_t)p2 << 32) + ((uint64_t)(int64_t)c[6] << 48));
}

// ---------------------------------------------------------------------------
// scores
// ---------------------------------------------------------------------------
template <int NR>
__host__ __device__ constexpr int qk_smem(int ns) { return 2 * kTrPlanes + ns * 4 * NR * 64 + 1024; }

template <int NR, bool VEC>
__global__ void __launch_bounds__(kQkThreads, NR == 16 ? 2 : 1) tree_qk(const __grid_constant__ TreeGroup g) {
  constexpr int kCols = 7 * NR, kTmem = NR == 16 ? 256 : 512;
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* planes = sm;                   // [2][4 digits][128 keys][64 B]
  unsigned char* qpl = sm + 2 * kTrPlanes;      // [chunk][4 NR rows][64 B]
  __shared__ __align__(8) uint64_t planes_full[2], mma_done[2], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_holder;
  __shared__ int s_fail;
  __shared__ __align__(8) unsigned char s_top[2][8];   // per converter warp: digit 3 is used in the stage
  // a value outside the digits' range in the tile.  Four slots: a converter
  // runs at most two stages, so at most two tiles, ahead of the MMAs, and those
  // at most two tiles ahead of the drain that reads the slot.
  __shared__ __align__(8) unsigned char s_over[4][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int d = g.d, ns = (d + 63) / 64, G = g.Hq / g.Hkv;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&planes_full[i], kTrConv / 32);
      mbar_init(&mma_done[i], 1);
      mbar_init(&acc_full[i], 2);
      mbar_init(&acc_empty[i], 4);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_fail = 0;
  }
  if (warp == 0) ta_alloc<kTmem>(&tmem_holder);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_holder;

  // item -> sequence, KV head, row block, key tiles [t0, t1)
  const int si = seq_of(g.qk_first, g.nseq, blockIdx.x);
  const TreeSeq& t = g.seq[si];
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, tiles = (t.len + kTrKeys - 1) / kTrKeys;
  const int per = (tiles + g.qk_tiles - 1) / g.qk_tiles;  // items of one row block
  const int it = blockIdx.x - g.qk_first[si];
  const int kvh = it / (per * nrb), rb = (it / per) % nrb;
  const int t0 = (it % per) * g.qk_tiles, t1 = min(tiles, t0 + g.qk_tiles);
  const int r0 = rb * NR, nr = min(NR, rows - r0);
  const int total = (t1 - t0) * ns;
  ta_wait();
  ta_go();

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_wait(bar, parity)) s_fail = 1;
  };
  // query row r (node * G + head of the group) of this block
  auto qrow = [&](int r) {
    const int rr = r0 + r;
    return g.q + ((int64_t)(t.node0 + rr / G) * g.Hq + kvh * G + rr % G) * d;
  };

  // a converter thread's part of a stage: keys 16 warp + 2 i + lane / 16, dims 4 (lane % 16) ..
  uint4 x[8];
  auto load = [&](int u) {
    const int key0 = (t0 + u / ns) * kTrKeys + 16 * warp + (lane >> 4), dim = (u % ns) * 64 + 4 * (lane & 15);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = key0 + 2 * i;
      x[i] = j < t.len ? load4<VEC>(key_row(t, kvh, t.lo + j, d), dim, d) : make_uint4(0, 0, 0, 0);
    }
  };
  if (warp < 8) load(0);

  // query digits: chunk s holds dims [64 s, 64 s + 64) of rows a * NR + r
  bool big_q = false;  // a value outside the digits' range
  for (int e = tid; e < NR * ns * 16; e += kQkThreads) {
    const int r = e / (ns * 16), dg = e % (ns * 16), s = dg >> 4;
    const uint4 v = r < nr ? load4<VEC>(qrow(r), 4 * dg, d) : make_uint4(0, 0, 0, 0);
    uint32_t o[4];
    ta_t4(ta_digits((int32_t)v.x), ta_digits((int32_t)v.y), ta_digits((int32_t)v.z), ta_digits((int32_t)v.w), o);
    big_q |= over(v);
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      *reinterpret_cast<uint32_t*>(qpl + s * (4 * NR * 64) + ta_sw(a * NR + r, (dg & 15) >> 2) + 4 * (dg & 3)) = o[a];
    }
  }
  ta_fence_async();
  const bool qover = __syncthreads_or(big_q);
  constexpr int na = 4;  // query digits

  if (warp < 8) {
    bool big = false;
    for (int u = 0; u < total; ++u) {
      const int pb = u & 1, tile = u / ns;
      if (u >= 2) wait(&mma_done[pb], ((u - 2) >> 1) & 1);
      unsigned char* pl = planes + pb * kTrPlanes;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t o[4];
        ta_t4(ta_digits((int32_t)x[i].x), ta_digits((int32_t)x[i].y), ta_digits((int32_t)x[i].z),
              ta_digits((int32_t)x[i].w), o);
        big |= over(x[i]);
        top |= o[3];
        const int r = 16 * warp + 2 * i + (lane >> 4);
        const int at = ta_sw(r, (lane & 15) >> 2) + 4 * (lane & 3);
#pragma unroll
        for (int b = 0; b < 4; ++b) *reinterpret_cast<uint32_t*>(pl + b * kTrPlane + at) = o[b];
      }
      if (u + 1 < total) load(u + 1);
      ta_fence_async();
      const bool anytop = __any_sync(0xffffffffu, top != 0);
      const bool last = (u + 1) % ns == 0;
      const bool anybig = last && __any_sync(0xffffffffu, big);
      if (lane == 0) {
        s_top[pb][warp] = anytop;
        if (last) s_over[tile & 3][warp] = anybig;
        mbar_arrive(&planes_full[pb]);
      }
      if (last) big = false;
    }
  } else if (warp == 12) {
    if (lane == 0) {
      const uint32_t full = ta_idesc(na * NR), low = ta_idesc((na - 1) * NR), one = ta_idesc(NR);
      for (int u = 0; u < total; ++u) {
        const int tile = u / ns, s = u % ns, pb = u & 1;
        if (s == 0 && tile >= 2) wait(&acc_empty[tile & 1], ((tile - 2) >> 1) & 1);
        wait(&planes_full[pb], (u >> 1) & 1);
        fence_after();
        const uint32_t pbase = su32(planes + pb * kTrPlanes), qbase = su32(qpl + s * (4 * NR * 64));
        const uint32_t dcol = tmem + (uint32_t)((tile & 1) * kCols);
        const uint64_t tops = *reinterpret_cast<volatile uint64_t*>(s_top[pb]);
        const int nb = tops ? 4 : 3;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          if (s == 0 && k == 0) {
            // the first products of a tile open its column blocks: digit b
            // adds to the blocks that the digits before it opened and opens
            // block b + na - 1
            mma_i8(dcol, smem_desc_sw64(pbase), smem_desc_sw64(qbase), full, 0);
            for (int b = 1; b < 4; ++b) {
              const uint64_t ad = smem_desc_sw64(pbase + b * kTrPlane);
              if (na > 1) mma_i8(dcol + b * NR, ad, smem_desc_sw64(qbase), low, 1);
              mma_i8(dcol + (b + na - 1) * NR, ad, smem_desc_sw64(qbase + (na - 1) * NR * 64), one, 0);
            }
          } else {
            for (int b = 0; b < nb; ++b)
              mma_i8(dcol + b * NR, smem_desc_sw64(pbase + b * kTrPlane + 32 * k), smem_desc_sw64(qbase + 32 * k), full, 1);
          }
        }
        mma_commit(&mma_done[pb]);
        if (s == ns - 1) {
          mma_commit(&acc_full[tile & 1]);
          mbar_arrive(&acc_full[tile & 1]);  // hands the converters' s_over on
        }
      }
    }
  } else {
    // warps 8-11: accumulator lane (key) 32 (warp % 4) + lane
    const int key = 32 * (warp & 3) + lane;
    int32_t* const sc = reinterpret_cast<int32_t*>(static_cast<unsigned char*>(g.ws)) + t.soff +
                        ((int64_t)kvh * rows + r0) * t.pad;
    for (int tile = 0; tile < t1 - t0; ++tile) {
      wait(&acc_full[tile & 1], (tile >> 1) & 1);
      fence_after();
      const int j = (t0 + tile) * kTrKeys + key;
      const bool slow = qover || *reinterpret_cast<volatile uint64_t*>(s_over[tile & 3]) != 0;
      const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)((tile & 1) * kCols);
      if (!slow) {
        for (int r = 0; r < nr; r += 4) {
          int32_t c[7][4];
#pragma unroll
          for (int b = 0; b < 7; ++b) ta_ld4(taddr + b * NR + r, c[b]);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t cc[7] = {c[0][i], c[1][i], c[2][i], c[3][i], c[4][i], c[5][i], c[6][i]};
            const int32_t sv = requantize(shift_sum(cc));
            if (r + i < nr && j < t.len) sc[(int64_t)(r + i) * t.pad + j] = sv;
          }
        }
      } else if (j < t.len) {
        const int32_t* k = key_row(t, kvh, t.lo + j, d);
        for (int r = 0; r < nr; ++r) {
          const int32_t* q = qrow(r);
          int64_t acc = 0;
          for (int i = 0; i < d; ++i) acc = mac_wide(acc, q[i], k[i]);
          sc[(int64_t)r * t.pad + j] = requantize(acc);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[tile & 1]);
    }
  }
  fence_before();
  __syncthreads();
  if (s_fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == 0) ta_dealloc<kTmem>(tmem);
}

// ---------------------------------------------------------------------------
// softmax: one cluster per row, its keys split over the CTAs in spans of 64
// ---------------------------------------------------------------------------
constexpr int kSmThreads = 256;
constexpr int kSmVec = 4;                                  // keys per thread and step
constexpr int kSmRegs = 4;                                 // steps whose terms stay in registers
constexpr int kSmRegKeys = kSmThreads * kSmVec * kSmRegs;  // keys per CTA of the register form

__device__ __forceinline__ uint64_t sm_warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ int64_t sm_warp_sum(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// REG: every thread keeps its keys' scores, terms and weights in registers;
// else they stay in the score scratch between the passes (longer rows).
template <int NR, bool REG>
__global__ void __launch_bounds__(kSmThreads) tree_softmax(const __grid_constant__ TreeGroup g) {
  cg::cluster_group cl = cg::this_cluster();
  const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  __shared__ uint64_t red[3][kSmThreads / 32], part[3];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = g.Hq / g.Hkv;
  // row of the group: (sequence, KV head, node, head of the KV head's group)
  const int grow = blockIdx.x / CL, si = seq_of(g.row_first, g.nseq, grow);
  const TreeSeq& t = g.seq[si];
  const int rows = t.n * G, lrow = grow - g.row_first[si], kvh = lrow / rows, rr = lrow % rows;
  const uint64_t mask = g.mask[t.node0 + rr / G];
  const int start = first_pos(g, t, mask);
  const int nrb = (rows + NR - 1) / NR, rb = rr / NR, r = rr % NR;
  unsigned char* const ws = static_cast<unsigned char*>(g.ws);
  int32_t* const sc = reinterpret_cast<int32_t*>(ws) + t.soff + (int64_t)lrow * t.pad;
  const int chunks = t.pad / 64;  // the CTA's span: chunks [c0, c1) of 64 keys
  const int c0 = (int)((int64_t)chunks * rank / CL), c1 = (int)((int64_t)chunks * (rank + 1) / CL);
  const int k0 = c0 * 64, k1 = c1 * 64;

  // block and cluster reduction number `i` of the row
  auto reduce = [&](uint64_t v, int i, bool mx) {
    v = mx ? sm_warp_max(v) : (uint64_t)sm_warp_sum((int64_t)v);
    if (lane == 0) red[i][warp] = v;
    __syncthreads();
    v = red[i][lane & (kSmThreads / 32 - 1)];
#pragma unroll
    for (int o = kSmThreads / 64; o > 0; o >>= 1) {
      const uint64_t u = __shfl_xor_sync(0xffffffffu, v, o);
      v = mx ? max(v, u) : v + u;
    }
    if (CL > 1) {
      if (tid == 0) part[i] = v;
      cl.sync();
      v = *cl.map_shared_rank(&part[i], lane < CL ? lane : 0);
      if (lane >= CL) v = 0;
      v = mx ? sm_warp_max(v) : (uint64_t)sm_warp_sum((int64_t)v);
    }
    return v;
  };
  auto key_of = [&](int step) { return k0 + (step * kSmThreads + tid) * kSmVec; };
  // weight digits of four keys into the value kernel's operand tiles
  unsigned char* const wpl = ws + t.woff + (int64_t)(kvh * nrb + rb) * chunks * (3 * NR * 64);
  auto put = [&](int j, const int32_t (&w)[4]) {
    uint32_t o[4];
    ta_t4(ta_digits(w[0]), ta_digits(w[1]), ta_digits(w[2]), ta_digits(w[3]), o);
    unsigned char* tile = wpl + (int64_t)(j >> 6) * (3 * NR * 64);
#pragma unroll
    for (int a = 0; a < 3; ++a)
      *reinterpret_cast<uint32_t*>(tile + ta_sw(a * NR + r, (j & 63) >> 4) + (j & 15)) = o[a];
  };

  ta_wait();
  ta_go();
  if (rank == 0) {
    // the value kernel's sums and counters of this row
    if (t.splits > 1) {
      int64_t* acc = reinterpret_cast<int64_t*>(ws + g.acc_off) + (int64_t)grow * g.d;
      for (int i = tid; i < g.d; i += kSmThreads) acc[i] = 0;
      if (r == 0 && tid < (g.d + 127) / 128)
        reinterpret_cast<uint32_t*>(ws + g.cnt_off)[(t.blk0 + kvh * nrb + rb) * 4 + tid] = 0;
    }
  }
  int32_t v[REG ? kSmRegs : 1][4];
  uint64_t b = 0;
  const int steps = (k1 - k0 + kSmThreads * kSmVec - 1) / (kSmThreads * kSmVec);
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s) {
      const int j = key_of(s);
      if (j < k1) *reinterpret_cast<int4*>(v[s]) = *reinterpret_cast<const int4*>(sc + j);
    }
  }
  // (value, lowest index): the node itself is always attended, so the row's key is never 0
  auto scan = [&](int j, const int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (sees(g, t, mask, start, t.lo + j + i))
        b = max(b, (uint64_t)((uint32_t)x[i] ^ 0x80000000u) << 32 | (uint32_t)~(j + i));
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) scan(key_of(s), v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        scan(j, v[0]);
      }
    }
  }
  b = reduce(b, 0, true);
  const int32_t m = (int32_t)((uint32_t)(b >> 32) ^ 0x80000000u);
  const int mi = (int)~(uint32_t)b;
  // exp terms as u32: the one value of 2^32 (a score equal to the maximum)
  // is coded 2^32 - 1, which no other score gives (the next lower score's
  // term is below 2^32 - 2^15)
  uint64_t sum = 0;
  auto terms = [&](int j, int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t e = sees(g, t, mask, start, t.lo + j + i) ? exp_term(x[i], m) : 0;
      sum += (uint64_t)e;
      x[i] = (int32_t)(uint32_t)(e == kOneAcc ? 0xffffffffu : (uint32_t)e);
    }
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) terms(key_of(s), v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        terms(j, v[0]);
        *reinterpret_cast<int4*>(sc + j) = *reinterpret_cast<const int4*>(v[0]);
      }
    }
  }
  sum = reduce(sum, 1, false);
  uint64_t wsum = 0;
  auto weights = [&](int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = (uint32_t)x[i];
      x[i] = u ? softmax_weight(u == 0xffffffffu ? kOneAcc : (int64_t)u, (int64_t)sum) : 0;
      wsum += (uint64_t)x[i];
    }
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) weights(v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        weights(v[0]);
        *reinterpret_cast<int4*>(sc + j) = *reinterpret_cast<const int4*>(v[0]);
      }
    }
  }
  wsum = reduce(wsum, 2, false);
  // what the roundings left goes to the first maximum (the sum is below 2^31:
  // at most 2^16 and half a unit per key)
  const int32_t left = sub_sat(kOneAct, (int32_t)wsum);
  auto finish = [&](int j, int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i == mi) x[i] = add_sat(x[i], left);
    const int32_t w[4] = {x[0], x[1], x[2], x[3]};
    put(j, w);
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) finish(key_of(s), v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        finish(j, v[0]);
      }
    }
  }
  if (CL > 1) cl.sync();  // every CTA's shared memory stays until it has been read
}

// ---------------------------------------------------------------------------
// weighted values
// ---------------------------------------------------------------------------
template <int NR>
__host__ __device__ constexpr int pv_smem() { return 2 * kTrPlanes + 2 * 3 * NR * 64 + 1024; }

template <int NR>
__global__ void __launch_bounds__(kPvThreads, 2) tree_pv(const __grid_constant__ TreeGroup g) {
  constexpr int kTmem = NR == 16 ? 128 : 256;
  constexpr int kW = 3 * NR * 64;               // one stage's weight tile
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* planes = sm;                   // [2][4 digits][128 dims][64 keys]
  unsigned char* wsm = sm + 2 * kTrPlanes;      // [2][3 NR rows][64 keys]
  __shared__ __align__(8) uint64_t planes_full[2], mma_done[2], acc_full;
  __shared__ uint32_t tmem_holder, s_last;
  __shared__ int s_fail;
  __shared__ __align__(8) unsigned char s_top[2][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int d = g.d, nd = (d + 127) / 128, G = g.Hq / g.Hkv;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&planes_full[i], kTrConv / 32);
      mbar_init(&mma_done[i], 1);
    }
    mbar_init(&acc_full, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_fail = 0;
  }
  if (warp == 0) ta_alloc<kTmem>(&tmem_holder);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_holder;

  // item -> sequence, KV head, row block, dim block, chunks [c0, c1) of 64 keys
  const int si = seq_of(g.pv_first, g.nseq, blockIdx.x);
  const TreeSeq& t = g.seq[si];
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, chunks = t.pad / 64, S = t.splits;
  int it = blockIdx.x - g.pv_first[si];
  const int sp = it % S, db = (it / S) % nd, rb = (it / (S * nd)) % nrb, kvh = it / (S * nd * nrb);
  const int c0 = (int)((int64_t)chunks * sp / S), c1 = (int)((int64_t)chunks * (sp + 1) / S);
  const int r0 = rb * NR, nr = min(NR, rows - r0), total = c1 - c0;
  unsigned char* const ws = static_cast<unsigned char*>(g.ws);
  const unsigned char* const wpl = ws + t.woff + ((int64_t)(kvh * nrb + rb) * chunks + c0) * kW;

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_wait(bar, parity)) s_fail = 1;
  };
  // a converter thread's part of a stage: dim tid % 128, keys 32 (tid / 128) .. + 32
  const int dl = tid & 127, half = (tid >> 7) & 1, dim = db * 128 + dl;
  int32_t x[32];
  auto load = [&](int u) {
    const int j0 = (c0 + u) * 64 + 32 * half;
    if (t.lo + j0 + 32 <= t.ctx && dim < d) {  // cache rows only
      const int32_t* p = t.v + (int64_t)kvh * t.kstride + (int64_t)(t.lo + j0) * d + dim;
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = __ldg(p + (int64_t)i * d);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        x[i] = j0 + i < t.len && dim < d ? value_row(t, kvh, t.lo + j0 + i, d)[dim] : 0;
    }
  };
  // The values do not depend on the softmax: their first stage loads before
  // the wait (this grid starts only after the score kernel has completed, and
  // with it everything before it).
  if (warp < 8) load(0);
  ta_wait();
  ta_go();

  bool big = false;
  if (warp < 8) {
    for (int u = 0; u < total; ++u) {
      const int pb = u & 1;
      if (u >= 2) wait(&mma_done[pb], ((u - 2) >> 1) & 1);
      unsigned char* pl = planes + pb * kTrPlanes;
      for (int e = tid; e < kW / 16; e += kTrConv)
        reinterpret_cast<uint4*>(wsm + pb * kW)[e] = reinterpret_cast<const uint4*>(wpl + (int64_t)u * kW)[e];
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {  // 16 keys: one 16-byte piece of each digit plane
        uint32_t o[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int j = 16 * c + 4 * k;
          uint32_t q[4];
          ta_t4(ta_digits(x[j]), ta_digits(x[j + 1]), ta_digits(x[j + 2]), ta_digits(x[j + 3]), q);
          big |= max(max(x[j], x[j + 1]), max(x[j + 2], x[j + 3])) > kTrMaxDigit;
          top |= q[3];
#pragma unroll
          for (int b = 0; b < 4; ++b) o[b][k] = q[b];
        }
#pragma unroll
        for (int b = 0; b < 4; ++b)
          *reinterpret_cast<uint4*>(pl + b * kTrPlane + ta_sw(dl, 2 * half + c)) =
              make_uint4(o[b][0], o[b][1], o[b][2], o[b][3]);
      }
      if (u + 1 < total) load(u + 1);
      ta_fence_async();
      const bool anytop = __any_sync(0xffffffffu, top != 0);
      if (lane == 0) {
        s_top[pb][warp] = anytop;
        mbar_arrive(&planes_full[pb]);
      }
    }
  } else if (lane == 0) {
    const uint32_t full = ta_idesc(3 * NR), low = ta_idesc(2 * NR), one = ta_idesc(NR);
    for (int u = 0; u < total; ++u) {
      const int pb = u & 1;
      wait(&planes_full[pb], (u >> 1) & 1);
      fence_after();
      const uint32_t pbase = su32(planes + pb * kTrPlanes), wbase = su32(wsm + pb * kW);
      const uint64_t tops = *reinterpret_cast<volatile uint64_t*>(s_top[pb]);
      const int nb = tops ? 4 : 3;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (u == 0 && k == 0) {  // opens the column blocks, as in the score kernel
          mma_i8(tmem, smem_desc_sw64(pbase), smem_desc_sw64(wbase), full, 0);
          for (int b = 1; b < 4; ++b) {
            const uint64_t ad = smem_desc_sw64(pbase + b * kTrPlane);
            mma_i8(tmem + b * NR, ad, smem_desc_sw64(wbase), low, 1);
            mma_i8(tmem + (b + 2) * NR, ad, smem_desc_sw64(wbase + 2 * NR * 64), one, 0);
          }
        } else {
          for (int b = 0; b < nb; ++b)
            mma_i8(tmem + b * NR, smem_desc_sw64(pbase + b * kTrPlane + 32 * k), smem_desc_sw64(wbase + 32 * k), full, 1);
        }
      }
      mma_commit(&mma_done[pb]);
      if (u == total - 1) mma_commit(&acc_full);
    }
    wait(&acc_full, 0);
  }
  // a value outside the digits' range: the block's sums are taken directly
  const bool slow = __syncthreads_or(big);
  fence_after();
  // ---- the block's partial sums: lane dl, rows split over the two halves
  const bool one_split = S == 1;
  int64_t* const acc = reinterpret_cast<int64_t*>(ws + g.acc_off) +
                       ((int64_t)g.row_first[si] + (int64_t)kvh * rows + r0) * d;
  auto orow = [&](int r) {
    const int rr = r0 + r;
    return g.out + ((int64_t)(t.node0 + rr / G) * g.Hq + kvh * G + rr % G) * d;
  };
  auto give = [&](int r, int64_t v) {
    if (r >= nr || dim >= d) return;
    if (one_split) orow(r)[dim] = requantize(v);
    else atomicAdd(reinterpret_cast<unsigned long long*>(acc + (int64_t)r * d + dim), (unsigned long long)v);
  };
  if (warp < 8) {
    if (!slow) {
      const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
      for (int r = half * (NR / 2); r < min(nr, (half + 1) * (NR / 2)); r += 4) {
        int32_t c[6][4];
#pragma unroll
        for (int b = 0; b < 6; ++b) ta_ld4(taddr + b * NR + r, c[b]);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t cc[7] = {c[0][i], c[1][i], c[2][i], c[3][i], c[4][i], c[5][i], 0};
          give(r + i, shift_sum(cc));
        }
      }
    } else {
      for (int r = half; r < nr; r += 2) {
        int64_t sum = 0;
        for (int j = c0 * 64; j < min(c1 * 64, t.len) && dim < d; ++j) {
          const unsigned char* tile = wpl + (int64_t)((j >> 6) - c0) * kW;
          int32_t w = 0;
          for (int a = 2; a >= 0; --a)
            w = w * 256 + (int8_t)tile[ta_sw(a * NR + r, (j & 63) >> 4) + (j & 15)];
          sum = mac_wide(sum, w, value_row(t, kvh, t.lo + j, d)[dim]);
        }
        give(r, sum);
      }
    }
  }
  if (!one_split) {
    // the block that arrives last rounds the sums of all splits (wrapping
    // integer sums: the order of the additions does not matter)
    __threadfence();
    __syncthreads();
    if (tid == 0)
      s_last = atomicAdd(reinterpret_cast<uint32_t*>(ws + g.cnt_off) + (t.blk0 + kvh * nrb + rb) * 4 + db, 1u) ==
               (uint32_t)S - 1;
    __syncthreads();
    if (s_last) {
      __threadfence();
      if (warp < 8 && dim < d)
        for (int r = half; r < nr; r += 2) orow(r)[dim] = requantize(__ldcg(reinterpret_cast<const long long*>(acc + (int64_t)r * d + dim)));
    }
  }
  fence_before();
  __syncthreads();
  if (s_fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == 0) ta_dealloc<kTmem>(tmem);
}

template <int NR, bool VEC>
void qk_attr() {
  cudaFuncSetAttribute(tree_qk<NR, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, qk_smem<NR>(8));
}

}  // namespace

void tree_attn_init() {
  qk_attr<16, true>();
  qk_attr<16, false>();
  qk_attr<32, true>();
  qk_attr<32, false>();
  cudaFuncSetAttribute(tree_pv<16>, cudaFuncAttributeMaxDynamicSharedMemorySize, pv_smem<16>());
  cudaFuncSetAttribute(tree_pv<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, pv_smem<32>());
}

int tree_attn_error_flag(bool reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_tree_err, sizeof(int));
  if (reset && v) {
    int z = 0;
    cudaMemcpyToSymbol(g_tree_err, &z, sizeof(int));
  }
  return v;
}

size_t tree_attn_plan(TreeGroup& g) {
  constexpr int kSms = 148;
  const int G = g.Hq / g.Hkv, nd = (g.d + 127) / 128;
  int maxrows = 0;
  for (int i = 0; i < g.nseq; ++i) maxrows = std::max(maxrows, g.seq[i].n * G);
  g.nr = maxrows <= 16 ? 16 : 32;
  int64_t soff = 0, tiles = 0, vitems = 0;
  int rows = 0, blocks = 0;
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    // the shallowest node's window is the lowest of the tree
    t.lo = g.window > 0 && t.ctx + 1 > g.window ? std::min(t.ctx, t.ctx + 1 - g.window) : 0;
    t.len = t.ctx - t.lo + t.n;
    t.pad = (t.len + 63) & ~63;
    t.soff = soff;
    const int nrb = (t.n * G + g.nr - 1) / g.nr;
    soff += (int64_t)t.pad * t.n * g.Hq;
    g.row_first[i] = rows;
    rows += t.n * g.Hq;
    t.blk0 = blocks;
    blocks += g.Hkv * nrb;
    tiles += (int64_t)g.Hkv * nrb * ((t.len + kTrKeys - 1) / kTrKeys);
    vitems += (int64_t)g.Hkv * nrb * nd * (t.pad / 64);
  }
  // key tiles of one score item, key chunks of one value item: enough items
  // for two waves, no more than needed
  g.qk_tiles = (int)std::max<int64_t>(1, std::min<int64_t>(16, tiles / (2 * kSms)));
  const int chunks_per = (int)std::max<int64_t>(2, std::min<int64_t>(kTrSplitKeys / 64, vitems / (2 * kSms)));
  int64_t off = soff * 4;
  int qk = 0, pv = 0;
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    const int nrb = (t.n * G + g.nr - 1) / g.nr, chunks = t.pad / 64;
    t.splits = (chunks + chunks_per - 1) / chunks_per;
    off = (off + 1023) & ~(int64_t)1023;
    t.woff = off;
    off += (int64_t)g.Hkv * nrb * chunks * (3 * g.nr * 64);
    g.qk_first[i] = qk;
    qk += g.Hkv * nrb * (((t.len + kTrKeys - 1) / kTrKeys + g.qk_tiles - 1) / g.qk_tiles);
    g.pv_first[i] = pv;
    pv += g.Hkv * nrb * nd * t.splits;
  }
  g.qk_items = qk;
  g.pv_items = pv;
  g.rows = rows;
  off = (off + 255) & ~(int64_t)255;
  g.acc_off = off;
  off += (int64_t)rows * g.d * 8;
  g.cnt_off = off;
  off += (int64_t)blocks * 4 * 4;
  return (size_t)((off + 255) & ~(int64_t)255);
}

template <int NR>
static void tree_launch(const TreeGroup& g, bool vec, cudaStream_t s) {
  const int ns = (g.d + 63) / 64;
  if (vec) ta_launch(tree_qk<NR, true>, dim3(g.qk_items), dim3(kQkThreads), qk_smem<NR>(ns), 1, s, g);
  else ta_launch(tree_qk<NR, false>, dim3(g.qk_items), dim3(kQkThreads), qk_smem<NR>(ns), 1, s, g);
  // CTAs per row: the register form's keys at most, and enough CTAs to fill the GPU
  int pad = 0;
  for (int i = 0; i < g.nseq; ++i) pad = std::max(pad, g.seq[i].pad);
  int CL = 1;
  while (CL < 8 && (pad > CL * kSmRegKeys || ((int64_t)g.rows * CL < 4 * 148 && pad > CL * 1024))) CL *= 2;
  // a CTA's span is a whole number of 64-key chunks, so it may exceed pad / CL by less than 64 keys
  if ((pad / 64 + CL - 1) / CL * 64 <= kSmRegKeys)
    ta_launch(tree_softmax<NR, true>, dim3(CL * g.rows), dim3(kSmThreads), 0, CL, s, g);
  else
    ta_launch(tree_softmax<NR, false>, dim3(CL * g.rows), dim3(kSmThreads), 0, CL, s, g);
  ta_launch(tree_pv<NR>, dim3(g.pv_items), dim3(kPvThreads), pv_smem<NR>(), 1, s, g);
}

void launch_tree_attn(const TreeGroup& g, cudaStream_t s) {
  uintptr_t bits = reinterpret_cast<uintptr_t>(g.q);
  for (int i = 0; i < g.nseq; ++i)
    bits |= reinterpret_cast<uintptr_t>(g.seq[i].k) | reinterpret_cast<uintptr_t>(g.seq[i].kt);
  const bool vec = g.d % 4 == 0 && (bits & 15) == 0;
  if (g.nr == 16) tree_launch<16>(g, vec, s);
  else tree_launch<32>(g, vec, s);
}

}  // namespace rdet
