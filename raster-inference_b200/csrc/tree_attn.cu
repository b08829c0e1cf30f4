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
constexpr int kTrConv = 512;           // converter threads (warps 0-15)
constexpr int kTrConvWarps = kTrConv / 32;
constexpr int kQkThreads = 672;        // + warps 16-19 drain the accumulators, warp 20 issues the MMAs
constexpr int kPvThreads = 544;        // + warp 16 issues the MMAs
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
__device__ __forceinline__ int32_t max4(int32_t m, const uint4& v) {
  return max(max(max(m, (int32_t)v.x), max((int32_t)v.y, (int32_t)v.z)), (int32_t)v.w);
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
__global__ void __launch_bounds__(kQkThreads, 1) tree_qk(const __grid_constant__ TreeGroup g) {
  constexpr int kCols = 7 * NR, kTmem = NR == 16 ? 256 : 512;
  constexpr int kSets = 2;                      // stages a converter holds in registers
  constexpr int na = 4;                         // query digits
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* planes = sm;                   // [2][4 digits][128 keys][64 B]
  unsigned char* qpl = sm + 2 * kTrPlanes;      // [chunk][4 NR rows][64 B]
  __shared__ __align__(8) uint64_t planes_full[2], mma_done[2], acc_full[2], acc_empty[2], last_full;
  __shared__ uint32_t tmem_holder;
  __shared__ int s_fail;
  // last stage (plus 1) of each plane buffer that uses digit 3
  __shared__ int s_top[2];
  // last tile (plus 1) with a value outside the digits' range.  Four slots: a
  // converter runs at most two stages, so at most two tiles, ahead of the MMAs,
  // and those at most two tiles ahead of the drain that reads the slot.
  __shared__ int s_over[4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // item -> sequence, KV head, row block, key tiles [t0, t1)
  const int si = seq_of(g.qk_first, g.nseq, blockIdx.x);
  const TreeSeq t = g.seq[si];
  const int d = g.d, ns = (d + 63) / 64, G = g.G, Hq = g.Hq;
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, tiles = (t.len + kTrKeys - 1) / kTrKeys, qt = g.qk_tiles;
  const int it = blockIdx.x - g.qk_first[si];
  const int blk = it / t.qk_per, t0 = (it - blk * t.qk_per) * qt, t1 = min(tiles, t0 + qt);
  const int kvh = blk / nrb, rb = blk - kvh * nrb;
  const int r0 = rb * NR, nr = min(NR, rows - r0);
  const int total = (t1 - t0) * ns;
  const int32_t* const kc = t.k + (int64_t)kvh * t.kstride;
  const int32_t* const kt = t.kt + (int64_t)kvh * t.tstride;
  const int32_t* const qb = g.q + ((int64_t)t.node0 * Hq + kvh * G) * d;
  int32_t* const sc = static_cast<int32_t*>(g.ws) + t.soff + ((int64_t)kvh * rows + r0) * t.pad;
  ta_wait();
  ta_go();

  // a converter thread's part of stage (tile, s): keys 8 warp + 2 i + lane / 16, dims 64 s + 4 (lane % 16) ..
  const uint32_t lkey = 8 * warp + (lane >> 4), off0 = (lkey * (uint32_t)d + 4 * (lane & 15)) * 4, step = 8 * (uint32_t)d;
  auto load = [&](uint4 (&x)[4], int tile, int s) {
    const int key0 = t.lo + (t0 + tile) * kTrKeys;
    if (VEC && key0 + kTrKeys <= t.ctx && s * 64 + 64 <= d) {  // cache rows and dims only
      const unsigned char* base = reinterpret_cast<const unsigned char*>(kc + (int64_t)key0 * d + s * 64);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __ldg(reinterpret_cast<const uint4*>(base + (off0 + i * step)));
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = key0 + (int)lkey + 2 * i;
      const int32_t* p = key < t.ctx ? kc + (int64_t)key * d : kt + (int64_t)(key - t.ctx) * d;
      x[i] = key < t.lo + t.len ? load4<VEC>(p, s * 64 + 4 * (lane & 15), d) : make_uint4(0, 0, 0, 0);
    }
  };
  uint4 x[kSets][4];
  int lt = 0, ls = 0;  // next stage to load
  auto next = [&](uint4 (&y)[4]) {
    if (lt < t1 - t0) load(y, lt, ls);
    if (++ls == ns) { ls = 0; ++lt; }
  };
  if (warp < kTrConvWarps) {
#pragma unroll
    for (int i = 0; i < kSets; ++i) next(x[i]);
  }

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&planes_full[i], kTrConvWarps);
      mbar_init(&mma_done[i], 1);
      mbar_init(&acc_full[i], 2);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&last_full, 2);
    s_top[0] = s_top[1] = s_over[0] = s_over[1] = s_over[2] = s_over[3] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_fail = 0;
  }
  if (warp == 20) ta_alloc<kTmem>(&tmem_holder);
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!ta_mbar_wait(bar, parity)) s_fail = 1;
  };
  // query row r (node * G + head of the group) of this block
  auto qrow = [&](int r) {
    const int rr = r0 + r, node = rr / G;
    return qb + ((int64_t)node * Hq + (rr - node * G)) * d;
  };
  // query digits: chunk s holds dims [64 s, 64 s + 64) of rows a * NR + r.
  // One row per warp and step, 16-byte pieces lane + 32 i of the row.
  int32_t qmax = INT32_MIN;
  for (int r = warp; r < NR; r += kQkThreads / 32) {
    const int32_t* q = r < nr ? qrow(r) : qb;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = r < nr && lane + 32 * i < ns * 16 ? load4<VEC>(q, 4 * (lane + 32 * i), d) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int dg = lane + 32 * i;
      if (dg >= ns * 16) break;
      uint32_t o[4];
      ta_t4(ta_digits((int32_t)v[i].x), ta_digits((int32_t)v[i].y), ta_digits((int32_t)v[i].z),
            ta_digits((int32_t)v[i].w), o);
      qmax = max4(qmax, v[i]);
#pragma unroll
      for (int a = 0; a < 4; ++a)
        *reinterpret_cast<uint32_t*>(qpl + (dg >> 4) * (4 * NR * 64) + ta_sw(a * NR + r, (dg & 15) >> 2) +
                                     4 * (dg & 3)) = o[a];
    }
  }
  ta_fence_async();
  fence_before();
  const bool qover = __syncthreads_or(qmax > kTrMaxDigit);
  fence_after();
  const uint32_t tmem = tmem_holder;

  // scores of rows [ra, re) of a drained tile, this thread's key
  const int lk = 32 * (warp & 3) + lane;
  auto drain = [&](int tile, int ra, int re) {
    const int j = (t0 + tile) * kTrKeys + lk;
    const bool slow = qover || *reinterpret_cast<volatile int*>(&s_over[tile & 3]) == tile + 1;
    const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + (uint32_t)((tile & 1) * kCols);
    int32_t* out = sc + (int64_t)ra * t.pad + j;
    if (!slow) {
      for (int r = ra; r < re; r += 4) {
        int32_t c[7][4];
#pragma unroll
        for (int b = 0; b < 7; ++b) ta_ld4(taddr + b * NR + r, c[b]);
        tmem_wait_ld();
        int32_t sv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t cc[7] = {c[0][i], c[1][i], c[2][i], c[3][i], c[4][i], c[5][i], c[6][i]};
          sv[i] = requantize(shift_sum(cc));
        }
        if (j < t.len) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (r + i < re) out[(int64_t)i * t.pad] = sv[i];
        }
        out += 4 * (int64_t)t.pad;
      }
    } else if (j < t.len) {
      const int key = t.lo + j;
      const int32_t* k = key < t.ctx ? kc + (int64_t)key * d : kt + (int64_t)(key - t.ctx) * d;
      for (int r = ra; r < re; ++r, out += t.pad) {
        const int32_t* q = qrow(r);
        int64_t acc = 0;
        for (int i = 0; i < d; ++i) acc = mac_wide(acc, q[i], k[i]);
        *out = requantize(acc);
      }
    }
  };
  // The last tile is drained by all five groups of four warps, a fifth of the
  // rows each (the converters are done by then).
  const int last_tile = t1 - t0 - 1, fifth = ((nr + 19) / 20) * 4;

  if (warp < kTrConvWarps) {
    int tile = 0, s = 0;
    // rows 8 warp + 2 i + lane / 16 of the planes: bits 1-2 of the row are i
    const int ch = (lane & 15) >> 2;
    unsigned char* const pl0 = planes + lkey * 64 + 4 * (lane & 3);
    unsigned char* const plx[4] = {pl0 + (ch << 4), pl0 + 128 + ((ch ^ 1) << 4), pl0 + 256 + ((ch ^ 2) << 4),
                                   pl0 + 384 + ((ch ^ 3) << 4)};
    for (int u = 0; u < total; u += kSets) {
#pragma unroll
      for (int p = 0; p < kSets; ++p) {
        if (u + p < total) {
          if (u + p >= 2) wait(&mma_done[p], ((u + p - 2) >> 1) & 1);
          uint32_t top = 0;
          int32_t mx = INT32_MIN;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t o[4];
            ta_t4(ta_digits((int32_t)x[p][i].x), ta_digits((int32_t)x[p][i].y), ta_digits((int32_t)x[p][i].z),
                  ta_digits((int32_t)x[p][i].w), o);
            mx = max4(mx, x[p][i]);
            top |= o[3];
#pragma unroll
            for (int b = 0; b < 4; ++b) *reinterpret_cast<uint32_t*>(plx[i] + p * kTrPlanes + b * kTrPlane) = o[b];
          }
          if (top) s_top[p] = u + p + 1;
          if (mx > kTrMaxDigit) s_over[tile & 3] = tile + 1;
          ta_fence_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&planes_full[p]);
          next(x[p]);
          if (++s == ns) { s = 0; ++tile; }
        }
      }
    }
    // a barrier of its own: a converter does not follow acc_full's phases, and
    // a parity tells neighbouring phases apart only
    wait(&last_full, 0);
    fence_after();
    const int ra = fifth * (1 + (warp >> 2));
    if (ra < nr) drain(last_tile, ra, min(nr, ra + fifth));
  } else if (warp == 20) {
    if (lane == 0) {
      const uint32_t full = ta_idesc(na * NR), low = ta_idesc((na - 1) * NR), one = ta_idesc(NR);
      const uint64_t pdesc = smem_desc_sw64(su32(planes)), qdesc = smem_desc_sw64(su32(qpl));
      int tile = 0, s = 0;
      for (int u = 0; u < total; ++u) {
        const int pb = u & 1;
        if (s == 0 && tile >= 2) wait(&acc_empty[tile & 1], ((tile - 2) >> 1) & 1);
        wait(&planes_full[pb], (u >> 1) & 1);
        fence_after();
        const uint64_t pd = ta_adv(pdesc, pb * kTrPlanes), qd = ta_adv(qdesc, s * (4 * NR * 64));
        const uint32_t dcol = tmem + (uint32_t)((tile & 1) * kCols);
        const bool top = *reinterpret_cast<volatile int*>(&s_top[pb]) == u + 1;
        if (s == 0) {
          // the first products of a tile open its column blocks: digit b adds
          // to the blocks that the digits before it opened and opens block
          // b + na - 1
          mma_i8(dcol, pd, qd, full, 0);
#pragma unroll
          for (int b = 1; b < 4; ++b) {
            mma_i8(dcol + b * NR, ta_adv(pd, b * kTrPlane), qd, low, 1);
            mma_i8(dcol + (b + na - 1) * NR, ta_adv(pd, b * kTrPlane), ta_adv(qd, (na - 1) * NR * 64), one, 0);
          }
        } else {
#pragma unroll
          for (int b = 0; b < 3; ++b) mma_i8(dcol + b * NR, ta_adv(pd, b * kTrPlane), qd, full, 1);
          if (top) mma_i8(dcol + 3 * NR, ta_adv(pd, 3 * kTrPlane), qd, full, 1);
        }
#pragma unroll
        for (int b = 0; b < 3; ++b) mma_i8(dcol + b * NR, ta_adv(pd, b * kTrPlane + 32), ta_adv(qd, 32), full, 1);
        if (top) mma_i8(dcol + 3 * NR, ta_adv(pd, 3 * kTrPlane + 32), ta_adv(qd, 32), full, 1);
        mma_commit(&mma_done[pb]);
        if (s == ns - 1) {
          mma_commit(&acc_full[tile & 1]);
          mbar_arrive(&acc_full[tile & 1]);  // hands the converters' s_over on
          if (u == total - 1) {
            mma_commit(&last_full);
            mbar_arrive(&last_full);
          }
          s = 0;
          ++tile;
        } else {
          ++s;
        }
      }
    }
  } else {
    // warps 16-19: accumulator lane (key) 32 (warp % 4) + lane
    for (int tile = 0; tile <= last_tile; ++tile) {
      wait(&acc_full[tile & 1], (tile >> 1) & 1);
      fence_after();
      drain(tile, 0, tile == last_tile ? min(nr, fifth) : nr);
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[tile & 1]);
    }
  }
  fence_before();
  __syncthreads();
  if (s_fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == 20) ta_dealloc<kTmem>(tmem);
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
  const int G = g.G;
  // row of the group: (sequence, KV head, node, head of the KV head's group)
  const int grow = blockIdx.x / CL, si = seq_of(g.row_first, g.nseq, grow);
  const TreeSeq t = g.seq[si];
  const int rows = t.n * G, lrow = grow - g.row_first[si], kvh = lrow / rows, rr = lrow - kvh * rows;
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
  // which of the keys j .. j + 3 the row attends
  auto seen = [&](int j) -> uint32_t {
    const int key = t.lo + j;
    if (key >= start && key + 3 < t.ctx) return 15u;
    uint32_t m = 0;
    for (int i = 0; i < 4; ++i) m |= sees(g, t, mask, start, key + i) ? 1u << i : 0u;
    return m;
  };
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

  int32_t v[REG ? kSmRegs : 1][4];
  uint32_t vis[REG ? kSmRegs : 1];
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s) vis[s] = key_of(s) < k1 ? seen(key_of(s)) : 0u;
  }
  ta_wait();
  ta_go();
  const int steps = (k1 - k0 + kSmThreads * kSmVec - 1) / (kSmThreads * kSmVec);
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) *reinterpret_cast<int4*>(v[s]) = *reinterpret_cast<const int4*>(sc + key_of(s));
  }
  // the thread's first maximum: its keys come in ascending order
  int32_t bv = INT32_MIN, bj = -1;
  auto scan = [&](int j, uint32_t m, const int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((m >> i & 1) && (x[i] > bv || bj < 0)) { bv = x[i]; bj = j + i; }
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s) scan(key_of(s), vis[s], v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        scan(j, seen(j), v[0]);
      }
    }
  }
  // (value, lowest index): the node itself is always attended, so the row's key is never 0
  const uint64_t b = reduce(bj >= 0 ? (uint64_t)((uint32_t)bv ^ 0x80000000u) << 32 | (uint32_t)~bj : 0, 0, true);
  const int32_t m = (int32_t)((uint32_t)(b >> 32) ^ 0x80000000u);
  const int mi = (int)~(uint32_t)b;
  // exp terms as u32: the one value of 2^32 (a score equal to the maximum)
  // is coded 2^32 - 1, which no other score gives (the next lower score's
  // term is below 2^32 - 2^15)
  uint64_t sum = 0;
  auto terms = [&](uint32_t mk, int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t D = (uint32_t)m - (uint32_t)x[i];  // below the maximum by D
      uint64_t e = 0;
      if ((mk >> i & 1) && D < (16u << 16)) e = exp_term_below(D);
      sum += e;
      x[i] = (int32_t)(uint32_t)(e >> 32 ? 0xffffffffu : (uint32_t)e);
    }
  };
  if (REG) {
#pragma unroll
    for (int s = 0; s < kSmRegs; ++s)
      if (key_of(s) < k1) terms(vis[s], v[s]);
  } else {
    for (int s = 0; s < steps; ++s) {
      const int j = key_of(s);
      if (j < k1) {
        *reinterpret_cast<int4*>(v[0]) = *reinterpret_cast<const int4*>(sc + j);
        terms(seen(j), v[0]);
        *reinterpret_cast<int4*>(sc + j) = *reinterpret_cast<const int4*>(v[0]);
      }
    }
  }
  sum = reduce(sum, 1, false);
  const uint32_t inv = softmax_inverse(sum);
  uint64_t wsum = 0;
  auto weights = [&](int32_t* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = softmax_weight_coded((uint32_t)x[i], inv, sum);
      wsum += (uint32_t)x[i];
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
// weighted values: one cluster per (sequence, KV head, row block, block of 128
// dims), its keys split over the CTAs in chunks of 64; the partial i64 sums
// meet in distributed shared memory
// ---------------------------------------------------------------------------
template <int NR>
__host__ __device__ constexpr int pv_smem() { return 2 * kTrPlanes + 2 * 3 * NR * 64 + 1024; }

template <int NR>
__global__ void __launch_bounds__(kPvThreads, 1) tree_pv(const __grid_constant__ TreeGroup g) {
  constexpr int kTmem = NR == 16 ? 128 : 256;
  constexpr int kW = 3 * NR * 64;               // one stage's weight tile
  extern __shared__ __align__(16) unsigned char tr_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(tr_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* planes = sm;                   // [2][4 digits][128 dims][64 keys]
  unsigned char* wsm = sm + 2 * kTrPlanes;      // [2][3 NR rows][64 keys]
  int64_t* const pacc = reinterpret_cast<int64_t*>(sm);  // [NR][128] partial sums, after the last MMA
  __shared__ __align__(8) uint64_t planes_full[2], mma_done[2], acc_full;
  __shared__ uint32_t tmem_holder;
  __shared__ int s_fail;
  __shared__ int s_top[2];  // last stage (plus 1) of each plane buffer that uses digit 3
  cg::cluster_group cl = cg::this_cluster();
  const int S = (int)cl.num_blocks(), sp = (int)cl.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int item = blockIdx.x / S, si = seq_of(g.pv_first, g.nseq, item);
  const TreeSeq t = g.seq[si];
  const int d = g.d, nd = (d + 127) / 128, G = g.G, Hq = g.Hq;
  const int rows = t.n * G, nrb = (rows + NR - 1) / NR, chunks = t.pad / 64;
  const int it = item - g.pv_first[si];
  const int blk = it / nd, db = it - blk * nd, kvh = blk / nrb, rb = blk - kvh * nrb;
  const int c0 = (int)((int64_t)chunks * sp / S), c1 = (int)((int64_t)chunks * (sp + 1) / S);
  const int r0 = rb * NR, nr = min(NR, rows - r0), total = c1 - c0;
  const unsigned char* const wpl =
      static_cast<unsigned char*>(g.ws) + t.woff + ((int64_t)blk * chunks + c0) * kW;
  const int32_t* const vc = t.v + (int64_t)kvh * t.kstride;
  const int32_t* const vt = t.vt + (int64_t)kvh * t.tstride;

  // a converter thread's part of a stage: dim tid % 128, keys 16 (tid / 128) .. + 16
  const int dl = tid & 127, quarter = (tid >> 7) & 3, dim = db * 128 + dl;
  const uint32_t off0 = ((uint32_t)(16 * quarter) * d + dl) * 4, step = 4 * (uint32_t)d;
  auto load = [&](int32_t (&x)[16], int u) {
    const int key0 = t.lo + (c0 + u) * 64;
    if (key0 + 64 <= t.ctx && db * 128 + 128 <= d) {  // cache rows and dims only
      const unsigned char* base = reinterpret_cast<const unsigned char*>(vc + (int64_t)key0 * d + db * 128);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __ldg(reinterpret_cast<const int32_t*>(base + (off0 + i * step)));
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = key0 + 16 * quarter + i;
        const int32_t* p = key < t.ctx ? vc + (int64_t)key * d : vt + (int64_t)(key - t.ctx) * d;
        x[i] = key < t.lo + t.len && dim < d ? p[dim] : 0;
      }
    }
  };
  int32_t x[2][16];  // two stages in flight
  uint4 wv;
  auto load_w = [&](int u) {
    if (tid < kW / 16) wv = reinterpret_cast<const uint4*>(wpl + (int64_t)u * kW)[tid];
  };
  static_assert(kW / 16 <= kTrConv, "one 16-byte piece of a weight tile per converter thread");
  // The values do not depend on the softmax: their first stage loads before
  // the wait (this grid starts only after the score kernel has completed, and
  // with it everything before it).
  if (warp < kTrConvWarps) {
    if (total > 0) load(x[0], 0);
    if (total > 1) load(x[1], 1);
  }
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&planes_full[i], kTrConvWarps);
      mbar_init(&mma_done[i], 1);
    }
    mbar_init(&acc_full, 1);
    s_top[0] = s_top[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    s_fail = 0;
  }
  if (warp == kTrConvWarps) ta_alloc<kTmem>(&tmem_holder);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_holder;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!ta_mbar_wait(bar, parity)) s_fail = 1;
  };

  int32_t mx = INT32_MIN;  // of the thread's values
  if (warp < kTrConvWarps) {
    for (int u0 = 0; u0 < total; u0 += 2) {
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int u = u0 + p;
        if (u < total) {
          if (u >= 2) wait(&mma_done[p], ((u - 2) >> 1) & 1);
          unsigned char* pl = planes + p * kTrPlanes + ta_sw(dl, quarter);
          uint32_t o[4][4], top = 0;  // one 16-byte piece of each digit plane
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int32_t x0 = x[p][4 * k], x1 = x[p][4 * k + 1], x2 = x[p][4 * k + 2], x3 = x[p][4 * k + 3];
            uint32_t q[4];
            ta_t4(ta_digits(x0), ta_digits(x1), ta_digits(x2), ta_digits(x3), q);
            mx = max(max(max(mx, x0), max(x1, x2)), x3);
            top |= q[3];
#pragma unroll
            for (int b = 0; b < 4; ++b) o[b][k] = q[b];
          }
#pragma unroll
          for (int b = 0; b < 4; ++b)
            *reinterpret_cast<uint4*>(pl + b * kTrPlane) = make_uint4(o[b][0], o[b][1], o[b][2], o[b][3]);
          if (u == 0) {
            ta_wait();  // the weights
            load_w(0);
          }
          if (tid < kW / 16) reinterpret_cast<uint4*>(wsm + p * kW)[tid] = wv;
          if (top) s_top[p] = u + 1;
          ta_fence_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&planes_full[p]);
          if (u + 1 < total) load_w(u + 1);
          if (u + 2 < total) load(x[p], u + 2);
        }
      }
    }
  } else if (lane == 0 && total > 0) {
    ta_wait();  // the converters' first stage waits for the weights: not within a bounded wait
    const uint32_t full = ta_idesc(3 * NR), low = ta_idesc(2 * NR), one = ta_idesc(NR);
    const uint64_t pdesc = smem_desc_sw64(su32(planes)), wdesc = smem_desc_sw64(su32(wsm));
    for (int u = 0; u < total; ++u) {
      const int pb = u & 1;
      wait(&planes_full[pb], (u >> 1) & 1);
      fence_after();
      const uint64_t pd = ta_adv(pdesc, pb * kTrPlanes), wd = ta_adv(wdesc, pb * kW);
      const bool top = *reinterpret_cast<volatile int*>(&s_top[pb]) == u + 1;
      if (u == 0) {  // opens the column blocks, as in the score kernel
        mma_i8(tmem, pd, wd, full, 0);
#pragma unroll
        for (int b = 1; b < 4; ++b) {
          mma_i8(tmem + b * NR, ta_adv(pd, b * kTrPlane), wd, low, 1);
          mma_i8(tmem + (b + 2) * NR, ta_adv(pd, b * kTrPlane), ta_adv(wd, 2 * NR * 64), one, 0);
        }
      } else {
#pragma unroll
        for (int b = 0; b < 3; ++b) mma_i8(tmem + b * NR, ta_adv(pd, b * kTrPlane), wd, full, 1);
        if (top) mma_i8(tmem + 3 * NR, ta_adv(pd, 3 * kTrPlane), wd, full, 1);
      }
#pragma unroll
      for (int b = 0; b < 3; ++b) mma_i8(tmem + b * NR, ta_adv(pd, b * kTrPlane + 32), ta_adv(wd, 32), full, 1);
      if (top) mma_i8(tmem + 3 * NR, ta_adv(pd, 3 * kTrPlane + 32), ta_adv(wd, 32), full, 1);
      mma_commit(&mma_done[pb]);
      if (u == total - 1) mma_commit(&acc_full);
    }
    wait(&acc_full, 0);
  }
  // a value outside the digits' range: the block's sums are taken directly
  const bool slow = __syncthreads_or(mx > kTrMaxDigit);
  ta_wait();
  ta_go();
  fence_after();
  // ---- the block's partial sums: lane dl, rows split over the four quarters
  auto orow = [&](int r) {
    const int rr = r0 + r, node = rr / G;
    return g.out + ((int64_t)(t.node0 + node) * Hq + kvh * G + (rr - node * G)) * d;
  };
  auto give = [&](int r, int64_t v) {
    if (r >= nr) return;
    if (S > 1) pacc[r * 128 + dl] = v;
    else if (dim < d) orow(r)[dim] = requantize(v);
  };
  if (warp < kTrConvWarps) {
    constexpr int kQ = NR / 4;
    if (total == 0) {
      for (int r = quarter; r < nr; r += 4) give(r, 0);
    } else if (!slow) {
      const uint32_t taddr = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
      for (int r = quarter * kQ; r < min(nr, (quarter + 1) * kQ); r += 4) {
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
      for (int r = quarter; r < nr; r += 4) {
        int64_t sum = 0;
        for (int j = c0 * 64; j < min(c1 * 64, t.len) && dim < d; ++j) {
          const unsigned char* tile = wpl + (int64_t)((j >> 6) - c0) * kW;
          int32_t w = 0;
          for (int a = 2; a >= 0; --a)
            w = w * 256 + (int8_t)tile[ta_sw(a * NR + r, (j & 63) >> 4) + (j & 15)];
          const int key = t.lo + j;
          const int32_t* p = key < t.ctx ? vc + (int64_t)key * d : vt + (int64_t)(key - t.ctx) * d;
          sum = mac_wide(sum, w, p[dim]);
        }
        give(r, sum);
      }
    }
  }
  fence_before();
  if (S > 1) {
    cl.sync();
    // rank sp rounds every S-th group of 32 sums of the block
    for (int e = warp * S + sp; e < nr * 4 && warp < kTrConvWarps; e += kTrConvWarps * S) {
      const int r = e >> 2, c = (e & 3) * 32 + lane;
      int64_t v[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) v[q] = q < S ? *cl.map_shared_rank(&pacc[r * 128 + c], q) : 0;
#pragma unroll
      for (int q = 1; q < 16; ++q) v[0] += v[q];
      if (db * 128 + c < d) orow(r)[db * 128 + c] = requantize(v[0]);
    }
    cl.sync();  // every CTA's shared memory stays until it has been read
  } else {
    __syncthreads();
  }
  if (s_fail && tid == 0) atomicExch(&g_tree_err, 1);
  fence_after();
  if (warp == kTrConvWarps) ta_dealloc<kTmem>(tmem);
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
  cudaFuncSetAttribute(tree_pv<16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  cudaFuncSetAttribute(tree_pv<32>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
  const int G = g.G = g.Hq / g.Hkv, nd = (g.d + 127) / 128;
  int maxrows = 0;
  for (int i = 0; i < g.nseq; ++i) maxrows = std::max(maxrows, g.seq[i].n * G);
  g.nr = maxrows <= 16 ? 16 : 32;
  int64_t soff = 0, tiles = 0;
  int rows = 0, pv = 0, maxchunks = 1;
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
    tiles += (int64_t)g.Hkv * nrb * ((t.len + kTrKeys - 1) / kTrKeys);
    maxchunks = std::max(maxchunks, t.pad / 64);
    g.pv_first[i] = pv;
    pv += g.Hkv * nrb * nd;
  }
  g.rows = rows;
  g.pv_items = pv;
  // key tiles of one score item: enough items for two waves, no more than needed
  g.qk_tiles = (int)std::max<int64_t>(1, std::min<int64_t>(16, tiles / (2 * kSms)));
  // CTAs of one value item: while they fit one wave and have two chunks of
  // their own, and at most kTrSplitKeys keys each
  g.splits = 1;
  while (g.splits < 16 && ((int64_t)pv * g.splits * 2 <= kSms && maxchunks >= g.splits * 4)) g.splits *= 2;
  while (g.splits < 16 && (maxchunks + g.splits - 1) / g.splits * 64 > kTrSplitKeys) g.splits *= 2;
  int64_t off = soff * 4;
  int qk = 0;
  for (int i = 0; i < g.nseq; ++i) {
    TreeSeq& t = g.seq[i];
    const int nrb = (t.n * G + g.nr - 1) / g.nr, chunks = t.pad / 64;
    off = (off + 1023) & ~(int64_t)1023;
    t.woff = off;
    off += (int64_t)g.Hkv * nrb * chunks * (3 * g.nr * 64);
    g.qk_first[i] = qk;
    t.qk_per = ((t.len + kTrKeys - 1) / kTrKeys + g.qk_tiles - 1) / g.qk_tiles;
    qk += g.Hkv * nrb * t.qk_per;
  }
  g.qk_items = qk;
  return (size_t)((off + 255) & ~(int64_t)255);
}

template <int NR>
static void tree_launch(const TreeGroup& g, bool vec, cudaStream_t s) {
  const int ns = (g.d + 63) / 64;
  if (vec) ta_launch(tree_qk<NR, true>, dim3(g.qk_items), dim3(kQkThreads), qk_smem<NR>(ns), 1, s, g);
  else ta_launch(tree_qk<NR, false>, dim3(g.qk_items), dim3(kQkThreads), qk_smem<NR>(ns), 1, s, g);
  // CTAs per row: the register form's keys at most, and enough CTAs to fill
  // the GPU while they have a step of their own
  int pad = 0;
  for (int i = 0; i < g.nseq; ++i) pad = std::max(pad, g.seq[i].pad);
  auto span = [&](int CL) { return (pad / 64 + CL - 1) / CL * 64; };
  int CL = 1;
  while (CL < 8 && (span(CL) > kSmRegKeys || ((int64_t)g.rows * CL < 148 && span(CL) > kSmThreads * kSmVec))) CL *= 2;
  if (span(CL) <= kSmRegKeys)
    ta_launch(tree_softmax<NR, true>, dim3(CL * g.rows), dim3(kSmThreads), 0, CL, s, g);
  else
    ta_launch(tree_softmax<NR, false>, dim3(CL * g.rows), dim3(kSmThreads), 0, CL, s, g);
  ta_launch(tree_pv<NR>, dim3(g.pv_items * g.splits), dim3(kPvThreads), pv_smem<NR>(), g.splits, s, g);
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
