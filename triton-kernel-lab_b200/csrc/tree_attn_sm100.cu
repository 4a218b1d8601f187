// Attention of a tree of drafted tokens over a key/value cache, on tcgen05.
//
// Query of node t of sequence b and query head h attends the first
// kv_lens[b] cache rows of KV head h / G and, of the tree's own keys, those
// of its ancestors and itself (parents[t] < t; a node whose parent is not
// one has only itself):
//   o = sum_n p_n v_n,  p = softmax(scale * q . k_n) over those keys,
// with the base-2 log-sum-exp (scale included) as the optional statistic.
// Nodes past a sequence's tree_sizes[b] give o = 0 and lse = -inf.
//
// The G T query rows of one KV head are contiguous, so they are the M rows of
// S = Q K^T and O += P V: each key and value is read once for all of them
// (about G T flop per byte: the cache's bytes bound it up to some 250 rows,
// the tensor cores beyond).  The formulation is the attention forward's
// (attn_fwd_sm100.cu): 128-key tiles by TMA, S and O in tensor memory, one
// thread per row for the base-2 online softmax, P written back over S as
// packed 16-bit pairs.  Keys of an item are its cache tiles, the last one cut
// at kv_lens[b], then the tree's tiles under a bit per (row, node).
//
// With 64 rows or fewer the M rows are filled with kRep = 2 or 4 copies of
// them: copy i's warps take the i-th part of every tile's keys, with a
// running maximum, sum and O of their own (the other keys' P is zero there),
// and the copies are joined through shared memory at the end of a segment.  A
// row's softmax step then takes half or a quarter of the time, which bounds
// short rows: one warp's 128 columns a row took about 3000 cycles a tile.
// 24 sequences of 0 to 4096 keys, 16 heads of 64, 5 nodes: 43 us with four
// copies, 48 with two, 66 with one; 32 sequences of 6144 keys on average, 8
// heads of 128, 32 rows: 134, 133 and 145 us.
//
// Work is cut where the lengths are known, on the device: an item is a (batch,
// KV head), its work its key tiles, and the items' tiles in one row are
// divided into equal runs, one per CTA (of each group of 128 kT rows), so a
// batch of any lengths keeps every SM busy to the end.  A run may begin and
// end inside an item: those (at most two) parts go to a workspace as fp32 O,
// m and l, and tree_attn_combine_kernel joins each row's parts in run order
// (bitwise reproducible, no atomics).
//
// Few items with few tiles are bound by latency, not by bytes: there each item
// gets a CTA to itself (one launch, no scan, no workspace; TreePlan::whole,
// tree_grid).  Rows are not copied then: joining the copies takes longer than
// they save on a few tiles.  (Clusters of CTAs that share an item and join it
// over distributed shared memory were no quicker than the second launch: 12.0
// against 12.3 us a call for 8 items of 9 tiles, 24.7 against 22.1 at 256 rows.)
//
// Cache rows past kv_lens, tree rows past tree_sizes and, for a row, nodes that
// it does not attend may hold anything: the scores of masked keys are replaced
// before they are used, and in shared memory a V tile's rows past the last valid
// key are cleared, and in tree tiles what is not finite (0 times it would be NaN
// in the product); the rows that attend the latter get it added at the end.
// An infinite value in a cache row, which every row attends, makes its column
// infinite, or NaN where a weight is 0: one that underflowed, or a copy's for
// the keys of the others.
//
// Measured, per call (cache bytes; useful flops), 32 sequences of 4096 to 8192
// keys, 8 KV heads of 128, bf16:
//   32 rows    134 us   6.0 TB/s, 94 % of a copy
//   256 rows   218 us   3.9 TB/s, 950 TFLOP/s on a rested device: two tiles'
//              softmax and their products in turn, the tensor pipe 45 %
//              active; called without a pause, at the power limit (1.45 GHz),
//              255 to 267 us
// and 2 sequences of 100000 to 131000 keys, 4 KV heads of 128, 104 rows, fp16:
//   83 us      5.7 TB/s, 89 % of a copy; 93 to 102 us at the power limit.
// The smallest call (8 items of 1000 keys, 32 rows) takes 9.1 us: two launches
// and a chain of loads, products and a join.  For 256 rows none of these was
// quicker than 218 to 223 us at the time: P announced in two parts, so that P V
// starts under the second part's exponentials (221 us); S and P in halves (232);
// S read twice, in loops that need fewer registers (227); two softmax
// warpgroups a tile (315).
//
// What numbers that are not finite cost, in such times: the search of the tree
// tiles' V, the maximum that carries NaN and the additions at the end 1.5 us of
// 62 for 8 sequences of 256 rows (2.5 %), 0.2 of 9 for the smallest call, nothing
// that can be told for the long cache.
#include <algorithm>

#include "attn_launch.h"
#include "pdl_launch.h"
#include "sm100_primitives.cuh"
#include "tree_attn_plan.h"

namespace tk {
namespace {

// D: kernel width (64 or 128); kT: 128-row query tiles per CTA; kRep: copies of
// the rows in the one tile (1, 2 or 4).
template <int D, int kT, int kRep>
struct TreeCfg {
  static_assert(kRep == 1 || kT == 1, "copies fill one tile");
  // One tile per CTA: a warpgroup of its own for the epilogue and two O
  // buffers, so a segment's end does not hold up the next one's tiles, and a
  // second S buffer, so S(j + 1) runs under the softmax of S(j).  Two tiles
  // cover each other instead (and fill tensor memory at D = 128).
  static constexpr bool kEpi = kT == 1;
  static constexpr int kLook = kEpi ? 2 : 1;
  static constexpr int kThreads = 128 * (1 + kT + (kEpi ? 1 : 0));
  // Stages of K and of V.
  static constexpr int kStages = (D == 64) ? 5 : 3;
  static constexpr int kVStages = (D == 64) ? 4 : (kT == 1 && kRep == 1) ? 3 : 2;
  static constexpr int kQBufs = (D == 64 && kT == 1) ? 2 : 1;
  static constexpr int kRows = kT * kTileRows / kRep;  // query rows per CTA
  // 0: launched with registers to spare, no redistribution.
  static constexpr int kLaunchRegs = (kRep == 1) ? 168 : 0;
  static constexpr int kRegsCtrl = 56;
  static constexpr int kRegsWork = 224;  // of the other warpgroups
  static_assert(kLaunchRegs == 0 || kRegsCtrl + (kThreads / 128 - 1) * kRegsWork <= kThreads / 128 * kLaunchRegs,
                "register split exceeds the launch");
  static constexpr int kTileBytes = kTileRows * D * 2;
  static constexpr int kKOff = kQBufs * kT * kTileBytes;
  static constexpr int kVOff = kKOff + kStages * kTileBytes;
  static constexpr int kJoinOff = kVOff + kVStages * kTileBytes;
  static constexpr int kJoinCols = 64;  // columns of O joined at a time (every copy, fp32)
  static constexpr int kBarOff = kJoinOff + (kRep > 1 ? kTileRows * kJoinCols * 4 : 0);
  // q_full[Q], q_empty[Q], k_full[S], k_empty[S], v_full[S], v_ok[S], v_empty[S], s_full[2], p_ready[2], o_final[2],
  // o_empty[2], l_ready[2], pv_done, drained
  static constexpr int kNumBars = 2 * kQBufs + 2 * kStages + 3 * kVStages + 12;
  static constexpr int kCtlOff = kBarOff + kNumBars * 8;
  static constexpr int kMlOff = (kCtlOff + 16 + 32 + 64 + 7) / 8 * 8;  // after control, first segment, scan
  // m and l of a segment's rows, two buffers.
  static constexpr int kSmemBytes = kMlOff + (kEpi ? 2 * kTileRows * 8 : 0);
  static constexpr uint32_t kTmemCols = 512;
  // O of query tile x, or O buffer x, at column x D; the S buffers from here.
  static constexpr uint32_t kColS0 = (kEpi ? 2 : kT) * D;
};

constexpr float kTreeRescale = 8.0f;  // as the forward's: P stays below 2^8 (2^15 in float16), O is rescaled rarely
// float16 has nothing below 2^-24: there exponents are taken from 7 below a
// row's maximum (m is that everywhere below), so that a weight is lost from P V
// only under 2^-32 of the largest.  (Taken from the maximum, it was lost under
// 2^-25: thousands of such keys were missing in O, though not in the sum, where
// the largest's own value was small.)  bfloat16 has float32's exponents.
template <bool kBf16>
constexpr float kTreeRaise = kBf16 ? 0.0f : 7.0f;

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, CtaControl* ctl, uint64_t timeout_ns,
                                          int* status, int site) {
  const bool ok = mbar_wait(bar, parity, ctl, timeout_ns, status, site);
  return __all_sync(0xffffffffu, ok);
}

// Sizes every role needs.
struct TreeShape {
  const int* kv_lens;
  const int* tree_sizes;
  const int* parents;
  long long parent_stride;
  const uint16_t* v_tree;  // the tree's values, at element strides
  long long v_batch, v_head, v_row;
  int B, Hkv, T, L, R;  // R = G T query rows per KV head
  int d_real;
};

__device__ __forceinline__ int cache_len(const TreeShape& s, int b) { return min(max(s.kv_lens[b], 0), s.L); }
__device__ __forceinline__ int tree_size(const TreeShape& s, int b) {
  return s.tree_sizes != nullptr ? min(max(s.tree_sizes[b], 0), s.T) : s.T;
}
__device__ __forceinline__ int tiles_of(int n) { return (n + kTileRows - 1) / kTileRows; }

// A part of an item: key tiles [j0, j1) of (b, h), which has n_cache cache
// tiles and n_all tiles.
struct TreeSeg {
  int b, h, j0, j1, n_cache, n_all, len;
};

// What an item costs beyond its tiles (its query load, first scores and
// epilogue), in tiles: runs are equal in tiles plus this, so that a CTA with
// many short items gets fewer tiles.  Sequences of 0 to 4096 keys, 64 wide, 24
// of them: with 0, the slowest CTA took 1.29 times the median's time.
constexpr int kItemCost = 2;
__device__ __forceinline__ int item_cost(const TreeShape& s, int b) {
  return tiles_of(cache_len(s, b)) + tiles_of(s.T) + kItemCost;
}

// Walks a CTA's run, one segment at a time.  u: place in the item's cost, its
// first kItemCost units holding no tile.
struct TreeWalk {
  int b, h, u, left;
  __device__ __forceinline__ bool next(const TreeShape& s, TreeSeg& seg) {
    while (left > 0) {
      seg.b = b;
      seg.h = h;
      seg.len = cache_len(s, b);
      seg.n_cache = tiles_of(seg.len);
      seg.n_all = seg.n_cache + tiles_of(s.T);
      const int end = min(seg.n_all + kItemCost, u + left);
      seg.j0 = max(u - kItemCost, 0);
      seg.j1 = max(end - kItemCost, 0);
      left -= end - u;
      u = 0;
      if (++h == s.Hkv) {
        h = 0;
        ++b;
      }
      if (seg.j1 > seg.j0) return true;
    }
    return false;
  }
};

// The start of the workspace, for the joining kernel: an entry per item or, if
// there are fewer runs, per run, written by the CTA that begins the item.
struct TreePlan {
  TreeCut* cut;
  int by_item;
  int whole;  // a CTA per item, grid (groups, items): nothing else of the plan or the workspace is used
};

// The maximum; with kNan NaN if one of them is.
template <bool kNan>
__device__ __forceinline__ float tile_max(float a, float b, float c) {
  return kNan ? fmax3_nan(a, b, c) : fmax3(a, b, c);
}

// One 128-key tile of one row: as the forward's softmax step, with `mask`
// (kMasked) a bit per key.  With copies (kRep > 1) only copy `copy`'s 128 /
// kRep keys; P of the others is zero.  The polynomial exponentials
// (kEmuPairs) take any NaN or -inf for 2^-126, so where they run the tile's
// maximum carries NaN, a row whose maximum is NaN or +inf (the formula's inf -
// inf) gets a sum of NaN, and one with only -inf so far a sum of 0.
template <bool kBf16, bool kMasked, int kEmuPairs, int kRep>
__device__ __forceinline__ void softmax_tile(uint32_t s_addr, int copy, const uint32_t (&mask)[4 / kRep], float scale_log2,
                                             float& m_run, float& l_run, float& alpha, bool& need) {
  constexpr int kBlocks = 4 / kRep;  // 32-key blocks
  constexpr bool kEmulates = !kMasked && kEmuPairs > 0;
  uint32_t s[kBlocks][32];
  const uint32_t own = s_addr + copy * (32 * kBlocks);
#pragma unroll
  for (int b = 0; b < (kBlocks + 1) / 2; ++b) tmem_ld32(own + 32 * b, s[b]);
  tmem_wait_ld();
#pragma unroll
  for (int b = 0; b < (kBlocks + 1) / 2; ++b) reg_fence(s[b]);
#pragma unroll
  for (int b = (kBlocks + 1) / 2; b < kBlocks; ++b) tmem_ld32(own + 32 * b, s[b]);
  float mx[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mx[i] = -INFINITY;
  bool live[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    if (kBlocks > 1 && b == kBlocks / 2) {
      tmem_wait_ld();
#pragma unroll
      for (int i = kBlocks / 2; i < kBlocks; ++i) reg_fence(s[i]);
    }
    // Blocks without a key of any row of the warp: cut tiles and small trees
    // leave much of a tile empty (80 to 73 us for 336 items of two tiles).
    live[b] = !kMasked || __any_sync(0xffffffffu, mask[b] != 0u);
    if (!live[b]) continue;
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      if constexpr (kMasked) {
        if (!((mask[b] >> c) & 1u)) s[b][c] = __float_as_uint(-INFINITY);
        if (!((mask[b] >> (c + 1)) & 1u)) s[b][c + 1] = __float_as_uint(-INFINITY);
      }
      mx[(c >> 1) & 7] = tile_max<kEmulates>(mx[(c >> 1) & 7], __uint_as_float(s[b][c]), __uint_as_float(s[b][c + 1]));
    }
  }
  const float mxa = tile_max<kEmulates>(mx[0], mx[1], mx[2]), mxb = tile_max<kEmulates>(mx[3], mx[4], mx[5]);
  const float m_tile = tile_max<kEmulates>(mxa, mxb, tile_max<kEmulates>(mx[6], mx[7], mx[7]));
  const float m_new = fmaxf(m_run, kBf16 ? m_tile * scale_log2 : fmaf(m_tile, scale_log2, -kTreeRaise<kBf16>));
  need = m_new > m_run + kTreeRescale;
  const float m_use = need ? m_new : m_run;
  alpha = (m_run == -INFINITY) ? 0.0f : ex2(m_run - m_use);
  const float ms = (m_use == -INFINITY) ? 0.0f : m_use;
  const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
  const uint64_t negm2 = f2_pack(-ms, -ms);
  uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
  if constexpr (kRep > 1) {
    // S is in registers: zero P everywhere else.
    const uint32_t zero[16] = {};
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (b / kBlocks != copy) tmem_st16(s_addr + b * 16, zero);
  }
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) {
    uint32_t pk[16] = {};
    if (live[b]) {
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        float x0, x1, p0, p1;
        f2_unpack(ffma2(f2_pack(__uint_as_float(s[b][c]), __uint_as_float(s[b][c + 1])), scale2, negm2), x0, x1);
        // Masked tiles keep every exponential on the MUFU so that masked
        // entries are exactly zero.
        if (kEmulates && ((c >> 1) & 7) >= 8 - kEmuPairs) {
          exp2_fma_pair(x0, x1, p0, p1);
        } else {
          p0 = ex2(x0);
          p1 = ex2(x1);
        }
        sum2[(c >> 1) & 1] = fadd2(sum2[(c >> 1) & 1], f2_pack(p0, p1));
        pk[c >> 1] = pack2<kBf16>(p0, p1);
      }
    }
    tmem_st16(s_addr + (copy * kBlocks + b) * 16, pk);
  }
  float sa0, sa1, sb0, sb1;
  f2_unpack(sum2[0], sa0, sa1);
  f2_unpack(sum2[1], sb0, sb1);
  l_run = l_run * alpha + ((sa0 + sa1) + (sb0 + sb1));
  if constexpr (kEmulates) {
    if (!(m_tile < INFINITY)) l_run = __uint_as_float(0x7fffffffu);
    if (m_use == -INFINITY && l_run == l_run) l_run = 0.0f;
  }
  m_run = m_use;
}

// The first n bits of W words (none below 0, all from 32 W on).
template <int W>
__device__ __forceinline__ void first_bits(int n, uint32_t (&mask)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const int k = n - 32 * i;
    mask[i] = k >= 32 ? 0xffffffffu : k > 0 ? (1u << k) - 1u : 0u;
  }
}

// Bit n of the W words: the row's node attends tree node lo + n.
template <int W>
__device__ __forceinline__ void tree_mask(const TreeShape& s, int b, int node, int size, int lo, uint32_t (&mask)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) mask[i] = 0;
  if (node >= size) return;
  if (s.parents == nullptr) {
    first_bits(node + 1 - lo, mask);
    return;
  }
  const int* up = s.parents + b * s.parent_stride;
  while (node >= lo) {  // ends: every step goes to a smaller node
    const int n = node - lo;
#pragma unroll
    for (int i = 0; i < W; ++i)
      if ((n >> 5) == i) mask[i] |= 1u << (n & 31);
    const int parent = up[node];
    node = parent < node ? parent : -1;
  }
}

template <bool kBf16>
__device__ __forceinline__ float half_value(uint16_t h) {
  if constexpr (kBf16) {
    return __uint_as_float(static_cast<uint32_t>(h) << 16);
  } else {
    return __half2float(__ushort_as_half(h));
  }
}

// The halves of a word that hold no finite number, as bits 15 and 31: their
// exponents are all ones, and one more carries into the sign's place.
template <bool kBf16>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  constexpr uint32_t kExp = kBf16 ? 0x7f807f80u : 0x7c007c00u, kOne = kBf16 ? 0x00800080u : 0x04000400u;
  return ((w & kExp) + kOne) & 0x80008000u;
}

// The larger magnitudes of two words' halves, NaN before all.
template <bool kBf16>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t w) {
  if constexpr (kBf16) {
    const __nv_bfloat162 m = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), __habs2(*reinterpret_cast<__nv_bfloat162*>(&w)));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __half2 m = __hmax2_nan(*reinterpret_cast<__half2*>(&a), __habs2(*reinterpret_cast<__half2*>(&w)));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}

// Clears what is not finite in the first `rows` rows of a V tile (one warp) and
// returns whether there was anything.  The search is a packed maximum a word:
// one warp has the whole tile to look at while others make its P.
template <int D, bool kBf16>
__device__ __forceinline__ bool clear_not_finite(uint8_t* tile, int rows, int lane) {
  constexpr int kFlight = 2;
  uint32_t top[kFlight] = {};
#pragma unroll 1
  for (int off = lane * 16; off < rows * kSwizzleBytes; off += kFlight * 32 * 16) {
    uint4 v[D / 64][kFlight];
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk)
#pragma unroll
      for (int i = 0; i < kFlight; ++i)  // (past the rows: loaded still, not looked at)
        v[blk][i] = *reinterpret_cast<const uint4*>(tile + blk * kBlockBytes + min(off + i * 32 * 16, kBlockBytes - 16));
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk)
#pragma unroll
      for (int i = 0; i < kFlight; ++i)
        if (off + i * 32 * 16 < rows * kSwizzleBytes)
          top[i] = larger<kBf16>(larger<kBf16>(larger<kBf16>(larger<kBf16>(top[i], v[blk][i].x), v[blk][i].y), v[blk][i].z),
                                 v[blk][i].w);
  }
  uint32_t found = 0;
#pragma unroll
  for (int i = 0; i < kFlight; ++i) found |= not_finite<kBf16>(top[i]);
  if (!__any_sync(0xffffffffu, found != 0)) return false;
#pragma unroll 1
  for (int blk = 0; blk < D / 64; ++blk)
#pragma unroll 1
    for (int off = lane * 4; off < rows * kSwizzleBytes; off += 32 * 4) {
      uint32_t* w = reinterpret_cast<uint32_t*>(tile + blk * kBlockBytes + off);
      *w &= ~((not_finite<kBf16>(*w) >> 15) * 0xffffu);
    }
  return true;
}

// Place of 8 columns of a part's row: blocks of four rows, within one the rows'
// 32 bytes of the same columns side by side.  Threads with a row each then
// fill whole lines, and a warp of the joining kernel reads four rows as one
// piece.  (With rows in sequence a store touched a line a lane: 4300 cycles
// for 256 rows of 128.)
template <int D>
__device__ __forceinline__ long long part_at(long long prow, int col) {
  return (prow >> 2) * (4 * D) + (col >> 3) * 32 + (prow & 3) * 8;
}

// The end of a segment for one row held by one thread: O from tensor memory
// to the output (whole items) or, unnormalised with m and l, to a part's row.
template <int D, bool kBf16>
__device__ __forceinline__ void finish_row(uint32_t o_addr, bool whole, bool live, bool row_ok, float m, float l,
                                           long long row_g, long long prow, int d_real, uint16_t* out, float* lse,
                                           float* part_ml, float* part_o) {
  if (whole) {
    const bool wide_store = (d_real % 16) == 0 && (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
    const float inv = (live && l != 0.0f) ? 1.0f / l : 0.0f;  // of a NaN: NaN
    uint16_t* orow = out + row_g * d_real;
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
      uint32_t o[32];
      tmem_ld32(o_addr + cb * 32, o);
      tmem_wait_ld();
      reg_fence(o);
      uint32_t w[16];
#pragma unroll
      for (int e = 0; e < 16; ++e)
        w[e] = live ? pack2<kBf16>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv) : 0u;
      if (row_ok) {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          const int col = cb * 32 + hh * 16;
          if (wide_store && col < d_real) {
            st_global_v8(orow + col, &w[hh * 8]);
          } else if (!wide_store) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if (col + q * 8 < d_real)
                *reinterpret_cast<uint4*>(orow + col + q * 8) = make_uint4(
                    w[hh * 8 + q * 4], w[hh * 8 + q * 4 + 1], w[hh * 8 + q * 4 + 2], w[hh * 8 + q * 4 + 3]);
          }
        }
      }
    }
    if (lse != nullptr && row_ok) lse[row_g] = live ? m + lg2(l) : -INFINITY;
  } else {
#pragma unroll
    for (int cb = 0; cb < D / 32; ++cb) {
      uint32_t o[32];
      tmem_ld32(o_addr + cb * 32, o);
      tmem_wait_ld();
      reg_fence(o);
      if (!live) {
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = 0u;
      }
      if (row_ok) {
#pragma unroll
        for (int q = 0; q < 4; ++q) st_global_v8(part_o + part_at<D>(prow, cb * 32 + q * 8), &o[q * 8]);
      }
    }
    if (row_ok) *reinterpret_cast<float2*>(part_ml + prow * 2) = live ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
  }
}

// Adds to columns [c0, c1) of a row that this thread has stored (as output, or
// as a part's row) the values that are not finite of the nodes in the segment's
// tree tiles that the row's node attends.  What was stored lacks them: in the
// product they would make NaN of every row, 0 times infinity, and not of those
// that attend them only.
template <int D, bool kBf16>
__device__ __forceinline__ void add_not_finite(const TreeShape& s, const TreeSeg& seg, int node, int c0, int c1, bool whole,
                                               uint16_t* out_row, float* part_o, long long prow) {
  const int lo = max(seg.j0 - seg.n_cache, 0) * kTileRows, hi = (seg.j1 - seg.n_cache) * kTileRows;
  const uint16_t* v = s.v_tree + seg.b * s.v_batch + seg.h * s.v_head;
  if (hi <= 0) return;
  asm volatile("" ::: "memory");  // after the stores, which were of other types
#pragma unroll 1
  for (int n = node; n >= lo;) {
    if (n < hi) {
#pragma unroll 1
      for (int c = c0; c < min(c1, s.d_real); ++c) {
        const uint16_t x = v[n * s.v_row + c];
        if (not_finite<kBf16>(x) == 0) continue;
        if (whole) {
          uint16_t* o = out_row + c;
          *o = static_cast<uint16_t>(pack2<kBf16>(half_value<kBf16>(*o) + half_value<kBf16>(x), 0.0f));
        } else {
          part_o[part_at<D>(prow, c & ~7) + (c & 7)] += half_value<kBf16>(x);
        }
      }
    }
    const int parent = s.parents != nullptr ? s.parents[seg.b * s.parent_stride + n] : n - 1;
    n = parent < n ? parent : -1;
  }
}

// Out of line for the epilogue warpgroup: a call that is hardly ever made, and
// whose code would delay the smallest ones (8.9 us, 9.2 with it in line).  With
// two tiles in line: there a call costs the softmax warps registers (53 us, 54).
template <int D, bool kBf16>
__device__ __noinline__ void call_add_not_finite(const TreeShape& s, const TreeSeg& seg, int node, int c0, int c1, bool whole,
                                                 uint16_t* out_row, float* part_o, long long prow) {
  add_not_finite<D, kBf16>(s, seg, node, c0, c1, whole, out_row, part_o, prow);
}

// The end of a segment whose rows are held as kRep copies: thread r holds row
// r % (128 / kRep) of copy r / (128 / kRep).  64 columns at a time, each row
// weighted by 2^(m - M) goes to shared memory (16-byte chunks XORed with the
// row), then kRep threads a row add the copies and store.  All 128 threads
// call it; `ok` only skips the work.
template <int D, int kRep, bool kBf16>
__device__ __forceinline__ void finish_copies(bool ok, uint32_t o_addr, int r, bool whole, const float2* ml, float4* join,
                                              const TreeShape& shape, const TreeSeg& seg, bool patch, long long item_row,
                                              long long slot_row, uint16_t* out, float* lse, float* part_ml,
                                              float* part_o) {
  const int R = shape.R, d_real = shape.d_real;
  constexpr int kCopyRows = kTileRows / kRep;
  constexpr int kCols = 64 / kRep;
  const int mrow = r % kCopyRows;  // the row it writes
  const int jrow = r / kRep, jpart = r % kRep;  // the row and columns it finishes
  float top = -INFINITY, jtop = -INFINITY, jl = 0.0f;
#pragma unroll
  for (int i = 0; i < kRep; ++i) {
    top = fmaxf(top, ml[i * kCopyRows + mrow].x);
    jtop = fmaxf(jtop, ml[i * kCopyRows + jrow].x);
  }
  // Weight 0: a copy without keys, or rows that no warp computed.
  const float w = ml[r].x == -INFINITY ? 0.0f : ex2(ml[r].x - top);
#pragma unroll
  for (int i = 0; i < kRep; ++i) {
    const float2 e = ml[i * kCopyRows + jrow];
    if (e.x != -INFINITY) jl += ex2(e.x - jtop) * e.y;
  }
  // (A sum of NaN makes NaN of its row, also where the copy that it is from
  // weighs nothing beside the others and its O is left out.)
  const float scale = whole ? (jl != 0.0f ? 1.0f / jl : 0.0f) : 1.0f;
  const bool jrow_ok = ok && jrow < R;
#pragma unroll
  for (int pass = 0; pass < D / 64; ++pass) {
    if (pass > 0) named_barrier_sync(1, 128);
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      uint32_t o[32];
      if (ok) {
        tmem_ld32(o_addr + pass * 64 + cb * 32, o);
        tmem_wait_ld();
        reg_fence(o);
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
        join[r * 16 + ((cb * 8 + q) ^ (r & 7))] =
            w != 0.0f ? make_float4(w * __uint_as_float(o[4 * q]), w * __uint_as_float(o[4 * q + 1]),
                                   w * __uint_as_float(o[4 * q + 2]), w * __uint_as_float(o[4 * q + 3]))
                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    named_barrier_sync(1, 128);
    if (!jrow_ok) continue;
#pragma unroll
    for (int c = 0; c < kCols; c += 8) {
      float4 f[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        f[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < kRep; ++i) {
          const int jr = i * kCopyRows + jrow;
          const float4 g = join[jr * 16 + (((jpart * kCols + c) / 4 + q) ^ (jr & 7))];
          f[q].x += g.x, f[q].y += g.y, f[q].z += g.z, f[q].w += g.w;
        }
      }
      const int col = pass * 64 + jpart * kCols + c;
      if (whole) {
        if (col < d_real)
          *reinterpret_cast<uint4*>(out + (item_row + jrow) * d_real + col) =
              make_uint4(pack2<kBf16>(f[0].x * scale, f[0].y * scale), pack2<kBf16>(f[0].z * scale, f[0].w * scale),
                         pack2<kBf16>(f[1].x * scale, f[1].y * scale), pack2<kBf16>(f[1].z * scale, f[1].w * scale));
      } else {
        float4* dst = reinterpret_cast<float4*>(part_o + part_at<D>(slot_row + jrow, col));
        dst[0] = f[0];
        dst[1] = f[1];
      }
    }
  }
  if (patch && jrow_ok && jl != 0.0f)
    for (int c = jpart * kCols; c < D; c += 64)
      call_add_not_finite<D, kBf16>(shape, seg, jrow % shape.T, c, c + kCols, whole, out + (item_row + jrow) * d_real,
                                    part_o, slot_row + jrow);
  if (jrow_ok && jpart == 0) {
    if (!whole)
      *reinterpret_cast<float2*>(part_ml + (slot_row + jrow) * 2) = make_float2(jtop, jl);
    else if (lse != nullptr)
      lse[item_row + jrow] = jl == 0.0f ? -INFINITY : jtop + lg2(jl);
  }
  __syncwarp();
  named_barrier_sync(1, 128);  // before the next segment's ml and columns
}

template <int D, int kT, int kRep, bool kBf16>
__global__ void __launch_bounds__(TreeCfg<D, kT, kRep>::kThreads, 1)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kt,
                     const __grid_constant__ CUtensorMap tm_vt, const __grid_constant__ TreeShape shape,
                     uint16_t* __restrict__ out, float* __restrict__ lse, TreePlan plan, float* __restrict__ part_ml,
                     float* __restrict__ part_o, float scale_log2, unsigned long long timeout_ns, int* status) {
  using C = TreeCfg<D, kT, kRep>;
  constexpr int kLook = C::kLook;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, kOk, kErrMisaligned);
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int wg = warp >> 2;
  const bool whole_item = kRep == 1 && plan.whole != 0;
  const int group = blockIdx.x;  // rows [group kRows, ...) of every item

  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::kKOff;
  uint8_t* sV = smem + C::kVOff;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* q_empty = q_full + C::kQBufs;
  uint64_t* k_full = q_empty + C::kQBufs;
  uint64_t* k_empty = k_full + C::kStages;
  uint64_t* v_full = k_empty + C::kStages;
  uint64_t* v_ok = v_full + C::kVStages;  // full, and cleared past the last valid key
  uint64_t* v_empty = v_ok + C::kVStages;
  uint64_t* s_full = v_empty + C::kVStages;  // [2]: query tile, or S buffer of the one tile
  uint64_t* p_ready = s_full + 2;           // [2]
  uint64_t* o_final = p_ready + 2;          // [2]: query tile, or O buffer
  uint64_t* o_empty = o_final + 2;          // [2]: O buffer read by the epilogue
  uint64_t* l_ready = o_empty + 2;          // [2]: m and l of O buffer's segment written
  uint64_t* pv_done = l_ready + 2;          // with two S buffers: P V of every tile
  uint64_t* drained = pv_done + 1;          // after a wait that gave up: every product
  CtaControl* ctl = reinterpret_cast<CtaControl*>(smem + C::kCtlOff);
  // Values that are not finite were taken out of a tree tile of this CTA.  Warp 3
  // sets it before v_ok of the tile; it is read after o_final of its segment.
  volatile int* patched = reinterpret_cast<int*>(smem + C::kCtlOff + sizeof(CtaControl));
  int* first = reinterpret_cast<int*>(smem + C::kCtlOff + 16);  // this CTA's run: b, h, u, length; the runs' length
  int* loads = first + 5;  // [3]: tiles of K (warp 0) and V (warp 2) and segments' Q (warp 3) that were asked for
  int* scan = first + 8;                                         // [warps]

  // Loads of the query rows of a segment (kT tiles of 128 rows, or kRep copies
  // of 128 / kRep) and of one of its key tiles.
  auto load_q = [&](const TreeSeg& sg, int qb) {
    mbar_arrive_expect_tx(&q_full[qb], kT * C::kTileBytes);
#pragma unroll
    for (int x = 0; x < kT * kRep; ++x)
#pragma unroll
      for (int blk = 0; blk < D / 64; ++blk)
        tma_load_3d(sQ + (qb * kT + x / kRep) * C::kTileBytes + blk * kBlockBytes +
                        (x % kRep) * (kTileRows / kRep) * kSwizzleBytes,
                    &tm_q, &q_full[qb], blk * 64, group * C::kRows + (kRep == 1 ? x * kTileRows : 0),
                    sg.b * shape.Hkv + sg.h);
  };
  auto load_tile = [&](const TreeSeg& sg, int j, bool is_k, int st) {
    uint64_t* full = is_k ? &k_full[st] : &v_full[st];
    mbar_arrive_expect_tx(full, C::kTileBytes);
    const bool on_cache = j < sg.n_cache;
    const CUtensorMap* map = on_cache ? (is_k ? &tm_k : &tm_v) : (is_k ? &tm_kt : &tm_vt);
    const int row = (on_cache ? j : j - sg.n_cache) * kTileRows;
#pragma unroll
    for (int blk = 0; blk < D / 64; ++blk)
      tma_load_4d((is_k ? sK : sV) + st * C::kTileBytes + blk * kBlockBytes, map, full, blk * 64, row, sg.h, sg.b);
  };

  // This CTA's work, by warp 0 alone unless the batch is large, so that it can
  // also start the first loads before the CTA has met.
  const bool by_warp = whole_item || shape.B <= 32;
  uint32_t early = 0;  // K tiles started (warp 0, lane 0)
  if (warp == 0) {
    // The barriers and descriptors, a lane each; what other kernels may have written from here on.
    if (lane == 0) tma_prefetch_map(&tm_q);
    if (lane == 1) tma_prefetch_map(&tm_k);
    if (lane == 2) tma_prefetch_map(&tm_kt);
    if (lane == 3) tma_prefetch_map(&tm_v);
    if (lane == 4) tma_prefetch_map(&tm_vt);
    for (int i = lane; i < C::kNumBars; i += 32) {
      uint64_t* bar = q_full + i;
      const bool by_warps = (bar >= p_ready && bar < p_ready + 2) || (bar >= o_empty && bar < o_empty + 4);
      mbar_init(bar, by_warps ? 4 : bar >= o_final && bar < o_final + 2 ? 2 : 1);
    }
    if (lane == 0) {
      ctl->abort = 0;
      *patched = 0;
    }
    fence_mbarrier_init();
    pdl_wait_prerequisites();
    const int cost = whole_item ? item_cost(shape, blockIdx.y / shape.Hkv)
                                : by_warp && lane < shape.B ? item_cost(shape, lane) : 0;
    __syncwarp();
    if (whole_item) {
      if (lane == 0) {
        first[0] = blockIdx.y / shape.Hkv;
        first[1] = blockIdx.y % shape.Hkv;
        first[2] = 0;
        first[3] = cost;
      }
    } else if (by_warp) {
      // A run: a scan of the batch's costs, a lane each.
      const int n = cost;
      int upto = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += o;
      }
      const int total = __shfl_sync(0xffffffffu, upto, 31) * shape.Hkv;
      const int run = (total + gridDim.y - 1) / gridDim.y;
      const int start = blockIdx.y * run, from = (upto - n) * shape.Hkv;
      if (n > 0 && start >= from && start < from + n * shape.Hkv) {
        first[0] = lane;
        first[1] = (start - from) / n;
        first[2] = (start - from) % n;
      }
      if (lane == 0) {
        first[3] = max(min(run, total - start), 0);
        first[4] = run;
      }
    }
    __syncwarp();
    if (by_warp && lane == 0) {
      TreeWalk ahead{first[0], first[1], first[2], first[3]};
      TreeSeg sg;
      if (ahead.next(shape, sg)) {
        load_q(sg, 0);
        for (int j = sg.j0; j < sg.j1 && early < C::kStages; ++j, ++early) load_tile(sg, j, true, early);
      }
    }
  }
  if (warp == 1) tmem_alloc(&ctl->tmem_base, C::kTmemCols);
  pdl_wait_prerequisites();
  if (!by_warp) {
    // A run: the scan by all threads, each over consecutive sequences.
    const int per = (shape.B + C::kThreads - 1) / C::kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, shape.B), b1 = min(b0 + per, shape.B);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += item_cost(shape, b);
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += o;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < C::kThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    before += upto - mine;
    total *= shape.Hkv;
    const int run = (total + gridDim.y - 1) / gridDim.y;
    const int start = blockIdx.y * run;
    if (threadIdx.x == 0) {
      first[3] = max(min(run, total - start), 0);
      first[4] = run;
    }
    for (int b = b0; b < b1; ++b) {
      const int n = item_cost(shape, b);
      const int from = before * shape.Hkv;
      if (start >= from && start < from + n * shape.Hkv) {
        first[0] = b;
        first[1] = (start - from) / n;
        first[2] = (start - from) % n;
      }
      before += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // (The grid is resident as a whole, so what starts early only waits.)
  pdl_launch_dependents();
  const uint32_t tmem = ctl->tmem_base;
  TreeWalk walk{first[0], first[1], first[2], first[3]};
  TreeSeg seg;

  // Every role walks the same segments; barrier phases follow running counts
  // of segments and key tiles, so consecutive segments pipeline.
  if (wg == 0) {
    if constexpr (C::kLaunchRegs != 0) warpgroup_reg_dec<C::kRegsCtrl>();
    if (warp == 0 || warp == 2) {
      // ---------------- TMA producers: warp 0 K, warp 2 V ----------------
      if (lane == 0) {
        const bool is_k = warp == 0;
        uint64_t* empty = is_k ? k_empty : v_empty;
        const uint32_t depth = is_k ? C::kStages : C::kVStages;
        uint32_t g = 0;
        bool ok = true;
        while (ok && walk.next(shape, seg)) {
          for (int j = seg.j0; j < seg.j1; ++j, ++g) {
            if (is_k && g < early) continue;
            const int st = g % depth;
            if (!(ok = mbar_wait(&empty[st], ((g / depth) & 1) ^ 1, ctl, timeout_ns, status, is_k ? 2 : 3))) break;
            load_tile(seg, j, is_k, st);
          }
        }
        loads[warp >> 1] = max(g, is_k ? early : 0u);
      }
    } else if (warp == 3) {
      // ---------------- Q, the tails of V, and the joining kernel's entries ----------------
      TreeCut mine{-1, 0, 0, 0};
      uint32_t g = 0;
      int asked = 0;
      bool ok = true;
      // (Every segment, failed or not: an entry is for the joining kernel to read.)
      for (int it = 0; walk.next(shape, seg); ++it) {
        if (lane == 0 && !whole_item && group == 0 && seg.j0 == 0) {
          const bool cut = seg.j1 < seg.n_all;
          const int item = seg.b * shape.Hkv + seg.h;
          const TreeCut e{cut ? item : -1, static_cast<int>(blockIdx.y), it > 0 ? 1 : 0,
                          1 + (seg.n_all - seg.j1 + first[4] - 1) / first[4]};
          if (plan.by_item)
            plan.cut[item] = e;
          else if (cut)
            mine = e;
        }
        const int qb = it % C::kQBufs;
        if (ok && it >= C::kQBufs) ok = warp_wait(&q_empty[qb], ((it / C::kQBufs) & 1) ^ 1, ctl, timeout_ns, status, 1);
        if (!ok) continue;
        if (!by_warp || it > 0) {
          if (lane == 0) load_q(seg, qb);
        }
        asked = it + 1;
        const int size = tree_size(shape, seg.b);
        for (int j = seg.j0; j < seg.j1; ++j, ++g) {
          const int st = g % C::kVStages;
          if (!(ok = warp_wait(&v_full[st], (g / C::kVStages) & 1, ctl, timeout_ns, status, 15))) break;
          // Rows of V past the last valid key: cleared.
          const int jt = j - seg.n_cache;
          const int valid = jt < 0 ? seg.len - j * kTileRows : size - jt * kTileRows;
          if (valid < kTileRows) {
            const int from = max(valid, 0) * kSwizzleBytes;
#pragma unroll
            for (int blk = 0; blk < D / 64; ++blk)
              for (int off = from + lane * 16; off < kBlockBytes; off += 32 * 16)
                *reinterpret_cast<uint4*>(sV + st * C::kTileBytes + blk * kBlockBytes + off) = make_uint4(0, 0, 0, 0);
          }
          // Not every row attends a tree row: what is not finite is taken out
          // (and added where it belongs at the segment's end).
          const bool odd = jt >= 0 && clear_not_finite<D, kBf16>(sV + st * C::kTileBytes, min(max(valid, 0), kTileRows), lane);
          if (odd && lane == 0) *patched = 1;
          if (odd || valid < kTileRows) fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_ok[st]);
        }
      }
      if (lane == 0 && !whole_item && group == 0 && !plan.by_item) plan.cut[blockIdx.y] = mine;
      if (lane == 0) loads[2] = asked;
    } else if (warp == 1) {
      // ---------------- MMA issuer ----------------
      const bool leader = elect_one();
      const uint32_t idesc_qk = idesc_f16(kBf16 ? 1u : 0u, 128, 128, 0, 0);
      const uint32_t idesc_pv = idesc_f16(kBf16 ? 1u : 0u, 128, D, 0, 1);
      const uint32_t q_lo0 = sdesc_lo_kmajor(smem_u32(sQ));
      const uint32_t k_lo0 = sdesc_lo_kmajor(smem_u32(sK));
      const uint32_t v_lo0 = sdesc_lo_mnmajor(smem_u32(sV), kTileRows);
      constexpr uint32_t kTileLo = C::kTileBytes >> 4;
      // Query tile x (kT = 2), or S buffer x of the one tile.
      auto issue_s = [&](int x, int qb, int st) {
        const uint32_t q_lo = q_lo0 + (kT == 2 ? x : qb) * kTileLo;
        const uint32_t k_lo = k_lo0 + st * kTileLo;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_ss_w(tmem + C::kColS0 + 128u * x, q_lo + kmajor_koff(kTileRows, kk * 16),
                      k_lo + kmajor_koff(kTileRows, kk * 16), idesc_qk, kk > 0 ? 1u : 0u);
          umma_commit(&s_full[x]);
        }
        __syncwarp();
      };
      auto issue_pv = [&](int x, int ob, int st, bool accumulate) {
        const uint32_t v_lo = v_lo0 + st * kTileLo;
        const uint32_t d = tmem + (kT == 2 ? D * x : D * ob);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < kTileRows / 16; ++kk)
            umma_ts_w(d, tmem + C::kColS0 + 128u * x + kk * 8, v_lo + mnmajor_koff(kk * 16), idesc_pv,
                      (kk > 0 || accumulate) ? 1u : 0u);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
        __syncwarp();
      };
      uint32_t g = 0;
      bool ok = true;
      for (int it = 0; ok && walk.next(shape, seg); ++it) {
        const int n = seg.j1 - seg.j0;
        const int qb = it % C::kQBufs;
        const int ob = C::kEpi ? it & 1 : 0;  // O buffer
        // S of tile i of the segment (every query tile), with what it frees.
        auto scores = [&](int i) -> bool {
          const int st = (g + i) % C::kStages;
          if (!warp_wait(&k_full[st], ((g + i) / C::kStages) & 1, ctl, timeout_ns, status, 4)) return false;
          tc_fence_after();
          if constexpr (kT == 1) issue_s((g + i) % kLook, qb, st);
          return true;
        };
        auto scores_done = [&](int i) {
          commit(&k_empty[(g + i) % C::kStages]);
          if (i == n - 1) commit(&q_empty[qb]);
        };
        if (!(ok = warp_wait(&q_full[qb], (it / C::kQBufs) & 1, ctl, timeout_ns, status, 5))) break;
        for (int i = 0; i < min(kLook, n); ++i) {
          if (!(ok = scores(i))) break;
          if constexpr (kT == 2) {
            issue_s(0, 0, g % C::kStages);
            issue_s(1, 0, g % C::kStages);
          }
          scores_done(i);
        }
        for (int j = 0; ok && j < n; ++j) {
          const uint32_t gj = g + j;
          const int st = gj % C::kVStages;
#pragma unroll
          for (int x = 0; x < kT; ++x) {
            const int buf = kT == 2 ? x : static_cast<int>(gj % kLook);
            if (!(ok = warp_wait(&p_ready[buf], (gj / kLook) & 1, ctl, timeout_ns, status, 6))) break;
            if (x == 0) {
              if (!(ok = warp_wait(&v_ok[st], (gj / C::kVStages) & 1, ctl, timeout_ns, status, 7))) break;
            }
            if (C::kEpi && j == 0 && it >= 2) {
              if (!(ok = warp_wait(&o_empty[ob], ((it >> 1) & 1) ^ 1, ctl, timeout_ns, status, 11))) break;
            }
            tc_fence_after();
            issue_pv(buf, ob, st, j > 0);
            if (x == kT - 1) commit(&v_empty[st]);
            if constexpr (kLook == 2) commit(pv_done);
            if (j == n - 1) {
              // The products' arrival, and one of this warp, which has waited for the
              // segment's v_ok: after both, `patched` is what warp 3 made it.
              commit(&o_final[C::kEpi ? ob : x]);
              if (lane == 0) mbar_arrive(&o_final[C::kEpi ? ob : x]);
            }
            if (j + kLook < n) {
              if constexpr (kT == 1) {
                if (!(ok = scores(j + kLook))) break;
              } else {
                if (x == 0 && !(ok = scores(j + 1))) break;
                issue_s(x, 0, (gj + 1) % C::kStages);
              }
              if (x == kT - 1) scores_done(j + kLook);
            }
          }
        }
        g += n;
      }
    }
  } else if (wg <= kT) {
    if constexpr (C::kLaunchRegs != 0) warpgroup_reg_inc<C::kRegsWork>();
    // ---------------- softmax and correction of query tile x (and its epilogue) ----------------
    const int x = wg - 1;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    constexpr int kCopyRows = kTileRows / kRep;
    const int copy = r / kCopyRows;
    const int row = group * C::kRows + x * kTileRows + r % kCopyRows;  // of the item's R rows
    const int node = row % shape.T;
    const bool any_row = row - lane < shape.R;  // some row of this warp exists
    // The bits of a tree of one tile serve all heads of its sequence: the walk to
    // the root took 3200 of the 14200 cycles of an item of two tiles (80 to 71 us
    // for 336 of them, 688 rows; 67 with the blocks left out).
    uint32_t kept[4 / kRep] = {};
    int kept_b = -1;
    uint32_t g = 0;
    bool ok = true;
    for (int it = 0; ok && walk.next(shape, seg); ++it) {
      const uint32_t o_addr = t_lane + D * (C::kEpi ? it & 1 : x);
      const int size = tree_size(shape, seg.b);
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = seg.j0; ok && j < seg.j1; ++j, ++g) {
        const int buf = kT == 2 ? x : static_cast<int>(g % kLook);
        const uint32_t s_addr = t_lane + C::kColS0 + 128u * buf;
        uint32_t mask[4 / kRep];
        const bool on_tree = j >= seg.n_cache;
        const int lim = seg.len - j * kTileRows;
        if (on_tree) {
          if (seg.b != kept_b || shape.T > kTileRows) {
            tree_mask(shape, seg.b, row < shape.R ? node : size, size, (j - seg.n_cache) * kTileRows + copy * kCopyRows,
                      kept);
            kept_b = seg.b;
          }
#pragma unroll
          for (int i = 0; i < 4 / kRep; ++i) mask[i] = kept[i];
        }
        if (!(ok = warp_wait(&s_full[buf], (g / kLook) & 1, ctl, timeout_ns, status, 8))) break;
        tc_fence_after();
        if (any_row) {
          float alpha;
          bool need;
          if (on_tree || lim < kTileRows) {
            if (!on_tree) first_bits(lim - copy * kCopyRows, mask);
            softmax_tile<kBf16, true, 0, kRep>(s_addr, copy, mask, scale_log2, m_run, l_run, alpha, need);
          } else {
            softmax_tile<kBf16, false, kLook == 2 ? 0 : 3, kRep>(s_addr, copy, mask, scale_log2, m_run, l_run, alpha,
                                                                 need);
          }
          // O may be rescaled once P V of the tile before is in it: with one S
          // buffer S(j) completing says so.
          if (j > seg.j0 && __any_sync(0xffffffffu, need)) {
            if constexpr (kLook == 2) {
              if (!(ok = warp_wait(pv_done, (g - 1) & 1, ctl, timeout_ns, status, 9))) break;
              tc_fence_after();
            }
#pragma unroll
            for (int cb = 0; cb < D / 32; ++cb) {
              uint32_t o[32];
              tmem_ld32(o_addr + cb * 32, o);
              tmem_wait_ld();
              reg_fence(o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
              tmem_st32(o_addr + cb * 32, o);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[buf]);
      }
      if (!ok) break;
      const bool live = node < size;  // other rows: nothing
      if constexpr (C::kEpi) {
        const int ob = it & 1;
        if (it >= 2 && !(ok = warp_wait(&o_empty[ob], ((it >> 1) & 1) ^ 1, ctl, timeout_ns, status, 12))) break;
        if (l_run != l_run) m_run = 0.0f;  // a NaN row stays one
        reinterpret_cast<float2*>(smem + C::kMlOff)[ob * kTileRows + r] =
            (any_row && live) ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.0f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_ready[ob]);
      } else {
        if (!(ok = warp_wait(&o_final[x], it & 1, ctl, timeout_ns, status, 10))) break;
        if (!any_row) continue;
        if (l_run != l_run) m_run = 0.0f;  // a NaN row stays one
        tc_fence_after();
        const long long slot_row =
            ((static_cast<long long>(blockIdx.y) * gridDim.x + group) * 2 + (it > 0 ? 1 : 0)) * C::kRows;
        finish_row<D, kBf16>(o_addr, seg.j0 == 0 && seg.j1 == seg.n_all, live, row < shape.R, m_run, l_run,
                             (static_cast<long long>(seg.b) * shape.Hkv + seg.h) * shape.R + row,
                             slot_row + x * kTileRows + r, shape.d_real, out, lse, part_ml, part_o);
        if (*patched && live && row < shape.R)
          add_not_finite<D, kBf16>(shape, seg, node, 0, D, seg.j0 == 0 && seg.j1 == seg.n_all,
                                   out + ((static_cast<long long>(seg.b) * shape.Hkv + seg.h) * shape.R + row) * shape.d_real,
                                   part_o, slot_row + x * kTileRows + r);
      }
    }
  } else {
    if constexpr (C::kLaunchRegs != 0) warpgroup_reg_inc<C::kRegsWork>();
    // ---------------- epilogue (kEpi) ----------------
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    bool ok = true;
    // (Every warp walks every segment, failed or not: the copies meet at
    // barriers.)
    for (int it = 0; walk.next(shape, seg); ++it) {
      const int ob = it & 1;
      if (ok) ok = warp_wait(&l_ready[ob], (it >> 1) & 1, ctl, timeout_ns, status, 13);
      if (ok) ok = warp_wait(&o_final[ob], (it >> 1) & 1, ctl, timeout_ns, status, 14);
      if (ok) tc_fence_after();
      const bool whole = seg.j0 == 0 && seg.j1 == seg.n_all;
      const long long item_row = (static_cast<long long>(seg.b) * shape.Hkv + seg.h) * shape.R;
      // A part's slot: 0 of this CTA for its first segment, 1 for its last.
      const long long slot_row =
          ((static_cast<long long>(blockIdx.y) * gridDim.x + group) * 2 + (it > 0 ? 1 : 0)) * C::kRows;
      const float2* ml = reinterpret_cast<const float2*>(smem + C::kMlOff) + ob * kTileRows;
      if constexpr (kRep > 1) {
        finish_copies<D, kRep, kBf16>(ok, t_lane + D * ob, r, whole, ml, reinterpret_cast<float4*>(smem + C::kJoinOff),
                                      shape, seg, *patched != 0, item_row, slot_row, out, lse, part_ml, part_o);
      } else if (ok && group * C::kRows + r - lane < shape.R) {
        const int row = group * C::kRows + r;
        finish_row<D, kBf16>(t_lane + D * ob, whole, ml[r].y != 0.0f, row < shape.R, ml[r].x, ml[r].y, item_row + row,
                             slot_row + r, shape.d_real, out, lse, part_ml, part_o);
        if (*patched && ml[r].y != 0.0f && row < shape.R)
          call_add_not_finite<D, kBf16>(shape, seg, row % shape.T, 0, D, whole, out + (item_row + row) * shape.d_real,
                                        part_o, slot_row + r);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[ob]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (ctl->abort != 0) {
    // A wait gave up: copies and products may be under way, which have to end
    // before the CTA's shared and tensor memory are another's.
    if (warp == 1) {
      if (elect_one()) umma_commit(drained);
      __syncwarp();
      mbar_drain(drained, 0);
      auto drain = [&](uint64_t* full, int depth, int n) {
#pragma unroll 1
        for (int i = max(n - depth, 0); i < n; ++i) mbar_drain(&full[i % depth], (i / depth) & 1);
      };
      drain(k_full, C::kStages, loads[0]);
      drain(v_full, C::kVStages, loads[1]);
      drain(q_full, C::kQBufs, loads[2]);
    }
    __syncthreads();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

constexpr int kJoinWarps = 8;

// Joins the parts of cut items: with M the largest m,
// o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over a row's parts in run
// order.  Bound by the latency of the loads (a row's parts are a few KB, in
// L2): a warp has four rows (part_at: a lane holds columns of one of them) and
// four parts of each in flight, and kShare warps divide the rows' parts.
template <int D, bool kBf16, int kShare>
__global__ void __launch_bounds__(32 * kJoinWarps)
    tree_attn_combine_kernel(const __grid_constant__ TreeShape shape, uint16_t* __restrict__ out,
                             float* __restrict__ lse, TreePlan plan, const float* __restrict__ part_ml,
                             const float* __restrict__ part_o, int groups, int runs, int group_rows) {
  constexpr int kVec = D / 32;  // float4 of a part's four rows a lane
  constexpr int kBatch = 4;
  pdl_launch_dependents();
  pdl_wait_prerequisites();
  const TreeCut cut = plan.cut[blockIdx.y];
  if (!tree_cut_ok(cut, shape.B * shape.Hkv, runs)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = warp % kShare;
  const int row0 = (blockIdx.x * (kJoinWarps / kShare) + warp / kShare) * 4;
  const int row = row0 + ((lane >> 1) & 3);
  const bool row_ok = row < shape.R;
  const int group = row0 / group_rows;
  float m = -INFINITY, l = 0.0f;
  float4 acc[kVec];
#pragma unroll
  for (int e = 0; e < kVec; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int p = share; p < cut.parts; p += kShare * kBatch) {
    float2 ml[kBatch];
    float4 v[kBatch][kVec];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int pi = p + i * kShare;
      ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[i][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (pi < cut.parts && row_ok) {
        const long long slot = (static_cast<long long>(cut.run + pi) * groups + group) * 2 + (pi == 0 ? cut.slot : 0);
        const long long prow0 = slot * group_rows + row0 % group_rows;
        ml[i] = *reinterpret_cast<const float2*>(part_ml + (prow0 + (row - row0)) * 2);
        const float4* src = reinterpret_cast<const float4*>(part_o + prow0 * D) + lane;
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[i][e] = src[32 * e];
      }
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) top = fmaxf(top, ml[i].x);
    if (top == -INFINITY) continue;
    const float keep = ex2(m - top);
    m = top;
    l *= keep;
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[e].x *= keep, acc[e].y *= keep, acc[e].z *= keep, acc[e].w *= keep;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const float w = ex2(ml[i].x - top);
      l += w * ml[i].y;
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        acc[e].x += w * v[i][e].x, acc[e].y += w * v[i][e].y;
        acc[e].z += w * v[i][e].z, acc[e].w += w * v[i][e].w;
      }
    }
  }
  if constexpr (kShare > 1) {
    __shared__ float4 s_acc[kJoinWarps][kVec][32];
    __shared__ float2 s_ml[kJoinWarps][32];
#pragma unroll
    for (int e = 0; e < kVec; ++e) s_acc[warp][e][lane] = acc[e];
    s_ml[warp][lane] = make_float2(m, l);
    __syncthreads();
    if (share != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kShare; ++i) m = fmaxf(m, s_ml[warp + i][lane].x);
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < kVec; ++e) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (m != -INFINITY) {
#pragma unroll
      for (int i = 0; i < kShare; ++i) {
        const float2 ml = s_ml[warp + i][lane];
        const float w = ex2(ml.x - m);
        l += w * ml.y;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float4 v = s_acc[warp + i][e][lane];
          acc[e].x += w * v.x, acc[e].y += w * v.y, acc[e].z += w * v.z, acc[e].w += w * v.w;
        }
      }
    }
  }
  if (!row_ok) return;
  const long long row_g = static_cast<long long>(cut.item) * shape.R + row;
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // of a NaN: NaN
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const int col = (4 * e + (lane >> 3)) * 8 + (lane & 1) * 4;
    if (col < shape.d_real)
      *reinterpret_cast<uint2*>(out + row_g * shape.d_real + col) =
          make_uint2(pack2<kBf16>(acc[e].x * inv, acc[e].y * inv), pack2<kBf16>(acc[e].z * inv, acc[e].w * inv));
  }
  if (lse != nullptr && (lane & 25) == 0) lse[row_g] = l == 0.0f ? -INFINITY : m + lg2(l);
}

// The launch: groups of kRows rows x runs, as many CTAs as are resident
// together (or as the items cost at full caches, if less).
struct TreeGrid {
  bool whole;     // a CTA per item (and group)
  int copies;     // of the rows
  int groups, runs;
  int cuts;  // entries of the plan: items or runs, whichever are fewer
  size_t plan_bytes, ml_bytes, o_bytes;
};

constexpr int tree_tiles_per_cta(int64_t R) { return R > kTileRows ? 2 : 1; }
constexpr int tree_copies(int64_t R) { return R <= 32 ? 4 : R <= 64 ? 2 : 1; }

constexpr int kFewTiles = 10;

TreeGrid tree_grid(int64_t B, int64_t Hkv, int64_t G, int64_t T, int64_t L, int64_t D, int sms) {
  const int64_t tile_rows = tree_tiles_per_cta(G * T) * kTileRows, items = B * Hkv;
  const int64_t item_tiles = (L + kTileRows - 1) / kTileRows + (T + kTileRows - 1) / kTileRows;
  TreeGrid t{};
  // A CTA per item, where that is quicker than runs: where an item's tiles, one
  // after another, take no longer than the runs' share of all of them (a CTA's
  // part of the items' cost) and what cutting the items adds, the plan, the
  // second launch and its join: 2 tiles, and with the rows 0 or 3/4 of the share
  // more (up to 64 rows runs have copies, which an item alone has not).  us a
  // call, runs / a CTA per item, 8 KV heads of 128:
  //   32 rows: 1 sequence of 2 cache tiles 8.8 / 8.6, of 4 9.1 / 10.9; 8 of
  //     2, 4 and 8 11.5 / 9.5, 12.5 / 11.5 and 14.3 / 16.6;
  //   256 rows: 1 of 2 12.3 / 12.8; 4 of 2 and 8 16.8 / 13.6 and 19.6 / 24.1;
  //     8 of 4 and 8 25.3 / 17.4 and 28.3 / 25.6.
  // The host does not see the lengths, and the longest item is what a CTA per
  // item waits for: only up to kFewTiles (58 sequences of 0 to 1809 keys in a
  // cache of 2256, 2 KV heads, 150 rows: 32.0 / 36.0).
  const int64_t groups = (G * T + tile_rows - 1) / tile_rows;
  const int64_t share4 = items * groups * (item_tiles + kItemCost) * (tree_copies(G * T) > 1 ? 4 : 7);
  if (items * groups <= sms && item_tiles <= kFewTiles && 4 * item_tiles * sms <= 8 * static_cast<int64_t>(sms) + share4) {
    t.whole = true;
    t.copies = 1;
    t.groups = static_cast<int>(groups);
    return t;
  }
  t.copies = tree_copies(G * T);
  const int64_t group_rows = tile_rows / t.copies, width = D > 64 ? 128 : 64;
  t.groups = static_cast<int>((G * T + group_rows - 1) / group_rows);
  t.runs = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(sms / t.groups, items * (item_tiles + kItemCost))));
  const size_t rows = static_cast<size_t>(t.groups) * t.runs * 2 * group_rows;
  t.cuts = static_cast<int>(std::min<int64_t>(items, t.runs));
  t.plan_bytes = (static_cast<size_t>(t.cuts) * sizeof(TreeCut) + 255) / 256 * 256;
  t.ml_bytes = rows * 8;
  t.o_bytes = rows * static_cast<size_t>(width) * 4;
  return t;
}

template <int D, bool kBf16, int kShare>
int launch_tree_combine(const TreeAttnArgs& a, const TreeGrid& t, const TreeShape& shape, const TreePlan& plan,
                        const float* part_ml, const float* part_o, int group_rows) {
  const int64_t per_block = kJoinWarps / kShare * 4;
  const dim3 grid(static_cast<unsigned>((a.G * a.T + per_block - 1) / per_block), static_cast<unsigned>(t.cuts));
  return launch_pdl(tree_attn_combine_kernel<D, kBf16, kShare>, grid, dim3(32 * kJoinWarps), 0, a.stream, 1, shape,
                    static_cast<uint16_t*>(a.o), a.lse, plan, part_ml, part_o, t.groups, t.runs, group_rows);
}

template <int D, int kT, int kRep, bool kBf16>
int launch_tree_t(const TreeAttnArgs& a, const TreeGrid& t) {
  using C = TreeCfg<D, kT, kRep>;
  static_assert(C::kSmemBytes <= 232448, "shared memory exceeds the sm_100 limit");
  auto kern = tree_attn_kernel<D, kT, kRep, kBf16>;
  if (int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::kSmemBytes, C::kLaunchRegs, nullptr)) return rc;
  const TreeShape shape{a.kv_lens, a.tree_sizes, a.parents, a.parent_stride, static_cast<const uint16_t*>(a.v_tree),
                        a.v_tree_stride[0], a.v_tree_stride[1], a.v_tree_stride[2], static_cast<int>(a.B),
                        static_cast<int>(a.Hkv), static_cast<int>(a.T), static_cast<int>(a.L),
                        static_cast<int>(a.G * a.T), static_cast<int>(a.D)};
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const TreePlan plan{reinterpret_cast<TreeCut*>(ws), a.B * a.Hkv <= t.runs ? 1 : 0, t.whole ? 1 : 0};
  float* part_ml = reinterpret_cast<float*>(ws + t.plan_bytes);
  float* part_o = reinterpret_cast<float*>(ws + t.plan_bytes + t.ml_bytes);
  const dim3 grid(static_cast<unsigned>(t.groups), static_cast<unsigned>(t.whole ? a.B * a.Hkv : t.runs));
  if (int rc = launch_pdl(kern, grid, dim3(C::kThreads), C::kSmemBytes, a.stream, 1, *a.tm_q, *a.tm_k, *a.tm_v, *a.tm_kt,
                          *a.tm_vt, shape, static_cast<uint16_t*>(a.o), a.lse, plan, part_ml, part_o, a.scale_log2,
                          a.timeout_ns, a.status))
    return rc;
  if (t.whole) return kOk;
  if (t.runs == 1) return kOk;  // nothing is cut
  // An item has about runs / items parts and one: with two or more, warps share
  // its rows' parts.
  const int64_t parts = t.runs / (a.B * a.Hkv);
  if (parts >= 8) return launch_tree_combine<D, kBf16, 8>(a, t, shape, plan, part_ml, part_o, C::kRows);
  if (parts >= 2) return launch_tree_combine<D, kBf16, 2>(a, t, shape, plan, part_ml, part_o, C::kRows);
  return launch_tree_combine<D, kBf16, 1>(a, t, shape, plan, part_ml, part_o, C::kRows);
}

template <int D, bool kBf16>
int launch_tree_r(const TreeAttnArgs& a, const TreeGrid& t) {
  switch (t.copies) {
    case 4: return launch_tree_t<D, 1, 4, kBf16>(a, t);
    case 2: return launch_tree_t<D, 1, 2, kBf16>(a, t);
    default: break;
  }
  if (tree_tiles_per_cta(a.G * a.T) == 2) return launch_tree_t<D, 2, 1, kBf16>(a, t);
  return launch_tree_t<D, 1, 1, kBf16>(a, t);
}

}  // namespace

int tree_attn_q_box_rows(int64_t B, int64_t Hkv, int64_t G, int64_t T, int64_t L, int64_t D, int sms) {
  return kTileRows / tree_grid(B, Hkv, G, T, L, D, sms).copies;
}

size_t tree_attn_workspace_bytes(int64_t B, int64_t Hkv, int64_t G, int64_t T, int64_t L, int64_t D, int sms) {
  const TreeGrid t = tree_grid(B, Hkv, G, T, L, D, sms);
  return t.plan_bytes + t.ml_bytes + t.o_bytes;
}

int launch_tree_attn(const TreeAttnArgs& a) {
  const TreeGrid t = tree_grid(a.B, a.Hkv, a.G, a.T, a.L, a.D, a.sms);
  if (a.D <= 64) return a.bf16 ? launch_tree_r<64, true>(a, t) : launch_tree_r<64, false>(a, t);
  return a.bf16 ? launch_tree_r<128, true>(a, t) : launch_tree_r<128, false>(a, t);
}

}  // namespace tk
