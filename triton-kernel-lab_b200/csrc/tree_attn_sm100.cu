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
// Work is cut where the lengths are known, on the device: an item is a (batch,
// KV head), its work its key tiles, and the items' tiles in one row are
// divided into equal runs, one per CTA (of each group of 128 kT rows), so a
// batch of any lengths keeps every SM busy to the end.  A run may begin and
// end inside an item: those (at most two) parts go to a workspace as fp32 O,
// m and l, and tree_attn_combine_kernel joins each row's parts in run order
// (bitwise reproducible, no atomics).
//
// Cache rows past kv_lens and tree rows past tree_sizes may hold anything: the
// scores of masked keys are replaced before they are used, and the rows of a
// V tile past the last valid key are cleared in shared memory (0 times NaN
// would be NaN in the product).
#include <algorithm>

#include "attn_launch.h"
#include "sm100_primitives.cuh"

namespace tk {
namespace {

// D: kernel width (64 or 128); kT: 128-row query tiles per CTA.
template <int D, int kT>
struct TreeCfg {
  static constexpr int kThreads = 128 * (1 + kT);
  static constexpr int kMinBlocks = D == 64 ? 2 : 1;
  // S buffers per query tile: with one tile per CTA and SM a second one lets
  // S(j + 1) run under the softmax of S(j); two CTAs or tiles cover each other.
  static constexpr int kLook = (D == 128 && kT == 1) ? 2 : 1;
  static constexpr int kStages = (kT == 1) ? 3 : 2;
  // 0: launched with registers to spare, no redistribution.
  static constexpr int kLaunchRegs = (D == 64) ? 128 : (kT == 2 ? 168 : 0);
  static constexpr int kRegsCtrl = 56;
  static constexpr int kRegsSoftmax = (D == 64) ? 200 : 224;
  static_assert(kLaunchRegs == 0 || kRegsCtrl + kT * kRegsSoftmax <= (1 + kT) * kLaunchRegs, "register split");
  static constexpr int kTileBytes = kTileRows * D * 2;
  static constexpr int kKOff = kT * kTileBytes;
  static constexpr int kVOff = kKOff + kStages * kTileBytes;
  static constexpr int kBarOff = kVOff + kStages * kTileBytes;
  // q_full, q_empty, k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2], p_ready[2], o_final[2], pv_done
  static constexpr int kNumBars = 2 + 4 * kStages + 7;
  static constexpr int kCtlOff = kBarOff + kNumBars * 8;
  static constexpr int kSmemBytes = kCtlOff + 16 + 32 + 64;  // control, first segment, scan
  static constexpr uint32_t kTmemCols = (D == 64) ? 256 : 512;
  static constexpr uint32_t kColS0 = kT * D;  // O of tile x at column x D, S buffers from here
};

constexpr float kTreeRescale = 8.0f;  // as the forward's: P stays below 2^8, O is rescaled rarely

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

// Walks a CTA's run, one segment at a time.
struct TreeWalk {
  int b, h, j, left;
  __device__ __forceinline__ bool next(const TreeShape& s, TreeSeg& seg) {
    if (left <= 0) return false;
    seg.b = b;
    seg.h = h;
    seg.len = cache_len(s, b);
    seg.n_cache = tiles_of(seg.len);
    seg.n_all = seg.n_cache + tiles_of(s.T);
    seg.j0 = j;
    seg.j1 = min(seg.n_all, j + left);
    left -= seg.j1 - seg.j0;
    j = 0;
    if (++h == s.Hkv) {
      h = 0;
      ++b;
    }
    return true;
  }
};

// The start of the workspace: the run length, then each batch's first tile
// (of one KV head's worth: multiply by Hkv).
struct TreePlan {
  int* run;
  int* base;
};

// One 128-key tile of one row: as the forward's softmax step, with `mask`
// (kMasked) a bit per key.
template <bool kBf16, bool kMasked, int kEmuPairs>
__device__ __forceinline__ void softmax_tile(uint32_t s_addr, const uint32_t (&mask)[4], float scale_log2, float& m_run,
                                             float& l_run, float& alpha, bool& need) {
  uint32_t s[4][32];
  tmem_ld32(s_addr, s[0]);
  tmem_ld32(s_addr + 32, s[1]);
  tmem_wait_ld();
  reg_fence(s[0]);
  reg_fence(s[1]);
  tmem_ld32(s_addr + 64, s[2]);
  tmem_ld32(s_addr + 96, s[3]);
  float mx[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) mx[i] = -INFINITY;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (b == 2) {
      tmem_wait_ld();
      reg_fence(s[2]);
      reg_fence(s[3]);
    }
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      if constexpr (kMasked) {
        if (!((mask[b] >> c) & 1u)) s[b][c] = __float_as_uint(-INFINITY);
        if (!((mask[b] >> (c + 1)) & 1u)) s[b][c + 1] = __float_as_uint(-INFINITY);
      }
      mx[(c >> 1) & 7] = fmax3(mx[(c >> 1) & 7], __uint_as_float(s[b][c]), __uint_as_float(s[b][c + 1]));
    }
  }
  const float mxa = fmax3(mx[0], mx[1], mx[2]), mxb = fmax3(mx[3], mx[4], mx[5]);
  const float m_tile = fmax3(mxa, mxb, fmaxf(mx[6], mx[7]));
  const float m_new = fmaxf(m_run, m_tile * scale_log2);
  need = m_new > m_run + kTreeRescale;
  const float m_use = need ? m_new : m_run;
  alpha = (m_run == -INFINITY) ? 0.0f : ex2(m_run - m_use);
  const float ms = (m_use == -INFINITY) ? 0.0f : m_use;
  const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
  const uint64_t negm2 = f2_pack(-ms, -ms);
  uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t pk[16];
#pragma unroll
    for (int c = 0; c < 32; c += 2) {
      float x0, x1, p0, p1;
      f2_unpack(ffma2(f2_pack(__uint_as_float(s[b][c]), __uint_as_float(s[b][c + 1])), scale2, negm2), x0, x1);
      // Masked tiles keep every exponential on the MUFU so that masked
      // entries are exactly zero.
      if (!kMasked && ((c >> 1) & 7) >= 8 - kEmuPairs) {
        exp2_fma_pair(x0, x1, p0, p1);
      } else {
        p0 = ex2(x0);
        p1 = ex2(x1);
      }
      sum2[(c >> 1) & 1] = fadd2(sum2[(c >> 1) & 1], f2_pack(p0, p1));
      pk[c >> 1] = pack2<kBf16>(p0, p1);
    }
    tmem_st16(s_addr + b * 16, pk);
  }
  float sa0, sa1, sb0, sb1;
  f2_unpack(sum2[0], sa0, sa1);
  f2_unpack(sum2[1], sb0, sb1);
  l_run = l_run * alpha + ((sa0 + sa1) + (sb0 + sb1));
  m_run = m_use;
}

// Bit n of the result: the row's node attends tree node 128 tile + n.
__device__ __forceinline__ void tree_mask(const TreeShape& s, int b, int node, int size, int tile, uint32_t (&mask)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) mask[i] = 0;
  if (node >= size) return;
  const int lo = tile * kTileRows;
  if (s.parents == nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = node + 1 - lo - 32 * i;  // nodes of this word up to and including the row's own
      mask[i] = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
    }
    return;
  }
  const int* up = s.parents + b * s.parent_stride;
  while (node >= lo) {  // ends: every step goes to a smaller node
    const int n = node - lo;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((n >> 5) == i) mask[i] |= 1u << (n & 31);
    const int parent = up[node];
    node = parent < node ? parent : -1;
  }
}

template <int D, int kT, bool kBf16>
__global__ void __launch_bounds__(TreeCfg<D, kT>::kThreads, TreeCfg<D, kT>::kMinBlocks)
    tree_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_kt,
                     const __grid_constant__ CUtensorMap tm_vt, const __grid_constant__ TreeShape shape,
                     uint16_t* __restrict__ out, float* __restrict__ lse, TreePlan plan, float* __restrict__ part_ml,
                     float* __restrict__ part_o, float scale_log2, unsigned long long timeout_ns, int* status) {
  using C = TreeCfg<D, kT>;
  constexpr int kLook = C::kLook;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(status, kOk, kErrMisaligned);
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int wg = warp >> 2;
  const int group = blockIdx.x;  // rows [group 128 kT, ...) of every item

  uint8_t* sQ = smem;
  uint8_t* sK = smem + C::kKOff;
  uint8_t* sV = smem + C::kVOff;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + C::kStages;
  uint64_t* v_full = k_empty + C::kStages;
  uint64_t* v_empty = v_full + C::kStages;
  uint64_t* s_full = v_empty + C::kStages;  // [2]: query tile, or S buffer of the one tile
  uint64_t* p_ready = s_full + 2;           // [2]
  uint64_t* o_final = p_ready + 2;          // [2]: query tile
  uint64_t* pv_done = o_final + 2;          // with two S buffers: P V of every tile
  CtaControl* ctl = reinterpret_cast<CtaControl*>(smem + C::kCtlOff);
  int* first = reinterpret_cast<int*>(smem + C::kCtlOff + 16);  // b, h, j, tiles of this CTA's run
  int* scan = first + 8;                                         // [warps]

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
      mbar_init(&o_final[i], 1);
    }
    mbar_init(pv_done, 1);
    ctl->abort = 0;
    fence_mbarrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_map(&tm_q);
    tma_prefetch_map(&tm_k);
    tma_prefetch_map(&tm_v);
    tma_prefetch_map(&tm_kt);
    tma_prefetch_map(&tm_vt);
  }
  if (warp == 1) tmem_alloc(&ctl->tmem_base, C::kTmemCols);

  // This CTA's run: a scan of the batch's tiles, each thread over consecutive sequences.
  {
    const int per = (shape.B + C::kThreads - 1) / C::kThreads;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, shape.B), b1 = min(b0 + per, shape.B);
    const int tree_tiles = tiles_of(shape.T);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(cache_len(shape, b)) + tree_tiles;
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
    if (threadIdx.x == 0) first[3] = max(min(run, total - start), 0);
    const bool writes = blockIdx.x == 0 && blockIdx.y == 0;
    if (writes && threadIdx.x == 0) *plan.run = run;
    for (int b = b0; b < b1; ++b) {
      const int n = tiles_of(cache_len(shape, b)) + tree_tiles;
      const int from = before * shape.Hkv;
      if (start >= from && start < from + n * shape.Hkv) {
        first[0] = b;
        first[1] = (start - from) / n;
        first[2] = (start - from) % n;
      }
      if (writes) plan.base[b] = before;
      before += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem_base;
  TreeWalk walk{first[0], first[1], first[2], first[3]};
  TreeSeg seg;

  // Every role walks the same segments; barrier phases follow running counts
  // of segments and key tiles, so consecutive segments pipeline.
  if (wg == 0) {
    if constexpr (C::kLaunchRegs != 0) warpgroup_reg_dec<C::kRegsCtrl>();
    if (warp == 0 || warp == 2) {
      // ---------------- TMA producers: warp 0 Q and K, warp 2 V ----------------
      if (lane == 0) {
        const bool is_k = warp == 0;
        uint8_t* ring = is_k ? sK : sV;
        uint64_t* full = is_k ? k_full : v_full;
        uint64_t* empty = is_k ? k_empty : v_empty;
        uint32_t g = 0;
        bool ok = true;
        for (int it = 0; ok && walk.next(shape, seg); ++it) {
          if (is_k) {
            if (it > 0 && !(ok = mbar_wait(q_empty, (it - 1) & 1, ctl, timeout_ns, status, 1))) break;
            mbar_arrive_expect_tx(q_full, kT * C::kTileBytes);
#pragma unroll
            for (int x = 0; x < kT; ++x)
#pragma unroll
              for (int blk = 0; blk < D / 64; ++blk)
                tma_load_3d(sQ + x * C::kTileBytes + blk * kBlockBytes, &tm_q, q_full, blk * 64,
                            (group * kT + x) * kTileRows, seg.b * shape.Hkv + seg.h);
          }
          for (int j = seg.j0; j < seg.j1; ++j, ++g) {
            const int st = g % C::kStages;
            if (!(ok = mbar_wait(&empty[st], ((g / C::kStages) & 1) ^ 1, ctl, timeout_ns, status, is_k ? 2 : 3))) break;
            mbar_arrive_expect_tx(&full[st], C::kTileBytes);
            const bool on_cache = j < seg.n_cache;
            const CUtensorMap* map = on_cache ? (is_k ? &tm_k : &tm_v) : (is_k ? &tm_kt : &tm_vt);
            const int row = (on_cache ? j : j - seg.n_cache) * kTileRows;
#pragma unroll
            for (int blk = 0; blk < D / 64; ++blk)
              tma_load_4d(ring + st * C::kTileBytes + blk * kBlockBytes, map, &full[st], blk * 64, row, seg.h, seg.b);
          }
        }
      }
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
      auto issue_s = [&](int x, int st) {
        const uint32_t q_lo = q_lo0 + (kT == 2 ? x * kTileLo : 0u);
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
      auto issue_pv = [&](int x, int st, bool accumulate) {
        const uint32_t v_lo = v_lo0 + st * kTileLo;
        const uint32_t d = tmem + (kT == 2 ? D * x : 0u);
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
        const int size = tree_size(shape, seg.b);
        // S of tile i of the segment (every query tile), with what it frees.
        auto scores = [&](int i) -> bool {
          const int st = (g + i) % C::kStages;
          if (!warp_wait(&k_full[st], ((g + i) / C::kStages) & 1, ctl, timeout_ns, status, 4)) return false;
          tc_fence_after();
          if constexpr (kT == 1) issue_s((g + i) % kLook, st);
          return true;
        };
        auto scores_done = [&](int i) {
          commit(&k_empty[(g + i) % C::kStages]);
          if (i == n - 1) commit(q_empty);
        };
        if (!(ok = warp_wait(q_full, it & 1, ctl, timeout_ns, status, 5))) break;
        for (int i = 0; i < min(kLook, n); ++i) {
          if (!(ok = scores(i))) break;
          if constexpr (kT == 2) {
            issue_s(0, g % C::kStages);
            issue_s(1, g % C::kStages);
          }
          scores_done(i);
        }
        for (int j = 0; ok && j < n; ++j) {
          const uint32_t gj = g + j;
          const int st = gj % C::kStages;
#pragma unroll
          for (int x = 0; x < kT; ++x) {
            const int buf = kT == 2 ? x : static_cast<int>(gj % kLook);
            if (!(ok = warp_wait(&p_ready[buf], (gj / kLook) & 1, ctl, timeout_ns, status, 6))) break;
            if (x == 0) {
              if (!(ok = warp_wait(&v_full[st], (gj / C::kStages) & 1, ctl, timeout_ns, status, 7))) break;
              // Rows of V past the last valid key: cleared.
              const int jt = seg.j0 + j - seg.n_cache;
              const int valid = jt < 0 ? seg.len - (seg.j0 + j) * kTileRows : size - jt * kTileRows;
              if (valid < kTileRows) {
                const int from = max(valid, 0) * kSwizzleBytes;
#pragma unroll
                for (int blk = 0; blk < D / 64; ++blk)
                  for (int off = from + lane * 16; off < kBlockBytes; off += 32 * 16)
                    *reinterpret_cast<uint4*>(sV + st * C::kTileBytes + blk * kBlockBytes + off) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            tc_fence_after();
            issue_pv(buf, st, j > 0);
            if (x == kT - 1) commit(&v_empty[st]);
            if constexpr (kLook == 2) commit(pv_done);
            if (j == n - 1) commit(&o_final[x]);
            if (j + kLook < n) {
              if constexpr (kT == 1) {
                if (!(ok = scores(j + kLook))) break;
              } else {
                if (x == 0 && !(ok = scores(j + 1))) break;
                issue_s(x, (gj + 1) % C::kStages);
              }
              if (x == kT - 1) scores_done(j + kLook);
            }
          }
        }
        g += n;
      }
    }
  } else {
    if constexpr (C::kLaunchRegs != 0) warpgroup_reg_inc<C::kRegsSoftmax>();
    // ---------------- softmax, correction and epilogue of query tile x ----------------
    const int x = wg - 1;
    const int q4 = warp & 3;
    const int r = q4 * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(q4 * 32) << 16);
    const uint32_t o_addr = t_lane + D * x;
    const int row = (group * kT + x) * kTileRows + r;  // of the item's R rows
    const int node = row % shape.T;
    const bool any_row = row - lane < shape.R;  // some row of this warp exists
    const bool wide_store = (shape.d_real % 16) == 0 && (reinterpret_cast<uintptr_t>(out) & 31u) == 0;
    uint32_t g = 0;
    bool ok = true;
    for (int it = 0; ok && walk.next(shape, seg); ++it) {
      const int size = tree_size(shape, seg.b);
      float m_run = -INFINITY, l_run = 0.0f;
      for (int j = seg.j0; ok && j < seg.j1; ++j, ++g) {
        const int buf = kT == 2 ? x : static_cast<int>(g % kLook);
        const uint32_t s_addr = t_lane + C::kColS0 + 128u * buf;
        uint32_t mask[4];
        const bool on_tree = j >= seg.n_cache;
        const int lim = seg.len - j * kTileRows;
        if (on_tree) tree_mask(shape, seg.b, row < shape.R ? node : size, size, j - seg.n_cache, mask);
        if (!(ok = warp_wait(&s_full[buf], (g / kLook) & 1, ctl, timeout_ns, status, 8))) break;
        tc_fence_after();
        if (any_row) {
          float alpha;
          bool need;
          if (on_tree || lim < kTileRows) {
            if (!on_tree) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int n = lim - 32 * i;
                mask[i] = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
              }
            }
            softmax_tile<kBf16, true, 0>(s_addr, mask, scale_log2, m_run, l_run, alpha, need);
          } else {
            softmax_tile<kBf16, false, kLook == 2 ? 0 : 3>(s_addr, mask, scale_log2, m_run, l_run, alpha, need);
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
      if (ok) ok = warp_wait(&o_final[x], it & 1, ctl, timeout_ns, status, 10);
      if (!ok || !any_row) continue;
      tc_fence_after();
      const bool whole = seg.j0 == 0 && seg.j1 == seg.n_all;
      const bool live = node < size;  // other rows: nothing
      const bool row_ok = row < shape.R;
      const long long row_g = (static_cast<long long>(seg.b) * shape.Hkv + seg.h) * shape.R + row;
      if (whole) {
        const float inv = (live && l_run > 0.0f) ? 1.0f / l_run : 0.0f;
        uint16_t* orow = out + row_g * shape.d_real;
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
              if (wide_store && col < shape.d_real) {
                st_global_v8(orow + col, &w[hh * 8]);
              } else if (!wide_store) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
                  if (col + q * 8 < shape.d_real)
                    *reinterpret_cast<uint4*>(orow + col + q * 8) = make_uint4(
                        w[hh * 8 + q * 4], w[hh * 8 + q * 4 + 1], w[hh * 8 + q * 4 + 2], w[hh * 8 + q * 4 + 3]);
              }
            }
          }
        }
        if (lse != nullptr && row_ok) lse[row_g] = live ? m_run + lg2(l_run) : -INFINITY;
      } else {
        // A part: unnormalised O, m and l.  Slot 0 of this CTA for its first segment, 1 for its last.
        const long long slot = (static_cast<long long>(blockIdx.y) * gridDim.x + group) * 2 + (it > 0 ? 1 : 0);
        const long long prow = slot * (kT * kTileRows) + x * kTileRows + r;
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
            for (int q = 0; q < 4; ++q) st_global_v8(part_o + prow * D + cb * 32 + q * 8, &o[q * 8]);
          }
        }
        if (row_ok)
          *reinterpret_cast<float2*>(part_ml + prow * 2) = live ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.0f);
      }
    }
  }
  pdl_launch_dependents();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

constexpr int kJoinWarps = 8;

// Joins the parts of the rows whose item was cut: with M the largest m,
// o = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over its parts in run
// order.  warps_per_row warps (1 to 8) share a row's parts.
template <int D, bool kBf16>
__global__ void __launch_bounds__(32 * kJoinWarps)
    tree_attn_combine_kernel(const __grid_constant__ TreeShape shape, uint16_t* __restrict__ out,
                             float* __restrict__ lse, TreePlan plan, const float* __restrict__ part_ml,
                             const float* __restrict__ part_o, int groups, int group_rows, int warps_per_row) {
  constexpr int kPer = D / 32;
  __shared__ float s_acc[kJoinWarps][D];
  __shared__ float s_ml[kJoinWarps][2];
  pdl_wait_prerequisites();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int share = warp % warps_per_row;
  const long long row_g = static_cast<long long>(blockIdx.x) * (kJoinWarps / warps_per_row) + warp / warps_per_row;
  const bool exists = row_g < static_cast<long long>(shape.B) * shape.Hkv * shape.R;
  int c0 = 0, c1 = 0, start = 0, row = 0;
  const int run = *plan.run;
  if (exists) {
    row = static_cast<int>(row_g % shape.R);
    const int item = static_cast<int>(row_g / shape.R);
    const int b = item / shape.Hkv, h = item % shape.Hkv;
    const int n = tiles_of(cache_len(shape, b)) + tiles_of(shape.T);
    start = plan.base[b] * shape.Hkv + h * n;
    c0 = start / run;
    c1 = (start + n - 1) / run;
  }
  const bool cut = c1 > c0;
  float acc[kPer], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
  if (cut) {
    const int group = row / group_rows;
    constexpr int kBatch = 8;  // parts loaded before any is used
    for (int c = c0 + share; c <= c1; c += warps_per_row * kBatch) {
      float2 ml[kBatch];
      float v[kBatch][kPer];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int ci = c + i * warps_per_row;
        ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[i][e] = 0.0f;
        if (ci <= c1) {
          const long long slot = (static_cast<long long>(ci) * groups + group) * 2 + (static_cast<long long>(ci) * run >= start ? 0 : 1);
          const long long prow = slot * group_rows + row % group_rows;
          ml[i] = *reinterpret_cast<const float2*>(part_ml + prow * 2);
          const float* src = part_o + prow * D + lane * kPer;
          if constexpr (kPer == 4) {
            const float4 q = *reinterpret_cast<const float4*>(src);
            v[i][0] = q.x, v[i][1] = q.y, v[i][2] = q.z, v[i][3] = q.w;
          } else {
            const float2 q = *reinterpret_cast<const float2*>(src);
            v[i][0] = q.x, v[i][1] = q.y;
          }
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
      for (int e = 0; e < kPer; ++e) acc[e] *= keep;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w = ex2(ml[i].x - top);
        l += w * ml[i].y;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] += w * v[i][e];
      }
    }
  }
  if (warps_per_row > 1) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) s_acc[warp][lane * kPer + e] = acc[e];
    if (lane == 0) {
      s_ml[warp][0] = m;
      s_ml[warp][1] = l;
    }
    __syncthreads();
    if (share != 0) return;
    float top = -INFINITY;
    for (int i = 0; i < warps_per_row; ++i) top = fmaxf(top, s_ml[warp + i][0]);
    m = top;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
    for (int i = 0; i < warps_per_row && top != -INFINITY; ++i) {
      const float w = ex2(s_ml[warp + i][0] - top);
      l += w * s_ml[warp + i][1];
#pragma unroll
      for (int e = 0; e < kPer; ++e) acc[e] += w * s_acc[warp + i][lane * kPer + e];
    }
  }
  if (!cut) return;
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  if (lane * kPer < shape.d_real) {
    uint16_t* dst = out + row_g * shape.d_real + lane * kPer;
    if constexpr (kPer == 4) {
      *reinterpret_cast<uint2*>(dst) =
          make_uint2(pack2<kBf16>(acc[0] * inv, acc[1] * inv), pack2<kBf16>(acc[2] * inv, acc[3] * inv));
    } else {
      *reinterpret_cast<uint32_t*>(dst) = pack2<kBf16>(acc[0] * inv, acc[1] * inv);
    }
  }
  if (lse != nullptr && lane == 0) lse[row_g] = l > 0.0f ? m + lg2(l) : -INFINITY;
}

// The launch: groups of 128 kT rows x runs, as many CTAs as are resident
// together (or as there are key tiles at full caches, if fewer).
struct TreeGrid {
  int groups, runs;
  size_t plan_bytes, ml_bytes, o_bytes;
};

constexpr int tree_tiles_per_cta(int64_t D, int64_t R) { return D > 64 && R > kTileRows ? 2 : 1; }

TreeGrid tree_grid(int64_t B, int64_t Hkv, int64_t G, int64_t T, int64_t L, int64_t D, int sms) {
  const int kT = tree_tiles_per_cta(D, G * T);
  const int64_t width = D > 64 ? 128 : 64;
  const int64_t resident = sms * (width == 64 ? 2 : 1);
  TreeGrid t;
  const int64_t groups = (G * T + kT * kTileRows - 1) / (kT * kTileRows);
  const int64_t tiles = B * Hkv * ((L + kTileRows - 1) / kTileRows + (T + kTileRows - 1) / kTileRows);
  t.groups = static_cast<int>(groups);
  t.runs = static_cast<int>(std::max<int64_t>(1, std::min(resident / groups, tiles)));
  const size_t rows = static_cast<size_t>(groups) * t.runs * 2 * kT * kTileRows;
  t.plan_bytes = (256 + static_cast<size_t>(B) * 4 + 255) / 256 * 256;
  t.ml_bytes = rows * 8;
  t.o_bytes = rows * static_cast<size_t>(width) * 4;
  return t;
}

template <int D, int kT, bool kBf16>
int launch_tree_t(const TreeAttnArgs& a, const TreeGrid& t) {
  using C = TreeCfg<D, kT>;
  static_assert(C::kSmemBytes + 1024 <= 233472 / C::kMinBlocks, "shared memory exceeds the SM's");
  auto kern = tree_attn_kernel<D, kT, kBf16>;
  if (int rc = prepare_kernel(reinterpret_cast<const void*>(kern), C::kSmemBytes, C::kLaunchRegs, nullptr)) return rc;
  const TreeShape shape{a.kv_lens, a.tree_sizes, a.parents, a.parent_stride, static_cast<int>(a.B),
                        static_cast<int>(a.Hkv), static_cast<int>(a.T), static_cast<int>(a.L),
                        static_cast<int>(a.G * a.T), static_cast<int>(a.D)};
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const TreePlan plan{reinterpret_cast<int*>(ws), reinterpret_cast<int*>(ws + 256)};
  float* part_ml = reinterpret_cast<float*>(ws + t.plan_bytes);
  float* part_o = reinterpret_cast<float*>(ws + t.plan_bytes + t.ml_bytes);
  const dim3 grid(static_cast<unsigned>(t.groups), static_cast<unsigned>(t.runs));
  kern<<<grid, C::kThreads, C::kSmemBytes, a.stream>>>(*a.tm_q, *a.tm_k, *a.tm_v, *a.tm_kt, *a.tm_vt, shape,
                                                      static_cast<uint16_t*>(a.o), a.lse, plan, part_ml, part_o,
                                                      a.scale_log2, a.timeout_ns, a.status);
  if (cudaGetLastError() != cudaSuccess) return kErrLaunch;
  if (t.runs == 1) return kOk;  // nothing is cut
  const int64_t rows = a.B * a.Hkv * a.G * a.T;
  // Few rows: several warps share a row's parts.
  int warps_per_row = kJoinWarps;
  while (warps_per_row > 1 && rows * warps_per_row > 148 * 32) warps_per_row /= 2;
  const int64_t per_block = kJoinWarps / warps_per_row;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((rows + per_block - 1) / per_block));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, tree_attn_combine_kernel<D, kBf16>, shape, static_cast<uint16_t*>(a.o),
                                             a.lse, plan, static_cast<const float*>(part_ml),
                                             static_cast<const float*>(part_o), t.groups, kT * kTileRows, warps_per_row);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return kErrLaunch;
  }
  return kOk;
}

template <bool kBf16>
int launch_tree_b(const TreeAttnArgs& a, const TreeGrid& t) {
  if (a.D <= 64) return launch_tree_t<64, 1, kBf16>(a, t);
  if (tree_tiles_per_cta(a.D, a.G * a.T) == 1) return launch_tree_t<128, 1, kBf16>(a, t);
  return launch_tree_t<128, 2, kBf16>(a, t);
}

}  // namespace

size_t tree_attn_workspace_bytes(int64_t B, int64_t Hkv, int64_t G, int64_t T, int64_t L, int64_t D, int sms) {
  const TreeGrid t = tree_grid(B, Hkv, G, T, L, D, sms);
  return t.plan_bytes + t.ml_bytes + t.o_bytes;
}

int launch_tree_attn(const TreeAttnArgs& a) {
  const TreeGrid t = tree_grid(a.B, a.Hkv, a.G, a.T, a.L, a.D, a.sms);
  return a.bf16 ? launch_tree_b<true>(a, t) : launch_tree_b<false>(a, t);
}

}  // namespace tk
