// Speculative decoding around the attention: acceptance of drafted tokens
// against the target's probabilities, and the write of the accepted tokens'
// keys and values into the cache.
//
// Verification.  Node 0 is the sequence's last known token; node c > 0
// carries a drafted token x_c that continues its parent n (parents[c] < c; a
// chain has n = c - 1).  p_n is the target's distribution after node n.  From
// node 0, the children of the current node are tried in index order with the
// given uniform numbers u_c in [0, 1):
//   exact drafts (no draft probabilities): accepted if u_c (1 - S_c) < p_n(x_c),
//     S_c the mass under p_n of the earlier siblings' (different) tokens; a
//     token tried before has nothing left and is refused;
//   drafts drawn from q_n (chains only): accepted if u_c q_n(x_c) < p_n(x_c).
// The walk goes on from an accepted child.  At the last accepted node n the
// next token is the winner of an exponential race, argmax_v w_v / e_v, with
// the residual weights w = p_n without the tried tokens, max(p_n - q_n, 0),
// or p_n where n has no child; p_n also where the residual has no mass left.
// The emitted tokens are then distributed as the target's own samples.
//
// Every node's probability is loaded at once; the walk itself is a warp's, over
// the visited nodes only.
#include <algorithm>

#include "attn_launch.h"
#include "pdl_launch.h"
#include "sm100_primitives.cuh"

namespace tk {
namespace {

template <int kType>
__device__ __forceinline__ float prob_at(const void* p, int64_t i) {
  if constexpr (kType == kProbF32) {
    return static_cast<const float*>(p)[i];
  } else if constexpr (kType == kProbBf16) {
    return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p)[i]) << 16);
  } else {
    return __half2float(static_cast<const __half*>(p)[i]);
  }
}

__device__ __forceinline__ long long token_at(const VerifyArgs& a, int64_t i) {
  return a.tokens_64 ? static_cast<const long long*>(a.tokens)[i] : static_cast<const int*>(a.tokens)[i];
}

// Two scores of the race in one order: the larger score, then the lower
// index (positive floats order like their bits); 0 is no token.
__device__ __forceinline__ unsigned long long race_key(float score, int v) {
  return (static_cast<unsigned long long>(__float_as_uint(score)) << 32) | (0xffffffffu - static_cast<unsigned>(v));
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned n;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}
// Every thread of every CTA of the cluster; sync orders shared-memory accesses.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_remote(const void* mine, unsigned rank, unsigned long long x) {
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %0, %1;\n\tst.shared::cluster.u64 [r], %2;\n\t}" ::"r"(
          smem_u32(mine)),
      "r"(rank), "l"(x)
      : "memory");
}

constexpr int kVerifyThreads = 512;
constexpr int kVerifyMaxCluster = 8;
constexpr int kFilterWords = 256;

// How the vocabulary is read: a thread's step is
//   kByFour     four entries by a vector load; every row starts on their word;
//   kByOne      one entry (rows of an odd vocabulary start anywhere);
//   kCutByFour  four 16-bit entries of such a row, cut out of the two words that
//               hold them by a shift that is the row's; the steps follow the
//               noise's words.  At the row's ends, where a word is not all the
//               row's, entry by entry.
// By one is bound by its many small requests: 20.1 us against 12.5 cut for 32
// trees over 128001 bf16 entries, 56 against 30 for 108 over 97835.  With float32
// or draft probabilities the cut words take registers that loads in flight
// need: 18.3 us by one, 23.7 cut for the 128 chains below.
enum { kByFour, kByOne, kCutByFour };

// Entries [i, i + N) of the row from p[at], whose first is `shift` past a word.
template <int kType, int N, bool kShifted>
__device__ __forceinline__ void load_step(const void* p, int64_t at, int i, int shift, float (&f)[N]) {
  if constexpr (N == 1) {
    f[0] = prob_at<kType>(p, at + i);
  } else if constexpr (kType == kProbF32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + i);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else {
    const uint16_t* x = static_cast<const uint16_t*>(p) + at + i;
    uint2 v;
    if constexpr (!kShifted) {
      v = *reinterpret_cast<const uint2*>(x);
    } else {
      const uint2* w = reinterpret_cast<const uint2*>(x - shift);
      const uint2 lo = w[0], hi = w[1];
      const bool two = shift & 2;
      const uint32_t a0 = two ? lo.y : lo.x, a1 = two ? hi.x : lo.y, a2 = two ? hi.y : hi.x;
      v.x = __funnelshift_r(a0, a1, (shift & 1) * 16);
      v.y = __funnelshift_r(a1, a2, (shift & 1) * 16);
    }
    const uint32_t u[2] = {v.x, v.y};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (kType == kProbBf16) {
        f[2 * k] = __uint_as_float(u[k] << 16);
        f[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
        f[2 * k] = h.x;
        f[2 * k + 1] = h.y;
      }
    }
  }
}

// Entries between p[at] and the word of four that it is in.
template <int kType>
__device__ __forceinline__ int word_shift(const void* p, int64_t at) {
  constexpr int kBytes = kType == kProbF32 ? 4 : 2;
  return static_cast<int>((reinterpret_cast<uintptr_t>(p) + at * kBytes) / kBytes % 4);
}

// One cluster per sequence, its CTAs over the vocabulary.  Every CTA of it
// walks the tree for itself (a few loads; sharing the result would cost a
// cluster barrier more).  Bound by the row of p (and q) and the noise where
// there are many sequences, by the chain of dependent loads (tokens, their
// probabilities, the row) and the walk where there are few.  (Bringing the
// noise, which depends on none of them, into L2 at the start held up those
// loads: 30.4 to 27.7 us without it for 128 trees of 64 nodes, 8.5 to 8.3 us
// for 8.)
//
// Measured, per call: 18.3 us for 128 chains of 5 over 50257 float32 entries
// (4.2 TB/s; 16.0 us, 4.8 TB/s for 50304, whose rows start on 16 bytes);
// 10.4 us for 32 trees of 64 over 128000 bf16 entries, 3 us of it the tree (1.7
// the loads of parents and tokens and then of their probabilities); 4.6 us for
// one chain of 6 over 32000.  With 128 or 256 threads a CTA and more CTAs the
// first took 18.1 to 19.0 us, the second 11.4 to 15.9.
//
// The race is run on w times the hardware reciprocal of e (a few operations an
// element, no branch); a thread then divides for its own best only, or, if its
// second is within 2^-19 of it (16-bit probabilities and small variates take few
// values, so that happens), its warp for all its elements: the result is that
// of the rounded quotients.  Dividing wherever a
// thread's or a warp's best so far might be beaten bound it: B = 32, 128000
// entries, bf16, 24 to 45 us.
template <int kType, int kRead, bool kDraft>
__global__ void __launch_bounds__(kVerifyThreads, 2) verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int N = kRead == kByOne ? 1 : 4;
  constexpr bool kShifted = kRead == kCutByFour;
  __shared__ int s_parent[kTreeMaxNodes], s_path[kTreeMaxNodes];
  __shared__ long long s_token[kTreeMaxNodes], s_list[kTreeMaxNodes];
  __shared__ float s_prob[kTreeMaxNodes], s_uniform[kTreeMaxNodes];
  __shared__ bool s_pass[kTreeMaxNodes];
  __shared__ int s_length, s_tried;
  __shared__ unsigned s_filter[kFilterWords];
  __shared__ unsigned long long s_warp[kVerifyThreads / 32], s_best[2][kVerifyMaxCluster];
  cluster_arrive();  // waited for before the first store to another CTA's shared memory
  pdl_wait_prerequisites();
  const unsigned rank = cluster_rank(), ranks = cluster_size();
  const int64_t b = blockIdx.x / ranks;
  const int T = static_cast<int>(a.T), V = static_cast<int>(a.V);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* noise = a.noise + b * V;
  // This CTA's part of the vocabulary, in steps of N: step i has the entries
  // from N i - lead on.
  const int lead = kShifted ? word_shift<kProbF32>(noise, 0) : 0;
  const int steps = (V + lead + N - 1) / N, per = (steps + ranks - 1) / ranks;
  const int first = min(static_cast<int>(rank) * per, steps), end = min(first + per, steps);
  const int size = a.tree_sizes != nullptr ? min(max(a.tree_sizes[b], 0), T) : T;
  for (int c = threadIdx.x; c < T; c += kVerifyThreads) {
    int n = c - 1;
    if (a.parents != nullptr && c > 0) n = a.parents[b * a.parent_stride + c];
    if (n >= c || n < 0 || c >= size) n = -1;  // hangs on nothing: never reached
    const long long x = token_at(a, b * T + c);
    const bool real = n >= 0 && x >= 0 && x < V;
    const float p = real ? prob_at<kType>(a.target, b * a.target_stride[0] + n * a.target_stride[1] + x) : 0.0f;
    const float u = a.uniforms[b * T + c];
    bool pass = false;
    if (kDraft && p > 0.0f)
      pass = u * prob_at<kType>(a.draft, b * a.draft_stride[0] + n * a.draft_stride[1] + x) < p;
    s_parent[c] = n;
    s_token[c] = x;
    s_prob[c] = p;
    s_uniform[c] = u;
    s_pass[c] = pass;
  }
  for (int i = threadIdx.x; i < kFilterWords; i += kVerifyThreads) s_filter[i] = 0;
  __syncthreads();
  if (warp == 0) {
    // The walk: at each node its children in order, 32 candidates at a time.
    int length = 0, tried = 0;
    for (int n = size > 0 ? 0 : -1; n >= 0;) {
      if (lane == 0) s_path[length] = n;
      ++length;
      tried = 0;
      int next = -1;
      float mass = 0.0f;  // of the children refused so far
      for (int c0 = (n + 1) & ~31; c0 < size; c0 += 32) {
        const int c = c0 + lane;
        const bool child = c > n && c < size && s_parent[c] == n;
        const unsigned all = __ballot_sync(0xffffffffu, child), before = all & ((1u << lane) - 1u);
        if (all == 0) continue;
        const long long x = child ? s_token[c] : -1;
        bool pass;
        if constexpr (kDraft) {
          pass = child && s_pass[c];
        } else {
          bool again = (__match_any_sync(0xffffffffu, x) & before) != 0;
          for (int t = 0; t < tried; ++t) again = again || s_list[t] == x;
          const float left = child && !again && s_prob[c] > 0.0f ? s_prob[c] : 0.0f;
          float upto = left;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const float o = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += o;
          }
          const float earlier = __shfl_up_sync(0xffffffffu, upto, 1);
          pass = left > 0.0f && s_uniform[c] * fmaxf(1.0f - (mass + (lane > 0 ? earlier : 0.0f)), 0.0f) < left;
          mass += __shfl_sync(0xffffffffu, upto, 31);
        }
        const unsigned passed = __ballot_sync(0xffffffffu, pass);
        if (passed != 0) {
          next = c0 + __ffs(passed) - 1;
          break;
        }
        if (child) s_list[tried + __popc(before)] = x;
        tried += __popc(all);
        __syncwarp();
      }
      n = next;
    }
    // A filter over the steps that hold a tried token.
    for (int t = lane; !kDraft && t < tried; t += 32)
      if (s_list[t] >= 0 && s_list[t] < V) {
        const unsigned i = (static_cast<unsigned>(s_list[t]) + lead) / N;
        atomicOr(&s_filter[(i >> 5) % kFilterWords], 1u << (i & 31));
      }
    if (lane == 0) {
      s_length = length;
      s_tried = tried;
    }
  }
  __syncthreads();
  cluster_wait();
  const int length = s_length, tried = s_tried;
  if (rank == 0) {
    for (int i = threadIdx.x; i < T; i += kVerifyThreads) a.path[b * T + i] = i < length ? s_path[i] : -1;
    if (threadIdx.x == 0) a.path_lens[b] = length;
  }
  if (length == 0) {  // the same in every CTA of the cluster
    if (rank == 0 && threadIdx.x == 0) {
      if (a.tokens_64)
        static_cast<long long*>(a.next)[b] = -1;
      else
        static_cast<int*>(a.next)[b] = -1;
    }
    return;
  }
  const int last = s_path[length - 1];
  const int64_t row = b * a.target_stride[0] + last * a.target_stride[1];
  const int64_t drow = kDraft ? b * a.draft_stride[0] + last * a.draft_stride[1] : 0;
  const int shift = kShifted ? (word_shift<kType>(a.target, row) + 4 - lead) % 4 : 0;  // of the steps in p
  for (int attempt = 0; attempt < 2; ++attempt) {
    const bool residual = attempt == 0 && tried > 0;
    const bool minus = kDraft && residual;
    const bool skips = !kDraft && residual;
    auto was_tried = [&](int v) {
      bool out = false;
      for (int t = 0; t < tried; ++t) out = out || s_list[t] == v;
      return out;
    };
    float best = 0.0f, second = 0.0f, best_w = 0.0f, best_e = 1.0f;
    int index = -1;
    // Steps loaded before any is used.  By one: 18.9 us with 8, 21.5 with 4,
    // 18.8 with 12 for the 128 chains; by four: 10.4 us with 4, 14.3 with 8 for
    // the 32 trees (fewer CTAs an SM); cut: the same with 2 and 4.
    constexpr int kFlight = kRead == kByOne ? 8 : kDraft || kShifted ? 2 : 4;
    for (int i0 = first + threadIdx.x; i0 < end; i0 += kVerifyThreads * kFlight) {
      float p[kFlight][N], q[kFlight][N], e[kFlight][N];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int i = i0 + k * kVerifyThreads, v = i * N - lead;
#pragma unroll
        for (int j = 0; j < N; ++j) p[k][j] = q[k][j] = 0.0f, e[k][j] = 1.0f;
        if (i < end) {
          if (kShifted && (v < shift || v + 8 > V)) {
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (v + j >= 0 && v + j < V) p[k][j] = prob_at<kType>(a.target, row + v + j), e[k][j] = noise[v + j];
          } else {
            load_step<kType, N, kShifted>(a.target, row, v, shift, p[k]);
            load_step<kProbF32, N, false>(noise, 0, v, 0, e[k]);
            if (minus) load_step<kType, N, false>(a.draft, drow, v, 0, q[k]);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int i = i0 + k * kVerifyThreads, v = i * N - lead;
        if (skips && ((s_filter[(i >> 5) % kFilterWords] >> (i & 31)) & 1u)) {
#pragma unroll
          for (int j = 0; j < N; ++j)
            if (was_tried(v + j)) p[k][j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
          float r;
          asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e[k][j]));
          const float w = kDraft ? p[k][j] - q[k][j] : p[k][j], score = w * r;
          const bool wins = score > best;
          second = fmaxf(second, wins ? best : score);
          best = wins ? score : best;
          index = wins ? v + j : index;
          if constexpr (kDraft) {
            best_w = wins ? w : best_w;
            best_e = wins ? e[k][j] : best_e;
          }
        }
      }
    }
    // The thread's exact best; where its second is too near, the warp divides
    // for all of its elements.
    auto exact = [&](int v) {
      float w = prob_at<kType>(a.target, row + v);
      if (minus) w -= prob_at<kType>(a.draft, drow + v);
      const float score = __fdiv_rn(w, noise[v]);
      return score > 0.0f && !(skips && was_tried(v)) ? race_key(score, v) : 0ull;
    };
    const bool clear = index < 0 || (second < best * 0.999998f && best < INFINITY);
    unsigned long long key = 0ull;
    if (clear && index >= 0) key = kDraft ? race_key(__fdiv_rn(best_w, best_e), index) : exact(index);
    for (unsigned close = __ballot_sync(0xffffffffu, !clear); close != 0; close &= close - 1) {
      for (int i = first + warp * 32 + __ffs(close) - 1 + lane * kVerifyThreads; i < end; i += 32 * kVerifyThreads)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int v = i * N - lead + j;
          const unsigned long long mine = v >= 0 && v < V ? exact(v) : 0ull;
          key = mine > key ? mine : key;
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, off);
      key = o > key ? o : key;
    }
    if (lane == 0) s_warp[warp] = key;
    __syncthreads();
    if (warp == 0) {
      key = lane < kVerifyThreads / 32 ? s_warp[lane] : 0ull;
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, key, off);
        key = o > key ? o : key;
      }
      if (lane < ranks) store_remote(&s_best[attempt][rank], lane, key);
    }
    cluster_sync();
    key = 0ull;
    for (unsigned r = 0; r < ranks; ++r) key = s_best[attempt][r] > key ? s_best[attempt][r] : key;
    // Nothing left after the refusals: once more, from p itself.  (The same
    // decision in every CTA: all see the same keys.)
    if (key == 0ull && residual) continue;
    if (rank == 0 && threadIdx.x == 0) {
      const int next = key != 0ull ? static_cast<int>(0xffffffffu - static_cast<unsigned>(key)) : 0;
      if (a.tokens_64)
        static_cast<long long*>(a.next)[b] = next;
      else
        static_cast<int*>(a.next)[b] = next;
    }
    return;
  }
}

constexpr int kCommitThreads = 256;
constexpr int kCommitHeads = 4;

// CTA (b and layer, four heads): a thread has one 16-byte chunk of a row and
// copies it for K and V of all its heads, eight loads in flight.  One layer's
// call is bound by the latency of path, row and store (2.1 us), every layer's
// by memory: 27.2 us (5.1 TB/s, 79 % of a copy, in pieces of 256 bytes) for 138
// MB; 27.5 us with two heads a thread, 28.1 with eight.
__global__ void __launch_bounds__(kCommitThreads) commit_kernel(const __grid_constant__ CommitArgs a, int chunks, int rows) {
  pdl_wait_prerequisites();
  const int64_t b = blockIdx.x % a.B, layer = blockIdx.x / a.B;
  const int h0 = blockIdx.y * kCommitHeads, heads = min(kCommitHeads, static_cast<int>(a.H) - h0);
  const int path_len = a.path_lens[b], kv_len = a.kv_lens[b];
  const int n = min(max(path_len, 0), static_cast<int>(a.T));
  const int start = min(max(kv_len, 0), static_cast<int>(a.L));
  const int fit = min(n, static_cast<int>(a.L) - start);
  if (h0 == 0 && layer == 0 && threadIdx.x == 0) {
    a.new_lens[b] = start + fit;
    if (fit < n) atomicCAS(a.status, kOk, kErrTooLarge);
    if (n != path_len || start != kv_len) atomicCAS(a.status, kOk, kErrInvalidArgument);
  }
  const int lane_row = threadIdx.x / chunks, c = threadIdx.x % chunks * 8;
  if (lane_row >= rows) return;
  const int64_t* st = a.strides;  // k, v, k_tree, v_tree x (layer, batch, head, row)
  uint16_t* k = static_cast<uint16_t*>(a.k) + layer * st[0] + b * st[1] + h0 * st[2] + c;
  uint16_t* v = static_cast<uint16_t*>(a.v) + layer * st[4] + b * st[5] + h0 * st[6] + c;
  const uint16_t* kt = static_cast<const uint16_t*>(a.k_tree) + layer * st[8] + b * st[9] + h0 * st[10] + c;
  const uint16_t* vt = static_cast<const uint16_t*>(a.v_tree) + layer * st[12] + b * st[13] + h0 * st[14] + c;
  for (int i = lane_row; i < fit; i += rows) {
    const int node = a.path[b * a.T + i];
    if (node < 0 || node >= a.T) {
      atomicCAS(a.status, kOk, kErrInvalidArgument);
      continue;
    }
    uint4 x[kCommitHeads], y[kCommitHeads];
#pragma unroll
    for (int h = 0; h < kCommitHeads; ++h)
      if (h < heads) {
        x[h] = *reinterpret_cast<const uint4*>(kt + h * st[10] + node * st[11]);
        y[h] = *reinterpret_cast<const uint4*>(vt + h * st[14] + node * st[15]);
      }
#pragma unroll
    for (int h = 0; h < kCommitHeads; ++h)
      if (h < heads) {
        *reinterpret_cast<uint4*>(k + h * st[2] + (start + i) * st[3]) = x[h];
        *reinterpret_cast<uint4*>(v + h * st[6] + (start + i) * st[7]) = y[h];
      }
  }
}

template <int kType, int kRead, bool kDraft>
int launch_verify_t(const VerifyArgs& a, int cluster) {
  static_assert(kRead != kCutByFour || (kType != kProbF32 && !kDraft), "16-bit probabilities alone are cut");
  return launch_pdl(verify_kernel<kType, kRead, kDraft>, dim3(static_cast<unsigned>(a.B * cluster)), dim3(kVerifyThreads),
                    0, a.stream, cluster, a);
}

template <int kType>
int launch_verify_n(const VerifyArgs& a, int cluster, bool wide) {
  if (a.draft != nullptr)
    return wide ? launch_verify_t<kType, kByFour, true>(a, cluster) : launch_verify_t<kType, kByOne, true>(a, cluster);
  return wide ? launch_verify_t<kType, kByFour, false>(a, cluster)
              : launch_verify_t<kType, kType == kProbF32 ? kByOne : kCutByFour, false>(a, cluster);
}

}  // namespace

int launch_verify(const VerifyArgs& a) {
  // CTAs of a sequence: about one an SM (each walks the tree again), as long as
  // each has a thread's worth of loads.  Two an SM: the same for 32 trees, 22.8
  // instead of 19.0 us for 128 chains; four: 30.9 us.
  int cluster = 1;
  while (cluster < kVerifyMaxCluster && a.B * cluster < 148 && a.V >= kVerifyThreads * 2 * cluster) cluster *= 2;
  // Whether every row starts on a word of four.
  const uintptr_t bytes = a.type == kProbF32 ? 16 : 8;
  bool wide = a.V % 4 == 0 && a.target_stride[0] % 4 == 0 && a.target_stride[1] % 4 == 0 &&
              reinterpret_cast<uintptr_t>(a.target) % bytes == 0 && reinterpret_cast<uintptr_t>(a.noise) % 16 == 0;
  if (a.draft != nullptr)
    wide = wide && a.draft_stride[0] % 4 == 0 && a.draft_stride[1] % 4 == 0 &&
           reinterpret_cast<uintptr_t>(a.draft) % bytes == 0;
  switch (a.type) {
    case kProbF32: return launch_verify_n<kProbF32>(a, cluster, wide);
    case kProbBf16: return launch_verify_n<kProbBf16>(a, cluster, wide);
    default: return launch_verify_n<kProbF16>(a, cluster, wide);
  }
}

int launch_commit(const CommitArgs& a) {
  // No more threads than a tree's rows have chunks: a CTA is short, and smaller
  // ones are more an SM (trees of 8, every layer: 8.1 us instead of 10.2).
  const int chunks = static_cast<int>(a.D / 8);
  const int threads = static_cast<int>(std::min<int64_t>(kCommitThreads, (a.T * chunks + 31) / 32 * 32));
  const dim3 grid(static_cast<unsigned>(a.layers * a.B), static_cast<unsigned>((a.H + kCommitHeads - 1) / kCommitHeads));
  return launch_pdl(commit_kernel, grid, dim3(threads), 0, a.stream, 1, a, chunks, threads / chunks);
}

}  // namespace tk
