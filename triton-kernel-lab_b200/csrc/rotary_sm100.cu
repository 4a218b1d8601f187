// Rotary positions on queries and keys at given positions: interleaved or
// half layout, all or part of the head, forward and backward.
//
// For a row x at position p, r rotated columns and the angle tables cos, sin
// (positions, r/2) in fp32, pair i of the row is columns (i, i + r/2) in the
// half layout and (2i, 2i + 1) in the interleaved one, and in fp32, rounded
// once,
//   y1 = x1 cos[p][i] - x2 sin[p][i]
//   y2 = x2 cos[p][i] + x1 sin[p][i];
// columns from r on are copied.  The backward is the transpose: the sine's
// sign changes (`transpose`).  Long-context scalings (and their factor on the
// tables) live in the tables, so they need nothing here.
//
// Bound by memory: 4 bytes an element and three operations.  A row's angles
// are fp32 and serve every head, so a thread keeps those of its columns and
// goes over the heads with them: loading them per head would be twice the
// data.  A thread has two chunks of W columns: the two sides of its pairs in
// the half layout, else two half a row apart, so that neighbouring threads
// have neighbouring chunks (with neighbouring chunks in one thread a request
// used half of each 32-byte sector it touched).
//
// Measured, forward and backward: 113.5 us (6.05 TB/s, 94 % of a copy) for
// (1, 16384) tokens of 32 + 8 heads of 128, all rotated; 29.6 us (5.1 TB/s)
// for (3, 2047) tokens of 16 + 16 heads of 96, 24 rotated in neighbouring
// pairs (36.8 us with neighbouring chunks and 256 threads a CTA).  These are the
// device's times: called through autograd the second takes 67 to 69 us, which
// the host's side of the backward pass does.  Forward for 32 x 24 tokens of 32 +
// 8 heads of 128: 4.0 us, of which 3 us are the latency of one call.
#include <algorithm>

#include "attn_launch.h"
#include "pdl_launch.h"
#include "rope_sm100.cuh"

namespace tk {
namespace {

// W 16-bit elements as they are loaded and stored.
template <int W>
struct alignas(2 * W) Chunk {
  uint16_t e[W];
};

template <bool kBf16>
__device__ __forceinline__ float from16(uint16_t h) {
  if constexpr (kBf16) {
    return __uint_as_float(static_cast<uint32_t>(h) << 16);
  } else {
    return __half2float(__ushort_as_half(h));
  }
}

template <bool kBf16>
__device__ __forceinline__ uint16_t to16(float x) {
  if constexpr (kBf16) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(x));
  } else {
    return __half_as_ushort(__float2half_rn(x));
  }
}

// Small CTAs even out the end of a short call: 29.6 us for the (3, 2047)
// case, 32.4 us with 256 threads.
constexpr int kRotaryThreads = 128;
// A thread with at most this many heads has four heads of loads in flight,
// one with more has two: fewer registers, so more threads an SM, whose loads
// overlap in place of a thread's own.  With 40 heads a thread 113.5 us with
// two and 116.7 with four; with 4 heads a thread 34.4 and 31.0 us (3 x 2047
// tokens, half layout), 4.5 and 4.3 us (32 x 24 tokens).
constexpr int kFewHeads = 8;

template <bool kBf16, bool kInterleaved, int W, int kFlight>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryArgs a, int units, int heads_per_block) {
  using C = Chunk<W>;
  pdl_wait_prerequisites();
  const int chunks = static_cast<int>(a.D) / W, turned = static_cast<int>(a.rotary_dim) / W;
  const long long u = static_cast<long long>(blockIdx.x) * kRotaryThreads + threadIdx.x;
  const long long tok = u / units;  // (b, s)
  if (tok >= a.B * a.S) return;
  const int unit = static_cast<int>(u - tok * units);
  const long long b = tok / a.S, s = tok - b * a.S;
  // The thread's chunks; the second may not exist (an odd number of copied ones).
  int c1, c2;
  bool turn1, turn2;
  if constexpr (kInterleaved) {
    c1 = unit;
    c2 = unit + (chunks + 1) / 2;
    turn1 = c1 < turned;
    turn2 = c2 < turned;
  } else {
    const int pairs = turned / 2;
    turn1 = turn2 = unit < pairs;
    c1 = turn1 ? unit : turned + (unit - pairs);
    c2 = turn1 ? unit + pairs : c1 + (chunks - turned + 1) / 2;
  }
  const bool has2 = c2 < chunks;
  // Angles of this thread's pairs: W of them (half: the chunks' columns;
  // interleaved: W / 2 a chunk).
  float cs[W], sn[W];
#pragma unroll
  for (int i = 0; i < W; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
  if (turn1) {
    long long pos = s;
    if (a.positions != nullptr)
      pos = a.positions_64 ? static_cast<const long long*>(a.positions)[tok] : static_cast<const int*>(a.positions)[tok];
    if (pos < 0 || pos >= a.table_rows) {
      // No table row: report it, leave the row as it is.
      atomicCAS(a.status, kOk, kErrInvalidArgument);
      turn1 = turn2 = false;
    } else {
      const long long t = pos * (a.rotary_dim / 2) + (kInterleaved ? c1 * (W / 2) : c1 * W);
      if constexpr (W == 8) {  // rows of a multiple of 4 angles: t is one too
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          if (kInterleaved && i > 0 && !turn2) break;
          const long long o = t + (kInterleaved && i > 0 ? (c2 - c1) * (W / 2) : i);
          const float4 c = *reinterpret_cast<const float4*>(a.cos + o);
          const float4 v = *reinterpret_cast<const float4*>(a.sin + o);
          cs[i] = c.x, cs[i + 1] = c.y, cs[i + 2] = c.z, cs[i + 3] = c.w;
          sn[i] = v.x, sn[i + 1] = v.y, sn[i + 2] = v.z, sn[i + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if (kInterleaved && i >= W / 2 && !turn2) break;
          const long long o = t + (kInterleaved && i >= W / 2 ? (c2 - c1 - 1) * (W / 2) + i : i);
          cs[i] = a.cos[o];
          sn[i] = a.sin[o];
        }
      }
#pragma unroll
      for (int i = 0; i < W; ++i) sn[i] = a.transpose ? -sn[i] : sn[i];
    }
  }
  const int heads = static_cast<int>(a.Hq + a.Hkv);
  const int h_end = min(heads, static_cast<int>(blockIdx.y + 1) * heads_per_block);
  for (int h0 = blockIdx.y * heads_per_block; h0 < h_end; h0 += kFlight) {
    C x1[kFlight], x2[kFlight];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int h = h0 + i;
      if (h >= h_end) break;
      const bool is_q = h < a.Hq;
      const int64_t* st = is_q ? a.q_stride : a.k_stride;
      const uint16_t* x = static_cast<const uint16_t*>(is_q ? a.q : a.k) + b * st[0] +
                          (is_q ? h : h - a.Hq) * st[1] + s * st[2];
      x1[i] = *reinterpret_cast<const C*>(x + c1 * W);
      if (has2) x2[i] = *reinterpret_cast<const C*>(x + c2 * W);
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int h = h0 + i;
      if (h >= h_end) break;
      C y1 = x1[i], y2 = x2[i];
      if constexpr (kInterleaved) {
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          const float p = from16<kBf16>(x1[i].e[e]), q = from16<kBf16>(x1[i].e[e + 1]);
          const float v = from16<kBf16>(x2[i].e[e]), w = from16<kBf16>(x2[i].e[e + 1]);
          const int k = e / 2, l = W / 2 + e / 2;
          if (turn1) {
            y1.e[e] = to16<kBf16>(p * cs[k] - q * sn[k]);
            y1.e[e + 1] = to16<kBf16>(q * cs[k] + p * sn[k]);
          }
          if (turn2) {
            y2.e[e] = to16<kBf16>(v * cs[l] - w * sn[l]);
            y2.e[e + 1] = to16<kBf16>(w * cs[l] + v * sn[l]);
          }
        }
      } else if (turn1) {
#pragma unroll
        for (int e = 0; e < W; ++e) {
          const float p = from16<kBf16>(x1[i].e[e]), q = from16<kBf16>(x2[i].e[e]);
          y1.e[e] = to16<kBf16>(p * cs[e] - q * sn[e]);
          y2.e[e] = to16<kBf16>(q * cs[e] + p * sn[e]);
        }
      }
      const bool is_q = h < a.Hq;
      uint16_t* y = static_cast<uint16_t*>(is_q ? a.q_out : a.k_out) +
                    ((is_q ? b * a.Hq + h : b * a.Hkv + (h - a.Hq)) * a.S + s) * a.D;
      *reinterpret_cast<C*>(y + c1 * W) = y1;
      if (has2) *reinterpret_cast<C*>(y + c2 * W) = y2;
    }
  }
}

template <bool kBf16, bool kInterleaved, int W>
int launch_rotary_w(const RotaryArgs& a) {
  const int64_t chunks = a.D / W, turned = a.rotary_dim / W;
  const int64_t units = kInterleaved ? (chunks + 1) / 2 : turned / 2 + (chunks - turned + 1) / 2;
  const int64_t heads = a.Hq + a.Hkv;
  const int64_t blocks = (a.B * a.S * units + kRotaryThreads - 1) / kRotaryThreads;
  if (blocks > INT32_MAX) return kErrTooLarge;
  // All heads in one thread where that fills the device (16 CTAs an SM), else
  // as few as it takes: short calls are bound by latency.
  const int64_t want = std::max<int64_t>(1, std::min<int64_t>((heads + 3) / 4, 148 * 16 / blocks));
  const int64_t per = (heads + want - 1) / want;
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>((heads + per - 1) / per));
  const bool few = per <= kFewHeads;
  return launch_pdl(few ? rotary_kernel<kBf16, kInterleaved, W, 4> : rotary_kernel<kBf16, kInterleaved, W, 2>, grid,
                    dim3(kRotaryThreads), 0, a.stream, 1, a, static_cast<int>(units), static_cast<int>(per));
}

// The widest chunk that rotated columns divide into: 16 bytes for the usual
// widths, down to one column for pairs like (i, i + 3).
template <bool kBf16>
int launch_rotary_b(const RotaryArgs& a) {
  if (a.interleaved) {
    if (a.rotary_dim % 8 == 0) return launch_rotary_w<kBf16, true, 8>(a);
    if (a.rotary_dim % 4 == 0) return launch_rotary_w<kBf16, true, 4>(a);
    return launch_rotary_w<kBf16, true, 2>(a);
  }
  if (a.rotary_dim % 16 == 0) return launch_rotary_w<kBf16, false, 8>(a);
  if (a.rotary_dim % 8 == 0) return launch_rotary_w<kBf16, false, 4>(a);
  if (a.rotary_dim % 4 == 0) return launch_rotary_w<kBf16, false, 2>(a);
  return launch_rotary_w<kBf16, false, 1>(a);
}

}  // namespace

int launch_rotary(const RotaryArgs& a) { return a.bf16 ? launch_rotary_b<true>(a) : launch_rotary_b<false>(a); }

}  // namespace tk
