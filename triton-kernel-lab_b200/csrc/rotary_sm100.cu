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
#include "attn_launch.h"
#include "rope_sm100.cuh"

namespace tk {
namespace {

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

// One thread per column pair or copied column of one row.
template <bool kBf16>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  const int half = a.rotary_dim / 2;
  const int units = half + a.D - a.rotary_dim;  // pairs, then copied columns
  const long long n = static_cast<long long>(a.B) * (a.Hq + a.Hkv) * a.S * units;
  const long long stride = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long u = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; u < n; u += stride) {
    const int unit = static_cast<int>(u % units);
    long long row = u / units;
    const int s = static_cast<int>(row % a.S);
    row /= a.S;
    int h = static_cast<int>(row % (a.Hq + a.Hkv));
    const long long b = row / (a.Hq + a.Hkv);
    const bool is_q = h < a.Hq;
    if (!is_q) h -= static_cast<int>(a.Hq);
    const int64_t* st = is_q ? a.q_stride : a.k_stride;
    const uint16_t* x = static_cast<const uint16_t*>(is_q ? a.q : a.k) + b * st[0] + h * st[1] + s * st[2];
    uint16_t* y = static_cast<uint16_t*>(is_q ? a.q_out : a.k_out) + ((b * (is_q ? a.Hq : a.Hkv) + h) * a.S + s) * a.D;
    if (unit >= half) {
      const int c = a.rotary_dim + unit - half;
      y[c] = x[c];
      continue;
    }
    long long pos = s;
    if (a.positions != nullptr)
      pos = a.positions_64 ? static_cast<const long long*>(a.positions)[b * a.S + s]
                           : static_cast<const int*>(a.positions)[b * a.S + s];
    const int c1 = a.interleaved ? 2 * unit : unit;
    const int c2 = a.interleaved ? c1 + 1 : unit + half;
    if (pos < 0 || pos >= a.table_rows) {
      // No table row: report it, leave the row as it is.
      atomicCAS(a.status, kOk, kErrInvalidArgument);
      y[c1] = x[c1];
      y[c2] = x[c2];
      continue;
    }
    const float cs = a.cos[pos * half + unit];
    const float sn = a.transpose ? -a.sin[pos * half + unit] : a.sin[pos * half + unit];
    const float x1 = from16<kBf16>(x[c1]), x2 = from16<kBf16>(x[c2]);
    y[c1] = to16<kBf16>(x1 * cs - x2 * sn);
    y[c2] = to16<kBf16>(x2 * cs + x1 * sn);
  }
}

}  // namespace

int launch_rotary(const RotaryArgs& a) {
  const long long n = static_cast<long long>(a.B) * (a.Hq + a.Hkv) * a.S * (a.D - a.rotary_dim / 2);
  const long long blocks = (n + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < 148LL * 64 ? blocks : 148LL * 64);
  if (a.bf16)
    rotary_kernel<true><<<grid, 256, 0, a.stream>>>(a);
  else
    rotary_kernel<false><<<grid, 256, 0, a.stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace tk
