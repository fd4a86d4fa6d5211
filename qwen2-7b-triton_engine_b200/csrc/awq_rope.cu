// awq_rope.cu -- rotary positions with several axes, out of place or in place.
//
// angle[t, i] = positions[axis(i), t] * inv_freq[i]; the pair (x_i, x_{i + half}) of every
// head of token t is turned by it (the rotate-half pairing of the reference's
// kernels/rope.py:7-66), in fp32, one fp16 rounding; channels from 2 half up pass through.
// The angle is reduced in fp64 in units of whole turns, so positions of a million and more
// lose nothing: |pos * inv_freq / 2 pi| keeps 53 bits before the whole turns go, and the
// fp32 remainder is exact to 2^-25 of a turn.
//
// Bound: HBM.  One block for four neighbouring tokens: it makes their sines and cosines once
// for all heads, then every thread turns pairs in 16-byte pieces, with its first loads under way
// while the angles are made.  8191 tokens, 28 + 4 heads of 128 channels: 26 us on B200 (134 MB,
// 5.2 TB/s, 79 % of a copy's rate); with the loads behind the angles 31 us.  Eight tokens: 4.3
// us, a launch and the reduction of the angles.  Channels that pass through, and all channels
// where half is no multiple of 8, go two bytes at a time: the same tokens with 80 of 128
// channels rotated take 66 us (62 in place), 32 heads of 64 with 40 rotated 35 us, against 20.5
// and 10.2 for the bytes.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "awq_common.cuh"
#include "awq_internal.h"

namespace awq {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 256;
constexpr int kTokens = 4;             // of a block

__device__ __forceinline__ int axis_of(const RopeCall& c, int i) {
  if (c.interleaved) {
    const int a = i % c.axes;
    return i / c.axes < c.sections[a] ? a : 0;
  }
  int a = 0, end = c.sections[0];
  while (i >= end && a + 1 < c.axes) end += c.sections[++a];
  return a;
}

// Where piece idx of a head lies: 8 pairs of channels (VEC) or one, from channel i of head h.
struct Piece {
  const __half* x;
  __half* y;
  int64_t xs, ys;      // token strides
  int i;
};
template <bool VEC>
__device__ __forceinline__ Piece piece(const RopeCall& c, int idx, int per) {
  Piece p;
  const int h = idx / per;
  p.i = (idx - h * per) * (VEC ? 8 : 1);
  const bool isq = h < c.q_heads;
  const int hk = h - c.q_heads;
  p.x = isq ? static_cast<const __half*>(c.q) + h * c.q_hs : static_cast<const __half*>(c.k) + hk * c.k_hs;
  p.y = isq ? static_cast<__half*>(c.out_q) + h * c.oq_hs : static_cast<__half*>(c.out_k) + hk * c.ok_hs;
  p.xs = isq ? c.q_ts : c.k_ts, p.ys = isq ? c.oq_ts : c.ok_ts;
  return p;
}

// A block turns kTokens neighbouring tokens.  The loads of a thread's first piece are under way
// while the block makes the tokens' sines and cosines.
template <bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeCall c) {
  __shared__ __align__(16) float s_cos[kTokens][kRopeMaxHalf], s_sin[kTokens][kRopeMaxHalf];
  const int heads = c.q_heads + c.k_heads, rest = c.dim - 2 * c.half;
  const int per = VEC ? c.half / 8 : c.half, pieces = heads * per;
  const int64_t t0 = (int64_t)blockIdx.x * kTokens;
  const int tokens = (int)(c.T - t0 < kTokens ? c.T - t0 : kTokens);
  Piece p = {};
  uint4 va[kTokens], vb[kTokens];
  auto fetch = [&](int idx) {
    p = piece<VEC>(c, idx, per);
    if constexpr (VEC) {
#pragma unroll
      for (int k = 0; k < kTokens; ++k)
        if (k < tokens) {
          const __half* x = p.x + (t0 + k) * p.xs + p.i;
          va[k] = *reinterpret_cast<const uint4*>(x);
          vb[k] = *reinterpret_cast<const uint4*>(x + c.half);
        }
    }
  };
  if ((int)threadIdx.x < pieces) fetch(threadIdx.x);
  for (int n = threadIdx.x; n < tokens * c.half; n += kRopeThreads) {
    const int k = n / c.half, i = n - k * c.half;
    const int64_t at = axis_of(c, i) * c.pos_as + t0 + k;
    const double pos = c.pos_is_64 ? (double)static_cast<const int64_t*>(c.positions)[at]
                                   : (double)static_cast<const int32_t*>(c.positions)[at];
    const double turns = pos * ((double)c.inv_freq[i] * 0.15915494309189533577);
    sincospif((float)(2.0 * (turns - rint(turns))), &s_sin[k][i], &s_cos[k][i]);
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < pieces; idx += kRopeThreads) {
    if (idx != (int)threadIdx.x) fetch(idx);
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
      if (k >= tokens) break;
      const float *cs = s_cos[k] + p.i, *sn = s_sin[k] + p.i;
      __half* y = p.y + (t0 + k) * p.ys + p.i;
      if constexpr (VEC) {
        const uint32_t a[4] = {va[k].x, va[k].y, va[k].z, va[k].w}, b[4] = {vb[k].x, vb[k].y, vb[k].z, vb[k].w};
        uint32_t ya[4], yb[4];
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const float4 c4 = *reinterpret_cast<const float4*>(cs + 2 * j);
          const float4 s4 = *reinterpret_cast<const float4*>(sn + 2 * j);
          const float2 a0 = __half22float2(u32_as_h2(a[j])), a1 = __half22float2(u32_as_h2(a[j + 1]));
          const float2 b0 = __half22float2(u32_as_h2(b[j])), b1 = __half22float2(u32_as_h2(b[j + 1]));
          ya[j] = h2_as_u32(__floats2half2_rn(a0.x * c4.x - b0.x * s4.x, a0.y * c4.y - b0.y * s4.y));
          yb[j] = h2_as_u32(__floats2half2_rn(b0.x * c4.x + a0.x * s4.x, b0.y * c4.y + a0.y * s4.y));
          ya[j + 1] = h2_as_u32(__floats2half2_rn(a1.x * c4.z - b1.x * s4.z, a1.y * c4.w - b1.y * s4.w));
          yb[j + 1] = h2_as_u32(__floats2half2_rn(b1.x * c4.z + a1.x * s4.z, b1.y * c4.w + a1.y * s4.w));
        }
        *reinterpret_cast<uint4*>(y) = make_uint4(ya[0], ya[1], ya[2], ya[3]);
        *reinterpret_cast<uint4*>(y + c.half) = make_uint4(yb[0], yb[1], yb[2], yb[3]);
      } else {
        const __half* x = p.x + (t0 + k) * p.xs + p.i;
        const float fa = __half2float(x[0]), fb = __half2float(x[c.half]);
        y[0] = __float2half_rn(fa * cs[0] - fb * sn[0]);
        y[c.half] = __float2half_rn(fb * cs[0] + fa * sn[0]);
      }
    }
  }
  if (rest > 0)
    for (int idx = threadIdx.x; idx < tokens * heads * rest; idx += kRopeThreads) {
      const int k = idx / (heads * rest), at = idx - k * heads * rest, h = at / rest;
      const int64_t t = t0 + k, i = 2 * c.half + at - h * rest;
      if (h < c.q_heads)
        static_cast<__half*>(c.out_q)[t * c.oq_ts + h * c.oq_hs + i] =
            static_cast<const __half*>(c.q)[t * c.q_ts + h * c.q_hs + i];
      else
        static_cast<__half*>(c.out_k)[t * c.ok_ts + (h - c.q_heads) * c.ok_hs + i] =
            static_cast<const __half*>(c.k)[t * c.k_ts + (h - c.q_heads) * c.k_hs + i];
    }
}

bool vec16(const void* p, int64_t ts, int64_t hs) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
}

}  // namespace

cudaError_t launch_rope(const RopeCall& c, int num_sms, cudaStream_t stream) {
  const bool q_ok = c.q_heads == 0 || (vec16(c.q, c.q_ts, c.q_hs) && vec16(c.out_q, c.oq_ts, c.oq_hs));
  const bool k_ok = c.k_heads == 0 || (vec16(c.k, c.k_ts, c.k_hs) && vec16(c.out_k, c.ok_ts, c.ok_hs));
  const unsigned blocks = (unsigned)((c.T + kTokens - 1) / kTokens);
  if (c.half % 8 == 0 && q_ok && k_ok)
    rope_kernel<true><<<blocks, kRopeThreads, 0, stream>>>(c);
  else
    rope_kernel<false><<<blocks, kRopeThreads, 0, stream>>>(c);
  return cudaGetLastError();
}

}  // namespace awq
