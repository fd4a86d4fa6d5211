// awq_rope.cu -- rotary positions with several axes, out of place or in place.
//
// angle[t, i] = positions[axis(i), t] * inv_freq[i]; the pair (x_i, x_{i + half}) of every
// head of token t is turned by it (the rotate-half pairing of the reference's
// kernels/rope.py:7-66), in fp32, one fp16 rounding; channels from 2 half up pass through.
// The angle is reduced in fp64 in units of whole turns, so positions of a million and more
// lose nothing: |pos * inv_freq / 2 pi| keeps 53 bits before the whole turns go, and the
// fp32 remainder is exact to 2^-25 of a turn.
//
// Bound: HBM.  One block per token: `half` threads make the token's sines and cosines once
// for all heads, then every thread turns pairs in 16-byte pieces.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "awq_common.cuh"
#include "awq_internal.h"

namespace awq {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxHalf = 256;

__device__ __forceinline__ int axis_of(const RopeCall& c, int i) {
  if (c.interleaved) {
    const int a = i % c.axes;
    return i / c.axes < c.sections[a] ? a : 0;
  }
  int a = 0, end = c.sections[0];
  while (i >= end && a + 1 < c.axes) end += c.sections[++a];
  return a;
}

template <bool VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeCall c) {
  __shared__ float s_cos[kRopeMaxHalf], s_sin[kRopeMaxHalf];
  const int heads = c.q_heads + c.k_heads;
  for (int64_t t = blockIdx.x; t < c.T; t += gridDim.x) {
    for (int i = threadIdx.x; i < c.half; i += kRopeThreads) {
      const int64_t at = axis_of(c, i) * c.pos_as + t;
      const double pos = c.pos_is_64 ? (double)static_cast<const int64_t*>(c.positions)[at]
                                     : (double)static_cast<const int32_t*>(c.positions)[at];
      const double turns = pos * ((double)c.inv_freq[i] * 0.15915494309189533577);
      sincospif((float)(2.0 * (turns - rint(turns))), &s_sin[i], &s_cos[i]);
    }
    __syncthreads();
    const int per = VEC ? c.half / 8 : c.half;
    for (int idx = threadIdx.x; idx < heads * per; idx += kRopeThreads) {
      const int h = idx / per, i = (idx - h * per) * (VEC ? 8 : 1);
      const bool isq = h < c.q_heads;
      const __half* x = isq ? static_cast<const __half*>(c.q) + t * c.q_ts + h * c.q_hs
                            : static_cast<const __half*>(c.k) + t * c.k_ts + (h - c.q_heads) * c.k_hs;
      __half* y = isq ? static_cast<__half*>(c.out_q) + t * c.oq_ts + h * c.oq_hs
                      : static_cast<__half*>(c.out_k) + t * c.ok_ts + (h - c.q_heads) * c.ok_hs;
      if constexpr (VEC) {
        const uint4 va = *reinterpret_cast<const uint4*>(x + i);
        const uint4 vb = *reinterpret_cast<const uint4*>(x + i + c.half);
        uint4 oa, ob;
        const __half2* a = reinterpret_cast<const __half2*>(&va);
        const __half2* b = reinterpret_cast<const __half2*>(&vb);
        __half2* ya = reinterpret_cast<__half2*>(&oa);
        __half2* yb = reinterpret_cast<__half2*>(&ob);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 fa = __half22float2(a[j]), fb = __half22float2(b[j]);
          const float c0 = s_cos[i + 2 * j], c1 = s_cos[i + 2 * j + 1];
          const float s0 = s_sin[i + 2 * j], s1 = s_sin[i + 2 * j + 1];
          ya[j] = __floats2half2_rn(fa.x * c0 - fb.x * s0, fa.y * c1 - fb.y * s1);
          yb[j] = __floats2half2_rn(fb.x * c0 + fa.x * s0, fb.y * c1 + fa.y * s1);
        }
        *reinterpret_cast<uint4*>(y + i) = oa;
        *reinterpret_cast<uint4*>(y + i + c.half) = ob;
      } else {
        const float fa = __half2float(x[i]), fb = __half2float(x[i + c.half]);
        y[i] = __float2half_rn(fa * s_cos[i] - fb * s_sin[i]);
        y[i + c.half] = __float2half_rn(fb * s_cos[i] + fa * s_sin[i]);
      }
    }
    const int rest = c.dim - 2 * c.half;
    for (int idx = threadIdx.x; idx < heads * rest; idx += kRopeThreads) {
      const int h = idx / rest, i = 2 * c.half + idx - h * rest;
      if (h < c.q_heads)
        static_cast<__half*>(c.out_q)[t * c.oq_ts + h * c.oq_hs + i] =
            static_cast<const __half*>(c.q)[t * c.q_ts + h * c.q_hs + i];
      else
        static_cast<__half*>(c.out_k)[t * c.ok_ts + (h - c.q_heads) * c.ok_hs + i] =
            static_cast<const __half*>(c.k)[t * c.k_ts + (h - c.q_heads) * c.k_hs + i];
    }
    __syncthreads();
  }
}

bool vec16(const void* p, int64_t ts, int64_t hs) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
}

}  // namespace

cudaError_t launch_rope(const RopeCall& c, int num_sms, cudaStream_t stream) {
  const bool q_ok = c.q_heads == 0 || (vec16(c.q, c.q_ts, c.q_hs) && vec16(c.out_q, c.oq_ts, c.oq_hs));
  const bool k_ok = c.k_heads == 0 || (vec16(c.k, c.k_ts, c.k_hs) && vec16(c.out_k, c.ok_ts, c.ok_hs));
  const int64_t most = (int64_t)num_sms * 64;
  const unsigned blocks = (unsigned)(c.T < most ? c.T : most);
  if (c.half % 8 == 0 && q_ok && k_ok)
    rope_kernel<true><<<blocks, kRopeThreads, 0, stream>>>(c);
  else
    rope_kernel<false><<<blocks, kRopeThreads, 0, stream>>>(c);
  return cudaGetLastError();
}

}  // namespace awq
