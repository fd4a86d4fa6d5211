// awq_kv4_args.cuh -- kernel arguments shared by the two attention kernels over the 4-bit
// cache (awq_kv4_attn.cu, awq_kv4_prefill.cu).
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "awq_common.cuh"

namespace awq {
namespace kv4 {

constexpr int kPrefixEntries = 1024;     // prefix sums held in shared memory
constexpr int kDescInts = 8;             // per CTA: the item that starts there and goes on
// The softmax reference M lies this many powers of two below the largest p s seen when it was
// set (or below a bound on it, in a step whose value scales lie close together), and moves when
// one passes 2^15 of M: fp16 weights reach 2^15, half of fp16's limit, and lose bits from 2^-21
// and vanish from 2^-32 of the largest on only.
constexpr float kBelowTop = 7.0f, kMoveAt = 8.0f;   // a new reference 2^kMoveAt above M replaces it

struct AttnArgs {
  const uint8_t* cache;
  const __half* q;
  __half* out;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu_q;
  int64_t q_ts, q_hs, o_ts, o_hs, table_rs;
  int64_t num_pages;
  int64_t tokens;
  // each kernel's own, as the two may overlap:
  float* part;        // [ctas][2] slots of items that cross CTAs
  float* warp_part;   // [ctas][warps] slots of items that cross warps, not a warp's last
  int* desc;          // [ctas][kDescInts]
  int* status;
  float scale_log2;
  int R, width, page_shift, kv_heads, G;
  int min_rows;       // requests with this many query rows per kv head are the prefill kernel's
};

// Launch of a kernel that may start while the one before it in the stream still runs, and
// waits for it (grid_dependency_wait) where it needs its results.
template <class K>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream,
                              const AttnArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

// Requests of one entry of the prefix sums: 1 << shift.
__device__ __forceinline__ int prefix_shift(const AttnArgs& a) {
  int shift = 0;
  while ((a.R >> shift) + 1 > kPrefixEntries) ++shift;
  return shift;
}
// Prefix sums pre[] of the requests' units of work (units(r), below 2^31), and their total.
// All THREADS threads call it.
template <int THREADS, class F>
__device__ __forceinline__ int scan_units(const AttnArgs& a, int* pre, F units) {
  constexpr int WARPS = THREADS / 32;
  static_assert(kPrefixEntries <= 1 << 10, "entries below 2^21 units do not overflow");
  __shared__ int wsum[WARPS];
  __shared__ int s_total, s_high;                        // high: entries of 2^21 and more, / 2^16
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  const int shift = prefix_shift(a), entries = (a.R + (1 << shift) - 1) >> shift;
  if (tid == 0) s_total = s_high = 0;
  for (int e0 = 0; e0 < entries; e0 += THREADS) {
    const int e = e0 + tid;
    uint32_t v = 0;
    if (e < entries)
      for (int r = e << shift; r < min(a.R, (e + 1) << shift); ++r)
        v = min(v + (uint32_t)units(r), 0x7fffffffu);
    int inc = (int)v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int nb = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += nb;
    }
    if (lane == 31) wsum[warp] = inc;
    if (__syncthreads_or(v >= 1u << 21)) atomicAdd(&s_high, (int)(v >> 16));
    const int part = lane < WARPS ? wsum[lane] : 0;
    const int before = s_total + __reduce_add_sync(0xffffffffu, lane < warp ? part : 0);
    if (e < entries) pre[e] = before + inc - (int)v;
    const int all = __reduce_add_sync(0xffffffffu, part);
    __syncthreads();
    if (tid == 0) s_total += all;
    __syncthreads();
  }
  // a list of 2^31 or more (requests that claim the same query rows): nothing is computed
  if (s_high <= 32767 && s_total >= 0) return s_total;
  if (tid == 0) atomicOr(a.status, kDevErrShape);
  return 0;
}

}  // namespace kv4
}  // namespace awq
