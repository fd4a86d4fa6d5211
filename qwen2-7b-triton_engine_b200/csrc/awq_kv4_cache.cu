// awq_kv4_cache.cu -- the paged 4-bit key/value cache: quantize-and-append, read-back, and
// the page bookkeeping of a step (block tables and slot maps from request lengths).
//
// Quantization of a group of g channels x (fp16): m = min x, s = fp16((max x - m) / 15),
// c = clamp(rne((x - m) / s), 0, 15), c = 0 where s = 0; both roundings are of the exact
// quotient.  A group holding a NaN or an infinity gets s = m = NaN, so that its token reads
// back as NaN instead of as some finite value.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "awq_common.cuh"
#include "awq_internal.h"
#include "awq_kv4.cuh"

namespace awq {

namespace {

struct Kv4IoArgs {
  const __half* k;
  const __half* v;
  int64_t k_ts, k_hs, v_ts, v_hs;   // token and head strides of k and v, elements
  const int64_t* slots;
  uint8_t* cache;
  __half* out_k;                    // gather: [T, H, D] contiguous
  __half* out_v;
  int64_t T, capacity;              // tokens; num_pages * page_size
  int H, page;
  int* status;
};

// Round-to-nearest-even of the exact (x - m) / s, 0..15.  The fp32 quotient is within
// 2^-21 of the exact one here (three roundings of 2^-24 each, quotient below 2^5), so only
// results that close to a tie take the double division, which decides every tie: x - m is
// exact in double, and an fp16 / fp16-difference quotient that is not a tie lies further
// than 2^-46 from one.
__device__ __forceinline__ uint32_t quant1(float x, float m, float s, float inv) {
  const float t = (x - m) * inv;
  float r = rintf(t);
  if (fabsf(t - r) > 0.4999f) r = (float)rint(((double)x - (double)m) / (double)s);
  return (uint32_t)fminf(fmaxf(r, 0.f), 15.f);
}

// The four codes of a lane's channels (nibble p = channel p), its group's scale and
// minimum.  LG lanes of four channels form a group.
template <int LG>
__device__ __forceinline__ uint32_t quant_quad(const float (&x)[4], __half& sh, __half& mh) {
  float lo = fminf(fminf(x[0], x[1]), fminf(x[2], x[3]));
  float hi = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  // a sum of differences that is not zero marks a NaN or an infinity
  bool bad = !((x[0] - x[0]) + (x[1] - x[1]) + (x[2] - x[2]) + (x[3] - x[3]) == 0.f);
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, o);
  }
  lo += 0.f, hi += 0.f;                              // one zero: -0 is stored as +0
  sh = __double2half(((double)hi - (double)lo) / 15.0);
  mh = __float2half_rn(lo);                          // exact: lo is one of the inputs
  if (bad) sh = mh = __ushort_as_half(0x7FFF);
  const float s = __half2float(sh);
  if (!(s > 0.f)) return 0;
  const float inv = 1.0f / s;
  uint32_t c = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p) c |= quant1(x[p], lo, s, inv) << (4 * p);
  return c;
}

__device__ __forceinline__ void load_quad(const __half* p, bool vec, float (&x)[4]) {
  if (vec) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(u32_as_h2(u.x)), b = __half22float2(u32_as_h2(u.y));
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __half2float(p[i]);
  }
}

// D/4 lanes per (token, head); grid-stride over the T * H rows, whole warps at a time so
// that the shuffles always see 32 lanes.
template <int D, int GROUP>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const Kv4IoArgs a, const int vec_k, const int vec_v) {
  constexpr int L = D / 4, ROWS = 32 / L, NG = D / GROUP;
  const int lane = threadIdx.x & 31, c = lane % L;
  const int64_t rows = a.T * a.H;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32) * ROWS;
  for (int64_t r0 = ((int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * ROWS; r0 < rows;
       r0 += step) {
    const int64_t row = r0 + lane / L;
    const bool in = row < rows;
    const int64_t tok = in ? row / a.H : 0;
    const int h = in ? (int)(row - tok * a.H) : 0;
    const int64_t slot = in ? a.slots[tok] : -1;
    float kx[4] = {}, vx[4] = {};
    if (in) {
      load_quad(a.k + tok * a.k_ts + h * a.k_hs + 4 * c, vec_k, kx);
      load_quad(a.v + tok * a.v_ts + h * a.v_hs + 4 * c, vec_v, vx);
    }
    __half ks, km, vs, vm;
    const uint32_t kc = quant_quad<GROUP / 4>(kx, ks, km);
    const uint32_t vc = quant_quad<GROUP / 4>(vx, vs, vm);
    const uint32_t kn = __shfl_down_sync(0xffffffffu, kc, 1);
    if (slot < 0) continue;                          // padding: nothing is written
    if (slot >= a.capacity) {
      if (c == 0) atomicOr(a.status, kDevErrShape);
      continue;
    }
    const int64_t page = slot / a.page;
    const int at = (int)(slot - page * a.page), b = at & 15;
    uint8_t* blk = a.cache + ((page * a.H + h) * (a.page / 16) + at / 16) * kv4::block_bytes(D, GROUP);
    if ((c & 1) == 0)
      *reinterpret_cast<uint32_t*>(blk + b * (D / 2) + 4 * kv4::k_word(D, c / 2)) = kc | kn << 16;
    *reinterpret_cast<uint16_t*>(blk + kv4::off_v(D) + (b / 2) * D + 4 * kv4::v_word(D, c) + 2 * (b & 1)) =
        (uint16_t)vc;
    if (c % (GROUP / 4) == 0) {
      const int gi = c / (GROUP / 4);
      reinterpret_cast<__half2*>(blk + kv4::off_kp(D))[b * NG + gi] = __halves2half2(ks, km);
      reinterpret_cast<__half2*>(blk + kv4::off_vp(D, GROUP))[b * NG + gi] = __halves2half2(vs, vm);
    }
  }
}

// fp16(code * scale + minimum) of the slots' keys and values; a negative slot reads as 0.
template <int D, int GROUP>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const Kv4IoArgs a) {
  constexpr int L = D / 4, NG = D / GROUP;
  const int64_t total = a.T * a.H * L;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / L, tok = row / a.H;
    const int c = (int)(i - row * L), h = (int)(row - tok * a.H);
    const int64_t slot = a.slots[tok];
    uint2 ko = make_uint2(0, 0), vo = make_uint2(0, 0);
    if (slot >= a.capacity) {
      if (c == 0) atomicOr(a.status, kDevErrShape);
    } else if (slot >= 0) {
      const int64_t page = slot / a.page;
      const int at = (int)(slot - page * a.page), b = at & 15;
      const uint8_t* blk = a.cache + ((page * a.H + h) * (a.page / 16) + at / 16) * kv4::block_bytes(D, GROUP);
      const uint32_t kc = *reinterpret_cast<const uint16_t*>(
          blk + b * (D / 2) + 4 * kv4::k_word(D, c / 2) + 2 * (c & 1));
      const uint32_t vc = *reinterpret_cast<const uint16_t*>(
          blk + kv4::off_v(D) + (b / 2) * D + 4 * kv4::v_word(D, c) + 2 * (b & 1));
      const int gi = c / (GROUP / 4);
      const float2 kp = __half22float2(reinterpret_cast<const __half2*>(blk + kv4::off_kp(D))[b * NG + gi]);
      const float2 vp = __half22float2(reinterpret_cast<const __half2*>(blk + kv4::off_vp(D, GROUP))[b * NG + gi]);
      float kf[4], vf[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        kf[p] = fmaf((float)((kc >> (4 * p)) & 15u), kp.x, kp.y);
        vf[p] = fmaf((float)((vc >> (4 * p)) & 15u), vp.x, vp.y);
      }
      ko = make_uint2(h2_as_u32(__floats2half2_rn(kf[0], kf[1])), h2_as_u32(__floats2half2_rn(kf[2], kf[3])));
      vo = make_uint2(h2_as_u32(__floats2half2_rn(vf[0], vf[1])), h2_as_u32(__floats2half2_rn(vf[2], vf[3])));
    }
    *reinterpret_cast<uint2*>(a.out_k + row * D + 4 * c) = ko;
    *reinterpret_cast<uint2*>(a.out_v + row * D + 4 * c) = vo;
  }
}

// ---- page bookkeeping -------------------------------------------------------------------
// One cluster does the whole step.  Every CTA scans all rows for itself (pages released,
// pages needed, tokens: three prefix sums kept in shared memory) and then takes a share of
// the flat lists of released pages, new pages and tokens, finding an element's row by
// bisection.  The cluster barriers separate the three uses of the free stack: push the
// released pages, read the popped ones, clear them.
struct PagesArgs {
  int32_t* table;
  int64_t table_rs;             // row stride of the block table
  int32_t* held;
  int32_t* free_pages;
  int32_t* free_count;
  const int32_t* lens;
  const int32_t* fresh_tokens;
  const uint8_t* reset;         // or null
  int64_t* slots;
  int32_t* positions;
  int32_t* cu_q;
  int32_t* new_lens;
  int32_t* status;
  int64_t max_tokens;
  int R, width, capacity, page;
};
constexpr int kPagesThreads = 512;

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

// Largest r with pre[r] <= j (pre[0] = 0, ascending).
__device__ __forceinline__ int row_of(const int* pre, int R, int j) {
  int lo = 0, hi = R;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= j) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPagesThreads) kv4_pages_kernel(const PagesArgs a) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int sm[];                        // pre[3][R + 1]
  __shared__ long long wsum[3][kPagesThreads / 32];
  __shared__ long long carry[3];
  __shared__ int s_bad;
  int* pre_gone = sm;
  int* pre_need = sm + (a.R + 1);
  int* pre_tok = sm + 2 * (a.R + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  if (tid < 3) carry[tid] = 0;
  if (tid == 0) s_bad = 0;
  __syncthreads();
  const int count = *a.free_count;
  for (int base = 0; base < a.R; base += kPagesThreads) {
    const int r = base + tid;
    long long v[3] = {0, 0, 0};
    if (r < a.R) {
      const long long h = a.held[r], len = a.lens[r], n = a.fresh_tokens[r];
      const bool rs = a.reset && a.reset[r];
      const long long need = (len + n + a.page - 1) / a.page, kept = rs ? 0 : h;
      if (h < 0 || h > a.width || len < 0 || n < 0 || len + n > 0x7fffffffLL || need > a.width)
        s_bad = 1;
      v[0] = rs ? h : 0;
      v[1] = need > kept ? need - kept : 0;
      v[2] = n;
    }
    long long inc[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      inc[k] = warp_scan(v[k], lane);
      if (lane == 31) wsum[k][warp] = inc[k];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const long long w = lane < kPagesThreads / 32 ? wsum[k][lane] : 0;
        const long long i = warp_scan(w, lane), before = carry[k];
        __syncwarp();                                // every lane has read the carry
        if (lane < kPagesThreads / 32) wsum[k][lane] = before + i - w;
        if (lane == 31) carry[k] = before + i;
      }
    }
    __syncthreads();
    // a sum past 32 bits is refused below, before any prefix is used
    if (r < a.R) {
      pre_gone[r] = (int)(wsum[0][warp] + inc[0] - v[0]);
      pre_need[r] = (int)(wsum[1][warp] + inc[1] - v[1]);
      pre_tok[r] = (int)(wsum[2][warp] + inc[2] - v[2]);
    }
    __syncthreads();
  }
  const long long gone = carry[0], need = carry[1], tokens = carry[2];
  int status = 0;
  if (s_bad || count < 0 || count + gone > a.capacity || tokens > a.max_tokens) status = -1;
  else if (need > count + gone) status = (int)(need - count - gone);
  if (tid == 0) pre_gone[a.R] = (int)gone, pre_need[a.R] = (int)need, pre_tok[a.R] = (int)tokens;
  __syncthreads();
  const bool ok = status == 0;
  const int top = ok ? count + (int)gone : 0;        // stack height between push and pop
  const int gt = (int)cluster.block_rank() * kPagesThreads + tid;
  const int gn = (int)cluster.num_blocks() * kPagesThreads;
  if (ok)
    for (int j = gt; j < (int)gone; j += gn) {       // push: the first released page on top
      const int r = row_of(pre_gone, a.R, j);
      int32_t* e = a.table + r * a.table_rs + (j - pre_gone[r]);
      a.free_pages[top - 1 - j] = *e;
      *e = -1;
    }
  cluster.sync();
  if (ok)
    for (int j = gt; j < (int)need; j += gn) {       // pop into the rows' next columns
      const int r = row_of(pre_need, a.R, j);
      const int kept = (a.reset && a.reset[r]) ? 0 : a.held[r];
      a.table[r * a.table_rs + kept + (j - pre_need[r])] = __ldcg(a.free_pages + top - 1 - j);
    }
  for (int64_t t = gt; t < a.max_tokens; t += gn) {
    int64_t slot = -1;
    int pos = 0;
    if (ok && t < tokens) {
      const int r = row_of(pre_tok, a.R, (int)t);
      const int kept = (a.reset && a.reset[r]) ? 0 : a.held[r];
      pos = a.lens[r] + ((int)t - pre_tok[r]);
      const int col = pos / a.page;
      const int pg = col < kept ? a.table[r * a.table_rs + col]
                                : __ldcg(a.free_pages + top - 1 - (pre_need[r] + col - kept));
      slot = pg < 0 ? -1 : (int64_t)pg * a.page + (pos - col * a.page);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  for (int r = gt; r <= a.R; r += gn) {
    a.cu_q[r] = ok ? pre_tok[r] : 0;
    if (r < a.R) a.new_lens[r] = a.lens[r] + (ok ? a.fresh_tokens[r] : 0);
  }
  cluster.sync();                                    // every reader of held and the stack is done
  if (ok) {
    for (int r = gt; r < a.R; r += gn) {
      const int kept = (a.reset && a.reset[r]) ? 0 : a.held[r];
      a.held[r] = kept + (pre_need[r + 1] - pre_need[r]);
    }
    for (int j = gt; j < (int)need; j += gn) a.free_pages[top - 1 - j] = -1;
  }
  if (gt == 0) {
    if (ok) *a.free_count = top - (int)need;
    *a.status = status;
  }
}

template <class F>
cudaError_t dispatch(int D, int group, F&& f) {
  if (D == 64 && group == 32) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 32>{});
  if (D == 64 && group == 64) return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
  if (D == 128 && group == 32) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, 32>{});
  if (D == 128 && group == 64) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, 64>{});
  if (D == 128 && group == 128) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{});
  return cudaErrorInvalidValue;
}

bool vec8(const void* p, int64_t ts, int64_t hs) {
  return (reinterpret_cast<uintptr_t>(p) & 7) == 0 && ts % 4 == 0 && hs % 4 == 0;
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Shape& c, const void* k, int64_t k_ts, int64_t k_hs,
                              const void* v, int64_t v_ts, int64_t v_hs, const int64_t* slots,
                              int64_t T, void* cache, int num_sms, int* dev_status,
                              cudaStream_t stream) {
  Kv4IoArgs a = {};
  a.k = static_cast<const __half*>(k), a.v = static_cast<const __half*>(v);
  a.k_ts = k_ts, a.k_hs = k_hs, a.v_ts = v_ts, a.v_hs = v_hs;
  a.slots = slots, a.cache = static_cast<uint8_t*>(cache);
  a.T = T, a.capacity = c.num_pages * c.page, a.H = c.heads, a.page = c.page;
  a.status = dev_status;
  const int vk = vec8(k, k_ts, k_hs), vv = vec8(v, v_ts, v_hs);
  return dispatch(c.dim, c.group, [&](auto d, auto g) {
    constexpr int kRows = 32 / (d.value / 4) * 8;    // (token, head) rows per block
    int64_t blocks = (T * c.heads + kRows - 1) / kRows;
    if (blocks > (int64_t)num_sms * 32) blocks = (int64_t)num_sms * 32;
    kv4_append_kernel<d.value, g.value><<<(unsigned)blocks, 256, 0, stream>>>(a, vk, vv);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv4_gather(const Kv4Shape& c, const void* cache, const int64_t* slots, int64_t T,
                              void* out_k, void* out_v, int num_sms, int* dev_status,
                              cudaStream_t stream) {
  Kv4IoArgs a = {};
  a.slots = slots, a.cache = static_cast<uint8_t*>(const_cast<void*>(cache));
  a.out_k = static_cast<__half*>(out_k), a.out_v = static_cast<__half*>(out_v);
  a.T = T, a.capacity = c.num_pages * c.page, a.H = c.heads, a.page = c.page;
  a.status = dev_status;
  return dispatch(c.dim, c.group, [&](auto d, auto g) {
    int64_t blocks = (T * c.heads * (d.value / 4) + 255) / 256;
    if (blocks > (int64_t)num_sms * 32) blocks = (int64_t)num_sms * 32;
    kv4_gather_kernel<d.value, g.value><<<(unsigned)blocks, 256, 0, stream>>>(a);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv4_pages(const Kv4PagesCall& c, cudaStream_t stream) {
  PagesArgs a = {};
  a.table = c.table, a.table_rs = c.table_rs, a.held = c.held;
  a.free_pages = c.free_pages, a.free_count = c.free_count;
  a.lens = c.lens, a.fresh_tokens = c.new_tokens, a.reset = c.reset;
  a.slots = c.slots, a.positions = c.positions, a.cu_q = c.cu_q, a.new_lens = c.new_lens;
  a.status = c.status, a.max_tokens = c.max_tokens;
  a.R = c.rows, a.width = c.width, a.capacity = c.capacity, a.page = c.page;
  const size_t smem = 3 * (size_t)(c.rows + 1) * sizeof(int);
  static PerDeviceOnce attr_once;
  const cudaError_t attr = attr_once.run([] {
    return cudaFuncSetAttribute(kv4_pages_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                3 * (kKv4MaxRows + 1) * (int)sizeof(int));
  });
  if (attr != cudaSuccess) return attr;
  cudaLaunchConfig_t cfg = {};
  const int ctas = c.rows <= kPagesThreads && c.max_tokens <= 4 * kPagesThreads ? 1 : 8;
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(kPagesThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ctas, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_pages_kernel, a);
}

}  // namespace awq
