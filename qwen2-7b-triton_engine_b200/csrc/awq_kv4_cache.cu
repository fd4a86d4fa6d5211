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
  int H, page_shift;
  int* status;
};

__device__ __forceinline__ uint32_t hmin2_u32(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hmax2_u32(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// fp16((hi - lo) / 15), rounded once.  The fp32 quotient is within 2^-22 of the exact one; where
// both ends of that interval round to the same fp16 value that is the result, otherwise (about
// one group in a thousand) the double quotient decides: hi - lo is exact in double, and an
// integer multiple of a power of two over 15 that is not a tie is far further than 2^-50 from
// one.
__device__ __forceinline__ __half scale_of(float lo, float hi) {
  const float q = (hi - lo) * (1.0f / 15.0f);
  const __half a = __float2half_rn(q * (1.0f - 0x1p-21f)), b = __float2half_rn(q * (1.0f + 0x1p-21f));
  if (__half_as_ushort(a) == __half_as_ushort(b)) return a;
  return __double2half(((double)hi - (double)lo) / 15.0);
}

// The codes of a lane's octet of channels (nibble p = channel p), its group's scale and minimum.
// LG lanes form a group; u: the eight fp16 values.  Every lane of the warp calls it.
//
// A code is the round-to-nearest-even of the exact (x - m) / s, at most 15.  The fp32 quotient
// is within 2^-18 of the exact one (three roundings of 2^-24 and a reciprocal of 2^-23, quotient
// below 2^5), so only results within 10^-5 of a tie take the double division, which decides
// every tie (x - m is exact in double).  So do groups whose scale is subnormal: elsewhere the
// scale's own rounding (2^-11) leaves the quotient below 15.5.
template <int LG>
__device__ __forceinline__ uint32_t quant_octet(const uint4 u, int lane, __half& sh, __half& mh) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  // (minimum, -maximum) of the group in one register
  const uint32_t lo2 = hmin2_u32(hmin2_u32(w[0], w[1]), hmin2_u32(w[2], w[3]));
  const uint32_t hi2 = hmax2_u32(hmax2_u32(w[0], w[1]), hmax2_u32(w[2], w[3])) ^ 0x80008000u;
  uint32_t v = hmin2_u32(__byte_perm(lo2, hi2, 0x5410), __byte_perm(lo2, hi2, 0x7632));
#pragma unroll
  for (int o = LG / 2; o > 0; o >>= 1) v = hmin2_u32(v, __shfl_xor_sync(0xffffffffu, v, o));
  // an exponent of all ones marks an infinity or a NaN
  uint32_t odd = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) odd |= (w[k] & 0x7FFF7FFFu) + 0x04000400u;
  const uint32_t group = ((1u << LG) - 1u) << (lane & ~(LG - 1));
  const bool bad = (__ballot_sync(0xffffffffu, (odd & 0x80008000u) != 0) & group) != 0;
  const float2 mm = __half22float2(u32_as_h2(v));
  const float lo = mm.x + 0.f, hi = 0.f - mm.y;      // one zero: -0 is stored as +0
  sh = bad ? __ushort_as_half(0x7FFF) : scale_of(lo, hi);
  mh = bad ? __ushort_as_half(0x7FFF) : __float2half_rn(lo);
  const float s = __half2float(sh);
  if (!(s > 0.f)) return 0;
  const float inv = __fdividef(1.0f, s);
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(u32_as_h2(w[k]));
    x[2 * k] = f.x, x[2 * k + 1] = f.y;
  }
  // t + 1.5 * 2^23 rounds t to an integer (ties to even) in the low bits of the float
  uint32_t b[8];
  float worst = 0.f;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float t = (x[p] - lo) * inv, m = t + 12582912.f;
    b[p] = __float_as_uint(m);
    worst = fmaxf(worst, fabsf(t - (m - 12582912.f)));
  }
  if (worst > 0.49999f || s < 6.1035156e-5f) {
#pragma unroll 1
    for (int p = 0; p < 8; ++p) {
      const uint32_t c = (uint32_t)fmin(rint(((double)__half2float(__ushort_as_half(
                             (uint16_t)(w[p >> 1] >> (16 * (p & 1))))) - (double)lo) / (double)s), 15.0);
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q == p) b[q] = 0x4B400000u + c;
    }
  }
  // 1.5 * 2^23 is 0x4B400000: of sum b[p] 16^p, 0x4B400000 (1 + 16 + 256) is the floats' own
  uint32_t c = b[0] - 0x4B400000u * 273u;
#pragma unroll
  for (int p = 1; p < 8; ++p) c += b[p] << (4 * p);
  return c;
}

__device__ __forceinline__ uint4 load_octet(const __half* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
  return make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                    h[6] | (uint32_t)h[7] << 16);
}

// D/8 lanes per token, one kv head per blockIdx.y; whole warps at a time, so that the shuffles
// always see 32 lanes.  A lane has an octet of channels of the K and of the V row: one 16-byte
// load each, the group's minimum and maximum over its lanes by shuffles.
// Bound: instructions.  8191 tokens, 4 heads of 128 channels in groups of 32 take 16 us on B200
// (22 MB read and written: 1.4 TB/s; the issue slots are 59 % busy, the logic pipe 41 %).  With
// 64-bit index divisions and fewer channels a lane this and the read-back took 30.9 us together
// in a graph, now 20.6.  The rows of a decode batch: a launch, 3 us.
template <int D, int GROUP>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const Kv4IoArgs a, const int vec_k, const int vec_v) {
  constexpr int L = D / 8, ROWS = 32 / L, NG = D / GROUP;
  const int lane = threadIdx.x & 31, o = lane % L, h = blockIdx.y;
  const int64_t step = (int64_t)gridDim.x * 8 * ROWS;
  for (int64_t t0 = ((int64_t)blockIdx.x * 8 + threadIdx.x / 32) * ROWS; t0 < a.T; t0 += step) {
    const int64_t tok = t0 + lane / L;
    const bool in = tok < a.T;
    const int64_t slot = in ? a.slots[tok] : -1;
    uint4 ku = make_uint4(0, 0, 0, 0), vu = ku;
    if (in) {
      ku = load_octet(a.k + tok * a.k_ts + h * a.k_hs + 8 * o, vec_k);
      vu = load_octet(a.v + tok * a.v_ts + h * a.v_hs + 8 * o, vec_v);
    }
    __half ks, km, vs, vm;
    const uint32_t kc = quant_octet<GROUP / 8>(ku, lane, ks, km);
    const uint32_t vc = quant_octet<GROUP / 8>(vu, lane, vs, vm);
    if (slot < 0) continue;                          // padding: nothing is written
    if (slot >= a.capacity) {
      if (o == 0) atomicOr(a.status, kDevErrShape);
      continue;
    }
    const int64_t page = slot >> a.page_shift;
    const int at = (int)slot & ((1 << a.page_shift) - 1), b = at & 15;
    uint8_t* blk = a.cache + (((page * a.H + h) << (a.page_shift - 4)) + (at >> 4)) * kv4::block_bytes(D, GROUP);
    *reinterpret_cast<uint32_t*>(blk + b * (D / 2) + 4 * kv4::k_word(D, o)) = kc;
    uint8_t* vrow = blk + kv4::off_v(D) + (b / 2) * D + 2 * (b & 1);
    *reinterpret_cast<uint16_t*>(vrow + 4 * kv4::v_word(D, 2 * o)) = (uint16_t)vc;
    *reinterpret_cast<uint16_t*>(vrow + 4 * kv4::v_word(D, 2 * o + 1)) = (uint16_t)(vc >> 16);
    if (o % (GROUP / 8) == 0) {
      const int gi = o / (GROUP / 8);
      reinterpret_cast<__half2*>(blk + kv4::off_kp(D))[b * NG + gi] = __halves2half2(ks, km);
      reinterpret_cast<__half2*>(blk + kv4::off_vp(D, GROUP))[b * NG + gi] = __halves2half2(vs, vm);
    }
  }
}

// fp16(code * scale + minimum) of the slots' keys and values; a negative slot reads as 0.  One
// thread per octet of channels of a token's K and V rows.
// Bound: instructions, the logic pipe.  8191 tokens, 4 heads of 128 channels in groups of 32
// take 9 us on B200 (22 MB: 2.4 TB/s; the logic pipe is 56 % busy, with the launch in it).
template <int D, int GROUP>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const Kv4IoArgs a) {
  constexpr int L = D / 8, NG = D / GROUP;
  const int o = threadIdx.x % L, h = blockIdx.y;
  const int64_t step = (int64_t)gridDim.x * (256 / L);
  for (int64_t tok = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L; tok < a.T; tok += step) {
    const int64_t slot = a.slots[tok];
    uint4 ko = make_uint4(0, 0, 0, 0), vo = make_uint4(0, 0, 0, 0);
    if (slot >= a.capacity) {
      if (o == 0) atomicOr(a.status, kDevErrShape);
    } else if (slot >= 0) {
      const int64_t page = slot >> a.page_shift;
      const int at = (int)slot & ((1 << a.page_shift) - 1), b = at & 15;
      const uint8_t* blk = a.cache + (((page * a.H + h) << (a.page_shift - 4)) + (at >> 4)) * kv4::block_bytes(D, GROUP);
      const uint32_t kc = *reinterpret_cast<const uint32_t*>(blk + b * (D / 2) + 4 * kv4::k_word(D, o));
      const uint8_t* vrow = blk + kv4::off_v(D) + (b / 2) * D + 2 * (b & 1);
      const uint32_t vc = *reinterpret_cast<const uint16_t*>(vrow + 4 * kv4::v_word(D, 2 * o)) |
                          (uint32_t)*reinterpret_cast<const uint16_t*>(vrow + 4 * kv4::v_word(D, 2 * o + 1)) << 16;
      const int gi = o / (GROUP / 8);
      const float2 kp = __half22float2(reinterpret_cast<const __half2*>(blk + kv4::off_kp(D))[b * NG + gi]);
      const float2 vp = __half22float2(reinterpret_cast<const __half2*>(blk + kv4::off_vp(D, GROUP))[b * NG + gi]);
      uint32_t kw[4], vw[4];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        kw[p] = h2_as_u32(__floats2half2_rn(fmaf((float)((kc >> (8 * p)) & 15u), kp.x, kp.y),
                                            fmaf((float)((kc >> (8 * p + 4)) & 15u), kp.x, kp.y)));
        vw[p] = h2_as_u32(__floats2half2_rn(fmaf((float)((vc >> (8 * p)) & 15u), vp.x, vp.y),
                                            fmaf((float)((vc >> (8 * p + 4)) & 15u), vp.x, vp.y)));
      }
      ko = make_uint4(kw[0], kw[1], kw[2], kw[3]);
      vo = make_uint4(vw[0], vw[1], vw[2], vw[3]);
    }
    const int64_t out = (tok * a.H + h) * D + 8 * o;
    *reinterpret_cast<uint4*>(a.out_k + out) = ko;
    *reinterpret_cast<uint4*>(a.out_v + out) = vo;
  }
}

// ---- page bookkeeping -------------------------------------------------------------------
// One cluster does the whole step.  Every CTA scans all rows for itself (pages released,
// pages needed, tokens: three prefix sums kept in shared memory) and then takes a share of
// the flat lists of released pages, new pages and tokens, finding an element's row by
// bisection.  The cluster barriers separate the three uses of the free stack: push the
// released pages, read the popped ones, clear them.
// Bound: latency, a chain of loads, scans, barriers and bisections; the bytes of the largest
// case below take 0.1 us.  Measured on B200: 64 requests, three of them replaced, 8.4 us; 2048
// requests, a hundred replaced by prompts of 301 tokens, 16.6 us (22.6 us with a scan for each
// list and one bisection at a time).
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
constexpr int kPagesThreads = 1024, kPagesFew = 256;

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

// Rows of N elements at once (the bisections overlap): the largest r with pre[r] <= j[n]
// (pre[0] = 0, ascending).
template <int N>
__device__ __forceinline__ void rows_of(const int* pre, int R, const int (&j)[N], int (&row)[N]) {
  int hi[N];
#pragma unroll
  for (int n = 0; n < N; ++n) row[n] = 0, hi[n] = R;
  for (int span = R; span > 1; span = (span + 1) >> 1)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int mid = (row[n] + hi[n]) >> 1;
      if (hi[n] - row[n] > 1) {
        if (pre[mid] <= j[n]) row[n] = mid; else hi[n] = mid;
      }
    }
}

// THREADS a CTA, up to PER rows a thread (THREADS = 256: one CTA, which needs no cluster).
template <int THREADS, int PER>
__global__ void __launch_bounds__(THREADS) kv4_pages_kernel(const PagesArgs a) {
  namespace cg = cooperative_groups;
  constexpr bool kAlone = THREADS == kPagesFew;
  auto everyone = [] {                               // all threads that share the step
    if constexpr (kAlone) __syncthreads();
    else cg::this_cluster().sync();
  };
  extern __shared__ int sm[];                        // pre[3][R + 1], kept [R], len [R]
  __shared__ long long wsum[3][THREADS / 32];
  __shared__ int s_bad;
  int* pre_gone = sm;
  int* pre_need = sm + (a.R + 1);
  int* pre_tok = sm + 2 * (a.R + 1);
  int* s_kept = sm + 3 * (a.R + 1);                  // pages the row keeps through the release
  int* s_len = s_kept + a.R;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  if (tid == 0) s_bad = 0;
  const int count = *a.free_count;
  __syncthreads();
  // a thread has `per` neighbouring rows, so that one scan over the block is enough
  const int per = (a.R + THREADS - 1) / THREADS;
  int g[PER], nd[PER], nw[PER];
  long long sum[3] = {0, 0, 0};
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * per + i;
    g[i] = nd[i] = nw[i] = 0;
    if (i < per && r < a.R) {
      const long long h = a.held[r], len = a.lens[r], n = a.fresh_tokens[r];
      const bool rs = a.reset && a.reset[r];
      const long long need = (len + n + a.page - 1) / a.page, kept = rs ? 0 : h;
      if (h < 0 || h > a.width || len < 0 || n < 0 || len + n > 0x7fffffffLL || need > a.width)
        s_bad = 1;
      g[i] = rs ? (int)h : 0;
      nd[i] = need > kept ? (int)(need - kept) : 0;
      nw[i] = (int)n;
      s_kept[r] = (int)kept;
      s_len[r] = (int)len;
      sum[0] += g[i], sum[1] += nd[i], sum[2] += nw[i];
    }
  }
  long long inc[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    inc[k] = warp_scan(sum[k], lane);
    if (lane == 31) wsum[k][warp] = inc[k];
  }
  __syncthreads();
  long long total[3], base[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const long long w = warp_scan(lane < THREADS / 32 ? wsum[k][lane] : 0, lane);
    total[k] = __shfl_sync(0xffffffffu, w, 31);
    const long long before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    base[k] = (warp ? before : 0) + inc[k] - sum[k];
  }
  const long long gone = total[0], need = total[1], tokens = total[2];
  int status = 0;
  if (s_bad || count < 0 || count + gone > a.capacity || tokens > a.max_tokens) status = -1;
  else if (need > count + gone) status = (int)min(need - count - gone, 0x7fffffffLL);
  const bool ok = status == 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int r = tid * per + i;
    if (i < per && r < a.R) {
      pre_gone[r] = (int)base[0], pre_need[r] = (int)base[1], pre_tok[r] = (int)base[2];
      base[0] += g[i], base[1] += nd[i], base[2] += nw[i];
    }
  }
  if (tid == 0) pre_gone[a.R] = (int)gone, pre_need[a.R] = (int)need, pre_tok[a.R] = (int)tokens;
  __syncthreads();
  const int top = ok ? count + (int)gone : 0;        // stack height between push and pop
  const int gt = (int)blockIdx.x * THREADS + tid, gn = (int)gridDim.x * THREADS;
  if (ok)
    for (int j = gt; j < (int)gone; j += gn) {       // push: the first released page on top
      int at[1] = {j}, r[1];
      rows_of(pre_gone, a.R, at, r);
      int32_t* e = a.table + r[0] * a.table_rs + (j - pre_gone[r[0]]);
      a.free_pages[top - 1 - j] = *e;
      *e = -1;
    }
  everyone();
  if (ok)
    for (int j = gt; j < (int)need; j += gn) {       // pop into the rows' next columns
      int at[1] = {j}, r[1];
      rows_of(pre_need, a.R, at, r);
      a.table[r[0] * a.table_rs + s_kept[r[0]] + (j - pre_need[r[0]])] = __ldcg(a.free_pages + top - 1 - j);
    }
  constexpr int N = 4;
  for (int64_t t0 = gt; t0 < a.max_tokens; t0 += (int64_t)N * gn) {
    int at[N], r[N], pos[N], pg[N], col[N];
#pragma unroll
    for (int n = 0; n < N; ++n) at[n] = (int)min((long long)t0 + (long long)n * gn, ok && tokens ? tokens - 1 : 0LL);
    if (ok && tokens) {
      rows_of(pre_tok, a.R, at, r);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        pos[n] = s_len[r[n]] + (at[n] - pre_tok[r[n]]);
        col[n] = pos[n] / a.page;
        const int kept = s_kept[r[n]];
        pg[n] = col[n] < kept ? a.table[r[n] * a.table_rs + col[n]]
                              : __ldcg(a.free_pages + top - 1 - (pre_need[r[n]] + col[n] - kept));
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int64_t t = t0 + (int64_t)n * gn;
      if (t >= a.max_tokens) continue;
      const bool live = ok && t < tokens;
      a.slots[t] = live && pg[n] >= 0 ? (int64_t)pg[n] * a.page + (pos[n] - col[n] * a.page) : -1;
      a.positions[t] = live ? pos[n] : 0;
    }
  }
  for (int r = gt; r <= a.R; r += gn) {
    a.cu_q[r] = ok ? pre_tok[r] : 0;
    if (r < a.R) a.new_lens[r] = s_len[r] + (ok ? pre_tok[r + 1] - pre_tok[r] : 0);
  }
  everyone();                                    // every reader of the stack and the state is done
  if (ok) {
    for (int r = gt; r < a.R; r += gn) a.held[r] = s_kept[r] + (pre_need[r + 1] - pre_need[r]);
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

int log2_of(int n) {
  int b = 0;
  while ((1 << b) < n) ++b;
  return b;
}

bool vec16(const void* p, int64_t ts, int64_t hs) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ts % 8 == 0 && hs % 8 == 0;
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
  a.T = T, a.capacity = c.num_pages * c.page, a.H = c.heads, a.page_shift = log2_of(c.page);
  a.status = dev_status;
  const int vk = vec16(k, k_ts, k_hs), vv = vec16(v, v_ts, v_hs);
  return dispatch(c.dim, c.group, [&](auto d, auto g) {
    constexpr int kTokens = 32 / (d.value / 8) * 8;  // of a block
    int64_t blocks = (T + kTokens - 1) / kTokens;
    if (blocks > (int64_t)num_sms * 64) blocks = (int64_t)num_sms * 64;
    kv4_append_kernel<d.value, g.value><<<dim3((unsigned)blocks, c.heads), 256, 0, stream>>>(a, vk, vv);
    return cudaGetLastError();
  });
}

cudaError_t launch_kv4_gather(const Kv4Shape& c, const void* cache, const int64_t* slots, int64_t T,
                              void* out_k, void* out_v, int num_sms, int* dev_status,
                              cudaStream_t stream) {
  Kv4IoArgs a = {};
  a.slots = slots, a.cache = static_cast<uint8_t*>(const_cast<void*>(cache));
  a.out_k = static_cast<__half*>(out_k), a.out_v = static_cast<__half*>(out_v);
  a.T = T, a.capacity = c.num_pages * c.page, a.H = c.heads, a.page_shift = log2_of(c.page);
  a.status = dev_status;
  return dispatch(c.dim, c.group, [&](auto d, auto g) {
    constexpr int kTokens = 256 / (d.value / 8);
    int64_t blocks = (T + kTokens - 1) / kTokens;
    if (blocks > (int64_t)num_sms * 64) blocks = (int64_t)num_sms * 64;
    kv4_gather_kernel<d.value, g.value><<<dim3((unsigned)blocks, c.heads), 256, 0, stream>>>(a);
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
  const size_t smem = (3 * (size_t)(c.rows + 1) + 2 * (size_t)c.rows) * sizeof(int);
  // One small CTA where its threads have a row and a few tokens each at most: a decode step of
  // 64 requests of which three are replaced takes 8.4 us on it, 10.4 us on a cluster of eight.
  if (c.rows <= kPagesFew && c.max_tokens <= 4 * kPagesFew) {
    kv4_pages_kernel<kPagesFew, 1><<<1, kPagesFew, smem, stream>>>(a);
    return cudaGetLastError();
  }
  static PerDeviceOnce attr_once;
  const cudaError_t attr = attr_once.run([] {
    return cudaFuncSetAttribute(kv4_pages_kernel<kPagesThreads, kKv4MaxRows / kPagesThreads>,
                                cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (5 * kKv4MaxRows + 3) * (int)sizeof(int));
  });
  if (attr != cudaSuccess) return attr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(8, 1, 1);
  cfg.blockDim = dim3(kPagesThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 8, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_pages_kernel<kPagesThreads, kKv4MaxRows / kPagesThreads>, a);
}

}  // namespace awq
