// awq_kv4_prefill.cu -- attention of many query rows over the paged 4-bit key/value cache, on
// tcgen05.  Same mathematics as awq_kv4_attn.cu, for requests with many query rows per kv
// head (prompt chunks), where the tensor work binds instead of the cache's bytes.
//
// One CTA works on 256 query rows (two row tiles A and B of 128) of a request's kv head, over
// steps of NTOK = 128 / NG tokens (NG scale groups per head):
//   S_g [128 x NTOK] = Q_g [128 x group] . C_g^T      codes as fp16 integers (subnormals)
//   x = scale sum_g (s_tg S_g + m_tg sum q_g)          fp32, one thread per query row
//   P_g = fp16(2^(x - M) v_tg)                         value scales, reference M as there
//   O_g [128 x group] += P_g . (C'_g - 8)
// so keys and values are never rounded: scales and minima are applied in fp32.  One group
// (NG = 1) is a plain flash step of 128 tokens; more groups trade tokens for accumulators, so
// that S always takes 128 columns of tensor memory, P 64 of them (over S, once it is read)
// and O head_dim: 2 x 256 columns in all.
//
// Roles (16 warps): two softmax warpgroups (one per row tile, one row per thread, so no
// shuffles), one warpgroup that spreads the packed codes into the MMAs' K-major 128-byte
// swizzled operands, a warp that issues the MMAs and one that fetches cache blocks with bulk
// copies.  While one tile's softmax runs, the tensor core works on the other tile.
//
// Work split: items (request, kv head, 256 rows) are cut into steps, causal lengths counted
// per item, and every CTA (one per SM) takes an equal share of the list of steps; items that
// cross CTAs are joined by kv4_prefill_merge in CTA order.
//
// Bound: the softmax warps' latency.  Measured on B200, four requests of 1 to 1024 query tokens
// and 777 to 8192 cached ones, 28 / 4 heads of 128 channels: 346 us, 0.52 PFLOP/s; a step of 256
// rows x 128 tokens takes 3.4 us, of which the MMAs need 1.1, the exponentials 1.1 and the
// operand traffic in shared memory 1.4; no pipe is busier than 43 % (shared memory).  A tile waits a third of
// the time for its S, which shares tensor memory with its P: 512 columns hold two tiles of S
// and O, and no third S.  Measured and not kept (same case, 380 us then): scales and minima as
// fp16 pairs in shared memory 463 us, all eight softmax warps on one tile after the other 417,
// S in two buffers of 64 tokens 399, half of the exponentials as polynomials 479, x kept in
// registers between the two passes 392 (184 registers) to 422.  The compiler holds the kernel at
// the launch's 128 registers a thread and spills 200 to 560 bytes a thread of its forms (128
// channels in groups of 128: 560); where, and what that costs, is not measured.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <type_traits>

#include "awq_common.cuh"
#include "awq_internal.h"
#include "awq_kv4.cuh"
#include "awq_kv4_args.cuh"
#include "awq_sm100.cuh"

namespace awq {

namespace {

using kv4::AttnArgs;
using kv4::kDescInts;
using kv4::kPrefixEntries;

constexpr int kThreads = 512;
constexpr int kRows = kKv4PrefillRows;   // 256: query rows of an item, two tiles of 128
// One stage of raw blocks is enough, as the unpacking warps hold a step's in registers; the
// room is better spent on a fourth operand slot (the header's case: 6 % less time).
constexpr int kKvSlots = 4, kRawStages = 1, kParStages = 2;
// Empty steps of an item, for its fixed cost (queries, first and last step, result).  Four
// requests of 1024 query and up to 8192 cached tokens, 28 / 4 heads: 1 375 us, 2 368 us, 4 360 us
// with a result that took 6 us; with today's 2 345 us, 3 344 us (three operand slots).
constexpr int kItemSteps = 3;
constexpr float kMaxSpread = 128.f;      // 2^kBelowTop
constexpr uint64_t kWaitNs = 2000000000ull;

template <int D_, int GROUP_>
struct Geo {
  static constexpr int D = D_, GROUP = GROUP_, NG = D / GROUP;
  static constexpr int NTOK = 128 / NG, NBLK = NTOK / 16, BLK = kv4::block_bytes(D, GROUP);
  static constexpr int RAW = NBLK * BLK;               // a step's cache blocks
  static constexpr int KA = D / 64;                    // 64-channel atoms of Q and K rows
  static constexpr int VA = (NTOK + 63) / 64;          // 64-token atoms of V rows
  static constexpr int QTILE = KA * 128 * 128, KSLOT = KA * NTOK * 128, VSLOT = VA * D * 128;
  static constexpr int SLOT = KSLOT > VSLOT ? KSLOT : VSLOT;
  // ks, km, vs, vm [NG][NTOK], log2 of a token's largest vs [NTOK], largest and least [4]
  static constexpr int PAR = 4 * 128 * 4 + NTOK * 4 + 32;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = OFF_Q + 2 * QTILE;
  static constexpr int OFF_RAW = OFF_KV + kKvSlots * SLOT;
  static constexpr int OFF_PAR = OFF_RAW + kRawStages * RAW;
  static constexpr int OFF_PRE = OFF_PAR + kParStages * PAR;
  static constexpr int OFF_BAR = OFF_PRE + (kPrefixEntries + 8) * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;    // + alignment slack
  static_assert(SMEM <= 227 * 1024 && QTILE % 1024 == 0 && SLOT % 1024 == 0 && RAW % 16 == 0 &&
                    PAR % 16 == 0, "shared memory");
};
enum Bar {
  RAW_FULL = 0,
  RAW_EMPTY = RAW_FULL + kRawStages,
  KV_FULL = RAW_EMPTY + kRawStages,
  KV_EMPTY = KV_FULL + kKvSlots,
  PAR_FULL = KV_EMPTY + kKvSlots,
  PAR_EMPTY = PAR_FULL + kParStages,
  Q_READY = PAR_EMPTY + kParStages,
  S_FULL = Q_READY + 2,
  P_READY = S_FULL + 2,
  O_FULL = P_READY + 2,
  DRAIN = O_FULL + 2,
  NBARS = DRAIN + 1
};
static_assert(NBARS * 8 <= 256, "barriers");

// A request's items: nrt row tiles of 256 per kv head, each with its causal number of steps
// and kItemSteps empty ones that stand for its fixed cost.
struct Item {
  int L, n, q0, nrt;
  int r, h, rt, step;
  int vis, steps;

  template <class G_>
  __device__ void request(const AttnArgs& a) {
    const int cap = (int)min((long long)a.width << a.page_shift, 0x7fffff00LL);
    L = min(max(a.lens[r], 0), cap);
    n = q0 = 0;
    if (a.cu_q) {
      const int b = a.cu_q[r], e = a.cu_q[r + 1];
      if (b >= 0 && e >= b && e <= a.tokens) q0 = b, n = e - b;
    } else {
      q0 = r, n = 1;
    }
    if ((long long)n * a.G < a.min_rows) n = 0;         // the other kernel's request
    nrt = (int)(((long long)n * a.G + kRows - 1) / kRows);
  }
  template <class G_>
  __device__ int steps_of(const AttnArgs& a, int tile, int* seen) const {
    const int last = min(n - 1, (int)(((long long)(tile + 1) * kRows - 1) / a.G));
    *seen = max(0, L - n + last + 1);
    return (*seen + G_::NTOK - 1) / G_::NTOK + kItemSteps;
  }
  template <class G_>
  __device__ int units(const AttnArgs& a) const {       // of one kv head
    // steps_of of every tile, its last row's token counted up instead of divided out
    const int dq = kRows / a.G, dr = kRows - dq * a.G;
    int s = 0, last = -1, rem = a.G - 1;                 // row -1: token -1, its last row
    for (int i = 0; i < nrt; ++i) {
      last += dq, rem += dr;
      if (rem >= a.G) rem -= a.G, ++last;
      const int seen = max(0, L - n + min(n - 1, last) + 1);
      s += (seen + G_::NTOK - 1) / G_::NTOK + kItemSteps;
    }
    return s;
  }
  template <class G_>
  __device__ void next(const AttnArgs& a) {
    step = 0;
    if (++rt == nrt) {
      rt = 0;
      if (++h == a.kv_heads) {
        h = 0;
        do {
          if (++r >= a.R) return;
          request<G_>(a);
        } while (nrt == 0);
      }
    }
    steps = steps_of<G_>(a, rt, &vis);
  }
};

// This CTA's part of an item.
struct Segment {
  int k0, count;        // first step, steps with tokens
  bool skip, whole, starts;
  bool two;             // the second row tile has rows
  __device__ Segment(const Item& it, const AttnArgs& a, int u, int u0, int u1) {
    const int ib = u - it.step, real = it.steps - kItemSteps;
    k0 = it.step;
    count = max(0, min(real, k0 + u1 - u) - k0);
    starts = ib >= u0;
    skip = count == 0 && (real > 0 || !starts);                       // only empty steps are left
    whole = starts && ib + max(1, real) <= u1;
    two = (long long)it.n * a.G > (long long)it.rt * kRows + 128;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 lanes in one instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}
// Byte offset of 16-byte chunk c (0..7) of a 128-byte row under the 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(int row, int c) { return row * 128 + ((c ^ (row & 7)) << 4); }

template <class G_>
__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const AttnArgs a) {
  constexpr int D = G_::D, GROUP = G_::GROUP, NG = G_::NG, NTOK = G_::NTOK, NBLK = G_::NBLK;
  constexpr int BLK = G_::BLK, PAR = G_::PAR;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024 - (sm100::smem_u32(smem_raw) & 1023)) & 1023);
  const uint32_t sbase = sm100::smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  int* pre = reinterpret_cast<int*>(smem + G_::OFF_PRE);
  const uint32_t bars = sbase + G_::OFF_BAR;
  __shared__ volatile int s_abort;
  __shared__ uint32_t s_tmem;
  __shared__ Item s_first;
  __shared__ int raw_ok[kRawStages], par_ok[kParStages];   // blocks of the step that are there

  if (tid == 0) {
    s_abort = 0;
    for (int i = 0; i < NBARS; ++i) {
      int count = 1;                                     // bulk copies, MMA commits
      if (i >= RAW_EMPTY && i < RAW_EMPTY + kRawStages) count = 128;
      if (i >= KV_FULL && i < KV_FULL + kKvSlots) count = 128;
      if (i >= PAR_FULL && i < PAR_FULL + kParStages) count = 128;
      if (i >= PAR_EMPTY && i < PAR_EMPTY + kParStages) count = 256;
      if (i >= Q_READY && i < Q_READY + 2) count = 128;
      if (i >= P_READY && i < P_READY + 2) count = 128;
      sm100::mbar_init(bars + 8 * i, count);
    }
    sm100::fence_mbar_init();
  }
  const int U = kv4::scan_units<kThreads>(a, pre, [&](int r) {
    Item it;
    it.r = r;
    it.request<G_>(a);
    return a.kv_heads * it.units<G_>(a);
  });
  sm100::grid_launch_dependents();                       // the other kernel fills SMs as they end
  const int cta = blockIdx.x, ctas = min((int)gridDim.x, U);
  if (cta >= ctas) {
    if (tid == 0) a.desc[cta * kDescInts] = 0;
    return;
  }
  const int uq = U / ctas, ur = U - uq * ctas;
  auto first_unit = [&](int c) { return uq * c + ur * c / ctas; };
  const int u0 = first_unit(cta), u1 = first_unit(cta + 1);
  if (warp == 0) {
    sm100::tmem_alloc(sm100::smem_u32(&s_tmem), 512);
    sm100::tmem_relinquish();
  }
  if (tid == 32) {
    const int shift = kv4::prefix_shift(a);
    int lo = 0, hi = (a.R + (1 << shift) - 1) >> shift;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u0) lo = mid; else hi = mid;
    }
    Item it = {};
    int rem = u0 - pre[lo], per = 0;
    it.r = lo << shift;
    for (;;) {
      it.request<G_>(a);
      per = it.units<G_>(a);
      if (rem < per * a.kv_heads || it.r + 1 >= a.R) break;
      rem -= per * a.kv_heads;
      ++it.r;
    }
    it.h = rem / per;
    rem -= it.h * per;
    for (it.rt = 0;; ++it.rt) {
      it.steps = it.steps_of<G_>(a, it.rt, &it.vis);
      if (rem < it.steps) break;
      rem -= it.steps;
    }
    it.step = rem;
    s_first = it;
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = s_tmem;
  auto bar = [&](int i) { return bars + 8 * i; };
  // A wait that runs out ends every later wait of the CTA at once.  The roles of one lane or
  // warp stop there; the softmax and unpacking warps, whose lanes vote and shuffle, run through
  // their remaining steps together, on whatever they find (the status says that the output is
  // wrong).  A vote behind every wait instead costs 2 %: 351 us for 344 in the header's case.
  auto wait = [&](int b, uint32_t parity) {
    if (s_abort) return false;
    if (sm100::mbar_wait_bounded(bar(b), parity, a.status, kWaitNs)) return true;
    s_abort = 1;
    return false;
  };
  Item it = s_first;

  if (warp < 8) {
    // ---- softmax: warpgroup T has row tile T, thread = row ---------------------------------
    sm100::setmaxnreg_inc<168>();
    const int T = warp >> 2, rloc = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + T * 128, tO = tmem + lanes + 256 + T * 128;
    const uint32_t qs_base = sbase + G_::OFF_Q + T * G_::QTILE;
    int np = 0, ns = 0, nq = 0;                          // steps, this tile's steps, segments
    for (int u = u0; u < u1; u += it.steps - it.step, it.next<G_>(a)) {
      const Segment sg(it, a, u, u0, u1);
      if (sg.skip) continue;
      const int row = it.rt * kRows + T * 128 + rloc;
      const bool in = row < it.n * a.G;
      const int head = it.h * a.G + row % a.G, tokq = it.q0 + row / a.G;
      const bool mine = T == 0 || sg.two;
      float qs[NG], ksc = 0.f, M = -CUDART_INF_F;
      F2 l2 = pack2(0.f, 0.f), pm2[NG];
#pragma unroll
      for (int k = 0; k < NG; ++k) qs[k] = 0.f, pm2[k] = pack2(0.f, 0.f);
      const int lim = in ? it.L - it.n + row / a.G : -1;
      if (sg.count > 0 && mine) {
        // queries into the A operand: the codes' order within an octet, odd channels / 16,
        // scaled up to just below fp16's limit
        uint4 v[D / 8];
        float big = 0.f;
        const __half* qp = a.q + (in ? (int64_t)tokq * a.q_ts + (int64_t)head * a.q_hs : 0);
#pragma unroll
        for (int o = 0; o < D / 8; ++o) {
          v[o] = make_uint4(0, 0, 0, 0);
          if (in) v[o] = *reinterpret_cast<const uint4*>(qp + 8 * o);
        }
#pragma unroll
        for (int o = 0; o < D / 8; ++o) {
          const uint32_t w[4] = {v[o].x, v[o].y, v[o].z, v[o].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(u32_as_h2(w[k]));
            qs[o * 8 / GROUP] += f.x + f.y;
            big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        const int e_big = (int)(__float_as_uint(big) >> 23) - 127;
        const int up2 = big > 0.f && e_big <= 15 ? 15 - e_big : 0;
        // (a negative scale turns the queries: the largest x is then the largest score)
        const float qmul = copysignf(__uint_as_float((uint32_t)(127 + up2) << 23), a.scale_log2);
        const float qodd = qmul * 0.0625f;
        // x = ksc (s S + m qs): codes enter the MMA times 2^-24, queries times qmul
        ksc = fmaxf(fabsf(a.scale_log2), 1e-30f) * 16777216.0f * __uint_as_float((uint32_t)(127 - up2) << 23);
#pragma unroll
        for (int k = 0; k < NG; ++k) qs[k] *= qmul * 5.9604645e-8f;
#pragma unroll
        for (int o = 0; o < D / 8; ++o) {
          const uint32_t ev[2] = {__byte_perm(v[o].x, v[o].z, 0x5410), __byte_perm(v[o].y, v[o].w, 0x5410)};
          const uint32_t od[2] = {__byte_perm(v[o].x, v[o].z, 0x7632), __byte_perm(v[o].y, v[o].w, 0x7632)};
          uint32_t c[4];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float2 e = __half22float2(u32_as_h2(ev[k])), f = __half22float2(u32_as_h2(od[k]));
            c[2 * k] = h2_as_u32(__floats2half2_rn(e.x * qmul, e.y * qmul));
            c[2 * k + 1] = h2_as_u32(__floats2half2_rn(f.x * qodd, f.y * qodd));
          }
          sm100::st_shared_v4(qs_base + (o / 8) * (128 * 128) + swz(rloc, o & 7), c[0], c[1], c[2], c[3]);
        }
        sm100::fence_proxy_async_smem();
        sm100::mbar_arrive(bar(Q_READY + T));
      }
      const int lim_lo = it.L - it.n + (it.rt * kRows + T * 128) / a.G;   // all rows see these
      for (int k = 0; k < sg.count; ++k, ++np) {
        const int ps = np % kParStages;
        wait(PAR_FULL + ps, (np / kParStages) & 1);
        if (!mine) {
          sm100::mbar_arrive(bar(PAR_EMPTY + ps));
          continue;
        }
        wait(S_FULL + T, ns & 1);
        ++ns;
        sm100::tc_fence_after();
        const int tok0 = (sg.k0 + k) * NTOK;
        const int ok = par_ok[ps];
        const float* par = reinterpret_cast<const float*>(smem + G_::OFF_PAR + ps * PAR);
        const float* ls = par + 512;
        // One step.  SLOW: some of its tokens may be unseen (past a row's limit, or in a page
        // the table does not name), or their value scales differ by more than 2^kBelowTop, so
        // that the reference has to look at every token's scale: with the step's largest in
        // their place it lies up to their spread too high, and never above the largest p s.
        const float4 hi4 = *reinterpret_cast<const float4*>(ls + NTOK);
        const float4 lo4 = *reinterpret_cast<const float4*>(ls + NTOK + 4);
        const float v_hi = fmaxf(fmaxf(hi4.x, hi4.y), fmaxf(hi4.z, hi4.w));
        const float v_lo = fminf(fminf(lo4.x, lo4.y), fminf(lo4.z, lo4.w));
        auto softmax_step = [&](auto slow) {
        constexpr bool SLOW = decltype(slow)::value;
        constexpr int CT = 32 / NG, NC = NTOK / CT;      // tokens of a chunk: 32 registers of S
        auto unseen = [&](int t) { return tok0 + t > lim || !((ok >> (t / 16)) & 1); };
        float top = -CUDART_INF_F;
        {
          // first pass: x / ksc of every token, back into the columns of S_0, and the largest
          uint32_t buf[2][NG][CT];
          auto load = [&](int b, int c) {
#pragma unroll
            for (int g = 0; g < NG; ++g) sm100::tmem_ld_32x32b<CT>(tS + g * NTOK + c * CT, buf[b][g]);
          };
          load(0, 0);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            sm100::tmem_ld_wait();
            if (c + 1 < NC) load((c + 1) & 1, c + 1);
            uint32_t x[CT];
#pragma unroll
            for (int t0 = 0; t0 < CT; t0 += 4) {
              const int t = c * CT + t0;
              F2 y[2];
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                const float4 s4 = *reinterpret_cast<const float4*>(par + g * NTOK + t);
                const float4 m4 = *reinterpret_cast<const float4*>(par + 128 + g * NTOK + t);
                const F2 q2 = pack2(qs[g], qs[g]);
                const uint32_t* S = buf[c & 1][g] + t0;
                const F2 a0 = pack2(__uint_as_float(S[0]), __uint_as_float(S[1]));
                const F2 a1 = pack2(__uint_as_float(S[2]), __uint_as_float(S[3]));
                const F2 b0 = pack2(m4.x, m4.y), b1 = pack2(m4.z, m4.w);
                y[0] = fma2(a0, pack2(s4.x, s4.y), g == 0 ? mul2(b0, q2) : fma2(b0, q2, y[0]));
                y[1] = fma2(a1, pack2(s4.z, s4.w), g == 0 ? mul2(b1, q2) : fma2(b1, q2, y[1]));
              }
              float2 y0 = unpack2(y[0]), y1 = unpack2(y[1]);
              if constexpr (SLOW) {
                if (unseen(t)) y0.x = -CUDART_INF_F;
                if (unseen(t + 1)) y0.y = -CUDART_INF_F;
                if (unseen(t + 2)) y1.x = -CUDART_INF_F;
                if (unseen(t + 3)) y1.y = -CUDART_INF_F;
                const float4 l4 = *reinterpret_cast<const float4*>(ls + t);
                top = fmaxf(top, fmaxf(fmaxf(fmaf(y0.x, ksc, l4.x), fmaf(y0.y, ksc, l4.y)),
                                       fmaxf(fmaf(y1.x, ksc, l4.z), fmaf(y1.y, ksc, l4.w))));
              } else {
                top = fmaxf(top, fmaxf(fmaxf(y0.x, y0.y), fmaxf(y1.x, y1.y)));
              }
              x[t0] = __float_as_uint(y0.x), x[t0 + 1] = __float_as_uint(y0.y);
              x[t0 + 2] = __float_as_uint(y1.x), x[t0 + 3] = __float_as_uint(y1.y);
            }
            sm100::tmem_st_32x32b<CT>(tS + c * CT, x);
          }
        }
        if constexpr (!SLOW) top = fmaf(top, ksc, lg2(v_hi));
        top -= kv4::kBelowTop;
        // the reference moves when it is more than 2^8 behind
        if (__any_sync(0xffffffffu, top > M + kv4::kMoveAt)) {
          const float m = fmaxf(M, top), f = M == m ? 1.0f : ex2(M - m);
          M = m;
          const F2 f2 = pack2(f, f);
          l2 = mul2(l2, f2);
#pragma unroll
          for (int g = 0; g < NG; ++g) pm2[g] = mul2(pm2[g], f2);
          if (k > 0) {                                   // the step before is in O already
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              sm100::tmem_ld_32x32b_x32(tO + 32 * c, o);
              sm100::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              sm100::tmem_st_32x32b_x32(tO + 32 * c, o);
            }
          }
        }
        const float Mu = M == -CUDART_INF_F ? 0.f : M;
        const F2 negM = pack2(-Mu, -Mu), ksc2 = pack2(ksc, ksc);
        sm100::tmem_st_wait();
        // second pass: weights, sums, and P_g over columns that have been read: 16 per chunk
        // of 32 tokens in the columns of S_g
        constexpr int PT = NTOK < 32 ? NTOK : 32;
        uint32_t xb[2][PT];
        sm100::tmem_ld_32x32b<PT>(tS, xb[0]);
#pragma unroll
        for (int c = 0; c < NTOK / PT; ++c) {
          sm100::tmem_ld_wait();
          if (c + 1 < NTOK / PT) sm100::tmem_ld_32x32b<PT>(tS + (c + 1) * PT, xb[(c + 1) & 1]);
          uint32_t w[NG][PT / 2];
#pragma unroll
          for (int t0 = 0; t0 < PT; t0 += 4) {
            const int t = c * PT + t0;
            const uint32_t* x = xb[c & 1] + t0;
            const float2 e0 = unpack2(fma2(pack2(__uint_as_float(x[0]), __uint_as_float(x[1])), ksc2, negM));
            const float2 e1 = unpack2(fma2(pack2(__uint_as_float(x[2]), __uint_as_float(x[3])), ksc2, negM));
            const F2 p0 = pack2(ex2(e0.x), ex2(e0.y)), p1 = pack2(ex2(e1.x), ex2(e1.y));
            l2 = add2(l2, add2(p0, p1));
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              float4 s4 = *reinterpret_cast<const float4*>(par + 256 + g * NTOK + t);
              float4 m4 = *reinterpret_cast<const float4*>(par + 384 + g * NTOK + t);
              if constexpr (SLOW) {                      // unseen tokens may hold anything
                if (unseen(t)) s4.x = m4.x = 0.f;
                if (unseen(t + 1)) s4.y = m4.y = 0.f;
                if (unseen(t + 2)) s4.z = m4.z = 0.f;
                if (unseen(t + 3)) s4.w = m4.w = 0.f;
              }
              pm2[g] = fma2(p0, pack2(m4.x, m4.y), pm2[g]);
              pm2[g] = fma2(p1, pack2(m4.z, m4.w), pm2[g]);
              const float2 w0 = unpack2(mul2(p0, pack2(s4.x, s4.y)));
              const float2 w1 = unpack2(mul2(p1, pack2(s4.z, s4.w)));
              w[g][t0 / 2] = h2_as_u32(__floats2half2_rn(w0.x, w0.y));
              w[g][t0 / 2 + 1] = h2_as_u32(__floats2half2_rn(w1.x, w1.y));
            }
          }
#pragma unroll
          for (int g = 0; g < NG; ++g) sm100::tmem_st_32x32b<PT / 2>(tS + g * NTOK + c * (PT / 2), w[g]);
        }
        };
        if (tok0 + NTOK - 1 > lim_lo || ok != (1 << NBLK) - 1 || !(v_hi <= kMaxSpread * v_lo))
          softmax_step(std::true_type{});
        else
          softmax_step(std::false_type{});
        sm100::mbar_arrive(bar(PAR_EMPTY + ps));
        sm100::tmem_st_wait();
        sm100::tc_fence_before();
        sm100::mbar_arrive(bar(P_READY + T));
      }
      if (!mine) continue;
      // ---- the rows' result ------------------------------------------------------------------
      if (sg.count > 0) {
        wait(O_FULL + T, nq & 1);
        ++nq;
        sm100::tc_fence_after();
      }
      const float2 lv = unpack2(l2);
      const float l = lv.x + lv.y;
      float pm[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float2 v = unpack2(pm2[g]);
        pm[g] = v.x + v.y;
      }
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      __half* op = a.out + (in ? (int64_t)tokq * a.o_ts + (int64_t)head * a.o_hs : 0);
      float* slot = a.part + (size_t)(cta * 2 + (sg.starts ? 1 : 0)) * (kRows * (D + 2));
      const int srow = T * 128 + rloc;
      // 32 channels at a time through the warp's rows of the Q tile, whose products are done,
      // so that eight lanes store a row's 128 (64) bytes
      const uint32_t mine_smem = qs_base + (warp & 3) * 4096;
      const uint32_t out_rows = __ballot_sync(0xffffffffu, in);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = 0;
        if (sg.count > 0) {
          sm100::tmem_ld_32x32b_x32(tO + 32 * c, o);
          sm100::tmem_ld_wait();
        }
        float m = pm[0];
#pragma unroll
        for (int g = 1; g < NG; ++g) m = c * 32 / GROUP == g ? pm[g] : m;
        const float mul = sg.whole ? inv : 1.f;
#pragma unroll
        for (int j = 0; j < 32; j += 4) {                // odd channels' codes entered times 2^-20
          float f[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            f[e] = fmaf(__uint_as_float(o[j + e]), (e & 1) ? 1048576.f : 16777216.f, m) * mul;
          sm100::st_shared_v4(mine_smem + swz(lane, j / 4), __float_as_uint(f[0]), __float_as_uint(f[1]),
                              __float_as_uint(f[2]), __float_as_uint(f[3]));
        }
        __syncwarp();
        const int ch = 32 * c + 4 * (lane & 7);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + lane / 8;
          const uint4 v = sm100::ld_shared_v4(mine_smem + swz(r, lane & 7));
          const __half* rp = reinterpret_cast<const __half*>(__shfl_sync(0xffffffffu, (unsigned long long)op, r));
          if (!sg.whole)
            *reinterpret_cast<uint4*>(slot + (size_t)(T * 128 + (warp & 3) * 32 + r) * D + ch) =
                v;
          else if ((out_rows >> r) & 1)
            *reinterpret_cast<uint2*>(const_cast<__half*>(rp) + ch) =
                make_uint2(h2_as_u32(__floats2half2_rn(__uint_as_float(v.x), __uint_as_float(v.y))),
                           h2_as_u32(__floats2half2_rn(__uint_as_float(v.z), __uint_as_float(v.w))));
        }
        __syncwarp();
      }
      if (!sg.whole) {
        slot[kRows * D + srow] = M;
        slot[kRows * D + kRows + srow] = l;
      }
      sm100::tc_fence_before();
    }
  } else if (warp < 12) {
    // ---- codes into operands ------------------------------------------------------------------
    sm100::setmaxnreg_dec<88>();
    const int i = tid - 256;
    int n = 0, kv = 0;                                   // steps, operand slots filled
    for (int u = u0; u < u1; u += it.steps - it.step, it.next<G_>(a)) {
      const Segment sg(it, a, u, u0, u1);
      for (int k = 0; k < sg.count; ++k, ++n) {
        const int rs = n % kRawStages, ps = n % kParStages;
        wait(RAW_FULL + rs, (n / kRawStages) & 1);
        const uint8_t* raw = smem + G_::OFF_RAW + rs * G_::RAW;
        // every load of the step's raw blocks first: K rows by quads of lanes (a phase of eight
        // lanes has rows r and r ^ 5, which meet neither in banks nor in swizzled chunks), V
        // in units of 8 tokens x D / 32 quads of channels (four runs of 8 tokens and two
        // quads in a phase)
        constexpr int KU = NTOK * 4 / 128;
        uint32_t kw[KU][D / 32], vw[4][D / 32];
        const int t = i & 3, pair = (i >> 3) & 3;
        const int tok_in = (i & 4) ? pair ^ 5 : pair;    // of the 8 tokens of an oct
#pragma unroll
        for (int x = 0; x < KU; ++x) {
          const int tok = ((i >> 5) + 4 * x) * 8 + tok_in;
          load_words<D / 32>(raw + (tok / 16) * BLK + (tok % 16) * (D / 2) + t * (D / 8), kw[x]);
        }
        const int run = (i & 3) + 4 * (i >> 5), h8 = (i >> 2) & 7;
        if (i < NTOK) {
          const uint8_t* src = raw + (run / 2) * BLK + kv4::off_v(D) + (run & 1) * 4 * D + h8 * (D / 8);
#pragma unroll
          for (int p = 0; p < 4; ++p) load_words<D / 32>(src + p * D, vw[p]);
        }
        // scales and minima as fp32, per group and token
        const int ptok = i / NG, pg = i % NG;
        const uint8_t* pblk = raw + (ptok / 16) * BLK;
        const float2 kp = __half22float2(reinterpret_cast<const __half2*>(pblk + kv4::off_kp(D))[(ptok % 16) * NG + pg]);
        const float2 vp = __half22float2(reinterpret_cast<const __half2*>(pblk + kv4::off_vp(D, GROUP))[(ptok % 16) * NG + pg]);
        const int ok = raw_ok[rs];
        sm100::mbar_arrive(bar(RAW_EMPTY + rs));         // all that is needed is in registers
        if (n >= kParStages) wait(PAR_EMPTY + ps, (n / kParStages - 1) & 1);
        {
          float* par = reinterpret_cast<float*>(smem + G_::OFF_PAR + ps * PAR);
          par[pg * NTOK + ptok] = kp.x, par[128 + pg * NTOK + ptok] = kp.y;
          par[256 + pg * NTOK + ptok] = vp.x, par[384 + pg * NTOK + ptok] = fmaf(8.f, vp.x, vp.y);
          float big = fmaxf(vp.x, 5.9604645e-8f);        // 2^-24, fp16's least scale
#pragma unroll
          for (int o = 1; o < NG; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
          if (pg == 0) par[512 + ptok] = lg2(big);
          // positive floats order as their bits
          const uint32_t hi = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
          const uint32_t lo = __reduce_min_sync(0xffffffffu, __float_as_uint(big));
          if (lane == 0) par[512 + NTOK + i / 32] = __uint_as_float(hi), par[516 + NTOK + i / 32] = __uint_as_float(lo);
          if (i == 0) par_ok[ps] = ok;
        }
        sm100::mbar_arrive(bar(PAR_FULL + ps));
        int slot = kv % kKvSlots;
        if (kv >= kKvSlots) wait(KV_EMPTY + slot, (kv / kKvSlots - 1) & 1);
        uint32_t dst = sbase + G_::OFF_KV + slot * G_::SLOT;
        // K: rows of tokens
#pragma unroll
        for (int x = 0; x < KU; ++x) {
          const int tok = ((i >> 5) + 4 * x) * 8 + tok_in;
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int o = 4 * j + t;                     // octet of the token's row
            const uint32_t w = kw[x][j], h = w >> 8;
            sm100::st_shared_v4(dst + (o / 8) * (NTOK * 128) + swz(tok, o & 7), w & kLoMask, w & kHiMask,
                                h & kLoMask, h & kHiMask);
          }
        }
        sm100::fence_proxy_async_smem();
        sm100::mbar_arrive(bar(KV_FULL + slot));
        ++kv;
        // V: rows of channels, codes less 8 (the odd ones times 16)
        auto lo = [](uint32_t w) { return hsub2_u32(w & kLoMask, 0x00080008u); };
        auto hi = [](uint32_t w) { return hsub2_u32(w & kHiMask, 0x00800080u); };
        slot = kv % kKvSlots;
        if (kv >= kKvSlots) wait(KV_EMPTY + slot, (kv / kKvSlots - 1) & 1);
        dst = sbase + G_::OFF_KV + slot * G_::SLOT + (run / 8) * (D * 128);
        if (i < NTOK) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const int ch = 4 * (8 * j + h8);             // first of the quad's channels
            const uint32_t a0 = vw[0][j], a1 = vw[1][j], a2 = vw[2][j], a3 = vw[3][j];
            sm100::st_shared_v4(dst + swz(ch, run & 7), lo(a0), lo(a1), lo(a2), lo(a3));
            sm100::st_shared_v4(dst + swz(ch + 1, run & 7), hi(a0), hi(a1), hi(a2), hi(a3));
            const uint32_t b0 = a0 >> 8, b1 = a1 >> 8, b2 = a2 >> 8, b3 = a3 >> 8;
            sm100::st_shared_v4(dst + swz(ch + 2, run & 7), lo(b0), lo(b1), lo(b2), lo(b3));
            sm100::st_shared_v4(dst + swz(ch + 3, run & 7), hi(b0), hi(b1), hi(b2), hi(b3));
          }
        }
        sm100::fence_proxy_async_smem();
        sm100::mbar_arrive(bar(KV_FULL + slot));
        ++kv;
      }
    }
  } else {
    sm100::setmaxnreg_dec<88>();
    if (warp == 12 && lane == 0) {
      // ---- MMA issue ---------------------------------------------------------------------------
      constexpr uint32_t idS = sm100::idesc_f16_f32(128, NTOK, 0, 0);
      constexpr uint32_t idO = sm100::idesc_f16_f32(128, GROUP, 0, 0);
      int kv = 0, np[2] = {0, 0}, nq[2] = {0, 0};
      bool live = true;
      // descriptors differ in their start address (low bits, in 16-byte units) only
      const uint64_t dq = sm100::umma_desc_sw128(sbase + G_::OFF_Q, 16, 1024);
      const uint64_t dkv = sm100::umma_desc_sw128(sbase + G_::OFF_KV, 16, 1024);
      auto issue_s = [&](int T, int slot) {
        const uint64_t q = dq + (uint32_t)(T * (G_::QTILE / 16)), kd = dkv + (uint32_t)(slot * (G_::SLOT / 16));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          sm100::umma_f16(tmem + T * 128 + (kk * 16 / GROUP) * NTOK, q + ((kk / 4) * (128 * 128) + (kk & 3) * 32) / 16,
                          kd + ((kk / 4) * (NTOK * 128) + (kk & 3) * 32) / 16, idS, kk * 16 % GROUP != 0);
        sm100::umma_commit(bar(S_FULL + T));
      };
      auto issue_o = [&](int T, int slot, bool first) {
        const uint64_t vd = dkv + (uint32_t)(slot * (G_::SLOT / 16));
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int kk = 0; kk < NTOK / 16; ++kk)
            sm100::umma_f16_ts(tmem + 256 + T * 128 + g * GROUP, tmem + T * 128 + g * NTOK + kk * 8,
                               vd + ((kk / 4) * (D * 128) + g * GROUP * 128 + (kk & 3) * 32) / 16, idO,
                               !first || kk != 0);
      };
      for (int u = u0; live && u < u1; u += it.steps - it.step, it.next<G_>(a)) {
        const Segment sg(it, a, u, u0, u1);
        if (sg.count == 0) continue;
        const int tiles = sg.two ? 2 : 1;
        // S of the first step
        if (!(live = wait(KV_FULL + kv % kKvSlots, (kv / kKvSlots) & 1))) break;
        for (int T = 0; T < tiles && live; ++T) {
          if (!(live = wait(Q_READY + T, nq[T] & 1))) break;
          ++nq[T];
          sm100::tc_fence_after();
          issue_s(T, kv % kKvSlots);
        }
        if (!live) break;
        sm100::umma_commit(bar(KV_EMPTY + kv % kKvSlots));
        ++kv;
        for (int k = 0; k < sg.count && live; ++k) {
          const int vs = kv % kKvSlots, vp = (kv / kKvSlots) & 1;
          ++kv;
          const int ks = kv % kKvSlots, kp = (kv / kKvSlots) & 1;
          const bool more = k + 1 < sg.count;
          if (!(live = wait(KV_FULL + vs, vp))) break;
          for (int T = 0; T < tiles; ++T) {
            if (!(live = wait(P_READY + T, np[T] & 1))) break;
            ++np[T];
            sm100::tc_fence_after();
            issue_o(T, vs, k == 0);
            if (T == tiles - 1) sm100::umma_commit(bar(KV_EMPTY + vs));
            if (more) {
              if (T == 0 && !(live = wait(KV_FULL + ks, kp))) break;
              sm100::tc_fence_after();
              issue_s(T, ks);
              if (T == tiles - 1) sm100::umma_commit(bar(KV_EMPTY + ks));
            } else {
              sm100::umma_commit(bar(O_FULL + T));
            }
          }
          if (more) ++kv;
        }
      }
      if (s_abort) {                                     // MMAs in flight finish before TMEM goes back
        sm100::umma_commit(bar(DRAIN));
        sm100::mbar_wait_bounded(bar(DRAIN), 0, nullptr, 100000000ull);
      }
    } else if (warp == 13) {
      // ---- cache blocks of a step: lane b copies block b ---------------------------------------
      const int bpp_shift = a.page_shift - 4;
      int n = 0;
      bool live = true;
      for (int u = u0; live && u < u1; u += it.steps - it.step, it.next<G_>(a)) {
        const Segment sg(it, a, u, u0, u1);
        auto page = [&](int k) {
          const int blk = (sg.k0 + k) * NBLK + lane;
          return lane < NBLK && k < sg.count && blk * 16 < it.vis
                     ? a.table[it.r * a.table_rs + (blk >> bpp_shift)] : -2;
        };
        int pid = page(0);
        for (int k = 0; k < sg.count; ++k, ++n) {
          const int rs = n % kRawStages;
          if (n >= kRawStages) live = wait(RAW_EMPTY + rs, (n / kRawStages - 1) & 1);
          live = __all_sync(0xffffffffu, live);
          if (!live) break;
          const bool have = pid >= 0 && pid < a.num_pages;
          if (pid != -2 && !have) atomicOr(a.status, kDevErrShape);
          const uint32_t ok = __ballot_sync(0xffffffffu, have);
          if (lane == 0) {
            raw_ok[rs] = (int)ok;
            sm100::mbar_arrive_expect_tx(bar(RAW_FULL + rs), __popc(ok) * BLK);
          }
          __syncwarp();
          if (have) {
            const int blk = (sg.k0 + k) * NBLK + lane;
            bulk_load(sbase + G_::OFF_RAW + rs * G_::RAW + lane * BLK,
                      a.cache + ((((int64_t)pid * a.kv_heads + it.h) << bpp_shift) +
                                 (blk & ((1 << bpp_shift) - 1))) * BLK,
                      BLK, bar(RAW_FULL + rs));
          }
          pid = page(k + 1);
        }
      }
      __syncwarp();
      if (lane == 0 && s_abort)                          // copies in flight land before the exit
        for (int k = max(0, n - kRawStages); k < n; ++k)
          sm100::mbar_wait_bounded(bar(RAW_FULL + k % kRawStages), (k / kRawStages) & 1, nullptr, 100000000ull);
    }
    __syncwarp();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  if (tid == 0) {
    // the item that starts here and goes on in the next CTAs, if there is one
    int* d = a.desc + cta * kDescInts;
    int span = 0;
    Item x = s_first;
    for (int u = u0; u < u1; u += x.steps - x.step, x.next<G_>(a)) {
      const Segment sg(x, a, u, u0, u1);
      if (!sg.whole && sg.starts) {
        const int end = u - x.step + max(1, x.steps - kItemSteps);     // past the last step with tokens
        span = (int)(((double)end * ctas - 1.0) / U) - cta + 1;
        d[1] = x.q0, d[2] = x.rt * kRows, d[3] = x.n * a.G, d[4] = x.h;
      }
    }
    d[0] = span;
  }
  if (warp == 0) sm100::tmem_dealloc(tmem, 512);
}

// Joins an item that crosses CTAs: block (c, y) takes rows [8 y, 8 y + 8) of the item that
// starts in CTA c, over the slots of CTAs c .. c + span - 1, a warp a row.  Lanes read 32
// parts' statistics at once and then their channels of one part after the other; the loads of
// eight parts are under way together (latency is all this kernel costs).
template <int D>
__global__ void __launch_bounds__(256) kv4_prefill_merge(const AttnArgs a) {
  sm100::grid_dependency_wait();
  const int cta = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
  const int* d = a.desc + cta * kDescInts;
  const int span = d[0];
  if (span == 0) return;
  const int r = blockIdx.y * 8 + tid / 32, ch = lane * (D / 32), row = d[2] + r;
  if (row >= d[3]) return;
  constexpr size_t kSlot = (size_t)kRows * (D + 2);
  auto part = [&](int k) { return a.part + (size_t)((cta + k) * 2 + (k == 0)) * kSlot; };
  float m = -CUDART_INF_F;
  for (int k = lane; k < span; k += 32) m = fmaxf(m, part(k)[kRows * D + r]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float o[D / 32] = {}, l = 0.f;
  for (int k0 = 0; k0 < span; k0 += 32) {
    float f = 0.f;
    if (k0 + lane < span) {
      const float* p = part(k0 + lane);
      const float mk = p[kRows * D + r];
      f = mk == m ? 1.0f : ex2(mk - m);
      l = fmaf(f, p[kRows * D + kRows + r], l);
    }
    const int n = min(32, span - k0);
#pragma unroll 8
    for (int k = 0; k < n; ++k) {
      const float* p = part(k0 + k) + (size_t)r * D + ch;
      const float fk = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
      for (int j = 0; j < D / 32; j += 2) {
        const float2 v = *reinterpret_cast<const float2*>(p + j);
        o[j] = fmaf(fk, v.x, o[j]), o[j + 1] = fmaf(fk, v.y, o[j + 1]);
      }
    }
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __half* op = a.out + (int64_t)(d[1] + row / a.G) * a.o_ts + (int64_t)(d[4] * a.G + row % a.G) * a.o_hs + ch;
#pragma unroll
  for (int j = 0; j < D / 32; j += 2)
    *reinterpret_cast<__half2*>(op + j) = __floats2half2_rn(o[j] * inv, o[j + 1] * inv);
}

template <int D, int GROUP>
cudaError_t launch_geo(const AttnArgs& a, int num_sms, cudaStream_t stream) {
  using G_ = Geo<D, GROUP>;
  static PerDeviceOnce attr_once;
  const cudaError_t attr = attr_once.run([] {
    return cudaFuncSetAttribute(kv4_prefill_kernel<G_>, cudaFuncAttributeMaxDynamicSharedMemorySize, G_::SMEM);
  });
  if (attr != cudaSuccess) return attr;
  kv4_prefill_kernel<G_><<<num_sms, kThreads, G_::SMEM, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv4_prefill(const kv4::AttnArgs& a, int head_dim, int group, int num_sms,
                               cudaStream_t stream) {
  if (head_dim == 64 && group == 32) return launch_geo<64, 32>(a, num_sms, stream);
  if (head_dim == 64 && group == 64) return launch_geo<64, 64>(a, num_sms, stream);
  if (head_dim == 128 && group == 32) return launch_geo<128, 32>(a, num_sms, stream);
  if (head_dim == 128 && group == 64) return launch_geo<128, 64>(a, num_sms, stream);
  if (head_dim == 128 && group == 128) return launch_geo<128, 128>(a, num_sms, stream);
  return cudaErrorInvalidValue;
}

cudaError_t launch_kv4_prefill_merge(const kv4::AttnArgs& a, int head_dim, int num_sms, cudaStream_t stream) {
  return kv4::launch_overlapped(head_dim == 64 ? kv4_prefill_merge<64> : kv4_prefill_merge<128>,
                                dim3(num_sms, kRows / 8), 256, 0, stream, a);
}

}  // namespace awq
