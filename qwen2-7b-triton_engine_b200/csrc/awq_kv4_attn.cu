// awq_kv4_attn.cu -- attention over the paged 4-bit key/value cache.
//
// Query row (i, h) of a request with L cached tokens and n query tokens sees the tokens
// t <= L - n + i:  o = sum_t softmax_t(scale q . k_t) v_t,  k_t = c s + m per channel group.
// Nothing is dequantized: with integer codes c,
//   scale q . k_t = scale sum_G ( s_tG (q_G . c_tG) + m_tG sum(q_G) )
//   o_G = ( sum_t (p_t s_tG) (c_tG - 8) + sum_t p_t (m_tG + 8 s_tG) ) / sum_t p_t
// so the tensor cores multiply fp16 queries, and fp16 weights p s, with the codes (fp16
// subnormals, one AND per two codes), and scales and minima are applied per token in fp32.
// The values' codes are taken from the middle of their range: against the mean of many values
// sum p s c is large and almost cancels sum p m, and the weights' rounding and the tensor
// cores' truncated sums would stay behind (0.06 % instead of 0.03 % of the result at 1000 tokens,
// 0.15 % at 8000).
// The odd codes of a word sit four bits higher, times 2^-20; the queries they meet are scaled
// by 1/16 for it, after an item's queries are scaled up together by a power of two so that
// the largest lies just below fp16's limit and nothing that matters becomes subnormal.  Of the
// values' codes one product takes the even ones and one whole bytes, even + 16 odd (each less
// 8); the odd sum is their difference over 16, exact to fp32's rounding.
// The softmax reference M runs over log2(p s) rather than log2(p), and lies 2^7 below the
// largest, so that the fp16 weights stay below 2^15 and near the top of the range whatever the
// size of the value scales (s is a token's largest: groups with scales up to 2^21 below it keep
// all bits of their weights); sums, statistics and accumulators are fp32.
//
// Operand order: scores are computed transposed (tokens are the MMA's 16 rows, the query
// rows of a kv head its 8 columns), as are the outputs (channels x query rows), so seven
// query heads of a group waste one column in eight instead of nine rows in sixteen.
//
// Work split (kv4_attn_kernel): the (request, kv head, 8 query rows) items are cut into tiles
// of 64 tokens, and the linear list of all tiles is dealt evenly to all warps of one CTA per
// SM; ragged batches balance to within a tile.  Every item has one empty tile more, which
// stands for its fixed cost.  A warp reads its tiles from a ring of its own; one more warp
// fills all rings with bulk copies, each of its lanes one (no CTA barrier in the loop).  Items
// that cross warps are joined in the CTA at its end; items that cross CTAs by
// kv4_merge_kernel, in CTA order, so results do not depend on timing.
//
// Bound: for large batches the instructions of the 11 warps an SM's registers hold (45 % of the
// issue slots, start and joins included; unpacking goes through the half-rate logic pipe, 31 %)
// and then the cache's bytes, for few tokens latency.  Measured on
// B200, 48 requests of 1 to 16384 tokens, 28 / 4 heads of 128 channels in groups of 64: 51 us
// (176 MB, 3.5 TB/s, 53 % of a copy's rate; 47.6 us before the values' codes were centred); 64-token tiles start within 4 us and the joins take
// 6.  One request of 1000 tokens: 12.5 us.
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

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// N words of shared memory (plain loads: the compiler schedules them and the MMAs freely
// between the barrier wait and the refill).
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// 2^x of the softmax: 2 ulp, results below 2^-126 are 0 (they are below 2^-100 of the sum).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
      ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

constexpr int kRows = 8;                               // query rows of an item

template <int D_, int GROUP_, int TB_, int WARPS_>
struct Geo {
  static constexpr int TB = TB_, TOKENS = 16 * TB_;    // blocks and tokens of a tile
  static constexpr int D = D_, GROUP = GROUP_, WARPS = WARPS_;
  static constexpr int THREADS = (WARPS + 1) * 32;     // and the producer warp
  static constexpr int NG = D / GROUP, W = D / 32, ROWS = kRows;
  static constexpr int BLK = kv4::block_bytes(D, GROUP), TILE = TB * BLK;
  static constexpr int BUDGET = 227 * 1024 - (kPrefixEntries + 8) * 4 - 5120;
  static constexpr int FIT = BUDGET / (WARPS * TILE);
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int SLOT = ROWS * (D + 2);          // floats: O [ROWS][D], M, l
  static constexpr int OFF_PRE = WARPS * STAGES * TILE;
  static constexpr int OFF_BAR = OFF_PRE + (kPrefixEntries + 8) * 4 / 16 * 16;
  static constexpr int OFF_META = OFF_BAR + WARPS * STAGES * 16;
  static constexpr int OFF_ENT = (OFF_META + WARPS * STAGES * 4 + 15) / 16 * 16;
  // join: the parts' factors per column, and M and l of their sum
  static constexpr int OFF_WGT = OFF_ENT + WARPS * 2 * 40;
  static constexpr int SMEM = OFF_WGT + (WARPS * 2 + 2) * ROWS * 4;
  static_assert(STAGES >= 2 && SLOT * 4 <= STAGES * TILE && SMEM <= 227 * 1024, "shared memory");
  static_assert(2 * WARPS <= 32 && WARPS * STAGES <= THREADS, "one lane per part, one thread per barrier");
};

// One request as the work split sees it.
struct Req {
  int L, n, q0, tiles, nrt;
};
template <class G_>
__device__ __forceinline__ Req request(const AttnArgs& a, int r) {
  Req x;
  const int cap = (int)min((long long)a.width << a.page_shift, 0x7fffff00LL);
  const int len = a.lens[r];
  x.L = min(max(len, 0), cap);
  if (len != x.L) atomicOr(a.status, kDevErrShape);
  if (a.cu_q) {
    const int b = a.cu_q[r], e = a.cu_q[r + 1];
    const bool ok = b >= 0 && e >= b && e <= a.tokens;
    if (!ok) atomicOr(a.status, kDevErrShape);
    x.q0 = ok ? b : 0;
    x.n = ok ? e - b : 0;
  } else {
    x.q0 = r;
    x.n = 1;
  }
  if ((long long)x.n * a.G >= a.min_rows) x.n = 0;      // the prefill kernel's request
  x.tiles = (x.L + G_::TOKENS - 1) / G_::TOKENS + 1;
  x.nrt = (x.n * a.G + G_::ROWS - 1) / G_::ROWS;
  return x;
}

// A position in the list of tiles: request, kv head, tile of query rows, tile of tokens.
struct Cursor {
  Req x;
  int r, h, rt, tile;
  int vis;      // tokens the last query row of the row tile sees

  template <class G_>
  __device__ bool has_tokens() const { return tile * G_::TOKENS < vis; }

  template <class G_>
  __device__ void set_vis(const AttnArgs& a) {
    const int last = min(x.n - 1, ((rt + 1) * G_::ROWS - 1) / a.G);
    vis = max(0, x.L - x.n + last + 1);
  }
  template <class G_>
  __device__ void locate(const AttnArgs& a, const int* pre, int u) {
    const int shift = kv4::prefix_shift(a);
    int lo = 0, hi = (a.R + (1 << shift) - 1) >> shift;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u) lo = mid; else hi = mid;
    }
    int rem = u - pre[lo];
    r = lo << shift;
    for (;;) {
      x = request<G_>(a, r);
      const int units = a.kv_heads * x.nrt * x.tiles;
      if (rem < units || r + 1 >= a.R) break;
      rem -= units;
      ++r;
    }
    const int item = rem / x.tiles;
    tile = rem - item * x.tiles;
    h = item / x.nrt;
    rt = item - h * x.nrt;
    set_vis<G_>(a);
  }
  template <class G_>
  __device__ void next_item(const AttnArgs& a) {
    tile = 0;
    if (++rt == x.nrt) {
      rt = 0;
      if (++h == a.kv_heads) {
        h = 0;
        do {
          if (++r >= a.R) return;
          x = request<G_>(a, r);
        } while (x.nrt == 0);
      }
    }
    set_vis<G_>(a);
  }
};

struct Entry {          // a part of an item, for the join at the CTA's end
  int ib, ie;           // the item's tiles in the list
  int q0, row0, rows, h;
  const float* ptr;     // slot, or null
  long long pad;
};
static_assert(sizeof(Entry) == 40, "entry size");

template <class G_>
__global__ void __launch_bounds__(G_::THREADS, 1) kv4_attn_kernel(const AttnArgs a) {
  constexpr int D = G_::D, NG = G_::NG, W = G_::W, ROWS = G_::ROWS;
  constexpr int TB = G_::TB, TOKENS = G_::TOKENS, THREADS = G_::THREADS;
  constexpr int WARPS = G_::WARPS, STAGES = G_::STAGES, BLK = G_::BLK, TILE = G_::TILE;
  constexpr int GW = W / NG;                           // words (32 channels) per group
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t sbase = sm100::smem_u32(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane / 4, t = lane & 3;
  int* pre = reinterpret_cast<int*>(smem + G_::OFF_PRE);
  int* meta = reinterpret_cast<int*>(smem + G_::OFF_META);     // [warp][stage] blocks that arrive
  Entry* ent = reinterpret_cast<Entry*>(smem + G_::OFF_ENT);
  const uint32_t bars = sbase + G_::OFF_BAR;           // [warp][stage] full, empty
  __shared__ volatile int s_abort;                     // a wait ran out: everyone stops

  if (tid < WARPS * STAGES) {
    sm100::mbar_init(bars + 16 * tid, 1);
    sm100::mbar_init(bars + 16 * tid + 8, 1);
    sm100::fence_mbar_init();
  }
  if (tid < 2 * WARPS) ent[tid].ptr = nullptr;

  if (tid == 0) s_abort = 0;
  const int U = kv4::scan_units<THREADS>(a, pre, [&](int r) {
    const Req x = request<G_>(a, r);
    return a.kv_heads * x.nrt * x.tiles;
  });
  const int ctas = min((int)gridDim.x, (U + WARPS - 1) / WARPS);
  const int cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) a.desc[cta * kDescInts] = 0;
    sm100::grid_dependency_wait();
    return;
  }
  // unit ranges: warp w of all Wt starts at floor(U w / Wt)
  const int Wt = ctas * WARPS, uq = U / Wt, ur = U - uq * Wt;
  auto first_unit = [&](int w) { return uq * w + ur * w / Wt; };

  if (warp == WARPS) {
    // ---- producer warp: lane i fills warp i's ring, all rings in step ---------------------
    if (lane < WARPS) {
      const int u1 = first_unit(cta * WARPS + lane + 1);
      int next = first_unit(cta * WARPS + lane);        // unit of lc
      const int bpp_shift = a.page_shift - 4;
      const int run_shift = min(bpp_shift, TB == 4 ? 2 : 1);   // blocks of a tile in one page
      const uint32_t ring = sbase + lane * STAGES * TILE;
      const uint32_t bar0 = bars + lane * STAGES * 16;
      Cursor lc = {};
      int copied = 0, pid = -1;
      auto settle = [&]() {                             // to the next tile that holds tokens
        while (next < u1 && !lc.has_tokens<G_>()) {
          if (++next < u1 && ++lc.tile == lc.x.tiles) lc.next_item<G_>(a);
        }
        if (next < u1) pid = a.table[lc.r * a.table_rs + ((lc.tile * TB) >> bpp_shift)];
      };
      if (next < u1) lc.locate<G_>(a, pre, next);
      settle();
      uint64_t t0 = sm100::globaltimer_ns();
      while (next < u1 && !s_abort) {
        const int s = copied % STAGES;
        if (copied >= STAGES && !sm100::mbar_test_wait(bar0 + 16 * s + 8, (copied / STAGES - 1) & 1)) {
          if (sm100::globaltimer_ns() - t0 > 2000000000ull) {
            atomicOr(a.status, kDevErrBarrierTimeout);
            s_abort = 1;
          }
          continue;
        }
        const int blk0 = lc.tile * TB;
        const int nb = min(TB, (lc.vis + kv4::kBlockTokens - 1) / kv4::kBlockTokens - blk0);
        const uint32_t dst = ring + s * TILE, bar = bar0 + 16 * s;
        int ok = 0;
        for (int b = 0; b < nb; b += 1 << run_shift) {  // a tile in one page takes one round
          if (b > 0) pid = a.table[lc.r * a.table_rs + ((blk0 + b) >> bpp_shift)];
          const int n = min(1 << run_shift, nb - b);
          if (pid < 0 || pid >= a.num_pages) {
            atomicOr(a.status, kDevErrShape);
            continue;
          }
          ok |= ((1 << n) - 1) << b;
          const int at = (blk0 + b) & ((1 << bpp_shift) - 1);
          sm100::mbar_expect_tx(bar, n * BLK);
          bulk_load(dst + b * BLK,
                    a.cache + ((((int64_t)pid * a.kv_heads + lc.h) << bpp_shift) + at) * BLK, n * BLK, bar);
        }
        meta[lane * STAGES + s] = ok;
        sm100::mbar_arrive(bar);
        ++copied;
        if (++next < u1 && ++lc.tile == lc.x.tiles) lc.next_item<G_>(a);
        settle();
        t0 = sm100::globaltimer_ns();
      }
      if (s_abort)                                       // copies in flight land before the exit
        for (int k = max(0, copied - STAGES); k < copied; ++k)
          sm100::mbar_wait_bounded(bar0 + 16 * (k % STAGES), (k / STAGES) & 1, nullptr, 100000000ull);
    }
    __syncwarp();
  } else if (first_unit(cta * WARPS + warp) < first_unit(cta * WARPS + warp + 1)) {
    const int u0 = first_unit(cta * WARPS + warp), u1 = first_unit(cta * WARPS + warp + 1);
    const uint8_t* stage0 = smem + warp * STAGES * TILE;
    const uint32_t bar0 = bars + warp * STAGES * 16;
    Cursor cc = {};
    cc.locate<G_>(a, pre, u0);
    bool dead = false;
    int u = u0, use = 0, phase = 0;                     // use: the stage to read next
    while (u < u1) {
      // ---- one item, or this warp's part of it ----------------------------------------
      const int rows = cc.x.n * a.G, row0 = cc.rt * ROWS;
      const int ib = u - cc.tile, ie = ib + cc.x.tiles, ue = min(u1, ie);
      uint32_t qa[W][2], qb[W][2];              // B operands: even / odd nibbles
      float qs[NG][2];                              // scale * sum of q over the group
      int lim[2];                                   // last visible token of the columns
      uint4 qv[W];
      float big = 0.f;
      const int row = row0 + g;
      const bool in = row < rows;
      const __half* qp = a.q + (in ? (int64_t)(cc.x.q0 + row / a.G) * a.q_ts +
                                         (int64_t)(cc.h * a.G + row % a.G) * a.q_hs
                                   : 0);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        qv[j] = make_uint4(0, 0, 0, 0);
        if (in) qv[j] = *reinterpret_cast<const uint4*>(qp + 8 * (4 * j + t));
      }
      float sum[NG] = {};
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint32_t w4[4] = {qv[j].x, qv[j].y, qv[j].z, qv[j].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(u32_as_h2(w4[k]));
          sum[j / GW] += f.x + f.y;
          big = fmaxf(big, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
#pragma unroll
      for (int k = 0; k < NG; ++k) {
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
        sum[k] *= a.scale_log2;
        qs[k][0] = __shfl_sync(0xffffffffu, sum[k], 8 * t);
        qs[k][1] = __shfl_sync(0xffffffffu, sum[k], 8 * t + 4);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
        lim[c] = cc.x.L - cc.x.n + (row0 + 2 * t + c) / a.G;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
      // 2^(15 - e) for the largest |q| in [2^e, 2^(e + 1)); 1 for zeros and infinities
      const int e_big = (int)(__float_as_uint(big) >> 23) - 127;
      const int up2 = big > 0.f && e_big <= 15 ? 15 - e_big : 0;
      const float qmul = __uint_as_float((uint32_t)(127 + up2) << 23);
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint4 v = qv[j];
        const uint32_t even[2] = {__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.y, v.w, 0x5410)};
        const uint32_t odd[2] = {__byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x7632)};
#pragma unroll
        for (int k = 0; k < 2; ++k) {                    // channels (0, 4), (2, 6); (1, 5), (3, 7)
          const float2 e = __half22float2(u32_as_h2(even[k])), o = __half22float2(u32_as_h2(odd[k]));
          qa[j][k] = h2_as_u32(__floats2half2_rn(e.x * qmul, e.y * qmul));
          qb[j][k] = h2_as_u32(__floats2half2_rn(o.x * (qmul * 0.0625f), o.y * (qmul * 0.0625f)));
        }
      }
      const int lim_all = cc.x.L - cc.x.n + row0 / a.G;  // every row sees tokens up to here
      // codes enter the MMA times 2^-24, queries times qmul
      const float ksc = a.scale_log2 * 16777216.0f * __uint_as_float((uint32_t)(127 - up2) << 23);
      float O[2 * W][4] = {}, M[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {}, pm[NG][2] = {};

      // One tile; EDGE: some of its tokens may be unseen (past a row's limit, or in a page the
      // table does not name).
      auto tile = [&](auto edge, const uint8_t* st, int tok0, int ok) {
        constexpr bool EDGE = decltype(edge)::value;
        auto unseen = [&](int b, int e, int c) {  // token g + 8 e of block b, column c
          return tok0 + b * 16 + g + e * 8 > lim[c] || !((ok >> b) & 1);
        };
        float x[TB][4];                         // [block][token g / g + 8, column]
        float ls[TB][2];                        // log2 of a token's largest value scale
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const uint8_t* blk = st + b * BLK;
          uint32_t k0[W], k1[W], p0[NG], p1[NG];
          load_words<W>(blk + g * (D / 2) + t * (4 * W), k0);
          load_words<W>(blk + (g + 8) * (D / 2) + t * (4 * W), k1);
          load_words<NG>(blk + kv4::off_kp(D) + g * (4 * NG), p0);
          load_words<NG>(blk + kv4::off_kp(D) + (g + 8) * (4 * NG), p1);
#pragma unroll
          for (int k = 0; k < NG; ++k) {
            const float2 f0 = __half22float2(u32_as_h2(p0[k])), f1 = __half22float2(u32_as_h2(p1[k]));
            const float s0 = f0.x * ksc, s1 = f1.x * ksc;
            float acc[4];
#pragma unroll
            for (int j = k * GW; j < (k + 1) * GW; ++j) {
              // x >> 8 as the high half of x 2^24: the multiplier has room, the logic pipe not
              const uint32_t h0 = __umulhi(k0[j], 1u << 24), h1 = __umulhi(k1[j], 1u << 24);
              if (j == k * GW)
                mma16816_first(acc, k0[j] & kLoMask, k1[j] & kLoMask, h0 & kLoMask, h1 & kLoMask,
                               qa[j][0], qa[j][1]);
              else
                mma16816(acc, k0[j] & kLoMask, k1[j] & kLoMask, h0 & kLoMask, h1 & kLoMask,
                         qa[j][0], qa[j][1]);
              mma16816(acc, k0[j] & kHiMask, k1[j] & kHiMask, h0 & kHiMask, h1 & kHiMask,
                       qb[j][0], qb[j][1]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float m = i < 2 ? f0.y : f1.y, q1 = qs[k][i & 1];
              const float base = k == 0 ? m * q1 : fmaf(m, q1, x[b][i]);
              x[b][i] = fmaf(acc[i], i < 2 ? s0 : s1, base);
            }
          }
          if constexpr (EDGE) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (unseen(b, i / 2, i & 1)) x[b][i] = -CUDART_INF_F;
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t pv[NG];
            load_words<NG>(blk + kv4::off_vp(D, G_::GROUP) + (g + 8 * e) * (4 * NG), pv);
            float top = 5.9604645e-8f;                   // 2^-24, fp16's least scale
#pragma unroll
            for (int k = 0; k < NG; ++k) top = fmaxf(top, __low2float(u32_as_h2(pv[k])));
            ls[b][e] = lg2(top);
          }
        }
        // the softmax reference moves only when it is more than 2^8 behind (kBelowTop);
        // -inf + 8 = -inf, so the first visible token sets it
        bool up = false;
        float nm[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = fmaxf(x[0][c] + ls[0][0], x[0][2 + c] + ls[0][1]);
#pragma unroll
          for (int b = 1; b < TB; ++b)
            m = fmaxf(m, fmaxf(x[b][c] + ls[b][0], x[b][2 + c] + ls[b][1]));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          nm[c] = m - kv4::kBelowTop;
          up |= nm[c] > M[c] + kv4::kMoveAt;
        }
        if (__any_sync(0xffffffffu, up)) {
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float m = fmaxf(M[c], nm[c]);
            f[c] = M[c] == m ? 1.0f : ex2(M[c] - m);
            M[c] = m;
            l[c] *= f[c];
#pragma unroll
            for (int k = 0; k < NG; ++k) pm[k][c] *= f[c];
          }
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) {
            O[i][0] *= f[0], O[i][1] *= f[1];
            O[i][2] *= f[0], O[i][3] *= f[1];
          }
        }
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const uint8_t* blk = st + b * BLK;
          uint32_t wb[NG][2];                            // B operands: weights p s per group
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t pv[NG];
            load_words<NG>(blk + kv4::off_vp(D, G_::GROUP) + (g + 8 * e) * (4 * NG), pv);
            float p[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              p[c] = ex2(x[b][2 * e + c] - (EDGE && M[c] == -CUDART_INF_F ? 0.f : M[c]));
              l[c] += p[c];
            }
#pragma unroll
            for (int k = 0; k < NG; ++k) {
              const float2 f = __half22float2(u32_as_h2(pv[k]));
              const float mid = fmaf(8.f, f.x, f.y);
              float w[2];
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                // an unseen token's scale and minimum may be anything: no 0 * NaN (a seen
                // one's weight may be 0 as well, and its NaN counts)
                const bool seen = !EDGE || !unseen(b, e, c);
                w[c] = seen ? p[c] * f.x : 0.f;
                pm[k][c] = seen ? fmaf(p[c], mid, pm[k][c]) : pm[k][c];
              }
              wb[k][e] = movmatrix(h2_as_u32(__floats2half2_rn(w[0], w[1])));
            }
          }
          // c - 8, and (c_even - 8) + 16 (c_odd - 8), as fp16 subnormals
          auto even = [](uint32_t v) { return hsub2_u32(v & kLoMask, 0x00080008u); };
          auto both = [](uint32_t v) { return hsub2_u32(v, 0x00880088u); };
          uint32_t v0[W], v1[W];
          load_words<W>(blk + kv4::off_v(D) + t * D + g * (4 * W), v0);
          load_words<W>(blk + kv4::off_v(D) + (t + 4) * D + g * (4 * W), v1);
#pragma unroll
          for (int i = 0; i < W; ++i) {
            // bytes: code p in the low nibble, code p + 1 in the high one
            const uint32_t a0 = __byte_perm(v0[i], 0, 0x4240), a1 = __byte_perm(v0[i], 0, 0x4341);
            const uint32_t a2 = __byte_perm(v1[i], 0, 0x4240), a3 = __byte_perm(v1[i], 0, 0x4341);
            mma16816(O[2 * i], even(a0), even(a1), even(a2), even(a3), wb[i / GW][0], wb[i / GW][1]);
            mma16816(O[2 * i + 1], both(a0), both(a1), both(a2), both(a3), wb[i / GW][0], wb[i / GW][1]);
          }
        }
      };

      for (; u < ue; ++u, ++cc.tile) {
        if (dead || !cc.has_tokens<G_>()) continue;
        const bool got = sm100::mbar_wait_bounded(bar0 + 16 * use, phase, a.status);
        dead = __any_sync(0xffffffffu, !got);            // one verdict for the whole warp
        if (dead) {
          s_abort = 1;
          continue;
        }
        const int tok0 = cc.tile * TOKENS;
        const int ok = *(volatile int*)(meta + warp * STAGES + use);
        if (tok0 + TOKENS - 1 > lim_all || ok != (1 << TB) - 1)
          tile(std::true_type{}, stage0 + use * TILE, tok0, ok);
        else
          tile(std::false_type{}, stage0 + use * TILE, tok0, ok);
        __syncwarp();                                    // the stage is read: it may be refilled
        if (lane == 0) sm100::mbar_arrive(bar0 + 16 * use + 8);
        if (++use == STAGES) use = 0, phase ^= 1;
      }

      // ---- the item's (part's) result ---------------------------------------------------
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
#pragma unroll
          for (int k = 0; k < NG; ++k) pm[k][c] += __shfl_xor_sync(0xffffffffu, pm[k][c], o);
        }
      }
      const bool whole = ib >= u0 && ie <= u1;
      float* slot = nullptr;
      if (!whole) {
        slot = ue == u1 ? reinterpret_cast<float*>(smem + warp * STAGES * TILE)
                        : a.warp_part + (size_t)(cta * WARPS + warp) * G_::SLOT;
        __syncwarp();
        if (lane == 0) {
          Entry& e = ent[2 * warp + (ue == u1)];
          e.ib = ib, e.ie = ie, e.q0 = cc.x.q0, e.row0 = row0, e.rows = rows, e.h = cc.h;
          e.ptr = slot;
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int col = 2 * t + c, row = row0 + col;
        const float inv = l[c] == 0.f ? 0.f : 1.0f / l[c];
        __half* op = nullptr;
        if (whole && row < rows)
          op = a.out + (int64_t)(cc.x.q0 + row / a.G) * a.o_ts + (int64_t)(cc.h * a.G + row % a.G) * a.o_hs;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float m = pm[i / GW][c];
          // 2 i: even codes less 8; 2 i + 1: those + 16 (odd codes less 8)
          const float e0 = O[2 * i][c], e1 = O[2 * i][2 + c];
          const float4 v = make_float4(fmaf(e0, 16777216.f, m),
                                       fmaf(O[2 * i + 1][c] - e0, 1048576.f, m),
                                       fmaf(e1, 16777216.f, m),
                                       fmaf(O[2 * i + 1][2 + c] - e1, 1048576.f, m));
          if (slot) {
            *reinterpret_cast<float4*>(slot + col * D + 32 * i + 4 * g) = v;
          } else if (op) {
            *reinterpret_cast<uint2*>(op + 32 * i + 4 * g) =
                make_uint2(h2_as_u32(__floats2half2_rn(v.x * inv, v.y * inv)),
                           h2_as_u32(__floats2half2_rn(v.z * inv, v.w * inv)));
          }
        }
        if (slot && g == 0) {
          slot[ROWS * D + col] = M[c];
          slot[ROWS * D + ROWS + col] = l[c];
        }
      }
      if (u < u1) cc.next_item<G_>(a);
    }
  }
  sm100::grid_launch_dependents();
  __syncthreads();

  // ---- join the items that cross this CTA's warps, in order ------------------------------
  // Lane k of every warp looks at part k (two per warp, in tile order); the parts of one item
  // are neighbours.
  const int cs = first_unit(cta * WARPS), ce = first_unit((cta + 1) * WARPS);
  float* wgt = reinterpret_cast<float*>(smem + G_::OFF_WGT);    // [part][column] factors
  float* tot = wgt + 2 * WARPS * ROWS;                          // [column] M, l of the sum
  const bool mine = lane < 2 * WARPS && ent[lane < 2 * WARPS ? lane : 0].ptr;
  const int my_ib = mine ? ent[lane].ib : -1;
  const float* my_ptr = mine ? ent[lane].ptr : nullptr;
  uint32_t left = __ballot_sync(0xffffffffu, mine);
  int span = 0;
  Entry head = {};
  while (left) {
    const int lead = __ffs(left) - 1;
    const int lead_ib = __shfl_sync(0xffffffffu, my_ib, lead);
    const uint32_t group = __ballot_sync(0xffffffffu, mine && my_ib == lead_ib);
    left &= ~group;
    const Entry e0 = ent[lead];
    const bool in = (group >> lane) & 1;
    // factors 2^(M_k - M) and the sum of l: warp w makes the columns w, w + WARPS + 1, ...
    for (int col = warp; col < ROWS; col += WARPS + 1) {
      const float mk = in ? my_ptr[ROWS * D + col] : -CUDART_INF_F;
      float m = mk;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float f = mk == m ? 1.0f : ex2(mk - m);
      float l = in ? f * my_ptr[ROWS * D + ROWS + col] : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (in) wgt[lane * ROWS + col] = f;
      if (lane == 0) tot[2 * col] = m, tot[2 * col + 1] = l;
    }
    __syncthreads();
    const bool done = e0.ib >= cs && e0.ie <= ce;
    float* slot = a.part + (size_t)(cta * 2 + (e0.ib < cs ? 0 : 1)) * G_::SLOT;
    if (!done && e0.ib >= cs) {                          // the item starts here and goes on
      // the last warp that starts at or before the item's last tile (exact in double)
      const int w = (int)(((double)e0.ie * Wt - 1.0) / U);
      span = w / WARPS - cta + 1;
      head = e0;
    }
    for (int idx = tid; idx < ROWS * (D / 4); idx += THREADS) {
      const int col = idx / (D / 4), ch = (idx - col * (D / 4)) * 4, row = e0.row0 + col;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t rest = group; rest; rest &= rest - 1) {
        const int k = __ffs(rest) - 1;
        const float f = wgt[k * ROWS + col];
        const float4 v = *reinterpret_cast<const float4*>(ent[k].ptr + col * D + ch);
        o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y);
        o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
      }
      const float m = tot[2 * col], l = tot[2 * col + 1];
      if (done) {
        if (row < e0.rows) {
          const float inv = l == 0.f ? 0.f : 1.0f / l;
          __half* op = a.out + (int64_t)(e0.q0 + row / a.G) * a.o_ts + (int64_t)(e0.h * a.G + row % a.G) * a.o_hs;
          *reinterpret_cast<uint2*>(op + ch) = make_uint2(h2_as_u32(__floats2half2_rn(o.x * inv, o.y * inv)),
                                                          h2_as_u32(__floats2half2_rn(o.z * inv, o.w * inv)));
        }
      } else {
        *reinterpret_cast<float4*>(slot + col * D + ch) = o;
        if (ch == 0) slot[ROWS * D + col] = m, slot[ROWS * D + ROWS + col] = l;
      }
    }
    if (left) __syncthreads();                           // the factors are free again
  }
  if (tid == 0) {
    int* d = a.desc + cta * kDescInts;
    d[0] = span, d[1] = head.q0, d[2] = head.row0, d[3] = head.rows, d[4] = head.h;
  }
  // The tcgen05 kernel may still run: this one has not ended before it, so that whoever waits
  // for this one has waited for both.
  sm100::grid_dependency_wait();
}

// Joins an item that crosses CTAs: block (c, col) sums column col of the item that starts in
// CTA c, over the slots of CTAs c .. c + span - 1, in four (eight) interleaved groups.  Latency
// is its cost: 2 us behind the attention kernel's end, whose tail hides the launch.
template <int D>
__global__ void __launch_bounds__(128) kv4_merge_kernel(const AttnArgs a) {
  constexpr int LANES = D / 4, GROUPS = 128 / LANES;
  __shared__ float s_m[4], s_l[GROUPS];
  __shared__ float4 s_o[GROUPS][LANES];
  sm100::grid_launch_dependents();
  sm100::grid_dependency_wait();
  const int cta = blockIdx.x, col = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const int* d = a.desc + cta * kDescInts;
  const int span = d[0];
  if (span == 0) return;
  const int row = d[2] + col;
  if (row >= d[3]) return;
  const size_t slot = (size_t)kRows * (D + 2);
  // CTA c's item is in its slot 1, the following CTAs' parts of it in their slots 0
  auto part = [&](int k) { return a.part + (size_t)((cta + k) * 2 + (k == 0)) * slot; };
  float m = -CUDART_INF_F;
  for (int k = tid; k < span; k += 128) m = fmaxf(m, part(k)[kRows * D + col]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) s_m[tid / 32] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const int grp = tid / LANES, ch = tid % LANES;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 4
  for (int k = grp; k < span; k += GROUPS) {
    const float* p = part(k);
    const float mk = p[kRows * D + col], f = mk == m ? 1.0f : ex2(mk - m);
    const float4 v = *reinterpret_cast<const float4*>(p + col * D + 4 * ch);
    l = fmaf(f, p[kRows * D + kRows + col], l);
    o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
  }
  s_o[grp][ch] = o;
  if (ch == 0) s_l[grp] = l;
  __syncthreads();
  if (grp != 0) return;
  l = s_l[0];
#pragma unroll
  for (int k = 1; k < GROUPS; ++k) {
    const float4 v = s_o[k][ch];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
    l += s_l[k];
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __half* op = a.out + (int64_t)(d[1] + row / a.G) * a.o_ts + (int64_t)(d[4] * a.G + row % a.G) * a.o_hs;
  *reinterpret_cast<uint2*>(op + 4 * ch) = make_uint2(h2_as_u32(__floats2half2_rn(o.x * inv, o.y * inv)),
                                                      h2_as_u32(__floats2half2_rn(o.z * inv, o.w * inv)));
}

// Consumer warps of a CTA.  With the producer 12: 168 registers a thread, what a 64-token tile
// of 8 query rows takes without spilling.  Measured on B200, 48 requests of 1 to 16384 tokens,
// 28 / 4 heads: 11 warps x 64 tokens 47.4 us, 15 warps x 32 tokens 53.5 us (more instructions
// per token: the logic pipe, which unpacks the codes, binds).  Items of 16 rows halve the
// unpacking but fit 7 warps only: 8 requests of 4096 tokens with 4 query tokens take 27.2 us
// (8 rows: 26.8), with 24 tokens 76 (78), with one token 30 (21).
constexpr int kWarps = 11;
constexpr int kNoPrefill = 0x7fffffff;                 // min_rows where only this kernel runs

template <class G_>
cudaError_t launch_geo(AttnArgs a, int num_sms, cudaStream_t stream) {
  static PerDeviceOnce attr_once;
  const cudaError_t attr = attr_once.run([] {
    return cudaFuncSetAttribute(kv4_attn_kernel<G_>, cudaFuncAttributeMaxDynamicSharedMemorySize, G_::SMEM);
  });
  if (attr != cudaSuccess) return attr;
  a.warp_part = a.part + (size_t)num_sms * 2 * G_::SLOT;
  cudaError_t e;
  if (a.min_rows == kNoPrefill) {
    kv4_attn_kernel<G_><<<num_sms, G_::THREADS, G_::SMEM, stream>>>(a);
    e = cudaGetLastError();
  } else {                                               // beside the end of the tcgen05 kernel
    e = kv4::launch_overlapped(kv4_attn_kernel<G_>, dim3(num_sms), G_::THREADS, G_::SMEM, stream, a);
  }
  if (e != cudaSuccess) return e;
  return kv4::launch_overlapped(kv4_merge_kernel<G_::D>, dim3(num_sms, kRows), 128, 0, stream, a);
}

template <int D, int GROUP>
cudaError_t launch_form(const AttnArgs& a, int num_sms, cudaStream_t stream) {
  // two stages must fit shared memory: 32-token tiles where a 64-token one takes 10 KB
  return launch_geo<Geo<D, GROUP, D / GROUP == 4 ? 2 : 4, kWarps>>(a, num_sms, stream);
}

cudaError_t launch_decode(const AttnArgs& a, int D, int g, int num_sms, cudaStream_t stream) {
  if (D == 64 && g == 32) return launch_form<64, 32>(a, num_sms, stream);
  if (D == 64 && g == 64) return launch_form<64, 64>(a, num_sms, stream);
  if (D == 128 && g == 32) return launch_form<128, 32>(a, num_sms, stream);
  if (D == 128 && g == 64) return launch_form<128, 64>(a, num_sms, stream);
  if (D == 128 && g == 128) return launch_form<128, 128>(a, num_sms, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

size_t kv4_attention_workspace(int head_dim, int64_t max_rows, int num_sms) {
  // per CTA a descriptor, 2 slots and one per warp; and for the prefill kernel, which the other
  // may overlap, a descriptor and 2 slots of 256 rows
  const size_t row = (size_t)(head_dim + 2) * 4;
  size_t bytes = kDescInts * 4 + (2 + kWarps) * kRows * row;
  if (max_rows >= kKv4PrefillMinRows) bytes += kDescInts * 4 + 2 * kKv4PrefillRows * row;
  return num_sms * bytes;
}

cudaError_t launch_kv4_attention(const Kv4AttnCall& c, int num_sms, int* dev_status,
                                 cudaStream_t stream) {
  AttnArgs a = {};
  a.cache = static_cast<const uint8_t*>(c.data);
  a.q = static_cast<const __half*>(c.q), a.out = static_cast<__half*>(c.out);
  a.table = c.table, a.lens = c.lens, a.cu_q = c.cu_q;
  a.q_ts = c.q_ts, a.q_hs = c.q_hs, a.o_ts = c.o_ts, a.o_hs = c.o_hs, a.table_rs = c.table_rs;
  a.num_pages = c.cache.num_pages, a.tokens = c.tokens;
  a.desc = static_cast<int*>(c.workspace);
  a.part = reinterpret_cast<float*>(a.desc + num_sms * kDescInts);
  a.status = dev_status;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.R = c.rows, a.width = c.width, a.kv_heads = c.cache.heads, a.G = c.q_heads / c.cache.heads;
  a.page_shift = 0;
  while ((1 << a.page_shift) < c.cache.page) ++a.page_shift;
  const int D = c.cache.dim, g = c.cache.group;
  if ((int64_t)c.max_q * a.G < kKv4PrefillMinRows) {
    a.min_rows = kNoPrefill;
    return launch_decode(a, D, g, num_sms, stream);
  }
  // requests with many query rows beside those with few; they share no output row
  a.min_rows = kKv4PrefillMinRows;
  AttnArgs p = a;
  p.desc = reinterpret_cast<int*>(a.part + (size_t)num_sms * (2 + kWarps) * kRows * (D + 2));
  p.part = reinterpret_cast<float*>(p.desc + num_sms * kDescInts);
  cudaError_t e = launch_kv4_prefill(p, D, g, num_sms, stream);
  if (e == cudaSuccess) e = launch_decode(a, D, g, num_sms, stream);
  if (e == cudaSuccess) e = launch_kv4_prefill_merge(p, D, num_sms, stream);
  return e;
}

}  // namespace awq
