// awq_kv4_args.cuh -- kernel arguments shared by the two attention kernels over the 4-bit
// cache (awq_kv4_attn.cu, awq_kv4_prefill.cu).
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace awq {
namespace kv4 {

constexpr int kPrefixEntries = 1024;     // prefix sums held in shared memory
constexpr int kDescInts = 8;             // per CTA: the item that starts there and goes on

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
  float* part;        // [ctas][2] slots of items that cross CTAs
  float* warp_part;   // [ctas][warps] slots of items that cross warps, not a warp's last
  int* desc;          // [ctas][kDescInts]
  int* status;
  float scale_log2;
  int R, width, page_shift, kv_heads, G;
  int min_rows;       // requests with this many query rows per kv head are the prefill kernel's
};

}  // namespace kv4
}  // namespace awq
