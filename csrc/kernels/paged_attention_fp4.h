// C ABI of the paged attention kernels over the 4-bit KV cache (no PyTorch types).
//
// Cache page of one (block, kv head): 64 tokens x D/2 code bytes (two e2m1 codes a byte, even dimension in the
// low nibble), then 64 tokens x D/16 e4m3 scales (one per 16 dimensions, sign bit clear): 64 (D/2 + D/16) bytes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

struct AttnFp4Params {
  __nv_bfloat16* out;            // [T, >= hq*D], row stride out_stride elements
  int64_t out_stride;
  const __nv_bfloat16* q;        // [T, >= hq*D], row stride q_stride; rows 16-byte aligned
  int64_t q_stride;
  const uint8_t* k_cache;        // [num_blocks, hk, 64 (D/2 + D/16)]
  const uint8_t* v_cache;
  const int32_t* block_tables;   // [B, bt_cols], row stride bt_stride
  int64_t bt_stride;
  const int64_t* seq_lens;       // [B] length including the new tokens
  const int64_t* q_start;        // [B + 1]
  float* part_o;                 // sh_paged_attention_fp4_workspace floats
  unsigned* tickets;             // zeroed words; every call leaves them zero
  int* err;                      // optional: the code of the first wait that ran out (the kernel for short queries has none)
  int64_t num_tokens;            // T
  int B, hq, hk, num_blocks, bt_cols;  // bt_cols: below 2^25, so that a position fits an int
  int whole_units;               // 1: a (request, head, row tile) is never split over CTAs
  float scale_log2;              // softmax scale x log2(e) x the key cache's scale
  float v_scale;                 // the value cache's scale
};

#ifdef __cplusplus
extern "C" {
#endif
// CTAs of the kernel for short queries at this head dimension and row tile (also the number of tickets), and the
// floats of partial results that they may write.  row_tile: query rows of one kv head a CTA holds, 8 * (1..4).
int sh_paged_attention_fp4_ctas(int head_dim, int row_tile);
int64_t sh_paged_attention_fp4_workspace(int head_dim, int row_tile);
// 0 on success; head_dim in {64, 128, 256}, block size 64.
int sh_paged_attention_fp4(const AttnFp4Params* p, int head_dim, int row_tile, cudaStream_t stream);
// The tensor-core kernel for many query rows: units of 256 rows (128 at head_dim 256), whole_units not supported, no
// tickets.
int64_t sh_paged_attention_fp4_tc_workspace(int head_dim);
int sh_paged_attention_fp4_tc(const AttnFp4Params* p, int head_dim, cudaStream_t stream);
#ifdef __cplusplus
}
#endif
