// C ABI of the 4-bit KV cache's row kernels (no PyTorch types): the writer, the reader and the page copy.  The page
// layout is stated in paged_attention_fp4.h.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#define SH_KV_COPY_MAX_TENSORS 128

struct KvFp4WriteParams {
  const __nv_bfloat16* qkv;   // [T, >= (hq + 2 hk) D], row stride qkv_stride
  int64_t qkv_stride;
  __nv_bfloat16* q_out;       // [T, >= hq D] rotated queries, row stride q_stride
  int64_t q_stride;
  const int64_t* positions;   // [T]
  const float* cos_sin;       // [max_pos, rot]: cos in [:rot/2], sin behind
  int64_t max_pos;
  const int64_t* slots;       // [T] cache slot, < 0: not cached
  uint8_t* k_cache;           // [num_blocks, hk, page bytes]
  uint8_t* v_cache;
  int64_t num_tokens, num_slots;  // slots: num_blocks * 64
  int hq, hk, rot;
  float k_inv, v_inv;         // 1 / the caches' scales
};

struct KvFp4ReadParams {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  __nv_bfloat16* k_out;       // [n, hk, D] contiguous
  __nv_bfloat16* v_out;
  const int64_t* slots;       // [n]; a slot outside the cache reads as zeros
  int64_t n, num_slots;
  int hk;
  float k_scale, v_scale;
};

struct KvCopyParams {
  uint8_t* base[SH_KV_COPY_MAX_TENSORS];
  int64_t page_bytes[SH_KV_COPY_MAX_TENSORS];  // multiples of 16
  int64_t pages[SH_KV_COPY_MAX_TENSORS];
  const int64_t* src;         // [n]
  const int64_t* dst;
  int64_t n;
  int tensors;
};

#ifdef __cplusplus
extern "C" {
#endif
int sh_kv_fp4_write(const KvFp4WriteParams* p, int head_dim, cudaStream_t stream);
int sh_kv_fp4_read(const KvFp4ReadParams* p, int head_dim, cudaStream_t stream);
int sh_kv_copy_pages(const KvCopyParams* p, cudaStream_t stream);
#ifdef __cplusplus
}
#endif
