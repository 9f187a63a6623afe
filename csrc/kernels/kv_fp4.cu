// The 4-bit KV cache's row kernels: RoPE + NVFP4 quantisation into the pages, the rows read back, page copies.
//
//   k' = rope(k) / g_k, v' = v / g_v (products with the fp32 reciprocals); per 16 dimensions
//   s = e4m3(clamp(max|x'| / 6, 2^-9, 448)),  code = e2m1(x' / s)   (both to nearest even, saturating)
// The floor keeps the scale of a block of zeros a positive number; with it, or with values beyond 2688 (infinities
// among them), codes saturate and the cache stays finite.  A NaN is stored as the block's largest magnitude.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_fp4.h"
#include "nvfp4_act.cuh"
#include "pdl.cuh"

namespace shk {
namespace kv4 {

constexpr int PAGE = 64;
constexpr int WRITE_THREADS = 256;

template <int D>
struct Geo {
  static constexpr int ROW = D / 2, SROW = D / 16;
  static constexpr int PAGE_BYTES = PAGE * (ROW + SROW);
};

// One CTA per token; D/16 neighbouring threads hold a head's 16-dimension blocks, and a thread keeps its block
// through all heads, so its cosines and sines are read once.
template <int D>
__global__ void __launch_bounds__(WRITE_THREADS) write_kernel(KvFp4WriteParams p) {
  constexpr int BLOCKS = D / 16;
  constexpr int HEADS = WRITE_THREADS / BLOCKS;  // heads in flight
  shk::pdl_trigger();
  shk::pdl_wait();
  const int64_t tok = blockIdx.x;
  const int blk = threadIdx.x % BLOCKS, d0 = blk * 16;
  const int half = p.rot / 2;
  int64_t pos = p.positions[tok];
  if (pos < 0 || pos >= p.max_pos) pos = 0;  // never past the table
  const float* cs = p.cos_sin + pos * p.rot;
  // The rotation of dimension d < rot pairs it with d +- half: x'[d] = x[d] c - x[d + half] s below half, and
  // x[d] c + x[d - half] s above.
  float c[16], s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int d = d0 + i;
    const int j = d < half ? d : d - half;
    c[i] = d < p.rot ? cs[j] : 1.f;
    s[i] = d < p.rot ? (d < half ? -cs[half + j] : cs[half + j]) : 0.f;
  }
  const int64_t slot = p.slots[tok];
  const bool cached = slot >= 0 && slot < p.num_slots;
  const int64_t page = slot / PAGE;
  const int off = static_cast<int>(slot % PAGE);
  const __nv_bfloat16* row = p.qkv + tok * p.qkv_stride;
  for (int h = threadIdx.x / BLOCKS; h < p.hq + 2 * p.hk; h += HEADS) {
    if (h >= p.hq && !cached) break;
    const __nv_bfloat16* hp = row + static_cast<int64_t>(h) * D;
    float x[16];
    nvq::load16(hp + d0, x);
    if (h < p.hq + p.hk && d0 < p.rot) {
      float y[16];
      if (half % 16 == 0) {  // the partners are another whole block
        nvq::load16(hp + (d0 < half ? d0 + half : d0 - half), y);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int d = d0 + i;
          y[i] = d < p.rot ? __bfloat162float(hp[d < half ? d + half : d - half]) : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = __fadd_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
    }
    if (h < p.hq) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
      }
      uint4* dst = reinterpret_cast<uint4*>(p.q_out + tok * p.q_stride + static_cast<int64_t>(h) * D + d0);
      dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
      dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
      continue;
    }
    const bool key = h < p.hq + p.hk;
    const int hk = key ? h - p.hq : h - p.hq - p.hk;
    const float inv = key ? p.k_inv : p.v_inv;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = __fmul_rn(x[i], inv);
      amax = fmaxf(amax, fabsf(x[i]));
    }
    const __nv_fp8_e4m3 sc(fminf(fmaxf(__fdiv_rn(amax, 6.f), 1.f / 512.f), 448.f));
    const float sf = static_cast<float>(sc);
    // a true quotient: multiplying by 1/s moves values that lie between two codes off their tie
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __fdiv_rn(x[i], sf);
    uint8_t* pg = (key ? p.k_cache : p.v_cache) + (page * p.hk + hk) * Geo<D>::PAGE_BYTES;
    *reinterpret_cast<uint2*>(pg + off * Geo<D>::ROW + blk * 8) = make_uint2(nvq::e2m1x8(x), nvq::e2m1x8(x + 8));
    pg[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + blk] = sc.__x;
  }
}

// One thread per (slot, head, 16-dimension block).
template <int D>
__global__ void __launch_bounds__(256) read_kernel(KvFp4ReadParams p) {
  constexpr int BLOCKS = D / 16;
  shk::pdl_trigger();
  shk::pdl_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t rows = p.n * p.hk;
  if (i >= rows * BLOCKS) return;
  const bool key = blockIdx.y == 0;
  const int blk = static_cast<int>(i % BLOCKS);
  const int64_t row = i / BLOCKS;
  const int64_t slot = p.slots[row / p.hk];
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot >= 0 && slot < p.num_slots) {
    const uint8_t* pg = (key ? p.k_cache : p.v_cache) + ((slot / PAGE) * p.hk + row % p.hk) * Geo<D>::PAGE_BYTES;
    const int off = static_cast<int>(slot % PAGE);
    const uint2 codes = *reinterpret_cast<const uint2*>(pg + off * Geo<D>::ROW + blk * 8);
    __nv_fp8_e4m3 sc;
    sc.__x = pg[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + blk];
    const float sf = static_cast<float>(sc), gs = key ? p.k_scale : p.v_scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t byte = ((j < 4 ? codes.x : codes.y) >> (8 * (j & 3))) & 0xff;
      float v[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t c = (byte >> (4 * e)) & 15, m = c & 7;
        // e2m1: 0, 0.5, then (1 + bit 0 / 2) 2^(bits 2..1 - 1)
        const float mag = m < 2 ? 0.5f * m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
        v[e] = (c & 8 ? -mag : mag) * sf * gs;
      }
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[0], v[1]);
      w[j] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  uint4* dst = reinterpret_cast<uint4*>((key ? p.k_out : p.v_out) + row * D + blk * 16);
  dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
  dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

// Page copies in every tensor: a CTA moves up to 16 KB of one page, four 16-byte loads a thread in flight.
constexpr int COPY_THREADS = 256;
constexpr int COPY_VECS = 4;
constexpr int64_t COPY_BYTES = COPY_THREADS * COPY_VECS * 16;

__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const __grid_constant__ KvCopyParams p, int parts) {
  shk::pdl_trigger();
  shk::pdl_wait();
  const int t = blockIdx.y;
  const int64_t pair = blockIdx.x / parts, part = blockIdx.x % parts;
  const int64_t s = p.src[pair], d = p.dst[pair], bytes = p.page_bytes[t];
  if (s < 0 || d < 0 || s >= p.pages[t] || d >= p.pages[t]) return;
  const uint8_t* from = p.base[t] + s * bytes;
  uint8_t* to = p.base[t] + d * bytes;
  const int64_t at = part * COPY_BYTES + threadIdx.x * 16;
  uint4 v[COPY_VECS];
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i) {
    const int64_t o = at + i * COPY_THREADS * 16;
    if (o < bytes) v[i] = *reinterpret_cast<const uint4*>(from + o);
  }
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i) {
    const int64_t o = at + i * COPY_THREADS * 16;
    if (o < bytes) *reinterpret_cast<uint4*>(to + o) = v[i];
  }
}

}  // namespace kv4
}  // namespace shk

using namespace shk::kv4;

extern "C" int sh_kv_fp4_write(const KvFp4WriteParams* params, int head_dim, cudaStream_t stream) {
  const KvFp4WriteParams& p = *params;
  if (p.num_tokens <= 0) return 0;
  if (p.num_tokens > 0x7fffffff || p.rot < 0 || p.rot > head_dim || p.rot % 2) return -1;
  if ((reinterpret_cast<uintptr_t>(p.qkv) & 15) || (p.qkv_stride & 7) || (reinterpret_cast<uintptr_t>(p.q_out) & 15) ||
      (p.q_stride & 7) || (reinterpret_cast<uintptr_t>(p.k_cache) & 15) || (reinterpret_cast<uintptr_t>(p.v_cache) & 15))
    return -3;
  const dim3 grid(static_cast<unsigned>(p.num_tokens)), block(WRITE_THREADS);
  cudaError_t e;
  switch (head_dim) {
    case 64: e = shk::launch(write_kernel<64>, grid, block, 0, stream, p); break;
    case 128: e = shk::launch(write_kernel<128>, grid, block, 0, stream, p); break;
    case 256: e = shk::launch(write_kernel<256>, grid, block, 0, stream, p); break;
    default: return -4;
  }
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

extern "C" int sh_kv_fp4_read(const KvFp4ReadParams* params, int head_dim, cudaStream_t stream) {
  const KvFp4ReadParams& p = *params;
  if (p.n <= 0) return 0;
  const int64_t ctas = (p.n * p.hk * (head_dim / 16) + 255) / 256;
  if (ctas > 0x7fffffff) return -1;
  const dim3 grid(static_cast<unsigned>(ctas), 2), block(256);
  cudaError_t e;
  switch (head_dim) {
    case 64: e = shk::launch(read_kernel<64>, grid, block, 0, stream, p); break;
    case 128: e = shk::launch(read_kernel<128>, grid, block, 0, stream, p); break;
    case 256: e = shk::launch(read_kernel<256>, grid, block, 0, stream, p); break;
    default: return -4;
  }
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}

extern "C" int sh_kv_copy_pages(const KvCopyParams* params, cudaStream_t stream) {
  const KvCopyParams& p = *params;
  if (p.n <= 0 || p.tensors <= 0) return 0;
  if (p.tensors > SH_KV_COPY_MAX_TENSORS) return -1;
  int64_t most = 0;
  for (int t = 0; t < p.tensors; ++t) {
    if (p.page_bytes[t] % 16 || (reinterpret_cast<uintptr_t>(p.base[t]) & 15)) return -3;
    most = most < p.page_bytes[t] ? p.page_bytes[t] : most;
  }
  const int64_t parts = (most + COPY_BYTES - 1) / COPY_BYTES;
  if (parts * p.n > 0x7fffffff) return -1;
  const cudaError_t e =
      shk::launch(copy_kernel, dim3(static_cast<unsigned>(parts * p.n), static_cast<unsigned>(p.tensors)),
                  dim3(COPY_THREADS), 0, stream, p, static_cast<int>(parts));
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
