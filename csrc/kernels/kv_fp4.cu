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
// Below, 256 threads a token, else 32 (head_dim 128: 768 tokens take 8.2 us against 10.4, 1500 take 15.7 against 12.2).
constexpr int64_t kFewTokens = 1200;

template <int D>
struct Geo {
  static constexpr int ROW = D / 2, SROW = D / 16;
  static constexpr int PAGE_BYTES = PAGE * (ROW + SROW);
};

// A block of 16 dimensions as loaded, and its values.
struct Raw {
  uint4 a, b;
};
__device__ __forceinline__ Raw fetch(const __nv_bfloat16* p) {
  return {__ldg(reinterpret_cast<const uint4*>(p)), __ldg(reinterpret_cast<const uint4*>(p) + 1)};
}
__device__ __forceinline__ void unpack(const Raw& r, float* v) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// A block of 16 rotated query dimensions in bf16.
__device__ __forceinline__ void put_query(__nv_bfloat16* dst, const float* x) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  uint4* d = reinterpret_cast<uint4*>(dst);
  d[0] = make_uint4(w[0], w[1], w[2], w[3]);
  d[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
// A block of 16 key or value dimensions into its page (block blk of token off).
template <int D>
__device__ __forceinline__ void put_cached(uint8_t* page, int off, int blk, float* x, float inv) {
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
  *reinterpret_cast<uint2*>(page + off * Geo<D>::ROW + blk * 8) = make_uint2(nvq::e2m1x8(x), nvq::e2m1x8(x + 8));
  page[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + blk] = sc.__x;
}

// TPT threads a token.  The rotation pairs dimension d < rot/2 with d + rot/2: where rot/2 is a whole number of blocks
// (WHOLE) a thread takes a block and its partner, reads their cosines and sines once and keeps them through its heads
// (every TPT / items-th one); the blocks behind rot go as they are.  Otherwise each block fetches its partners singly.
//
// Memory bound: 16384 tokens of 32 + 2 x 8 heads of 128 (363 MB) take 86 us, 65% of the copy rate; what is left is the
// loads in flight, which 121 registers a thread hold to 16 warps an SM (at 80 registers it spills: 96 us; fetching a
// head ahead takes 139: 165 us).  With 32 threads a token a thread's cosines serve five heads; with 256 a single token's
// heads are all in flight.
template <int D, int TPT, bool WHOLE>
__global__ void __launch_bounds__(WRITE_THREADS, (TPT == 32 && D < 256 ? 2 : 3)) write_kernel(KvFp4WriteParams p) {
  constexpr int BLOCKS = D / 16;
  shk::pdl_trigger();
  shk::pdl_wait();
  const int64_t tok = static_cast<int64_t>(blockIdx.x) * (WRITE_THREADS / TPT) + threadIdx.x / TPT;
  if (tok >= p.num_tokens) return;
  const int tid = threadIdx.x % TPT;
  const int half = p.rot / 2;
  int64_t pos = p.positions[tok];
  if (pos < 0 || pos >= p.max_pos) pos = 0;  // never past the table
  const float* cs = p.cos_sin + pos * p.rot;
  const int64_t slot = p.slots[tok];
  const bool cached = slot >= 0 && slot < p.num_slots;
  const int64_t page = cached ? slot / PAGE : 0;
  const int off = static_cast<int>(slot % PAGE);
  const __nv_bfloat16* row = p.qkv + tok * p.qkv_stride;
  const int heads = cached ? p.hq + p.hk : p.hq;
  auto put = [&](int h, int blk, float* x) {
    if (h < p.hq) put_query(p.q_out + tok * p.q_stride + static_cast<int64_t>(h) * D + blk * 16, x);
    else put_cached<D>(p.k_cache + (page * p.hk + h - p.hq) * Geo<D>::PAGE_BYTES, off, blk, x, p.k_inv);
  };
  if constexpr (WHOLE) {
    const int pairs = half / 16, items = BLOCKS - pairs, step = TPT / items;
    const int item = tid % items;
    int h = tid / items;
    if (h < step) {
      if (item < pairs) {
        float c[16], s[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *reinterpret_cast<float4*>(c + 4 * i) = reinterpret_cast<const float4*>(cs + item * 16)[i];
          *reinterpret_cast<float4*>(s + 4 * i) = reinterpret_cast<const float4*>(cs + half + item * 16)[i];
        }
        for (; h < heads; h += step) {
          const __nv_bfloat16* hp = row + static_cast<int64_t>(h) * D + item * 16;
          const Raw xa = fetch(hp), ya = fetch(hp + half);
          float x[16], y[16], z[16];
          unpack(xa, x);
          unpack(ya, y);
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
          put(h, item, z);
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(x[i], s[i]));
          put(h, item + pairs, z);
        }
      } else {
        for (; h < heads; h += step) {
          float x[16];
          unpack(fetch(row + static_cast<int64_t>(h) * D + (item + pairs) * 16), x);
          put(h, item + pairs, x);
        }
      }
    }
  } else {
    const int blk = tid % BLOCKS, d0 = blk * 16;
    for (int h = tid / BLOCKS; h < heads; h += TPT / BLOCKS) {
      const __nv_bfloat16* hp = row + static_cast<int64_t>(h) * D;
      float x[16];
      unpack(fetch(hp + d0), x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = d0 + i;
        if (d >= p.rot) break;
        const int j = d < half ? d : d - half;
        const float y = __bfloat162float(hp[d < half ? d + half : j]);
        const float u = __fmul_rn(x[i], cs[j]), v = __fmul_rn(y, cs[half + j]);
        x[i] = d < half ? __fsub_rn(u, v) : __fadd_rn(u, v);
      }
      put(h, blk, x);
    }
  }
  if (!cached) return;
  const int blk = tid % BLOCKS;
  constexpr int STEP = TPT / BLOCKS;
  for (int h = tid / BLOCKS; h < p.hk; h += STEP) {
    float x[16];
    unpack(fetch(row + static_cast<int64_t>(p.hq + p.hk + h) * D + blk * 16), x);
    put_cached<D>(p.v_cache + (page * p.hk + h) * Geo<D>::PAGE_BYTES, off, blk, x, p.v_inv);
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

namespace {
template <int D, int TPT>
cudaError_t launch_write(const KvFp4WriteParams& p, cudaStream_t stream) {
  constexpr int TOKENS = WRITE_THREADS / TPT;
  const dim3 grid(static_cast<unsigned>((p.num_tokens + TOKENS - 1) / TOKENS)), block(WRITE_THREADS);
  return p.rot % 32 == 0 ? shk::launch(write_kernel<D, TPT, true>, grid, block, 0, stream, p)
                         : shk::launch(write_kernel<D, TPT, false>, grid, block, 0, stream, p);
}
template <int D>
cudaError_t launch_write(const KvFp4WriteParams& p, cudaStream_t stream) {
  return p.num_tokens < kFewTokens ? launch_write<D, 256>(p, stream) : launch_write<D, 32>(p, stream);
}
}  // namespace

extern "C" int sh_kv_fp4_write(const KvFp4WriteParams* params, int head_dim, cudaStream_t stream) {
  const KvFp4WriteParams& p = *params;
  if (p.num_tokens <= 0) return 0;
  if (p.num_tokens > 0x7fffffff || p.rot < 0 || p.rot > head_dim || p.rot % 2) return -1;
  if ((reinterpret_cast<uintptr_t>(p.qkv) & 15) || (p.qkv_stride & 7) || (reinterpret_cast<uintptr_t>(p.q_out) & 15) ||
      (p.q_stride & 7) || (reinterpret_cast<uintptr_t>(p.k_cache) & 15) || (reinterpret_cast<uintptr_t>(p.v_cache) & 15))
    return -3;
  cudaError_t e;
  switch (head_dim) {
    case 64: e = launch_write<64>(p, stream); break;
    case 128: e = launch_write<128>(p, stream); break;
    case 256: e = launch_write<256>(p, stream); break;
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
