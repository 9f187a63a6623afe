// The 4-bit KV cache's row kernels: RoPE + NVFP4 quantisation into the pages, the rows read back, page copies.
//
//   k' = rope(k) / g_k, v' = v / g_v (products with the fp32 reciprocals); per 16 dimensions
//   s = e4m3(clamp(max|x'| / 6, 2^-9, 448)),  code = e2m1(x' / s)   (both to nearest even, saturating)
// The floor keeps the scale of a block of zeros a positive number; with it, or with values beyond 2688 (infinities
// among them), codes saturate and the cache stays finite.  A NaN is stored as the block's largest magnitude.
#include <float.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
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
// Below, 256 threads a token, from there the kernel whose warps each take a run of heads.  In us for 420, 600, 900 and 1200
// tokens: 32 + 2 x 8 heads of 128: 3.7, 5.4, 6.8, 8.9 against 6.2, 6.8, 7.7, 8.8; as many of 256: 6.8, 10.9, 16.2, 19.4 against
// 8.3, 9.9, 12.6, 14.4; 8 + 2 x 2 of 64: 3.1, 5.1, 6.3, 7.4 against 3.2, 3.6, 3.9, 4.6.
constexpr int64_t kFewTokens = 600;
constexpr int STREAM_CTAS = 2, DEPTH = 4;
constexpr int READ_THREADS = 128, READ_UNITS = 4;

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
// The block's scale, and codes of x / scale.  The quotient is x (rh + rl) with rh + rl = 1 / scale in two words, rounded
// once (but for 2^-24 of a unit).  The ties t between codes have at most 3 bits and a scale 4, so t * scale is exact; if x
// is that, the result is t; the next x is further away than the rounding reaches: every code is that of the true
// quotient.  One product with rh alone moves values off their ties; a division per value made the writer's arithmetic a
// third longer (16384 tokens of 48 heads of 128: 32 million warp instructions).
struct Scale {
  __nv_fp8_e4m3 e4m3;
  float s, rh, rl;
};
__device__ __forceinline__ Scale block_scale(float amax) {
  Scale r;
  r.e4m3 = __nv_fp8_e4m3(fminf(fmaxf(__fdiv_rn(amax, 6.f), 1.f / 512.f), 448.f));
  r.s = static_cast<float>(r.e4m3);
  r.rh = __frcp_rn(r.s);
  r.rl = __fmul_rn(__fmaf_rn(-r.rh, r.s, 1.f), r.rh);
  return r;
}
template <int N>
__device__ __forceinline__ void quotients(float* x, float amax, const Scale& sc) {
  if (amax <= FLT_MAX) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmaf_rn(x[i], sc.rh, __fmul_rn(x[i], sc.rl));
  } else {  // an infinity times a zero rl would be no number
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], sc.rh);
  }
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
  const Scale sc = block_scale(amax);
  quotients<16>(x, amax, sc);
  *reinterpret_cast<uint2*>(page + off * Geo<D>::ROW + blk * 8) = make_uint2(nvq::e2m1x8(x), nvq::e2m1x8(x + 8));
  page[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + blk] = sc.e4m3.__x;
}

// TPT threads a token.  The rotation pairs dimension d < rot/2 with d + rot/2: where rot/2 is a whole number of blocks
// (WHOLE) a thread takes a block and its partner, reads their cosines and sines once and keeps them through its heads
// (every TPT / items-th one); the blocks behind rot go as they are.  Otherwise each block fetches its partners singly.
//
// Bound by latency: a single token of 32 + 2 x 8 heads of 128 takes 2.4 us, 389 take 3.7.  With 256 threads a token all
// of its heads are in flight.
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

// Eight dimensions, a thread's unit in the kernels below: one 16-byte access.
__device__ __forceinline__ void unpack8(const uint4& r, float* v) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// A unit of a key or value into its page, with the other half of its block, which lane ^ 1 brings; the whole warp calls.
template <int D>
__device__ __forceinline__ void put_unit(uint8_t* page, int off, int unit, float* x, float inv, bool live) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = __fmul_rn(x[i], inv);
    amax = fmaxf(amax, fabsf(x[i]));
  }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const Scale sc = block_scale(amax);
  quotients<8>(x, amax, sc);
  if (!live) return;
  *reinterpret_cast<uint32_t*>(page + off * Geo<D>::ROW + unit * 4) = nvq::e2m1x8(x);
  if (!(unit & 1)) page[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + (unit >> 1)] = sc.e4m3.__x;
}

__device__ __forceinline__ void async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Many tokens.  A token is a row of steps of STEP heads each, queries, keys and values.  A lane holds two units of a head:
// one and the unit that it is rotated with, or two behind rot (or of a value), so that the blocks' halves are neighbours.
// The steps of all tokens, end to end, are cut into one run per warp.  A lane copies what it will read into its own
// places of shared memory, DEPTH - 1 steps ahead: loads are always in flight and nobody waits for another thread.
//
// Memory bound, with 65% of the issue slots taken.  16384 tokens of 32 + 2 x 8 heads of 128 (363 MB with the cosines)
// take 70 us, 80% of the copy rate, of 16 + 2 x 2 heads of 256 (303 MB) 55 us, 85%; 256 threads a token take 117 and 137 there, and a warp a token with its
// loads in registers 87 and 125.  (Three CTAs an SM, three or two steps deep: the same for many tokens, 1 us more for a
// thousand; four CTAs, two deep: 97, for 64 registers spill.  Products of pairs, mul.f32x2 and add.f32x2, were fused by
// the compiler, against the reference's two roundings, and no faster.)
template <int D>
__global__ void __launch_bounds__(WRITE_THREADS, STREAM_CTAS) write_stream_kernel(KvFp4WriteParams p) {
  constexpr int UNITS = D / 8, ITEMS = UNITS / 2, STEP = 32 / ITEMS;
  extern __shared__ uint4 ring[];  // [DEPTH][6][WRITE_THREADS]: the two units, cosines (2), sines (2)
  shk::pdl_trigger();
  shk::pdl_wait();
  const int item = threadIdx.x % ITEMS, h0 = threadIdx.x % 32 / ITEMS;
  const int half = p.rot / 2, pairs = half / 8;
  const bool rotates = item < pairs;
  const int unit = rotates ? item : item + pairs, other = rotates ? pairs : ITEMS - pairs;  // its second unit is unit + other
  const int heads = p.hq + 2 * p.hk, all = (heads + STEP - 1) / STEP;
  const int64_t runs = static_cast<int64_t>(gridDim.x) * (WRITE_THREADS / 32);
  const int64_t run = static_cast<int64_t>(blockIdx.x) * (WRITE_THREADS / 32) + threadIdx.x / 32;
  const int64_t total = p.num_tokens * all, first = run * total / runs;
  const int count = static_cast<int>((run + 1) * total / runs - first);
  if (count <= 0) return;

  const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(ring + threadIdx.x));
  auto place = [](int s, int k) { return static_cast<uint32_t>((s * 6 + k) * WRITE_THREADS * 16); };
  // where the copies are, and where the reads are
  int64_t ft = first / all, ct = ft;
  int fe = static_cast<int>(first - ft * all), ce = fe, asked = 0;
  int64_t fpos = p.positions[ft], npos = ft + 1 < p.num_tokens ? p.positions[ft + 1] : 0;
  bool fresh = true;  // the copies' token has no cosines yet
  auto fetch = [&]() {
    if (asked < count) {
      const uint32_t to = base + place(asked % DEPTH, 0);
      const int h = fe * STEP + h0;
      if (h < heads) {
        const __nv_bfloat16* src = p.qkv + ft * p.qkv_stride + static_cast<int64_t>(h) * D + unit * 8;
        async16(to, src);
        async16(to + place(0, 1), src + other * 8);
      }
      if (fresh && rotates) {
        const int64_t pos = fpos < 0 || fpos >= p.max_pos ? 0 : fpos;  // never past the table
        const float* cs = p.cos_sin + pos * p.rot + item * 8;
        async16(to + place(0, 2), cs);
        async16(to + place(0, 3), cs + 4);
        async16(to + place(0, 4), cs + half);
        async16(to + place(0, 5), cs + half + 4);
      }
      fresh = false;
      ++asked;
      if (++fe == all) {
        fe = 0;
        ++ft;
        fresh = true;
        fpos = npos;
        npos = ft + 1 < p.num_tokens ? p.positions[ft + 1] : 0;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < DEPTH - 1; ++i) fetch();

  int64_t slot = p.slots[ct], next_slot = ct + 1 < p.num_tokens ? p.slots[ct + 1] : 0;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = 1.f, s[i] = 0.f;
  bool stale = true;
#pragma unroll 1
  for (int n = 0; n < count; ++n) {
    fetch();
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    const uint4* at = ring + (n % DEPTH) * 6 * WRITE_THREADS + threadIdx.x;
    if (stale && rotates) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<uint4*>(c + 4 * i) = at[(2 + i) * WRITE_THREADS];
        *reinterpret_cast<uint4*>(s + 4 * i) = at[(4 + i) * WRITE_THREADS];
      }
    }
    stale = false;
    const bool cached = slot >= 0 && slot < p.num_slots;
    const int h = ce * STEP + h0;
    const bool pages = cached && ce * STEP + STEP > p.hq;  // some of the step's heads go into the cache
    if (h < p.hq || pages) {
      float x[8], y[8];
      const uint4 zero = make_uint4(0, 0, 0, 0);
      unpack8(h < heads ? at[0] : zero, x);
      unpack8(h < heads ? at[WRITE_THREADS] : zero, y);
      if (rotates && h < p.hq + p.hk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = __fsub_rn(__fmul_rn(x[i], c[i]), __fmul_rn(y[i], s[i]));
          y[i] = __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(x[i], s[i]));
          x[i] = u;
        }
      }
      if (h < p.hq) {
        uint4* dst = reinterpret_cast<uint4*>(p.q_out + ct * p.q_stride + static_cast<int64_t>(h) * D) + unit;
        dst[0] = pack8(x);
        dst[other] = pack8(y);
      }
      if (pages) {
        const int j = h - p.hq;
        const bool key = j < p.hk;
        uint8_t* pg = (key ? p.k_cache : p.v_cache) + (slot / PAGE * p.hk + (key ? j : j - p.hk)) * Geo<D>::PAGE_BYTES;
        const int off = static_cast<int>(slot % PAGE);
        const float inv = key ? p.k_inv : p.v_inv;
        const bool live = j >= 0 && h < heads;
        put_unit<D>(pg, off, unit, x, inv, live);
        put_unit<D>(pg, off, unit + other, y, inv, live);
      }
    }
    if (++ce == all) {
      ce = 0;
      ++ct;
      stale = true;
      slot = next_slot;
      next_slot = ct + 1 < p.num_tokens ? p.slots[ct + 1] : 0;
    }
  }
}

// A thread reads READ_UNITS units of 8 dimensions, a CTA's in one run, in flight together.  Divisions by a slot's units
// are done in 32 bits, within the CTA (in 64 bits, for each thread: 25 us instead of 17).
// 16384 slots of 2 x 8 heads of 128 (86 MB) take 17 us, 78% of the copy rate; one takes 1.4 us.
template <int D>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(KvFp4ReadParams p) {
  constexpr int UNITS = D / 8;
  shk::pdl_trigger();
  shk::pdl_wait();
  const bool key = blockIdx.y == 0;
  const unsigned units = p.hk * UNITS;  // of a slot
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * (READ_THREADS * READ_UNITS);
  const int64_t n0 = begin / units;
  const unsigned r0 = static_cast<unsigned>(begin - n0 * units) + threadIdx.x;
  const uint8_t* cache = key ? p.k_cache : p.v_cache;
  const float gs = key ? p.k_scale : p.v_scale;
  uint4* out = reinterpret_cast<uint4*>(key ? p.k_out : p.v_out) + begin + threadIdx.x;
  const int64_t left = p.n * units - begin - threadIdx.x;
  uint32_t codes[READ_UNITS] = {};
  uint8_t sc[READ_UNITS] = {};
#pragma unroll
  for (int i = 0; i < READ_UNITS; ++i) {
    if (i * READ_THREADS >= left) break;
    const unsigned r = r0 + i * READ_THREADS, n = r / units, u = r - n * units;
    const int64_t slot = p.slots[n0 + n];
    if (slot < 0 || slot >= p.num_slots) continue;
    const uint8_t* pg = cache + (slot / PAGE * p.hk + u / UNITS) * Geo<D>::PAGE_BYTES;
    const int off = static_cast<int>(slot % PAGE), unit = u % UNITS;
    codes[i] = *reinterpret_cast<const uint32_t*>(pg + off * Geo<D>::ROW + unit * 4);
    sc[i] = pg[PAGE * Geo<D>::ROW + off * Geo<D>::SROW + (unit >> 1)];
  }
#pragma unroll
  for (int i = 0; i < READ_UNITS; ++i) {
    if (i * READ_THREADS >= left) break;
    __nv_fp8_e4m3 e;
    e.__x = sc[i];
    const float sf = static_cast<float>(e);
    uint32_t w[4];
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
        " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
        : "r"(codes[i]));
    float x[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
      x[2 * k] = v.x * sf * gs;
      x[2 * k + 1] = v.y * sf * gs;
    }
    out[i * READ_THREADS] = pack8(x);
  }
}

// Page copies in every tensor: a CTA moves up to 16 KB of one page, four 16-byte loads a thread in flight.  1023 blocks of
// 64 tensors (4.8 GB read and written) take 720 us, 103% of the rate of a plain copy; one block's 64 pages take 2.7 us.
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
template <int D, int TPT, bool WHOLE>
cudaError_t launch_write(const KvFp4WriteParams& p, cudaStream_t stream) {
  constexpr int TOKENS = WRITE_THREADS / TPT;
  const dim3 grid(static_cast<unsigned>((p.num_tokens + TOKENS - 1) / TOKENS));
  return shk::launch(write_kernel<D, TPT, WHOLE>, grid, dim3(WRITE_THREADS), 0, stream, p);
}
template <int D>
cudaError_t launch_stream(const KvFp4WriteParams& p, cudaStream_t stream) {
  constexpr int kMaxDevices = 64;
  constexpr size_t smem = static_cast<size_t>(DEPTH) * 6 * WRITE_THREADS * 16;
  static int sms[kMaxDevices];  // 0: this device has not been set up
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!sms[dev]) {
    int n = 0;
    if ((e = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(write_stream_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(smem))) != cudaSuccess)
      return e;
    sms[dev] = n;
  }
  return shk::launch(write_stream_kernel<D>, dim3(sms[dev] * STREAM_CTAS), dim3(WRITE_THREADS), smem, stream, p);
}
template <int D>
cudaError_t launch_write(const KvFp4WriteParams& p, cudaStream_t stream) {
  // a table that does not start on 16 bytes is read singly
  const bool whole = p.rot % 32 == 0 && !(reinterpret_cast<uintptr_t>(p.cos_sin) & 15);
  const bool few = p.num_tokens < kFewTokens;
  if (whole) return few ? launch_write<D, 256, true>(p, stream) : launch_stream<D>(p, stream);
  return few ? launch_write<D, 256, false>(p, stream) : launch_write<D, 32, false>(p, stream);
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
  if ((reinterpret_cast<uintptr_t>(p.k_cache) & 3) || (reinterpret_cast<uintptr_t>(p.v_cache) & 3) ||
      (reinterpret_cast<uintptr_t>(p.k_out) & 15) || (reinterpret_cast<uintptr_t>(p.v_out) & 15))
    return -3;
  constexpr int64_t per = READ_THREADS * READ_UNITS;
  const int64_t ctas = (p.n * p.hk * (head_dim / 8) + per - 1) / per;
  if (ctas > 0x7fffffff) return -1;
  const dim3 grid(static_cast<unsigned>(ctas), 2), block(READ_THREADS);
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
