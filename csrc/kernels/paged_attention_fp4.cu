// Paged GQA attention over the 4-bit KV cache: decode, verify windows and (any length) short query runs.
//
//   o[t, h] = g_v sum_j softmax_j(q[t, h] . k[j] g_k scale) v[j],   j <= position of t
//   k[j], v[j] = e2m1 code x e4m3 block scale (16 dimensions), read as they lie in the pages.
//
// Work.  A unit is (request, kv head, tile of NT * 8 packed query rows); packed row r of a request is token r / G,
// head r % G of the group, so the heads of a group and the tokens of a verify window share one read of the keys.
// The units' pages, laid end to end, are cut into equal runs, one per CTA (2 CTAs an SM for one 8-row tile): a
// ragged batch loads every SM alike and no length has to be known on the host.  A unit cut by a run's end leaves an
// fp32 partial (O, max, sum); the last of its CTAs to finish (a ticket, which it resets) merges them in page order,
// so the result does not depend on the order of arrival.
//
// A CTA's 8 warps take the run's 16-token chunks in turn, each through a ring of its own in shared memory, filled
// with cp.async three chunks ahead: no barrier between the warps while they stream.  Per chunk and warp, with
// m16n8k16 (f16 in, fp32 out) and the KEYS on the M side, so 8 query rows fill the N side that decode has:
//   S^T (16 tokens x rows) = K Q^T,   O^T (D x rows) += V^T P^T.
// Both products are free to permute the dimension they sum over, or the rows of the result: thread (g, t) of the
// quad layout takes D/4 consecutive dimensions of a key as its share of K's columns, and D/8 consecutive dimensions
// as its share of V^T's rows, so its codes are one 8- to 32-byte run of a row and one or two scales cover them.
// V^T's pairs of adjacent tokens come from interleaving the nibbles of two tokens' words (a shift and a lop3 per 8
// codes).  e2m1 -> f16 is exact, and so is the product with the e4m3 scale (at most 6 significant bits, between
// 2^-10 and 2688).  Q goes to f16 after a multiplication by a power of two per row (its largest element into
// [2^13, 2^14), which keeps bf16's 8 bits for elements down to 2^-38 of it); the power leaves with the softmax scale.
// P is rounded to f16: 11 bits, where bf16 would cost as much again as the output's own rounding.
//
// The softmax keeps, per row, a reference m that moves only when a score exceeds it by more than 8 (in log2 units):
// P <= 2^8 stays far from f16's range, and a chunk costs one vote instead of a reduction over the tokens.
//
// Rows that see no key give 0.  Tokens past the end of a sequence are read (they lie in its last page) with V's
// scale replaced by 0 and their scores by -inf, so what an earlier owner left there does not matter.
#include <float.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_attention_fp4.h"
#include "pdl.cuh"

namespace shk {
namespace attn4 {

constexpr int WARPS = 8;
constexpr int THREADS = WARPS * 32;
constexpr int CHUNK = 16;  // tokens of one warp step
constexpr int PAGE = 64;   // tokens of a page
constexpr float kSlack = 8.f;
constexpr int kMinPages = 2;  // shortest run: a chunk for every warp

template <int D>
struct Geo {
  static constexpr int ROW = D / 2;              // code bytes of a token
  static constexpr int SROW = D / 16;            // scale bytes of a token
  static constexpr int PAGE_BYTES = PAGE * (ROW + SROW);
  static constexpr int CODES = CHUNK * ROW;
  static constexpr int SCALES = CHUNK * SROW;
  static constexpr int STAGE = 2 * (CODES + SCALES);
  static constexpr int PIECES = ROW / 16;        // 16-byte pieces of a token's codes
};
template <int D, int NT>
struct Cfg {
  static constexpr int CTAS = (D <= 128 && NT == 1) ? 2 : 1;  // per SM
  static constexpr int STAGES = CTAS == 2 ? 4 : (D == 256 ? 3 : 6);
  static constexpr int MSTRIDE = D + 4;  // floats of a merge row
  static constexpr int RING = WARPS * STAGES * Geo<D>::STAGE;
  static constexpr int MERGE = WARPS * 8 * MSTRIDE * 4;
  static constexpr int STATS = 2 * WARPS * 8 * NT * 4;
  static constexpr int SMEM = RING + MERGE + STATS;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// The four code pairs of a word as f16 pairs (low nibble in the low half).
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t* o) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}
// Two e4m3 scales (low and next byte) as an f16 pair.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t w) {
  uint32_t r;
  asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Byte of 16-byte piece p of token r in a chunk's key (value) codes.  A warp's 16-, 8- or 4-byte reads of the
// fragments then fall into different banks: keys are read as neighbouring rows, values as every second row.
template <int D>
__device__ __forceinline__ int key_at(int r, int p) {
  if constexpr (D == 256) p ^= r & 1;
  return r * Geo<D>::ROW + p * 16;
}
template <int D>
__device__ __forceinline__ int value_at(int r, int p) {
  if constexpr (D == 256) p ^= ((r >> 1) & 3) << 1;
  if constexpr (D == 128) {
    const int line = r >> 1, q = ((r & 1) << 2 | p) ^ ((line & 3) << 1);
    return line * 128 + q * 16;
  }
  if constexpr (D == 64) {
    const int line = r >> 2, q = ((r & 3) << 1 | p) ^ ((line & 1) << 1);
    return line * 128 + q * 16;
  }
  return r * Geo<D>::ROW + p * 16;
}

// What a request asks for, clipped to the tensors it indexes.
struct Request {
  int64_t qs, seq;
  int q_len, tiles, pages;
};
__device__ __forceinline__ Request request(const AttnFp4Params& p, int b, int rows) {
  Request r;
  const int64_t q0 = p.q_start[b], q1 = p.q_start[b + 1];
  r.qs = q0 < 0 ? 0 : q0;
  const int64_t n = (q1 < p.num_tokens ? q1 : p.num_tokens) - r.qs;
  r.q_len = n > 0 ? static_cast<int>(n) : 0;
  r.seq = p.seq_lens[b];
  if (r.seq < 0) r.seq = 0;
  const int64_t cap = static_cast<int64_t>(p.bt_cols) * PAGE;
  if (r.seq > cap) r.seq = cap;
  r.tiles = static_cast<int>((static_cast<int64_t>(r.q_len) * (p.hq / p.hk) + rows - 1) / rows);
  r.pages = static_cast<int>((r.seq + PAGE - 1) / PAGE);
  if (r.pages < 1) r.pages = 1;  // a request without keys still has its rows to write
  return r;
}
__device__ __forceinline__ int64_t weight(const AttnFp4Params& p, const Request& r) {
  return static_cast<int64_t>(r.tiles) * p.hk * r.pages;
}

// One unit's part in a CTA's run.
struct Segment {
  int64_t u0, u1;  // the unit's place among all pages
  int b, h, row0, pg0, pg1, pages, c0, c1;  // c0, c1: chunks with keys that some row sees
  int64_t qs, ctx0, kv_end;
  int rows;
};
// Walks a CTA's run [pos, end) of the pages laid end to end; `base` is the place of request b's first page.
struct Cursor {
  int64_t pos, end, base;
  int b;
  Request r;
};
template <int ROWS>
__device__ __forceinline__ bool next_segment(const AttnFp4Params& p, Cursor& c, Segment& s) {
  const int g = p.hq / p.hk;
  int64_t unit;
  while (true) {
    if (c.pos >= c.end) return false;
    while (c.pos >= c.base + weight(p, c.r)) {
      c.base += weight(p, c.r);
      c.r = request(p, ++c.b, ROWS);
    }
    unit = (c.pos - c.base) / c.r.pages;
    const int64_t at = c.base + unit * c.r.pages;
    if (!p.whole_units || at == c.pos) break;
    c.pos = at + c.r.pages;  // whole units: one that began in an earlier run belongs to that run's CTA
  }
  s.b = c.b;
  s.h = static_cast<int>(unit % p.hk);
  const int tile = static_cast<int>(unit / p.hk);
  s.row0 = tile * ROWS;
  const int64_t left = static_cast<int64_t>(c.r.q_len) * g - s.row0;
  s.rows = left < ROWS ? static_cast<int>(left) : ROWS;
  s.u0 = c.base + unit * c.r.pages;
  s.u1 = s.u0 + c.r.pages;
  s.pages = c.r.pages;
  s.pg0 = static_cast<int>(c.pos - s.u0);
  s.pg1 = p.whole_units || c.end >= s.u1 ? c.r.pages : static_cast<int>(c.end - s.u0);
  c.pos = s.u0 + s.pg1;
  s.qs = c.r.qs;
  s.ctx0 = c.r.seq - c.r.q_len;
  int64_t kv = s.ctx0 + (s.row0 + s.rows - 1) / g + 1;  // keys the tile's last row sees
  if (kv > c.r.seq) kv = c.r.seq;
  if (kv < 0) kv = 0;
  s.kv_end = kv;
  const int64_t last = (kv + CHUNK - 1) / CHUNK;
  s.c0 = s.pg0 * (PAGE / CHUNK);
  s.c1 = s.pg1 * (PAGE / CHUNK);
  if (s.c1 > last) s.c1 = static_cast<int>(last);
  return true;
}

template <int D, int NT>
__global__ void __launch_bounds__(THREADS, (Cfg<D, NT>::CTAS)) attn_fp4_kernel(AttnFp4Params p) {
  using G = Geo<D>;
  using K = Cfg<D, NT>;
  constexpr int ROWS = 8 * NT;
  constexpr int STAGES = K::STAGES;
  constexpr int KSTEPS = D / 16;
  constexpr int MT = D / 16;
  constexpr int KW = D / 32;  // words of a key in a thread (D/4 codes)
  constexpr int VB = D / 16;  // bytes of a value in a thread (D/8 codes)
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge_o = reinterpret_cast<float*>(smem + K::RING);
  float* merge_m = reinterpret_cast<float*>(smem + K::RING + K::MERGE);  // [WARPS][ROWS]
  float* merge_l = merge_m + WARPS * ROWS;
  __shared__ int64_t scan[WARPS + 1];
  __shared__ int64_t start_base;
  __shared__ int start_b;
  __shared__ int last_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = p.hq / p.hk;
  shk::pdl_trigger();
  shk::pdl_wait();  // lengths, tables, queries and the new tokens' rows come from earlier kernels

  // ---------------------------------------------------------------- this CTA's run
  int64_t total = 0;
  for (int b = threadIdx.x; b < p.B; b += THREADS) total += weight(p, request(p, b, ROWS));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) scan[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < WARPS; ++w) total += scan[w];
  __syncthreads();
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < kMinPages) per = kMinPages;
  Cursor cons;
  cons.pos = per * blockIdx.x;
  cons.end = cons.pos + per;
  if (cons.end > total) cons.end = total;
  if (cons.pos >= cons.end) return;
  for (int64_t done = 0, b0 = 0; b0 < p.B; b0 += THREADS) {
    const int b = static_cast<int>(b0) + threadIdx.x;
    const int64_t w = b < p.B ? weight(p, request(p, b, ROWS)) : 0;
    int64_t incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int64_t before = done;
    for (int i = 0; i < warp; ++i) before += scan[i];
    const int64_t hi = before + incl, lo = hi - w;
    if (lo <= cons.pos && cons.pos < hi) {
      start_b = b;
      start_base = lo;
    }
    for (int i = 0; i < WARPS; ++i) done += scan[i];
    __syncthreads();
    if (done > cons.pos) break;
  }
  cons.b = start_b;
  cons.base = start_base;
  cons.r = request(p, cons.b, ROWS);

  // ---------------------------------------------------------------- loads of this warp's chunks
  const uint32_t ring = smem_addr(smem) + warp * STAGES * G::STAGE;
  Cursor prod = cons;
  Segment ps;
  bool pmore = next_segment<ROWS>(p, prod, ps);
  int pc = pmore ? ps.c0 + warp : 0;
  int page = 0;  // cache block of chunk pc, fetched one chunk ahead of its use
  auto settle = [&]() {  // moves pc to this warp's next chunk and looks its block up
    while (pmore && pc >= ps.c1) {
      pmore = next_segment<ROWS>(p, prod, ps);
      pc = ps.c0 + warp;
    }
    if (pmore) {
      page = p.block_tables[static_cast<int64_t>(ps.b) * p.bt_stride + pc / (PAGE / CHUNK)];
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) page = 0;
    }
  };
  auto fetch = [&](int stage) {
    if (pmore) {
      const int64_t off = (static_cast<int64_t>(page) * p.hk + ps.h) * G::PAGE_BYTES;
      const int sub = pc % (PAGE / CHUNK);
      const uint32_t dst = ring + stage * G::STAGE;
      const uint8_t* kc = p.k_cache + off + sub * G::CODES;
      const uint8_t* vc = p.v_cache + off + sub * G::CODES;
#pragma unroll
      for (int i = 0; i < CHUNK * G::PIECES / 32; ++i) {
        const int idx = i * 32 + lane, r = idx / G::PIECES, q = idx % G::PIECES;
        cp16(dst + key_at<D>(r, q), kc + idx * 16);
        cp16(dst + G::CODES + value_at<D>(r, q), vc + idx * 16);
      }
      const int half = lane >> 4, i = lane & 15;
      if (i < G::SCALES / 16)
        cp16(dst + 2 * G::CODES + half * G::SCALES + i * 16,
             (half ? p.v_cache : p.k_cache) + off + PAGE * G::ROW + sub * G::SCALES + i * 16);
      pc += WARPS;
      settle();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  settle();
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(s);

  // ---------------------------------------------------------------- segments
  int it = 0;
  Segment s;
  while (next_segment<ROWS>(p, cons, s)) {
    uint32_t qf[NT][KSTEPS][2];
    float cs[NT][2], m[NT][2], l[NT][2];
    int64_t pos[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int n = 8 * j + g;
      float f = 1.f, inv = 1.f;
      uint4 raw[D / 32];
      if (n < s.rows) {
        const int rr = s.row0 + n;
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (s.qs + rr / group) * p.q_stride +
                                                          static_cast<int64_t>(s.h * group + rr % group) * D + t * (D / 4));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) raw[i] = src[i];
      } else {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) raw[i] = make_uint4(0, 0, 0, 0);
      }
      uint32_t top = 0;  // largest magnitude's bf16 bits: its exponent is all that is needed
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = min(267 - static_cast<int>(top >> 7), 253);  // biased exponent of the row's factor
      f = __uint_as_float(static_cast<uint32_t>(e) << 23);
      inv = __uint_as_float(static_cast<uint32_t>(254 - e) << 23) * p.scale_log2;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          qf[j][2 * i + k / 2][k & 1] =
              pack_f16(__uint_as_float(w[k] << 16) * f, __uint_as_float(w[k] & 0xffff0000u) * f);
      }
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        cs[j][e2] = __shfl_sync(0xffffffffu, inv, (2 * t + e2) * 4);
        pos[j][e2] = s.ctx0 + (s.row0 + 8 * j + 2 * t + e2) / group;
        m[j][e2] = -FLT_MAX;
        l[j][e2] = 0.f;
      }
    }
    const int64_t safe = s.ctx0 + s.row0 / group;  // the tile's first position: keys up to it need no mask
    float o[NT][MT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;

#pragma unroll 1
    for (int c = s.c0 + warp; c < s.c1; c += WARPS, ++it) {
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      fetch((it + STAGES - 1) % STAGES);
      const uint8_t* st = smem + warp * STAGES * G::STAGE + (it % STAGES) * G::STAGE;
      const int64_t key0 = static_cast<int64_t>(c) * CHUNK;
      const bool edge = key0 + CHUNK - 1 > safe;
      // -------- S^T = K Q^T
      float sc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
      {
        uint32_t kw[2][KW];
        uint32_t ksc[2][D / 64];  // the scale of each 16 dimensions, twice
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int r = g + 8 * hf;
          if constexpr (D == 64) {
            const uint2 v = *reinterpret_cast<const uint2*>(st + key_at<D>(r, t >> 1) + (t & 1) * 8);
            kw[hf][0] = v.x;
            kw[hf][1] = v.y;
          } else {
#pragma unroll
            for (int i = 0; i < D / 128; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(st + key_at<D>(r, t * (D / 128) + i));
              kw[hf][4 * i] = v.x;
              kw[hf][4 * i + 1] = v.y;
              kw[hf][4 * i + 2] = v.z;
              kw[hf][4 * i + 3] = v.w;
            }
          }
          const uint8_t* sp = st + 2 * G::CODES + r * G::SROW + t * (D / 64);
          uint32_t w;
          if constexpr (D == 64) w = *sp;
          if constexpr (D == 128) w = *reinterpret_cast<const uint16_t*>(sp);
          if constexpr (D == 256) w = *reinterpret_cast<const uint32_t*>(sp);
#pragma unroll
          for (int i = 0; i < D / 64; i += 2) {
            const uint32_t pr = e4m3x2(w >> (8 * i));
            ksc[hf][i] = __byte_perm(pr, 0, 0x1010);
            if constexpr (D > 64) ksc[hf][i + 1] = __byte_perm(pr, 0, 0x3232);
          }
        }
#pragma unroll
        for (int w = 0; w < KW; ++w) {  // 8 codes: two k-steps
          uint32_t lo[4], hi[4];
          e2m1x8(kw[0][w], lo);
          e2m1x8(kw[1][w], hi);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t a[4] = {hmul2(lo[2 * k], ksc[0][w / 2]), hmul2(hi[2 * k], ksc[1][w / 2]),
                                   hmul2(lo[2 * k + 1], ksc[0][w / 2]), hmul2(hi[2 * k + 1], ksc[1][w / 2])};
#pragma unroll
            for (int j = 0; j < NT; ++j) mma(sc[j], a, qf[j][2 * w + k][0], qf[j][2 * w + k][1]);
          }
        }
      }
      // -------- softmax over the tokens (rows g and g + 8; columns 2t and 2t + 1)
      bool grow = false;
      float x[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[j][e] = fmaf(sc[j][e], cs[j][e & 1], -m[j][e & 1]);
          if (edge && key0 + g + 8 * (e >> 1) > pos[j][e & 1]) x[j][e] = -INFINITY;
          grow |= x[j][e] > kSlack;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // the scores themselves: x holds their distance from m, which is no help while m is -FLT_MAX
            float mx = -FLT_MAX;
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              if (!(edge && key0 + g + 8 * hf > pos[j][e])) mx = fmaxf(mx, sc[j][e + 2 * hf] * cs[j][e]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            // a row moves by its own scores alone, whatever its neighbours do
            const float to = mx - m[j][e] > kSlack ? mx : m[j][e];
            const float al = ex2(m[j][e] - to);
            m[j][e] = to;
            l[j][e] *= al;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[j][i][e] *= al;
              o[j][i][2 + e] *= al;
            }
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              if (!(edge && key0 + g + 8 * hf > pos[j][e])) x[j][e + 2 * hf] = fmaf(sc[j][e + 2 * hf], cs[j][e], -to);
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = ex2(x[j][e]);
        l[j][0] += pr[0] + pr[2];
        l[j][1] += pr[1] + pr[3];
        pb[j][0] = transpose8x8(pack_f16(pr[0], pr[1]));
        pb[j][1] = transpose8x8(pack_f16(pr[2], pr[3]));
      }
      // -------- O^T += V^T P^T
      {
        const uint8_t* vs = st + G::CODES;
        uint32_t vw[4][VB / 4];
        uint32_t vsc[2][D / 128 + (D == 64)];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
          const int r = 2 * t + (i & 1) + 8 * (i >> 1);
          if constexpr (D == 64) vw[i][0] = *reinterpret_cast<const uint32_t*>(vs + value_at<D>(r, g >> 2) + (g & 3) * 4);
          if constexpr (D == 128) {
            const uint2 v = *reinterpret_cast<const uint2*>(vs + value_at<D>(r, g >> 1) + (g & 1) * 8);
            vw[i][0] = v.x;
            vw[i][1] = v.y;
          }
          if constexpr (D == 256) {
            const uint4 v = *reinterpret_cast<const uint4*>(vs + value_at<D>(r, g));
            vw[i][0] = v.x;
            vw[i][1] = v.y;
            vw[i][2] = v.z;
            vw[i][3] = v.w;
          }
        }
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const int r = 2 * t + 8 * pr;
          const uint8_t* sp = st + 2 * G::CODES + G::SCALES + r * G::SROW;
          uint32_t a, b;
          if constexpr (D == 64) {
            a = sp[g >> 1];
            b = sp[G::SROW + (g >> 1)];
          }
          if constexpr (D == 128) {
            a = sp[g];
            b = sp[G::SROW + g];
          }
          if constexpr (D == 256) {
            a = *reinterpret_cast<const uint16_t*>(sp + 2 * g);
            b = *reinterpret_cast<const uint16_t*>(sp + G::SROW + 2 * g);
          }
          if (edge) {  // a token that no sequence owns: its codes are finite, its scale may be anything
            if (key0 + r >= s.kv_end) a = 0;
            if (key0 + r + 1 >= s.kv_end) b = 0;
          }
          if constexpr (D == 256) {
            vsc[pr][0] = e4m3x2(__byte_perm(a, b, 0x0040));
            vsc[pr][1] = e4m3x2(__byte_perm(a, b, 0x0051));
          } else {
            vsc[pr][0] = e4m3x2(a | (b << 8));
          }
        }
#pragma unroll
        for (int w = 0; w < VB / 4; ++w) {  // 8 dimensions: four M tiles
          uint32_t ev[2][4], od[2][4];
#pragma unroll
          for (int pr = 0; pr < 2; ++pr) {
            const uint32_t a = vw[2 * pr][w], b = vw[2 * pr + 1][w];
            e2m1x8((a & 0x0f0f0f0fu) | ((b << 4) & 0xf0f0f0f0u), ev[pr]);  // even dimensions, tokens 2t | 2t + 1
            e2m1x8(((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u), od[pr]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t s0 = vsc[0][D == 256 ? w / 2 : 0], s1 = vsc[1][D == 256 ? w / 2 : 0];
            const uint32_t a[4] = {hmul2(ev[0][i], s0), hmul2(od[0][i], s0), hmul2(ev[1][i], s1), hmul2(od[1][i], s1)};
#pragma unroll
            for (int j = 0; j < NT; ++j) mma(o[j][4 * w + i], a, pb[j][0], pb[j][1]);
          }
        }
      }
    }

    // -------------------------------------------------------------- the warps' states become one
    const bool whole = s.pg0 == 0 && s.pg1 == s.pages;
    const int slot = 2 * blockIdx.x + (s.pg0 > 0 ? 0 : 1);
    float* part = p.part_o + static_cast<int64_t>(slot) * ROWS * (D + 2);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = l[j][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) {
          merge_m[warp * ROWS + 8 * j + 2 * t + e] = m[j][e];
          merge_l[warp * ROWS + 8 * j + 2 * t + e] = v;
        }
      }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (8 * j >= s.rows) break;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float* dst = merge_o + (warp * 8 + 2 * t + e) * K::MSTRIDE + g * (D / 8);
#pragma unroll
        for (int i = 0; i < MT; i += 2)
          *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[j][i][e], o[j][i][2 + e], o[j][i + 1][e], o[j][i + 1][2 + e]);
      }
      __syncthreads();
      constexpr int DT = D / 32;  // dimensions of a thread: warp w holds row w of the tile
      const int row = 8 * j + warp;
      float top = -FLT_MAX, sum = 0.f, acc[DT];
#pragma unroll
      for (int i = 0; i < DT; ++i) acc[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge_m[w * ROWS + row]);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float wt = ex2(merge_m[w * ROWS + row] - top);
        sum += wt * merge_l[w * ROWS + row];
        const float* src = merge_o + (w * 8 + warp) * K::MSTRIDE + lane * DT;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] += wt * src[i];
      }
      if (row < s.rows) {
        if (whole) {
          const float inv = sum == 0.f ? 0.f : p.v_scale / sum;  // no key at all: 0 (a NaN stays one)
          const int rr = s.row0 + row;
          __nv_bfloat16* dst = p.out + (s.qs + rr / group) * p.out_stride + static_cast<int64_t>(s.h * group + rr % group) * D + lane * DT;
#pragma unroll
          for (int i = 0; i < DT; i += 2)
            *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
        } else {
          float* dst = part + row * D + lane * DT;
#pragma unroll
          for (int i = 0; i < DT; ++i) dst[i] = acc[i];
          if (lane == 0) {
            part[ROWS * D + 2 * row] = top;
            part[ROWS * D + 2 * row + 1] = sum;
          }
        }
      }
      __syncthreads();
    }
    if (!whole) {
      const int first = static_cast<int>(s.u0 / per), last = static_cast<int>((s.u1 - 1) / per);
      if (threadIdx.x == 0) {
        __threadfence();
        const unsigned n = atomicAdd(&p.tickets[first], 1u);
        last_flag = n == static_cast<unsigned>(last - first);
        if (last_flag) p.tickets[first] = 0;
        __threadfence();
      }
      __syncthreads();
      if (last_flag) {
        constexpr int DT = D / 32;
        for (int row = warp; row < s.rows; row += WARPS) {
          float top = -FLT_MAX, sum = 0.f, acc[DT];
#pragma unroll
          for (int i = 0; i < DT; ++i) acc[i] = 0.f;
          auto at = [&](int c) {
            return p.part_o + static_cast<int64_t>(2 * c + (c == first ? 1 : 0)) * ROWS * (D + 2);
          };
          for (int c = first + lane; c <= last; c += 32) top = fmaxf(top, __ldcg(at(c) + ROWS * D + 2 * row));
#pragma unroll
          for (int o2 = 16; o2 > 0; o2 >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o2));
#pragma unroll 4
          for (int c = first; c <= last; ++c) {
            const float* src = at(c);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + ROWS * D + 2 * row));
            const float wt = ex2(ml.x - top);
            sum += wt * ml.y;
#pragma unroll
            for (int i = 0; i < DT; i += 2) {
              const float2 v = __ldcg(reinterpret_cast<const float2*>(src + row * D + lane * DT + i));
              acc[i] += wt * v.x;
              acc[i + 1] += wt * v.y;
            }
          }
          const float inv = sum == 0.f ? 0.f : p.v_scale / sum;  // no key at all: 0 (a NaN stays one)
          const int rr = s.row0 + row;
          __nv_bfloat16* dst = p.out + (s.qs + rr / group) * p.out_stride + static_cast<int64_t>(s.h * group + rr % group) * D + lane * DT;
#pragma unroll
          for (int i = 0; i < DT; i += 2)
            *reinterpret_cast<__nv_bfloat162*>(dst + i) = __floats2bfloat162_rn(acc[i] * inv, acc[i + 1] * inv);
        }
      }
      __syncthreads();  // last_flag is rewritten by the next segment
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

}  // namespace attn4
}  // namespace shk

using namespace shk::attn4;

namespace {
constexpr int kMaxDevices = 64;

int num_sms() {
  static int sms[kMaxDevices] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms[dev];
}

template <int D, int NT>
int launch(const AttnFp4Params& p, cudaStream_t st) {
  using K = Cfg<D, NT>;
  static_assert(K::CTAS * (K::SMEM + 1200) <= 227 * 1024, "shared-memory budget");
  static bool ready[kMaxDevices] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -5;
  auto k = attn_fp4_kernel<D, NT>;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, K::SMEM);
    if (e != cudaSuccess) return 300 + static_cast<int>(e);
    ready[dev] = true;
  }
  const int ctas = K::CTAS * num_sms();
  if (ctas <= 0) return -5;
  const cudaError_t e = shk::launch(k, dim3(ctas), dim3(THREADS), K::SMEM, st, p);
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
}  // namespace

// f(D, NT) of the instantiation for (head_dim, row_tile); `none` for a pair that has none.
#define SH_ATTN4_DISPATCH(head_dim, row_tile, none, ...)          \
  switch ((head_dim) * 8 + (row_tile) / 8) {                      \
    case 64 * 8 + 1: { constexpr int D = 64, NT = 1; __VA_ARGS__ }  \
    case 64 * 8 + 2: { constexpr int D = 64, NT = 2; __VA_ARGS__ }  \
    case 64 * 8 + 3: { constexpr int D = 64, NT = 3; __VA_ARGS__ }  \
    case 64 * 8 + 4: { constexpr int D = 64, NT = 4; __VA_ARGS__ }  \
    case 128 * 8 + 1: { constexpr int D = 128, NT = 1; __VA_ARGS__ } \
    case 128 * 8 + 2: { constexpr int D = 128, NT = 2; __VA_ARGS__ } \
    case 128 * 8 + 3: { constexpr int D = 128, NT = 3; __VA_ARGS__ } \
    case 128 * 8 + 4: { constexpr int D = 128, NT = 4; __VA_ARGS__ } \
    case 256 * 8 + 1: { constexpr int D = 256, NT = 1; __VA_ARGS__ } \
    case 256 * 8 + 2: { constexpr int D = 256, NT = 2; __VA_ARGS__ } \
    default: return none;                                         \
  }

extern "C" int sh_paged_attention_fp4_ctas(int head_dim, int row_tile) {
  SH_ATTN4_DISPATCH(head_dim, row_tile, 0, return Cfg<D, NT>::CTAS * num_sms();)
}

extern "C" int64_t sh_paged_attention_fp4_workspace(int head_dim, int row_tile) {
  return static_cast<int64_t>(sh_paged_attention_fp4_ctas(head_dim, row_tile)) * 2 * row_tile * (head_dim + 2);
}

extern "C" int sh_paged_attention_fp4(const AttnFp4Params* params, int head_dim, int row_tile, cudaStream_t stream) {
  const AttnFp4Params& p = *params;
  if (p.num_tokens <= 0 || p.B <= 0) return 0;
  if (p.hk <= 0 || p.hq % p.hk != 0 || p.num_blocks <= 0 || p.bt_cols <= 0) return -1;
  if (p.part_o == nullptr || p.tickets == nullptr) return -2;
  if ((reinterpret_cast<uintptr_t>(p.k_cache) & 15) || (reinterpret_cast<uintptr_t>(p.v_cache) & 15) ||
      (reinterpret_cast<uintptr_t>(p.q) & 15) || (p.q_stride & 7) || (reinterpret_cast<uintptr_t>(p.out) & 3) ||
      (p.out_stride & 1))
    return -3;
  SH_ATTN4_DISPATCH(head_dim, row_tile, -4, return launch<D, NT>(p, stream);)
}
