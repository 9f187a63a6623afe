// Paged GQA attention over the 4-bit KV cache on the 5th-generation tensor cores: prompts, chunks of prompts and
// wide verify windows (paged_attention_fp4.cu states the mathematics and serves short queries).
//
// Work.  A unit is (request, kv head, NQ tiles of 128 packed query rows) that share every key tile, so a key is decoded
// once per 256 rows (128 at head_dim 256, where two accumulators do not fit TMEM).  The units are laid end to end,
// each as long as its share of the causal triangle (w_i = (ctx + c) G + (i + 1) ROWS for row tile i, less the rows before
// the first key, c for a unit's start and end: integers with a closed-form sum, so any place is found by bisection), and
// cut into one run per SM.  A unit cut by a run's end leaves fp32 partials, which a second kernel merges in order.  (The
// last CTA of a unit doing it alone, as the short-query kernel does, pulls 133 KB per partial through one SM: 64 tokens
// over 20000 took 101 us.)
//
// Per CTA (16 warps; 13 at head_dim 256):
//   4 NQ warps       a warpgroup per query tile: load its rows, scale each by a power of two into f16's range and store
//                    it for the MMA; then a row a thread (= its TMEM lane): per key tile read S, softmax in the exp2
//                    domain against a reference that moves only when a score passes it by more than 8, write P (f16)
//                    over S; at the end O / l, or the partial;
//   3 + 3 (4 + 4)    decode 64-key tiles (a page's head) of K and of V into f16 tiles (exact) in shared memory; the next
//                    two tiles' codes are on their way in registers (head_dim 256 with 3 + 3: a prompt of 4096 with 16
//                    heads took 360 us, with 5 + 5 255, with 4 + 4, a whole number of pieces a thread, 240);
//   NQ warps         issue the MMAs of a query tile each: S_q = Q_q K^T into one of two buffers, O_q += P_q V.  S of the
//                    next tile is issued before P of this one is waited for, so the softmax never waits for a product
//                    it could have had, and the products run under the other tile's (or buffer's) softmax.
// TMEM: S_q,b (64 columns each, P in their first 32), O_q (D columns each) from column 256.
//
// What bounds it.  No single pipe: a prompt of 8192 with 32 heads of 128 takes 626 us (878 TFLOP/s, 53% of the rate of a
// large bf16 product), a chunk of 2000 at 32768 keys 1088 us (957 TFLOP/s, 57%), calls among others with their merges;
// a prompt of 4096 has about half of the issue slots, half of the tensor pipe's cycles and 40% of the special-function
// unit's.  In a probe where the chunk took 1020, it took 808 without the softmax and 1014 without the decoding: the chain
// S, weights, product of one query tile hides behind the other's only in part.  Registers decide much: with the run's
// cursor in them, not in shared memory, both took 3% more, and with the search for the first unit in each role's walk a
// prompt of 4096 with 16 heads of 256 took 212 us, not 199.
// Tried and slower: 128-key tiles with one S buffer, setmaxnreg splits (1110 us: the producers spill), a third tile's
// codes in registers (1090), the tile's sum as the sign that the reference must move, in place of its maximum (1081), S
// of two tiles in one product (1247, where the same code took 1079 with one), results through shared memory (1078).  A
// prompt of 4096 with 16 heads of 256 takes 199 us (690 TFLOP/s, 41%): one query tile, whose softmax and products wait
// for each other.  One of 8192 with 8 heads of 64 takes 142 us (485 TFLOP/s, 29%): half the products for each exponential.
//
// Every wait is bounded (2 s); one that runs out records 600 + role (1 producers, 2 products, 3 softmax) in *err and
// raises the CTA's abort flag, the rows of the CTA's units become NaN, and the CTA drains its MMAs and frees its TMEM
// before it returns.
#include <float.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_attention_fp4.h"
#include "pdl.cuh"
#include "tcgen05_common.cuh"

namespace shk {
namespace attn4tc {

using namespace shk::tc;

constexpr int PAGE = 64;
constexpr int KT = PAGE;  // keys per tile
constexpr float kSlack = 8.f;
constexpr int kMergeDims = 16;
constexpr int kMinTiles = 4;  // shortest piece of a unit that is cut
constexpr int kUnit = 512;  // a unit's start and end in keys (measured: 256 and 1024 leave the SMs less even)

template <int D>
struct Smem {
  static constexpr int NQ = D == 256 ? 1 : 2;     // query tiles
  static constexpr int ROWS = 128 * NQ;           // query rows per unit
  static constexpr int FIRST = 4 * NQ;            // first producer warp
  static constexpr int PRODUCERS = NQ == 1 ? 4 : 3;       // warps each for K and V
  static constexpr int MMA_WARP = FIRST + 2 * PRODUCERS;  // and one for each query tile
  static constexpr int THREADS = (MMA_WARP + NQ) * 32;
  static constexpr int STAGES = D == 256 ? 2 : 4;
  static constexpr int SLABS = D / 64;            // 64 dimensions: one 128-byte swizzle row
  static constexpr int QSLAB = 128 * 128;         // 128 rows of one slab
  static constexpr int KSLAB = KT * 128;
  static constexpr int QTILE = SLABS * QSLAB;
  static constexpr int KTILE = SLABS * KSLAB;
  static constexpr int Q = 0;                     // [NQ]
  static constexpr int K = Q + NQ * QTILE;        // [STAGES]
  static constexpr int V = K + STAGES * KTILE;    // [STAGES]
  static constexpr int BAR = V + STAGES * KTILE;
  static constexpr int TOTAL = BAR + 512 + 1024;  // + alignment slack
};

__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFF);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFF) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFF) << 32;
  d |= static_cast<uint64_t>(1) << 46;  // version
  d |= static_cast<uint64_t>(2) << 61;  // SWIZZLE_128B
  return d;
}
// kind::f16, D f32, A and B f16, A K-major, B K- or MN-major.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_mn_major) {
  return (1u << 4) | (b_mn_major ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(
          d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// 32 columns of this thread's lane, without a wait; ld_wait() names the registers, so their uses stay behind it.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void e2m1x8(uint32_t w, uint32_t* o) {
  asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
      " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
      " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}
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
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float2 ex2_pair(uint64_t v) {
  const float2 x = unpair(v);
  return make_float2(ex2(x.x), ex2(x.y));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}

// What a request asks for, clipped to the tensors it indexes.
struct Request {
  int64_t qs, seq, ctx;  // ctx: tokens before the new ones (negative: as many new ones come before the first key)
  int q_len, tiles;
};
template <int ROWS>
__device__ __forceinline__ Request request(const AttnFp4Params& p, int b) {
  Request r;
  const int64_t q0 = p.q_start[b], q1 = p.q_start[b + 1];
  r.qs = q0 < 0 ? 0 : q0;
  const int64_t n = (q1 < p.num_tokens ? q1 : p.num_tokens) - r.qs;
  r.q_len = n > 0 ? static_cast<int>(n) : 0;
  r.seq = p.seq_lens[b];
  if (r.seq < 0) r.seq = 0;
  const int64_t cap = static_cast<int64_t>(p.bt_cols) * PAGE;
  if (r.seq > cap) r.seq = cap;
  r.ctx = r.seq - r.q_len;
  r.tiles = static_cast<int>((static_cast<int64_t>(r.q_len) * (p.hq / p.hk) + ROWS - 1) / ROWS);
  return r;
}
// Cost of a request's row tile i, one kv head: the keys it sees (times the group) and kUnit keys for what a unit costs
// besides; and of its first n tiles.  Rows before the first key count for nothing: a cost that ran ahead of a unit's key
// tiles would leave some run in the unit's middle without one, and the merge expects a partial of each.
template <int ROWS>
__device__ __forceinline__ int64_t tile_cost(const Request& r, int group, int64_t i) {
  const int64_t w = (r.ctx + kUnit) * group + (i + 1) * ROWS, least = kUnit * group;
  return w > least ? w : least;
}
template <int ROWS>
__device__ __forceinline__ int64_t cost(const Request& r, int group, int64_t n) {
  const int64_t a = r.ctx < 0 ? -r.ctx * group / ROWS : 0;  // tiles without a key
  const int64_t seen = n > a ? (n - a) * r.ctx * group + ROWS * ((n * (n + 1) - a * (a + 1)) / 2) : 0;
  return n * kUnit * group + seen;
}

// A unit of `tiles` key tiles and cost w, cut where `at` of w lies behind: the tile there, moved to an end of the unit
// where a piece would be short.
__device__ __forceinline__ int cut_tile(int64_t at, int64_t tiles, int64_t w) {
  const int64_t t = at * tiles / w;
  if (t < kMinTiles) return 0;
  return static_cast<int>(t > tiles - kMinTiles ? tiles : t);
}

struct Segment {
  int64_t u0, u1;  // the unit's place among all costs
  int64_t qs, ctx0, kv_end;
  int b, h, row0, rows, k0, k1;  // key tiles [k0, k1) of the unit
  bool whole, head;              // all of the unit; its beginning
  bool none;                     // this run has no part in it
};
// Walks a CTA's run [pos, end) of the units laid end to end; each one follows from the last without a division.
struct Cursor {
  int64_t pos, end, r0;  // r0: what of the first unit lies before the run
  int b, tile, h;
  Request r;
};
template <int ROWS>
__device__ __forceinline__ bool next_segment(const AttnFp4Params& p, Cursor& c, Segment& s) {
  if (c.pos >= c.end) return false;
  const int g = p.hq / p.hk;
  const int64_t r0 = c.r0;
  c.r0 = 0;
  if (++c.h == p.hk) {
    c.h = 0;
    ++c.tile;
    while (c.tile >= c.r.tiles) {
      c.r = request<ROWS>(p, ++c.b);
      c.tile = 0;
    }
  }
  s.b = c.b;
  s.h = c.h;
  s.row0 = c.tile * ROWS;
  const int64_t left = static_cast<int64_t>(c.r.q_len) * g - s.row0;
  s.rows = left < ROWS ? static_cast<int>(left) : ROWS;
  s.qs = c.r.qs;
  s.ctx0 = c.r.ctx;
  int64_t kv = s.ctx0 + (s.row0 + s.rows - 1) / g + 1;  // keys the tile's last row sees
  if (kv > c.r.seq) kv = c.r.seq;
  if (kv < 0) kv = 0;
  s.kv_end = kv;
  const int64_t tiles = (kv + KT - 1) / KT, w = tile_cost<ROWS>(c.r, g, c.tile);
  s.u0 = c.pos - r0;
  s.u1 = s.u0 + w;
  s.k0 = r0 == 0 ? 0 : cut_tile(r0, tiles, w);
  s.k1 = c.end >= s.u1 ? static_cast<int>(tiles) : cut_tile(c.end - s.u0, tiles, w);
  // a piece without tiles is nobody's, but a unit without any belongs to the run that ends it
  s.none = s.k0 >= s.k1 && !(tiles == 0 && c.end >= s.u1);
  s.head = s.k0 == 0;
  s.whole = s.head && s.k1 == tiles;
  c.pos = c.end < s.u1 ? c.end : s.u1;
  return true;
}

// Run `run` of `runs`: its place among all units and the request it begins in.  Every thread of the block calls it;
// returns the length of a run.
template <int ROWS, int N>
__device__ __forceinline__ int64_t find_run(const AttnFp4Params& p, int run, int runs, Cursor& cur) {
  __shared__ int64_t scan[N / 32];
  __shared__ int64_t start_base;
  __shared__ int start_b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = p.hq / p.hk;
  auto weight = [&](int64_t b) {
    if (b >= p.B) return int64_t(0);
    const Request r = request<ROWS>(p, static_cast<int>(b));
    return cost<ROWS>(r, group, r.tiles) * p.hk;
  };
  int64_t total = 0;
  for (int64_t b = threadIdx.x; b < p.B; b += N) total += weight(b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) scan[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < N / 32; ++w) total += scan[w];
  __syncthreads();
  int64_t per = (total + runs - 1) / runs;
  // A run in the middle of a unit is never without a tile: a unit of kv keys costs at most (kv + kUnit) G + ROWS, so for
  // the 9 tiles or more that leave cuts in its middle (kv > 512) a tile costs less than 2 KT G + ROWS / 9 < 4 KT G.
  const int64_t least = static_cast<int64_t>(kMinTiles) * KT * group;
  if (per < least) per = least;
  cur.pos = per * run;
  cur.end = cur.pos + per < total ? cur.pos + per : total;
  if (cur.pos < cur.end) {
    for (int64_t done = 0, b0 = 0; b0 < p.B; b0 += N) {
      const int64_t w = weight(b0 + threadIdx.x);
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
      if (lo <= cur.pos && cur.pos < hi) {
        start_b = static_cast<int>(b0) + threadIdx.x;
        start_base = lo;
      }
      for (int i = 0; i < N / 32; ++i) done += scan[i];
      __syncthreads();
      if (done > cur.pos) break;
    }
    cur.b = start_b;
    cur.r = request<ROWS>(p, cur.b);
    const int64_t off = cur.pos - start_base;
    int lo = 0, hi = cur.r.tiles - 1;  // the tile that holds `off`: its predecessors cost at most that
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cost<ROWS>(cur.r, group, mid) * p.hk <= off) lo = mid;
      else hi = mid - 1;
    }
    const int64_t in = off - cost<ROWS>(cur.r, group, lo) * p.hk, w = tile_cost<ROWS>(cur.r, group, lo);
    cur.tile = lo;
    cur.h = static_cast<int>(in / w) - 1;  // the cursor stands before it
    cur.r0 = in % w;
  }
  return per;
}

// A unit's partial of run c: O, then the reference and the sum, [D + 2][128] with the row last.  A run leaves two at
// most, the one that begins in it (and ends later) and the one that began earlier.
struct Split {
  int64_t qs;
  int last, rows, row0, h;  // the run that ends the unit (the own one or less: nothing to merge) and the unit
};
template <int D>
__device__ __forceinline__ Split* splits(const AttnFp4Params& p, int runs) {
  return reinterpret_cast<Split*>(p.part_o + static_cast<int64_t>(runs) * 2 * Smem<D>::NQ * (D + 2) * 128);
}
template <int D>
__device__ __forceinline__ float* partial(const AttnFp4Params& p, int c, bool begins, int q, int row) {
  return p.part_o + (static_cast<int64_t>(2 * c + (begins ? 1 : 0)) * Smem<D>::NQ + q) * (D + 2) * 128 + row;
}

// The last run that holds a piece of a unit that is cut: cut_tile of its beginning leaves tiles behind.
__device__ __forceinline__ int last_run(const Segment& s, int64_t per) {
  const int64_t w = s.u1 - s.u0, tiles = (s.kv_end + KT - 1) / KT;
  const int64_t at = (w * (tiles - kMinTiles + 1) - 1) / tiles;  // the last place with floor(at tiles / w) <= tiles - kMinTiles
  return static_cast<int>((s.u0 + at) / per);
}

// Eight values, one 16-byte chunk: 8 codes times their block's scale.
__device__ __forceinline__ uint4 decode8(uint32_t w, uint32_t s2) {
  uint32_t o[4];
  e2m1x8(w, o);
  return make_uint4(hmul2(o[0], s2), hmul2(o[1], s2), hmul2(o[2], s2), hmul2(o[3], s2));
}

template <int D>
__global__ void __launch_bounds__(Smem<D>::THREADS, 1) attn_fp4_tc_kernel(AttnFp4Params p) {
  using M = Smem<D>;
  constexpr int ROWS = M::ROWS, NQ = M::NQ, STAGES = M::STAGES, MMA_WARP = M::MMA_WARP;
  constexpr uint32_t T_S = 0, T_O = 256, T_COLS = 512;
  constexpr int PAGE_BYTES = PAGE * (D / 2 + D / 16);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + M::BAR);  // [2]
  uint64_t* kfull = qfull + 2;                                   // [STAGES], as the next three
  uint64_t* kempty = kfull + STAGES;
  uint64_t* vfull = kempty + STAGES;
  uint64_t* vempty = vfull + STAGES;
  uint64_t* sfull = vempty + STAGES;                             // [q][buffer]
  uint64_t* pfull = sfull + 4;                                   // [q][buffer]
  uint64_t* pvdone = pfull + 4;                                  // [q][buffer]: the product of that P is in O
  uint64_t* drain = pvdone + 4;                                  // [q]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = p.hq / p.hk;
  auto raise = [&](int role) {  // a wait ran out, here or in the warp whose code stands already
    if (lane != 0) return;
    if (p.err != nullptr) atomicCAS(p.err, 0, 600 + role);
    *abort_flag = 1;
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&qfull[i], 4);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&kfull[i], M::PRODUCERS);
      mbar_init(&kempty[i], NQ);
      mbar_init(&vfull[i], M::PRODUCERS);
      mbar_init(&vempty[i], NQ);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sfull[i], 1);
      mbar_init(&pfull[i], 4);
      mbar_init(&pvdone[i], 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(T_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  shk::pdl_trigger();
  shk::pdl_wait();  // lengths, tables, queries and the new tokens' rows come from earlier kernels

  __shared__ Cursor saved[4 * NQ];
  Cursor cur;
  const int64_t per = find_run<ROWS, M::THREADS>(p, blockIdx.x, gridDim.x, cur);
  if (threadIdx.x == 0) splits<D>(p, gridDim.x)[blockIdx.x].last = -1;
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  Segment s = {};

  if (warp >= M::FIRST && warp < MMA_WARP) {
    // ------------------------------------------------------------------ producers
    // A thread decodes 16-byte pieces (32 dimensions of a key): piece i of a tile is dimensions 32 (i % PR) .. of
    // key i / PR, so a warp's loads are one run of memory.
    constexpr int PR = D / 32, PIECES = KT * PR, STEP = M::PRODUCERS * 32, N = (PIECES + STEP - 1) / STEP;
    const bool value = warp >= M::FIRST + M::PRODUCERS;  // this warp's matrix
    const int tid = threadIdx.x - (M::FIRST + (value ? M::PRODUCERS : 0)) * 32;
    const uint8_t* cache = value ? p.v_cache : p.k_cache;
    struct Codes {
      uint4 w[N];
      uint32_t sc[N];
    };
    bool more;
    int asked = 0;  // tiles asked for so far
    int kt, blk, nxt;  // the tile whose codes are asked for next, its block and the following tile's
    auto block_of = [&](int tile) {
      int b = static_cast<int64_t>(tile) * KT < s.kv_end ? p.block_tables[static_cast<int64_t>(s.b) * p.bt_stride + tile] : 0;
      return static_cast<unsigned>(b) < static_cast<unsigned>(p.num_blocks) ? b : 0;
    };
    auto settle = [&]() {  // the next unit with keys
      do {
        more = next_segment<ROWS>(p, cur, s);
      } while (more && s.k0 >= s.k1);
      kt = s.k0;
      if (more) {
        blk = block_of(kt);
        nxt = block_of(kt + 1);
      }
    };
    auto fetch = [&]() {  // the next tile's codes, wherever its unit
      Codes c = {};
      if (!more) return c;
      ++asked;
      const uint8_t* pg = cache + (static_cast<int64_t>(blk) * p.hk + s.h) * PAGE_BYTES;
      const int64_t left = s.kv_end - static_cast<int64_t>(kt) * KT;
      const int live = left < KT ? static_cast<int>(left) * PR : PIECES;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int idx = i * STEP + tid;
        if (idx < live) {  // a key that no row sees is a zero, whatever its page holds
          c.w[i] = *reinterpret_cast<const uint4*>(pg + idx * 16);
          c.sc[i] = *reinterpret_cast<const uint16_t*>(pg + PAGE * (D / 2) + idx * 2);
        }
      }
      if (++kt == s.k1) {
        settle();
      } else {
        blk = nxt;
        nxt = block_of(kt + 1);
      }
      return c;
    };
    // A thread's pieces are all the same 32 dimensions.  The threads of the second 64 write their four chunks in the
    // order 2, 3, 0, 1: in step with the first 64's they would meet in the same banks.
    static_assert(STEP % PR == 0, "a thread keeps its dimensions");
    const int d = tid % PR;
    const bool turned = D > 64 && (d & 2);
    const int ch = (d & 1) * 4 + (turned ? 2 : 0);
    auto store = [&](uint8_t* tile, const Codes& c) {
      uint8_t* slab = tile + (d >> 1) * M::KSLAB;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int idx = i * STEP + tid, r = idx / PR;
        if (idx >= PIECES) break;
        const uint32_t pr = e4m3x2(c.sc[i]);
        const uint32_t sa = __byte_perm(pr, 0, turned ? 0x3232 : 0x1010), sb = __byte_perm(pr, 0, turned ? 0x1010 : 0x3232);
        const uint32_t a0 = turned ? c.w[i].z : c.w[i].x, a1 = turned ? c.w[i].w : c.w[i].y;
        const uint32_t b0 = turned ? c.w[i].x : c.w[i].z, b1 = turned ? c.w[i].y : c.w[i].w;
        uint8_t* row = slab + r * 128;
        const int at = ch ^ (r & 7);  // chunk positions differ from it in their low two bits
        *reinterpret_cast<uint4*>(row + (at << 4)) = decode8(a0, sa);
        *reinterpret_cast<uint4*>(row + ((at ^ 1) << 4)) = decode8(a1, sa);
        *reinterpret_cast<uint4*>(row + ((at ^ 2) << 4)) = decode8(b0, sb);
        *reinterpret_cast<uint4*>(row + ((at ^ 3) << 4)) = decode8(b1, sb);
      }
      fence_proxy_async_smem();  // the decoded tile is read by the tensor cores
      __syncwarp();
    };
    uint64_t* full = value ? vfull : kfull;
    uint64_t* empty = value ? vempty : kempty;
    bool ok = true;
    settle();
    Codes now = fetch(), then = fetch();
#pragma unroll 1
    for (int n = 0; n < asked; ++n) {  // tile n fills stage n % STAGES
      const int st = n % STAGES, turn = n / STAGES;
      if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait(empty + st, (turn - 1) & 1, abort_flag))) {
        ok = false;
        break;
      }
      store(smem + (value ? M::V : M::K) + st * M::KTILE, now);
      if (lane == 0) mbar_arrive(full + st);
      now = then;
      then = fetch();
    }
    if (!ok) raise(1);
  } else if (warp >= MMA_WARP && warp < MMA_WARP + NQ) {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the loop, on values that the compiler can see to be uniform, and one elected lane (the same
    // each time) issues: operands then stay in uniform registers, where a lone lane's would be moved there for every
    // MMA (about 125 cycles an MMA instead of 25).
    constexpr uint32_t IS = idesc_f16(128, KT, false), IP = idesc_f16(128, D, true);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t sbase = __shfl_sync(0xffffffffu, smem_addr(smem), 0);
    const uint64_t kd = sw128_desc(sbase + M::K);
    const uint64_t vd = sw128_mn_desc(sbase + M::V, M::KSLAB, 1024);
    const int q = warp - MMA_WARP;
    const uint64_t qd = sw128_desc(sbase + M::Q + q * M::QTILE);
    const uint32_t ts = tm + T_S + q * 2 * KT, to = tm + T_O + q * D;
    int kc = 0, vc = 0, qc = 0, sc = 0, pc = 0;  // K and V tiles, queries, S and P so far
    bool ok = true;
    auto wait = [&](uint64_t* bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
    while (ok) {
      const bool more = next_segment<ROWS>(p, cur, s);
      if (!__shfl_sync(0xffffffffu, static_cast<int>(more), 0)) break;
      const bool mine = __shfl_sync(0xffffffffu, s.rows, 0) > q * 128;  // this tile has rows
      const int tiles = __shfl_sync(0xffffffffu, max(s.k1 - s.k0, 0), 0);
      if (tiles > 0 && mine) {
        ok = wait(&qfull[q], qc & 1);
        ++qc;
      }
#pragma unroll 1
      for (int j = -1; ok && j < tiles; ++j) {
        if (j + 1 < tiles) {  // S of tile j + 1
          const int st = kc % STAGES;
          ok = wait(&kfull[st], (kc / STAGES) & 1);
          if (!ok) break;
          ++kc;
          fence_after();
          if (elect_one()) {
            if (mine) {
              const uint64_t b = kd + static_cast<uint64_t>((st * M::KTILE) >> 4);
              const uint32_t d = ts + (sc & 1) * KT;
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk)
                mma_ss(d, qd + static_cast<uint64_t>(((kk >> 2) * M::QSLAB + (kk & 3) * 32) >> 4),
                       b + static_cast<uint64_t>(((kk >> 2) * M::KSLAB + (kk & 3) * 32) >> 4), IS, kk ? 1u : 0u);
              mma_commit(&sfull[q * 2 + (sc & 1)]);
            }
            mma_commit(&kempty[st]);
          }
          __syncwarp();
          sc += mine ? 1 : 0;
        }
        if (j >= 0) {  // O += P V of tile j
          const int st = vc % STAGES, buf = pc & 1;
          ok = wait(&vfull[st], (vc / STAGES) & 1) && (!mine || wait(&pfull[q * 2 + buf], (pc >> 1) & 1));
          if (!ok) break;
          ++vc;
          fence_after();
          if (elect_one()) {
            if (mine) {
              const uint64_t b = vd + static_cast<uint64_t>((st * M::KTILE) >> 4);
#pragma unroll
              for (int kk = 0; kk < KT / 16; ++kk)
                mma_ts(to, ts + buf * KT + kk * 8, b + static_cast<uint64_t>((kk * 2048) >> 4), IP, (j > 0 || kk > 0) ? 1u : 0u);
              mma_commit(&pvdone[q * 2 + buf]);
            }
            mma_commit(&vempty[st]);
          }
          __syncwarp();
          pc += mine ? 1 : 0;
        }
      }
    }
    if (!ok) raise(2);
    if (elect_one()) {
      mma_commit(&drain[q]);
      (void)mbar_wait_drain(&drain[q], 0);
    }
    __syncwarp();
  } else if (warp < 4 * NQ) {
    // ------------------------------------------------------------------ softmax + epilogue
    const int q = warp >> 2, r = threadIdx.x & 127;
    const uint32_t tl = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + tl + T_O + q * D;
    // S tiles seen so far.  A barrier belongs to one buffer: its next phase cannot complete before this warp has been
    // through the last, so a parity is never two phases old.
    int ns = 0;
    bool ok = true;
    // This thread's row of a unit: where it comes from and goes to, its scale, the last key it sees.
    struct Row {
      const uint4* src;
      __nv_bfloat16* dst;
      int64_t pos;
      float cs;
      bool valid;
    };
    auto advance = [&](Segment& sg) {  // the next unit in which this query tile has rows
      bool more;
      Cursor c = saved[warp];  // kept out of the registers, which the softmax needs
      do {
        more = next_segment<ROWS>(p, c, sg);
      } while (more && (q * 128 >= sg.rows || sg.none));
      __syncwarp();
      if (lane == 0) saved[warp] = c;
      __syncwarp();
      return more;
    };
    auto row_of = [&](const Segment& sg) {
      Row w;
      const int n = q * 128 + r, rr = sg.row0 + n;
      const int64_t tok = sg.qs + rr / group, col = static_cast<int64_t>(sg.h * group + rr % group) * D;
      w.valid = n < sg.rows;
      w.src = reinterpret_cast<const uint4*>(p.q + tok * p.q_stride + col);
      w.dst = p.out + tok * p.out_stride + col;
      w.pos = sg.ctx0 + rr / group;
      w.cs = 0.f;
      return w;
    };
    // A warp's 32 rows, scaled and in f16, into their tile.  A row is read by D / 8 lanes (read by its own thread alone,
    // each access touched 32 lines, and a unit waited 8 us for its queries).
    auto load_rows = [&](Row& w) {
      constexpr int LANES = D / 8, AT_ONCE = 32 / LANES, BATCH = 8;
      uint8_t* tile = smem + M::Q + q * M::QTILE + (warp & 3) * 32 * 128;
      const int i = lane % LANES;
      const uint64_t from = w.valid ? reinterpret_cast<uint64_t>(w.src) : 0;
      int own = 0;  // the exponent of this thread's row
#pragma unroll 1
      for (int b = 0; b < LANES; b += BATCH) {
        uint4 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const uint4* row = reinterpret_cast<const uint4*>(__shfl_sync(0xffffffffu, from, (b + k) * AT_ONCE + lane / LANES));
          v[k] = row != nullptr ? row[i] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int n = (b + k) * AT_ONCE + lane / LANES;
          const uint32_t w4[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          uint32_t top = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) top = max(top, max(w4[j] & 0x7fffu, (w4[j] >> 16) & 0x7fffu));
          if constexpr (LANES == 32) {
            top = __reduce_max_sync(0xffffffffu, top);
          } else {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
          }
          // its largest element goes into [2^13, 2^14); the softmax scale's sign goes with the row (0: a zero row), so
          // that cs > 0 and the largest S is the largest score
          const int e = min(267 - static_cast<int>(top >> 7), 253);
          const float f = p.scale_log2 == 0.f ? 0.f : copysignf(__uint_as_float(static_cast<uint32_t>(e) << 23), p.scale_log2);
          const int there = __shfl_sync(0xffffffffu, e, lane % AT_ONCE * LANES);
          if (lane / AT_ONCE == b + k) own = there;
          uint32_t o[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = pack_f16(__uint_as_float(w4[j] << 16) * f, __uint_as_float(w4[j] & 0xffff0000u) * f);
          *reinterpret_cast<uint4*>(tile + n * 128 + (i >> 3) * M::QSLAB + (((i & 7) ^ (n & 7)) << 4)) =
              make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
      w.cs = fmaxf(__uint_as_float(static_cast<uint32_t>(254 - own) << 23) * fabsf(p.scale_log2), FLT_MIN);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&qfull[q]);
    };
    if (lane == 0) saved[warp] = cur;
    __syncwarp();
    Segment sn;
    bool have = advance(sn), stored = false;
    Row next = {};
    if (have) next = row_of(sn);
    while (have) {
      s = sn;
      float m = -FLT_MAX, l = 0.f;
      const bool keys = s.k0 < s.k1;
      if (keys && ok && !stored) load_rows(next);
      const Row w = next;
      const float cs = w.cs;
      if (keys && ok) {
        // key tiles from here on hold keys that some row of this query tile does not see
        const int64_t seen = s.ctx0 + (s.row0 + q * 128) / group + 1;
        const int free_tiles = seen > 0 ? static_cast<int>(seen / KT) : 0;
        for (int kt = s.k0; kt < s.k1; ++kt, ++ns) {
          const int buf = q * 2 + (ns & 1);
          const uint32_t tS = tmem + tl + T_S + buf * KT;
          if (!__all_sync(0xffffffffu, mbar_wait(&sfull[buf], (ns >> 1) & 1, abort_flag))) {
            ok = false;
            break;
          }
          fence_after();
          uint64_t sum[2] = {0, 0};
          uint32_t x[64];
          ld32(tS, x);
          ld32(tS + 32, x + 32);
          ld_wait(x);
          ld_wait(x + 32);
          if (kt >= free_tiles) {
            // keys [0, lim) of the tile are this row's
            const int lim = static_cast<int>(min(max(w.pos + 1 - static_cast<int64_t>(kt) * KT, int64_t(0)), int64_t(KT)));
#pragma unroll
            for (int i = 0; i < 64; ++i)
              if (i >= lim) x[i] = __float_as_uint(-INFINITY);
          }
          const float* f = reinterpret_cast<const float*>(x);
          float t4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) t4[i] = max3(f[i], f[4 + i], f[8 + i]);
#pragma unroll
          for (int j = 12; j < 60; j += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i) t4[i] = max3(t4[i], f[j + i], f[j + 4 + i]);
#pragma unroll
          for (int i = 0; i < 4; ++i) t4[i] = fmaxf(t4[i], f[60 + i]);
          const float mx = fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]);
          const bool grow = fmaf(mx, cs, -m) > kSlack;
          if (__any_sync(0xffffffffu, grow)) {  // rare
            const float to = grow ? mx * cs : m;
            const float al = ex2(m - to);
            m = to;
            l *= al;
            if (kt > s.k0) {  // O must hold every earlier tile of the unit
              if (!__all_sync(0xffffffffu, mbar_wait(&pvdone[q * 2 + ((ns - 1) & 1)], ((ns - 1) >> 1) & 1, abort_flag))) {
                ok = false;
                break;
              }
              fence_after();
#pragma unroll 1
              for (int i = 0; i < D; i += 8) {
                uint32_t o[8];
                ld8(tO + i, o);
#pragma unroll
                for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * al);
                st8(tO + i, o);
              }
              st_wait();
            }
          }
          const uint64_t cs2 = pair(cs, cs), nm2 = pair(-m, -m);
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t v = fma2(pair(f[h + 2 * i], f[h + 2 * i + 1]), cs2, nm2);
              const float2 e = ex2_pair(v);
              sum[i & 1] = add2(sum[i & 1], pair(e.x, e.y));
              pk[i] = pack_f16(e.x, e.y);
            }
            st16(tS + h / 2, pk);
          }
          {
            const float2 a = unpair(sum[0]), b = unpair(sum[1]);
            l += (a.x + a.y) + (b.x + b.y);
          }
          st_wait();
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pfull[buf]);
        }
      }
      // the next unit's rows take the place of this one's, whose last S has been seen, under its last product
      have = advance(sn);
      if (have) next = row_of(sn);
      stored = have && ok && sn.k0 < sn.k1;
      if (stored) load_rows(next);
      if (keys) {
        if (ok && !__all_sync(0xffffffffu, mbar_wait(&pvdone[q * 2 + ((ns - 1) & 1)], ((ns - 1) >> 1) & 1, abort_flag)))
          ok = false;
        if (!ok) raise(3);
        fence_after();
      }
      if (!ok) l = __uint_as_float(0x7fc00000u);  // a wait ran out: NaN, not numbers
      const bool none = !keys || !ok;
      if (s.whole) {
        const float inv = l == 0.f ? 0.f : p.v_scale / l;  // no key at all: 0 (a NaN stays one)
        __nv_bfloat16* dst = w.dst;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (none) {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0;
          } else {
            ld32(tO + c, o);
            ld_wait(o);
          }
          if (w.valid) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                v[i] = pack_bf16(__uint_as_float(o[8 * k + 2 * i]) * inv, __uint_as_float(o[8 * k + 2 * i + 1]) * inv);
              *reinterpret_cast<uint4*>(dst + c + 8 * k) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        continue;
      }
      if (q == 0 && r == 0 && s.head)
        splits<D>(p, gridDim.x)[blockIdx.x] = {s.qs, last_run(s, per), s.rows, s.row0, s.h};
      float* mine = partial<D>(p, blockIdx.x, s.head, q, r);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        if (none) {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0;
        } else {
          ld32(tO + c, o);
          ld_wait(o);
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) mine[(c + k) * 128] = __uint_as_float(o[k]);
      }
      mine[D * 128] = m;
      mine[(D + 1) * 128] = l;
    }
  }
  fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(T_COLS));
  }
}

// The unit that run blockIdx.x begins and a later one ends, if there is one: its partials, in order.  blockIdx.y: query
// tile and kMergeDims of the dimensions; a thread holds a row.
template <int D>
__global__ void __launch_bounds__(128) merge_kernel(AttnFp4Params p, int runs) {
  constexpr int DC = kMergeDims;
  shk::pdl_trigger();
  shk::pdl_wait();
  const int q = blockIdx.y / (D / DC), d0 = blockIdx.y % (D / DC) * DC, r = threadIdx.x;
  const Split s = splits<D>(p, runs)[blockIdx.x];
  const int first = blockIdx.x, last = s.last;
  if (last <= first || q * 128 + r >= s.rows) return;
  float top = -FLT_MAX, den = 0.f, acc[DC];
#pragma unroll
  for (int k = 0; k < DC; ++k) acc[k] = 0.f;
#pragma unroll 8
  for (int c = first; c <= last; ++c) top = fmaxf(top, __ldcg(partial<D>(p, c, c == first, q, r) + D * 128));
  constexpr int BATCH = 4;  // partials whose loads are in flight together
  for (int c0 = first; c0 <= last; c0 += BATCH) {
    float v[BATCH][DC], m[BATCH], l[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int c = c0 + i <= last ? c0 + i : last;
      const float* src = partial<D>(p, c, c == first, q, r);
      m[i] = __ldcg(src + D * 128);
      l[i] = __ldcg(src + (D + 1) * 128);
#pragma unroll
      for (int k = 0; k < DC; ++k) v[i][k] = __ldcg(src + (d0 + k) * 128);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (c0 + i > last) break;
      const float wt = ex2(m[i] - top);
      den += wt * l[i];
#pragma unroll
      for (int k = 0; k < DC; ++k) acc[k] += wt * v[i][k];
    }
  }
  const float inv = den == 0.f ? 0.f : p.v_scale / den;  // no key at all: 0 (a NaN stays one)
  const int group = p.hq / p.hk, rr = s.row0 + q * 128 + r;
  __nv_bfloat16* dst = p.out + (s.qs + rr / group) * p.out_stride + static_cast<int64_t>(s.h * group + rr % group) * D + d0;
#pragma unroll
  for (int k = 0; k < DC; k += 8)
    *reinterpret_cast<uint4*>(dst + k) =
        make_uint4(pack_bf16(acc[k] * inv, acc[k + 1] * inv), pack_bf16(acc[k + 2] * inv, acc[k + 3] * inv),
                   pack_bf16(acc[k + 4] * inv, acc[k + 5] * inv), pack_bf16(acc[k + 6] * inv, acc[k + 7] * inv));
}

}  // namespace attn4tc
}  // namespace shk

using namespace shk::attn4tc;

namespace {
constexpr int kMaxDevices = 64;

int num_sms() {
  static int sms[kMaxDevices] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return sms[dev];
}

template <int D>
int launch(const AttnFp4Params& p, cudaStream_t st) {
  static_assert(Smem<D>::TOTAL + 256 <= 227 * 1024, "shared-memory budget");
  static bool ready[kMaxDevices] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return -5;
  auto k = attn_fp4_tc_kernel<D>;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D>::TOTAL);
    if (e != cudaSuccess) return 300 + static_cast<int>(e);
    ready[dev] = true;
  }
  const int ctas = num_sms();
  if (ctas <= 0) return -5;
  cudaError_t e = shk::launch(k, dim3(ctas), dim3(Smem<D>::THREADS), Smem<D>::TOTAL, st, p);
  if (e == cudaSuccess) e = shk::launch(merge_kernel<D>, dim3(ctas, Smem<D>::NQ * D / kMergeDims), dim3(128), 0, st, p, ctas);
  return e == cudaSuccess ? 0 : 400 + static_cast<int>(e);
}
}  // namespace

extern "C" int64_t sh_paged_attention_fp4_tc_workspace(int head_dim) {
  const int query_tiles = head_dim == 256 ? Smem<256>::NQ : Smem<128>::NQ;
  return static_cast<int64_t>(num_sms()) * (2 * query_tiles * (head_dim + 2) * 128 + sizeof(Split) / 4);
}

extern "C" int sh_paged_attention_fp4_tc(const AttnFp4Params* params, int head_dim, cudaStream_t stream) {
  const AttnFp4Params& p = *params;
  if (p.num_tokens <= 0 || p.B <= 0) return 0;
  if (p.hk <= 0 || p.hq % p.hk != 0 || p.num_blocks <= 0 || p.bt_cols <= 0 || p.whole_units) return -1;
  if (p.part_o == nullptr) return -2;
  if ((reinterpret_cast<uintptr_t>(p.k_cache) & 15) || (reinterpret_cast<uintptr_t>(p.v_cache) & 15) ||
      (reinterpret_cast<uintptr_t>(p.q) & 15) || (p.q_stride & 7) || (reinterpret_cast<uintptr_t>(p.out) & 15) ||
      (p.out_stride & 7))
    return -3;
  switch (head_dim) {
    case 64: return launch<64>(p, stream);
    case 128: return launch<128>(p, stream);
    case 256: return launch<256>(p, stream);
    default: return -4;
  }
}
