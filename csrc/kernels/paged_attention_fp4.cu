// Paged GQA attention over the 4-bit KV cache: decode, verify windows and (any length) short query runs.
//
//   o[t, h] = g_v sum_j softmax_j(q[t, h] . k[j] g_k scale) v[j],   j <= position of t
//   k[j], v[j] = e2m1 code x e4m3 block scale (16 dimensions), read as they lie in the pages.
//
// Work.  A unit is (request, kv head, tile of NT * 8 packed query rows); packed row r of a request is token r / G,
// head r % G of the group, so the heads of a group and the tokens of a verify window share one read of the keys.
// The units, each as long as its pages and a constant for its start and end, are laid end to end and cut into equal
// runs, one per CTA: a ragged batch loads every SM alike and no length has to be known on the host.  A unit that a run's
// end leaves in two or more pieces has fp32 partials (O, max, sum); the last of its CTAs to finish (a ticket, which it
// resets) merges them in page order, so the result does not depend on the order of arrival.
//
// A CTA's warps take the run's 32-token chunks in turn, each through a ring of its own in shared memory, filled with
// cp.async: no barrier between the warps while they stream.  Per chunk and warp, with m16n8k16 (f16 in, fp32 out) and
// the KEYS on the M side, so 8 query rows fill the N side that decode has:
//   S^T (tokens x rows) = K Q^T,   O^T (D x rows) += V^T P^T.
// Both products are free to permute the dimension they sum over, or the rows of the result: thread (g, t) of the
// quad layout takes D/4 consecutive dimensions of a key as its share of K's columns, and D/8 consecutive dimensions
// as its share of V^T's rows, so its codes are one 8- to 32-byte run of a row and one or two scales cover them.
// V^T's pairs of adjacent tokens come from interleaving the nibbles of two tokens' words (a shift and a lop3 per 8
// codes).  e2m1 -> f16 is exact, and so is the product with the e4m3 scale (at most 6 significant bits, between
// 2^-10 and 2688).  Q goes to f16 after a multiplication by a power of two per row (its largest element into
// [2^13, 2^14), which keeps bf16's 8 bits for elements down to 2^-30 of it; smaller ones lose bits, and below 2^-38 they
// vanish); the power leaves with the softmax scale.  P is rounded to f16: 11 bits, where bf16 would cost as much again as
// the output's own rounding.  Against the reference's 1 a weight below 2^-14 has fewer bits, and one below 2^-25 counts in
// the sum alone.
//
// The softmax keeps, per row, a reference m that moves only when a score exceeds it by more than 8 (in log2 units):
// P <= 2^8 stays far from f16's range, and a chunk costs one vote instead of a reduction over the tokens.
//
// What bounds it (times of a call among others).  Many keys and 8 rows: memory, behind the decoding (8 requests of 131072
// keys, 32 heads of 128, 8 kv heads: 1.18 GB in 261 us, 69% of the copy rate).  Short runs: the way to the first key and
// the merges, about 10 us of latency around 22 pages (64 requests of 2048: 115 MB in 36 us, 49%; 24 of 4000 at head_dim
// 256: 40 MB in 23 us, 27%; 64 of 4096 with 8 heads of 64: 29 MB in 18 us, 24%).  Wide windows: 255 registers leave two
// warps a scheduler, which wait for their own results (32 windows of 6 tokens, 24 rows: 233 MB in 97 us, 37%, 43% of the
// issue slots and 41% of the tensor pipe's cycles).
// Whole units (batch-invariant calls) are never cut: those 8 requests then run on 64 CTAs, in 2260 us, and a prompt of
// 8192 takes 4000 us here where the tensor-core kernel takes 620.
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

constexpr int PAGE = 64;  // tokens of a page
constexpr float kSlack = 8.f;
constexpr int kUnit = 8;       // pages' worth of work that a unit costs besides its pages
constexpr int kTable = 16;     // requests of a run that are kept in shared memory

template <int D>
struct Geo {
  static constexpr int ROW = D / 2;              // code bytes of a token
  static constexpr int SROW = D / 16;            // scale bytes of a token
  static constexpr int PAGE_BYTES = PAGE * (ROW + SROW);
  static constexpr int PIECES = ROW / 16;        // 16-byte pieces of a token's codes
};
// Warps of a CTA, CTAs of an SM, 16-token groups of a warp step (a chunk) and ring stages.  O^T takes D / 4 registers a
// thread for every 8 rows: with 32 of them a thread fits 128 registers and an SM 16 warps, beyond that 8 (255).  At
// head_dim 128 the CTAs have 4 warps, so that their starts, merges and ends fall under one another's streaming (decode
// 64 x 2048: 42 us against 48 with CTAs of 8; 32 rows over 32 x 6000: 142 against 153); elsewhere 8 are better (decode
// 64 x 4096 at 64: 20 us against 23, 24 x 4000 at 256: 24 against 33).  Twelve or sixteen warps for the wider tiles, or
// a pair of warps to share a tile's dimensions, were slower (24 rows: 157 and 131 us against 109): they spill.
template <int D, int NT>
struct Cfg {
  static constexpr int REGS_O = D / 4 * NT;
  static constexpr int SUB = REGS_O <= 96 && NT <= 3 ? 2 : 1;
  static constexpr int WARPS = D == 128 ? 4 : 8;
  static constexpr int CTAS = (REGS_O <= 32 ? 16 : 8) / WARPS;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int CHUNK = 16 * SUB;
  static constexpr int CODES = CHUNK * Geo<D>::ROW;
  static constexpr int SCALES = CHUNK * Geo<D>::SROW;
  static constexpr int STAGE = 2 * (CODES + SCALES);
  static constexpr int MSTRIDE = D + 4;  // floats of a merge row
  static constexpr int MERGE = WARPS * 8 * MSTRIDE * 4;
  static constexpr int QUERY = 2 * NT * D * 16;  // the fragments of two row tiles, this unit's and the next one's
  static constexpr int STATS = 2 * WARPS * 8 * NT * 4 + 2 * 2 * 8 * NT * 4;
  static constexpr int ROOM = (227 - 2 * CTAS) * 1024 / CTAS - QUERY - STATS;
  // with two stages that leave no room for the merge area, it takes the ring's place after each unit
  static constexpr bool SHARED = 2 * WARPS * STAGE + MERGE > ROOM;
  static constexpr int FIT = (SHARED ? ROOM : ROOM - MERGE) / (WARPS * STAGE);
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int SMEM = (SHARED ? (RING > MERGE ? RING : MERGE) : RING + MERGE) + QUERY + STATS;
  static_assert(STAGES >= 2, "a chunk in flight while another is used");
  // A unit's start and end cost about as much as kUnit pages, and it is cut into pieces of two chunks a warp at least.
  static constexpr int MIN_PAGES = 2 * WARPS * CHUNK / PAGE > 1 ? 2 * WARPS * CHUNK / PAGE : 1;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
template <int DST, int SRC>
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0+%2], [%1+%3], 16;" ::"r"(dst), "l"(src), "n"(DST), "n"(SRC) : "memory");
}
// Pieces I, I + 1, ... < N of this lane, 512 bytes apart on both sides; the odd ones go to another base.
template <int I, int N>
__device__ __forceinline__ void cp_pieces(uint32_t even, uint32_t odd, const void* src) {
  if constexpr (I < N) {
    cp16<512 * I, 512 * I>(I & 1 ? odd : even, src);
    cp_pieces<I + 1, N>(even, odd, src);
  }
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
  int64_t qs;
  int seq, q_len, tiles, pages;
};
__device__ __forceinline__ Request request(const AttnFp4Params& p, int b, int rows) {
  Request r;
  const int64_t q0 = p.q_start[b], q1 = p.q_start[b + 1];
  r.qs = q0 < 0 ? 0 : q0;
  const int64_t n = (q1 < p.num_tokens ? q1 : p.num_tokens) - r.qs;
  r.q_len = n > 0 ? static_cast<int>(n) : 0;
  int64_t seq = p.seq_lens[b];
  if (seq < 0) seq = 0;
  const int64_t cap = static_cast<int64_t>(p.bt_cols) * PAGE;  // below 2^31: bt_cols is at most 2^25 - 1
  r.seq = static_cast<int>(seq < cap ? seq : cap);
  r.tiles = static_cast<int>((static_cast<int64_t>(r.q_len) * (p.hq / p.hk) + rows - 1) / rows);
  r.pages = (r.seq + (PAGE - 1)) / PAGE;
  if (r.pages < 1) r.pages = 1;  // a request without keys still has its rows to write
  return r;
}
__device__ __forceinline__ int64_t weight(const AttnFp4Params& p, const Request& r) {
  return static_cast<int64_t>(r.tiles) * p.hk * (r.pages + kUnit);
}
// A unit of `pages` cut `at` its start + at: the page there, moved to an end of the unit where a piece would be short.
template <int MIN_PAGES>
__device__ __forceinline__ int cut_page(int64_t at, int pages) {
  const int64_t page = at - kUnit;
  if (page < MIN_PAGES) return 0;
  return page > pages - MIN_PAGES ? pages : static_cast<int>(page);
}

// a / b of non-negative numbers, short where both are short.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// One unit's part in a CTA's run.
struct Segment {
  int64_t u0;  // the unit's place among all
  int64_t qs;
  int b, h, row0, rows, ctx0, kv_end, pages;
  int c0, c1;        // chunks with keys that some row sees
  bool whole, head;  // all of the unit; its beginning
};
// Walks a CTA's run [pos, end) of the units laid end to end; each one follows from the last without a division.
struct Cursor {
  int64_t pos, end, next;  // the run, and where the next unit begins
  int b, tile, h;
  Request r;
};
template <int ROWS, int CHUNK, int MIN_PAGES>
__device__ __forceinline__ bool next_segment(const AttnFp4Params& p, const Request* table, int table_b, Cursor& c, Segment& s) {
  const int g = p.hq / p.hk;
  while (true) {
    if (c.next >= c.end) return false;
    if (++c.h == p.hk) {
      c.h = 0;
      ++c.tile;
    }
    while (c.tile >= c.r.tiles) {
      ++c.b;
      c.r = table != nullptr && c.b - table_b < kTable ? table[c.b - table_b] : request(p, c.b, ROWS);
      c.tile = 0;
    }
    s.u0 = c.next;
    s.pages = c.r.pages;
    c.next = s.u0 + s.pages + kUnit;
    // whole units belong to the run that they begin in; others to each run that holds enough of them
    int pg0, pg1;
    if (p.whole_units) {
      if (s.u0 < c.pos) continue;
      pg0 = 0;
      pg1 = s.pages;
    } else {
      pg0 = s.u0 >= c.pos ? 0 : cut_page<MIN_PAGES>(c.pos - s.u0, s.pages);
      pg1 = c.next <= c.end ? s.pages : cut_page<MIN_PAGES>(c.end - s.u0, s.pages);
      if (pg0 >= pg1) continue;
    }
    s.head = pg0 == 0;
    s.whole = s.head && pg1 == s.pages;
    s.b = c.b;
    s.h = c.h;
    s.row0 = c.tile * ROWS;
    const int64_t left = static_cast<int64_t>(c.r.q_len) * g - s.row0;
    s.rows = left < ROWS ? static_cast<int>(left) : ROWS;
    s.qs = c.r.qs;
    s.ctx0 = c.r.seq - c.r.q_len;
    int kv = s.ctx0 + (s.row0 + s.rows - 1) / g + 1;  // keys the tile's last row sees
    kv = kv < 0 ? 0 : (kv < c.r.seq ? kv : c.r.seq);
    s.kv_end = kv;
    s.c0 = pg0 * (PAGE / CHUNK);
    const int last = kv / CHUNK + (kv % CHUNK ? 1 : 0);
    s.c1 = pg1 * (PAGE / CHUNK) < last ? pg1 * (PAGE / CHUNK) : last;
    return true;
  }
}
// The first and the last run that hold a piece of the unit (by the rule of cut_page, on runs of `per`).
template <int MIN_PAGES>
__device__ __forceinline__ int2 runs_of(const Segment& s, int64_t per) {
  const int64_t end = s.u0 + s.pages + kUnit;
  const int64_t at_end = quotient(end - 1, per);
  const int64_t a = quotient(s.u0 + kUnit + MIN_PAGES + per - 1, per) - 1;  // its end leaves a piece behind it
  const int64_t first = a < at_end ? a : at_end;
  const int64_t z = s.pages >= MIN_PAGES ? quotient(s.u0 + kUnit + s.pages - MIN_PAGES, per) : first;
  const int64_t last = z < at_end ? z : at_end;
  return make_int2(static_cast<int>(first), static_cast<int>(last < first ? first : last));
}

template <int D, int NT>
__global__ void __launch_bounds__(Cfg<D, NT>::THREADS, (Cfg<D, NT>::CTAS)) attn_fp4_kernel(AttnFp4Params p) {
  using G = Geo<D>;
  using K = Cfg<D, NT>;
  constexpr int ROWS = 8 * NT, WARPS = K::WARPS, THREADS = K::THREADS, STAGES = K::STAGES;
  constexpr int CHUNK = K::CHUNK, SUB = K::SUB;
  constexpr int SCOUT = THREADS - 32;  // walks the run's units, in the last warp: it has the fewest queries to convert
  constexpr int MT = D / 16;  // M tiles of O^T
  constexpr int KW = D / 32;  // words of a key in a thread (D/4 codes), two k-steps each
  constexpr int VW = D / 64;  // words of a value in a thread (D/8 codes), four M tiles each
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge_o = reinterpret_cast<float*>(smem + (K::SHARED ? 0 : K::RING));
  uint4* query2 = reinterpret_cast<uint4*>(smem + K::SMEM - K::STATS - K::QUERY);  // [2][NT][KW][32 lanes]
  float* merge_m = reinterpret_cast<float*>(smem + K::SMEM - K::STATS);           // [WARPS][ROWS]
  float* merge_l = merge_m + WARPS * ROWS;
  float* row_scale2 = merge_l + WARPS * ROWS;                      // [2][ROWS]
  int* row_pos2 = reinterpret_cast<int*>(row_scale2 + 2 * ROWS);  // [2][ROWS] last key a row sees
  __shared__ int64_t scan[WARPS];
  __shared__ int start_b;
  __shared__ Request table[kTable];  // of requests start_b, start_b + 1, ...
  __shared__ Cursor cursor;
  // this unit, the next one and the one behind it; the one before may still be read when that one is written
  __shared__ Segment segs[4];
  __shared__ int seg_ok[4];
  __shared__ Segment open[2];  // units that this CTA has a partial of: at most the run's first and last
  __shared__ int last_flag[2];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int group = p.hq / p.hk;
  shk::pdl_trigger();
  shk::pdl_wait();  // lengths, tables, queries and the new tokens' rows come from earlier kernels

  // ---------------------------------------------------------------- this CTA's run
  // The first THREADS requests' pages are summed and searched in one pass, which is all for most batches.
  int64_t first_w = 0, rest = 0;
  Request mine = {};
  if (threadIdx.x < p.B) {
    mine = request(p, threadIdx.x, ROWS);
    first_w = weight(p, mine);
  }
  for (int b = threadIdx.x + THREADS; b < p.B; b += THREADS) rest += weight(p, request(p, b, ROWS));
  auto scan_warps = [&](int64_t w, int64_t& all) {  // inclusive over the block; a barrier lies between two calls
    int64_t incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    int64_t before = 0;
    all = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      before += i < warp ? scan[i] : 0;
      all += scan[i];
    }
    return before + incl;
  };
  int64_t total = 0, done;
  if (p.B > THREADS) {
    (void)scan_warps(rest, total);
    __syncthreads();
  }
  int64_t incl = scan_warps(first_w, done);
  total += done;
  int64_t per = quotient(total + gridDim.x - 1, gridDim.x);
  if (per < K::MIN_PAGES) per = K::MIN_PAGES;
  const int64_t run = per * blockIdx.x;
  if (run >= total) return;
  auto advance = [&](Cursor c, const Request* known, int slot) {  // one thread: the next unit of the run
    Segment sg;
    seg_ok[slot] = next_segment<ROWS, CHUNK, K::MIN_PAGES>(p, known, start_b, c, sg);
    segs[slot] = sg;
    cursor = c;
  };
  // The thread whose request the run begins in goes to its first unit at once.
  auto take = [&](int b, const Request& r, int64_t base) {
    start_b = b;
    Cursor c;
    c.pos = run;
    c.end = run + per < total ? run + per : total;
    c.r = r;
    const int64_t unit = quotient(run - base, r.pages + kUnit);
    c.b = b;
    c.tile = static_cast<int>(quotient(unit, p.hk));
    c.h = static_cast<int>(unit - static_cast<int64_t>(c.tile) * p.hk) - 1;  // the cursor stands before it
    c.next = base + unit * (r.pages + kUnit);
    advance(c, nullptr, 0);
  };
  if (incl - first_w <= run && run < incl) take(threadIdx.x, mine, incl - first_w);
  for (int64_t b0 = THREADS; done <= run; b0 += THREADS) {
    __syncthreads();
    const int64_t b = b0 + threadIdx.x;
    Request other = {};
    int64_t w = 0, all;
    if (b < p.B) {
      other = request(p, static_cast<int>(b), ROWS);
      w = weight(p, other);
    }
    incl = done + scan_warps(w, all);
    if (incl - w <= run && run < incl) take(static_cast<int>(b), other, incl - w);
    done += all;
  }
  __syncthreads();

  // ---------------------------------------------------------------- loads of this warp's chunks
  const uint32_t ring = smem_addr(smem) + warp * STAGES * K::STAGE;
  // where this lane's pieces of a chunk go: piece i * 32 + lane is row i * 512 / ROW + lane / PIECES
  const uint32_t kdst = ring + key_at<D>(lane / G::PIECES, lane % G::PIECES);
  const uint32_t vdst = ring + K::CODES + value_at<D>(lane / G::PIECES, lane % G::PIECES);
  // The loads run ahead into the next unit at most.
  int pc = 0, pc1 = 0, page = 0;  // this warp's next chunk, the unit's end, the chunk's cache block
  int at = -1, asked = 0;         // the unit whose chunks are being asked for; chunks asked for so far
  const int32_t* pages = nullptr;
  int64_t head = 0;  // the unit's head inside a block
  auto look_up = [&]() {
    page = pages[pc / (PAGE / CHUNK)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_blocks)) page = 0;
  };
  auto begin = [&](const Segment& sg) {
    pc = sg.c0 + warp;
    pc1 = sg.c1;
    pages = p.block_tables + static_cast<int64_t>(sg.b) * p.bt_stride;
    head = static_cast<int64_t>(sg.h) * G::PAGE_BYTES;
    ++at;
    if (pc < pc1) look_up();
  };
  auto fetch = [&]() {  // the next chunk, if there is one
    if (pc < pc1) {
      const int stage = asked % STAGES;
      ++asked;
      const int64_t off = static_cast<int64_t>(page) * p.hk * G::PAGE_BYTES + head;
      const int part = pc % (PAGE / CHUNK);
      const uint32_t kd = kdst + stage * K::STAGE, vd = vdst + stage * K::STAGE;
      cp_pieces<0, K::CODES / 512>(kd, kd, p.k_cache + off + part * K::CODES + lane * 16);
      // head_dim 256: a value row's place in its line turns with every second row, so with every second piece
      cp_pieces<0, K::CODES / 512>(vd, D == 256 ? vd ^ 64 : vd, p.v_cache + off + part * K::CODES + lane * 16);
      constexpr int N = K::SCALES / 16;  // pieces of the scales: the keys' for the first half of the warp
      const int half = lane >> 4, i = lane & 15;
      const uint8_t* sc = (half ? p.v_cache : p.k_cache) + off + PAGE * G::ROW + part * K::SCALES + i * 16;
      const uint32_t sd = ring + stage * K::STAGE + 2 * K::CODES + half * K::SCALES + i * 16;
      if (i < N) cp16<0, 0>(sd, sc);
      if constexpr (N > 16) cp16<256, 256>(sd, sc);
      pc += WARPS;
      if (pc < pc1) look_up();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int it = 0;

  // per-lane places of the fragments in a chunk: keys g (+ 8, ...), values 2 t and 2 t + 1 (+ 8, ...)
  const int koff0 = key_at<D>(g, D == 64 ? t >> 1 : t * (D / 128)) + (D == 64 ? (t & 1) * 8 : 0);
  const int koff1 = D == 256 ? key_at<D>(g, t * 2 + 1) : 0;
  const int vp = D == 256 ? g : (D == 128 ? g >> 1 : g >> 2), vb = D == 256 ? 0 : (D == 128 ? (g & 1) * 8 : (g & 3) * 4);
  const int voff0 = K::CODES + value_at<D>(2 * t, vp) + vb, voff1 = K::CODES + value_at<D>(2 * t + 1, vp) + vb;
  const int ksoff = 2 * K::CODES + g * G::SROW + t * (D / 64);
  const int vsoff = 2 * K::CODES + K::SCALES + 2 * t * G::SROW + (D == 64 ? g >> 1 : (D == 128 ? g : 2 * g));

  // ---------------------------------------------------------------- segments
  int opened = 0, unit = 0;  // partials left and units done so far; unit's parity: its half of query2
  auto row_of = [&](const Segment& sg, int n) {  // row n's queries, this lane's dimensions
    const int rr = sg.row0 + n;
    return reinterpret_cast<const uint4*>(p.q + (sg.qs + rr / group) * p.q_stride +
                                          static_cast<int64_t>(sg.h * group + rr % group) * D + t * (D / 4));
  };
  // The row tile's fragments, a warp per 8 rows: lane (g, t) has dimensions [t D/4, (t + 1) D/4) of row g, word u of its
  // codes against query2[half][j][u][lane].
  static_assert(NT <= WARPS, "a warp per 8 rows");
  struct Rows {
    uint4 raw[D / 32];
  };
  auto load_rows = [&](const Segment& sg) {
    Rows x;
    const int n = 8 * warp + g;
    const bool valid = warp < NT && n < sg.rows;
    const uint4* src = row_of(sg, valid ? n : 0);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) x.raw[i] = valid ? src[i] : make_uint4(0, 0, 0, 0);
    return x;
  };
  auto convert = [&](const Segment& sg, int half, const Rows& x) {
    if (warp < NT) {
      const int j = warp, n = 8 * j + g;
      const uint4* raw = x.raw;
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
      const float f = __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = pack_f16(__uint_as_float(w[k] << 16) * f, __uint_as_float(w[k] & 0xffff0000u) * f);
        query2[((half * NT + j) * KW + i) * 32 + lane] = make_uint4(o[0], o[1], o[2], o[3]);
      }
      if (t == 0) {
        row_scale2[half * ROWS + n] = __uint_as_float(static_cast<uint32_t>(254 - e) << 23) * p.scale_log2;
        row_pos2[half * ROWS + n] = sg.ctx0 + (sg.row0 + n) / group;
      }
    }
  };
  Rows first = {};
  if (seg_ok[0]) {
    first = load_rows(segs[0]);
    begin(segs[0]);  // the first keys are on their way before the queries are looked at
    do fetch();
    while (asked < STAGES - 1 && pc < pc1);
  }
  {
    const int i = static_cast<int>(threadIdx.x) - start_b;  // start_b + i is this thread's request, if it is among the first
    if (i >= 0 && i < kTable && threadIdx.x < p.B) table[i] = mine;
    if (start_b + kTable > THREADS && threadIdx.x < kTable && start_b + threadIdx.x >= THREADS && start_b + threadIdx.x < p.B)
      table[threadIdx.x] = request(p, start_b + threadIdx.x, ROWS);
  }
  __syncthreads();
  if (seg_ok[0]) {
    if (threadIdx.x == SCOUT) advance(cursor, table, 1);
    convert(segs[0], 0, first);
  }
  __syncthreads();
  for (; seg_ok[unit % 4]; ++unit) {
    const Segment& s = segs[unit % 4];
    const Segment& sn = segs[(unit + 1) % 4];
    const bool have = seg_ok[(unit + 1) % 4];
    const int turn = unit & 1, c_end = s.c1, kv_end = s.kv_end;
    const uint4* query = query2 + turn * NT * KW * 32;
    const float* row_scale = row_scale2 + turn * ROWS;
    const int* row_pos = row_pos2 + turn * ROWS;
    if (have && warp < NT && 8 * warp + g < sn.rows)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(row_of(sn, 8 * warp + g)));
    // what of the ring could not be filled under the unit before
    if (at < unit) begin(s);
    while (asked < it + STAGES - 1 && pc < pc1) fetch();
    float cs[NT][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        cs[j][e] = row_scale[8 * j + 2 * t + e];
        m[j][e] = -FLT_MAX;
        l[j][e] = 0.f;
      }
    const int safe = row_pos[0];  // the tile's first position: keys up to it need no mask
    float o[NT][MT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) o[j][i][0] = o[j][i][1] = o[j][i][2] = o[j][i][3] = 0.f;

#pragma unroll 1
    for (int c = s.c0 + warp; c < c_end; c += WARPS, ++it) {
      // a group per chunk: with a full ring STAGES - 2 later ones may still be under way
      if (asked - it < STAGES - 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
      __syncwarp();
      if (!K::SHARED && pc >= pc1 && at == unit && have) begin(sn);
      fetch();
      const uint8_t* st = smem + warp * STAGES * K::STAGE + (it % STAGES) * K::STAGE;
      const int key0 = c * CHUNK;
      const bool edge = key0 + CHUNK - 1 > safe;
      // -------- S^T = K Q^T
      float sc[SUB][NT][4];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int j = 0; j < NT; ++j) sc[u][j][0] = sc[u][j][1] = sc[u][j][2] = sc[u][j][3] = 0.f;
      {
        uint32_t kw[2 * SUB][KW];
        uint32_t ksc[2 * SUB][D / 64];  // the scale of each 16 dimensions, twice
#pragma unroll
        for (int hf = 0; hf < 2 * SUB; ++hf) {  // rows g + 8 hf
          const uint8_t* kp = st + koff0 + 8 * hf * G::ROW;
          if constexpr (D == 64) {
            const uint2 v = *reinterpret_cast<const uint2*>(kp);
            kw[hf][0] = v.x;
            kw[hf][1] = v.y;
          } else {
#pragma unroll
            for (int i = 0; i < D / 128; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(i ? st + koff1 + 8 * hf * G::ROW : kp);
              kw[hf][4 * i] = v.x;
              kw[hf][4 * i + 1] = v.y;
              kw[hf][4 * i + 2] = v.z;
              kw[hf][4 * i + 3] = v.w;
            }
          }
          const uint8_t* sp = st + ksoff + 8 * hf * G::SROW;
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
          uint4 qf[NT];
#pragma unroll
          for (int j = 0; j < NT; ++j) qf[j] = query[(j * KW + w) * 32 + lane];
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            uint32_t lo[4], hi[4];
            e2m1x8(kw[2 * u][w], lo);
            e2m1x8(kw[2 * u + 1][w], hi);
            const uint32_t s0 = ksc[2 * u][w / 2], s1 = ksc[2 * u + 1][w / 2];
            const uint32_t a0[4] = {hmul2(lo[0], s0), hmul2(hi[0], s1), hmul2(lo[1], s0), hmul2(hi[1], s1)};
            const uint32_t a1[4] = {hmul2(lo[2], s0), hmul2(hi[2], s1), hmul2(lo[3], s0), hmul2(hi[3], s1)};
#pragma unroll
            for (int j = 0; j < NT; ++j) mma(sc[u][j], a0, qf[j].x, qf[j].y);
#pragma unroll
            for (int j = 0; j < NT; ++j) mma(sc[u][j], a1, qf[j].z, qf[j].w);
          }
        }
      }
      // -------- softmax over the tokens (rows g and g + 8; columns 2t and 2t + 1)
      // token 16 u + g + 8 (e >> 1) of the chunk, row 8 j + 2 t + (e & 1)
      uint32_t hidden = 0;  // bit (u, j, e): the row does not see the key
      if (edge) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int behind = key0 + g + 8 * (e >> 1) - row_pos[8 * j + 2 * t + (e & 1)];
#pragma unroll
            for (int u = 0; u < SUB; ++u) hidden |= static_cast<uint32_t>(behind + 16 * u > 0) << ((u * NT + j) * 4 + e);
          }
      }
      float x[SUB][NT][4];
      float far = -FLT_MAX;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][j][e] = fmaf(sc[u][j][e], cs[j][e & 1], -m[j][e & 1]);
      if (edge) {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hidden >> ((u * NT + j) * 4 + e) & 1) x[u][j][e] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) far = fmaxf(far, x[u][j][e]);
      if (__any_sync(0xffffffffu, far > kSlack)) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // the scores themselves: x holds their distance from m, which is no help while m is -FLT_MAX
            float mx = -FLT_MAX;
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf)
                if (!(hidden >> ((u * NT + j) * 4 + e + 2 * hf) & 1)) mx = fmaxf(mx, sc[u][j][e + 2 * hf] * cs[j][e]);
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
            for (int u = 0; u < SUB; ++u)
#pragma unroll
              for (int hf = 0; hf < 2; ++hf)
                if (!(hidden >> ((u * NT + j) * 4 + e + 2 * hf) & 1))
                  x[u][j][e + 2 * hf] = fmaf(sc[u][j][e + 2 * hf], cs[j][e], -to);
          }
      }
      uint32_t pb[SUB][NT][2];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) pr[e] = ex2(x[u][j][e]);
          l[j][0] += pr[0] + pr[2];
          l[j][1] += pr[1] + pr[3];
          pb[u][j][0] = transpose8x8(pack_f16(pr[0], pr[1]));
          pb[u][j][1] = transpose8x8(pack_f16(pr[2], pr[3]));
        }
      // -------- O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        uint32_t vw[4][VW];
        uint32_t vsc[2][D == 256 ? 2 : 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // tokens 2t, 2t + 1, 2t + 8, 2t + 9
          const uint8_t* vpt = st + (i & 1 ? voff1 : voff0) + (16 * u + 8 * (i >> 1)) * G::ROW;
          if constexpr (D == 64) vw[i][0] = *reinterpret_cast<const uint32_t*>(vpt);
          if constexpr (D == 128) {
            const uint2 v = *reinterpret_cast<const uint2*>(vpt);
            vw[i][0] = v.x;
            vw[i][1] = v.y;
          }
          if constexpr (D == 256) {
            const uint4 v = *reinterpret_cast<const uint4*>(vpt);
            vw[i][0] = v.x;
            vw[i][1] = v.y;
            vw[i][2] = v.z;
            vw[i][3] = v.w;
          }
        }
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) {
          const int r = 16 * u + 8 * pr;
          const uint8_t* sp = st + vsoff + r * G::SROW;
          uint32_t a, b;
          if constexpr (D == 256) {
            a = *reinterpret_cast<const uint16_t*>(sp);
            b = *reinterpret_cast<const uint16_t*>(sp + G::SROW);
          } else {
            a = sp[0];
            b = sp[G::SROW];
          }
          if (edge) {  // a token that no sequence owns: its codes are finite, its scale may be anything
            if (key0 + r + 2 * t >= kv_end) a = 0;
            if (key0 + r + 2 * t + 1 >= kv_end) b = 0;
          }
          if constexpr (D == 256) {
            vsc[pr][0] = e4m3x2(__byte_perm(a, b, 0x0040));
            vsc[pr][1] = e4m3x2(__byte_perm(a, b, 0x0051));
          } else {
            vsc[pr][0] = e4m3x2(a | (b << 8));
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {  // 8 dimensions: four M tiles
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
            for (int j = 0; j < NT; ++j) mma(o[j][4 * w + i], a, pb[u][j][0], pb[u][j][1]);
          }
        }
      }
    }

    // (the barriers below stand before the use of both)
    if (have) convert(sn, turn ^ 1, load_rows(sn));
    if (threadIdx.x == SCOUT) {
      if (have) advance(cursor, table, (unit + 2) % 4);
      else seg_ok[(unit + 2) % 4] = 0;
    }
    // -------------------------------------------------------------- the warps' states become one
    if constexpr (K::SHARED) {  // no copy may land in the merge area
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
    }
    const bool whole = s.whole;
    const int slot = 2 * blockIdx.x + (s.head ? 1 : 0);
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
      constexpr int DT = D / 32;  // dimensions of a thread; a warp takes a row at a time
#pragma unroll 1
      for (int rt = warp; rt < 8; rt += WARPS) {
        const int row = 8 * j + rt;
        if (row >= s.rows) break;
        float top = -FLT_MAX, sum = 0.f, acc[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge_m[w * ROWS + row]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const float wt = ex2(merge_m[w * ROWS + row] - top);
          sum += wt * merge_l[w * ROWS + row];
          const float* src = merge_o + (w * 8 + rt) * K::MSTRIDE + lane * DT;
#pragma unroll
          for (int i = 0; i < DT; ++i) acc[i] += wt * src[i];
        }
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
      if (threadIdx.x == 0) open[opened] = s;
      ++opened;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (opened == 0) return;
  // ---------------------------------------------------------------- units cut by a run's end: the last CTA merges
  __syncthreads();
  if (threadIdx.x < opened) {
    const Segment& u = open[threadIdx.x];
    const int2 runs = runs_of<K::MIN_PAGES>(u, per);
    __threadfence();
    const bool mine = atomicAdd(&p.tickets[runs.x], 1u) == static_cast<unsigned>(runs.y - runs.x);
    if (mine) p.tickets[runs.x] = 0;
    last_flag[threadIdx.x] = mine;
    __threadfence();
  }
  __syncthreads();
  for (int i = 0; i < opened; ++i) {
    if (!last_flag[i]) continue;
    const Segment u = open[i];
    const int2 runs = runs_of<K::MIN_PAGES>(u, per);
    const int first = runs.x, last = runs.y;
    constexpr int DT = D / 32, BATCH = 4;
    auto at = [&](int c) { return p.part_o + static_cast<int64_t>(2 * c + (c == first ? 1 : 0)) * ROWS * (D + 2); };
    for (int row = warp; row < u.rows; row += WARPS) {
      float top = -FLT_MAX, sum = 0.f, acc[DT];
#pragma unroll
      for (int k = 0; k < DT; ++k) acc[k] = 0.f;
      for (int c0 = first; c0 <= last; c0 += BATCH) {
        float2 ml[BATCH], v[BATCH][DT / 2];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const float* src = at(c0 + b <= last ? c0 + b : last);
          ml[b] = __ldcg(reinterpret_cast<const float2*>(src + ROWS * D + 2 * row));
#pragma unroll
          for (int k = 0; k < DT / 2; ++k) v[b][k] = __ldcg(reinterpret_cast<const float2*>(src + row * D + lane * DT + 2 * k));
        }
        float to = top;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) to = fmaxf(to, ml[b].x);
        const float al = ex2(top - to);  // the batches before, on the new reference
        top = to;
        sum *= al;
#pragma unroll
        for (int k = 0; k < DT; ++k) acc[k] *= al;
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          if (c0 + b > last) break;
          const float wt = ex2(ml[b].x - top);
          sum += wt * ml[b].y;
#pragma unroll
          for (int k = 0; k < DT / 2; ++k) {
            acc[2 * k] += wt * v[b][k].x;
            acc[2 * k + 1] += wt * v[b][k].y;
          }
        }
      }
      const float inv = sum == 0.f ? 0.f : p.v_scale / sum;  // no key at all: 0 (a NaN stays one)
      const int rr = u.row0 + row;
      __nv_bfloat16* dst = p.out + (u.qs + rr / group) * p.out_stride + static_cast<int64_t>(u.h * group + rr % group) * D + lane * DT;
#pragma unroll
      for (int k = 0; k < DT; k += 2)
        *reinterpret_cast<__nv_bfloat162*>(dst + k) = __floats2bfloat162_rn(acc[k] * inv, acc[k + 1] * inv);
    }
  }
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
  static_assert(K::CTAS * (K::SMEM + 1300) <= 228 * 1024 && K::SMEM <= 226 * 1024, "shared-memory budget");
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
  const cudaError_t e = shk::launch(k, dim3(ctas), dim3(K::THREADS), K::SMEM, st, p);
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
  if (p.hk <= 0 || p.hq % p.hk != 0 || p.num_blocks <= 0 || p.bt_cols <= 0 || p.bt_cols >= 1 << 25) return -1;
  if (p.part_o == nullptr || p.tickets == nullptr) return -2;
  if ((reinterpret_cast<uintptr_t>(p.k_cache) & 15) || (reinterpret_cast<uintptr_t>(p.v_cache) & 15) ||
      (reinterpret_cast<uintptr_t>(p.q) & 15) || (p.q_stride & 7) || (reinterpret_cast<uintptr_t>(p.out) & 3) ||
      (p.out_stride & 1))
    return -3;
  SH_ATTN4_DISPATCH(head_dim, row_tile, -4, return launch<D, NT>(p, stream);)
}
