// Causal attention of several new tokens a sequence over a paged cache in 8 bits (fp8.cuh), on the 5th-generation tensor cores.
//
//   o_t = sum_j 2^(s_tj) c_j 2^(ev_j) / sum_j 2^(s_tj),   s_tj = scale log2(e) (q_t . k_j) 2^(ek_j),   j seen by t     (k, c: codes)
//
// Rows. A key/value head is read once for all of its query heads: the rows of a 128-row operand are (token, query head) pairs,
// 128 / G tokens of the G heads that share the key/value head. A block has two such tiles, A and B, with a softmax warpgroup
// each (a thread a row, its scores of a step in registers) and an issuing thread each; while one's softmax works, the tensor core is
// busy with the other's.
//
// Keys and values become half-precision numbers (exactly) on their way into shared memory: four warps load codes into
// registers a tile ahead, convert them and write the tensor core's operand layout. Their exponents stay out of the products:
// a block of 16 positions has one for its keys, which multiplies a score, and one for its values, which is added to it. So
// w = 2^(s + ev - R + 7) is what the codes of the values are weighted with, and the softmax's denominator takes w 2^(-ev).
// R is a running bound that follows the largest s + ev of the row only when that has grown by more than 8: w stays below
// 2^15, half precision holds it with 11 digits down to 2^-21 of the row's largest, and the sums in tensor memory have to be
// multiplied by 2^(R - R') in few tiles only. Queries are brought to half precision with a power of two a row, which keeps
// every digit of bfloat16. Weights go back to tensor memory as the second product's first operand.
//
// Work. A block takes one (sequence, tile of tokens, key/value head), or one of several equal runs of its key tiles where the
// step has too few of them for the GPU: how many runs a sequence's tiles are cut into is worked out on the device from the
// lengths that are there, so that a run is about a 148th of the step. Runs leave partial results, which a second kernel joins in order.
//
// Numbers that are not finite: a score that is NaN makes its row NaN by itself. A value that is NaN must reach the rows that see it
// and no other, and a product with a zero weight would spread it; so such codes enter the product as zeros, the tile is marked,
// and the rows that see one are told column by column.
#include "fp8.cuh"
#include "tcgen05.cuh"
#include <math.h>

namespace llmie {
using namespace tc;

constexpr int kPfRows = 128;         // rows of a tile
constexpr int kPfKeys = 128;         // keys of a step
constexpr int kPfThreads = 512;      // warps 0-3, 4-7: softmax of tiles A and B; 8-11: conversion; 12, 13: the products of A, of B; 14, 15: nothing
constexpr int kPfSub = kPfRows * 128;        // bytes of 128 rows of 64 half-precision numbers
constexpr int kPfSms = 148;
constexpr int kPfRing = 8;
constexpr int kPfNeedsScratch = -5;  // the answer to a call without scratch that cannot do without
constexpr int kPfLeast = 4;          // key tiles that a run has at least, on average
constexpr int kPfSlots = 200;        // partial results at once (see pf_run)
constexpr int kPfFew = 128;          // tiles of tokens that can always be cut into runs for which there are SMs (see pf_run)
constexpr float kPfTop = 7.f;        // the bound's own weight is 2^7
constexpr float kPfSlack = 8.f;      // how far scores may outgrow the bound, in units of log2

template <int HD> struct PfCfg {
  static constexpr int kSubs = HD / 64;
  static constexpr int kQBytes = kSubs * kPfSub;             // one tile of queries
  static constexpr int kKvBytes = kSubs * kPfSub;            // 128 keys, or values
  static constexpr int kStages = 2;
  static constexpr int kSmem = 2 * kQBytes + 2 * kStages * kKvBytes + 1024;
  static constexpr bool kOwnP = HD == 64;                    // tensor memory has room for the weights beside the scores
  static constexpr int kSCol = 0, kOCol = 256, kPCol = 384;  // columns: scores of A and B, sums of A and B, weights
  static constexpr int kRecord = 2 * kPfRows * (HD + 2);     // floats of a partial result: sums, then bounds, then denominators
};

// Registers that a thread of a softmax, the conversion and the last warpgroup keeps of the 128 that it is launched with: a row's 128
// scores stay in registers, a converting thread has a step's codes in them. (Head size 128, 192 / 176 for the softmax: pieces of 60
// to 1,500 tokens 84.9 / 87.8 us; where the tiles take turns and the conversion sets the pace, 24 sequences of 2 to 8 tokens, 70.2 / 58.5.)
template <int HD, bool TURNS> struct PfRegs {
  static constexpr int kSoftmax = HD == 64 ? 200 : TURNS ? 176 : 192, kConvert = HD == 64 ? 80 : TURNS ? 112 : 88,
                       kIssue = HD == 64 ? 32 : TURNS ? 48 : 40;
  static_assert(2 * kSoftmax + kConvert + kIssue == 4 * 128, "more than the block has would never be granted");
  static_assert(kSoftmax >= 128 && kConvert <= 128 && kIssue <= 128, "inc may only raise, dec only lower");
};

struct PrefillArgs {
  const __nv_bfloat16* q;
  const unsigned char* k;            // [pages, n_kv, 64, HD] codes
  const unsigned char* v;
  const signed char* k_exp;          // [pages, n_kv, 4]
  const signed char* v_exp;
  __nv_bfloat16* out;
  float* part;
  int* status;
  const int* cu_q;
  const int* seq_slot;
  const int* seq_start;
  const int* block_table;
  int max_pages, n_seqs, n_q, n_kv;
  float scale2;
  int window;
  int run;                           // no run is shorter: what the host counted blocks and scratch by
};

__device__ __forceinline__ float pf_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pf_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float pf_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// D[tmem] (+)= A[tmem] * B[smem], half precision
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void pf_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__host__ __device__ constexpr uint32_t pf_instr_desc(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);   // float32 += half * half
}

// ------------------------------------------------------------------------------------------ the cut of the work
// Key tiles of a sequence's tile of tokens [t0, t0 + n): from `lo` on, `count` of them. None behind the table's last page.
__device__ __forceinline__ void pf_tiles(const PrefillArgs& a, int start, int t0, int n, int& lo, int& count) {
  lo = first_visible_key(start + t0, a.window) / kPfKeys;
  count = max((min(start + t0 + n, a.max_pages * kFp8Page) - 1) / kPfKeys - lo + 1, 0);
}
// What a lane knows of its sequence: tiles of tokens, the key tiles of the first and the last of them.
struct PfSequence {
  int q_begin, q_len, start, slot, tiles, first, last;
};
__device__ __forceinline__ PfSequence pf_sequence(const PrefillArgs& a, int s, int tok) {
  PfSequence q{0, 0, 0, 0, 0, 0, 0};
  if (s < a.n_seqs) {
    q.q_begin = a.cu_q[s];
    q.q_len = a.cu_q[s + 1] - q.q_begin;
    q.start = a.seq_start[s];
    q.slot = a.seq_slot[s];
    q.tiles = (q.q_len + tok - 1) / tok;
    if (q.tiles > 0) {
      int lo;
      pf_tiles(a, q.start, 0, min(tok, q.q_len), lo, q.first);
      pf_tiles(a, q.start, (q.tiles - 1) * tok, q.q_len - (q.tiles - 1) * tok, lo, q.last);
    }
  }
  return q;
}
// Runs that each of a sequence's tiles of tokens is cut into: last / run, to the nearest.
__device__ __forceinline__ int pf_runs(int last, int run) { return max(1, (last + run / 2) / run); }
// Key tiles that a run has on average. With T the sum of (first + last) / 2 over all tiles of tokens and heads:
// Where those are no more than the SMs: the least, from T / 148 on, with which every run finds an SM at once, since one that does
// not costs a whole round (24 sequences of 2 to 8 tokens behind 300 to 6,000, 96 tiles: 67 us in 170 runs, 58 in 148). Where they
// are more, or no such length is found: 2 T / 148, so that a sequence is cut only if one of its tiles alone would hold up the step.
// How many runs come of it: a sequence that is cut has last >= 1.5 run, so at most 4/3 last / run runs, and at most last / run of
// them more than tiles; and last <= first + last, whose sum is 2 T. With run >= 2 T / 148 all cut sequences have 4/3 148 < kPfSlots
// runs, and 148 more than tiles. The search goes on to 16 T / 148, where there are 18 more than tiles: up to kPfFew it finds one.
// `mine`: the lane's first sequence. All lanes of a warp call it, and every block gets the same answer.
__device__ __forceinline__ int pf_run(const PrefillArgs& a, int tok, const PfSequence& mine) {
  const int lane = threadIdx.x & 31;
  float twice = (float)mine.tiles * (float)(mine.first + mine.last);
  int tiles = mine.tiles;
  for (int s = lane + 32; s < a.n_seqs; s += 32) {
    const PfSequence q = pf_sequence(a, s, tok);
    twice += (float)q.tiles * (float)(q.first + q.last);
    tiles += q.tiles;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) twice += __shfl_xor_sync(0xffffffffu, twice, o);
  const float share = twice * (float)a.n_kv / kPfSms;                        // 2 T / 148
  const int most = max(a.run, max(kPfLeast, (int)fminf(ceilf(share), 1e9f)));
  if ((int)__reduce_add_sync(0xffffffffu, (unsigned)tiles) * a.n_kv > kPfSms) return most;
  int run = max(a.run, max(kPfLeast, (int)fminf(ceilf(share * 0.5f), 1e9f)));
  for (int i = 0; i < 24; ++i, run += (run + 7) / 8) {                       // (9/8)^24 > 16
    unsigned runs = mine.tiles * pf_runs(mine.last, run);
    for (int s = lane + 32; s < a.n_seqs; s += 32) {
      const PfSequence q = pf_sequence(a, s, tok);
      runs += q.tiles * pf_runs(q.last, run);
    }
    if ((int)__reduce_add_sync(0xffffffffu, runs) * a.n_kv <= kPfSms) return run;
  }
  return most;
}

struct PfWork {
  int q_begin, q_len, start, page_row;           // the sequence's rows in the step, what it held, its slot
  int tile, hk, part, parts, slot;               // slot: of the partial result; parts: 0 where there is no such piece
};
// Piece `index` of the step's work, or (WHOLE) tile `index` with all its runs. All lanes of a warp call it. Late tiles of a
// sequence, which see the most keys, come first, all heads of one after another.
template <bool WHOLE>
__device__ __forceinline__ PfWork pf_find(const PrefillArgs& a, int tok, int index) {
  const int lane = threadIdx.x & 31;
  const PfSequence mine = pf_sequence(a, lane, tok);
  const int run = pf_run(a, tok, mine);
  PfWork w{0, 0, 0, 0, 0, 0, 0, 0, 0};
  int before = 0, slots = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    const PfSequence q = s0 == 0 ? mine : pf_sequence(a, s0 + lane, tok);
    const int parts = pf_runs(q.last, run);
    const int all = q.tiles * parts * a.n_kv, own = WHOLE ? q.tiles * a.n_kv : all, cut = parts > 1 ? all : 0;
    int incl = own, cuts = cut;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o), y = __shfl_up_sync(0xffffffffu, cuts, o);
      if (lane >= o) {
        incl += x;
        cuts += y;
      }
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + incl > index);
    if (here) {
      const int src = __ffs(here) - 1;
      const int local = index - before - __shfl_sync(0xffffffffu, incl - own, src);
      w.q_begin = __shfl_sync(0xffffffffu, q.q_begin, src);
      w.q_len = __shfl_sync(0xffffffffu, q.q_len, src);
      w.start = __shfl_sync(0xffffffffu, q.start, src);
      w.page_row = __shfl_sync(0xffffffffu, q.slot, src);
      w.parts = __shfl_sync(0xffffffffu, parts, src);
      const int item = WHOLE ? local : local / w.parts;
      w.part = WHOLE ? 0 : local - item * w.parts;
      const int t = item / a.n_kv;
      w.hk = item - t * a.n_kv;
      w.tile = __shfl_sync(0xffffffffu, q.tiles, src) - 1 - t;
      w.slot = slots + __shfl_sync(0xffffffffu, cuts - cut, src) + item * w.parts + w.part;
      return w;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
    slots += __shfl_sync(0xffffffffu, cuts, 31);
  }
  return w;
}

struct PfShared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], x_full[kPfRing];
  uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], last[2];
  uint32_t tmem_base;
  int abort;
  // Of the key tiles in flight, by step % 8: factors of scores, addends, factors of the denominator's terms, and the step (+ 1)
  // that last had NaN among its values. x_full: all of them are there. (A step's place is written again eight steps on, when the
  // scores of the step six on are done; and those were let begin behind the softmax's last look at this step.)
  float k_scale[kPfRing][8], v_add[kPfRing][8], v_back[kPfRing][8];
  int v_nan[kPfRing];
  float handed[2][kPfRows];          // where B has A's rows: its bounds and denominators
  PfWork work;
};

// ------------------------------------------------------------------------------------------ the kernel
// TURNS: every tile's tokens fit into one operand tile; B then has the same rows as A, and the two take the key tiles in turn: two
// steps are under way at a time, and the results meet at the end.
template <int HD, bool TURNS>
__global__ void __launch_bounds__(kPfThreads, 1) prefill_fp8_kernel(const PrefillArgs a) {
  using Cfg = PfCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PfShared sh;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_smem = base;
  uint8_t* k_smem = q_smem + 2 * Cfg::kQBytes;
  uint8_t* v_smem = k_smem + Cfg::kStages * Cfg::kKvBytes;
  const int warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();

  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = TURNS ? tok_x : 2 * tok_x;      // tokens of a tile, of a block
  // one warp looks for the block's piece of work while others set it up
  if (warp == 0) {
    const PfWork found = pf_find<false>(a, tok, blockIdx.x);
    if (threadIdx.x == 0) sh.work = found;
  } else if (threadIdx.x == 32) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh.k_full[s], 128);
      mbar_init(&sh.k_empty[s], 2);
      mbar_init(&sh.v_full[s], 128);
      mbar_init(&sh.v_empty[s], 2);
      mbar_init(&sh.s_full[s], 1);
      mbar_init(&sh.s_free[s], 128);
      mbar_init(&sh.p_ready[s], 128);
      mbar_init(&sh.pv_done[s], 1);
      mbar_init(&sh.last[s], 1);
    }
    for (int i = 0; i < kPfRing; ++i) {
      mbar_init(&sh.x_full[i], 128);
      sh.v_nan[i] = 0;
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  const PfWork w = sh.work;
  if (w.parts == 0) return;          // the whole block alike
  if (warp == 12) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  const int q_begin = w.q_begin, q_len = w.q_len, start = w.start;
  const int t0 = w.tile * tok, n_tok = min(tok, q_len - t0);
  int lo_tile, tiles;
  pf_tiles(a, start, t0, n_tok, lo_tile, tiles);
  // this run's key tiles: [c0, c1) of the tiles of the block's tokens
  const int c0 = lo_tile + tiles * w.part / w.parts, c1 = lo_tile + tiles * (w.part + 1) / w.parts;
  const int last_key = min(start + t0 + n_tok, a.max_pages * kFp8Page) - 1;
  // Steps of the two tiles: A's tokens come first and may not see the last key tiles.
  const int n_tok_a = min(n_tok, tok_x);
  const int n_tok_b = TURNS ? n_tok_a : n_tok - n_tok_a;
  const int n_steps = c1 - c0;
  const int n_a = TURNS ? (n_steps + 1) / 2 : max(0, min(c1, (start + t0 + n_tok_a - 1) / kPfKeys + 1) - c0), n_b = TURNS ? n_steps / 2 : n_tok_b > 0 ? n_steps : 0;

  // What needs no barrier begins before the block meets: the rows' queries go to shared memory, the first codes are asked for.
  const bool softmax = warp < 8;
  const int x = warp >> 2 & 1, r = threadIdx.x & 127;        // tile and row of a softmax thread
  const int first_tok = t0 + (TURNS ? 0 : x * tok_x), n_tok_x = x ? n_tok_b : n_tok_a;
  const int rt = r / G, rh = r - rt * G;                     // token of the tile, query head of the group
  const bool there = softmax && rt < n_tok_x;
  const size_t row_off = ((size_t)(q_begin + first_tok + rt) * a.n_q + w.hk * G + rh) * HD;
  float f = 0.f;                                             // of the row's scores: scale log2(e) and the row's power of two
  constexpr int kPer = HD / 16;                              // pieces of 16 codes a row, and pieces that a converting thread has
  constexpr int kStep = 128 / kPer;                          // its rows: row0, row0 + kStep, ...
  const int ct = threadIdx.x & 127, piece = ct % kPer, row0 = ct / kPer;
  const int* pages = a.block_table + (size_t)w.page_row * a.max_pages;
  uint4 kr[kPer], vr[kPer];
  // Everything is asked for well before it is looked at: a tile's pages a step before its codes, its codes and exponents a step
  // before they are written out. (Where an exponent was clamped, or a page's address made, as soon as it was asked for, the
  // conversion waited for memory twice a tile, and the whole kernel for the conversion: 3,500 clocks a step.)
  int pg0 = 0, pg1 = 0;                                      // pages of the tile to be asked for next
  signed char ke = 0, ve = 0;                                // a thread's two exponents
  auto page_at = [&](int lp) { return lp * kFp8Page <= last_key ? pages[lp] : 0; };
  auto load = [&](uint4 (&reg)[kPer], const unsigned char* cache, int tile) {
    const unsigned char* at0 = cache + (((size_t)pg0 * a.n_kv + w.hk) * kFp8Page + row0) * HD + piece * 16;
    const unsigned char* at1 = cache + (((size_t)pg1 * a.n_kv + w.hk) * kFp8Page + row0) * HD + piece * 16;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      reg[i] = make_uint4(0u, 0u, 0u, 0u);                   // rows behind the block's last key: nothing that may be NaN
      if (tile * kPfKeys + row0 + i * kStep <= last_key)
        reg[i] = *reinterpret_cast<const uint4*>((i < kPer / 2 ? at0 + i * kStep * HD : at1 + (i - kPer / 2) * kStep * HD));
    }
  };
  // Exponents of the tile's eight blocks, a thread a block (one behind the last key: anything, nobody sees its scores).
  auto load_exps = [&]() {
    if (ct < 8) {
      const size_t at = ((size_t)(ct < 4 ? pg0 : pg1) * a.n_kv + w.hk) * kPageExps + (ct & 3);
      ke = a.k_exp[at];
      ve = a.v_exp[at];
    }
  };
  if (softmax) {
    uint4 raw[HD / 8];
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      raw[i] = there ? *reinterpret_cast<const uint4*>(a.q + row_off + i * 8) : make_uint4(0u, 0u, 0u, 0u);
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw[i]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = __bfloat1622float2(h[e]);
        big = fmaxf(big, fmaxf(fabsf(y.x), fabsf(y.y)));
      }
    }
    const int eb = (int)(__float_as_uint(big) >> 23);
    const int shift = eb == 255 ? 0 : min(max(141 - eb, -100), 100);         // the largest number into [2^14, 2^15)
    const float up = pow2_of(shift);
    f = a.scale2 * pow2_of(-shift);
    uint8_t* dst = q_smem + x * Cfg::kQBytes;
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) {
      const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw[i]);
      uint32_t o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 y = __bfloat1622float2(h[e]);
        o[e] = pf_half2(y.x * up, y.y * up);
      }
      *reinterpret_cast<uint4*>(dst + (i >> 3) * kPfSub + swizzle128_offset(r, i & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    fence_proxy_async_smem();
  } else if (warp < 12 && n_steps > 0) {
    pg0 = page_at(c0 * 2);
    pg1 = page_at(c0 * 2 + 1);
    const int next0 = page_at(c0 * 2 + 2), next1 = page_at(c0 * 2 + 3);
    load(kr, a.k, c0);
    load(vr, a.v, c0);
    load_exps();
    pg0 = next0;
    pg1 = next1;
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
#define LLMIE_FAIL(code) do { if (!*abort) { *abort = 1; atomicExch(a.status, (code)); } } while (0)

  if (softmax) {
    // ------------------------------------------------------------------ softmax: a thread a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PfRegs<HD, TURNS>::kSoftmax));
    const int n_x = x ? n_b : n_a;
    const int qpos = start + first_tok + min(rt, max(n_tok_x - 1, 0));
    const int lo = first_visible_key(qpos, a.window);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + Cfg::kSCol + x * 128, o_addr = tmem + lanes + Cfg::kOCol + x * (HD == 64 ? 64 : 128);
    const uint32_t p_addr = Cfg::kOwnP ? tmem + lanes + Cfg::kPCol + x * 64 : s_addr;
    // a score's factor is never 0: times -inf, which stands where the row does not look, that would be NaN
    auto factor = [&](float k_scale) { return fminf(fmaxf(f * k_scale, 1.2e-38f), 3.4e38f); };
    float R = -INFINITY, l = 0.f;
    uint32_t nan_cols[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) nan_cols[i] = 0u;
    bool ok = true;
    // the first and last keys that every row of the tile sees
    const int all_to = start + first_tok, all_from = first_visible_key(start + first_tok + max(n_tok_x - 1, 0), a.window);
    for (int j = 0; j < n_x; ++j) {            // this tile's j-th step is the block's `step`
      const int step = TURNS ? 2 * j + x : j;
      // every decision to give up is taken by the whole warp: reads of tensor memory are warp-wide instructions
      if (!__all_sync(0xffffffffu, mbar_wait(&sh.x_full[step % kPfRing], (step / kPfRing) & 1, abort) && mbar_wait(&sh.s_full[x], j & 1, abort))) {
        LLMIE_FAIL(kStatusTimeoutMma);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const int kbase = (c0 + step) * kPfKeys, ring = step % kPfRing;
      const bool edge = kbase + kPfKeys - 1 > all_to || kbase < all_from;
      const int nan_step = sh.v_nan[ring];
      // the row's scores; those that it does not see are -inf
      uint32_t v[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_addr + c * 32, v[c]);
      float fk[8];
#pragma unroll
      for (int b = 0; b < 8; ++b) fk[b] = factor(sh.k_scale[ring][b]);
      tmem_ld_wait();
      if (Cfg::kOwnP) {
        // they are in registers: the next scores may be written
        tc_fence_before_sync();
        mbar_arrive(&sh.s_free[x]);
      }
      if (edge) {
        const int from = lo - kbase;
        const unsigned span = (unsigned)(qpos - lo);
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if ((unsigned)(i - from) > span) v[i >> 5][i & 31] = 0xff800000u;
      }
      float mx = -INFINITY;          // the largest s + ev
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        const uint32_t* y = v[b >> 1] + (b & 1) * 16;
        float m0 = __uint_as_float(y[0]), m1 = __uint_as_float(y[1]);
#pragma unroll
        for (int i = 2; i < 14; i += 4) {
          m0 = pf_max3(m0, __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
          m1 = pf_max3(m1, __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
        }
        m0 = pf_max3(m0, __uint_as_float(y[14]), __uint_as_float(y[15]));
        mx = fmaxf(mx, fmaf(fmaxf(m0, m1), fk[b], sh.v_add[ring][b]));
      }
      const bool grow = mx > R + kPfSlack || R == -INFINITY;
      if (__any_sync(0xffffffffu, grow && j > 0)) {
        // the sums so far are brought to the new bound (rows that keep theirs: times 1)
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.pv_done[x], (j - 1) & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const float alpha = !grow ? 1.f : R == -INFINITY ? 0.f : pf_exp2(R - mx);
        l *= alpha;
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t y[16];
          tmem_ld_32x16(o_addr + c * 16, y);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
          pf_tmem_st16(o_addr + c * 16, y);
        }
        tmem_st_wait();
      }
      if (grow) R = mx;
      const float shift = (R == -INFINITY ? 0.f : R) - kPfTop;
      if (Cfg::kOwnP && j > 0) {
        // the weights of the tile before have to be through the product before they are written over
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.pv_done[x], (j - 1) & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
      }
      // the weights, over the scores they come from or in columns of their own
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t o[16];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float add = sh.v_add[ring][c * 2 + b] - shift;
          const uint32_t* y = v[c] + b * 16;
          float sum[4];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x0 = pf_exp2(fmaf(__uint_as_float(y[i]), fk[c * 2 + b], add)), x1 = pf_exp2(fmaf(__uint_as_float(y[i + 1]), fk[c * 2 + b], add));
            sum[i & 2] = i < 4 ? x0 : sum[i & 2] + x0;
            sum[(i & 2) + 1] = i < 4 ? x1 : sum[(i & 2) + 1] + x1;
            o[b * 8 + i / 2] = pf_half2(x0, x1);
          }
          l = fmaf((sum[0] + sum[1]) + (sum[2] + sum[3]), sh.v_back[ring][c * 2 + b], l);
        }
        pf_tmem_st16(p_addr + c * 16, o);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&sh.p_ready[x]);
      if (nan_step == step + 1) {
        // rare: which columns of the values that this row sees are NaN
        for (int p = max(lo, kbase); p <= min(min(qpos, last_key), kbase + kPfKeys - 1); ++p) {
          const unsigned* row = reinterpret_cast<const unsigned*>(a.v + (((size_t)pages[p / kFp8Page] * a.n_kv + w.hk) * kFp8Page + p % kFp8Page) * HD);
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            uint32_t bits = 0u;
#pragma unroll 1
            for (int e = 0; e < 32; ++e) bits |= ((row[i * 8 + e / 4] >> (e % 4 * 8) & 0x7fu) == 0x7fu ? 1u : 0u) << e;
            nan_cols[i] |= bits;
          }
        }
      }
    }
    if (ok && n_x > 0) {
      if (!__all_sync(0xffffffffu, mbar_wait(&sh.pv_done[x], (n_x - 1) & 1, abort))) {
        LLMIE_FAIL(kStatusTimeoutMma);
        ok = false;
      }
      tc_fence_after_sync();
    }
    if (TURNS) {
      // B hands its results to A through the place of the keys, which nobody reads any more once both tiles' products are done
      float* handed = reinterpret_cast<float*>(k_smem) + r * HD;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (x == 1) {
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t y[32];
          if (ok && n_x > 0) {
            tmem_ld_32x32(o_addr + c * 32, y);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = 0u;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {          // places of a row shifted by the row: other banks for other rows
            float4 z;
            z.x = (nan_cols[c] >> i & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(y[i]);
            z.y = (nan_cols[c] >> (i + 1) & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(y[i + 1]);
            z.z = (nan_cols[c] >> (i + 2) & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(y[i + 2]);
            z.w = (nan_cols[c] >> (i + 3) & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(y[i + 3]);
            *reinterpret_cast<float4*>(handed + (c * 32 + i + r * 4) % HD) = z;
          }
        }
        sh.handed[0][r] = R;
        sh.handed[1][r] = l;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    // ---- the row's result: the output, or a partial one. Where a wait gave up: NaN.
    if (!TURNS || x == 0) {
      float mine_f = 1.f, b_f = 0.f;
      if (TURNS) {
        const float Rb = sh.handed[0][r], M = fmaxf(R, Rb), Mu = M == -INFINITY ? 0.f : M;
        mine_f = R == -INFINITY ? 0.f : pf_exp2(R - Mu);
        b_f = Rb == -INFINITY ? 0.f : pf_exp2(Rb - Mu);
        l = fmaf(l, mine_f, sh.handed[1][r] * b_f);
        R = M;
      }
      const float* handed = reinterpret_cast<const float*>(k_smem) + r * HD;
      float* rec = a.part + (size_t)w.slot * Cfg::kRecord;
      const int pr = x * kPfRows + r;
      if (w.parts > 1 && there) {
        rec[2 * kPfRows * HD + pr] = R;
        rec[2 * kPfRows * (HD + 1) + pr] = ok ? l : __int_as_float(0x7fffffff);
      }
      const float inv = 1.f / l;
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t y[32];
        if (ok && n_x > 0) {
          tmem_ld_32x32(o_addr + c * 32, y);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0u;
        }
        if (there) {                   // (reads of tensor memory are warp-wide: only what follows them goes by the row)
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float v8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              v8[e] = (nan_cols[c] >> (i + e) & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(y[i + e]);
            if (TURNS) {
#pragma unroll
              for (int e = 0; e < 8; e += 4) {
                const float4 z = *reinterpret_cast<const float4*>(handed + (c * 32 + i + e + r * 4) % HD);
                v8[e] = fmaf(v8[e], mine_f, z.x * b_f);
                v8[e + 1] = fmaf(v8[e + 1], mine_f, z.y * b_f);
                v8[e + 2] = fmaf(v8[e + 2], mine_f, z.z * b_f);
                v8[e + 3] = fmaf(v8[e + 3], mine_f, z.w * b_f);
              }
            }
            if (w.parts > 1) {
              store8(rec + (size_t)pr * HD + c * 32 + i, v8);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) v8[e] *= inv;
              store8(a.out + row_off + c * 32 + i, v8);
            }
          }
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ conversion: 128 threads, 16 codes at a time
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PfRegs<HD, TURNS>::kConvert));
    auto put = [&](uint8_t* dst, const uint4 (&reg)[kPer]) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int row = row0 + i * kStep;
        const unsigned c[4] = {reg[i].x, reg[i].y, reg[i].z, reg[i].w};
        uint32_t h[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[2 * e] = e4m3x2_to_half2((unsigned short)(c[e] & 0xffffu));
          h[2 * e + 1] = e4m3x2_to_half2((unsigned short)(c[e] >> 16));
        }
        uint8_t* at = dst + (piece >> 2) * kPfSub;
        const int ch = (piece & 3) * 2, odd = piece >> 2 & 1;          // the two 64-column halves of a row in turn: other banks
        const uint4 lo4 = make_uint4(h[0], h[1], h[2], h[3]), hi4 = make_uint4(h[4], h[5], h[6], h[7]);
        *reinterpret_cast<uint4*>(at + swizzle128_offset(row, ch + odd)) = odd ? hi4 : lo4;
        *reinterpret_cast<uint4*>(at + swizzle128_offset(row, ch + 1 - odd)) = odd ? lo4 : hi4;
      }
    };
    for (int j = 0; j < n_steps; ++j) {
      const int st = j & 1, ring = j % kPfRing;
      const int next0 = page_at((c0 + j + 2) * 2), next1 = page_at((c0 + j + 2) * 2 + 1);
      if (j >= 2 && !mbar_wait(&sh.k_empty[st], ((j >> 1) - 1) & 1, abort)) {
        LLMIE_FAIL(kStatusTimeoutEmpty);
        break;
      }
      if (ct < 8) {
        const int k = clamp_exponent(ke), v = clamp_exponent(ve);
        sh.k_scale[ring][ct] = pow2_of(k);
        sh.v_add[ring][ct] = (float)v;
        sh.v_back[ring][ct] = pow2_of(-v);
      }
      // NaN among the values: such codes become zeros here
      unsigned any = 0u;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        any |= ((vr[i].x & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].y & 0x7f7f7f7fu) + 0x01010101u) |
               ((vr[i].z & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].w & 0x7f7f7f7fu) + 0x01010101u);
      put(k_smem + st * Cfg::kKvBytes, kr);
      if (j + 1 < n_steps) {
        load(kr, a.k, c0 + j + 1);
        load_exps();
      }
      fence_proxy_async_smem();
      if (any & 0x80808080u) {
        sh.v_nan[ring] = j + 1;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          unsigned* c = reinterpret_cast<unsigned*>(&vr[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned bad = ((c[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            c[e] &= ~(bad | (bad - (bad >> 7)));             // the whole byte
          }
        }
      }
      mbar_arrive(&sh.x_full[ring]);
      mbar_arrive(&sh.k_full[st]);
      if (j >= 2 && !mbar_wait(&sh.v_empty[st], ((j >> 1) - 1) & 1, abort)) {
        LLMIE_FAIL(kStatusTimeoutEmpty);
        break;
      }
      put(v_smem + st * Cfg::kKvBytes, vr);
      if (j + 1 < n_steps) load(vr, a.v, c0 + j + 1);
      pg0 = next0;
      pg1 = next1;
      fence_proxy_async_smem();
      mbar_arrive(&sh.v_full[st]);
    }
  } else {
    // ------------------------------------------------------------------ the tensor core: a thread a tile, so that neither waits for the other's
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PfRegs<HD, TURNS>::kIssue));
    if (warp < 14 && elect_one()) {
      constexpr uint32_t idesc_s = pf_instr_desc(kPfRows, kPfKeys, 0), idesc_o = pf_instr_desc(kPfRows, HD, 1);
      const int tx = warp - 12, n_x = tx ? n_b : n_a;
      const uint32_t s_col = tmem + Cfg::kSCol + tx * 128, o_col = tmem + Cfg::kOCol + tx * (HD == 64 ? 64 : 128);
      const uint32_t p_col = Cfg::kOwnP ? tmem + Cfg::kPCol + tx * 64 : s_col;
      // descriptors of the operands' first 16 columns; the rest lie a fixed number of 16-byte units on
      const uint64_t q_desc = make_smem_desc(smem_u32(q_smem + tx * Cfg::kQBytes), 16, 1024);
      const uint64_t k_desc = make_smem_desc(smem_u32(k_smem), 16, 1024), v_desc = make_smem_desc(smem_u32(v_smem), kPfSub, 1024);
      auto wait_for = [&](uint64_t* bar, uint32_t parity, int code) {
        if (mbar_wait(bar, parity, abort)) return true;
        LLMIE_FAIL(code);
        return false;
      };
      // a stage is free when both tiles have let go of it; where they take steps in turn, the one that has it lets go twice
      auto let_go = [&](uint64_t* bar) {
        mma_commit(bar);
        if (TURNS) mma_commit(bar);
      };
      auto scores = [&](int j) -> bool {                     // S = Q K^T of this tile's j-th step
        const int step = TURNS ? 2 * j + tx : j;
        if (!wait_for(&sh.k_full[step & 1], (step >> 1) & 1, kStatusTimeoutFull)) return false;
        tc_fence_after_sync();
        const uint64_t kd = k_desc + (uint64_t)((step & 1) * (Cfg::kKvBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const int off = ((kk >> 2) * kPfSub + (kk & 3) * 32) >> 4;
          mma_bf16_ss(s_col, q_desc + off, kd + off, idesc_s, kk > 0 ? 1u : 0u);
        }
        mma_commit(&sh.s_full[tx]);
        let_go(&sh.k_empty[step & 1]);
        return true;
      };
      auto sums = [&](int j) -> bool {                       // O (+)= W V of it
        const int step = TURNS ? 2 * j + tx : j;
        if (!wait_for(&sh.v_full[step & 1], (step >> 1) & 1, kStatusTimeoutFull)) return false;
        if (!wait_for(&sh.p_ready[tx], j & 1, kStatusTimeoutMma)) return false;
        tc_fence_after_sync();
        const uint64_t vd = v_desc + (uint64_t)((step & 1) * (Cfg::kKvBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < kPfKeys / 16; ++kk)            // 16 weights are 8 columns; 16 keys are 16 rows of the values
          pf_mma_ts(o_col, p_col + kk * 8, vd + kk * (2048 >> 4), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&sh.pv_done[tx]);
        let_go(&sh.v_empty[step & 1]);
        return true;
      };
      bool ok = n_x == 0 || scores(0);
      for (int j = 0; ok && j < n_x; ++j) {
        // where the weights have columns of their own, the next scores as soon as these are in registers; else they are written
        // where these weights are read from
        if (Cfg::kOwnP && j + 1 < n_x) ok = wait_for(&sh.s_free[tx], j & 1, kStatusTimeoutMma) && scores(j + 1);
        ok = ok && sums(j);
        if (!Cfg::kOwnP && ok && j + 1 < n_x) ok = wait_for(&sh.pv_done[tx], j & 1, kStatusTimeoutMma) && scores(j + 1);
      }
      // steps that are the other tile's alone
      for (int j = n_x; ok && !TURNS && j < n_steps; ++j) {
        ok = wait_for(&sh.k_full[j & 1], (j >> 1) & 1, kStatusTimeoutFull);
        if (ok) mbar_arrive(&sh.k_empty[j & 1]);
        ok = ok && wait_for(&sh.v_full[j & 1], (j >> 1) & 1, kStatusTimeoutFull);
        if (ok) mbar_arrive(&sh.v_empty[j & 1]);
      }
      // nothing may be in flight when the tensor memory is given back
      mma_commit(&sh.last[tx]);
      for (unsigned spin = 0; spin < (1u << 20) && !mbar_test(&sh.last[tx], 0); ++spin) __nanosleep(32);
    }
  }
#undef LLMIE_FAIL
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the runs of the tiles that were cut. grid (tiles of tokens x key/value heads, 8): an eighth of a tile's rows a block, a warp a row.
constexpr int kPfJoinWarps = 8, kPfJoinSide = 8;
template <int HD, bool TURNS> __global__ void __launch_bounds__(kPfJoinWarps * 32) prefill_fp8_join_kernel(const PrefillArgs a) {
  pdl_launch_dependents();
  using Cfg = PfCfg<HD>;
  const int lane = threadIdx.x & 31;
  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = TURNS ? tok_x : 2 * tok_x;
  const PfWork w = pf_find<true>(a, tok, blockIdx.x);
  // The lengths are older than the kernel that leaves the partial results (it lets this one begin behind its own wait). Blocks with
  // nothing to join wait too: the kernel behind this one waits for this one alone, and reads what the one in front wrote.
  pdl_wait();
  if (w.parts <= 1) return;
  const float* base = a.part + (size_t)w.slot * Cfg::kRecord;
  for (int row = blockIdx.y * kPfJoinWarps + (threadIdx.x >> 5); row < 2 * kPfRows; row += kPfJoinSide * kPfJoinWarps) {
    const int x = row / kPfRows, rt = row % kPfRows / G, rh = row % kPfRows - rt * G, t = w.tile * tok + x * tok_x + rt;
    if (rt >= tok_x || t >= w.q_len) continue;
    const float* rec = base + (size_t)row * HD + lane * (HD / 32);
    float M = -INFINITY, den = 0.f, num[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) num[i] = 0.f;
    // eight runs at a time, all asked for at once
    for (int p0 = 0; p0 < w.parts; p0 += 8) {
      float m[8], l[8], v[8][HD / 32];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const bool there = p0 + p < w.parts;
        const float* r = base + (size_t)(p0 + p) * Cfg::kRecord;
        m[p] = there ? __ldcg(r + 2 * kPfRows * HD + row) : -INFINITY;
        l[p] = there ? __ldcg(r + 2 * kPfRows * (HD + 1) + row) : 0.f;
        const float* c = rec + (size_t)(there ? p0 + p : 0) * Cfg::kRecord;
        if (HD == 64) {
          const float2 y = __ldcg(reinterpret_cast<const float2*>(c));
          v[p][0] = y.x;
          v[p][1] = y.y;
        } else {
          const float4 y = __ldcg(reinterpret_cast<const float4*>(c));
          v[p][0] = y.x;
          v[p][1] = y.y;
          v[p][HD / 32 - 2] = y.z;
          v[p][HD / 32 - 1] = y.w;
        }
      }
      float M8 = M;
#pragma unroll
      for (int p = 0; p < 8; ++p) M8 = fmaxf(M8, m[p]);
      const float Mu = M8 == -INFINITY ? 0.f : M8, back = M == -INFINITY ? 0.f : pf_exp2(M - Mu);
      den *= back;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) num[i] *= back;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float f = pf_exp2(m[p] - Mu);
        den = fmaf(f, l[p], den);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) num[i] = p0 + p < w.parts ? fmaf(f, v[p][i], num[i]) : num[i];
      }
      M = M8;
    }
    __nv_bfloat16* o = a.out + ((size_t)(w.q_begin + t) * a.n_q + w.hk * G + rh) * HD + lane * (HD / 32);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[i] = __float2bfloat16_rn(num[i] / den);
  }
}

template <int HD, bool TURNS>
static int launch_prefill_fp8(PrefillArgs a, int n_tokens, int max_q_len, cudaStream_t stream) {
  using Cfg = PfCfg<HD>;
  cudaError_t e = cudaFuncSetAttribute(prefill_fp8_kernel<HD, TURNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return (int)e;
  const int tok = (TURNS ? 1 : 2) * (kPfRows / (a.n_q / a.n_kv));
  // Pieces of work: the tiles of tokens, and the runs that they may be cut into (see pf_run). The most runs that a tile can have
  // follow from the most keys that the table has room for and the least work that so many tokens are.
  const long long items = max_q_len <= tok ? (long long)a.n_seqs * a.n_kv : ((long long)n_tokens / tok + a.n_seqs) * a.n_kv;
  double least = (double)n_tokens / tok * a.n_kv;
  long long most_tiles = ((long long)a.max_pages * kFp8Page + kPfKeys - 1) / kPfKeys;
  if (a.window == 0) {
    least *= (1.0 + (double)n_tokens / ((double)kPfKeys * a.n_seqs)) / 2;
  } else {
    const long long w = a.window < 0 ? -(long long)a.window : a.window;
    most_tiles = min(most_tiles, (w + tok) / kPfKeys + 2);
  }
  // (tokens that do not fill their tiles may leave fewer tiles than SMs after all, where runs may be half as long)
  long long run = (long long)(least * ((double)n_tokens / tok * a.n_kv > kPfSms ? 2 : 1) / kPfSms);
  run = min(max(run, (long long)kPfLeast), 1LL << 30);
  const bool cut = (most_tiles + run / 2) / run > 1;
  if (cut && !a.part) return kPfNeedsScratch;
  a.run = (int)run;
  const long long blocks = !cut ? items : items <= kPfFew ? kPfSms : items + kPfSms;
  if (blocks * most_tiles > 0x3fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  launch_k(prefill_fp8_kernel<HD, TURNS>, dim3((unsigned)blocks), dim3(kPfThreads), Cfg::kSmem, stream, a);
  LLMIE_LAUNCH_CHECK();
  if (cut) {
    launch_k(prefill_fp8_join_kernel<HD, TURNS>, dim3((unsigned)items, kPfJoinSide), dim3(kPfJoinWarps * 32), 0, stream, a);
    LLMIE_LAUNCH_CHECK();
  }
  return LLMIE_OK;
}

}  // namespace llmie

using namespace llmie;

// float32 numbers of scratch that a call may need
extern "C" int llmie_attention_prefill_fp8_scratch(int hd) {
  return kPfSlots * (hd == 64 ? PfCfg<64>::kRecord : PfCfg<128>::kRecord);
}

// q, out bfloat16 [n_tokens, n_q hd], hd 64 or 128, at most 128 query heads a key/value head; sequences packed one after another
// (cu_q [n_seqs + 1]); caches e4m3 [pages, n_kv, 64, hd] with exponents int8 [pages, n_kv, 4]; seq_start[i]: tokens that sequence i
// held before this step, whose keys are in the cache already; max_q_len: the most tokens that one brings. scale > 0. window: as in the other attention kernels.
// scratch: llmie_attention_prefill_fp8_scratch floats, 16-byte aligned; null: a call that needs it launches nothing and returns -5.
extern "C" int llmie_attention_prefill_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_exp,
                                           const void* v_exp, void* out, float* scratch, int* status, const int* cu_q,
                                           const int* seq_slot, const int* seq_start, const int* block_table, int max_pages,
                                           int n_tokens, int n_seqs, int max_q_len, int n_q, int n_kv, int hd, float scale,
                                           int window, cudaStream_t stream) {
  if (n_tokens < 0 || n_seqs < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0 || !status) return LLMIE_ERR_BAD_ARG;
  if (!(scale > 0.f)) return LLMIE_ERR_BAD_ARG;              // a row's bound is taken before scores are scaled
  if ((hd != 64 && hd != 128) || n_q / n_kv > kPfRows) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(scratch)) return LLMIE_ERR_ALIGNMENT;
  if (n_tokens == 0 || n_seqs == 0 || max_q_len <= 0) return LLMIE_OK;
  const PrefillArgs a{(const __nv_bfloat16*)q, (const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp,
                      (const signed char*)v_exp, (__nv_bfloat16*)out, scratch, status, cu_q, seq_slot, seq_start, block_table,
                      max_pages, n_seqs, n_q, n_kv, scale * 1.4426950408889634f, window, 0};
  const bool turns = max_q_len <= kPfRows / (n_q / n_kv);
#define LLMIE_PREFILL(HD) return turns ? launch_prefill_fp8<HD, true>(a, n_tokens, max_q_len, stream) : launch_prefill_fp8<HD, false>(a, n_tokens, max_q_len, stream)
  if (hd == 64) LLMIE_PREFILL(64);
  LLMIE_PREFILL(128);
#undef LLMIE_PREFILL
}
