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
// every digit of bfloat16 (of what is above 2^-31 of the row's largest number; the rest is off by 2^-39 of that at most). Weights go back
// to tensor memory as the second product's first operand.
//
// Work. A piece is a (sequence, tile of tokens, key/value head), or one of several equal runs of its key tiles where the step has
// too few of them for the GPU: how many runs a sequence's tiles are cut into is worked out on the device from the lengths that
// are there. Runs leave partial results, which a second kernel joins in order. A block per piece is launched, and a block that is
// about to be done takes over the piece of one that has not begun (cluster launch control): keys of the next piece are converted
// while this one's last scores are worked on, its queries are brought while its last product runs. (6 sequences of 60 to 1,500
// tokens, head size 128, steps of 128 keys: 76.4 us with a block a piece, which spent 26,000 of 42,000 clocks on finding, bringing and
// writing, 68.0 so. With steps of 64 keys 60.0.)
//
// What bounds it. At head size 64 a step of 128 rows twice and 128 keys is 32,768 exponentials, 2,050 clocks, and takes 4,100 (48.2 us
// for a prompt of 2,048 tokens, 32 / 8 heads: 357 TFLOP/s of products); what the other half goes into is not broken down. At 128 a step has 64
// keys, 16,384 exponentials and as many codes to convert, and takes 2,500. Between pieces some 9,000 clocks pass at head size 128 for
// results, queries and the first scores.
//
// Code. What a block does once is written in loops that stay loops, and each search for work is there once: a kernel of 140 to 250 KB
// of instructions, as the compiler lays them out by itself, spends thousands of clocks a piece on fetching them.
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
constexpr int kPfThreads = 512;      // warps 0-3, 4-7: softmax of tiles A and B; 8-11: conversion; 12, 13: the products of A, of B; 14: work; 15: nothing
constexpr int kPfSub = kPfRows * 128;        // bytes of 128 rows of 64 half-precision numbers
constexpr int kPfSms = 148;
constexpr int kPfRing = 16;
constexpr int kPfStages = 4;         // at most
constexpr int kPfAhead = 4;          // places for pieces of work
constexpr int kPfReaders = 14;       // who reads one: eight softmax warps, four converting ones, two issuing threads
constexpr int kPfNeedsScratch = -5;  // the answer to a call without scratch that cannot do without
constexpr int kPfLeast = 256;        // keys that a run has at least, on average
constexpr int kPfWhole = 768;        // a step is not cut where no token sees more keys
constexpr int kPfSlots = 200;        // partial results at once (see pf_run)
constexpr int kPfFew = 128;          // tiles of tokens that can always be cut into runs for which there are SMs (see pf_run)
constexpr float kPfTop = 7.f;        // the bound's own weight is 2^7
constexpr float kPfSlack = 8.f;      // how far scores may outgrow the bound, in units of log2

template <int HD> struct PfCfg {
  static constexpr int kSubs = HD / 64;
  static constexpr int kQBytes = kSubs * kPfSub;             // one tile of queries
  // Keys of a step. Where there is room for it in tensor memory, 128: 64 would be the same work with twice the waits (a prompt of 2,048
  // tokens 53.4 us for 48.8). At head size 128 there is not, and with weights that lay over the scores, the next scores had to
  // wait for this step's second product (pieces of 60 to 1,500 tokens 68.0 us with 128 keys, 60.5 with 64).
  static constexpr int kKeys = HD == 64 ? 128 : 64;
  static constexpr int kKvSub = kKeys * 128;
  static constexpr int kKvBytes = kSubs * kKvSub;            // a step's keys, or values
  static constexpr int kStages = 256 / kKeys;
  static constexpr int kBlocks = kKeys / kExpBlock;          // of the cache, a step
  static constexpr int kOutBytes = 8 * 2048;                 // a warp turns 32 rows of 32 numbers at a time
  static constexpr int kSmem = 2 * kQBytes + 2 * kStages * kKvBytes + kOutBytes + 1024;
  // Columns of tensor memory: sums of A and B, scores of either, weights. There is room for the weights beside the scores, which lets
  // a step's scores be made while the softmax works on the step before.
  static constexpr int kOCol = 0, kSCol = 2 * HD, kPCol = kSCol + 2 * kKeys;
  static_assert(kPCol + kKeys <= 512, "tensor memory has 512 columns");
  static constexpr int kRecord = 2 * kPfRows * (HD + 2);     // floats of a partial result: sums [HD / 4][rows][4], then bounds, then denominators
};

// Registers that a thread of a softmax, the conversion and the last warpgroup keeps of the 128 that it is launched with: a row's scores
// of a step stay in registers.
template <int HD> struct PfRegs {
  static constexpr int kSoftmax = HD == 64 ? 192 : 152, kConvert = HD == 64 ? 72 : 120, kIssue = HD == 64 ? 56 : 88;
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
  int run;                           // no run is shorter: what the host counted blocks and scratch by; 0: it counted on whole tiles
};

__device__ __forceinline__ float pf_exp2(float x) { return exp2_ftz(x); }
__device__ __forceinline__ uint32_t pf_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float pf_max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// mbar_wait in few instructions.
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  unsigned spin = 0;
#pragma unroll 1
  while (!mbar_test(bar, parity)) {
    if (++spin > 64) {
      __nanosleep(spin > 4096 ? 256 : 32);
      if (*abort || spin > kSpinLimit) return false;
    }
  }
  return true;
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
// Key tiles of a sequence's tile of tokens [t0, t0 + n): from `lo` on, `count` of them. None behind the table's last page: tokens at
// positions that the table has no room for (a caller's mistake) see what one at its last position sees.
template <int KEYS> __device__ __forceinline__ void pf_tiles(const PrefillArgs& a, int start, int t0, int n, int& lo, int& count) {
  const int room = a.max_pages * kFp8Page;
  lo = first_visible_key(min(start + t0, room - 1), a.window) / KEYS;
  count = max((min(start + t0 + n, room) - 1) / KEYS - lo + 1, 0);
}
// What a lane knows of its sequence: tiles of tokens, the key tiles of the first and the last of them.
struct PfSequence {
  int q_begin, q_len, start, slot, tiles, first, last;
};
template <int KEYS> __device__ __forceinline__ PfSequence pf_sequence(const PrefillArgs& a, int s, int tok) {
  PfSequence q{0, 0, 0, 0, 0, 0, 0};
  if (s < a.n_seqs) {
    q.q_begin = a.cu_q[s];
    q.q_len = a.cu_q[s + 1] - q.q_begin;
    q.start = a.seq_start[s];
    q.slot = a.seq_slot[s];
    q.tiles = (q.q_len + tok - 1) / tok;
    if (q.tiles > 0) {
      int lo;
      pf_tiles<KEYS>(a, q.start, 0, min(tok, q.q_len), lo, q.first);
      pf_tiles<KEYS>(a, q.start, (q.tiles - 1) * tok, q.q_len - (q.tiles - 1) * tok, lo, q.last);
    }
  }
  return q;
}
// Runs that each of a sequence's tiles of tokens is cut into, by pf_run's answer: none longer than it where all of them find an SM at
// once (answers below 0), else last / run to the nearest.
__device__ __forceinline__ int pf_runs(int last, int run) { return run < 0 ? max(1, (last - run - 1) / -run) : max(1, (last + run / 2) / run); }
// How long runs are, in key tiles. A step whose tokens see at most kPfWhole keys is left whole: the join takes about as long as it would
// save (2 sequences of 600 tokens, 16 heads: 25 us whole, 30.5 in runs of 256 keys; 6 of up to 50 behind up to 800 13.9 and 18.5;
// 4 of up to 156 behind up to 1,592 38.9 and 27.8). With T the sum of (first + last) / 2 over all tiles of tokens and heads:
// Where those are no more than the SMs: the least, from T / 148 on, with which every run finds an SM at once and none is longer
// (answered below 0; 24 sequences of 2 to 8 tokens behind 300 to 6,000, 96 tiles: 52.4 us, and 55.0 where runs are last / run to the
// nearest, half as long again at worst). Where they are more, or no such length is found: 2 T / 148, so that a sequence is cut only
// if one of its tiles alone would hold up the step.
// How many runs come of it: in the first case at most 148. In the second a sequence that is cut has last >= 1.5 run, so at most
// 4/3 last / run runs, and at most last / run of them more than tiles; and last <= first + last, whose sum is 2 T. So all cut
// sequences have 4/3 148 < kPfSlots runs, and 148 more than tiles. The search goes on beyond 15 T / 148, where there are 19 more than
// tiles at most: up to kPfFew it finds one.
// Where the host has counted on whole tiles (a.run 0), they stay whole, whatever the lengths are: there is no scratch then, no join, and a
// block for each tile. It goes by the rows of the step, of which the sequences may have few.
// `mine`: the lane's first sequence. All lanes of a warp call it, and every block gets the same answer.
template <int KEYS> __device__ __forceinline__ int pf_run(const PrefillArgs& a, int tok, const PfSequence& mine) {
  const int lane = threadIdx.x & 31;
  float twice = (float)mine.tiles * (float)(mine.first + mine.last);
  int tiles = mine.tiles, longest = mine.last;
#pragma unroll 1
  for (int s = lane + 32; s < a.n_seqs; s += 32) {
    const PfSequence q = pf_sequence<KEYS>(a, s, tok);
    twice += (float)q.tiles * (float)(q.first + q.last);
    tiles += q.tiles;
    longest = max(longest, q.last);
  }
  if (a.run == 0 || __reduce_max_sync(0xffffffffu, longest) <= kPfWhole / KEYS) return 1 << 30;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) twice += __shfl_xor_sync(0xffffffffu, twice, o);
  const float share = twice * (float)a.n_kv / kPfSms;                        // 2 T / 148
  const int most = max(a.run, max(kPfLeast / KEYS, (int)fminf(ceilf(share), 1e9f)));
  if ((int)__reduce_add_sync(0xffffffffu, (unsigned)tiles) * a.n_kv > kPfSms) return most;
  int run = max(a.run, max(kPfLeast / KEYS, (int)fminf(ceilf(share * 0.5f), 1e9f)));
#pragma unroll 1
  for (int i = 0; i < 24; ++i, run += (run + 7) / 8) {                       // the last is (9/8)^23 > 15 times the first
    unsigned runs = mine.tiles * pf_runs(mine.last, -run);
#pragma unroll 1
    for (int s = lane + 32; s < a.n_seqs; s += 32) {
      const PfSequence q = pf_sequence<KEYS>(a, s, tok);
      runs += q.tiles * pf_runs(q.last, -run);
    }
    if ((int)__reduce_add_sync(0xffffffffu, runs) * a.n_kv <= kPfSms) return -run;
  }
  return most;
}

struct PfWork {
  int q_begin, q_len, start, page_row;           // the sequence's rows in the step, what it held, its slot
  int tile, hk, part, parts, slot;               // slot: of the partial result; parts: 0 where there is no such piece
};
// Piece `index` of the step's work, or (WHOLE) tile `index` with all its runs. All lanes of a warp call it. Late tiles of a
// sequence, which see the most keys, come first, all heads of one after another. `mine`: the lane's first sequence; run: pf_run's.
template <bool WHOLE, int KEYS>
__device__ __forceinline__ PfWork pf_find(const PrefillArgs& a, int tok, int index, const PfSequence& mine, int run) {
  const int lane = threadIdx.x & 31;
  PfWork w{0, 0, 0, 0, 0, 0, 0, 0, 0};
  int before = 0, slots = 0;
#pragma unroll 1
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    const PfSequence q = s0 == 0 ? mine : pf_sequence<KEYS>(a, s0 + lane, tok);
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

// What the block's parts need of a piece, worked out by who found it.
struct PfPiece {
  int parts, slot, hk, page_row;
  int row0, pos0;                    // of its first token: row of the step, position
  int n_tok_a, n_tok_b;              // tokens of the two tiles
  int c0, n_steps, n_a, n_b;         // its first key tile; its steps and those of either tile
  int last_key;
};
template <bool TURNS, int KEYS> __device__ __forceinline__ PfPiece pf_piece(const PrefillArgs& a, const PfWork& w, int tok_x) {
  PfPiece p;
  const int tok = TURNS ? tok_x : 2 * tok_x, t0 = w.tile * tok, n_tok = min(tok, w.q_len - t0), parts = max(w.parts, 1);
  p.parts = w.parts;
  p.slot = w.slot;
  p.hk = w.hk;
  p.page_row = w.page_row;
  p.row0 = w.q_begin + t0;
  p.pos0 = w.start + t0;
  int lo_tile, tiles;
  pf_tiles<KEYS>(a, w.start, t0, n_tok, lo_tile, tiles);
  // this run's key tiles: [c0, c1) of the tiles of the block's tokens
  p.c0 = lo_tile + tiles * w.part / parts;
  const int c1 = lo_tile + tiles * (w.part + 1) / parts;
  p.last_key = min(p.pos0 + n_tok, a.max_pages * kFp8Page) - 1;
  // Steps of the two tiles: A's tokens come first and may not see the last key tiles.
  p.n_tok_a = min(n_tok, tok_x);
  p.n_tok_b = TURNS ? p.n_tok_a : n_tok - p.n_tok_a;
  p.n_steps = c1 - p.c0;
  p.n_a = TURNS ? (p.n_steps + 1) / 2 : max(0, min(c1, (p.pos0 + p.n_tok_a - 1) / KEYS + 1) - p.c0);
  p.n_b = TURNS ? p.n_steps / 2 : p.n_tok_b > 0 ? p.n_steps : 0;
  return p;
}

struct PfShared {
  uint64_t k_full[kPfStages], k_empty[kPfStages], v_full[kPfStages], v_empty[kPfStages], x_full[kPfRing];
  uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], q_ready[2], last[2];
  uint64_t a_scored, b_handed, a_read;             // where the tiles take turns
  uint64_t work_full[kPfAhead], work_empty[kPfAhead], want, answered, tmem_ready;
  uint32_t tmem_base;
  int abort;
  // Of the key tiles in flight, by step % 16 (steps are counted through all the block's pieces): factors of scores, addends, factors of
  // the denominator's terms, and the step (+ 1) that last had NaN among its values. x_full: all of them are there. (A step's place is
  // written again sixteen steps on. The conversion is at most four steps ahead of what both tiles have scored or let go of; a tile
  // lets steps go only behind its softmax's last step of a piece, three at most, and scores a piece's first step only when its
  // softmax has done with the piece before.)
  float k_scale[kPfRing][8], v_add[kPfRing][8], v_back[kPfRing][8];
  int v_nan[kPfRing];
  float handed[2][kPfRows];          // where B has A's rows: its bounds and denominators
  PfPiece work[kPfAhead];            // the block's pieces, by their number % 4
  alignas(16) uint32_t answer[4];    // to the last asking for another
};

// Asks for a thread block of this launch that has not begun, in whose stead this one works on; false: there is none any more (and
// nobody may ask again). All lanes of a warp call it; `asked`: how often it has been called.
__device__ __forceinline__ bool pf_another(PfShared& sh, int asked, int& index, volatile int* abort) {
  if ((threadIdx.x & 31) == 0) {
    fence_proxy_async_smem();        // the last answer has been read
    mbar_arrive_expect_tx(&sh.answered, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 ::"r"(smem_u32(sh.answer)), "r"(smem_u32(&sh.answered)) : "memory");
  }
  __syncwarp();
  if (!__all_sync(0xffffffffu, pf_wait(&sh.answered, asked & 1, abort))) {
    if ((threadIdx.x & 31) == 0) *abort = 1;
    return false;
  }
  uint32_t got, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(got), "=r"(x)
      : "r"(smem_u32(sh.answer))
      : "memory");
  __syncwarp();
  index = (int)x;
  return got != 0;
}

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
  uint8_t* out_smem = v_smem + Cfg::kStages * Cfg::kKvBytes;
  const int warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();

  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = TURNS ? tok_x : 2 * tok_x;      // tokens of a tile, of a block
  // one warp looks for the block's pieces of work while others set it up
  PfSequence mine;
  int run = 0;
  if (warp == 14) {
    mine = pf_sequence<Cfg::kKeys>(a, threadIdx.x & 31, tok);
    run = pf_run<Cfg::kKeys>(a, tok, mine);
    const PfWork found = pf_find<false, Cfg::kKeys>(a, tok, blockIdx.x, mine, run);
    if ((threadIdx.x & 31) == 0) sh.work[0] = pf_piece<TURNS, Cfg::kKeys>(a, found, tok_x);
  } else if (threadIdx.x == 32) {
    for (int s = 0; s < Cfg::kStages; ++s) {
      mbar_init(&sh.k_full[s], 128);
      mbar_init(&sh.k_empty[s], 2);
      mbar_init(&sh.v_full[s], 128);
      mbar_init(&sh.v_empty[s], 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh.s_full[s], 1);
      mbar_init(&sh.s_free[s], 128);
      mbar_init(&sh.p_ready[s], 128);
      mbar_init(&sh.pv_done[s], 1);
      mbar_init(&sh.q_ready[s], 128);
      mbar_init(&sh.last[s], 1);
    }
    for (int i = 0; i < kPfRing; ++i) {
      mbar_init(&sh.x_full[i], 128);
      sh.v_nan[i] = 0;
    }
    for (int i = 0; i < kPfAhead; ++i) {
      mbar_init(&sh.work_full[i], 1);
      mbar_init(&sh.work_empty[i], kPfReaders);
    }
    mbar_init(&sh.a_scored, 128);
    mbar_init(&sh.b_handed, 128);
    mbar_init(&sh.a_read, 128);
    mbar_init(&sh.want, 1);
    mbar_init(&sh.answered, 1);
    mbar_init(&sh.tmem_ready, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (sh.work[0].parts == 0) return; // the whole block alike
  volatile int* abort = &sh.abort;
#define LLMIE_FAIL(code) do { if (!*abort) { *abort = 1; atomicExch(a.status, (code)); } } while (0)
  // Whether there is a piece number n for this block (in sh.work until it is given back): false at the end of the work, or where a
  // wait gave up. All lanes of a warp call it, or one thread alone.
  auto piece_there = [&](int n) -> bool {
    if (!pf_wait(&sh.work_full[n % kPfAhead], (n / kPfAhead) & 1, abort)) {
      LLMIE_FAIL(kStatusTimeoutFull);
      return false;
    }
    return sh.work[n % kPfAhead].parts > 0;
  };

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax: a thread a row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PfRegs<HD>::kSoftmax));
    const int x = warp >> 2, r = threadIdx.x & 127;          // tile and row
    const int rt = r / G, rh = r - rt * G;                   // token of the tile, query head of the group
    const int lane = threadIdx.x & 31;
    constexpr int kPieces = HD / 8, kRowsAtOnce = 32 / kPieces, kLoads = 32 / kRowsAtOnce;   // of 16 bytes a row; rows a load of the warp's
    const uint32_t q_mine = smem_u32(q_smem + x * Cfg::kQBytes) + (lane % kPieces >> 3) * kPfSub;
    // where the i-th piece that this lane brings lies
    auto q_place = [&](int i) { return q_mine + swizzle128_offset((warp & 3) * 32 + i * kRowsAtOnce + lane / kPieces, lane & 7); };
    // which row of the queries and the output is this thread's (-1: none)
    auto row_of = [&](const PfPiece& p) {
      return rt < (x ? p.n_tok_b : p.n_tok_a) ? (p.row0 + (TURNS ? 0 : x * tok_x) + rt) * a.n_q + p.hk * G + rh : -1;
    };
    // A warp asks for its 32 rows of queries, a row by neighbouring lanes; rows that are not there are zeros.
    auto ask_for_queries = [&](const PfPiece& p) {
      const int mine = row_of(p);
#pragma unroll 4
      for (int i = 0; i < kLoads; ++i) {
        const int row = __shfl_sync(0xffffffffu, mine, i * kRowsAtOnce + lane / kPieces);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(q_place(i)), "l"(a.q + (size_t)max(row, 0) * HD + lane % kPieces * 8), "r"(row >= 0 ? 16 : 0) : "memory");
      }
    };
    bool more = __all_sync(0xffffffffu, piece_there(0));
    if (more) ask_for_queries(sh.work[0]);
    int gs = 0, gx = 0;              // steps of the block, and of this tile, before this piece
    int turns = 0;                   // pieces whose results B handed over
    bool ok = true;
    uint32_t tmem = 0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
#pragma unroll 1
    for (int n = 0; more; ++n) {
      const PfPiece& w = sh.work[n % kPfAhead];
      const int n_x = x ? w.n_b : w.n_a, c0 = w.c0;
      const int first = w.pos0 + (TURNS ? 0 : x * tok_x), n_more = max((x ? w.n_tok_b : w.n_tok_a) - 1, 0);
      const int end = a.max_pages * kFp8Page - 1;            // the last position that the table has room for
      const int qpos = min(first + min(rt, n_more), end), lo = first_visible_key(qpos, a.window);
      // the first and last keys that every row of the tile sees
      const int all_to = min(first, end), all_from = first_visible_key(min(first + n_more, end), a.window);
      // Queries become half precision where they lie, a row by its thread, with the power of two that brings its largest number into
      // [2^14, 2^15): 2^-113 at least, 2^126 at most (numbers below 2^-112 end up from 2^-7 on, with all digits of bfloat16).
      float f;                         // of the row's scores: scale log2(e) and the power of two
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncwarp();
      {
        const uint32_t row = smem_u32(q_smem + x * Cfg::kQBytes);
        auto piece_at = [&](int i) { return row + (i >> 3) * kPfSub + swizzle128_offset(r, i & 7); };
        uint32_t big[4] = {0u, 0u, 0u, 0u};      // the largest magnitudes by their bits, which are ordered as the numbers, what is not finite on top
#pragma unroll 8
        for (int i = 0; i < kPieces; ++i) {
          uint32_t u[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(piece_at(i)) : "memory");
#pragma unroll
          for (int e = 0; e < 4; ++e) big[e] = max(big[e], max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
        }
        const int eb = (int)(max(max(big[0], big[1]), max(big[2], big[3])) >> 7), shift = eb == 255 ? 0 : min(141 - eb, 126);
        const float up = pow2_of(shift);
        f = a.scale2 * pow2_of(-shift);
#pragma unroll 4
        for (int i = 0; i < kPieces; ++i) {
          uint32_t u[4];
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(piece_at(i)) : "memory");
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[e]));
            u[e] = pf_half2(y.x * up, y.y * up);
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(i)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&sh.q_ready[x]);
      if (n == 0) {
        if (!__all_sync(0xffffffffu, pf_wait(&sh.tmem_ready, 0, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          break;
        }
        tc_fence_after_sync();
        tmem = sh.tmem_base;
      }
      const uint32_t s_addr = tmem + lanes + Cfg::kSCol + x * Cfg::kKeys, o_addr = tmem + lanes + Cfg::kOCol + x * HD;
      const uint32_t p_addr = tmem + lanes + Cfg::kPCol + x * (Cfg::kKeys / 2);
      // a score's factor is never 0: times -inf, which stands where the row does not look, that would be NaN
      auto factor = [&](float k_scale) { return fminf(fmaxf(f * k_scale, 1.2e-38f), 3.4e38f); };
      float R = -INFINITY, l = 0.f;
      uint32_t nan_cols[HD / 32];
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) nan_cols[i] = 0u;
      // Rare: NaN where this row has seen a value that is NaN.
      auto poison = [&](auto put) {
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) {
#pragma unroll 1
          for (uint32_t bits = nan_cols[i]; bits; bits &= bits - 1) put(i * 32 + __ffs(bits) - 1);
        }
      };
      // Of a step whose values are all there. Rare: which columns of the values that this row sees are NaN.
      auto nan_values = [&](int step) {
        if (sh.v_nan[step % kPfRing] != step + 1) return;
        const int kbase = (c0 + step - gs) * Cfg::kKeys;
        const int* pages = a.block_table + (size_t)w.page_row * a.max_pages;
        const int last_key = w.last_key;
#pragma unroll 1
        for (int p = max(lo, kbase); p <= min(min(qpos, last_key), kbase + Cfg::kKeys - 1); ++p) {
          const unsigned* row = reinterpret_cast<const unsigned*>(a.v + (((size_t)pages[p / kFp8Page] * a.n_kv + w.hk) * kFp8Page + p % kFp8Page) * HD);
#pragma unroll
          for (int i = 0; i < HD / 32; ++i) {
            uint32_t bits = 0u;
#pragma unroll 1
            for (int e = 0; e < 32; ++e) bits |= ((row[i * 8 + e / 4] >> (e % 4 * 8) & 0x7fu) == 0x7fu ? 1u : 0u) << e;
            nan_cols[i] |= bits;
          }
        }
      };
      // Rare: the row's denominator by the scores alone (see fp8.cuh), four keys at a time, while the rest of the block waits: 800 clocks a
      // key at head size 64, 1,300 at 128 (2,048 tokens 0.9 and 2.2 ms; the waits' limit is reached behind more than a million keys).
      auto by_scores = [&]() {
        const int row = row_of(w);
        if (row < 0) return;
        const uint32_t* q = reinterpret_cast<const uint32_t*>(a.q + (size_t)row * HD);
        uint32_t big = 0u;
#pragma unroll 1
        for (int i = 0; i < HD / 2; ++i) big = max(big, max(q[i] & 0x7fffu, q[i] >> 16 & 0x7fffu));
        const int eb = (int)(big >> 7);
        const float up = pow2_of(eb == 255 ? 0 : min(141 - eb, 126)), shift = R - kPfTop;
        const int* pages = a.block_table + (size_t)w.page_row * a.max_pages;
        l = 0.f;
#pragma unroll 1
        for (int j = 0; j < n_x; ++j) {
          const int kbase = (c0 + (TURNS ? 2 * j + x : j)) * Cfg::kKeys;
#pragma unroll 1
          for (int p = max(lo, kbase) & ~3; p <= min(qpos, kbase + Cfg::kKeys - 1); p += 4) {
            const size_t head = (size_t)pages[p / kFp8Page] * a.n_kv + w.hk;
            const uint4* k = reinterpret_cast<const uint4*>(a.k + (head * kFp8Page + p % kFp8Page) * HD);
            const float fk = factor(pow2_of(clamp_exponent(a.k_exp[head * kPageExps + p % kFp8Page / kExpBlock])));
            float dot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int i = 0; i < HD / 16; ++i) {
              uint32_t y[8];
              *reinterpret_cast<uint4*>(y) = reinterpret_cast<const uint4*>(q)[2 * i];
              *reinterpret_cast<uint4*>(y + 4) = reinterpret_cast<const uint4*>(q)[2 * i + 1];
              uint4 z[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) z[e] = k[e * (HD / 16) + i];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const unsigned c[4] = {z[e].x, z[e].y, z[e].z, z[e].w};
#pragma unroll
                for (int h = 0; h < 8; ++h) {
                  const float2 u = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[h]));
                  const float2 o = e4m3x2_to_float2((unsigned short)(c[h >> 1] >> (h & 1) * 16 & 0xffffu));
                  dot[e] = fmaf(u.x * up, o.x, dot[e]);
                  dot[e] = fmaf(u.y * up, o.y, dot[e]);
                }
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (p + e >= lo && p + e <= qpos) l += exp2_term(fmaf(dot[e], fk, -shift));
          }
        }
      };
#pragma unroll 1
      for (int j = 0; j < n_x; ++j) {            // this tile's j-th step is the block's `step`
        const int step = gs + (TURNS ? 2 * j + x : j);
        // every decision to give up is taken by the whole warp: reads of tensor memory are warp-wide instructions
        if (!__all_sync(0xffffffffu, pf_wait(&sh.x_full[step % kPfRing], (step / kPfRing) & 1, abort) && pf_wait(&sh.s_full[x], (gx + j) & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const int kbase = (c0 + step - gs) * Cfg::kKeys, ring = step % kPfRing;
        const bool edge = kbase + Cfg::kKeys - 1 > all_to || kbase < all_from;
        // the row's scores; those that it does not see are -inf
        uint32_t v[Cfg::kKeys / 32][32];
#pragma unroll
        for (int c = 0; c < Cfg::kKeys / 32; ++c) tmem_ld_32x32(s_addr + c * 32, v[c]);
        float fk[Cfg::kBlocks];
#pragma unroll
        for (int b = 0; b < Cfg::kBlocks; ++b) fk[b] = factor(sh.k_scale[ring][b]);
        tmem_ld_wait();
        // they are in registers: the next scores may be written
        tc_fence_before_sync();
        mbar_arrive(&sh.s_free[x]);
        if (edge) {
          const int from = lo - kbase;
          const unsigned span = (unsigned)(qpos - lo);
#pragma unroll
          for (int i = 0; i < Cfg::kKeys; ++i)
            if ((unsigned)(i - from) > span) v[i >> 5][i & 31] = 0xff800000u;
        }
        float mx = -INFINITY;          // the largest s + ev
#pragma unroll
        for (int b = 0; b < Cfg::kBlocks; ++b) {
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
          if (!__all_sync(0xffffffffu, pf_wait(&sh.pv_done[x], (gx + j - 1) & 1, abort))) {
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
        if (j > 0) {
          // the weights of the tile before have to be through the product before they are written over
          if (!__all_sync(0xffffffffu, pf_wait(&sh.pv_done[x], (gx + j - 1) & 1, abort))) {
            LLMIE_FAIL(kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          nan_values(step - (TURNS ? 2 : 1));
        }
        // the weights, in columns of their own
#pragma unroll
        for (int c = 0; c < Cfg::kKeys / 32; ++c) {
          uint32_t o[16];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float add = sh.v_add[ring][c * 2 + b] - shift;
            const uint32_t* y = v[c] + b * 16;
            float sum[4];
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float x0 = pf_exp2(fmaf(__uint_as_float(y[i]), fk[c * 2 + b], add));
              const float x1 = pf_exp2(fmaf(__uint_as_float(y[i + 1]), fk[c * 2 + b], add));
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
      }
      if (ok && __float_as_uint(l) - 1u < __float_as_uint(kLeastDenominator) - 1u) by_scores();
      // the queries of the piece after this one are asked for while the last product runs
      const int at_end = gs + (TURNS ? 2 * (n_x - 1) + x : n_x - 1);             // this tile's last step
      gx += n_x;
      const bool early = ok && __all_sync(0xffffffffu, mbar_test(&sh.work_full[(n + 1) % kPfAhead], ((n + 1) / kPfAhead) & 1));
      const bool merge = TURNS && w.parts == 1;      // then the place of the queries is wanted first
      if (early && !merge && sh.work[(n + 1) % kPfAhead].parts > 0) ask_for_queries(sh.work[(n + 1) % kPfAhead]);
      if (ok && n_x > 0) {
        if (!__all_sync(0xffffffffu, pf_wait(&sh.pv_done[x], (gx - 1) & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
        }
        tc_fence_after_sync();
        if (ok) nan_values(at_end);
      }
      gs += w.n_steps;
      if (merge) {
        // B hands its results to A through the place of the queries, which nobody reads any more once both tiles' scores are done
        // (partial ones are joined later, B's with A's)
        float* handed = reinterpret_cast<float*>(q_smem) + r * HD;
        if (x == 0) mbar_arrive(&sh.a_scored);
        if (!__all_sync(0xffffffffu, x == 0 || pf_wait(&sh.a_scored, turns & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
        }
        if (x == 1) {
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t y[32];
            tmem_ld_32x32(o_addr + c * 32, y);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; i += 4)            // places of a row shifted by the row: other banks for other rows
              *reinterpret_cast<uint4*>(handed + (c * 32 + i + r * 4) % HD) =
                  n_x > 0 ? make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]) : make_uint4(0u, 0u, 0u, 0u);
          }
          poison([&](int d) { handed[(d + r * 4) % HD] = __int_as_float(0x7fffffff); });
          sh.handed[0][r] = R;
          sh.handed[1][r] = l;
          mbar_arrive(&sh.b_handed);
        }
        if (!__all_sync(0xffffffffu, x == 1 || pf_wait(&sh.b_handed, turns & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
        }
      }
      // ---- the row's result: the output, or a partial one. Where a wait gave up: NaN.
      if (!merge || x == 0) {
        float mine_f = 1.f, b_f = 0.f;
        if (merge) {
          const float Rb = sh.handed[0][r], M = fmaxf(R, Rb), Mu = M == -INFINITY ? 0.f : M;
          mine_f = R == -INFINITY ? 0.f : pf_exp2(R - Mu);
          b_f = Rb == -INFINITY ? 0.f : pf_exp2(Rb - Mu);
          l = add_times_exp2(l, mine_f, R - Mu, times_exp2(sh.handed[1][r], b_f, Rb - Mu));
        }
        if (!ok) l = __int_as_float(0x7fffffff);
        const float* handed = reinterpret_cast<const float*>(q_smem) + r * HD;
        const int row = row_of(w);
        const bool cut = w.parts > 1;
        float* rec = a.part + (size_t)w.slot * Cfg::kRecord + (x * kPfRows + r) * 4;
        if (cut && row >= 0) {
          rec[2 * kPfRows * HD - (x * kPfRows + r) * 3] = R;
          rec[2 * kPfRows * (HD + 1) - (x * kPfRows + r) * 3] = l;
        }
        const float by = cut ? 1.f : mine_f / l, b_by = b_f / l;
        // 32 columns at a time: partial ones lie row beside row, four columns a piece; the output's are turned in shared memory, so that
        // neighbouring lanes write a row's
        const uint32_t turn = smem_u32(out_smem) + warp * 2048;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t y[32];
          tmem_ld_32x32(o_addr + c * 32, y);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = n_x > 0 ? __float_as_uint(__uint_as_float(y[i]) * by) : 0u;
          if (merge) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 z = *reinterpret_cast<const float4*>(handed + (c * 32 + i + r * 4) % HD);
              y[i] = __float_as_uint(fmaf(z.x, b_by, __uint_as_float(y[i])));
              y[i + 1] = __float_as_uint(fmaf(z.y, b_by, __uint_as_float(y[i + 1])));
              y[i + 2] = __float_as_uint(fmaf(z.z, b_by, __uint_as_float(y[i + 2])));
              y[i + 3] = __float_as_uint(fmaf(z.w, b_by, __uint_as_float(y[i + 3])));
            }
          }
          if (cut) {
            if (row >= 0) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4*>(rec + (size_t)(c * 8 + i / 4) * 8 * kPfRows) = make_uint4(y[i], y[i + 1], y[i + 2], y[i + 3]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              uint32_t o[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(y[i + 2 * e]), __uint_as_float(y[i + 2 * e + 1]));
                o[e] = *reinterpret_cast<const uint32_t*>(&h);
              }
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                           ::"r"(turn + lane * 64 + ((i / 8) ^ (lane >> 1 & 3)) * 16), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int of = i * 8 + lane / 4, to = __shfl_sync(0xffffffffu, row, of);
              uint4 z;
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(z.x), "=r"(z.y), "=r"(z.z), "=r"(z.w)
                           : "r"(turn + of * 64 + ((lane & 3) ^ (of >> 1 & 3)) * 16) : "memory");
              if (to >= 0) *reinterpret_cast<uint4*>(a.out + (size_t)to * HD + c * 32 + (lane & 3) * 8) = z;
            }
            __syncwarp();
          }
        }
        // columns of values that are NaN, or, where B handed them over, were (then they are so already)
        if (row >= 0 && cut) poison([&](int d) { rec[(size_t)(d / 4) * 8 * kPfRows + d % 4] = __int_as_float(0x7fffffff); });
        if (row >= 0 && !cut) poison([&](int d) { a.out[(size_t)row * HD + d] = __float2bfloat16_rn(__int_as_float(0x7fffffff)); });
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.work_empty[n % kPfAhead]);
      more = ok && __all_sync(0xffffffffu, piece_there(n + 1));
      if (merge) {
        // the place is the queries' again when all of A's rows have been read
        if (x == 0) mbar_arrive(&sh.a_read);
        if (more && !__all_sync(0xffffffffu, pf_wait(&sh.a_read, turns & 1, abort))) {
          LLMIE_FAIL(kStatusTimeoutMma);
          ok = false;
        }
        ++turns;
      }
      if (more && (!early || merge)) ask_for_queries(sh.work[(n + 1) % kPfAhead]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");         // nothing in flight at the end, where a wait gave up either
  } else if (warp < 12) {
    // ------------------------------------------------------------------ conversion: 128 threads, 16 codes at a time
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PfRegs<HD>::kConvert));
    constexpr int kPieces = HD / 16, kStep = 128 / kPieces;  // pieces of 16 codes a row; a thread's rows: row0, row0 + kStep, ...
    constexpr int kPer = Cfg::kKeys / kStep, kPages = Cfg::kKeys / kFp8Page;
    const int ct = threadIdx.x & 127, piece = ct % kPieces, row0 = ct / kPieces;
    uint4 kr[kPer], vr[kPer];        // a step's codes
    // Everything is asked for before it is looked at: a tile's pages a step before its codes, its codes and exponents a step
    // before they are written out. (Where an exponent was clamped, or a page's address made, as soon as it was asked for, the
    // conversion waited for memory twice a tile, and the whole kernel for the conversion: 3,500 clocks a step.)
    int pg0 = 0, pg1 = 0;            // pages of the tile to be asked for next
    signed char ke = 0, ve = 0;      // a thread's two exponents
    int last_key = 0, hk = 0;
    const int* pages = nullptr;
    auto page_at = [&](int lp) { return lp * kFp8Page <= last_key ? pages[lp] : 0; };
    // piece i of a tile's keys, or values. Rows behind the block's last key: zeros, nothing that may be NaN.
    auto load = [&](uint4& to, int i, const unsigned char* at0, const unsigned char* at1, int first) {
      to = make_uint4(0u, 0u, 0u, 0u);
      if (first + i * kStep <= last_key) to = *reinterpret_cast<const uint4*>((i * kStep < kFp8Page ? at0 + i * kStep * HD : at1 + (i * kStep - kFp8Page) * HD));
    };
    // where this thread's pieces of a page begin
    auto in_page = [&](int page) { return (((size_t)page * a.n_kv + hk) * kFp8Page + row0) * HD + piece * 16; };
    // Exponents of the tile's eight blocks, a thread a block (one behind the last key: anything, nobody sees its scores).
    auto load_exps = [&]() {
      if (ct < Cfg::kBlocks) {
        const size_t at = ((size_t)(ct < 4 ? pg0 : pg1) * a.n_kv + hk) * kPageExps + (ct & 3);
        ke = a.k_exp[at];
        ve = a.v_exp[at];
      }
    };
    auto put = [&](uint8_t* dst, const uint4& from, int i) {
      const int row = row0 + i * kStep;
      const unsigned c[4] = {from.x, from.y, from.z, from.w};
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        h[2 * e] = e4m3x2_to_half2((unsigned short)(c[e] & 0xffffu));
        h[2 * e + 1] = e4m3x2_to_half2((unsigned short)(c[e] >> 16));
      }
      uint8_t* at = dst + (piece >> 2) * Cfg::kKvSub;
      const int ch = (piece & 3) * 2, odd = piece >> 2 & 1;            // the two 64-column halves of a row in turn: other banks
      const uint4 lo4 = make_uint4(h[0], h[1], h[2], h[3]), hi4 = make_uint4(h[4], h[5], h[6], h[7]);
      *reinterpret_cast<uint4*>(at + swizzle128_offset(row, ch + odd)) = odd ? hi4 : lo4;
      *reinterpret_cast<uint4*>(at + swizzle128_offset(row, ch + 1 - odd)) = odd ? lo4 : hi4;
    };
    int gs = 0;                      // steps so far
    bool ok = true;
#pragma unroll 1
    for (int n = 0; ok && __all_sync(0xffffffffu, piece_there(n)); ++n) {
      const PfPiece& w = sh.work[n % kPfAhead];
      const int n_steps = w.n_steps, c0 = w.c0;
      last_key = w.last_key;
      hk = w.hk;
      pages = a.block_table + (size_t)w.page_row * a.max_pages;
      __syncwarp();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.work_empty[n % kPfAhead]);
      if (n_steps > 0) {
        pg0 = page_at(c0 * kPages);
        if (kPages > 1) pg1 = page_at(c0 * kPages + 1);
        const int next0 = page_at((c0 + 1) * kPages), next1 = kPages > 1 ? page_at((c0 + 1) * kPages + 1) : 0;
        const size_t at0 = in_page(pg0), at1 = in_page(pg1);
#pragma unroll
        for (int i = 0; i < kPer; ++i) load(kr[i], i, a.k + at0, a.k + at1, c0 * Cfg::kKeys + row0);
#pragma unroll
        for (int i = 0; i < kPer; ++i) load(vr[i], i, a.v + at0, a.v + at1, c0 * Cfg::kKeys + row0);
        load_exps();
        pg0 = next0;
        pg1 = next1;
      } else if (ct == 0) {
        mbar_arrive(&sh.want);
      }
#pragma unroll 1
      for (int j = 0; j < n_steps; ++j, ++gs) {
        const int st = gs % Cfg::kStages, ring = gs % kPfRing;
        if (ct == 0 && j == max(n_steps - 2, 0)) mbar_arrive(&sh.want);
        // the next step's pages are pg0, pg1; those of the one behind it:
        const int next0 = page_at((c0 + j + 2) * kPages), next1 = kPages > 1 ? page_at((c0 + j + 2) * kPages + 1) : 0;
        if (gs >= Cfg::kStages && !pf_wait(&sh.k_empty[st], (gs / Cfg::kStages - 1) & 1, abort)) {
          LLMIE_FAIL(kStatusTimeoutEmpty);
          ok = false;
          break;
        }
        if (ct < Cfg::kBlocks) {
          const int k = clamp_exponent(ke), v = clamp_exponent(ve);
          sh.k_scale[ring][ct] = pow2_of(k);
          sh.v_add[ring][ct] = (float)v;
          sh.v_back[ring][ct] = pow2_of(-v);
        }
        const int ahead = j + 1 < n_steps ? (c0 + j + 1) * Cfg::kKeys + row0 : 0x40000000;       // no tile after the last one
        const size_t at0 = in_page(pg0), at1 = in_page(pg1);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          put(k_smem + st * Cfg::kKvBytes, kr[i], i);
          load(kr[i], i, a.k + at0, a.k + at1, ahead);
        }
        if (j + 1 < n_steps) load_exps();
        fence_proxy_async_smem();
        mbar_arrive(&sh.x_full[ring]);
        mbar_arrive(&sh.k_full[st]);
        if (gs >= Cfg::kStages && !pf_wait(&sh.v_empty[st], (gs / Cfg::kStages - 1) & 1, abort)) {
          LLMIE_FAIL(kStatusTimeoutEmpty);
          ok = false;
          break;
        }
        // NaN among the values: such codes become zeros here
        unsigned any = 0u;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          any |= ((vr[i].x & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].y & 0x7f7f7f7fu) + 0x01010101u) |
                 ((vr[i].z & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].w & 0x7f7f7f7fu) + 0x01010101u);
        if (any & 0x80808080u) {
          sh.v_nan[ring] = gs + 1;
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
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          put(v_smem + st * Cfg::kKvBytes, vr[i], i);
          load(vr[i], i, a.v + at0, a.v + at1, ahead);
        }
        pg0 = next0;
        pg1 = next1;
        fence_proxy_async_smem();
        mbar_arrive(&sh.v_full[st]);
      }
    }
  } else {
    // ------------------------------------------------------------------ the tensor core: a thread a tile, so that neither waits for the other's
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PfRegs<HD>::kIssue));
    if (warp == 12) {
      tmem_alloc(&sh.tmem_base, 512);
      tmem_relinquish();
      tc_fence_before_sync();
      if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.tmem_ready);
    }
    if (warp == 14) {
      // ---------------------------------------------------------------- more work: asked for when the block has two steps left, so that
      // who is done first goes on with what is left
      if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.work_full[0]);
      bool others = true;
#pragma unroll 1
      for (int n = 1, asked = 0; others; ++n) {
        if (!__all_sync(0xffffffffu, pf_wait(&sh.want, (n - 1) & 1, abort))) break;
        int index;
        PfWork w{0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
        do {                         // (there are more blocks than pieces: nobody has to begin those behind the last piece)
          others = pf_another(sh, asked++, index, abort);
          if (others) w = pf_find<false, Cfg::kKeys>(a, tok, index, mine, run);
        } while (others && w.parts == 0);
        if (n >= kPfAhead && !__all_sync(0xffffffffu, pf_wait(&sh.work_empty[n % kPfAhead], (n / kPfAhead - 1) & 1, abort))) break;
        if ((threadIdx.x & 31) == 0) {
          sh.work[n % kPfAhead] = pf_piece<TURNS, Cfg::kKeys>(a, w, tok_x);
          mbar_arrive(&sh.work_full[n % kPfAhead]);
        }
      }
    }
    if (warp < 14 && elect_one()) {
      constexpr uint32_t idesc_s = pf_instr_desc(kPfRows, Cfg::kKeys, 0), idesc_o = pf_instr_desc(kPfRows, HD, 1);
      const int tx = warp - 12;
      bool ok = pf_wait(&sh.tmem_ready, 0, abort);
      if (!ok) LLMIE_FAIL(kStatusTimeoutMma);
      tc_fence_after_sync();
      const uint32_t tmem = sh.tmem_base;
      int gs = 0, gx = 0;            // steps of the block, and of this tile, before this piece
      const uint32_t s_col = tmem + Cfg::kSCol + tx * Cfg::kKeys, o_col = tmem + Cfg::kOCol + tx * HD;
      const uint32_t p_col = tmem + Cfg::kPCol + tx * (Cfg::kKeys / 2);
      // descriptors of the operands' first 16 columns; the rest lie a fixed number of 16-byte units on
      const uint64_t q_desc = make_smem_desc(smem_u32(q_smem + tx * Cfg::kQBytes), 16, 1024);
      const uint64_t k_desc = make_smem_desc(smem_u32(k_smem), 16, 1024), v_desc = make_smem_desc(smem_u32(v_smem), Cfg::kKvSub, 1024);
      auto wait_for = [&](uint64_t* bar, uint32_t parity, int code) {
        if (pf_wait(bar, parity, abort)) return true;
        LLMIE_FAIL(code);
        return false;
      };
      // a stage is free when both tiles have let go of it; where they take steps in turn, the one that has it lets go twice
      auto let_go = [&](uint64_t* bar) {
        mma_commit(bar);
        if (TURNS) mma_commit(bar);
      };
      auto scores = [&](int j) -> bool {                     // S = Q K^T of this tile's j-th step
        const int step = gs + (TURNS ? 2 * j + tx : j);
        if (!wait_for(&sh.k_full[step % Cfg::kStages], (step / Cfg::kStages) & 1, kStatusTimeoutFull)) return false;
        tc_fence_after_sync();
        const uint64_t kd = k_desc + (uint64_t)((step % Cfg::kStages) * (Cfg::kKvBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const int q_off = ((kk >> 2) * kPfSub + (kk & 3) * 32) >> 4, k_off = ((kk >> 2) * Cfg::kKvSub + (kk & 3) * 32) >> 4;
          mma_bf16_ss(s_col, q_desc + q_off, kd + k_off, idesc_s, kk > 0 ? 1u : 0u);
        }
        mma_commit(&sh.s_full[tx]);
        let_go(&sh.k_empty[step % Cfg::kStages]);
        return true;
      };
      auto sums = [&](int j) -> bool {                       // O (+)= W V of it
        const int step = gs + (TURNS ? 2 * j + tx : j);
        if (!wait_for(&sh.v_full[step % Cfg::kStages], (step / Cfg::kStages) & 1, kStatusTimeoutFull)) return false;
        if (!wait_for(&sh.p_ready[tx], (gx + j) & 1, kStatusTimeoutMma)) return false;
        tc_fence_after_sync();
        const uint64_t vd = v_desc + (uint64_t)((step % Cfg::kStages) * (Cfg::kKvBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < Cfg::kKeys / 16; ++kk)            // 16 weights are 8 columns; 16 keys are 16 rows of the values
          pf_mma_ts(o_col, p_col + kk * 8, vd + kk * (2048 >> 4), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
        mma_commit(&sh.pv_done[tx]);
        let_go(&sh.v_empty[step % Cfg::kStages]);
        return true;
      };
#pragma unroll 1
      for (int n = 0; ok && piece_there(n); ++n) {
        const int n_x = tx ? sh.work[n % kPfAhead].n_b : sh.work[n % kPfAhead].n_a, n_steps = sh.work[n % kPfAhead].n_steps;
        mbar_arrive(&sh.work_empty[n % kPfAhead]);
        // the softmax has done with the piece before, and the queries of this one are there
        ok = wait_for(&sh.q_ready[tx], n & 1, kStatusTimeoutFull);
        tc_fence_after_sync();
        ok = ok && (n_x == 0 || scores(0));
#pragma unroll 1
        for (int j = 0; ok && j < n_x; ++j) {
          // the next scores as soon as these are in registers
          if (j + 1 < n_x) ok = wait_for(&sh.s_free[tx], (gx + j) & 1, kStatusTimeoutMma) && scores(j + 1);
          ok = ok && sums(j);
        }
        // steps that are the other tile's alone
#pragma unroll 1
        for (int j = n_x; ok && !TURNS && j < n_steps; ++j) {
          const int step = gs + j;
          ok = wait_for(&sh.k_full[step % Cfg::kStages], (step / Cfg::kStages) & 1, kStatusTimeoutFull);
          if (ok) mbar_arrive(&sh.k_empty[step % Cfg::kStages]);
          ok = ok && wait_for(&sh.v_full[step % Cfg::kStages], (step / Cfg::kStages) & 1, kStatusTimeoutFull);
          if (ok) mbar_arrive(&sh.v_empty[step % Cfg::kStages]);
        }
        gs += n_steps;
        gx += n_x;
      }
      // nothing may be in flight when the tensor memory is given back
      mma_commit(&sh.last[tx]);
#pragma unroll 1
      for (unsigned spin = 0; spin < (1u << 20) && !mbar_test(&sh.last[tx], 0); ++spin) __nanosleep(32);
    }
  }
#undef LLMIE_FAIL
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after_sync();
    tmem_dealloc(sh.tmem_base, 512);
  }
}

// Joins the runs of the tiles that were cut. grid (tiles of tokens x key/value heads, 8).
constexpr int kPfJoinWarps = 8, kPfJoinSide = 8;
template <int HD, bool TURNS> __global__ void __launch_bounds__(kPfJoinWarps * 32) prefill_fp8_join_kernel(const PrefillArgs a) {
  pdl_launch_dependents();
  using Cfg = PfCfg<HD>;
  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = TURNS ? tok_x : 2 * tok_x;
  const PfSequence mine = pf_sequence<Cfg::kKeys>(a, threadIdx.x & 31, tok);
  const PfWork w = pf_find<true, Cfg::kKeys>(a, tok, blockIdx.x, mine, pf_run<Cfg::kKeys>(a, tok, mine));
  // The lengths are older than the kernel that leaves the partial results (it lets this one begin behind its own wait). Blocks with
  // nothing to join wait too: the kernel behind this one waits for this one alone, and reads what the one in front wrote.
  pdl_wait();
  if (w.parts <= 1) return;
  // a thread four columns of a row, neighbouring threads neighbouring rows, as the results lie
  constexpr int kRows = TURNS ? kPfRows : 2 * kPfRows, kHalves = TURNS ? 2 : 1;              // in turns, both halves of a result are of the same rows
  const int results = w.parts * kHalves;
  const float* base = a.part + (size_t)w.slot * Cfg::kRecord;
  for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < kRows * (HD / 4); it += gridDim.y * blockDim.x) {
    const int row = it % kRows, group = it / kRows;
    const int x = row / kPfRows, rt = row % kPfRows / G, rh = row % kPfRows - rt * G, t = w.tile * tok + x * tok_x + rt;
    if (rt >= tok_x || t >= w.q_len) continue;
    float M = -INFINITY, den = 0.f, num[4] = {0.f, 0.f, 0.f, 0.f};
    // eight runs at a time, all asked for at once
    for (int p0 = 0; p0 < results; p0 += 8) {
      float m[8], l[8];
      float4 v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const bool there = p0 + p < results;
        const int at = there ? p0 + p : 0;
        const float* r = base + (size_t)(at / kHalves) * Cfg::kRecord;
        const int in = at % kHalves * kPfRows + row;
        m[p] = there ? __ldcg(r + 2 * kPfRows * HD + in) : -INFINITY;
        l[p] = there ? __ldcg(r + 2 * kPfRows * (HD + 1) + in) : 0.f;
        v[p] = there ? __ldcg(reinterpret_cast<const float4*>(r) + (size_t)group * 2 * kPfRows + in) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float M8 = M;
#pragma unroll
      for (int p = 0; p < 8; ++p) M8 = fmaxf(M8, m[p]);
      const float Mu = M8 == -INFINITY ? 0.f : M8, back = M == -INFINITY ? 0.f : pf_exp2(M - Mu);
      if (M != -INFINITY) den = times_exp2(den, back, M - Mu);             // (without a bound there is nothing yet, or NaN, which stays)
#pragma unroll
      for (int i = 0; i < 4; ++i) num[i] *= back;
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float f = pf_exp2(m[p] - Mu);
        den = add_times_exp2(l[p], f, m[p] - Mu, den);
        num[0] = fmaf(f, v[p].x, num[0]);
        num[1] = fmaf(f, v[p].y, num[1]);
        num[2] = fmaf(f, v[p].z, num[2]);
        num[3] = fmaf(f, v[p].w, num[3]);
      }
      M = M8;
    }
    const float inv = 1.f / den;
    uint2 o;
    __nv_bfloat162 h = __floats2bfloat162_rn(num[0] * inv, num[1] * inv);
    o.x = *reinterpret_cast<const uint32_t*>(&h);
    h = __floats2bfloat162_rn(num[2] * inv, num[3] * inv);
    o.y = *reinterpret_cast<const uint32_t*>(&h);
    *reinterpret_cast<uint2*>(a.out + ((size_t)(w.q_begin + t) * a.n_q + w.hk * G + rh) * HD + group * 4) = o;
  }
}

// What the host settles of a call before it launches. Nothing of the lengths is known but that they are n_tokens together at most.
struct PfPlan {
  int run;                           // PrefillArgs::run
  bool cut;                          // whether tiles of tokens may be cut into runs: scratch, and a join
  long long items, blocks;           // tiles of tokens x key/value heads at most; thread blocks of the kernel
  long long most_tiles;              // key tiles that a token may see
};
template <int HD> static PfPlan pf_plan(int n_tokens, int n_seqs, int max_q_len, int max_pages, int n_q, int n_kv, int window) {
  using Cfg = PfCfg<HD>;
  PfPlan p;
  const int tok_x = kPfRows / (n_q / n_kv), tok = (max_q_len <= tok_x ? 1 : 2) * tok_x;
  // Pieces of work: the tiles of tokens, and the runs that they may be cut into (see pf_run). The most runs that a tile can have
  // follow from the most keys that the table has room for and the least work that so many tokens are.
  p.items = max_q_len <= tok ? (long long)n_seqs * n_kv : ((long long)n_tokens / tok + n_seqs) * n_kv;
  double least = (double)n_tokens / tok * n_kv;
  p.most_tiles = ((long long)max_pages * kFp8Page + Cfg::kKeys - 1) / Cfg::kKeys;
  if (window == 0) {
    least *= (1.0 + (double)n_tokens / ((double)Cfg::kKeys * n_seqs)) / 2;
  } else {
    const long long w = window < 0 ? -(long long)window : window;
    p.most_tiles = min(p.most_tiles, (w + tok) / Cfg::kKeys + 2);
  }
  const bool many = (double)n_tokens / tok * n_kv > kPfSms;                  // more tiles than SMs whatever the sequences' lengths
  long long run = (long long)(least * (many ? 2 : 1) / kPfSms);
  run = min(max(run, (long long)kPfLeast / Cfg::kKeys), 1LL << 30);
  p.cut = p.most_tiles > kPfWhole / Cfg::kKeys && (many ? (p.most_tiles + run / 2) / run > 1 : p.most_tiles > run);
  p.run = p.cut ? (int)run : 0;
  p.blocks = !p.cut ? p.items : p.items <= kPfFew ? kPfSms : p.items + kPfSms;
  return p;
}

template <int HD, bool TURNS>
static int launch_prefill_fp8(PrefillArgs a, const PfPlan& plan, cudaStream_t stream) {
  using Cfg = PfCfg<HD>;
  if (plan.cut && !a.part) return kPfNeedsScratch;
  if (plan.blocks * plan.most_tiles > 0x3fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  cudaError_t e = cudaFuncSetAttribute(prefill_fp8_kernel<HD, TURNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return (int)e;
  a.run = plan.run;
  launch_k(prefill_fp8_kernel<HD, TURNS>, dim3((unsigned)plan.blocks), dim3(kPfThreads), Cfg::kSmem, stream, a);
  LLMIE_LAUNCH_CHECK();
  if (plan.cut) {
    const unsigned side = (unsigned)max(1LL, min((long long)kPfJoinSide, 8LL * kPfSms / plan.items));
    launch_k(prefill_fp8_join_kernel<HD, TURNS>, dim3((unsigned)plan.items, side), dim3(kPfJoinWarps * 32), 0, stream, a);
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
  if (max_pages > kMostPages) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!(scale > 0.f)) return LLMIE_ERR_BAD_ARG;              // a row's bound is taken before scores are scaled
  if ((hd != 64 && hd != 128) || n_q / n_kv > kPfRows) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(scratch)) return LLMIE_ERR_ALIGNMENT;
  if (n_tokens == 0 || n_seqs == 0 || max_q_len <= 0) return LLMIE_OK;
  const PrefillArgs a{(const __nv_bfloat16*)q, (const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp,
                      (const signed char*)v_exp, (__nv_bfloat16*)out, scratch, status, cu_q, seq_slot, seq_start, block_table,
                      max_pages, n_seqs, n_q, n_kv, scale * 1.4426950408889634f, window, 0};
  const bool turns = max_q_len <= kPfRows / (n_q / n_kv);
#define LLMIE_PREFILL(HD)                                                                                    \
  const PfPlan plan = pf_plan<HD>(n_tokens, n_seqs, max_q_len, max_pages, n_q, n_kv, window);               \
  return turns ? launch_prefill_fp8<HD, true>(a, plan, stream) : launch_prefill_fp8<HD, false>(a, plan, stream)
  if (hd == 64) {
    LLMIE_PREFILL(64);
  }
  LLMIE_PREFILL(128);
#undef LLMIE_PREFILL
}

// How such a call is laid out, on the host: plan[0] the length of a run that the device's cut goes by, in key tiles of 128 (head size 64) or 64
// (128) keys, plan[1] whether tiles may be cut (scratch and a join), plan[2] thread blocks, plan[3] the partial results that there is room for.
extern "C" int llmie_attention_prefill_fp8_plan(int n_tokens, int n_seqs, int max_q_len, int max_pages, int n_q, int n_kv, int hd,
                                                int window, long long* plan) {
  if (n_tokens <= 0 || n_seqs <= 0 || max_q_len <= 0 || max_pages <= 0 || n_kv <= 0 || n_q % n_kv || n_q / n_kv < 1 ||
      n_q / n_kv > kPfRows)
    return LLMIE_ERR_BAD_ARG;
  if (hd != 64 && hd != 128) return LLMIE_ERR_UNSUPPORTED_SIZE;
  const PfPlan p = hd == 64 ? pf_plan<64>(n_tokens, n_seqs, max_q_len, max_pages, n_q, n_kv, window)
                            : pf_plan<128>(n_tokens, n_seqs, max_q_len, max_pages, n_q, n_kv, window);
  plan[0] = p.run;
  plan[1] = p.cut;
  plan[2] = p.blocks;
  plan[3] = kPfSlots;
  return LLMIE_OK;
}

// The same by one address, with the arguments one behind another as they are above: a caller from another language converts one
// argument instead of 22, which takes as long as the launch.
struct PrefillCall {
  const void *q, *k_cache, *v_cache, *k_exp, *v_exp;
  void* out;
  float* scratch;
  int* status;
  const int *cu_q, *seq_slot, *seq_start, *block_table;
  int max_pages, n_tokens, n_seqs, max_q_len, n_q, n_kv, hd;
  float scale;
  int window;
  cudaStream_t stream;
};
extern "C" int llmie_attention_prefill_fp8_call(const PrefillCall* c) {
  return llmie_attention_prefill_fp8(c->q, c->k_cache, c->v_cache, c->k_exp, c->v_exp, c->out, c->scratch, c->status, c->cu_q, c->seq_slot,
                                     c->seq_start, c->block_table, c->max_pages, c->n_tokens, c->n_seqs, c->max_q_len, c->n_q, c->n_kv,
                                     c->hd, c->scale, c->window, c->stream);
}
