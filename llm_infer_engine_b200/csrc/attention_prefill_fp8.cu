// Causal attention of several new tokens a sequence over a paged cache in 8 bits (fp8.cuh), on the 5th-generation tensor cores.
//
//   o_t = sum_j 2^(s_tj) c_j 2^(ev_j) / sum_j 2^(s_tj),   s_tj = scale log2(e) (q_t . k_j) 2^(ek_j),   j seen by t     (k, c: codes)
//
// Rows. A key/value head is read once for all of its query heads: the rows of a 128-row operand are (token, query head) pairs,
// 128 / G tokens of the G heads that share the key/value head. A block has two such tiles, A and B, with a softmax warpgroup
// each (a thread a row); while one works on its scores the tensor core is busy with the other's.
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
constexpr int kPfThreads = 512;      // warps 0-3, 4-7: softmax of tiles A and B; 8-11: conversion; 12: the tensor core; 13-15 idle
constexpr int kPfSub = kPfRows * 128;        // bytes of 128 rows of 64 half-precision numbers
constexpr int kPfSms = 148;
constexpr int kPfNeedsScratch = -5;  // the answer to a call without scratch that cannot do without
constexpr int kPfLeast = 4;          // key tiles that a run has at least, on average
constexpr int kPfSlots = 400;        // partial results at once (see pf_plan)
constexpr float kPfSlack = 8.f;      // how far scores may outgrow R, in units of log2

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

struct PfShared {
  uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], x_full[4];
  uint64_t s_full[2], p_ready[2], pv_done[2], last;
  uint32_t tmem_base;
  int abort;
  // Of the key tiles in flight, by step % 4: factors of scores, addends, factors of the denominator's terms, and the step (+ 1)
  // that last had NaN among its values. x_full: all of them are there. (A step's place is written again four steps on, when
  // the scores of the step two on are done, which both tiles' softmax has let begin behind its last look at this step.)
  float k_scale[4][8], v_add[4][8], v_back[4][8];
  int v_nan[4];
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
__device__ __forceinline__ uint64_t pf_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
// (y0, y1) = (x0, x1) * b + c, one rounding each
__device__ __forceinline__ void pf_fma2(float& y0, float& y1, float x0, float x1, uint64_t b, uint64_t c) {
  uint64_t y;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(y) : "l"(pf_pair(x0, x1)), "l"(b), "l"(c));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y0), "=f"(y1) : "l"(y));
}
__device__ __forceinline__ void pf_add2(uint64_t& acc, float x0, float x1) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(pf_pair(x0, x1)));
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
// Key tiles of a sequence's tile of tokens [t0, t0 + n): from `lo` on, `count` of them.
__device__ __forceinline__ void pf_tiles(int start, int t0, int n, int window, int& lo, int& count) {
  lo = first_visible_key(start + t0, window) / kPfKeys;
  count = (start + t0 + n - 1) / kPfKeys - lo + 1;
}
// Tiles of tokens of a sequence, and the key tiles of its first and last one.
__device__ __forceinline__ void pf_sequence(const PrefillArgs& a, int s, int tok, int& tiles, int& first, int& last) {
  const int len = a.cu_q[s + 1] - a.cu_q[s], start = a.seq_start[s];
  tiles = (len + tok - 1) / tok;
  first = last = 0;
  if (tiles > 0) {
    int lo;
    pf_tiles(start, 0, min(tok, len), a.window, lo, first);
    pf_tiles(start, (tiles - 1) * tok, len - (tiles - 1) * tok, a.window, lo, last);
  }
}
// Key tiles that a run has on average: a 148th of the step (first and last tile of tokens stand for all of a sequence).
// All lanes of a warp call it.
__device__ __forceinline__ int pf_run(const PrefillArgs& a, int tok) {
  const int lane = threadIdx.x & 31;
  long long twice = 0;
  for (int s = lane; s < a.n_seqs; s += 32) {
    int n, f, l;
    pf_sequence(a, s, tok, n, f, l);
    twice += (long long)n * (f + l);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) twice += __shfl_xor_sync(0xffffffffu, twice, o);
  const long long c = (twice * a.n_kv + 2 * kPfSms - 1) / (2 * kPfSms);
  return (int)(c < kPfLeast ? kPfLeast : c > (1 << 28) ? (1 << 28) : c);
}
// Runs that each of a sequence's tiles of tokens is cut into. A sequence that is cut has last >= 1.5 run, so that runs <= 4/3
// last / run; and last <= 2 (first + last) / 2: all cut sequences together have at most 8/3 * 148 < kPfSlots runs.
__device__ __forceinline__ int pf_runs(int last, int run) { return max(1, (int)(((long long)last + run / 2) / run)); }

struct PfWork {
  int seq, tile, hk, part, parts, slot;          // slot: of the partial result
};
// The piece of work of block `index`; false if there is none. All lanes of a warp call it. Late tiles of a sequence, which see
// the most keys, come first, all heads of one after another.
__device__ __forceinline__ bool pf_find(const PrefillArgs& a, int tok, long long index, PfWork& w) {
  const int lane = threadIdx.x & 31;
  const int run = pf_run(a, tok);
  long long before = 0, slots = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    int n = 0, f = 0, l = 0, parts = 1;
    if (s0 + lane < a.n_seqs) {
      pf_sequence(a, s0 + lane, tok, n, f, l);
      parts = pf_runs(l, run);
    }
    const long long own = (long long)n * parts * a.n_kv, cut = parts > 1 ? own : 0;
    long long incl = own, cuts = cut;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o), y = __shfl_up_sync(0xffffffffu, cuts, o);
      if (lane >= o) {
        incl += x;
        cuts += y;
      }
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + incl > index);
    if (here) {
      const int src = __ffs(here) - 1;
      const int local = (int)(index - before - __shfl_sync(0xffffffffu, incl - own, src));
      n = __shfl_sync(0xffffffffu, n, src);
      w.parts = __shfl_sync(0xffffffffu, parts, src);
      w.slot = (int)(slots + __shfl_sync(0xffffffffu, cuts - cut, src)) + local;
      w.seq = s0 + src;
      w.part = local % w.parts;
      w.hk = local / w.parts % a.n_kv;
      w.tile = n - 1 - local / w.parts / a.n_kv;
      return true;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
    slots += __shfl_sync(0xffffffffu, cuts, 31);
  }
  return false;
}

// ------------------------------------------------------------------------------------------ the kernel
template <int HD>
__global__ void __launch_bounds__(kPfThreads, 1) prefill_fp8_kernel(const PrefillArgs a) {
  using Cfg = PfCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PfShared sh;
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_smem = base;
  uint8_t* k_smem = q_smem + 2 * Cfg::kQBytes;
  uint8_t* v_smem = k_smem + Cfg::kStages * Cfg::kKvBytes;
  const int warp = threadIdx.x >> 5;
  pdl_launch_dependents();
  pdl_wait();

  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = 2 * tok_x;      // tokens of a tile, of a block
  PfWork w;
  if (!pf_find(a, tok, blockIdx.x, w)) return;               // the whole block alike
  const int q_begin = a.cu_q[w.seq], q_len = a.cu_q[w.seq + 1] - q_begin, start = a.seq_start[w.seq];
  const int t0 = w.tile * tok, n_tok = min(tok, q_len - t0);
  int lo_tile, tiles;
  pf_tiles(start, t0, n_tok, a.window, lo_tile, tiles);
  // this run's key tiles: [c0, c1) of the tiles of the block's tokens
  const int c0 = lo_tile + (int)((long long)tiles * w.part / w.parts), c1 = lo_tile + (int)((long long)tiles * (w.part + 1) / w.parts);
  const int last_key = min(start + t0 + n_tok, a.max_pages * kFp8Page) - 1;
  // steps of the two tiles: A's tokens come first and may not see the last key tiles
  const int n_tok_a = min(n_tok, tok_x), n_tok_b = n_tok - n_tok_a;
  const int n_a = max(0, min(c1, (start + t0 + n_tok_a - 1) / kPfKeys + 1) - c0), n_b = n_tok_b > 0 ? c1 - c0 : 0;
  const int n_steps = max(n_a, n_b);

  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 256);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh.k_full[s], 128);
      mbar_init(&sh.k_empty[s], 1);
      mbar_init(&sh.v_full[s], 128);
      mbar_init(&sh.v_empty[s], 1);
      mbar_init(&sh.s_full[s], 1);
      mbar_init(&sh.p_ready[s], 128);
      mbar_init(&sh.pv_done[s], 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sh.x_full[i], 128);
      sh.v_nan[i] = 0;
    }
    mbar_init(&sh.last, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = sh.tmem_base;
  volatile int* abort = &sh.abort;
#define LLMIE_FAIL(code) do { if (!*abort) { *abort = 1; atomicExch(a.status, (code)); } } while (0)

  if (warp < 8) {
    // ------------------------------------------------------------------ softmax: a thread a row
    const int x = warp >> 2, r = threadIdx.x & 127;
    const int n_x = x ? n_b : n_a, first_tok = t0 + x * tok_x, n_tok_x = x ? n_tok_b : n_tok_a;
    const int rt = r / G, rh = r - rt * G;                   // token of the tile, query head of the group
    const bool there = rt < n_tok_x;
    const int qpos = start + first_tok + min(rt, max(n_tok_x - 1, 0));
    const int lo = first_visible_key(qpos, a.window);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + Cfg::kSCol + x * 128, o_addr = tmem + lanes + Cfg::kOCol + x * (HD == 64 ? 64 : 128);
    const uint32_t p_addr = Cfg::kOwnP ? tmem + lanes + Cfg::kPCol + x * 64 : s_addr;
    const int head = w.hk * G + rh;
    const size_t row_off = ((size_t)(q_begin + first_tok + rt) * a.n_q + head) * HD;
    float f;                                                 // of a score: scale log2(e) and the power of two of the row
    {
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
      const int shift = eb == 255 ? 0 : min(max(141 - eb, -100), 100);       // the largest number into [2^14, 2^15)
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
      mbar_arrive(&sh.q_full);
    }
    // a score's factor is never 0: times -inf, which stands where the row does not look, that would be NaN
    auto factor = [&](float k_scale) { return fminf(fmaxf(f * k_scale, 1.2e-38f), 3.4e38f); };
    float R = -INFINITY, l = 0.f;
    uint32_t nan_cols[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) nan_cols[i] = 0u;
    bool ok = true;
    // the first and last keys that every row of the tile sees
    const int all_to = start + first_tok, all_from = first_visible_key(start + first_tok + max(n_tok_x - 1, 0), a.window);
    for (int j = 0; j < n_x; ++j) {
      // every decision to give up is taken by the whole warp: reads of tensor memory are warp-wide instructions
      if (!__all_sync(0xffffffffu, mbar_wait(&sh.x_full[j & 3], (j >> 2) & 1, abort) && mbar_wait(&sh.s_full[x], j & 1, abort))) {
        LLMIE_FAIL(kStatusTimeoutMma);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const int kbase = (c0 + j) * kPfKeys, ring = j & 3;
      const bool edge = kbase + kPfKeys - 1 > all_to || kbase < all_from;
      // pass 1: the largest s + ev of the row; scores that the row does not see become -inf, in tensor memory too
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_ld_32x32(s_addr + c * 32, v);
        tmem_ld_wait();
        if (edge) {
          const int from = lo - kbase - c * 32;
          const unsigned span = (unsigned)(qpos - lo);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((unsigned)(i - from) > span) v[i] = 0xff800000u;
          tmem_st_32x32(s_addr + c * 32, v);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            m0 = fmaxf(m0, __uint_as_float(v[b * 16 + i]));
            m1 = fmaxf(m1, __uint_as_float(v[b * 16 + i + 1]));
          }
          mx = fmaxf(mx, fmaf(fmaxf(m0, m1), factor(sh.k_scale[ring][c * 2 + b]), sh.v_add[ring][c * 2 + b]));
        }
      }
      if (edge) tmem_st_wait();
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
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t v[32];
          tmem_ld_32x32(o_addr + c * 32, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
          tmem_st_32x32(o_addr + c * 32, v);
        }
        tmem_st_wait();
      }
      if (grow) R = mx;
      const float shift = (R == -INFINITY ? 0.f : R) - 7.f;
      // pass 2: the weights
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32], o[16];
        tmem_ld_32x32(s_addr + c * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float fk = factor(sh.k_scale[ring][c * 2 + b]), add = sh.v_add[ring][c * 2 + b] - shift;
          const uint64_t fk2 = pf_pair(fk, fk), add2 = pf_pair(add, add);
          uint64_t sum0 = 0ull, sum1 = 0ull;
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x0, x1;
            pf_fma2(x0, x1, __uint_as_float(v[b * 16 + i]), __uint_as_float(v[b * 16 + i + 1]), fk2, add2);
            x0 = pf_exp2(x0);
            x1 = pf_exp2(x1);
            if (i & 2) pf_add2(sum1, x0, x1);
            else pf_add2(sum0, x0, x1);
            o[b * 8 + i / 2] = pf_half2(x0, x1);
          }
          asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum0) : "l"(sum1));
          float y0, y1;
          asm("mov.b64 {%0, %1}, %2;" : "=f"(y0), "=f"(y1) : "l"(sum0));
          l = fmaf(y0 + y1, sh.v_back[ring][c * 2 + b], l);
        }
        if (Cfg::kOwnP && c == 0 && j > 0) {
          // the weights of the tile before have to be through the product before they are written over
          if (!__all_sync(0xffffffffu, mbar_wait(&sh.pv_done[x], (j - 1) & 1, abort))) {
            LLMIE_FAIL(kStatusTimeoutMma);
            ok = false;
            break;
          }
          tc_fence_after_sync();
        }
        pf_tmem_st16(p_addr + c * 16, o);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before_sync();
      mbar_arrive(&sh.p_ready[x]);
      if (sh.v_nan[ring] == j + 1) {
        // rare: which columns of the values that this row sees are NaN
        const int* pages = a.block_table + (size_t)a.seq_slot[w.seq] * a.max_pages;
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
    // ---- the row's result: the output, or a partial one. Where a wait gave up: NaN.
    float* rec = a.part + (size_t)w.slot * Cfg::kRecord;
    const int pr = x * kPfRows + r;
    if (w.parts > 1 && there) {
      rec[2 * kPfRows * HD + pr] = R;
      rec[2 * kPfRows * (HD + 1) + pr] = ok ? l : __int_as_float(0x7fffffff);
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t v[32];
      if (ok && n_x > 0) {
        tmem_ld_32x32(o_addr + c * 32, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0u;
      }
      if (!there) continue;
      float y[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) y[i] = (nan_cols[c] >> i & 1u) || !ok ? __int_as_float(0x7fffffff) : __uint_as_float(v[i]);
      if (w.parts > 1) {
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          *reinterpret_cast<float4*>(rec + (size_t)pr * HD + c * 32 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float v8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v8[e] = y[i + e] * inv;
          store8(a.out + row_off + c * 32 + i, v8);
        }
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------------ conversion: 128 threads, 16 codes at a time
    constexpr int kPer = HD / 16;                            // pieces of 16 codes a row, and pieces a thread
    const int ct = threadIdx.x - 256;
    const int piece = ct % kPer, row0 = ct / kPer;           // rows row0, row0 + 128 / kPer, ...
    constexpr int kStep = 128 / kPer;
    const int* pages = a.block_table + (size_t)a.seq_slot[w.seq] * a.max_pages;
    const int last_page = last_key / kFp8Page;
    uint4 kr[kPer], vr[kPer];
    auto page_row = [&](int tile, int half) -> size_t {      // (page, head) of a half of a key tile
      const int lp = tile * 2 + half;
      return (size_t)(lp <= last_page ? pages[lp] : 0) * a.n_kv + w.hk;
    };
    auto load = [&](uint4 (&reg)[kPer], const unsigned char* cache, int tile) {
      const size_t p0 = page_row(tile, 0), p1 = page_row(tile, 1);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int row = row0 + i * kStep;
        reg[i] = make_uint4(0u, 0u, 0u, 0u);                 // rows behind the block's last key: nothing that may be NaN
        if (tile * kPfKeys + row <= last_key)
          reg[i] = *reinterpret_cast<const uint4*>(cache + ((row < 64 ? p0 : p1) * kFp8Page + (row & 63)) * HD + piece * 16);
      }
    };
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
    load(kr, a.k, c0);
    load(vr, a.v, c0);
    bool ok = true;
    for (int j = 0; ok && j < n_steps; ++j) {
      const int st = j & 1, ring = j & 3;
      if (j >= 2 && !mbar_wait(&sh.k_empty[st], ((j >> 1) - 1) & 1, abort)) {
        LLMIE_FAIL(kStatusTimeoutEmpty);
        break;
      }
      if (ct < 8) {
        // the exponents of the tile's eight blocks (a block behind the last key: anything, nobody sees its scores)
        const size_t pr = page_row(c0 + j, ct >> 2);
        const int ke = clamp_exponent(a.k_exp[pr * kPageExps + (ct & 3)]), ve = clamp_exponent(a.v_exp[pr * kPageExps + (ct & 3)]);
        sh.k_scale[ring][ct] = pow2_of(ke);
        sh.v_add[ring][ct] = (float)ve;
        sh.v_back[ring][ct] = pow2_of(-ve);
      }
      // NaN among the values: such codes become zeros here
      unsigned any = 0u;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        any |= ((vr[i].x & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].y & 0x7f7f7f7fu) + 0x01010101u) |
               ((vr[i].z & 0x7f7f7f7fu) + 0x01010101u) | ((vr[i].w & 0x7f7f7f7fu) + 0x01010101u);
      put(k_smem + st * Cfg::kKvBytes, kr);
      if (j + 1 < n_steps) load(kr, a.k, c0 + j + 1);
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
      fence_proxy_async_smem();
      mbar_arrive(&sh.v_full[st]);
    }
  } else if (warp == 12) {
    // ------------------------------------------------------------------ the tensor core
    if (elect_one()) {
      constexpr uint32_t idesc_s = pf_instr_desc(kPfRows, kPfKeys, 0), idesc_o = pf_instr_desc(kPfRows, HD, 1);
      bool ok = mbar_wait(&sh.q_full, 0, abort);
      if (!ok) LLMIE_FAIL(kStatusTimeoutFull);
      auto scores = [&](int x, int j) {                      // S = Q K^T of tile x, step j (its keys are there)
        const uint32_t qa = smem_u32(q_smem + x * Cfg::kQBytes), ka = smem_u32(k_smem + (j & 1) * Cfg::kKvBytes);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kPfSub + (kk & 3) * 32;
          mma_bf16_ss(tmem + Cfg::kSCol + x * 128, make_smem_desc(qa + off, 16, 1024), make_smem_desc(ka + off, 16, 1024), idesc_s,
                      kk > 0 ? 1u : 0u);
        }
        mma_commit(&sh.s_full[x]);
      };
      auto keys = [&](int j) -> bool {
        if (mbar_wait(&sh.k_full[j & 1], (j >> 1) & 1, abort)) return true;
        LLMIE_FAIL(kStatusTimeoutFull);
        return false;
      };
      if (ok && n_steps > 0 && (ok = keys(0))) {
        tc_fence_after_sync();
        if (n_a > 0) scores(0, 0);
        if (n_b > 0) scores(1, 0);
        mma_commit(&sh.k_empty[0]);
      }
      for (int j = 0; ok && j < n_steps; ++j) {
        if (!mbar_wait(&sh.v_full[j & 1], (j >> 1) & 1, abort)) {
          LLMIE_FAIL(kStatusTimeoutFull);
          break;
        }
        const uint32_t va = smem_u32(v_smem + (j & 1) * Cfg::kKvBytes);
        for (int x = 0; ok && x < 2; ++x) {
          const int n_x = x ? n_b : n_a;
          if (j < n_x) {
            if (!mbar_wait(&sh.p_ready[x], j & 1, abort)) {
              LLMIE_FAIL(kStatusTimeoutMma);
              ok = false;
              break;
            }
            tc_fence_after_sync();
            // where the weights have columns of their own the next scores may be written at once
            if (Cfg::kOwnP && j + 1 < n_x) {
              if (!(ok = keys(j + 1))) break;
              tc_fence_after_sync();
              scores(x, j + 1);
            }
            const uint32_t pa = tmem + (Cfg::kOwnP ? Cfg::kPCol + x * 64 : Cfg::kSCol + x * 128);
            const uint32_t od = tmem + Cfg::kOCol + x * (HD == 64 ? 64 : 128);
#pragma unroll
            for (int kk = 0; kk < kPfKeys / 16; ++kk)        // 16 weights are 8 columns; 16 keys are 16 rows of the values
              pf_mma_ts(od, pa + kk * 8, make_smem_desc(va + kk * 2048, kPfSub, 1024), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
            mma_commit(&sh.pv_done[x]);
            if (!Cfg::kOwnP && j + 1 < n_x) {
              // the next scores are written where these weights are read from
              if (!mbar_wait(&sh.pv_done[x], j & 1, abort)) {
                LLMIE_FAIL(kStatusTimeoutMma);
                ok = false;
                break;
              }
              if (!(ok = keys(j + 1))) break;
              tc_fence_after_sync();
              scores(x, j + 1);
            }
          }
        }
        if (!ok) break;
        mma_commit(&sh.v_empty[j & 1]);
        if (j + 1 < n_steps) mma_commit(&sh.k_empty[(j + 1) & 1]);
      }
      // nothing may be in flight when the tensor memory is given back
      mma_commit(&sh.last);
      for (unsigned spin = 0; spin < (1u << 20) && !mbar_test(&sh.last, 0); ++spin) __nanosleep(32);
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

// Joins the runs of the tiles that were cut: a warp a (token, query head). grid (tokens, ceil(n_q / 4)).
template <int HD> __global__ void __launch_bounds__(128) prefill_fp8_join_kernel(const PrefillArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  using Cfg = PfCfg<HD>;
  const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), t = blockIdx.x;
  if (head >= a.n_q) return;
  const int G = a.n_q / a.n_kv, tok_x = kPfRows / G, tok = 2 * tok_x, hk = head / G;
  const int run = pf_run(a, tok);
  long long slots = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
    int n = 0, f = 0, l = 0, parts = 1, q0 = 0, q1 = 0;
    if (s0 + lane < a.n_seqs) {
      pf_sequence(a, s0 + lane, tok, n, f, l);
      parts = pf_runs(l, run);
      q0 = a.cu_q[s0 + lane];
      q1 = a.cu_q[s0 + lane + 1];
    }
    const long long cut = parts > 1 ? (long long)n * parts * a.n_kv : 0;
    long long cuts = cut;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, cuts, o);
      if (lane >= o) cuts += y;
    }
    const unsigned here = __ballot_sync(0xffffffffu, t >= q0 && t < q1);
    if (!here) {
      slots += __shfl_sync(0xffffffffu, cuts, 31);
      continue;
    }
    const int src = __ffs(here) - 1;
    parts = __shfl_sync(0xffffffffu, parts, src);
    if (parts == 1) return;
    n = __shfl_sync(0xffffffffu, n, src);
    const int place = t - __shfl_sync(0xffffffffu, q0, src), tile = place / tok, in = place - tile * tok;
    const int row = in / tok_x * kPfRows + in % tok_x * G + head % G;
    const long long slot = slots + __shfl_sync(0xffffffffu, cuts - cut, src) + ((long long)(n - 1 - tile) * a.n_kv + hk) * parts;
    const float* rec = a.part + slot * Cfg::kRecord;
    float M = -INFINITY;
    for (int p = lane; p < parts; p += 32) M = fmaxf(M, __ldcg(rec + (size_t)p * Cfg::kRecord + 2 * kPfRows * HD + row));
    M = warp_max(M);
    const float Mu = M == -INFINITY ? 0.f : M;
    float num[HD / 32], den = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) num[i] = 0.f;
    for (int p0 = 0; p0 < parts; p0 += 32) {
      float fac = 0.f;
      if (p0 + lane < parts) {
        const float* r = rec + (size_t)(p0 + lane) * Cfg::kRecord;
        fac = pf_exp2(__ldcg(r + 2 * kPfRows * HD + row) - Mu);
        den = fmaf(fac, __ldcg(r + 2 * kPfRows * (HD + 1) + row), den);
      }
      const int m = min(32, parts - p0);
      for (int p = 0; p < m; ++p) {
        const float g = __shfl_sync(0xffffffffu, fac, p);
        const float* r = rec + (size_t)(p0 + p) * Cfg::kRecord + (size_t)row * HD;
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) num[i] = fmaf(g, __ldcg(r + lane + 32 * i), num[i]);
      }
    }
    den = warp_sum(den);
    __nv_bfloat16* o = a.out + ((size_t)t * a.n_q + head) * HD;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) o[lane + 32 * i] = __float2bfloat16_rn(num[i] / den);
    return;
  }
}

template <int HD>
static int launch_prefill_fp8(const PrefillArgs& a, int n_tokens, cudaStream_t stream) {
  using Cfg = PfCfg<HD>;
  cudaError_t e = cudaFuncSetAttribute(prefill_fp8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem);
  if (e != cudaSuccess) return (int)e;
  const int tok = 2 * (kPfRows / (a.n_q / a.n_kv));
  // Pieces of work: the tiles of tokens, and the runs that they may be cut into. The most runs that a tile can have follow from
  // the most keys that the table has room for and the least work that so many tokens are.
  const long long items = ((long long)n_tokens / tok + a.n_seqs) * a.n_kv;
  double least = (double)n_tokens / tok * a.n_kv;
  long long most_tiles = ((long long)a.max_pages * kFp8Page + kPfKeys - 1) / kPfKeys;
  if (a.window == 0) {
    least *= (1.0 + (double)n_tokens / ((double)kPfKeys * a.n_seqs)) / 2;
  } else {
    const long long w = a.window < 0 ? -(long long)a.window : a.window;
    most_tiles = min(most_tiles, (w + tok) / kPfKeys + 2);
  }
  long long run = (long long)(least / kPfSms);
  if (run < kPfLeast) run = kPfLeast;
  const long long parts = (most_tiles + run / 2) / run;
  const bool cut = parts > 1;
  if (cut && !a.part) return kPfNeedsScratch;
  const long long blocks = cut ? min(items * parts, items + kPfSlots) : items;
  if (blocks > 0x7fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  launch_k(prefill_fp8_kernel<HD>, dim3((unsigned)blocks), dim3(kPfThreads), Cfg::kSmem, stream, a);
  LLMIE_LAUNCH_CHECK();
  if (cut) {
    launch_k(prefill_fp8_join_kernel<HD>, dim3(n_tokens, (a.n_q + 3) / 4), dim3(128), 0, stream, a);
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
// held before this step, whose keys are in the cache already. scale > 0. window: as in the other attention kernels.
// scratch: llmie_attention_prefill_fp8_scratch floats, 16-byte aligned; null: a call that needs it launches nothing and returns -5.
extern "C" int llmie_attention_prefill_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_exp,
                                           const void* v_exp, void* out, float* scratch, int* status, const int* cu_q,
                                           const int* seq_slot, const int* seq_start, const int* block_table, int max_pages,
                                           int n_tokens, int n_seqs, int n_q, int n_kv, int hd, float scale, int window,
                                           cudaStream_t stream) {
  if (n_tokens < 0 || n_seqs < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0 || !status) return LLMIE_ERR_BAD_ARG;
  if (!(scale > 0.f)) return LLMIE_ERR_BAD_ARG;              // a row's bound is taken before scores are scaled
  if ((hd != 64 && hd != 128) || n_q / n_kv > kPfRows || (n_q + 3) / 4 > 65535) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(scratch)) return LLMIE_ERR_ALIGNMENT;
  if (n_tokens == 0 || n_seqs == 0) return LLMIE_OK;
  const PrefillArgs a{(const __nv_bfloat16*)q, (const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp,
                      (const signed char*)v_exp, (__nv_bfloat16*)out, scratch, status, cu_q, seq_slot, seq_start, block_table,
                      max_pages, n_seqs, n_q, n_kv, scale * 1.4426950408889634f, window};
  return hd == 64 ? launch_prefill_fp8<64>(a, n_tokens, stream) : launch_prefill_fp8<128>(a, n_tokens, stream);
}
