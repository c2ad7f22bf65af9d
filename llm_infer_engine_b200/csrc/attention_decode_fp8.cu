// Attention of one token a sequence over a paged cache in 8 bits (fp8.cuh), on the tensor cores.
//
//   o = sum_j 2^(s_j) c_j 2^(ev_j) / sum_j 2^(s_j),     s_j = scale log2(e) (q . k_j) 2^(ek_j)      (k, c: codes of keys, values)
//
// A warp works on 32 positions of a KV head at a time, which are two blocks of the cache: a block's keys have one exponent, its
// values another. A value's exponent is added to the score, so that one exponential gives the weight that its codes get:
// with R a running bound, w_j = 2^(s_j + ev_j - R + 7) goes into the second product in half precision, and the softmax's
// denominator is sum_j w_j 2^(-ev_j), kept in float32 relative to the same R. R follows the largest s_j + ev_j only when that
// has outgrown it by 8, so that w_j stays below 2^15 (half precision then holds what is within 2^-21 of the largest weight with
// 11 digits) and the sums have to be rescaled a few times in a sequence, not with every block.
//
// Both products are mma.sync.m16n8k16 with the cache as the 16-row operand and the query heads of the KV head as the 8
// columns: S^T = K Q^T and O^T = V^T W^T. Codes become half-precision numbers (exactly) in registers, and which k
// index stands for which column of a head is free as long as both operands agree: a lane reads 16 neighbouring codes of a key
// (and 8 or 16 of a value), whole sectors every time, through a ring of asynchronous copies of its own.
// W^T comes out of S^T's accumulators by one 8x8 transpose between lanes (movmatrix). Queries are brought to half precision
// with a power of two per head (their largest number in [2^14, 2^15)), which keeps every digit of bfloat16 (of what is above 2^-31 of the
// head's largest number; the rest is off by 2^-39 of that at most).
//
// Work is cut by blocks of positions, not by sequences: all (sequence, KV head) items one after another make one line of
// units, and every thread block takes an equal share of it, wherever it begins and ends. Lengths are read on the device, so
// a captured step costs what its sequences hold. An item that lies in several shares leaves partial results, and a second
// small kernel joins them in the order of the shares: no atomics, no counters, nothing kept between calls.
#include "fp8.cuh"
#include "tcgen05.cuh"
#include <math.h>

namespace llmie {

constexpr int kDfWarps = 4;          // of a block (of a large one, where an item has its blocks to itself: twice as many)
constexpr int kDfUnit = 2 * kExpBlock;
constexpr int kDfThreads = kDfWarps * 32;
constexpr int kSms = 148;
constexpr int kNeedsScratch = -5;    // the answer to a call without scratch that cannot do without
constexpr float kDfSlack = 8.f;      // how far scores may outgrow a head's bound, in units of log2
constexpr float kDfTop = 7.f;        // the bound's own weight is 2^7: none is above 2^15
constexpr int kDfFew = 12;           // units a warp up to which an item is one cluster's

__device__ __forceinline__ float df_exp2(float x) { return exp2_ftz(x); }
__device__ __forceinline__ void df_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned df_transpose(unsigned v) {
  unsigned r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ unsigned df_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const unsigned*>(&h);
}
__device__ __forceinline__ unsigned df_lo(unsigned w) { return e4m3x2_to_half2((unsigned short)(w & 0xffffu)); }
__device__ __forceinline__ unsigned df_hi(unsigned w) { return e4m3x2_to_half2((unsigned short)(w >> 16)); }
// What is beyond float32 as its largest number (NaN stays): infinity times a product that is zero would be NaN.
__device__ __forceinline__ float df_finite(float x) {
  float y;
  asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, 0f7f7fffff;\n\tmax.NaN.f32 %0, t, 0fff7fffff;\n\t}" : "=f"(y) : "f"(x));
  return y;
}
struct DecodeArgs {
  const unsigned char* k;            // [pages, n_kv, 64, HD] codes
  const unsigned char* v;
  const signed char* k_exp;          // [pages, n_kv, 4]
  const signed char* v_exp;
  __nv_bfloat16* out;                // [n_seqs, n_q HD]
  float* part;                       // partial results, two a thread block
  const int* seq_slot;
  const int* seq_kvlen;
  const int* block_table;
  int max_pages, n_seqs, n_q, n_kv;
  float scale2;                      // scale * log2(e)
  int window;
};

// Units of 32 positions (two blocks of the cache) in which a sequence's newest token sees some: [first, first + count).
__device__ __forceinline__ void df_units(const DecodeArgs& a, int len, int& first, int& count) {
  len = min(len, a.max_pages * kFp8Page);              // what the table has room for
  if (len <= 0) {
    first = count = 0;
    return;
  }
  first = first_visible_key(len - 1, a.window) / kDfUnit;
  count = (len - 1) / kDfUnit - first + 1;
}

// Units of all sequences together (every item of a sequence has as many as the sequence). All lanes of a warp call it.
__device__ __forceinline__ int df_total(const DecodeArgs& a) {
  const int lane = threadIdx.x & 31;
  int t = 0;
#pragma unroll 1
  for (int s = lane; s < a.n_seqs; s += 32) {
    int f, c;
    df_units(a, a.seq_kvlen[s], f, c);
    t += c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

// Units that a thread block takes: an equal share, and four at least (one a warp).
__device__ __forceinline__ int df_share(int total_units, int blocks) {
  const int s = (total_units + blocks - 1) / blocks;
  return s < kDfWarps ? kDfWarps : s;
}

template <int HD, int NH> struct DfCfg {
  static constexpr int kHeads = 8 * NH;
  static constexpr int kPitch = HD + 4;                          // floats between two heads' sums: lanes 4 banks apart
  static constexpr int kRecord = kHeads * (HD + 2);              // floats of a partial result: sums, then bounds and denominators
};
// Thread blocks that an SM holds at once. (Head size 64, five instead of four, 102 registers a thread: 64 sequences of 700 to 3,900 keys
// 34.9 us where four took 29.3; one of 517 4.75 and 4.4. Head size 128, two instead of three: 48 of 1,000 to 16,000 100 and 92.5, with a
// third stage 94. The looks at small denominators came later: 30.0 and 93.1 now.)
template <int HD, int NH> __host__ __device__ constexpr int df_per_sm() { return HD == 64 ? (NH == 1 ? 4 : 3) : NH == 1 ? 3 : 2; }
template <int HD, int NH> __host__ __device__ constexpr int df_large_per_sm() { return HD == 64 && NH == 1 ? 2 : 1; }
template <int HD, int NH> constexpr int df_blocks() { return kSms * df_per_sm<HD, NH>(); }
// Where column d of a head stands among a head's sums: as the second product's accumulators hold them.
template <int HD> __device__ __forceinline__ int df_place(int d) {
  constexpr int R = HD / 8;
  return (d % R / 2) * 16 + (d & 1) * 8 + d / R;
}

// A step's projections as they come, [n_seqs, (n_q + 2 n_kv) HD], and what the new key and value need (rope == null: q is
// rotated already, and the cache holds the step's keys and values).
struct DecodeStep {
  const float4* rope;                // (cos, sin) [table_len, HD / 2]
  int table_len;
  unsigned char* k;                  // the cache, to be written
  unsigned char* v;
  signed char* k_exp;
  signed char* v_exp;
};

// Writes position len - 1 of (sequence, KV head) into its block: rotated key and value, the block's exponents, the earlier codes
// lowered where an exponent rises (cache_fp8.cu has the rules; the numbers are the same bit for bit). One warp; what it wrote
// is there for the whole warp when it returns.
template <int HD>
__device__ __forceinline__ void df_append(const __nv_bfloat16* qkv_row, const DecodeArgs& a, const DecodeStep& st, int hk, int len, int page) {
  const int lane = threadIdx.x & 31;
  const int pos = len - 1, in = pos % kExpBlock;
  const size_t head = (size_t)page * a.n_kv + hk;
  const size_t at = head * kPageExps + pos % kFp8Page / kExpBlock;
  const size_t row = (head * kFp8Page + pos % kFp8Page) * HD;
  constexpr int kN = HD / 64;        // neighbouring columns a lane has in each half of the head
  const int d = lane * kN;
  const float2* cs = reinterpret_cast<const float2*>(st.rope) + (size_t)min(pos, st.table_len - 1) * (HD / 2) + d;
  const __nv_bfloat16* kp = qkv_row + (size_t)(a.n_q + hk) * HD + d;
  const __nv_bfloat16* vp = kp + (size_t)a.n_kv * HD;
  float x[2][2][kN];
  unsigned big[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const float2 c = cs[i];
    const float k0 = __bfloat162float(kp[i]), k1 = __bfloat162float(kp[i + HD / 2]);
    x[0][0][i] = __fsub_rn(__fmul_rn(k0, c.x), __fmul_rn(k1, c.y));
    x[0][1][i] = __fadd_rn(__fmul_rn(k1, c.x), __fmul_rn(k0, c.y));
    x[1][0][i] = __bfloat162float(vp[i]);
    x[1][1][i] = __bfloat162float(vp[i + HD / 2]);
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
#pragma unroll
    for (int i = 0; i < kN; ++i) big[w] = max(big[w], max(finite_magnitude(x[w][0][i]), finite_magnitude(x[w][1][i])));
    big[w] = __reduce_max_sync(0xffffffffu, big[w]);
    signed char* exp_at = (w ? st.v_exp : st.k_exp) + at;
    unsigned char* codes = (w ? st.v : st.k) + row;
    int e = exponent_for(big[w]);
    if (in > 0) {
      const int before = clamp_exponent(*exp_at);
      e = max(e, before);
      if (e > before) {
        const float f = lower_factor(before, e);
        unsigned* old = reinterpret_cast<unsigned*>(codes - (size_t)in * HD);
#pragma unroll 1
        for (int i = lane; i < in * HD / 4; i += 32) old[i] = lower_codes(old[i], f);
      }
    }
    const float f = pow2_of(-e);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (kN == 2) {
        *reinterpret_cast<unsigned short*>(codes + d + h * (HD / 2)) = to_e4m3x2(x[w][h][0] * f, x[w][h][kN - 1] * f);
      } else {
        codes[d + h * (HD / 2)] = (unsigned char)(to_e4m3x2(x[w][h][0] * f, 0.f) & 0xffu);
      }
    }
    __syncwarp();                    // every lane has read the old exponent
    if (lane == 0) *exp_at = (signed char)e;
  }
  __syncwarp();
}

// A warp's pipeline of units: a ring of stages in shared memory, filled by asynchronous copies of whole lines. A unit's keys are one
// run of memory, its values another; 16-byte pieces lie in lines of 128 bytes, their places in a line permuted so that no two
// lanes of a quarter warp meet in a bank when the fragments are read: keys by 4 neighbouring pieces of 2 rows, values by one piece
// of 4 rows 2 apart. Fragments: lane (g, t) reads, of keys g, g + 8, g + 16 and g + 24, 16 codes from column 16 t on of every
// 64; of the values of positions 2t, 2t + 1, 2t + 8, 2t + 9 and those 16 on, HD / 8 codes from column g HD / 8 on.
// (Lanes that copied what they read themselves, 64 bytes of a line at a time, needed no barrier but reached 64 % of the copy
// bandwidth at head size 128 with the arithmetic left out.)
template <int HD> __device__ __forceinline__ int df_swizzle(int line) {
  return HD == 64 ? (line & 3) << 1 : ((line >> 1 & 3) << 1) ^ ((line & 1) << 2);
}
// byte offset of piece p of row r in a unit
template <int HD> __device__ __forceinline__ int df_at(int r, int p) {
  const int l = r * (HD / 16) + p, line = l >> 3;
  return line * 128 + ((l & 7) ^ df_swizzle<HD>(line)) * 16;
}
template <int HD, int NH, int W = kDfWarps> struct DfPipe {
  static constexpr int kStages = 2;
  static constexpr int kHalf = kDfUnit * HD;                 // bytes of a unit's keys, or values
  static constexpr int kUnit = 2 * kHalf + 128;              // and the exponents; whole lines

  static constexpr int kWarp = kStages * kUnit;
  static constexpr int kSums = DfCfg<HD, NH>::kHeads * (DfCfg<HD, NH>::kPitch + 2) * 4;        // a warp's results, in the same place afterwards
  static constexpr int kPerWarp = ((kWarp > kSums ? kWarp : kSums) + 127) / 128 * 128;
  static constexpr int kSmem = W * kPerWarp;
};
__device__ __forceinline__ void df_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void df_copy4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// A piece of an item: units [u_begin, u_end) of the `count` that sequence seq's newest token sees (unit 0 of them is `first`),
// KV head hk, ng query heads from g0 of its group on. All warps of the block; each leaves its sums (df_place), bounds and
// denominators in its own part of shared memory: [heads][pitch], [heads], [heads] floats.
template <int HD, int NH, bool ROPE, int W>
__device__ __forceinline__ void df_piece(const __nv_bfloat16* q, const DecodeArgs& a, const DecodeStep& st, unsigned char* smem, int seq,
                                         int len, int hk, int g0, int ng, int first, int count, int u_begin, int u_end) {
  using Cfg = DfCfg<HD, NH>;
  using Pipe = DfPipe<HD, NH>;
  constexpr int KS = HD / 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = a.n_q / a.n_kv;
  const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.max_pages;
  const int lo = first_visible_key(len - 1, a.window);
  unsigned char* mine = smem + warp * Pipe::kPerWarp;
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(mine);

  int u = first + u_begin + warp;
  const int u_stop = first + u_end;
  auto page_of = [&](int v) { return v < u_stop ? pages[v >> 1] : 0; };
  auto issue = [&](int v, int page, int stage) {
    if (v < u_stop) {
      const size_t row = (size_t)page * a.n_kv + hk;
      const size_t off = (row * kFp8Page + (v & 1) * kDfUnit) * HD + lane * 16;
      const uint32_t dst = ring + stage * Pipe::kUnit;
#pragma unroll
      for (int i = 0; i < Pipe::kHalf / 512; ++i) {
        const int line = i * 4 + (lane >> 3), to = line * 128 + ((lane & 7) ^ df_swizzle<HD>(line)) * 16;
        df_copy16(dst + to, a.k + off + i * 512);
        df_copy16(dst + Pipe::kHalf + to, a.v + off + i * 512);
      }
      if (lane < 2) df_copy4(dst + 2 * Pipe::kHalf + lane * 4, (lane ? a.v_exp : a.k_exp) + row * kPageExps);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const size_t q_pitch = (size_t)(ROPE ? a.n_q + 2 * a.n_kv : a.n_q) * HD;
  // (a sequence that is longer than its table: there is no place for the position)
  if (ROPE && u_end == count && u_begin < count && (count - 1 - u_begin) % W == warp && a.seq_kvlen[seq] == len)
    df_append<HD>(q + seq * q_pitch, a, st, hk, len, pages[(first + count - 1) >> 1]);            // this warp reads that block itself
  int pg_next;                       // page of the next unit to be asked for
  {
    int pg[Pipe::kStages];
#pragma unroll
    for (int i = 0; i < Pipe::kStages; ++i) pg[i] = page_of(u + i * W);
#pragma unroll
    for (int i = 0; i < Pipe::kStages - 1; ++i) issue(u + i * W, pg[i], i);
    pg_next = pg[Pipe::kStages - 1];
  }

  // the queries: for head g of each group of 8, columns in the order of the keys' codes
  unsigned qb[NH][KS][2];
  float q_scale[NH][2];              // of heads 2t, 2t + 1: scale log2(e) 2^(what the queries were shifted by)
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
    const bool there = nh * 8 + g < ng;
    const __nv_bfloat16* row = q + seq * q_pitch + (size_t)(hk * G + g0 + (there ? nh * 8 + g : 0)) * HD;
    uint2 raw[KS];
    float big = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int col = (ks >> 2) * 64 + t * 16 + (ks & 3) * 4;
      raw[ks] = there ? *reinterpret_cast<const uint2*>(row + col) : make_uint2(0u, 0u);
      if (ROPE) {
        // four columns and the four that they are rotated with, half a head away
        const bool upper = col >= HD / 2;
        const uint2 other = there ? *reinterpret_cast<const uint2*>(row + (upper ? col - HD / 2 : col + HD / 2)) : make_uint2(0u, 0u);
        const float4* cs = st.rope + ((size_t)min(len - 1, st.table_len - 1) * (HD / 2) + (upper ? col - HD / 2 : col)) / 2;
        const float4 c0 = cs[0], c1 = cs[1];
        auto turned = [&](unsigned x, unsigned y, const float4& c) {
          const float2 u2 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
          const float2 v2 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y));
          const float p0 = __fmul_rn(u2.x, c.x), p1 = __fmul_rn(u2.y, c.z), r0 = __fmul_rn(v2.x, c.y), r1 = __fmul_rn(v2.y, c.w);
          const __nv_bfloat162 z = upper ? __floats2bfloat162_rn(__fadd_rn(p0, r0), __fadd_rn(p1, r1))
                                         : __floats2bfloat162_rn(__fsub_rn(p0, r0), __fsub_rn(p1, r1));
          return *reinterpret_cast<const unsigned*>(&z);
        };
        raw[ks] = make_uint2(turned(raw[ks].x, other.x, c0), turned(raw[ks].y, other.y, c1));
      }
      const float2 y0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
      const float2 y1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
      big = fmaxf(big, fmaxf(fmaxf(fabsf(y0.x), fabsf(y0.y)), fmaxf(fabsf(y1.x), fabsf(y1.y))));
    }
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    // The exponent that brings the largest number into [2^14, 2^15): 141 - eb, -113 at least. (Below 2^-112 it stays lower, in [2^-7, 2^14):
    // half precision has all digits of bfloat16 there too.) A head that is not finite stays as it is.
    const int eb = (int)(__float_as_uint(big) >> 23);
    const int shift = eb == 255 ? 0 : min(141 - eb, 126);
    const float f = pow2_of(shift);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const float2 y0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].x));
      const float2 y1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[ks].y));
      qb[nh][ks][0] = df_half2(y0.x * f, y0.y * f);
      qb[nh][ks][1] = df_half2(y1.x * f, y1.y * f);
    }
    const float back = a.scale2 * pow2_of(-shift);
    q_scale[nh][0] = __shfl_sync(0xffffffffu, back, 8 * t);
    q_scale[nh][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
  }
  float o[NH][KS][4];
  float R[NH][2], l[NH][2];          // a head's bound, and this lane's share of its denominator
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
    for (int i = 0; i < KS; ++i) o[nh][i][0] = o[nh][i][1] = o[nh][i][2] = o[nh][i][3] = 0.f;
    R[nh][0] = R[nh][1] = -INFINITY;
    l[nh][0] = l[nh][1] = 0.f;
  }

  int stage = 0, ahead = Pipe::kStages - 1;                  // where this unit lies, and where the one to be asked for goes
  for (; u < u_stop; u += W) {
    asm volatile("cp.async.wait_group %0;" ::"n"(Pipe::kStages - 2) : "memory");
    __syncwarp();                    // everyone's share of the unit is there, and everyone has read the unit before
    issue(u + (Pipe::kStages - 1) * W, pg_next, ahead);
    pg_next = page_of(u + Pipe::kStages * W);
    const unsigned char* at = mine + stage * Pipe::kUnit;
    ahead = stage;
    stage = stage + 1 == Pipe::kStages ? 0 : stage + 1;
    // S^T = K Q^T, block by block
    float s[2][NH][4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) s[b][nh][0] = s[b][nh][1] = s[b][nh][2] = s[b][nh][3] = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) {
      uint4 k4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k4[i] = *reinterpret_cast<const uint4*>(at + df_at<HD>(g + 8 * i, c * 4 + t));
#pragma unroll
      for (int w = 0; w < 4; ++w) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const unsigned ka = w == 0 ? k4[2 * b].x : w == 1 ? k4[2 * b].y : w == 2 ? k4[2 * b].z : k4[2 * b].w;
          const unsigned kb = w == 0 ? k4[2 * b + 1].x : w == 1 ? k4[2 * b + 1].y : w == 2 ? k4[2 * b + 1].z : k4[2 * b + 1].w;
          const unsigned a0 = df_lo(ka), a1 = df_lo(kb), a2 = df_hi(ka), a3 = df_hi(kb);
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) df_mma(s[b][nh], a0, a1, a2, a3, qb[nh][c * 4 + w][0], qb[nh][c * 4 + w][1]);
        }
      }
    }
    unsigned exps = lane < 2 ? *reinterpret_cast<const unsigned*>(at + 2 * Pipe::kHalf + lane * 4) : 0u;
    exps >>= (u & 1) * 16;
    const unsigned kes = __shfl_sync(0xffffffffu, exps, 0), ves = __shfl_sync(0xffffffffu, exps, 1);
    const int p0 = u * kDfUnit;
    const bool edge = p0 < lo || p0 + kDfUnit > len;
    float back[2];
    bool grow = false;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int ke = clamp_exponent((int)(signed char)(kes >> (8 * b) & 0xffu)), ve = clamp_exponent((int)(signed char)(ves >> (8 * b) & 0xffu));
      const float kf = pow2_of(ke), add = (float)ve;
      back[b] = pow2_of(-ve);
      const int p = p0 + b * kExpBlock + g;
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) {
        const float f0 = df_finite(q_scale[nh][0] * kf), f1 = df_finite(q_scale[nh][1] * kf);
        float* x = s[b][nh];
        x[0] = fmaf(x[0], f0, add);
        x[1] = fmaf(x[1], f1, add);
        x[2] = fmaf(x[2], f0, add);
        x[3] = fmaf(x[3], f1, add);
        if (edge) {
          if (p < lo || p >= len) x[0] = x[1] = -INFINITY;
          if (p + 8 < lo || p + 8 >= len) x[2] = x[3] = -INFINITY;
        }
        grow |= fmaxf(x[0], x[2]) > R[nh][0] + kDfSlack || fmaxf(x[1], x[3]) > R[nh][1] + kDfSlack;
      }
    }
    if (__any_sync(0xffffffffu, grow)) {
      // a head has outgrown its bound: all of them follow their largest score
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) {
        float mx0 = fmaxf(fmaxf(s[0][nh][0], s[0][nh][2]), fmaxf(s[1][nh][0], s[1][nh][2]));
        float mx1 = fmaxf(fmaxf(s[0][nh][1], s[0][nh][3]), fmaxf(s[1][nh][1], s[1][nh][3]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
        }
        const float r0 = fmaxf(R[nh][0], mx0), r1 = fmaxf(R[nh][1], mx1);
        const float al0 = R[nh][0] == -INFINITY ? 0.f : df_exp2(R[nh][0] - r0), al1 = R[nh][1] == -INFINITY ? 0.f : df_exp2(R[nh][1] - r1);
        R[nh][0] = r0;
        R[nh][1] = r1;
        l[nh][0] *= al0;
        l[nh][1] *= al1;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[nh][i][0] *= al0;
          o[nh][i][1] *= al1;
          o[nh][i][2] *= al0;
          o[nh][i][3] *= al1;
        }
      }
    }
    unsigned wb[2][NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
      const float c0 = (R[nh][0] == -INFINITY ? 0.f : R[nh][0]) - kDfTop, c1 = (R[nh][1] == -INFINITY ? 0.f : R[nh][1]) - kDfTop;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float* x = s[b][nh];
        const float w0 = df_exp2(x[0] - c0), w1 = df_exp2(x[1] - c1), w2 = df_exp2(x[2] - c0), w3 = df_exp2(x[3] - c1);
        l[nh][0] = fmaf(w0 + w2, back[b], l[nh][0]);
        l[nh][1] = fmaf(w1 + w3, back[b], l[nh][1]);
        wb[b][nh][0] = df_transpose(df_half2(w0, w1));
        wb[b][nh][1] = df_transpose(df_half2(w2, w3));
      }
    }
    // O^T += V^T W^T
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      unsigned v[4][HD / 32];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned char* p = at + Pipe::kHalf + df_at<HD>(b * kExpBlock + 2 * t + (i & 1) + (i >> 1) * 8, HD == 64 ? g >> 1 : g) +
                                 (HD == 64 ? (g & 1) * 8 : 0);
        if (HD == 64) {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          v[i][0] = w.x;
          v[i][1] = w.y;
        } else {
          const uint4 w = *reinterpret_cast<const uint4*>(p);
          v[i][0] = w.x;
          v[i][1] = w.y;
          v[i][HD / 32 - 2] = w.z;
          v[i][HD / 32 - 1] = w.w;
        }
        if (edge) {
          // values that nobody sees may be anything (a page has had other owners): they must not meet a weight, not even zero
          const int pos = p0 + b * kExpBlock + 2 * t + (i & 1) + (i >> 1) * 8;
          if (pos < lo || pos >= len) {
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) v[i][c] = 0u;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) {
        // four columns of two positions each, interleaved into pairs of neighbouring positions
        const unsigned e0 = __byte_perm(v[0][c], v[1][c], 0x5140), e1 = __byte_perm(v[0][c], v[1][c], 0x7362);
        const unsigned h0 = __byte_perm(v[2][c], v[3][c], 0x5140), h1 = __byte_perm(v[2][c], v[3][c], 0x7362);
        const unsigned b0 = df_lo(e0), b1 = df_hi(e0), b2 = df_lo(h0), b3 = df_hi(h0);
        const unsigned d0 = df_lo(e1), d1 = df_hi(e1), d2 = df_lo(h1), d3 = df_hi(h1);
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
          df_mma(o[nh][2 * c], b0, b1, b2, b3, wb[b][nh][0], wb[b][nh][1]);
          df_mma(o[nh][2 * c + 1], d0, d1, d2, d3, wb[b][nh][0], wb[b][nh][1]);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();                      // no lane reads its units any more: the place becomes the results'
  float* sums = reinterpret_cast<float*>(mine);
  float* bounds = sums + Cfg::kHeads * Cfg::kPitch;
  // The denominators of the whole warp, in every lane.
  auto all_lanes = [&]() {
#pragma unroll
    for (int nh = 0; nh < NH; ++nh)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[nh][0] += __shfl_xor_sync(0xffffffffu, l[nh][0], d);
        l[nh][1] += __shfl_xor_sync(0xffffffffu, l[nh][1], d);
      }
  };
  all_lanes();
  unsigned least = 0xffffffffu;      // by their bits less one: without a key there is no denominator, and none is small
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) least = min(least, min(__float_as_uint(l[nh][0]) - 1u, __float_as_uint(l[nh][1]) - 1u));
  if (__any_sync(0xffffffffu, least < __float_as_uint(kLeastDenominator) - 1u)) {
    // rare: by the scores alone (see fp8.cuh), the warp's units once more, codes straight from the cache
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) l[nh][0] = l[nh][1] = 0.f;
#pragma unroll 1
    for (int v = first + u_begin + warp; v < u_stop; v += W) {
      const size_t row = (size_t)pages[v >> 1] * a.n_kv + hk;
#pragma unroll 1
      for (int b = 0; b < 2; ++b) {
        const int in = (v & 1) * 2 + b, p = v * kDfUnit + b * kExpBlock + g;
        const unsigned char* key = a.k + (row * kFp8Page + in * kExpBlock + g) * HD + t * 16;
        float x[NH][4];
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) x[nh][0] = x[nh][1] = x[nh][2] = x[nh][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const unsigned ka = *reinterpret_cast<const unsigned*>(key + (ks >> 2) * 64 + (ks & 3) * 4);
          const unsigned kb = *reinterpret_cast<const unsigned*>(key + 8 * HD + (ks >> 2) * 64 + (ks & 3) * 4);
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) df_mma(x[nh], df_lo(ka), df_lo(kb), df_hi(ka), df_hi(kb), qb[nh][ks][0], qb[nh][ks][1]);
        }
        const float kf = pow2_of(clamp_exponent(a.k_exp[row * kPageExps + in]));
#pragma unroll
        for (int nh = 0; nh < NH; ++nh) {
          const float f0 = df_finite(q_scale[nh][0] * kf), f1 = df_finite(q_scale[nh][1] * kf);
          const float c0 = kDfTop - (R[nh][0] == -INFINITY ? 0.f : R[nh][0]), c1 = kDfTop - (R[nh][1] == -INFINITY ? 0.f : R[nh][1]);
          const bool here = p >= lo && p < len, there = p + 8 >= lo && p + 8 < len;
          l[nh][0] += (here ? exp2_term(fmaf(x[nh][0], f0, c0)) : 0.f) + (there ? exp2_term(fmaf(x[nh][2], f0, c0)) : 0.f);
          l[nh][1] += (here ? exp2_term(fmaf(x[nh][1], f1, c1)) : 0.f) + (there ? exp2_term(fmaf(x[nh][3], f1, c1)) : 0.f);
        }
        __syncwarp();                // the products are the whole warp's
      }
    }
    all_lanes();
  }
#pragma unroll
  for (int nh = 0; nh < NH; ++nh) {
    if (g == 0) {
      bounds[nh * 8 + 2 * t] = R[nh][0];
      bounds[nh * 8 + 2 * t + 1] = R[nh][1];
      bounds[Cfg::kHeads + nh * 8 + 2 * t] = l[nh][0];
      bounds[Cfg::kHeads + nh * 8 + 2 * t + 1] = l[nh][1];
    }
    float* dst = sums + (nh * 8 + 2 * t) * Cfg::kPitch + g;
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      dst[i * 16] = o[nh][i][0];
      dst[i * 16 + Cfg::kPitch] = o[nh][i][1];
      dst[i * 16 + 8] = o[nh][i][2];
      dst[i * 16 + 8 + Cfg::kPitch] = o[nh][i][3];
    }
  }
}

// One number of a block's result: head h, place `at` of its sums; its bound and denominator with it. Behind a barrier. (What is relative to
// a bound d below the common one is times 2^(d / 2) twice: 2^d alone may be below float32 where the denominator's part is not, see
// fp8.cuh. By cases, d above -100 or not, a step of one sequence of 517 keys took 4.50 us; 4.39 so, and 4.37 with 2^d alone.)
template <int HD, int NH, int W>
__device__ __forceinline__ void df_of_warps(const unsigned char* smem, int h, int at, float& M, float& num, float& den) {
  using Cfg = DfCfg<HD, NH>;
  const float* s[W];
#pragma unroll
  for (int w = 0; w < W; ++w) s[w] = reinterpret_cast<const float*>(smem + w * DfPipe<HD, NH>::kPerWarp);
  M = -INFINITY;
#pragma unroll
  for (int w = 0; w < W; ++w) M = fmaxf(M, s[w][Cfg::kHeads * Cfg::kPitch + h]);
  const float Mu = M == -INFINITY ? 0.f : M;
  num = den = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float f = df_exp2(0.5f * (s[w][Cfg::kHeads * Cfg::kPitch + h] - Mu));
    num = fmaf(f * f, s[w][h * Cfg::kPitch + at], num);
    den = fmaf(f * s[w][Cfg::kHeads * (Cfg::kPitch + 1) + h], f, den);
  }
}

// Equal shares of the line of all units.
template <int HD, int NH, bool ROPE>
__global__ void __launch_bounds__(kDfThreads, df_per_sm<HD, NH>())
decode_fp8_kernel(const __nv_bfloat16* q, const DecodeArgs a, const DecodeStep st) {
  pdl_wait();
  pdl_launch_dependents();
  using Cfg = DfCfg<HD, NH>;
  extern __shared__ __align__(16) unsigned char df_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.n_q / a.n_kv, chunks = (G + Cfg::kHeads - 1) / Cfg::kHeads, per_seq = a.n_kv * chunks;
  const int total = df_total(a) * per_seq, share = df_share(total, gridDim.x);
  int cur = blockIdx.x * share;
  const int end = min(cur + share, total);
  if (blockIdx.x == 0) {
    // sequences that hold nothing: zeros
#pragma unroll 1
    for (int s = warp; s < a.n_seqs; s += kDfWarps)
      if (a.seq_kvlen[s] <= 0)
#pragma unroll 1
        for (int i = lane; i < a.n_q * HD; i += 32) a.out[(size_t)s * a.n_q * HD + i] = __float2bfloat16_rn(0.f);
  }
  if (cur >= end) return;
  // the sequence in which the share begins
  int seq = 0, first, count;
  int begin = 0;                     // where the sequence's units begin on the line
  {
    int before = 0;
#pragma unroll 1
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
      int f, c = 0;
      if (s0 + lane < a.n_seqs) df_units(a, a.seq_kvlen[s0 + lane], f, c);
      int incl = c * per_seq;
      const int own = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const unsigned here = __ballot_sync(0xffffffffu, before + incl > cur);
      if (here) {
        const int src = __ffs(here) - 1;
        seq = s0 + src;
        begin = before + __shfl_sync(0xffffffffu, incl - own, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
#pragma unroll 1
  while (cur < end) {
    const int len = min(a.seq_kvlen[seq], a.max_pages * kFp8Page);
    df_units(a, len, first, count);
    if (count == 0) {
      ++seq;
      continue;
    }
    const int item = (cur - begin) / count;                      // (KV head, chunk of query heads)
    const int u_begin = cur - begin - item * count;
    const int u_end = min(count, u_begin + (end - cur));
    const int hk = item / chunks, g0 = item % chunks * Cfg::kHeads, ng = min(Cfg::kHeads, G - g0);
    df_piece<HD, NH, ROPE, kDfWarps>(q, a, st, df_smem, seq, len, hk, g0, ng, first, count, u_begin, u_end);
    __syncthreads();
    const bool starts = u_begin == 0, whole = starts && u_end == count;
    float* rec = a.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * Cfg::kRecord;
#pragma unroll 1
    for (int i = threadIdx.x; i < ng * HD; i += kDfThreads) {
      const int h = i / HD, d = i % HD;
      float M, num, den;
      df_of_warps<HD, NH, kDfWarps>(df_smem, h, whole ? df_place<HD>(d) : d, M, num, den);      // a partial result stays in the order of the sums
      if (whole) {
        a.out[((size_t)seq * a.n_q + hk * G + g0 + h) * HD + d] = __float2bfloat16_rn(num / den);
      } else {
        rec[h * HD + d] = num;
        if (d == 0) {
          rec[Cfg::kHeads * HD + h] = M;
          rec[Cfg::kHeads * HD + Cfg::kHeads + h] = den;
        }
      }
    }
    __syncthreads();                 // shared memory may be written again
    cur += u_end - u_begin;
    if (item + 1 == per_seq && u_end == count) {
      begin += count * per_seq;
      ++seq;
    }
  }
}

// Few short sequences: an item is one cluster's, its units in equal runs over the cluster's blocks, which read one another's
// results from shared memory. grid (blocks of a cluster, items of a sequence, sequences). One launch, no partial results.
template <int HD, int NH, bool ROPE, int W>
__global__ void __launch_bounds__(W * 32, W > kDfWarps ? df_large_per_sm<HD, NH>() : df_per_sm<HD, NH>())
decode_fp8_cluster_kernel(const __nv_bfloat16* q, const DecodeArgs a, const DecodeStep st) {
  pdl_launch_dependents();
  pdl_wait();
  using Cfg = DfCfg<HD, NH>;
  extern __shared__ __align__(16) unsigned char df_smem[];
  __shared__ float joined[Cfg::kHeads * (HD + 2)];           // this block's result: sums, bounds, denominators
  const int G = a.n_q / a.n_kv, chunks = (G + Cfg::kHeads - 1) / Cfg::kHeads;
  const int seq = blockIdx.z, hk = blockIdx.y / chunks, g0 = blockIdx.y % chunks * Cfg::kHeads, ng = min(Cfg::kHeads, G - g0);
  const int len = min(a.seq_kvlen[seq], a.max_pages * kFp8Page);
  int first, count;
  df_units(a, len, first, count);
  __nv_bfloat16* out = a.out + ((size_t)seq * a.n_q + hk * G + g0) * HD;
  if (count == 0) {                  // the whole cluster alike
    for (int i = blockIdx.x * W * 32 + threadIdx.x; i < ng * HD; i += gridDim.x * W * 32) out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  const int u_begin = count * blockIdx.x / gridDim.x, u_end = count * (blockIdx.x + 1) / gridDim.x;
  df_piece<HD, NH, ROPE, W>(q, a, st, df_smem, seq, len, hk, g0, ng, first, count, u_begin, u_end);
  __syncthreads();
#pragma unroll 1
  for (int i = threadIdx.x; i < ng * HD; i += W * 32) {
    const int h = i / HD, d = i % HD;
    float M, num, den;
    df_of_warps<HD, NH, W>(df_smem, h, df_place<HD>(d), M, num, den);
    if (gridDim.x == 1) {
      out[i] = __float2bfloat16_rn(num / den);
      continue;
    }
    joined[i] = num;
    if (d == 0) {
      joined[Cfg::kHeads * HD + h] = M;
      joined[Cfg::kHeads * (HD + 1) + h] = den;
    }
  }
  if (gridDim.x == 1) return;
  tc::cluster_sync_all();
  const uint32_t here = (uint32_t)__cvta_generic_to_shared(joined);
#pragma unroll 1
  for (int i = blockIdx.x * W * 32 + threadIdx.x; i < ng * HD; i += gridDim.x * W * 32) {
    const int h = i / HD;
    float m[8], n[8], l[8], M = -INFINITY;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      if (b >= gridDim.x) continue;
      const uint32_t there = tc::map_to_block(here, b);
      m[b] = tc::ld_cluster_f32(there + (Cfg::kHeads * HD + h) * 4);
      n[b] = tc::ld_cluster_f32(there + i * 4);
      l[b] = tc::ld_cluster_f32(there + (Cfg::kHeads * (HD + 1) + h) * 4);
    }
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (b < gridDim.x) M = fmaxf(M, m[b]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      if (b >= gridDim.x) continue;
      const float f = df_exp2(0.5f * (m[b] - Mu));
      num = fmaf(f * f, n[b], num);
      den = fmaf(f * l[b], f, den);
    }
    out[i] = __float2bfloat16_rn(num / den);
  }
  tc::cluster_sync_all();            // nobody's shared memory goes before everyone has read it
}

// Joins the partial results of the items that lie in several shares. grid (items of all sequences, heads side by side); four threads
// a column, a quarter of the partial results each.
constexpr int kDfSlices = 4;
template <int HD, int NH>
__global__ void __launch_bounds__(kDfSlices * HD) decode_fp8_join_kernel(const DecodeArgs a, int blocks) {
  pdl_launch_dependents();
  using Cfg = DfCfg<HD, NH>;
  __shared__ float factor[kSms * 6], denom[kSms * 6], part_num[kDfSlices][HD], part_den[kDfSlices * HD / 32], top[kDfSlices * HD / 32];
  const int G = a.n_q / a.n_kv, chunks = (G + Cfg::kHeads - 1) / Cfg::kHeads, per_seq = a.n_kv * chunks;
  const int seq = blockIdx.x / per_seq, item = blockIdx.x % per_seq;
  const int hk = item / chunks, g0 = item % chunks * Cfg::kHeads, ng = min(Cfg::kHeads, G - g0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int first, count;
  int all = 0, ahead = 0;
#pragma unroll 1
  for (int s = lane; s < a.n_seqs; s += 32) {
    int f, c;
    df_units(a, a.seq_kvlen[s], f, c);
    all += c;
    ahead += s < seq ? c : 0;
  }
  df_units(a, a.seq_kvlen[seq], first, count);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  }
  const int share = df_share(all * per_seq, blocks);
  const int begin = ahead * per_seq + item * count;
  const int c0 = begin / share, n = count == 0 ? 0 : (begin + count - 1) / share - c0 + 1;
  // The lengths are older than the kernel that leaves the partial results (it lets this one begin behind its own wait). Blocks with
  // nothing to join wait too: the kernel behind this one waits for this one alone, and reads what the one in front wrote.
  pdl_wait();
  if (n <= 1) return;
  // partial result i: the first lies where a piece begins with its item, the others where one goes on
  const float* base = a.part + (size_t)c0 * 2 * Cfg::kRecord;
  auto record = [&](int i) { return base + (size_t)(i == 0 ? 1 : 2 * i) * Cfg::kRecord; };
  __nv_bfloat16* out = a.out + ((size_t)seq * a.n_q + hk * G + g0) * HD;
  // the column whose sum is at place d
  auto column = [](int d) { return (d % 8) * (HD / 8) + (d / 16) * 2 + (d / 8 & 1); };
  if (n <= 4) {
    // few of them (many sequences): a thread a column, everything asked for at once
#pragma unroll 1
    for (int x = blockIdx.y * kDfSlices * HD + threadIdx.x; x < ng * HD; x += gridDim.y * kDfSlices * HD) {
      const int h = x / HD;
      float m[4], l[4], v[4], M = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = i < n ? __ldcg(record(i) + Cfg::kHeads * HD + h) : -INFINITY;
        l[i] = i < n ? __ldcg(record(i) + Cfg::kHeads * (HD + 1) + h) : 0.f;
        v[i] = i < n ? __ldcg(record(i) + x) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) M = fmaxf(M, m[i]);
      const float Mu = M == -INFINITY ? 0.f : M;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = df_exp2(0.5f * (m[i] - Mu));
        num = fmaf(f * f, v[i], num);
        den = fmaf(f * l[i], f, den);
      }
      out[h * HD + column(x % HD)] = __float2bfloat16_rn(num / den);
    }
    return;
  }
  const int d = threadIdx.x % HD, slice = threadIdx.x / HD;
  for (int h = blockIdx.y; h < ng; h += gridDim.y) {
    // the first numbers are asked for before their factors are known
    float v[8];
    int i = slice;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = i + e * kDfSlices < n ? __ldcg(record(i + e * kDfSlices) + h * HD + d) : 0.f;
    float M = -INFINITY;
    for (int k = threadIdx.x; k < n; k += kDfSlices * HD) {
      const float m = __ldcg(record(k) + Cfg::kHeads * HD + h);
      factor[k] = m;
      denom[k] = __ldcg(record(k) + Cfg::kHeads * (HD + 1) + h);
      M = fmaxf(M, m);
    }
    M = warp_max(M);
    if (lane == 0) top[warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kDfSlices * HD / 32; ++w) M = fmaxf(M, top[w]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float den = 0.f;
    for (int k = threadIdx.x; k < n; k += kDfSlices * HD) {
      const float f = df_exp2(0.5f * (factor[k] - Mu));
      factor[k] = f * f;
      den = fmaf(f * denom[k], f, den);
    }
    den = warp_sum(den);
    if (lane == 0) part_den[warp] = den;
    __syncthreads();
    float num = 0.f;
    while (i < n) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e * kDfSlices < n) num = fmaf(factor[i + e * kDfSlices], v[e], num);
      i += 8 * kDfSlices;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = i + e * kDfSlices < n ? __ldcg(record(i + e * kDfSlices) + h * HD + d) : 0.f;
    }
    part_num[slice][d] = num;
    __syncthreads();
    if (slice == 0) {
      den = 0.f;
#pragma unroll
      for (int w = 0; w < kDfSlices * HD / 32; ++w) den += part_den[w];
#pragma unroll
      for (int e = 1; e < kDfSlices; ++e) num += part_num[e][d];
      out[h * HD + column(d)] = __float2bfloat16_rn(num / den);
    }
    __syncthreads();
  }
}

template <int HD, int NH, bool ROPE, int W>
static int launch_cluster(const void* q, const DecodeArgs& a, const DecodeStep& st, int items_of_seq, int cluster, cudaStream_t stream) {
  cudaError_t e = cudaFuncSetAttribute(decode_fp8_cluster_kernel<HD, NH, ROPE, W>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       DfPipe<HD, NH, W>::kSmem);
  if (e != cudaSuccess) return (int)e;
  launch_k_cluster(decode_fp8_cluster_kernel<HD, NH, ROPE, W>, dim3(cluster, items_of_seq, a.n_seqs), dim3(W * 32), DfPipe<HD, NH, W>::kSmem,
                   stream, cluster, (const __nv_bfloat16*)q, a, st);
  LLMIE_LAUNCH_CHECK();
  return LLMIE_OK;
}

template <int HD, int NH, bool ROPE>
static int launch_decode(const void* q, const DecodeArgs& a, const DecodeStep& st, int max_kv_len, cudaStream_t stream) {
  const int G = a.n_q / a.n_kv, chunks = (G + 8 * NH - 1) / (8 * NH);
  const long long items = (long long)a.n_seqs * a.n_kv * chunks;
  // units of the longest sequence, as far as the caller knows
  long long units = max_kv_len > 0 ? max_kv_len : (long long)a.max_pages * kFp8Page;
  if (a.window > 0 && (long long)a.window + kDfUnit < units) units = (long long)a.window + kDfUnit;
  if (a.window < 0 && -(long long)a.window < units) units = -(long long)a.window;
  units = (units + kDfUnit - 1) / kDfUnit;
  int cluster = 1;                   // blocks that share an item
  while (cluster < 8 && 2 * cluster * items <= df_blocks<HD, NH>() && 2 * cluster * kDfWarps <= units) cluster *= 2;
  if (units <= (long long)cluster * kDfWarps * kDfFew && items <= df_blocks<HD, NH>() && items <= 65535) {
    // Where these blocks would share SMs, half as many large ones, or one instead of two that have to meet (37 sequences, window of
    // 1,024, 148 items: 14.1 us with two blocks an item, 10.8 with one; 18 of 1,050 keys, head size 64: 10.7 and 7.7. One sequence of
    // 517: 4.4 with four blocks an item, 4.9 with two).
    if (cluster > 1 && items * cluster > kSms && items * (cluster / 2) <= kSms * df_large_per_sm<HD, NH>())
      return launch_cluster<HD, NH, ROPE, 2 * kDfWarps>(q, a, st, a.n_kv * chunks, cluster / 2, stream);
    return launch_cluster<HD, NH, ROPE, kDfWarps>(q, a, st, a.n_kv * chunks, cluster, stream);
  }
  if (!a.part) return kNeedsScratch;
  cudaError_t e = cudaFuncSetAttribute(decode_fp8_kernel<HD, NH, ROPE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       DfPipe<HD, NH>::kSmem);
  if (e != cudaSuccess) return (int)e;
  constexpr int blocks = df_blocks<HD, NH>();
  launch_k(decode_fp8_kernel<HD, NH, ROPE>, dim3(blocks), dim3(kDfThreads), DfPipe<HD, NH>::kSmem, stream, (const __nv_bfloat16*)q, a, st);
  LLMIE_LAUNCH_CHECK();
  const int side = (int)max(1LL, min((long long)min(G, 8 * NH), 4 * kSms / items));
  launch_k(decode_fp8_join_kernel<HD, NH>, dim3((unsigned)items, side), dim3(kDfSlices * HD), 0, stream, a, blocks);
  LLMIE_LAUNCH_CHECK();
  return LLMIE_OK;
}

}  // namespace llmie

using namespace llmie;

// float32 numbers of scratch that a call needs
extern "C" int llmie_attention_decode_fp8_scratch(int n_q, int n_kv, int hd) {
  if (n_kv <= 0 || n_q <= 0 || n_q % n_kv) return 0;
  const bool one = n_q / n_kv <= 8;
  if (hd == 64) return one ? 2 * df_blocks<64, 1>() * DfCfg<64, 1>::kRecord : 2 * df_blocks<64, 2>() * DfCfg<64, 2>::kRecord;
  return one ? 2 * df_blocks<128, 1>() * DfCfg<128, 1>::kRecord : 2 * df_blocks<128, 2>() * DfCfg<128, 2>::kRecord;
}

static int decode_fp8_entry(const void* q, const void* k_cache, const void* v_cache, const void* k_exp, const void* v_exp, void* out,
                            float* scratch, const float* rope, int table_len, const int* seq_slot, const int* seq_kvlen,
                            const int* block_table, int max_pages, int n_seqs, int n_q, int n_kv, int hd, float scale, int window,
                            int max_kv_len, cudaStream_t stream) {
  if (n_seqs < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0 || max_pages > (1 << 24)) return LLMIE_ERR_BAD_ARG;
  if (hd != 64 && hd != 128) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache)) return LLMIE_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(k_exp) | reinterpret_cast<uintptr_t>(v_exp)) & 3u) return LLMIE_ERR_ALIGNMENT;   // a page's four at once
  if (n_seqs == 0) return LLMIE_OK;
  // The line of units is counted in 32 bits: of a (sequence, KV head, chunk of 8 or 16 query heads) as many as its table has room for, or as
  // its window or chunk can touch.
  const long long chunks = n_q / n_kv <= 8 ? 1 : (n_q / n_kv + 15) / 16, back = window < 0 ? -(long long)window : window;
  const long long units = back ? min(2LL * max_pages, back / kDfUnit + 2) : 2LL * max_pages;
  if ((double)n_seqs * n_kv * chunks * units > 2.0e9) return LLMIE_ERR_UNSUPPORTED_SIZE;
  const DecodeArgs a{(const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp, (const signed char*)v_exp,
                     (__nv_bfloat16*)out, scratch, seq_slot, seq_kvlen, block_table, max_pages, n_seqs, n_q, n_kv,
                     scale * 1.4426950408889634f, window};
  const DecodeStep st{(const float4*)rope, table_len, (unsigned char*)k_cache, (unsigned char*)v_cache, (signed char*)k_exp, (signed char*)v_exp};
  const bool one = n_q / n_kv <= 8;
#define LLMIE_DECODE(HD, NH) return rope ? launch_decode<HD, NH, true>(q, a, st, max_kv_len, stream) : launch_decode<HD, NH, false>(q, a, st, max_kv_len, stream)
  if (hd == 64 && one) LLMIE_DECODE(64, 1);
  if (hd == 64) LLMIE_DECODE(64, 2);
  if (one) LLMIE_DECODE(128, 1);
  LLMIE_DECODE(128, 2);
#undef LLMIE_DECODE
}

// q, out bfloat16 [n_seqs, n_q hd], hd 64 or 128; caches e4m3 [pages, n_kv, 64, hd] with exponents int8 [pages, n_kv, 4];
// seq_kvlen: keys that each sequence holds, this step's among them (0: its rows become zeros). window as in the other attention
// kernels. max_kv_len: no sequence is longer (0: not known); the choice of the kernel goes by it, not its result.
// scratch: llmie_attention_decode_fp8_scratch floats, 16-byte aligned; null: a call that needs it launches nothing and returns -5.
extern "C" int llmie_attention_decode_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_exp,
                                          const void* v_exp, void* out, float* scratch, const int* seq_slot, const int* seq_kvlen,
                                          const int* block_table, int max_pages, int n_seqs, int n_q, int n_kv, int hd,
                                          float scale, int window, int max_kv_len, cudaStream_t stream) {
  return decode_fp8_entry(q, k_cache, v_cache, k_exp, v_exp, out, scratch, nullptr, 0, seq_slot, seq_kvlen, block_table, max_pages,
                          n_seqs, n_q, n_kv, hd, scale, window, max_kv_len, stream);
}

// The same from a step's projections: qkv bfloat16 [n_seqs, (n_q + 2 n_kv) hd], rope float32 [table_len, hd / 2, 2] the (cos, sin) of
// every position; the new key (rotated) and value of sequence i are written for position seq_kvlen[i] - 1 and read with the rest. A
// KV head must be one block's work (at most 16 query heads): the others would read what one of them writes.
extern "C" int llmie_attention_decode_fp8_rope(const void* qkv, void* k_cache, void* v_cache, void* k_exp, void* v_exp, void* out,
                                               float* scratch, const float* rope, int table_len, const int* seq_slot,
                                               const int* seq_kvlen, const int* block_table, int max_pages, int n_seqs, int n_q,
                                               int n_kv, int hd, float scale, int window, int max_kv_len, cudaStream_t stream) {
  if (!rope || table_len <= 0 || n_kv <= 0 || n_q / n_kv > 16) return LLMIE_ERR_BAD_ARG;
  if (!aligned16(rope)) return LLMIE_ERR_ALIGNMENT;
  return decode_fp8_entry(qkv, k_cache, v_cache, k_exp, v_exp, out, scratch, rope, table_len, seq_slot, seq_kvlen, block_table,
                          max_pages, n_seqs, n_q, n_kv, hd, scale, window, max_kv_len, stream);
}

// Both by one address, with the arguments one behind another as they are above: a caller from another language converts one
// argument instead of some twenty, which takes as long as the launch.
struct DecodeCall {
  const void *q, *k_cache, *v_cache, *k_exp, *v_exp;
  void* out;
  float* scratch;
  const int *seq_slot, *seq_kvlen, *block_table;
  int max_pages, n_seqs, n_q, n_kv, hd;
  float scale;
  int window, max_kv_len;
  cudaStream_t stream;
};
extern "C" int llmie_attention_decode_fp8_call(const DecodeCall* c) {
  return llmie_attention_decode_fp8(c->q, c->k_cache, c->v_cache, c->k_exp, c->v_exp, c->out, c->scratch, c->seq_slot, c->seq_kvlen,
                                    c->block_table, c->max_pages, c->n_seqs, c->n_q, c->n_kv, c->hd, c->scale, c->window,
                                    c->max_kv_len, c->stream);
}
struct DecodeRopeCall {
  const void* qkv;
  void *k_cache, *v_cache, *k_exp, *v_exp, *out;
  float* scratch;
  const float* rope;
  int table_len;
  const int *seq_slot, *seq_kvlen, *block_table;
  int max_pages, n_seqs, n_q, n_kv, hd;
  float scale;
  int window, max_kv_len;
  cudaStream_t stream;
};
extern "C" int llmie_attention_decode_fp8_rope_call(const DecodeRopeCall* c) {
  return llmie_attention_decode_fp8_rope(c->qkv, c->k_cache, c->v_cache, c->k_exp, c->v_exp, c->out, c->scratch, c->rope, c->table_len,
                                         c->seq_slot, c->seq_kvlen, c->block_table, c->max_pages, c->n_seqs, c->n_q, c->n_kv, c->hd,
                                         c->scale, c->window, c->max_kv_len, c->stream);
}
