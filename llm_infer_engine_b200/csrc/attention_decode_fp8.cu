// Attention of one token a sequence over a paged cache in 8 bits (fp8.cuh), on the tensor cores.
//
//   o = sum_j 2^(s_j) c_j 2^(ev_j) / sum_j 2^(s_j),     s_j = scale log2(e) (q . k_j) 2^(ek_j)      (k, c: codes of keys, values)
//
// A warp works on 16 positions of a KV head at a time, which is one block of the cache: its keys have one exponent, its
// values another. A value's exponent is added to the score, so that one exponential gives the weight that its codes get:
// with R >= s_j + ev_j a running bound, w_j = 2^(s_j + ev_j - R + 15) lies in (0, 2^15] and goes into the second product
// in half precision (its normal range reaches 2^-29 below the largest weight), and the softmax's denominator is sum_j w_j
// 2^(-ev_j), kept in float32 relative to the same R.
//
// Both products are mma.sync.m16n8k16 with the cache as the 16-row operand and the query heads of the KV head as the 8
// columns: S^T = K Q^T and O^T = V^T W^T. Codes become half-precision numbers (exactly) in registers, so the cache goes from
// global memory to the multiplier without shared memory: which k index stands for which column of a head is free as long as
// both operands agree, so a lane reads 16 neighbouring codes of a key (and 8 or 16 of a value), whole sectors every time.
// W^T comes out of S^T's accumulators by one 8x8 transpose between lanes (movmatrix). Queries are brought to half precision
// with a power of two per head (their largest number in [2^14, 2^15)), which keeps every digit of bfloat16.
//
// Work is cut by blocks of positions, not by sequences: all (sequence, KV head) items one after another make one line of
// units, and every thread block takes an equal share of it, wherever it begins and ends. Lengths are read on the device, so
// a captured step costs what its sequences hold. An item that lies in several shares leaves partial results, and a second
// small kernel joins them in the order of the shares: no atomics, no counters, nothing kept between calls.
#include "fp8.cuh"
#include <math.h>

namespace llmie {

constexpr int kDfWarps = 4;
constexpr int kDfThreads = kDfWarps * 32;
constexpr int kSms = 148;

__device__ __forceinline__ float df_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
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
// The cache is read once: past the first-level cache.
__device__ __forceinline__ uint4 df_load16(const unsigned char* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 df_load8(const unsigned char* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
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

// Blocks of 16 positions that a sequence's newest token sees: [first, first + count).
__device__ __forceinline__ void df_units(const DecodeArgs& a, int len, int& first, int& count) {
  len = min(len, a.max_pages * kFp8Page);              // what the table has room for
  if (len <= 0) {
    first = count = 0;
    return;
  }
  first = first_visible_key(len - 1, a.window) / kExpBlock;
  count = (len - 1) / kExpBlock - first + 1;
}

// Units of all sequences together (every item of a sequence has as many as the sequence). All lanes of a warp call it.
__device__ __forceinline__ long long df_total(const DecodeArgs& a) {
  const int lane = threadIdx.x & 31;
  long long t = 0;
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
__device__ __forceinline__ long long df_share(long long total_units, int blocks) {
  const long long s = (total_units + blocks - 1) / blocks;
  return s < kDfWarps ? kDfWarps : s;
}

template <int HD, int NH> struct DfCfg {
  static constexpr int kHeads = 8 * NH;
  static constexpr int kPitch = HD + 4;                          // floats between two heads' sums: lanes 4 banks apart
  static constexpr int kRecord = kHeads * (HD + 2);              // floats of a partial result: sums, then bounds and denominators
};
// Thread blocks that an SM holds at once.
template <int HD, int NH> __host__ __device__ constexpr int df_per_sm() { return HD == 64 ? (NH == 1 ? 4 : 3) : NH == 1 ? 3 : 2; }
template <int HD, int NH> constexpr int df_blocks() { return kSms * df_per_sm<HD, NH>(); }
// Where column d of a head stands among a head's sums: as the second product's accumulators hold them.
template <int HD> __device__ __forceinline__ int df_place(int d) {
  constexpr int R = HD / 8;
  return (d % R / 2) * 16 + (d & 1) * 8 + d / R;
}

// One unit as a warp's lanes hold it: lane (g, t) has keys g and g + 8, 16 columns from 16 t on of every 64; and the values
// of positions 2t, 2t + 1, 2t + 8, 2t + 9, HD / 8 columns from g HD / 8 on.
template <int HD> struct DfUnit {
  uint4 k[2][HD / 64];
  uint2 v[4][HD / 64];
  int ke, ve;
};

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

template <int HD, int NH, bool ROPE>
__global__ void __launch_bounds__(kDfThreads, df_per_sm<HD, NH>())
decode_fp8_kernel(const __nv_bfloat16* q, const DecodeArgs a, const DecodeStep st) {
  pdl_launch_dependents();
  pdl_wait();
  using Cfg = DfCfg<HD, NH>;
  constexpr int KS = HD / 16;
  __shared__ float sums[kDfWarps][Cfg::kHeads * Cfg::kPitch];
  __shared__ float bound_[kDfWarps][Cfg::kHeads], denom_[kDfWarps][Cfg::kHeads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int G = a.n_q / a.n_kv, chunks = (G + Cfg::kHeads - 1) / Cfg::kHeads, per_seq = a.n_kv * chunks;
  const long long total = df_total(a) * per_seq;
  const long long share = df_share(total, gridDim.x);
  long long cur = (long long)blockIdx.x * share;
  const long long end = min(cur + share, total);
  if (blockIdx.x == 0) {
    // sequences that hold nothing: zeros
    for (int s = warp; s < a.n_seqs; s += kDfWarps)
      if (a.seq_kvlen[s] <= 0)
        for (int i = lane; i < a.n_q * HD; i += 32) a.out[(size_t)s * a.n_q * HD + i] = __float2bfloat16_rn(0.f);
  }
  if (cur >= end) return;
  // the sequence in which the share begins
  int seq = 0, first, count;
  long long begin = 0;               // where the sequence's units begin on the line
  {
    long long before = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
      int f, c = 0;
      if (s0 + lane < a.n_seqs) df_units(a, a.seq_kvlen[s0 + lane], f, c);
      long long incl = (long long)c * per_seq;
      const long long own = incl;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
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

  while (cur < end) {
    const int len = min(a.seq_kvlen[seq], a.max_pages * kFp8Page);
    df_units(a, len, first, count);
    if (count == 0) {
      ++seq;
      continue;
    }
    const int item = (int)((cur - begin) / count);               // (KV head, chunk of query heads)
    const int u_begin = (int)((cur - begin) - (long long)item * count);
    const int u_end = (int)min((long long)count, u_begin + (end - cur));
    const int hk = item / chunks, g0 = item % chunks * Cfg::kHeads, ng = min(Cfg::kHeads, G - g0);
    const int* pages = a.block_table + (size_t)a.seq_slot[seq] * a.max_pages;
    const int lo = first_visible_key(len - 1, a.window);

    auto load = [&](DfUnit<HD>& x, int u, int page) {
      const size_t row = (size_t)page * a.n_kv + hk;
      const int b = u & (kPageExps - 1);
      const unsigned char* kp = a.k + (row * kFp8Page + b * kExpBlock) * HD;
      const unsigned char* vp = a.v + (row * kFp8Page + b * kExpBlock) * HD;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) x.k[i][c] = df_load16(kp + (g + 8 * i) * HD + c * 64 + t * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned char* p = vp + (2 * t + (i & 1) + (i >> 1) * 8) * HD + g * (HD / 8);
        if (HD == 64) {
          x.v[i][0] = df_load8(p);
        } else {
          const uint4 w = df_load16(p);
          x.v[i][0] = make_uint2(w.x, w.y);
          x.v[i][HD / 64 - 1] = make_uint2(w.z, w.w);
        }
      }
      x.ke = clamp_exponent(a.k_exp[row * kPageExps + b]);
      x.ve = clamp_exponent(a.v_exp[row * kPageExps + b]);
    };
    auto page_of = [&](int u) { return pages[u / kPageExps]; };

    int u = first + u_begin + warp;
    const int u_stop = first + u_end;
    DfUnit<HD> x0, x1;
    int pg_next = 0;
    const size_t q_pitch = (size_t)(ROPE ? a.n_q + 2 * a.n_kv : a.n_q) * HD;
    if (ROPE && u_begin + 1 <= count && u_end == count && (count - 1 - u_begin) % kDfWarps == warp)
      df_append<HD>(q + seq * q_pitch, a, st, hk, len, page_of(first + count - 1));     // this warp reads that block itself
    if (u < u_stop) load(x0, u, page_of(u));
    if (u + kDfWarps < u_stop) pg_next = page_of(u + kDfWarps);

    // the queries: for head g of each group of 8, columns in the order of the keys' codes
    unsigned qb[NH][KS][2];
    float q_scale[NH][2];            // of heads 2t, 2t + 1: scale log2(e) 2^(what the queries were shifted by)
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
      // the exponent that brings the largest number into [2^14, 2^15); a head that is not finite stays as it is
      const int eb = (int)(__float_as_uint(big) >> 23);
      const int shift = eb == 255 ? 0 : min(max(141 - eb, -100), 100);
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
    float R[NH][2], l[NH][2];
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
      for (int i = 0; i < KS; ++i) o[nh][i][0] = o[nh][i][1] = o[nh][i][2] = o[nh][i][3] = 0.f;
      R[nh][0] = R[nh][1] = -INFINITY;
      l[nh][0] = l[nh][1] = 0.f;
    }

    auto work = [&](DfUnit<HD>& x, int uu) {
      float s[NH][4];
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) s[nh][0] = s[nh][1] = s[nh][2] = s[nh][3] = 0.f;
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        const unsigned ka[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w};
        const unsigned kb[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const unsigned a0 = df_lo(ka[w]), a1 = df_lo(kb[w]), a2 = df_hi(ka[w]), a3 = df_hi(kb[w]);
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) df_mma(s[nh], a0, a1, a2, a3, qb[nh][c * 4 + w][0], qb[nh][c * 4 + w][1]);
        }
      }
      const int p0 = uu * kExpBlock;
      const bool edge = p0 < lo || p0 + kExpBlock > len;
      const bool see_a = p0 + g >= lo && p0 + g < len, see_b = p0 + g + 8 >= lo && p0 + g + 8 < len;
      if (edge) {
        // values that nobody sees may be anything (a page has had other owners): they must not meet a weight, not even zero
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = p0 + 2 * t + (i & 1) + (i >> 1) * 8;
          if (p < lo || p >= len) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) x.v[i][c] = make_uint2(0u, 0u);
          }
        }
      }
      const float kf = pow2_of(x.ke), ve = (float)x.ve, back = pow2_of(-x.ve);
      unsigned wb[NH][2];
#pragma unroll
      for (int nh = 0; nh < NH; ++nh) {
        const float f0 = q_scale[nh][0] * kf, f1 = q_scale[nh][1] * kf;
        s[nh][0] = fmaf(s[nh][0], f0, ve);
        s[nh][1] = fmaf(s[nh][1], f1, ve);
        s[nh][2] = fmaf(s[nh][2], f0, ve);
        s[nh][3] = fmaf(s[nh][3], f1, ve);
        if (edge) {
          if (!see_a) s[nh][0] = s[nh][1] = -INFINITY;
          if (!see_b) s[nh][2] = s[nh][3] = -INFINITY;
        }
        float mx0 = fmaxf(s[nh][0], s[nh][2]), mx1 = fmaxf(s[nh][1], s[nh][3]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
        }
        const float r0 = fmaxf(R[nh][0], mx0), r1 = fmaxf(R[nh][1], mx1);
        const float c0 = r0 == -INFINITY ? 0.f : r0 - 15.f, c1 = r1 == -INFINITY ? 0.f : r1 - 15.f;
        const float al0 = df_exp2(R[nh][0] - 15.f - c0), al1 = df_exp2(R[nh][1] - 15.f - c1);   // 0 while R is -inf
        R[nh][0] = r0;
        R[nh][1] = r1;
        const float w0 = df_exp2(s[nh][0] - c0), w1 = df_exp2(s[nh][1] - c1), w2 = df_exp2(s[nh][2] - c0), w3 = df_exp2(s[nh][3] - c1);
        l[nh][0] = fmaf(l[nh][0], al0, (w0 + w2) * back);
        l[nh][1] = fmaf(l[nh][1], al1, (w1 + w3) * back);
        wb[nh][0] = df_transpose(df_half2(w0, w1));
        wb[nh][1] = df_transpose(df_half2(w2, w3));
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          o[nh][i][0] *= al0;
          o[nh][i][1] *= al1;
          o[nh][i][2] *= al0;
          o[nh][i][3] *= al1;
        }
      }
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          // four columns of two positions each, interleaved into pairs of neighbouring positions
          const unsigned va = w ? x.v[0][c].y : x.v[0][c].x, vb = w ? x.v[1][c].y : x.v[1][c].x;
          const unsigned vc = w ? x.v[2][c].y : x.v[2][c].x, vd = w ? x.v[3][c].y : x.v[3][c].x;
          const unsigned e0 = __byte_perm(va, vb, 0x5140), e1 = __byte_perm(va, vb, 0x7362);
          const unsigned h0 = __byte_perm(vc, vd, 0x5140), h1 = __byte_perm(vc, vd, 0x7362);
          const int i = (c * 2 + w) * 2;
#pragma unroll
          for (int nh = 0; nh < NH; ++nh) {
            df_mma(o[nh][i], df_lo(e0), df_hi(e0), df_lo(h0), df_hi(h0), wb[nh][0], wb[nh][1]);
            df_mma(o[nh][i + 1], df_lo(e1), df_hi(e1), df_lo(h1), df_hi(h1), wb[nh][0], wb[nh][1]);
          }
        }
      }
    };

    while (u < u_stop) {
      if (u + kDfWarps < u_stop) load(x1, u + kDfWarps, pg_next);
      if (u + 2 * kDfWarps < u_stop) pg_next = page_of(u + 2 * kDfWarps);
      work(x0, u);
      u += kDfWarps;
      if (u >= u_stop) break;
      if (u + kDfWarps < u_stop) load(x0, u + kDfWarps, pg_next);
      if (u + 2 * kDfWarps < u_stop) pg_next = page_of(u + 2 * kDfWarps);
      work(x1, u);
      u += kDfWarps;
    }

    // ---- the warps' results meet
#pragma unroll
    for (int nh = 0; nh < NH; ++nh) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        l[nh][0] += __shfl_xor_sync(0xffffffffu, l[nh][0], d);
        l[nh][1] += __shfl_xor_sync(0xffffffffu, l[nh][1], d);
      }
      if (g == 0) {
        bound_[warp][nh * 8 + 2 * t] = R[nh][0];
        bound_[warp][nh * 8 + 2 * t + 1] = R[nh][1];
        denom_[warp][nh * 8 + 2 * t] = l[nh][0];
        denom_[warp][nh * 8 + 2 * t + 1] = l[nh][1];
      }
      float* mine = sums[warp] + (nh * 8 + 2 * t) * Cfg::kPitch + g;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        mine[i * 16] = o[nh][i][0];
        mine[i * 16 + Cfg::kPitch] = o[nh][i][1];
        mine[i * 16 + 8] = o[nh][i][2];
        mine[i * 16 + 8 + Cfg::kPitch] = o[nh][i][3];
      }
    }
    __syncthreads();
    const bool starts = u_begin == 0, ends = u_end == count;
    float* rec = a.part + ((size_t)blockIdx.x * 2 + (starts ? 1 : 0)) * Cfg::kRecord;
    for (int i = threadIdx.x; i < ng * HD; i += kDfThreads) {
      const int h = i / HD, d = i % HD;
      const int at = (starts && ends) ? df_place<HD>(d) : d;     // a partial result stays in the order of the sums
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kDfWarps; ++w) M = fmaxf(M, bound_[w][h]);
      const float Mu = M == -INFINITY ? 0.f : M;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < kDfWarps; ++w) {
        const float f = df_exp2(bound_[w][h] - Mu);
        num = fmaf(f, sums[w][h * Cfg::kPitch + at], num);
        den = fmaf(f, denom_[w][h], den);
      }
      if (starts && ends) {
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
    if (item + 1 == per_seq && ends) {
      begin += (long long)count * per_seq;
      ++seq;
    }
  }
}

// Joins the partial results of the items that lie in several shares. grid (n_seqs * items of a sequence, heads of an item); HD threads.
template <int HD, int NH>
__global__ void __launch_bounds__(HD) decode_fp8_join_kernel(const DecodeArgs a, int blocks) {
  pdl_launch_dependents();
  pdl_wait();
  using Cfg = DfCfg<HD, NH>;
  const int G = a.n_q / a.n_kv, chunks = (G + Cfg::kHeads - 1) / Cfg::kHeads, per_seq = a.n_kv * chunks;
  const int seq = blockIdx.x / per_seq, item = blockIdx.x % per_seq;
  const int hk = item / chunks, g0 = item % chunks * Cfg::kHeads, h = blockIdx.y;
  if (h >= min(Cfg::kHeads, G - g0)) return;
  const int lane = threadIdx.x & 31;
  int first, count;
  df_units(a, a.seq_kvlen[seq], first, count);
  if (count == 0) return;
  long long all = 0, ahead = 0;
  for (int s = lane; s < a.n_seqs; s += 32) {
    int f, c;
    df_units(a, a.seq_kvlen[s], f, c);
    all += c;
    ahead += s < seq ? c : 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  }
  const long long share = df_share(all * per_seq, blocks);
  const long long begin = ahead * per_seq + (long long)item * count;
  const int c0 = (int)(begin / share), c1 = (int)((begin + count - 1) / share);
  if (c0 == c1) return;
  auto record = [&](int c) { return a.part + ((size_t)c * 2 + (c == c0 ? 1 : 0)) * Cfg::kRecord; };
  float M = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, __ldcg(record(c) + Cfg::kHeads * HD + h));
  M = warp_max(M);
  const float Mu = M == -INFINITY ? 0.f : M;
  const int d = threadIdx.x;
  float num = 0.f, den = 0.f;
  for (int b = c0; b <= c1; b += 32) {
    float f = 0.f;
    if (b + lane <= c1) {
      const float* r = record(b + lane) + Cfg::kHeads * HD;
      f = df_exp2(__ldcg(r + h) - Mu);
      den = fmaf(f, __ldcg(r + Cfg::kHeads + h), den);
    }
    const int n = min(32, c1 - b + 1);
#pragma unroll 8
    for (int i = 0; i < n; ++i) num = fmaf(__shfl_sync(0xffffffffu, f, i), __ldcg(record(b + i) + h * HD + d), num);
  }
  den = warp_sum(den);
  // this thread's sum stands for the column whose place it is
  constexpr int R = HD / 8;
  const int col = (d % 8) * R + (d / 16) * 2 + (d / 8 & 1);
  a.out[((size_t)seq * a.n_q + hk * G + g0 + h) * HD + col] = __float2bfloat16_rn(num / den);
}

template <int HD, int NH>
static int launch_decode(const void* q, const DecodeArgs& a, const DecodeStep& st, cudaStream_t stream) {
  constexpr int blocks = df_blocks<HD, NH>();
  if (st.rope) launch_k(decode_fp8_kernel<HD, NH, true>, dim3(blocks), dim3(kDfThreads), 0, stream, (const __nv_bfloat16*)q, a, st);
  else launch_k(decode_fp8_kernel<HD, NH, false>, dim3(blocks), dim3(kDfThreads), 0, stream, (const __nv_bfloat16*)q, a, st);
  LLMIE_LAUNCH_CHECK();
  const int G = a.n_q / a.n_kv, chunks = (G + 8 * NH - 1) / (8 * NH);
  launch_k(decode_fp8_join_kernel<HD, NH>, dim3((unsigned)(a.n_seqs * a.n_kv * chunks), min(G, 8 * NH)), dim3(HD), 0, stream, a, blocks);
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
                            cudaStream_t stream) {
  if (n_seqs < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0 || max_pages > (1 << 24) || !scratch) return LLMIE_ERR_BAD_ARG;
  if (hd != 64 && hd != 128) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache)) return LLMIE_ERR_ALIGNMENT;
  if (n_seqs == 0) return LLMIE_OK;
  if ((long long)n_seqs * n_q > 0x7fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  const DecodeArgs a{(const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp, (const signed char*)v_exp,
                     (__nv_bfloat16*)out, scratch, seq_slot, seq_kvlen, block_table, max_pages, n_seqs, n_q, n_kv,
                     scale * 1.4426950408889634f, window};
  const DecodeStep st{(const float4*)rope, table_len, (unsigned char*)k_cache, (unsigned char*)v_cache, (signed char*)k_exp, (signed char*)v_exp};
  const bool one = n_q / n_kv <= 8;
  if (hd == 64) return one ? launch_decode<64, 1>(q, a, st, stream) : launch_decode<64, 2>(q, a, st, stream);
  return one ? launch_decode<128, 1>(q, a, st, stream) : launch_decode<128, 2>(q, a, st, stream);
}

// q, out bfloat16 [n_seqs, n_q hd], hd 64 or 128; caches e4m3 [pages, n_kv, 64, hd] with exponents int8 [pages, n_kv, 4];
// seq_kvlen: keys that each sequence holds, this step's among them (0: its rows become zeros). window as in the other attention
// kernels. scratch: llmie_attention_decode_fp8_scratch floats, 16-byte aligned.
extern "C" int llmie_attention_decode_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_exp,
                                          const void* v_exp, void* out, float* scratch, const int* seq_slot, const int* seq_kvlen,
                                          const int* block_table, int max_pages, int n_seqs, int n_q, int n_kv, int hd,
                                          float scale, int window, cudaStream_t stream) {
  return decode_fp8_entry(q, k_cache, v_cache, k_exp, v_exp, out, scratch, nullptr, 0, seq_slot, seq_kvlen, block_table, max_pages,
                          n_seqs, n_q, n_kv, hd, scale, window, stream);
}

// The same from a step's projections: qkv bfloat16 [n_seqs, (n_q + 2 n_kv) hd], rope float32 [table_len, hd / 2, 2] the (cos, sin) of
// every position; the new key (rotated) and value of sequence i are written for position seq_kvlen[i] - 1 and read with the rest. A
// KV head must be one block's work (at most 16 query heads): the others would read what one of them writes.
extern "C" int llmie_attention_decode_fp8_rope(const void* qkv, void* k_cache, void* v_cache, void* k_exp, void* v_exp, void* out,
                                               float* scratch, const float* rope, int table_len, const int* seq_slot,
                                               const int* seq_kvlen, const int* block_table, int max_pages, int n_seqs, int n_q,
                                               int n_kv, int hd, float scale, int window, cudaStream_t stream) {
  if (!rope || table_len <= 0 || n_kv <= 0 || n_q / n_kv > 16) return LLMIE_ERR_BAD_ARG;
  if (!aligned16(rope)) return LLMIE_ERR_ALIGNMENT;
  return decode_fp8_entry(qkv, k_cache, v_cache, k_exp, v_exp, out, scratch, rope, table_len, seq_slot, seq_kvlen, block_table,
                          max_pages, n_seqs, n_q, n_kv, hd, scale, window, stream);
}
