// Keys and values of a step go into a paged cache in 8 bits, with the position rotation on the way.
//
//   (y_i, y_{i + R/2}) = (x_i c_i - x_{i + R/2} s_i,  x_{i + R/2} c_i + x_i s_i)        i < R/2, R the rotated size
//
// for queries and keys, (c, s) the cosine and sine of the token's position from a float32 table; every product and every
// sum is rounded once to float32 (no fused multiply-add: keys then have the same codes wherever they are made). Queries go
// out in their own type; keys and values become codes of their block of 16 positions (fp8.cuh).
//
// A block of positions and a KV head is one thread block's work, with the query heads that belong to it: it knows all of
// the block's new numbers, so the block's exponent needs no atomics and comes out the same in any order. A block that
// already holds earlier positions keeps the larger of its own exponent and the new numbers'; if that raises it, the earlier
// codes are rounded to it. Rows behind the sequence's last one are left as they are.
#include "fp8.cuh"

namespace llmie {

constexpr int kStoreThreads = 128;

struct StoreArgs {
  unsigned char* k;                  // [pages, n_kv, 64, hd] codes
  unsigned char* v;
  signed char* k_exp;                // [pages, n_kv, 4]
  signed char* v_exp;
  const int* cu_q;
  const int* seq_slot;
  const int* seq_start;
  const int* block_table;
  int max_pages, n_q, n_kv, hd, rot_dim, table_len, write_kv;
  int n_seqs, packed;                // packed: a block's place in the line of all sequences' blocks of 16, instead of one in its sequence's
};

// What a thread block works on: positions [p0, p1) of sequence `seq`, all in one block of 16.
struct StoreBlock {
  int p0, p1, tok0;                  // tok0: row of p0 in the packed step
  int lead;                          // positions of the block that were there before
  size_t row;                        // page * n_kv + head, the page that holds the block
  int in_page;                       // row of the block's first position in its page
};
// Blocks of 16 that a sequence's new positions lie in.
__device__ __forceinline__ int store_blocks(const StoreArgs& a, int seq) {
  const int n_new = a.cu_q[seq + 1] - a.cu_q[seq], start = a.seq_start[seq];
  return n_new > 0 ? (start + n_new - 1) / kExpBlock - start / kExpBlock + 1 : 0;
}
// Finds the sequence whose blocks the block's place in the line lies among, a sequence a thread at a time, and `at`, its place there.
__device__ __forceinline__ bool store_find(const StoreArgs& a, int& seq, int& at) {
  __shared__ int total[kStoreThreads / 32], found[2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, index = blockIdx.x;
  int before = 0;
  if (threadIdx.x == 0) found[0] = -1;
#pragma unroll 1
  for (int s0 = 0; s0 < a.n_seqs; s0 += kStoreThreads) {
    const int s = s0 + threadIdx.x, own = s < a.n_seqs ? store_blocks(a, s) : 0;
    int incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) total[warp] = incl;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < kStoreThreads / 32; ++w) {
      if (w < warp) incl += total[w];
      all += total[w];
    }
    if (before + incl > index && before + incl - own <= index) {
      found[0] = s;
      found[1] = index - before - (incl - own);
    }
    __syncthreads();
    before += all;
    if (before > index) break;
  }
  seq = found[0];
  at = found[1];
  return seq >= 0;
}
__device__ __forceinline__ bool store_block(const StoreArgs& a, int hk, StoreBlock& b) {
  int seq = blockIdx.z, at = blockIdx.x;
  if (a.packed && !store_find(a, seq, at)) return false;
  const int start = a.seq_start[seq], t0 = a.cu_q[seq], n_new = a.cu_q[seq + 1] - t0;
  const int first = (start / kExpBlock + at) * kExpBlock;
  b.p0 = max(start, first);
  b.p1 = min(start + n_new, first + kExpBlock);
  if (b.p0 >= b.p1 || first / kFp8Page >= a.max_pages) return false;
  b.tok0 = t0 + b.p0 - start;
  b.lead = b.p0 - first;
  b.in_page = first % kFp8Page;
  b.row = 0;
  if (a.write_kv) {
    const int page = a.block_table[(size_t)a.seq_slot[seq] * a.max_pages + first / kFp8Page];
    b.row = (size_t)page * a.n_kv + hk;
  }
  return true;
}

// The exponent of a block that holds `lead` earlier positions at `at`; raises it, and lowers the earlier codes, if need be.
// All threads of the block call it; `need`: the bits of the new numbers' largest magnitude.
__device__ __forceinline__ int settle_exponent(signed char* at, unsigned char* codes, int lead, int hd, unsigned need) {
  int e = exponent_for(need);
  if (lead > 0) {
    const int before = clamp_exponent(*at);
    e = max(e, before);
    if (e > before) {
      const float f = lower_factor(before, e);
#pragma unroll 1
      for (int i = threadIdx.x; i < lead * hd / 4; i += kStoreThreads) {
        unsigned* w = reinterpret_cast<unsigned*>(codes) + i;
        *w = lower_codes(*w, f);
      }
    }
  }
  return e;
}

// Every size: any even rotation up to the head size (or none), one number at a time through shared memory.
template <typename T>
__global__ void __launch_bounds__(kStoreThreads)
rope_store_fp8_kernel(const T* qkv, T* __restrict__ q_out, const float2* LLMIE_WEIGHT table, const StoreArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ float staged[];  // [2][16][hd]: the block's new keys and values
  __shared__ unsigned largest[2];
  const int hk = blockIdx.y, G = a.n_q / a.n_kv, hd = a.hd, half = a.rot_dim >> 1;
  StoreBlock b;
  if (!store_block(a, hk, b)) return;
  const int n = b.p1 - b.p0;
  const size_t row_w = (size_t)(a.n_q + 2 * a.n_kv) * hd;
  if (threadIdx.x < 2) largest[threadIdx.x] = 0u;
  __syncthreads();
  // rotated number i of the row x at position p
  auto turned = [&](const T* x, int i, int p) {
    if (!table || i >= a.rot_dim) return to_f32(x[i]);
    const float2 c = table[(size_t)min(p, a.table_len - 1) * half + (i < half ? i : i - half)];
    const float x1 = to_f32(x[i < half ? i : i - half]), x2 = to_f32(x[i < half ? i + half : i]);
    return i < half ? __fsub_rn(__fmul_rn(x1, c.x), __fmul_rn(x2, c.y)) : __fadd_rn(__fmul_rn(x2, c.x), __fmul_rn(x1, c.y));
  };
  for (int it = threadIdx.x; it < n * G * hd; it += kStoreThreads) {
    const int i = it % hd, g = it / hd % G, r = it / hd / G;
    const size_t col = (size_t)(hk * G + g) * hd;
    q_out[(size_t)(b.tok0 + r) * a.n_q * hd + col + i] = from_f32<T>(turned(qkv + (b.tok0 + r) * row_w + col, i, b.p0 + r));
  }
  if (!a.write_kv) return;
  for (int which = 0; which < 2; ++which) {
    unsigned big = 0u;
    for (int it = threadIdx.x; it < n * hd; it += kStoreThreads) {
      const int i = it % hd, r = it / hd;
      const T* x = qkv + (b.tok0 + r) * row_w + (size_t)(a.n_q + which * a.n_kv + hk) * hd;
      const float y = which ? to_f32(x[i]) : turned(x, i, b.p0 + r);
      staged[which * kExpBlock * hd + it] = y;
      big = max(big, finite_magnitude(y));
    }
    atomicMax(&largest[which], big);
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    signed char* at = (which ? a.v_exp : a.k_exp) + b.row * kPageExps + b.in_page / kExpBlock;
    unsigned char* codes = (which ? a.v : a.k) + (b.row * kFp8Page + b.in_page) * hd;
    const int e = settle_exponent(at, codes, b.lead, hd, largest[which]);
    const float f = pow2_of(-e);
    unsigned short* dst = reinterpret_cast<unsigned short*>(codes + (size_t)b.lead * hd);
    const float* src = staged + which * kExpBlock * hd;
    for (int it = threadIdx.x; it < n * hd / 2; it += kStoreThreads) dst[it] = to_e4m3x2(src[2 * it] * f, src[2 * it + 1] * f);
    __syncthreads();                 // everyone has read the old exponent
    if (threadIdx.x == 0) *at = (signed char)e;
  }
}

// Head size 64 or 128, the whole head rotated (or none), rows on 16 bytes: a thread has eight neighbouring columns and their
// partners half a head on, of one position, for all the heads there are; the angles are read once for all of them.
// (2,048 tokens: 47 MB in 12.2 us, 3.9 TB/s, of which about 4 us are what a launch and four loads that wait for one another take. Four
// blocks an SM: three 13.6, 9 pieces of 3 to 700 tokens 6.5 and 6.2; 256 threads a block 15.7 and 7.0.)
template <typename T, int HD>
__global__ void __launch_bounds__(kStoreThreads, 4)
rope_store_fp8_vec_kernel(const T* qkv, T* __restrict__ q_out, const float4* LLMIE_WEIGHT table, const StoreArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kLanes = HD / 16;                            // threads a row
  constexpr int kParts = kStoreThreads / (kExpBlock * kLanes);         // 1: a thread has keys and values; 2: one of them
  __shared__ unsigned largest[2];
  const int hk = blockIdx.y, G = a.n_q / a.n_kv;
  StoreBlock b;
  if (!store_block(a, hk, b)) return;
  const int n = b.p1 - b.p0;
  if (threadIdx.x < 2) largest[threadIdx.x] = 0u;
  __syncthreads();
  const int lane = threadIdx.x % kLanes, row = threadIdx.x / kLanes % kExpBlock, part = threadIdx.x / (kLanes * kExpBlock);
  const bool active = row < n;
  const size_t row_w = (size_t)(a.n_q + 2 * a.n_kv) * HD;
  const T* src = qkv + (size_t)(b.tok0 + (active ? row : 0)) * row_w + lane * 8;
  float c[8], s[8];
  if (table) {
    const float4* cs = table + ((size_t)min(b.p0 + row, a.table_len - 1) * (HD / 2) + lane * 8) / 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = cs[i];
      c[2 * i] = v.x;
      s[2 * i] = v.y;
      c[2 * i + 1] = v.z;
      s[2 * i + 1] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = 1.f;
      s[i] = 0.f;
    }
  }
  auto turn = [&](float (&x)[8], float (&y)[8]) {
    if (!table) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float u = x[i], v = y[i];
      x[i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(v, s[i]));
      y[i] = __fadd_rn(__fmul_rn(v, c[i]), __fmul_rn(u, s[i]));
    }
  };
  // keys and values: which of them this thread has, as numbers. They are asked for before the queries are worked on.
  float x[3 - kParts][2][8];
  if (a.write_kv) {
#pragma unroll
    for (int i = 0; i < 3 - kParts; ++i) {
      const T* p = src + (size_t)(a.n_q + (kParts == 1 ? i : part) * a.n_kv + hk) * HD;
      load8(p, x[i][0]);
      load8(p + HD / 2, x[i][1]);
    }
  }
  if (active) {
    T* dst = q_out + (size_t)(b.tok0 + row) * a.n_q * HD + lane * 8;
    // four heads are asked for before one is worked on (2,048 tokens, 32 / 8 heads of 128: 14.5 us one by one, 12.2 so, with two 12.9; a
    // token of each of 64 sequences 4.4, 4.0, 4.3)
#pragma unroll 1
    for (int g0 = part; g0 < G; g0 += 4 * kParts) {
      float u[4][8], v[4][8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int g = min(g0 + k * kParts, G - 1);
        const size_t col = (size_t)(hk * G + g) * HD;
        load8(src + col, u[k]);
        load8(src + col + HD / 2, v[k]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int g = g0 + k * kParts;
        if (g >= G) break;
        const size_t col = (size_t)(hk * G + g) * HD;
        turn(u[k], v[k]);
        store8(dst + col, u[k]);
        store8(dst + col + HD / 2, v[k]);
      }
    }
  }
  if (a.write_kv) {
#pragma unroll
    for (int i = 0; i < 3 - kParts; ++i) {
      const int which = kParts == 1 ? i : part;
      if (which == 0) turn(x[i][0], x[i][1]);
      unsigned big = 0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) big = max(big, max(finite_magnitude(x[i][0][e]), finite_magnitude(x[i][1][e])));
      big = __reduce_max_sync(0xffffffffu, active ? big : 0u);
      if ((threadIdx.x & 31) == 0) atomicMax(&largest[which], big);
    }
  }
  if (!a.write_kv) return;
  __syncthreads();
  int e[2];
#pragma unroll
  for (int which = 0; which < 2; ++which)
    e[which] = settle_exponent((which ? a.v_exp : a.k_exp) + b.row * kPageExps + b.in_page / kExpBlock,
                               (which ? a.v : a.k) + (b.row * kFp8Page + b.in_page) * HD, b.lead, HD, largest[which]);
  if (active) {
#pragma unroll
    for (int i = 0; i < 3 - kParts; ++i) {
      const int which = kParts == 1 ? i : part;
      const float f = pow2_of(-(which ? e[1] : e[0]));
      unsigned char* dst = (which ? a.v : a.k) + (b.row * kFp8Page + b.in_page + b.lead + row) * HD + lane * 8;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        unsigned w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          w[j] = (unsigned)to_e4m3x2(x[i][h][4 * j] * f, x[i][h][4 * j + 1] * f) |
                 ((unsigned)to_e4m3x2(x[i][h][4 * j + 2] * f, x[i][h][4 * j + 3] * f) << 16);
        *reinterpret_cast<uint2*>(dst + h * (HD / 2)) = make_uint2(w[0], w[1]);
      }
    }
  }
  if (b.lead > 0) __syncthreads();   // everyone has read the old exponents
  if (threadIdx.x < 2) (threadIdx.x ? a.v_exp : a.k_exp)[b.row * kPageExps + b.in_page / kExpBlock] = (signed char)(threadIdx.x ? e[1] : e[0]);
}

template <typename T>
static int launch_store(const void* qkv, void* q_out, const float2* table, const StoreArgs& a, dim3 grid, cudaStream_t stream) {
  const bool vec = (a.rot_dim == a.hd || !table) && aligned16(qkv) && aligned16(q_out) && aligned16(table);
  if (vec && (a.hd == 64 || a.hd == 128)) {
    if (a.hd == 64)
      launch_k(rope_store_fp8_vec_kernel<T, 64>, grid, dim3(kStoreThreads), 0, stream, (const T*)qkv,
               (T*)q_out, (const float4*)table, a);
    else
      launch_k(rope_store_fp8_vec_kernel<T, 128>, grid, dim3(kStoreThreads), 0, stream, (const T*)qkv,
               (T*)q_out, (const float4*)table, a);
    LLMIE_LAUNCH_CHECK();
    return LLMIE_OK;
  }
  const size_t smem = (size_t)2 * kExpBlock * a.hd * sizeof(float);
  launch_k(rope_store_fp8_kernel<T>, grid, dim3(kStoreThreads), smem, stream, (const T*)qkv, (T*)q_out,
           table, a);
  LLMIE_LAUNCH_CHECK();
  return LLMIE_OK;
}

}  // namespace llmie

using namespace llmie;

// qkv [T, (n_q + 2 n_kv) hd], q_out [T, n_q hd] of one type; caches e4m3 [pages, n_kv, 64, hd] with exponents int8 [pages, n_kv,
// 4]; table float32 [table_len, rot_dim / 2, 2] or null (no rotation). cu_q [n_seqs + 1], seq_slot, seq_start [n_seqs]:
// sequence i brings rows cu_q[i] .. cu_q[i + 1] - 1, at positions from seq_start[i] on. n_tokens: rows of qkv; max_q_len: the most that one brings.
extern "C" int llmie_rope_store_fp8(const void* qkv, void* q_out, void* k_cache, void* v_cache, void* k_exp, void* v_exp,
                                    const float* table, const int* cu_q, const int* seq_slot, const int* seq_start,
                                    const int* block_table, int max_pages, int n_tokens, int n_seqs, int max_q_len, int n_q,
                                    int n_kv, int hd, int rot_dim, int table_len, int write_kv, int dtype, cudaStream_t stream) {
  if (n_tokens < 0 || n_seqs < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0) return LLMIE_ERR_BAD_ARG;
  if (hd < 16 || hd > 256 || hd % 16) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (table && (rot_dim <= 0 || rot_dim % 2 || rot_dim > hd || table_len <= 0)) return LLMIE_ERR_BAD_ARG;
  if (write_kv && (!aligned16(k_cache) || !aligned16(v_cache))) return LLMIE_ERR_ALIGNMENT;
  if (table && (reinterpret_cast<uintptr_t>(table) & 7u)) return LLMIE_ERR_ALIGNMENT;
  if (n_tokens == 0 || n_seqs == 0 || max_q_len <= 0) return LLMIE_OK;
  if (n_kv > 65535) return LLMIE_ERR_UNSUPPORTED_SIZE;
  StoreArgs a{(unsigned char*)k_cache, (unsigned char*)v_cache, (signed char*)k_exp, (signed char*)v_exp, cu_q, seq_slot,
                    seq_start, block_table, max_pages, n_q, n_kv, hd, table ? rot_dim : 0, table_len, write_kv ? 1 : 0, n_seqs, 0};
  // A run of L positions lies in at most (L + 14) / 16 + 1 blocks of 16. A block finds its sequence by its index, or, where most
  // sequences bring much less than the longest, by the lengths. (A prompt of 2,048 tokens
  // beside 63 single ones, 32 / 8 heads of 128: 75.9 us by index, 14.2 by the lengths; 9 pieces of 3 to 700 tokens 6.95 and 6.66.)
  const long long longest = (max_q_len + kExpBlock - 2) / kExpBlock + 1, line = (long long)n_tokens / kExpBlock + 2LL * n_seqs;
  a.packed = longest * n_seqs > 2 * line || n_seqs > 65535 ? 1 : 0;
  if (line > 0x7fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  const dim3 grid = a.packed ? dim3((unsigned)line, n_kv, 1) : dim3((unsigned)longest, n_kv, n_seqs);
  if (dtype == LLMIE_F32) return launch_store<float>(qkv, q_out, (const float2*)table, a, grid, stream);
  if (dtype == LLMIE_BF16) return launch_store<__nv_bfloat16>(qkv, q_out, (const float2*)table, a, grid, stream);
  return LLMIE_ERR_DTYPE;
}

// The same by one address, with the arguments one behind another as they are above: a caller from another language converts one
// argument instead of 23, which takes as long as the launch.
struct RopeStoreCall {
  const void* qkv;
  void *q_out, *k_cache, *v_cache, *k_exp, *v_exp;
  const float* table;
  const int *cu_q, *seq_slot, *seq_start, *block_table;
  int max_pages, n_tokens, n_seqs, max_q_len, n_q, n_kv, hd, rot_dim, table_len, write_kv, dtype;
  cudaStream_t stream;
};
extern "C" int llmie_rope_store_fp8_call(const RopeStoreCall* c) {
  return llmie_rope_store_fp8(c->qkv, c->q_out, c->k_cache, c->v_cache, c->k_exp, c->v_exp, c->table, c->cu_q, c->seq_slot, c->seq_start,
                              c->block_table, c->max_pages, c->n_tokens, c->n_seqs, c->max_q_len, c->n_q, c->n_kv, c->hd, c->rot_dim,
                              c->table_len, c->write_kv, c->dtype, c->stream);
}
