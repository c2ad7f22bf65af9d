// Plain attention over a paged cache in 8 bits (fp8.cuh), for any number of new tokens a sequence, any head size that is a
// multiple of 16 up to 256, float32 and bfloat16: the kernel that every call can go to, and the one that the tensor-core
// kernels of such a cache are checked against.
//
//   o_t = sum_j w_tj v_j / sum_j w_tj,   w_tj = exp(scale q_t . k_j - max_j),   j over the keys that token t sees
//
// One warp per (token, query head): a key a lane for the scores, a run of columns a lane for the sum over the values. All in
// float32; a block's two exponents multiply the score and the weight. Keys that a token does not see are not read. The sums over the
// values are kept 2^24 smaller: of 2^16 values near the largest number there is, the sum is not infinite where the mean is none.
#include "fp8.cuh"
#include <math.h>

namespace llmie {

constexpr int kPlainWarps = 4;
constexpr int kPlainHd = 256;
constexpr int kPlainDown = 24;

template <typename T>
__global__ void __launch_bounds__(kPlainWarps * 32)
attention_paged_fp8_kernel(const T* q, const unsigned char* k_cache, const unsigned char* v_cache, const signed char* k_exp,
                           const signed char* v_exp, T* __restrict__ out, const int* tok_pos, const int* tok_seq,
                           const int* seq_slot, const int* block_table, int max_pages, int n_items, int n_q, int n_kv, int hd,
                           float scale, int window) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float q_smem[kPlainWarps][kPlainHd];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kPlainWarps + warp;
  if (item >= n_items) return;       // whole warps: no barrier of the block below
  const int t = (int)(item / n_q), h = (int)(item % n_q), hk = h / (n_q / n_kv);
  const int pos = min(tok_pos[t], max_pages * kFp8Page - 1);           // what the table has room for
  const int* pages = block_table + (size_t)seq_slot[tok_seq[t]] * max_pages;
  const int lo = first_visible_key(pos, window);
  float* qs = q_smem[warp];
  for (int i = lane; i < hd; i += 32) qs[i] = to_f32(q[((size_t)t * n_q + h) * hd + i]) * scale;
  __syncwarp();
  constexpr int kAcc = kPlainHd / 32;
  float acc[kAcc];
#pragma unroll
  for (int i = 0; i < kAcc; ++i) acc[i] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int base = lo; base <= pos; base += 32) {
    const int j = base + lane;
    float s = -INFINITY, ev = 0.f;
    long long row = 0;
    if (j <= pos) {
      const long long pr = (long long)pages[j / kFp8Page] * n_kv + hk;
      const int in = j % kFp8Page;
      row = pr * kFp8Page + in;
      const uint4* kr = reinterpret_cast<const uint4*>(k_cache + row * hd);
      float dot = 0.f;
      for (int c = 0; c < hd / 16; ++c) {
        const uint4 w4 = kr[c];
        const unsigned w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 a = e4m3x2_to_float2((unsigned short)(w[i] & 0xffffu)), b = e4m3x2_to_float2((unsigned short)(w[i] >> 16));
          const float* x = qs + c * 16 + i * 4;
          dot = fmaf(x[0], a.x, dot);
          dot = fmaf(x[1], a.y, dot);
          dot = fmaf(x[2], b.x, dot);
          dot = fmaf(x[3], b.y, dot);
        }
      }
      s = dot * pow2_of(clamp_exponent(k_exp[pr * kPageExps + in / kExpBlock]));
      ev = pow2_of(clamp_exponent(v_exp[pr * kPageExps + in / kExpBlock]) - kPlainDown);
    }
    const float m_new = fmaxf(m, warp_max(s));
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float p = j <= pos ? expf(s - m_use) : 0.f;
    const float alpha = expf(m - m_use);
    l = l * alpha + warp_sum(p);
    m = m_new;
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[i] *= alpha;
    const float pv = p * ev;
    const int n_here = min(32, pos - base + 1);
    for (int jj = 0; jj < n_here; ++jj) {
      const float pj = __shfl_sync(0xffffffffu, pv, jj);
      const long long rj = __shfl_sync(0xffffffffu, row, jj);
#pragma unroll
      for (int i = 0; i < kAcc / 2; ++i) {
        const int d = 2 * lane + 64 * i;
        if (d < hd) {
          const float2 x = e4m3x2_to_float2(*reinterpret_cast<const unsigned short*>(v_cache + rj * hd + d));
          acc[2 * i] = fmaf(pj, x.x, acc[2 * i]);
          acc[2 * i + 1] = fmaf(pj, x.y, acc[2 * i + 1]);
        }
      }
    }
  }
  T* o = out + ((size_t)t * n_q + h) * hd;
  const bool none = lo > pos;        // a position below zero: a lane without a sequence
#pragma unroll
  for (int i = 0; i < kAcc / 2; ++i) {
    const int d = 2 * lane + 64 * i;
    if (d < hd) {
      o[d] = from_f32<T>(none ? 0.f : acc[2 * i] / l * pow2_of(kPlainDown));
      o[d + 1] = from_f32<T>(none ? 0.f : acc[2 * i + 1] / l * pow2_of(kPlainDown));
    }
  }
}

}  // namespace llmie

using namespace llmie;

// q, out [T, n_q hd]; caches e4m3 [pages, n_kv, 64, hd] with exponents int8 [pages, n_kv, 4]; window as in the other attention
// kernels: 0 every earlier key, n > 0 the last n, -n < 0 the token's own chunk of n positions.
extern "C" int llmie_attention_paged_fp8(const void* q, const void* k_cache, const void* v_cache, const void* k_exp,
                                         const void* v_exp, void* out, const int* tok_pos, const int* tok_seq,
                                         const int* seq_slot, const int* block_table, int max_pages, int n_tokens, int n_q,
                                         int n_kv, int hd, float scale, int window, int dtype, cudaStream_t stream) {
  if (n_tokens < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv || max_pages <= 0) return LLMIE_ERR_BAD_ARG;
  if (max_pages > kMostPages) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (hd < 16 || hd > kPlainHd || hd % 16) return LLMIE_ERR_UNSUPPORTED_SIZE;
  if (!aligned16(k_cache) || !aligned16(v_cache)) return LLMIE_ERR_ALIGNMENT;
  if (n_tokens == 0) return LLMIE_OK;
  const long long items = (long long)n_tokens * n_q;
  if (items > 0x7fffffffLL) return LLMIE_ERR_UNSUPPORTED_SIZE;
  const dim3 grid((unsigned)((items + kPlainWarps - 1) / kPlainWarps)), block(kPlainWarps * 32);
  if (dtype == LLMIE_F32)
    launch_k(attention_paged_fp8_kernel<float>, grid, block, 0, stream, (const float*)q, (const unsigned char*)k_cache,
             (const unsigned char*)v_cache, (const signed char*)k_exp, (const signed char*)v_exp, (float*)out, tok_pos, tok_seq,
             seq_slot, block_table, max_pages, (int)items, n_q, n_kv, hd, scale, window);
  else if (dtype == LLMIE_BF16)
    launch_k(attention_paged_fp8_kernel<__nv_bfloat16>, grid, block, 0, stream, (const __nv_bfloat16*)q,
             (const unsigned char*)k_cache, (const unsigned char*)v_cache, (const signed char*)k_exp, (const signed char*)v_exp,
             (__nv_bfloat16*)out, tok_pos, tok_seq, seq_slot, block_table, max_pages, (int)items, n_q, n_kv, hd, scale, window);
  else
    return LLMIE_ERR_DTYPE;
  LLMIE_LAUNCH_CHECK();
  return LLMIE_OK;
}
