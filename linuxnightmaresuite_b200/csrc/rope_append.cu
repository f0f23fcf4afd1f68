// Position rotation of q and k, and the append of k and v to a paged cache.
//
// With a = position * inv_freq[i] a pair (x1, x2) becomes
//   (x1 cos a - x2 sin a, x2 cos a + x1 sin a).
// The angle is formed and reduced to [-pi, pi] in 64 bits (a position of 2^20
// leaves an f32 angle with errors of a tenth), sin and cos are f32.
//
// One CTA per (token, part of its heads): the CTA computes the token's rot / 2
// (cos, sin) pairs once into shared memory, then its threads walk the pairs of
// its heads.  Bound by memory for prompts, by latency for single tokens.
#include <math.h>

#include "paged_cache.cuh"

namespace moe {

constexpr int kRopeThreads = 256;

struct RopeArgs {
  moe_paged_cache c;
  const float *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, qo_ts, qo_hs;
  float* q_out;
  const int32_t *positions, *seq_ids;
  const double* inv_freq;
  int* status;
  int hq, rot, interleaved;
};

__device__ __forceinline__ float2 rope_cos_sin(int pos, double freq) {
  const double kTwoPi = 6.283185307179586476925;
  const double a = (double)pos * freq;
  const double r = a - kTwoPi * rint(a / kTwoPi);
  const float hi = (float)r;
  const float lo = (float)(r - (double)hi);   // what the f32 angle leaves out
  float s, c;
  sincosf(hi, &s, &c);
  return make_float2(fmaf(-s, lo, c), fmaf(c, lo, s));
}

__device__ __forceinline__ void cache_put(__half* p, float x, float) { *p = __float2half_rn(x); }
__device__ __forceinline__ void cache_put(__nv_bfloat16* p, float x, float) {
  *p = __float2bfloat16_rn(x);
}
__device__ __forceinline__ void cache_put(__nv_fp8_e4m3* p, float x, float scale) {
  p->__x = __nv_cvt_float_to_fp8(__fdiv_rn(x, scale), __NV_SATFINITE, __NV_E4M3);
}

template <int DT>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeArgs A) {
  using T = typename CacheType<DT>::T;
  __shared__ float2 cs[kMaxHeadDim / 2];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x;
  const int pos = A.positions[t];
  if (pos < 0) return;
  const int seq = A.seq_ids ? A.seq_ids[t] : t;
  int64_t slot = -1;   // the token's slot in both caches, -1: none
  if (seq >= 0 && seq < A.c.seqs && pos / A.c.page_size < A.c.table_width) {
    const int page = A.c.block_table[(int64_t)seq * A.c.table_stride + pos / A.c.page_size];
    if (page >= 0 && page < A.c.pages)
      slot = (int64_t)page * A.c.page_stride + (int64_t)(pos % A.c.page_size) * A.c.token_stride;
  }
  if (slot < 0 && threadIdx.x == 0) set_status(A.status, MOE_STATUS_BAD_PAGE);
  const int h = A.rot / 2;
  for (int i = threadIdx.x; i < h; i += blockDim.x) cs[i] = rope_cos_sin(pos, A.inv_freq[i]);
  __syncthreads();
  const int half = A.c.head_dim / 2;                 // pairs per head
  const int heads = A.hq + 2 * A.c.kv_heads;
  for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < heads * half;
       it += gridDim.y * blockDim.x) {
    int j = it / half;
    const int i = it - j * half;
    const bool turn = j < A.hq + A.c.kv_heads && i < h;
    const int e0 = turn && !A.interleaved ? i : 2 * i;
    const int e1 = turn && !A.interleaved ? i + h : 2 * i + 1;
    const float* src;
    if (j < A.hq) {
      src = A.q + t * A.q_ts + j * A.q_hs;
    } else if (j < A.hq + A.c.kv_heads) {
      src = A.k + t * A.k_ts + (j - A.hq) * A.k_hs;
    } else {
      src = A.v + t * A.v_ts + (j - A.hq - A.c.kv_heads) * A.v_hs;
    }
    float x0 = src[e0], x1 = src[e1];
    if (turn) {
      const float2 w = cs[i];
      const float y0 = fmaf(x0, w.x, -x1 * w.y);
      x1 = fmaf(x1, w.x, x0 * w.y);
      x0 = y0;
    }
    if (j < A.hq) {
      float* dst = A.q_out + t * A.qo_ts + j * A.qo_hs;
      dst[e0] = x0;
      dst[e1] = x1;
    } else if (slot >= 0) {
      j -= A.hq;
      const bool is_k = j < A.c.kv_heads;
      T* dst = static_cast<T*>(is_k ? A.c.k : A.c.v) + slot +
               (int64_t)(is_k ? j : j - A.c.kv_heads) * A.c.head_stride;
      const float scale = is_k ? A.c.k_scale : A.c.v_scale;
      cache_put(dst + e0, x0, scale);
      cache_put(dst + e1, x1, scale);
    }
  }
}

}  // namespace moe

extern "C" {

int moe_rope_append(const moe_paged_cache* cache, const float* q, int64_t q_tok_stride,
                    int64_t q_head_stride, const float* k, int64_t k_tok_stride,
                    int64_t k_head_stride, const float* v, int64_t v_tok_stride,
                    int64_t v_head_stride, int T, int q_heads, const int32_t* positions,
                    const int32_t* seq_ids, const double* inv_freq, int rot, int interleaved,
                    float* q_out, int64_t qo_tok_stride, int64_t qo_head_stride, int32_t* status,
                    moe_stream_t stream) {
  MOE_REQUIRE(cache, MOE_ERR_INVALID, "null cache");
  MOE_CHECK(moe::check_cache(*cache));
  MOE_REQUIRE(T >= 0 && q_heads >= 0, MOE_ERR_INVALID, "negative size");
  MOE_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= cache->head_dim, MOE_ERR_INVALID,
              "rot %d: an even number up to head_dim %d is needed", rot, cache->head_dim);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(k && v && positions && (rot == 0 || inv_freq), MOE_ERR_INVALID, "null pointer");
  MOE_REQUIRE(q_heads == 0 || (q && q_out), MOE_ERR_INVALID, "null q or q_out");
  MOE_REQUIRE(seq_ids || T <= cache->seqs, MOE_ERR_INVALID,
              "%d tokens for %d sequences need seq_ids", T, cache->seqs);
  moe::RopeArgs a = {*cache, q, k, v, q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                     v_tok_stride, v_head_stride, qo_tok_stride, qo_head_stride, q_out, positions,
                     seq_ids, inv_freq, status, q_heads, rot, interleaved};
  moe::normalise_strides(a.c);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  dim3 grid((unsigned)T, 1);
  {
    ::moe::ProfScope _prof(MOE_K_ROPE_APPEND, s);
    auto kern = cache->dtype == MOE_CACHE_F16    ? moe::rope_append_kernel<MOE_CACHE_F16>
                : cache->dtype == MOE_CACHE_BF16 ? moe::rope_append_kernel<MOE_CACHE_BF16>
                                                 : moe::rope_append_kernel<MOE_CACHE_E4M3>;
    MOE_CUDA(moe::launch_pdl(kern, grid, dim3(moe::kRopeThreads), 0, s, a));
  }
  return moe::check_launch("rope_append");
}

}  // extern "C"
