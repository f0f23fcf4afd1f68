// Attention of one new token per sequence over a paged cache.
//
// First form: one CTA per (sequence, query head), four warps taking keys in
// turn, each with its own running maximum and sum; joined in shared memory.
#include <math.h>

#include "paged_cache.cuh"

namespace moe {

constexpr int kAttWarps = 4;

struct AttArgs {
  moe_paged_cache c;
  const float* q;
  int64_t q_ss, q_hs;
  const int32_t* seq_lens;
  float *out, *lse;
  int* status;
  int hq, window;
  float scale, cap;
};

template <int DT>
__global__ void __launch_bounds__(kAttWarps * 32) attention_kernel(const AttArgs A) {
  using T = typename CacheType<DT>::T;
  __shared__ float sm[kAttWarps], sl[kAttWarps], so[kAttWarps][kMaxHeadDim];
  pdl_trigger();
  pdl_wait();
  const int s = blockIdx.y, h = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int D = A.c.head_dim, kvh = h / (A.hq / A.c.kv_heads);
  int len = A.seq_lens[s];
  const int most = A.c.table_width * A.c.page_size;
  if (len > most) {
    if (threadIdx.x == 0) set_status(A.status, MOE_STATUS_BAD_PAGE);
    len = most;
  }
  const int first = A.window > 0 && len > A.window ? len - A.window : 0;
  float q[kMaxHeadDim / 32], o[kMaxHeadDim / 32];
#pragma unroll
  for (int i = 0; i < kMaxHeadDim / 32; ++i) {
    o[i] = 0.f;
    q[i] = 32 * i + lane < D ? A.q[s * A.q_ss + h * A.q_hs + 32 * i + lane] : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = first + warp; j < len; j += kAttWarps) {
    const int page = A.c.block_table[(int64_t)s * A.c.table_stride + j / A.c.page_size];
    if (page < 0 || page >= A.c.pages) {
      if (lane == 0) set_status(A.status, MOE_STATUS_BAD_PAGE);
      continue;
    }
    const int64_t at = (int64_t)page * A.c.page_stride +
                       (int64_t)(j % A.c.page_size) * A.c.token_stride +
                       (int64_t)kvh * A.c.head_stride;
    const T* k = static_cast<const T*>(A.c.k) + at;
    const T* v = static_cast<const T*>(A.c.v) + at;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
      if (32 * i + lane < D) x = fmaf(q[i], (float)k[32 * i + lane], x);
#pragma unroll
    for (int b = 16; b > 0; b >>= 1) x += __shfl_xor_sync(0xffffffffu, x, b);
    x *= A.scale * A.c.k_scale;
    if (A.cap > 0.f) x = A.cap * tanhf(x / A.cap);
    const float mn = fmaxf(m, x);
    const float keep = m == -INFINITY ? 0.f : expf(m - mn), p = expf(x - mn);
    m = mn;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
      if (32 * i + lane < D) o[i] = fmaf(p, (float)v[32 * i + lane], o[i] * keep);
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  for (int i = 0; i < kMaxHeadDim / 32; ++i) so[warp][32 * i + lane] = o[i];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < kAttWarps; ++w) M = fmaxf(M, sm[w]);
  float L = 0.f;
  for (int w = 0; w < kAttWarps; ++w) L += M == -INFINITY ? 0.f : sl[w] * expf(sm[w] - M);
  for (int i = threadIdx.x; i < D; i += blockDim.x) {
    float y = 0.f;
    for (int w = 0; w < kAttWarps; ++w)
      y += M == -INFINITY ? 0.f : so[w][i] * expf(sm[w] - M);
    A.out[((int64_t)s * A.hq + h) * D + i] = L > 0.f || L != L ? y / L * A.c.v_scale : 0.f;
  }
  if (threadIdx.x == 0 && A.lse) A.lse[(int64_t)s * A.hq + h] = M + logf(L);
}

}  // namespace moe

extern "C" {

int moe_paged_attention_workspace_bytes(int seqs, int q_heads, int kv_heads, int head_dim,
                                        size_t* bytes) {
  MOE_REQUIRE(bytes, MOE_ERR_INVALID, "null output pointer");
  MOE_REQUIRE(seqs >= 0 && kv_heads > 0 && head_dim > 0 && head_dim <= moe::kMaxHeadDim,
              MOE_ERR_INVALID, "bad attention shape");
  MOE_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0, MOE_ERR_INVALID,
              "%d query heads for %d key heads", q_heads, kv_heads);
  *bytes = 256;
  return MOE_OK;
}

int moe_paged_attention(const moe_paged_cache* cache, const float* q, int64_t q_seq_stride,
                        int64_t q_head_stride, const int32_t* seq_lens, int q_heads, int max_len,
                        int window, float scale, float softcap, float* out, float* lse,
                        void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  MOE_REQUIRE(cache, MOE_ERR_INVALID, "null cache");
  MOE_CHECK(moe::check_cache(*cache));
  MOE_REQUIRE(q_heads > 0 && q_heads % cache->kv_heads == 0, MOE_ERR_INVALID,
              "%d query heads for %d key heads", q_heads, cache->kv_heads);
  MOE_REQUIRE(max_len >= 0 && window >= 0, MOE_ERR_INVALID, "negative length or window");
  MOE_REQUIRE(isfinite(scale) && isfinite(softcap) && softcap >= 0.f, MOE_ERR_INVALID,
              "scale and softcap must be finite, softcap >= 0");
  if (cache->seqs == 0) return MOE_OK;
  MOE_REQUIRE(q && seq_lens && out && workspace, MOE_ERR_INVALID, "null pointer");
  size_t need = 0;
  MOE_CHECK(moe_paged_attention_workspace_bytes(cache->seqs, q_heads, cache->kv_heads,
                                                cache->head_dim, &need));
  MOE_REQUIRE(workspace_bytes >= need, MOE_ERR_WORKSPACE, "workspace %zu < %zu bytes",
              workspace_bytes, need);
  moe::AttArgs a = {*cache, q, q_seq_stride, q_head_stride, seq_lens, out, lse,
                    static_cast<int*>(workspace), q_heads, window, scale, softcap};
  moe::normalise_strides(a.c);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  {
    ::moe::ProfScope _prof(MOE_K_ATTENTION, s);
    auto kern = cache->dtype == MOE_CACHE_F16    ? moe::attention_kernel<MOE_CACHE_F16>
                : cache->dtype == MOE_CACHE_BF16 ? moe::attention_kernel<MOE_CACHE_BF16>
                                                 : moe::attention_kernel<MOE_CACHE_E4M3>;
    MOE_CUDA(moe::launch_pdl(kern, dim3((unsigned)q_heads, (unsigned)cache->seqs),
                             dim3(moe::kAttWarps * 32), 0, s, a));
  }
  return moe::check_launch("paged_attention");
}

}  // extern "C"
