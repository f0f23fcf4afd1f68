// Position rotation of q and k, and the append of k and v to a paged cache.
//
// With a = position * inv_freq[i] a pair (x1, x2) becomes
//   (x1 cos a - x2 sin a, x2 cos a + x1 sin a).
// The angle is formed and reduced to [-pi, pi] in 64 bits (a position of 2^20
// leaves an f32 angle with errors of a tenth), sin and cos are f32.
//
// One CTA per (token, part of its heads): the CTA computes the token's rot / 2
// (cos, sin) pairs once into shared memory, one thread follows the page table to
// the token's slot, then all walk the heads four elements at a time.  Bound by
// memory for prompts (8191 tokens, 32 + 2 x 8 heads of 128: 65.5 us for 0.37 GB, 86 %
// of the copy bandwidth; the rest is the latency of position, page and slot,
// which the resident CTAs of an SM do not hide altogether), by latency for single
// tokens (2.0 us).
#include <math.h>

#include <algorithm>

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
  int nr, ni, nv;                      // items: rotated and all of a turned head, of a value head
  uint32_t mi, mv;                     // 2^32 / ni, 2^32 / nv rounded up: it / ni = hi(it * mi),
};                                     // exact for it < 2^24 since ni, nv <= 256

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

// Four elements at a time; VEC 1 takes them one by one (rows that are not
// aligned to 16 bytes, rotations that end inside four elements).
template <int VEC> struct Elems { float v[VEC]; };

template <int VEC>
__device__ __forceinline__ Elems<VEC> load_elems(const float* p) {
  Elems<VEC> e;
  if (VEC == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    e.v[0] = f.x;
    e.v[1 % VEC] = f.y;
    e.v[2 % VEC] = f.z;
    e.v[3 % VEC] = f.w;
  } else {
    e.v[0] = *p;
  }
  return e;
}
template <int VEC>
__device__ __forceinline__ void store_f32(float* p, const Elems<VEC>& e) {
  if (VEC == 4)
    *reinterpret_cast<float4*>(p) = make_float4(e.v[0], e.v[1 % VEC], e.v[2 % VEC], e.v[3 % VEC]);
  else
    *p = e.v[0];
}
template <int VEC, typename T>
__device__ __forceinline__ void store_cache(T* p, const Elems<VEC>& e, float scale) {
  struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; } out;
#pragma unroll
  for (int i = 0; i < VEC; ++i) cache_put(&out.v[i], e.v[i], scale);
  *reinterpret_cast<Pack*>(p) = out;
}

// An item is one load, or for a pair half a head apart two.
template <int DT, int VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const RopeArgs A) {
  using T = typename CacheType<DT>::T;
  __shared__ float2 cs[kMaxHeadDim / 2];
  __shared__ int64_t sh_slot;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x;
  const int pos = A.positions[t];
  if (pos < 0) return;
  if (threadIdx.x == blockDim.x - 1) {           // the token's slot in both caches, -1: none
    const int seq = A.seq_ids ? A.seq_ids[t] : t, n = pos / A.c.page_size;
    int64_t slot = -1;
    if (seq >= 0 && seq < A.c.seqs && n < A.c.table_width) {
      const int page = A.c.block_table[(int64_t)seq * A.c.table_stride + n];
      if (page >= 0 && page < A.c.pages)
        slot = (int64_t)page * A.c.page_stride +
               (int64_t)(pos - n * A.c.page_size) * A.c.token_stride;
    }
    if (slot < 0) set_status(A.status, MOE_STATUS_BAD_PAGE);
    sh_slot = slot;
  }
  const int h = A.rot / 2;
  for (int i = threadIdx.x; i < h; i += blockDim.x) cs[i] = rope_cos_sin(pos, A.inv_freq[i]);
  __syncthreads();
  const int64_t slot = sh_slot;
  // items of a head: of the rotated half (h / VEC), or of all rotated elements
  // where pairs are adjacent, then of the rest
  const int hk = A.c.kv_heads, nr = A.nr, ni = A.ni, nv = A.nv;
  const int turned = (A.hq + hk) * ni, total = turned + hk * nv;
  for (int it = blockIdx.y * blockDim.x + threadIdx.x; it < total; it += gridDim.y * blockDim.x) {
    if (it >= turned) {                        // a value: copied
      const int k = it - turned, j = nv == 1 ? k : (int)__umulhi((uint32_t)k, A.mv);
      const int e = (k - j * nv) * VEC;
      if (slot >= 0)
        store_cache<VEC>(static_cast<T*>(A.c.v) + slot + (int64_t)j * A.c.head_stride + e,
                         load_elems<VEC>(A.v + t * A.v_ts + j * A.v_hs + e), A.c.v_scale);
      continue;
    }
    const int j = ni == 1 ? it : (int)__umulhi((uint32_t)it, A.mi), i = it - j * ni;
    const bool is_q = j < A.hq;
    const float* src = is_q ? A.q + t * A.q_ts + j * A.q_hs : A.k + t * A.k_ts + (j - A.hq) * A.k_hs;
    const int e0 = i < nr ? i * VEC : A.rot + (i - nr) * VEC;
    const bool two = i < nr && (!A.interleaved || VEC == 1);
    const int e1 = A.interleaved ? e0 + 1 : e0 + h;   // partner, in another load
    Elems<VEC> a, b;
    if (VEC == 1 && A.interleaved && i < nr) {
      if (i & 1) continue;                     // its pair's first element does both
    }
    a = load_elems<VEC>(src + e0);
    if (two) {
      b = load_elems<VEC>(src + e1);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float2 w = cs[A.interleaved ? e0 / 2 : e0 + k];
        const float x0 = a.v[k], x1 = b.v[k];
        a.v[k] = fmaf(x0, w.x, -x1 * w.y);
        b.v[k] = fmaf(x1, w.x, x0 * w.y);
      }
    } else if (i < nr) {
#pragma unroll
      for (int k = 0; k + 1 < VEC; k += 2) {
        const float2 w = cs[(e0 + k) / 2];
        const float x0 = a.v[k], x1 = a.v[k + 1];
        a.v[k] = fmaf(x0, w.x, -x1 * w.y);
        a.v[k + 1] = fmaf(x1, w.x, x0 * w.y);
      }
    }
    if (is_q) {
      float* dst = A.q_out + t * A.qo_ts + j * A.qo_hs;
      store_f32<VEC>(dst + e0, a);
      if (two) store_f32<VEC>(dst + e1, b);
    } else if (slot >= 0) {
      T* dst = static_cast<T*>(A.c.k) + slot + (int64_t)(j - A.hq) * A.c.head_stride;
      store_cache<VEC>(dst + e0, a, A.c.k_scale);
      if (two) store_cache<VEC>(dst + e1, b, A.c.k_scale);
    }
  }
}

template <int DT>
static int launch_rope(RopeArgs& a, int T, cudaStream_t s) {
  auto aligned = [](const void* p, int64_t ts, int64_t hs) {
    return (uintptr_t)p % 16 == 0 && ts % 4 == 0 && hs % 4 == 0;
  };
  const bool vec = a.rot % (a.interleaved ? 4 : 8) == 0 && aligned(a.k, a.k_ts, a.k_hs) &&
                   aligned(a.v, a.v_ts, a.v_hs) &&
                   (a.hq == 0 || (aligned(a.q, a.q_ts, a.q_hs) && aligned(a.q_out, a.qo_ts, a.qo_hs)));
  const int V = vec ? 4 : 1;
  a.nr = a.interleaved ? a.rot / V : a.rot / 2 / V;
  a.ni = a.nr + (a.c.head_dim - a.rot) / V;
  a.nv = a.c.head_dim / V;
  a.mi = 0xffffffffu / (uint32_t)a.ni + 1;
  a.mv = 0xffffffffu / (uint32_t)a.nv + 1;
  // a token's heads over several CTAs while there are fewer tokens than SMs
  const int items = (a.hq + 2 * a.c.kv_heads) * a.c.head_dim / (vec ? 4 : 1);
  const int parts = std::max(1, std::min(sm_count() / T, items / kRopeThreads));
  // many tokens: smaller CTAs, more of which are resident and wait for their
  // tokens' pages at a time (8191 tokens: 256 threads 68 us, 128 threads 65.5 us; 64
  // tokens 2.4 and 2.9 us)
  const int threads = T > 8 * sm_count() ? 128 : kRopeThreads;
  auto kern = vec ? rope_append_kernel<DT, 4> : rope_append_kernel<DT, 1>;
  MOE_CUDA(launch_pdl(kern, dim3((unsigned)T, (unsigned)parts), dim3((unsigned)threads), 0, s, a));
  return MOE_OK;
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
  moe_paged_cache c;
  MOE_CHECK(moe::take_cache(cache, c));
  MOE_CHECK(moe::check_cache_rows_apart(c));
  MOE_REQUIRE(T >= 0 && q_heads >= 0, MOE_ERR_INVALID, "negative size");
  MOE_REQUIRE(q_heads <= 32767 && cache->kv_heads <= 16383, MOE_ERR_UNSUPPORTED, "too many heads");
  MOE_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= cache->head_dim, MOE_ERR_INVALID,
              "rot %d: an even number up to head_dim %d is needed", rot, cache->head_dim);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(k && v && positions && (rot == 0 || inv_freq), MOE_ERR_INVALID, "null pointer");
  MOE_REQUIRE(q_heads == 0 || (q && q_out), MOE_ERR_INVALID, "null q or q_out");
  if (q_heads > 0) {
    MOE_REQUIRE((T == 1 || qo_tok_stride >= c.head_dim || -qo_tok_stride >= c.head_dim) &&
                    (q_heads == 1 || qo_head_stride >= c.head_dim || -qo_head_stride >= c.head_dim),
                MOE_ERR_INVALID, "rows of q_out overlap");
    MOE_REQUIRE(q_out != q || ((T == 1 || qo_tok_stride == q_tok_stride) &&
                               (q_heads == 1 || qo_head_stride == q_head_stride)),
                MOE_ERR_INVALID, "q_out is q with other strides");
    MOE_REQUIRE(q_out != k && q_out != v, MOE_ERR_INVALID, "q_out overlaps k or v");
  }
  MOE_REQUIRE(seq_ids || T <= cache->seqs, MOE_ERR_INVALID,
              "%d tokens for %d sequences need seq_ids", T, cache->seqs);
  moe::RopeArgs a = {c, q, k, v, q_tok_stride, q_head_stride, k_tok_stride, k_head_stride,
                     v_tok_stride, v_head_stride, qo_tok_stride, qo_head_stride, q_out, positions,
                     seq_ids, inv_freq, status, q_heads, rot, interleaved};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  {
    ::moe::ProfScope _prof(MOE_K_ROPE_APPEND, s);
    MOE_CHECK(cache->dtype == MOE_CACHE_F16    ? moe::launch_rope<MOE_CACHE_F16>(a, T, s)
              : cache->dtype == MOE_CACHE_BF16 ? moe::launch_rope<MOE_CACHE_BF16>(a, T, s)
                                               : moe::launch_rope<MOE_CACHE_E4M3>(a, T, s));
  }
  return moe::check_launch("rope_append");
}

int moe_rope_append_record(const moe_rope_append_args* a) {
  MOE_REQUIRE(a, MOE_ERR_INVALID, "null arguments");
  return moe_rope_append(&a->cache, a->q, a->q_tok_stride, a->q_head_stride, a->k, a->k_tok_stride,
                         a->k_head_stride, a->v, a->v_tok_stride, a->v_head_stride, a->T,
                         a->q_heads, a->positions, a->seq_ids, a->inv_freq, a->rot, a->interleaved,
                         a->q_out, a->qo_tok_stride, a->qo_head_stride, a->status, a->stream);
}

}  // extern "C"
