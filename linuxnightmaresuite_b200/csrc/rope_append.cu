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
#include <cmath>
#include <type_traits>

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

// Whether all rows can be taken four elements at a time.
static bool four_at_a_time(const RopeArgs& a) {
  auto aligned = [](const void* p, int64_t ts, int64_t hs) {
    return (uintptr_t)p % 16 == 0 && ts % 4 == 0 && hs % 4 == 0;
  };
  return a.rot % (a.interleaved ? 4 : 8) == 0 && aligned(a.k, a.k_ts, a.k_hs) &&
         aligned(a.v, a.v_ts, a.v_hs) &&
         (a.hq == 0 || (aligned(a.q, a.q_ts, a.q_hs) && aligned(a.q_out, a.qo_ts, a.qo_hs)));
}

template <int DT>
static int launch_rope(RopeArgs& a, int T, cudaStream_t s) {
  const bool vec = four_at_a_time(a);
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

// ---------------------------------------------------------------------------
// The append with a norm of each query and key head in front of the rotation,
//
//   y = x / sqrt(mean(x^2) + eps) * w      (or 1 + w),
//
// cache slots apart from the positions, and the slots' ledger (accumulated
// attention weight, position held).
//
// A norm needs its whole head before any element turns, so here a group of GL lanes
// owns a row: it loads the row once, in the items of the rotation (both halves of a
// pair meet in one lane), sums the squares by shuffles and turns what it holds.  Rows
// of a token go to the groups of its CTA; each group has the loads of kRowsAhead rows
// under way before it waits for the angles and the slot.  Bound by memory for
// prompts, by latency for single tokens, like the form without norms.
// ---------------------------------------------------------------------------
struct NormArgs {
  const float *q_norm, *k_norm;        // null: that head is not normed
  const int32_t* slots;                // null: the positions
  float* mass;                         // ledgers, null: none
  int32_t* held;
  int64_t ledger_row;                  // slots of a (sequence, head) in them
  float eps, plus;                     // weights are plus + w
};

constexpr int kRowsAhead = 3;
constexpr int kNormThreads = 128;

template <int VEC>
struct NormRow {
  Elems<VEC> a, b;
};

// The factors of a lane's item for all rows of a token: with a norm's weights w, or 1,
//   (x0, x1) -> (x0 w0 cos - x1 w1 sin, x1 w1 cos + x0 w0 sin) / norm,
// pair k in (k, VEC + k) of a and b, or adjacent ones of a; without a turn cos 1, sin 0.
template <int VEC, bool PAIRS>
struct NormFactors {
  float c0[VEC], s1[VEC], c1[VEC], s0[VEC];      // w0 cos, w1 sin, w1 cos, w0 sin
};

// Norm, rotation, append.  GL lanes own a row: its sum of squares is a few shuffles, no barrier,
// and a lane's factors serve all rows of a token, q's, then k's; values are copied after them.
// Bound by memory: 8191 tokens of 32 + 2 x 8 heads of 128, bf16 cache, 78 us, 369 MB at 4.7 TB/s, 72 %
// of a copy's rate (a row's loads, its sum and its quotient follow one another, and 28 warps of
// an SM do not hide all of it); weights and angles multiplied row by row took 136.
//
// Items of a lane: one, or (M > 1, a row of 16 lanes would be too few) M; PAIRS: an item of
// the rotation is two loads
template <int DT, int VEC, int GL, int M, bool PAIRS>
__global__ void __launch_bounds__(kNormThreads, M == 1 ? 7 : 3)
norm_append_kernel(const RopeArgs A, const NormArgs N) {
  using T = typename CacheType<DT>::T;
  __shared__ float2 cs[kMaxHeadDim / 2];
  __shared__ int64_t sh_slot;
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x;
  const int pos = A.positions[t];
  const int at = N.slots ? N.slots[t] : pos;
  if (pos < 0 || at < 0) return;
  const int hk = A.c.kv_heads, d = A.c.head_dim, nr = A.nr, ni = A.ni, nv = A.nv;
  const int h = A.rot / 2;
  constexpr int GROUPS = kNormThreads / GL;
  constexpr int HALF = VEC > 1 ? VEC / 2 : 1;    // adjacent pairs of an item
  const int gl = threadIdx.x % GL;
  const int g0 = blockIdx.y * GROUPS + threadIdx.x / GL, step = gridDim.y * GROUPS;
  const int apart = A.interleaved ? 1 : h;
  auto first_of = [&](int i) {
    return i < nr ? i * VEC * (VEC == 1 && A.interleaved ? 2 : 1) : A.rot + (i - nr) * VEC;
  };
  const float* const qp = A.q + t * A.q_ts;
  const float* const kp = A.k + t * A.k_ts;
  // q's rows, then k's, group by group
  auto fetch = [&](int row, const float* base, int64_t hs, int rows, NormRow<VEC> (&r)[M]) {
    if (row >= rows) return;
    const float* src = base + row * hs;
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int i = gl + m * GL, e = first_of(i);
      if (i < ni) r[m].a = load_elems<VEC>(src + e);
      if (PAIRS && i < nr) r[m].b = load_elems<VEC>(src + e + apart);
    }
  };
  NormRow<VEC> ahead[kRowsAhead][M];
#pragma unroll
  for (int k = 0; k < kRowsAhead; ++k) fetch(g0 + k * step, qp, A.q_hs, A.hq, ahead[k]);

  if (threadIdx.x == blockDim.x - 1) {           // the token's slot in both caches, -1: none
    const int seq = A.seq_ids ? A.seq_ids[t] : t, n = at / A.c.page_size;
    int64_t slot = -1;
    if (seq >= 0 && seq < A.c.seqs && n < A.c.table_width && (!N.mass || at < N.ledger_row)) {
      const int page = A.c.block_table[(int64_t)seq * A.c.table_stride + n];
      if (page >= 0 && page < A.c.pages)
        slot = (int64_t)page * A.c.page_stride +
               (int64_t)(at - n * A.c.page_size) * A.c.token_stride;
    }
    if (slot < 0) set_status(A.status, MOE_STATUS_BAD_PAGE);
    sh_slot = slot;
    if (slot >= 0 && N.mass && blockIdx.y == 0)
      for (int j = 0; j < hk; ++j) {
        const int64_t e = ((int64_t)seq * hk + j) * N.ledger_row + at;
        N.mass[e] = 0.f;
        N.held[e] = pos;
      }
  }
  for (int i = threadIdx.x; i < h; i += kNormThreads) cs[i] = rope_cos_sin(pos, A.inv_freq[i]);
  __syncthreads();
  const int64_t slot = sh_slot;

  NormFactors<VEC, PAIRS> f[M];
  auto factors = [&](const float* w) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int i = gl + m * GL, e = first_of(i);
      auto weight = [&](int x) { return w ? N.plus + w[x] : 1.f; };
      if (PAIRS) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float2 c = i < nr ? cs[A.interleaved ? e / 2 : e + k] : make_float2(1.f, 0.f);
          const float w0 = i < ni ? weight(e + k) : 0.f, w1 = i < nr ? weight(e + apart + k) : 0.f;
          f[m].c0[k] = w0 * c.x;
          f[m].s1[k] = w1 * c.y;
          f[m].c1[k] = w1 * c.x;
          f[m].s0[k] = w0 * c.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < HALF; ++k) {
          const float2 c = i < nr ? cs[e / 2 + k] : make_float2(1.f, 0.f);
          const float w0 = i < ni ? weight(e + 2 * k) : 0.f;
          const float w1 = i < ni ? weight(e + 2 * k + 1) : 0.f;
          f[m].c0[k] = w0 * c.x;
          f[m].s1[k] = w1 * c.y;
          f[m].c1[k] = w1 * c.x;
          f[m].s0[k] = w0 * c.y;
        }
      }
    }
  };
  const float per = 1.f / (float)d;
  // the sum of squares is the same for all lanes of a group
  auto turn = [&](NormRow<VEC> (&r)[M], bool normed) {
    float inv = 1.f;
    if (normed) {
      float ss = 0.f;
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int i = gl + m * GL;
        if (i < ni) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) ss = fmaf(r[m].a.v[k], r[m].a.v[k], ss);
        }
        if (PAIRS && i < nr) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) ss = fmaf(r[m].b.v[k], r[m].b.v[k], ss);
        }
      }
      const uint32_t mask = GL == 32 ? 0xffffffffu
                                     : ((1u << GL % 32) - 1u) << (threadIdx.x % 32 / GL * GL);
#pragma unroll
      for (int o = GL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      inv = 1.f / sqrtf(fmaf(ss, per, N.eps));
    }
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int i = gl + m * GL;
      if (PAIRS) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float x0 = r[m].a.v[k] * inv, x1 = i < nr ? r[m].b.v[k] * inv : 0.f;
          r[m].a.v[k] = i < nr ? fmaf(x0, f[m].c0[k], -x1 * f[m].s1[k]) : x0 * f[m].c0[k];
          r[m].b.v[k] = fmaf(x1, f[m].c1[k], x0 * f[m].s0[k]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < HALF; ++k) {
          const float x0 = r[m].a.v[2 * k] * inv, x1 = r[m].a.v[(2 * k + 1) % VEC] * inv;
          r[m].a.v[2 * k] = i < nr ? fmaf(x0, f[m].c0[k], -x1 * f[m].s1[k]) : x0 * f[m].c0[k];
          r[m].a.v[(2 * k + 1) % VEC] =
              i < nr ? fmaf(x1, f[m].c1[k], x0 * f[m].s0[k]) : x1 * f[m].c1[k];
        }
      }
    }
  };
  if (A.hq > 0) {
    factors(N.q_norm);
    float* const to = A.q_out + t * A.qo_ts;
    for (int row0 = g0; row0 < A.hq; row0 += kRowsAhead * step) {
#pragma unroll
      for (int k = 0; k < kRowsAhead; ++k) {
        const int row = row0 + k * step;
        if (row < A.hq) {
          turn(ahead[k], N.q_norm != nullptr);
          float* out = to + row * A.qo_hs;
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const int i = gl + m * GL, e = first_of(i);
            if (i < ni) store_f32<VEC>(out + e, ahead[k][m].a);
            if (PAIRS && i < nr) store_f32<VEC>(out + e + apart, ahead[k][m].b);
          }
        }
        fetch(row + kRowsAhead * step, qp, A.q_hs, A.hq, ahead[k]);
      }
    }
  }
  if (slot < 0) return;
#pragma unroll
  for (int k = 0; k < kRowsAhead; ++k) fetch(g0 + k * step, kp, A.k_hs, hk, ahead[k]);
  factors(N.k_norm);
  {
    T* const to = static_cast<T*>(A.c.k) + slot;
    for (int row0 = g0; row0 < hk; row0 += kRowsAhead * step) {
#pragma unroll
      for (int k = 0; k < kRowsAhead; ++k) {
        const int row = row0 + k * step;
        if (row < hk) {
          turn(ahead[k], N.k_norm != nullptr);
          T* out = to + (int64_t)row * A.c.head_stride;
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const int i = gl + m * GL, e = first_of(i);
            if (i < ni) store_cache<VEC>(out + e, ahead[k][m].a, A.c.k_scale);
            if (PAIRS && i < nr) store_cache<VEC>(out + e + apart, ahead[k][m].b, A.c.k_scale);
          }
        }
        fetch(row + kRowsAhead * step, kp, A.k_hs, hk, ahead[k]);
      }
    }
  }
  // ---- values: copied
  const int total = hk * nv, every = gridDim.y * kNormThreads;
  T* const to = static_cast<T*>(A.c.v) + slot;
#pragma unroll 2
  for (int it = blockIdx.y * kNormThreads + threadIdx.x; it < total; it += every) {
    const int j = nv == 1 ? it : (int)__umulhi((uint32_t)it, A.mv), e = (it - j * nv) * VEC;
    store_cache<VEC>(to + (int64_t)j * A.c.head_stride + e,
                     load_elems<VEC>(A.v + t * A.v_ts + j * A.v_hs + e), A.c.v_scale);
  }
}

template <int DT>
static int launch_norm_append(RopeArgs& a, const NormArgs& n, int T, cudaStream_t s) {
  const bool vec = four_at_a_time(a);
  const int d = a.c.head_dim;
  if (vec) {
    a.nr = a.interleaved ? a.rot / 4 : a.rot / 8;
    a.ni = a.nr + (d - a.rot) / 4;
    a.nv = d / 4;
  } else {                             // items are pairs, then single elements
    a.nr = a.rot / 2;
    a.ni = a.nr + (d - a.rot);
    a.nv = d;
  }
  a.mv = 0xffffffffu / (uint32_t)a.nv + 1;
  // lanes of a row: one item each where 32 are enough
  const bool pairs = !a.interleaved || !vec;
  const int gl = !vec || a.ni > 16 ? 32 : a.ni > 8 ? 16 : 8;
  auto pick = [&](auto p) {
    constexpr bool P = decltype(p)::value;
    return !vec        ? norm_append_kernel<DT, 1, 32, 8, true>
           : a.ni > 32 ? norm_append_kernel<DT, 4, 32, 2, P>
           : gl == 32  ? norm_append_kernel<DT, 4, 32, 1, P>
           : gl == 16  ? norm_append_kernel<DT, 4, 16, 1, P>
                       : norm_append_kernel<DT, 4, 8, 1, P>;
  };
  auto kern = pairs ? pick(std::true_type{}) : pick(std::false_type{});
  const int rows = a.hq + a.c.kv_heads;
  const int parts = std::max(1, std::min(sm_count() / T, rows * gl / kNormThreads));
  MOE_CUDA(launch_pdl(kern, dim3((unsigned)T, (unsigned)parts), dim3(kNormThreads), 0, s, a, n));
  return MOE_OK;
}

}  // namespace moe

namespace moe {

// The arguments that both forms of the append share.
static int take_append(const moe_rope_append_args* r, RopeArgs& a) {
  const moe_paged_cache* cache = &r->cache;
  moe_paged_cache c;
  MOE_CHECK(take_cache(cache, c));
  MOE_CHECK(check_cache_rows_apart(c));
  const int T = r->T, q_heads = r->q_heads, rot = r->rot;
  const float *q = r->q, *k = r->k, *v = r->v;
  float* q_out = r->q_out;
  MOE_REQUIRE(T >= 0 && q_heads >= 0, MOE_ERR_INVALID, "negative size");
  MOE_REQUIRE(q_heads <= 32767 && cache->kv_heads <= 16383, MOE_ERR_UNSUPPORTED, "too many heads");
  MOE_REQUIRE(rot >= 0 && rot % 2 == 0 && rot <= cache->head_dim, MOE_ERR_INVALID,
              "rot %d: an even number up to head_dim %d is needed", rot, cache->head_dim);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(k && v && r->positions && (rot == 0 || r->inv_freq), MOE_ERR_INVALID, "null pointer");
  MOE_REQUIRE(q_heads == 0 || (q && q_out), MOE_ERR_INVALID, "null q or q_out");
  if (q_heads > 0) {
    MOE_REQUIRE((T == 1 || r->qo_tok_stride >= c.head_dim || -r->qo_tok_stride >= c.head_dim) &&
                    (q_heads == 1 || r->qo_head_stride >= c.head_dim ||
                     -r->qo_head_stride >= c.head_dim),
                MOE_ERR_INVALID, "rows of q_out overlap");
    MOE_REQUIRE(q_out != q || ((T == 1 || r->qo_tok_stride == r->q_tok_stride) &&
                               (q_heads == 1 || r->qo_head_stride == r->q_head_stride)),
                MOE_ERR_INVALID, "q_out is q with other strides");
    MOE_REQUIRE(q_out != k && q_out != v, MOE_ERR_INVALID, "q_out overlaps k or v");
  }
  MOE_REQUIRE(r->seq_ids || T <= cache->seqs, MOE_ERR_INVALID,
              "%d tokens for %d sequences need seq_ids", T, cache->seqs);
  a = {c, q, k, v, r->q_tok_stride, r->q_head_stride, r->k_tok_stride, r->k_head_stride,
       r->v_tok_stride, r->v_head_stride, r->qo_tok_stride, r->qo_head_stride, q_out, r->positions,
       r->seq_ids, r->inv_freq, r->status, q_heads, rot, r->interleaved};
  return MOE_OK;
}

}  // namespace moe

extern "C" {

int moe_rope_append_record(const moe_rope_append_args* r) {
  MOE_REQUIRE(r, MOE_ERR_INVALID, "null arguments");
  moe::RopeArgs a = {};
  MOE_CHECK(moe::take_append(r, a));
  if (r->T == 0) return MOE_OK;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r->stream);
  {
    ::moe::ProfScope _prof(MOE_K_ROPE_APPEND, s);
    const int dt = a.c.dtype;
    MOE_CHECK(dt == MOE_CACHE_F16    ? moe::launch_rope<MOE_CACHE_F16>(a, r->T, s)
              : dt == MOE_CACHE_BF16 ? moe::launch_rope<MOE_CACHE_BF16>(a, r->T, s)
                                     : moe::launch_rope<MOE_CACHE_E4M3>(a, r->T, s));
  }
  return moe::check_launch("rope_append");
}

int moe_rope_append(const moe_paged_cache* cache, const float* q, int64_t q_tok_stride,
                    int64_t q_head_stride, const float* k, int64_t k_tok_stride,
                    int64_t k_head_stride, const float* v, int64_t v_tok_stride,
                    int64_t v_head_stride, int T, int q_heads, const int32_t* positions,
                    const int32_t* seq_ids, const double* inv_freq, int rot, int interleaved,
                    float* q_out, int64_t qo_tok_stride, int64_t qo_head_stride, int32_t* status,
                    moe_stream_t stream) {
  MOE_REQUIRE(cache, MOE_ERR_INVALID, "null cache");
  const moe_rope_append_args a = {*cache, q, k, v, q_tok_stride, q_head_stride, k_tok_stride,
                                  k_head_stride, v_tok_stride, v_head_stride, positions, seq_ids,
                                  inv_freq, q_out, qo_tok_stride, qo_head_stride, status, stream, T,
                                  q_heads, rot, interleaved};
  return moe_rope_append_record(&a);
}

int moe_norm_append_record(const moe_norm_append_args* r) {
  MOE_REQUIRE(r, MOE_ERR_INVALID, "null arguments");
  moe::RopeArgs a = {};
  MOE_CHECK(moe::take_append(&r->append, a));
  const int T = r->append.T;
  MOE_REQUIRE(std::isfinite(r->eps) && r->eps >= 0.f, MOE_ERR_INVALID, "eps must be finite, >= 0");
  MOE_REQUIRE(!r->mass == !r->held, MOE_ERR_INVALID, "mass and held come together");
  MOE_REQUIRE(!r->mass || r->ledger_slots > 0, MOE_ERR_INVALID, "bad ledger");
  if (T == 0) return MOE_OK;
  const moe::NormArgs n = {r->q_norm, r->k_norm, r->slots, r->mass, r->held, r->ledger_slots, r->eps,
                           r->gemma_style ? 1.f : 0.f};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r->append.stream);
  {
    ::moe::ProfScope _prof(MOE_K_ROPE_APPEND, s);
    const int dt = a.c.dtype;
    MOE_CHECK(dt == MOE_CACHE_F16    ? moe::launch_norm_append<MOE_CACHE_F16>(a, n, T, s)
              : dt == MOE_CACHE_BF16 ? moe::launch_norm_append<MOE_CACHE_BF16>(a, n, T, s)
                                     : moe::launch_norm_append<MOE_CACHE_E4M3>(a, n, T, s));
  }
  return moe::check_launch("norm_append");
}

}  // extern "C"
