// Attention weight that the slots of a paged cache receive in a decode step, added to a
// running sum:
//
//   out[s, h, j] = mass[s, h, j] + sum over the query heads g of key head h of
//                  exp(scale q_g.k_j - lse_g)
//
// with the log sums that the attention of the step returned.  Given those, every key
// stands by itself: no running maximum, no join, any split.
//
// Bound by memory: the keys are read once (again for every further 32 query heads of a
// key head), values not at all, 8 bytes per slot for the sums.  The products go to mma.sync (m16n8k16)
// as in the attention kernel, the heads' parts in the 16 rows of M (attention_frag.cuh);
// on CUDA cores 4 heads would take 2 instructions per head and element and be issue-bound.  But no key
// passes through shared memory: the order of a product's terms is free, so lane (g, t)
// of a warp loads 16-byte chunks t, t + 4, ... of key g straight into the registers of the B
// operand, and q's parts, in shared memory, are laid out in that order.  A warp has
// KEYS keys' loads under way at a time and the mass of its keys behind them; that 16
// warps of an SM alternate between loading and multiplying keeps the memory busy.
#include <math.h>

#include <algorithm>
#include <cmath>

#include "attention_frag.cuh"

namespace moe {

constexpr int kMassWarps = 8;
constexpr int kMassGroups = 4;         // groups of 8 query heads at one reading of the keys

struct MassArgs {
  moe_paged_cache c;
  const float* q;
  int64_t q_ss, q_hs;
  const int32_t* seq_lens;
  const float *lse, *mass;
  float* out;
  int64_t row;                         // slots of a (sequence, head) in mass and out
  int* status;
  int hq, window, chunk, chunks;       // keys of a CTA at a time, CTAs of a (sequence, head)
  float scale, cap;
};

template <int DT, int DP, bool PACK> struct MassCfg {
  static constexpr bool kBf = DT == MOE_CACHE_BF16;
  using Frag = AFrag<kBf, PACK>;
  static constexpr int kElem = DT == MOE_CACHE_E4M3 ? 1 : 2;
  static constexpr int kChunks = DP * kElem / 64;          // 16-byte chunks of a lane and key
  static constexpr int kTiles = DP > 128 ? 2 : 4;          // 8-key tiles of a warp
  static constexpr int kKeys = 8 * kTiles;
  static constexpr int kGroup = DP / 16 * Frag::kBytes;
};

template <int DT, int DP, bool PACK>
__global__ void __launch_bounds__(kMassWarps * 32, 2) mass_kernel(const MassArgs A) {
  using Cfg = MassCfg<DT, DP, PACK>;
  using Frag = typename Cfg::Frag;
  constexpr int CH = Cfg::kChunks, NT = Cfg::kTiles, KEYS = Cfg::kKeys;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float sh_scale[kMassGroups][kAttHeads], sh_lse[kMassGroups][kAttHeads];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int D = A.c.head_dim, G = A.hq / A.c.kv_heads, ps = A.c.page_size;
  const int unit = blockIdx.x / A.chunks, chunk0 = blockIdx.x - unit * A.chunks;
  const int seq = unit / A.c.kv_heads, head = unit - seq * A.c.kv_heads;
  pdl_trigger();
  pdl_wait();
  const int64_t most = std::min<int64_t>((int64_t)A.c.table_width * ps, A.row);
  const int told = A.seq_lens[seq], len = (int)min((int64_t)max(told, 0), most);
  if (told > most && chunk0 == 0 && head == 0 && threadIdx.x == 0)
    set_status(A.status, MOE_STATUS_BAD_PAGE);
  const int first = A.window > 0 && len > A.window ? len - A.window : 0;
  if ((int64_t)chunk0 * A.chunk >= len) return;
  const int32_t* table = A.c.block_table + (int64_t)seq * A.c.table_stride;
  const uint8_t* keys = static_cast<const uint8_t*>(A.c.k) +
                        (int64_t)head * A.c.head_stride * Cfg::kElem;
  const int row_chunks = D * Cfg::kElem / 16;
  const int groups = (G + kAttHeads - 1) / kAttHeads;
  const float* mass = A.mass + (int64_t)unit * A.row;
  float* out = A.out + (int64_t)unit * A.row;

  for (int pass = 0; pass < groups; pass += kMassGroups) {
    const int ng = min(kMassGroups, groups - pass);
    if (pass) __syncthreads();
    // q's parts, a warp per group: scaled by a power of two to [2^10, 2^11)
    if (warp < ng) {
      const int h = (pass + warp) * kAttHeads + (PACK ? g & 3 : g);
      const bool live = h < G && (!PACK || g < 4);
      const float* q = A.q + (int64_t)seq * A.q_ss + ((int64_t)head * G + h) * A.q_hs;
      // element of step i, register k: step i belongs to chunk t + 4 (i / per)
      constexpr int PER = Cfg::kElem == 2 ? 2 : 4, ES = 16 / Cfg::kElem;
      float v[DP / 16][4], mx = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = (t + 4 * (i / PER)) * ES + 4 * (i % PER) + k;
          v[i][k] = h < G && e < D ? q[e] : 0.f;
          mx = fmaxf(mx, fabsf(v[i][k]));
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const int ex = (int)(__float_as_uint(mx) >> 23);
      const int e = mx > 0.f && ex < 255 ? 137 - max(ex, 1) : 0;
      const int e1 = e / 2, e2 = e - e1;       // 2^e may lie outside the exponents of a float
      const float f1 = __uint_as_float((uint32_t)(127 + e1) << 23);
      const float f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
      if (t == 0) {
        sh_scale[warp][g] = ldexpf(A.scale * A.c.k_scale, -e);
        // a head that is not there, or has seen no key, gives nothing
        const float l = live ? A.lse[(int64_t)seq * A.hq + (int64_t)head * G + h] : -INFINITY;
        sh_lse[warp][g] = l == -INFINITY ? INFINITY : l * kLog2e;
      }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        Frag f;
        f.set(v[i][0] * f1 * f2, v[i][1] * f1 * f2, v[i][2] * f1 * f2, v[i][3] * f1 * f2, g);
        f.store(smem + warp * Cfg::kGroup + i * Frag::kBytes, lane);
      }
    }
    __syncthreads();

    for (int64_t c0 = (int64_t)chunk0 * A.chunk; c0 < len; c0 += (int64_t)A.chunks * A.chunk) {
      const int c1 = (int)min((int64_t)len, c0 + A.chunk);
      for (int base = (int)c0 + warp * KEYS; base < c1; base += kMassWarps * KEYS) {
        // lane i < KEYS follows key base + i to its row, -1: not there or not seen
        const int key = base + (lane & (KEYS - 1));
        int64_t at = -1;
        if (key < c1 && key >= first) {
          const int n = key / ps, page = table[n];
          if (page >= 0 && page < A.c.pages)
            at = ((int64_t)page * A.c.page_stride + (int64_t)(key - n * ps) * A.c.token_stride) *
                 Cfg::kElem;
          else
            set_status(A.status, MOE_STATUS_BAD_PAGE);
        }
        uint4 k[NT][CH];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int64_t from = __shfl_sync(0xffffffffu, at, 8 * n + g);
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            k[n][c] = make_uint4(0, 0, 0, 0);
            if (from >= 0 && t + 4 * c < row_chunks)
              asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                           : "=r"(k[n][c].x), "=r"(k[n][c].y), "=r"(k[n][c].z), "=r"(k[n][c].w)
                           : "l"(keys + from + (t + 4 * c) * 16));
          }
        }
        // the key whose sum this lane will hold
        const int mine = NT == 4 ? 8 * (lane >> 3) + 2 * t + ((lane >> 2) & 1)
                                 : 8 * (lane >> 4) + 2 * t + ((lane >> 3) & 1);
        const bool there = __shfl_sync(0xffffffffu, at, mine) >= 0;
        const bool writes = base + mine < c1 && (NT == 4 || !(lane & 4));
        float sum = 0.f;
        if (writes) sum = (pass ? out : mass)[base + mine];

        float w[NT][2];                        // keys 8n + 2t, 8n + 2t + 1 of head g
#pragma unroll
        for (int n = 0; n < NT; ++n) w[n][0] = w[n][1] = 0.f;
        for (int gr = 0; gr < ng; ++gr) {
          const uint8_t* qs = smem + gr * Cfg::kGroup;
          float x[NT][2];
#pragma unroll
          for (int k4 = 0; k4 < DP / 64; ++k4) {         // four steps in an accumulator
            float a[NT][4];
#pragma unroll
            for (int i = 4 * k4; i < 4 * k4 + 4; ++i) {
              Frag f;
              f.load(qs + i * Frag::kBytes, lane);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                uint32_t b0, b1;
                if (Cfg::kElem == 2) {
                  const uint4& v = k[n][i / 2 % CH];
                  b0 = i % 2 ? v.z : v.x;
                  b1 = i % 2 ? v.w : v.y;
                } else {
                  const uint4& v = k[n][i / 4 % CH];
                  e4m3x4_f16x2(i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w, b0,
                               b1);
                }
                if (i == 4 * k4) f.template mul<true>(a[n], b0, b1);
                else f.mul(a[n], b0, b1);
              }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              x[n][0] = (k4 ? x[n][0] : 0.f) + (a[n][0] + a[n][2]);
              x[n][1] = (k4 ? x[n][1] : 0.f) + (a[n][1] + a[n][3]);
            }
          }
          const float scale = sh_scale[gr][g], lse2 = sh_lse[gr][g];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float y = x[n][h];
              if (PACK) y += __shfl_xor_sync(0xffffffffu, y, 16);
              y *= scale;
              if (A.cap > 0.f) y = A.cap * tanhf(y / A.cap);
              const float p = ex2(fmaf(y, kLog2e, -lse2));
              w[n][h] += lse2 == INFINITY ? 0.f : p;
            }
        }
        // over the heads, which the lanes with the same t hold: halves are
        // exchanged until one key is left
        float r;
        if (NT == 4) {
          float u[4], v[2];
          const bool hi = lane & 16, mid = lane & 8, lo = lane & 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float keep = hi ? w[2 + i / 2][i % 2] : w[i / 2][i % 2];
            const float give = hi ? w[i / 2][i % 2] : w[2 + i / 2][i % 2];
            u[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float keep = mid ? u[2 + i] : u[i], give = mid ? u[i] : u[2 + i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, 8);
          }
          r = (lo ? v[1] : v[0]) + __shfl_xor_sync(0xffffffffu, lo ? v[0] : v[1], 4);
        } else {
          float u[2];
          const bool hi = lane & 16, mid = lane & 8;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float keep = hi ? w[1][i] : w[0][i], give = hi ? w[0][i] : w[1][i];
            u[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
          }
          r = (mid ? u[1] : u[0]) + __shfl_xor_sync(0xffffffffu, mid ? u[0] : u[1], 8);
          r += __shfl_xor_sync(0xffffffffu, r, 4);
        }
        if (writes) out[base + mine] = there ? sum + r : sum;
      }
    }
  }
}

template <int DT, int DP, bool PACK>
static int launch_mass(MassArgs& a, int64_t longest, cudaStream_t s) {
  using Cfg = MassCfg<DT, DP, PACK>;
  auto kern = mass_kernel<DT, DP, PACK>;
  const int groups = std::min(kMassGroups, (a.hq / a.c.kv_heads + kAttHeads - 1) / kAttHeads);
  const int smem = groups * Cfg::kGroup;
  if (smem > 48 * 1024 - 1024)
    MOE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // A CTA's start (lengths, q, its parts) costs about as much as 256 keys: chunks as
  // long as leave some six CTAs for each that is resident
  const int64_t units = (int64_t)a.c.seqs * a.c.kv_heads, step = kMassWarps * Cfg::kKeys;
  const int64_t even = units * longest / (12 * sm_count());
  a.chunk = (int)(std::max<int64_t>(1, std::min<int64_t>(16, even / step)) * step);
  a.chunks = (int)std::max<int64_t>(1, (longest + a.chunk - 1) / a.chunk);
  MOE_REQUIRE(units * a.chunks <= 0x7fffffff, MOE_ERR_UNSUPPORTED, "%d sequences are too many",
              a.c.seqs);
  MOE_CUDA(launch_pdl(kern, dim3((unsigned)(units * a.chunks)), dim3(kMassWarps * 32),
                      (size_t)smem, s, a));
  return MOE_OK;
}

template <int DT, bool PACK>
static int launch_mass_dt(MassArgs& a, int64_t longest, cudaStream_t s) {
  const int d = a.c.head_dim;
  return d <= 64    ? launch_mass<DT, 64, PACK>(a, longest, s)
         : d <= 128 ? launch_mass<DT, 128, PACK>(a, longest, s)
                    : launch_mass<DT, 256, PACK>(a, longest, s);
}

}  // namespace moe

extern "C" {

int moe_attention_mass_record(const moe_attention_mass_args* r) {
  MOE_REQUIRE(r, MOE_ERR_INVALID, "null arguments");
  moe::MassArgs a = {};
  MOE_CHECK(moe::take_cache(&r->cache, a.c));
  MOE_REQUIRE(r->q_heads > 0 && r->q_heads % a.c.kv_heads == 0, MOE_ERR_INVALID,
              "%d query heads for %d key heads", r->q_heads, a.c.kv_heads);
  MOE_REQUIRE(r->max_len >= 0 && r->window >= 0, MOE_ERR_INVALID, "negative length or window");
  MOE_REQUIRE(std::isfinite(r->scale) && std::isfinite(r->softcap) && r->softcap >= 0.f,
              MOE_ERR_INVALID, "scale and softcap must be finite, softcap >= 0");
  MOE_REQUIRE(r->ledger_slots > 0, MOE_ERR_INVALID, "bad ledger");
  if (a.c.seqs == 0) return MOE_OK;
  MOE_REQUIRE(r->q && r->seq_lens && r->lse && r->mass && r->out, MOE_ERR_INVALID, "null pointer");
  const int64_t ledger = (int64_t)a.c.seqs * a.c.kv_heads * r->ledger_slots;
  const int64_t apart = (int64_t)((uintptr_t)r->out - (uintptr_t)r->mass);
  MOE_REQUIRE(apart == 0 || apart >= 4 * ledger || -apart >= 4 * ledger, MOE_ERR_INVALID,
              "mass and out overlap, and are not the same");
  a.q = r->q;
  a.q_ss = r->q_seq_stride;
  a.q_hs = r->q_head_stride;
  a.seq_lens = r->seq_lens;
  a.lse = r->lse;
  a.mass = r->mass;
  a.out = r->out;
  a.row = r->ledger_slots;
  a.status = r->status;
  a.hq = r->q_heads;
  a.window = r->window;
  a.scale = r->scale;
  a.cap = r->softcap;
  const int64_t most = std::min<int64_t>((int64_t)a.c.table_width * a.c.page_size, a.row);
  const int64_t longest = r->max_len > 0 ? std::min<int64_t>(r->max_len, most) : most;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r->stream);
  {
    ::moe::ProfScope _prof(MOE_K_ATTENTION_MASS, s);
    if (a.c.dtype == MOE_CACHE_F16)
      MOE_CHECK((moe::launch_mass_dt<MOE_CACHE_F16, false>(a, longest, s)));
    else if (a.c.dtype == MOE_CACHE_E4M3)
      MOE_CHECK((moe::launch_mass_dt<MOE_CACHE_E4M3, false>(a, longest, s)));
    else if (a.hq / a.c.kv_heads <= 4)
      MOE_CHECK((moe::launch_mass_dt<MOE_CACHE_BF16, true>(a, longest, s)));
    else
      MOE_CHECK((moe::launch_mass_dt<MOE_CACHE_BF16, false>(a, longest, s)));
  }
  return moe::check_launch("attention_mass");
}

}  // extern "C"
