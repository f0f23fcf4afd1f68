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
// key head), values not at all, 8 bytes per slot for the sums.  The products go to mma.sync
// (m16n8k16) as in the attention kernel, the heads' parts in the 16 rows of M
// (attention_frag.cuh); on CUDA cores 4 heads would take 2 instructions per head and element and be
// issue-bound.
//
// Work.  A unit is a (sequence, key head), cut into rounds of KEYS keys per warp.  All units in
// order, each at the cost of its rounds and one more for its start (q and its parts), are dealt
// out in equal contiguous runs to the CTAs of one resident grid, whatever the lengths.  A warp
// takes a tile of KEYS keys of each round through a ring of its own, filled by TMA in boxes that
// lie in one page (as in the attention kernel); the loads run on across the ends of units, page
// ids are fetched a tile ahead of them.  (Keys loaded by the lanes themselves, straight
// into the operands of the products, took 367 instructions for 16 keys, most of them for
// addresses: 64 sequences of up to 4096 keys, 8 heads of 128, bf16, 89 us; now 50, 78 % of
// the memory's rate: 254 MB at 5.1 TB/s.)
#include <math.h>

#include <algorithm>
#include <cmath>

#include "attention_frag.cuh"
#include "tc_common.cuh"

namespace moe {

constexpr int kMassWarps = 8, kMassThreads = kMassWarps * 32;
constexpr int kMassGroups = 4;         // groups of 8 query heads at one reading of the keys, at most
constexpr int kMassSlots = 3;

struct MassArgs {
  moe_paged_cache c;
  CacheMap map;
  const float* q;
  int64_t q_ss, q_hs;
  const int32_t* seq_lens;
  const float *lse, *mass;
  float* out;
  int64_t row;                         // slots of a (sequence, head) in mass and out
  int* status;
  int hq, window, pass;                // the first of the groups of heads of this launch
  float scale, cap;
};

template <int DT, int DP, bool PACK> struct MassCfg {
  static constexpr bool kBf = DT == MOE_CACHE_BF16;
  using Frag = AFrag<kBf, PACK>;
  static constexpr int kElem = DT == MOE_CACHE_E4M3 ? 1 : 2;
  static constexpr int kRow = DP * kElem < kLine ? kLine : DP * kElem;     // bytes in the ring
  static constexpr int kLines = kRow / kLine;
  static constexpr int kKeys = kRow <= 128 ? 32 : 16;      // keys of a tile
  static constexpr int kSlot = kKeys * kRow;
  static constexpr int kRing = kMassWarps * kMassSlots * kSlot;
  static constexpr int kGroup = DP / 16 * Frag::kBytes;
  static constexpr int kGroups = kRing + kMassGroups * kGroup <= 220 * 1024 ? kMassGroups : 2;
  static_assert(kRing + kGroups * kGroup <= 225 * 1024, "");
  static constexpr int kRound = kMassWarps * kKeys;
  static constexpr int kCtas = kSlot <= 4096 ? 2 : 1;
};

// A cursor over a CTA's rounds: round r of r1 of a unit.
struct MassCursor {
  int seq, head, len, first, r, r1, cost;
  long long at;                        // where the unit's cost begins
};

struct MassShared {
  long long scan[kMassWarps], base;
  int seq, dead;
  uint64_t bars[kMassWarps][kMassSlots];
  float scale[kMassGroups][kAttHeads], lse[kMassGroups][kAttHeads];
};

template <int DT, int DP, bool PACK>
__global__ void __launch_bounds__(kMassThreads, (MassCfg<DT, DP, PACK>::kCtas))
mass_kernel(const __grid_constant__ CUtensorMap kmap, const MassArgs A) {
  using Cfg = MassCfg<DT, DP, PACK>;
  using Frag = typename Cfg::Frag;
  constexpr int KEYS = Cfg::kKeys, RK = Cfg::kRound, NS = kMassSlots, LINES = Cfg::kLines;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ MassShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int D = A.c.head_dim, hk = A.c.kv_heads, G = A.hq / hk, S = A.c.seqs;
  const uint32_t ps = A.c.page_size;
  const int ng = min(Cfg::kGroups, (G + kAttHeads - 1) / kAttHeads - A.pass);
  const int most = (int)min((int64_t)A.c.table_width * A.c.page_size, A.row);
  if (lane < NS) {
    mbar_init(&sh.bars[warp][lane], 1);
    fence_mbar_init();
  }
  if (tid == 0) {
    sh.dead = 0;
    prefetch_map(&kmap);
  }
  pdl_trigger();
  pdl_wait();

  // ---- this CTA's run
  auto len_of = [&](int s) { return min(max(A.seq_lens[s], 0), most); };
  auto cost_of = [&](int s) {                  // of one head of the sequence
    const int n = len_of(s);
    return n ? (n + RK - 1) / RK + 1 : 0;
  };
  const int per = (S + kMassThreads - 1) / kMassThreads, s0 = min(S, tid * per), s1 = min(S, s0 + per);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) {
    mine += (long long)cost_of(s) * hk;
    if (blockIdx.x == 0 && A.seq_lens[s] > most) set_status(A.status, MOE_STATUS_BAD_PAGE);
  }
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  long long total = 0, before = incl - mine;
#pragma unroll
  for (int w = 0; w < kMassWarps; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  const long long quota = (total + gridDim.x - 1) / gridDim.x, start = blockIdx.x * quota;
  const long long end = min(total, start + quota);
  if (start >= end) return;
  if (mine > 0 && before <= start && start < before + mine) {
    int s = s0;
    for (;;) {
      const long long n = (long long)cost_of(s) * hk;
      if (start < before + n) break;
      before += n;
      ++s;
    }
    sh.seq = s;
    sh.base = before;
  }
  __syncthreads();

  auto open = [&](MassCursor& c) {             // its rounds r .. r1 of this run; false: none
    c.len = len_of(c.seq);
    c.first = A.window > 0 && c.len > A.window ? c.len - A.window : 0;
    c.r = (int)max(0ll, start - c.at - 1);
    c.r1 = (int)min((long long)c.cost - 1, end - c.at - 1);
    return c.r < c.r1;
  };
  auto next_unit = [&](MassCursor& c) {        // false: that was the last
    do {
      c.at += c.cost;
      if (c.at >= end) return false;
      if (++c.head == hk) {
        c.head = 0;
        do {
          c.cost = cost_of(++c.seq);           // there is one: at < end <= total
        } while (c.cost == 0);
      }
    } while (!open(c));
    return true;
  };
  MassCursor C;                                // of the arithmetic
  C.seq = sh.seq;
  C.cost = cost_of(C.seq);
  C.head = (int)((start - sh.base) / C.cost);
  C.at = sh.base + (long long)C.head * C.cost;
  bool more = open(C) || next_unit(C);
  if (!more) return;                           // the run is the start of a unit whose rounds are not in it

  // ---- loads: a cursor that runs NS - 1 tiles ahead, across the ends of units
  MassCursor W = C;
  bool wmore = true;
  const uint32_t ring = smem_u32(smem) + warp * NS * Cfg::kSlot;
  const int box = 1 << A.map.box_shift, boxes = KEYS >> A.map.box_shift;
  int lslot = 0, page = -1;
  uint32_t pslot = 0;
  bool in = false;
  auto ask = [&]() {                           // page of this lane's box of the cursor's tile
    const int key = W.r * RK + warp * KEYS + (lane << A.map.box_shift);
    in = wmore && lane < boxes && key < W.len && key + box > W.first;
    if (in) {
      const uint32_t n = (uint32_t)key / ps;
      pslot = (uint32_t)key - n * ps;
      page = A.c.block_table[(int64_t)W.seq * A.c.table_stride + n];
    }
  };
  auto load = [&]() -> uint32_t {              // the cursor's tile; which keys are there and seen
    if (!wmore) return 0u;
    if (in && (page < 0 || page >= A.c.pages)) {
      set_status(A.status, MOE_STATUS_BAD_PAGE);
      in = false;
    }
    const uint32_t ok = __ballot_sync(0xffffffffu, in);
    uint64_t* bar = &sh.bars[warp][lslot];
    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(__popc(ok) * LINES * kLine) << A.map.box_shift);
    __syncwarp();
    if (in) {
      const uint32_t to = ring + lslot * Cfg::kSlot + (lane << A.map.box_shift) * kLine;
      const int row = page * A.map.page_units + W.head * A.map.head_units;
#pragma unroll
      for (int b = 0; b < LINES; ++b)
        tma_load_3d(to + b * KEYS * kLine, &kmap, b * (kLine / Cfg::kElem), row, (int)pslot, bar);
    }
    lslot = lslot + 1 == NS ? 0 : lslot + 1;
    const int key = W.r * RK + warp * KEYS + (lane & (KEYS - 1));
    const uint32_t seen = __ballot_sync(0xffffffffu, key >= W.first && key < W.len &&
                                                         ((ok >> ((lane & (KEYS - 1)) >> A.map.box_shift)) & 1u));
    if (++W.r == W.r1) wmore = next_unit(W);
    ask();
    return seen;
  };
  ask();
  uint32_t seen_of[NS - 1];
#pragma unroll
  for (int i = 0; i < NS - 1; ++i) seen_of[i] = load();

  // Bounded; after a timeout anywhere in the CTA no wait takes long any more.
  int cslot = 0;
  uint32_t cphase = 0;
  auto wait_slot = [&]() {
    uint64_t* bar = &sh.bars[warp][cslot];
    if (!mbar_test(bar, cphase) && !*(volatile int*)&sh.dead && !mbar_wait(bar, cphase)) {
      sh.dead = 1;
      set_status(A.status, MOE_STATUS_TIMEOUT);
    }
    __syncwarp();
    const uint32_t a = ring + cslot * Cfg::kSlot;
    if (++cslot == NS) {
      cslot = 0;
      cphase ^= 1u;
    }
    return a;
  };
  uint8_t* const qs = smem + Cfg::kRing;

  // fragment addresses: byte offset of 16-byte chunk c of row r, blocks of KEYS lines
  auto slot_at = [](int r, int c) {
    return (uint32_t)((c >> 3) * KEYS * kLine + r * kLine + (((c & 7) ^ (r & 7)) << 4));
  };
  const int krow = Cfg::kElem == 2 ? (lane >> 4) * 8 + (lane & 7)
                                   : ((lane >> 3) & 1) * 8 + (lane & 7);
  const int kch = Cfg::kElem == 2 ? (lane >> 3) & 1 : lane >> 4;
  constexpr int PPL = kLine / 32;              // chunk pairs of a line
  uint32_t kof[PPL];
#pragma unroll
  for (int j = 0; j < PPL; ++j) kof[j] = slot_at(krow, 2 * j + kch);
  // the key whose sum this lane will hold
  constexpr int NT = KEYS / 8;
  const int own = NT == 4 ? 8 * (lane >> 3) + 2 * t + ((lane >> 2) & 1)
                          : 8 * (lane >> 4) + 2 * t + ((lane >> 3) & 1);

  for (bool first_unit = true;; first_unit = false) {
    // ---- q's parts, a warp per group: scaled by a power of two to [2^10, 2^11)
    if (!first_unit) __syncthreads();          // those before these have been read
    if (warp < ng) {
      const int h = (A.pass + warp) * kAttHeads + (PACK ? g & 3 : g);
      const bool live = h < G && (!PACK || g < 4);
      const float* q = A.q + (int64_t)C.seq * A.q_ss + ((int64_t)C.head * G + h) * A.q_hs;
      // columns of a step: 2t, 2t + 1, 2t + 8, 2t + 9, of e4m3 keys 4t .. 4t + 3
      auto column = [&](int i, int k) {
        return 16 * i + (Cfg::kElem == 1 ? 4 * t + k : 2 * t + (k & 1) + 8 * (k >> 1));
      };
      float v[DP / 16][4], mx = 0.f;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int e = column(i, k);
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
        sh.scale[warp][g] = ldexpf(A.scale * A.c.k_scale, -e);
        // a head that is not there, or has seen no key, gives nothing
        const float l = live ? A.lse[(int64_t)C.seq * A.hq + (int64_t)C.head * G + h] : -INFINITY;
        sh.lse[warp][g] = l == -INFINITY ? INFINITY : l * kLog2e;
      }
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        Frag f;
        f.set(v[i][0] * f1 * f2, v[i][1] * f1 * f2, v[i][2] * f1 * f2, v[i][3] * f1 * f2, g);
        f.store(qs + warp * Cfg::kGroup + i * Frag::kBytes, lane);
      }
    }
    __syncthreads();
    const int64_t unit = ((int64_t)C.seq * hk + C.head) * A.row;
    const float* mass = A.mass + unit;
    float* out = A.out + unit;

    for (; C.r < C.r1; ++C.r) {
      const int key = C.r * RK + warp * KEYS + own;
      const bool writes = key < C.len && (NT == 4 || !(lane & 4));
      const float sum = writes ? mass[key] : 0.f;
      const uint32_t ka = wait_slot();
      const uint32_t seen = seen_of[0];
#pragma unroll
      for (int i = 0; i + 1 < NS - 1; ++i) seen_of[i] = seen_of[i + 1];
      seen_of[NS - 2] = load();

      float w[NT][2];                          // keys 8n + 2t, 8n + 2t + 1 of head g
#pragma unroll
      for (int n = 0; n < NT; ++n) w[n][0] = w[n][1] = 0.f;
#pragma unroll 1
      for (int gr = 0; gr < ng; ++gr) {
        const uint8_t* qg = qs + gr * Cfg::kGroup;
        float y[NT][2];
#pragma unroll
        for (int k4 = 0; k4 < DP / 64; ++k4) {             // four steps in an accumulator
          float a[NT][4];
#pragma unroll
          for (int kk = 4 * k4; kk < 4 * k4 + 4; kk += 3 - Cfg::kElem) {
            Frag q0, q1;
            q0.load(qg + kk * Frag::kBytes, lane);
            if (Cfg::kElem == 1) q1.load(qg + (kk + 1) * Frag::kBytes, lane);
            const int j = Cfg::kElem == 2 ? kk : kk / 2;   // chunk pair
#pragma unroll
            for (int kb = 0; kb < KEYS / 16; ++kb) {
              uint32_t b[4];
              ldsm4(b, ka + kof[j % PPL] + (j / PPL) * KEYS * kLine + kb * 16 * kLine);
              if (Cfg::kElem == 2) {
                if (kk == 4 * k4) {
                  q0.template mul<true>(a[2 * kb], b[0], b[1]);
                  q0.template mul<true>(a[2 * kb + 1], b[2], b[3]);
                } else {
                  q0.mul(a[2 * kb], b[0], b[1]);
                  q0.mul(a[2 * kb + 1], b[2], b[3]);
                }
              } else {
                uint32_t f[4][2];
#pragma unroll
                for (int i = 0; i < 4; ++i) e4m3x4_f16x2(b[i], f[i][0], f[i][1]);
                if (kk == 4 * k4) {
                  q0.template mul<true>(a[2 * kb], f[0][0], f[0][1]);
                  q0.template mul<true>(a[2 * kb + 1], f[1][0], f[1][1]);
                } else {
                  q0.mul(a[2 * kb], f[0][0], f[0][1]);
                  q0.mul(a[2 * kb + 1], f[1][0], f[1][1]);
                }
                q1.mul(a[2 * kb], f[2][0], f[2][1]);
                q1.mul(a[2 * kb + 1], f[3][0], f[3][1]);
              }
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            y[n][0] = (k4 ? y[n][0] : 0.f) + (a[n][0] + a[n][2]);
            y[n][1] = (k4 ? y[n][1] : 0.f) + (a[n][1] + a[n][3]);
          }
        }
        const float scale = sh.scale[gr][g], lse2 = sh.lse[gr][g];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float z = y[n][h];
            if (PACK) z += __shfl_xor_sync(0xffffffffu, z, 16);
            z *= scale;
            if (A.cap > 0.f) z = A.cap * tanhf(z / A.cap);
            const float p = ex2(fmaf(z, kLog2e, -lse2));
            w[n][h] += lse2 == INFINITY ? 0.f : p;
          }
      }
      // over the heads, which the lanes with the same t hold: halves are exchanged until one
      // key is left
      float r;
      const bool hi = lane & 16, mid = lane & 8, lo = lane & 4;
      if (NT == 4) {
        float u[4], v[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float keep = hi ? w[(2 + i / 2) % NT][i % 2] : w[i / 2][i % 2];
          const float give = hi ? w[i / 2][i % 2] : w[(2 + i / 2) % NT][i % 2];
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
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float keep = hi ? w[1][i] : w[0][i], give = hi ? w[0][i] : w[1][i];
          u[i] = keep + __shfl_xor_sync(0xffffffffu, give, 16);
        }
        r = (mid ? u[1] : u[0]) + __shfl_xor_sync(0xffffffffu, mid ? u[0] : u[1], 8);
        r += __shfl_xor_sync(0xffffffffu, r, 4);
      }
      // (what the ring holds for a key that is not there is anything)
      if (writes) out[key] = (seen >> own) & 1u ? sum + r : sum;
    }
    if (!next_unit(C)) break;
  }
  // after a timeout copies may still be under way: give them time to land
  if (*(volatile int*)&sh.dead)
    for (int i = 0; i < NS; ++i) {
      mbar_wait(&sh.bars[warp][i], 0);
      mbar_wait(&sh.bars[warp][i], 1);
    }
}

template <int DT, int DP, bool PACK>
static int launch_mass(MassArgs& a, int64_t longest, cudaStream_t s) {
  using Cfg = MassCfg<DT, DP, PACK>;
  auto kern = mass_kernel<DT, DP, PACK>;
  const int all = (a.hq / a.c.kv_heads + kAttHeads - 1) / kAttHeads;
  CUtensorMap kmap;
  MOE_CHECK(make_cache_map(&kmap, a.c, a.c.k, Cfg::kKeys, &a.map));
  const int64_t units = (int64_t)a.c.seqs * a.c.kv_heads;
  const int64_t rounds = units * std::max<int64_t>(1, (longest + Cfg::kRound - 1) / Cfg::kRound);
  const int grid = (int)std::min<int64_t>(rounds, (int64_t)Cfg::kCtas * sm_count());
  for (a.pass = 0; a.pass < all; a.pass += Cfg::kGroups) {
    const int smem = Cfg::kRing + std::min(Cfg::kGroups, all - a.pass) * Cfg::kGroup;
    MOE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  Cfg::kRing + Cfg::kGroups * Cfg::kGroup));
    MOE_CUDA(launch_pdl(kern, dim3((unsigned)grid), dim3(kMassThreads), (size_t)smem, s, kmap, a));
    a.mass = a.out;                    // further groups of heads add to the sums of the first
  }
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
