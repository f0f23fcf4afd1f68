// Attention of one new token per sequence where all sequences begin with the same pages.
//
//   out_s = (sum_{j < P} e^{s_j} v_j + sum_{P <= j < len} e^{s_j} v_j) / (sum of the e^{s_j})
//
// The first sums are over the same keys for every sequence: R = seqs x (query heads of a
// key head) rows meet each key at one reading, which makes them matrix products for the
// 5th-generation tensor cores.  The second ones are the paged attention's (attention.cu) from key P
// on.  A last kernel joins both: every part is (maximum, sum, values) of a softmax.
//
// The prefix kernel.  M = 128 rows of one key head, N = KT keys:
//   S = Q K^T   tcgen05.mma, Q and K in shared memory (K-major), S in tensor memory
//   P = exp(S - m), split in 16-bit parts, written over S
//   O = P V     tcgen05.mma, P from tensor memory, V in shared memory as TMA left it (MN-major)
// q's rows and P are f32.  They enter as hi + lo fp16 (22 bits), for bf16 caches as three bf16 parts
// (24): as in the paged attention, whose place this one takes by size.  (P in two bf16 parts leaves
// room for a third score tile and is a sixth fewer products, but its error of up to 2^-16 of a
// probability was most of the whole: 256 sequences behind 32768 tokens, 2.5e-6 of the norm, now
// 6e-7; an f32 form has 1.4e-6.)  The tensor core truncates where it adds, so the low parts go first,
// an O takes one tile of keys, and sums over tiles are f32 adds in registers.
//
// Roles.  Two warpgroups take every other tile's exponentials each (bf16: half of every tile's), a
// row to a thread; their references (maxima that move only when a score is more than 2^8 above
// them) go from tile to tile through shared memory (bf16: both find them).  A third one adds up the
// tiles' O.  Two threads issue the products, one S, up to three tiles ahead (bf16: two), and one O;
// two warps load pages by TMA, a tile ahead.  e4m3 keys and values are widened to fp16 (exact) by
// four more warps.  At 256 columns a CTA makes 128 columns of O: two CTAs form the same scores.
//
// Work.  A key head has RU row units (128 rows, or half of their columns).  m of them
// (all, up to 16) are a team: CTAs that take the same keys at the same time, so that the
// pages come from memory once, for one CTA of a team, and from L2 for the others.  Teams get equal
// runs of tiles, across heads; a run that crosses into the next head writes two parts.
// Bound by the tensor pipe for large batches: 256 sequences behind 32768 tokens, 8 key heads of 128
// with 4 query heads, bf16, 358 us with the rows' parts and the join: 412 executed GFLOP (q and P in
// three parts) at 1.15 PFLOP/s, 70 % of what a library product reaches in bursts.  Bound by
// starts for small ones (launches, the first pages, the join: 15 to 20 us), which therefore go
// sequence by sequence.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention_frag.cuh"
#include "tc_common.cuh"

namespace moe {

constexpr int kPrefixRows = 128;
constexpr int kTeamMost = 16;

struct PrefixArgs {
  moe_paged_cache c;                   // its block table is not used here
  CacheMap map;
  const uint8_t* q;                    // the rows' parts, as prefix_rows_kernel lays them out
  const float* qscale;                 // score = product * qscale
  const int32_t* pages;
  int* status;
  float2* part_ml;                     // [slot][warpgroup][row] (reference in powers of two, sum)
  float* part_o;                       // [slot][row][column of the unit], for the larger reference
  int rows, row_tiles, keys;           // of a key head, keys of the prefix
  int RU, m, RG, tiles, quota, parts;  // row units, team, row groups; tiles of a head; parts of a unit
  uint32_t total;                      // tiles of all teams
  float cap;
};

template <int DT, int DQ> struct PrefixCfg {
  static constexpr bool kBf = DT == MOE_CACHE_BF16, kE4 = DT == MOE_CACHE_E4M3;
  static constexpr int kParts = kBf ? 3 : 2;
  // bf16 rows of 256: the third part is an operand in tensor memory, there is no room for
  // it beside the others
  static constexpr bool kTmemQ = kBf && DQ == 256;
  static constexpr int kSmemParts = kTmemQ ? 2 : kParts;
  static constexpr int kDV = DQ < 128 ? DQ : 128;
  static constexpr int kHalves = DQ / kDV;
  static constexpr int kKT = DQ == 256 ? 64 : 128;
  static constexpr int kQPart = DQ / 64 * kPrefixRows * 128;
  static constexpr int kQ = kSmemParts * kQPart;
  static constexpr int kK = kKT * DQ * 2, kV = kKT * kDV * 2;
  // stages of keys and of values; of e4m3 the loads need two of their own more than V does
  static constexpr int kStages = kE4 && DQ == 256 ? 1 : DQ == 64 ? 3 : 2;
  static constexpr int kStagesV = kE4 && DQ == 128 ? 1 : kStages;
  static constexpr int kRawK = kE4 ? kKT * (DQ < 128 ? 128 : DQ) : 0, kRawV = kE4 ? kKT * 128 : 0;
  static constexpr int kRawStages = kE4 ? 2 : 0;
  static constexpr int kSmem =
      kQ + kStages * kK + kStagesV * kV + kRawStages * (kRawK + kRawV);
  static constexpr int kThreads = kE4 ? 640 : 512;
  // registers of a thread by warpgroup: what the block was launched with, dealt out again
  static constexpr int kRegsSoft = kE4 ? 104 : 136, kRegsSum = kE4 ? 168 : 176;
  static constexpr int kRegsIssue = kE4 ? 48 : 64, kRegsWiden = 56;
  static constexpr int kRegsAll = 2 * kRegsSoft + kRegsSum + kRegsIssue + (kE4 ? kRegsWiden : 0);
  static_assert(kRegsAll <= 65536 / kThreads / 8 * 8 * (kThreads / 128), "");
  // tensor memory: tiles of S (two parts of P over them, a third one behind them), O, then q's
  // third part
  static constexpr int kTiles = kBf ? 2 : 3;
  // Whether both softmax warpgroups work on a tile, half of its keys each.  With two tiles the
  // pipe would wait for a warpgroup that has a tile to itself (256 sequences behind 32768 tokens,
  // 393 us; 358 shared)
  static constexpr bool kShared = kBf;
  static constexpr int kPCols = kKT / 2 * kParts;
  static constexpr int kOCol = kTiles * kPCols, kQCol = kOCol + kDV;
  static_assert(kQCol + (kTmemQ ? DQ / 2 : 0) <= kTmemCols, "");
  static constexpr uint32_t kIdesc16 = (kBf ? (1u << 7) | (1u << 10) : 0u);
};

struct PrefixShared {
  uint64_t q_full, q_empty, k_full[3], k_empty[3], v_full[3], v_empty[3];
  uint64_t rk_full[2], rk_empty[2], rv_full[2], rv_empty[2];
  uint64_t s_full[3], p_full[3], p_read[3], m_ready[4], o_full, o_empty, drain[2];
  uint32_t tmem;
  int dead;
  // keys of a tile that are there, tile t at t % 8: the loads of tile t + 8 begin when S of tile
  // t + 3 at least has been formed (e4m3 heads of up to 64: two stages of loads, three of keys),
  // in the place of P of tile t.  So its last readers are the warp that issues O of tile t, which
  // meets between the reads and the issue
  uint4 seen[8];
  // references, tile t at t % 4.  Warps of a warpgroup may be two tiles apart where a piece ends
  // between them, since its first tile waits for no reference; four are not, for O of the tile before
  // takes the probabilities of all of them
  float m[4][kPrefixRows];
};

// 32 columns of this thread's row, on their way until tmem_wait_ld
__device__ __forceinline__ void tmem_get32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
      "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
// waits for all loads; r is read behind it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st1(uint32_t addr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(addr), "r"(r) : "memory");
}
__device__ __forceinline__ uint32_t tmem_ld1(uint32_t addr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;"
               : "=r"(r)
               : "r"(addr)
               : "memory");
  return r;
}
// two f32 at a time
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// D (tensor memory) += A (tensor memory) B (shared memory)
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t b_hi,
                                          uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %5, 0;\n mov.b64 db, {%2, %3};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// ---------------------------------------------------------------------------
// q's rows as the tiles of the products: parts of [block of 64 columns][row][128 bytes],
// swizzled, so that a CTA fetches a tile by a few bulk copies.  A warp per row; rows that
// fill up the last tile are zero.  (Done by the CTAs of the prefix kernel themselves, at the start of
// each piece, this took 14000 cycles of theirs.)
// ---------------------------------------------------------------------------
struct PrefixRowsArgs {
  const float* q;
  int64_t q_ss, q_hs;
  uint8_t* tiles;
  float* qscale;
  int G, rows, row_tiles, heads, d, vec;
  float scale, k_scale;
};

template <bool BF, int DQ>
__global__ void __launch_bounds__(256) prefix_rows_kernel(const PrefixRowsArgs A) {
  constexpr int PARTS = BF ? 3 : 2, PART = DQ / 64 * kPrefixRows * 128;
  pdl_wait();
  pdl_trigger();                       // in this order: see the loads of the prefix kernel
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t tile = id / kPrefixRows;                 // head, row tile
  if (tile >= (int64_t)A.heads * A.row_tiles) return;
  const int r = (int)(id % kPrefixRows), head = (int)(tile / A.row_tiles);
  const int at = (int)(tile - (int64_t)head * A.row_tiles) * kPrefixRows + r, s = at / A.G;
  const bool in = at < A.rows;
  const float* q = A.q + s * A.q_ss + ((int64_t)head * A.G + at - (int64_t)s * A.G) * A.q_hs;
  constexpr int PER = DQ / 32, VW = PER < 4 ? PER : 4;   // values of a lane: VW lane + 128 i ..
  float v[PER], mx = 0.f;
#pragma unroll
  for (int i = 0; i < PER; i += VW) {
    const int e = VW * lane + 32 * i;
    if (VW == 4 && A.vec) {
      const float4 f = in && e < A.d ? *reinterpret_cast<const float4*>(q + e)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
      v[i] = f.x;
      v[i + 1] = f.y;
      v[(i + 2) % PER] = f.z;
      v[(i + 3) % PER] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < VW; ++k) v[i + k] = in && e + k < A.d ? q[e + k] : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) mx = fmaxf(mx, fabsf(v[i]));
  mx = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx)));
  // scaled by a power of two to [2^10, 2^11), in two factors, since 2^e may lie outside the
  // exponents of a float; a negative scale turns q, and one that vanishes stays above zero
  const int ex = (int)(__float_as_uint(mx) >> 23);
  const int e = mx > 0.f && ex < 255 ? 137 - max(ex, 1) : 0, e1 = e / 2, e2 = e - e1;
  const float f1 = copysignf(__uint_as_float((uint32_t)(127 + e1) << 23), A.scale);
  const float f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
  if (lane == 0) A.qscale[id] = fmaxf(ldexpf(fabsf(A.scale) * A.k_scale, -e), 1e-30f);
#pragma unroll
  for (int i = 0; i < PER; i += VW) {
    const int c = VW * lane + 32 * i;
    uint8_t* to = A.tiles + tile * PARTS * PART + (c >> 6) * (kPrefixRows * 128) + r * 128 +
                  ((((c & 63) >> 3) ^ (r & 7)) << 4) + (c & 7) * 2;
    uint32_t lo[PARTS], hi[PARTS];
    split2<BF, PARTS>(v[i] * f1 * f2, v[i + 1] * f1 * f2, lo);
    if (VW == 4) split2<BF, PARTS>(v[(i + 2) % PER] * f1 * f2, v[(i + 3) % PER] * f1 * f2, hi);
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      if (VW == 4) *reinterpret_cast<uint2*>(to + k * PART) = make_uint2(lo[k], hi[k]);
      else *reinterpret_cast<uint32_t*>(to + k * PART) = lo[k];
    }
  }
}

// A CTA's pieces: tiles t0 .. t0 + n of row unit `unit` of a head, part j of its parts.
struct PrefixPiece {
  int head, ru, t0, n, slot;
};
struct PrefixRun {
  const PrefixArgs& A;
  uint32_t at, end;
  int team, member;
  __device__ explicit PrefixRun(const PrefixArgs& a) : A(a) {
    team = blockIdx.x / A.m;
    member = blockIdx.x - team * A.m;
    at = (uint32_t)team * A.quota;
    end = min(A.total, at + A.quota);
  }
  __device__ bool next(PrefixPiece& p) {
    while (at < end) {
      const uint32_t unit = at / (uint32_t)A.tiles;    // head and row group
      p.t0 = (int)(at - unit * A.tiles);
      p.n = (int)min(A.tiles - p.t0, end - at);
      const uint32_t first = unit * A.tiles / (uint32_t)A.quota;
      at += p.n;
      p.head = (int)unit / A.RG;
      p.ru = ((int)unit - p.head * A.RG) * A.m + member;
      p.slot = ((int)unit * A.m + member) * A.parts + team - (int)first;
      if (p.ru < A.RU) return true;
    }
    return false;
  }
};

template <int DT, int DQ>
__global__ void __launch_bounds__(PrefixCfg<DT, DQ>::kThreads, 1)
prefix_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
              const PrefixArgs A) {
  using Cfg = PrefixCfg<DT, DQ>;
  constexpr bool BF = Cfg::kBf, E4 = Cfg::kE4;
  constexpr int KT = Cfg::kKT, DV = Cfg::kDV, NS = Cfg::kStages, NV = Cfg::kStagesV, RS = Cfg::kRawStages;
  constexpr int BLK = KT * 128;        // a block of 64 columns of a key or value tile
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ PrefixShared sh;
  static_assert(Cfg::kSmem + (sizeof(PrefixShared) + 1023) / 1024 * 1024 <= 227 * 1024, "");
  uint8_t* const ks = smem + Cfg::kQ;
  uint8_t* const vs = ks + NS * Cfg::kK;
  uint8_t* const rk = vs + NV * Cfg::kV;
  uint8_t* const rv = rk + RS * Cfg::kRawK;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    mbar_init(&sh.q_full, Cfg::kTmemQ ? 9 : 1);  // the copies, and the warps that store third parts
    mbar_init(&sh.q_empty, 1);
    mbar_init(&sh.drain[0], 1);
    mbar_init(&sh.drain[1], 1);
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.k_full[i], E4 ? 4 : 1);
      mbar_init(&sh.v_full[i], E4 ? 4 : 1);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.rk_full[i], 1);
      mbar_init(&sh.rv_full[i], 1);
      mbar_init(&sh.rk_empty[i], 4);
      mbar_init(&sh.rv_empty[i], 4);
    }
    for (int i = 0; i < Cfg::kTiles; ++i) {
      mbar_init(&sh.s_full[i], 2);
      mbar_init(&sh.p_full[i], Cfg::kShared ? 256 : 128);
      mbar_init(&sh.p_read[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&sh.m_ready[i], 128);
    mbar_init(&sh.o_full, 2);
    mbar_init(&sh.o_empty, 128);
    sh.dead = 0;
    fence_mbar_init();
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  const uint32_t tmem = tc_alloc_all(&sh.tmem, warp);
  pdl_trigger();
  // Keys and values need not wait for q's rows: the kernel that lays those out lets this one
  // start when all before it is done.
  if (warp != 13 && warp != 14) pdl_wait();

  // Bounded; after a timeout anywhere in the CTA no wait takes long any more, nothing more
  // is issued, and the kernel ends.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!mbar_test(bar, parity) && !*(volatile int*)&sh.dead && !mbar_wait(bar, parity)) {
      *(volatile int*)&sh.dead = 1;
      set_status(A.status, MOE_STATUS_TIMEOUT);
    }
  };
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) {
    wait(bar, parity);
    __syncwarp();
  };
  PrefixRun run(A);
  PrefixPiece p;
  constexpr int NT = Cfg::kTiles, PC = Cfg::kPCols;
  int n = 0;                           // tiles so far: S n % NT, not shared: warpgroup n & 1

  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoft));
    const int w = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tm = tmem + lanes;
    while (run.next(p)) {
      const int64_t tile = (int64_t)p.head * A.row_tiles + p.ru / Cfg::kHalves;
      const float qscale = A.qscale[tile * kPrefixRows + row];
      if (Cfg::kTmemQ) {               // third parts: this thread's row, half of its columns
        asm volatile("bar.sync 1, 256;" ::: "memory");     // S of the piece before has been formed
        const uint8_t* q = A.q + (tile * Cfg::kParts + 2) * Cfg::kQPart + row * 128;
#pragma unroll 1
        for (int c = w * (DQ / 2); c < (w + 1) * (DQ / 2); c += 64) {
          uint32_t x[32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(
                q + (c >> 6) * (kPrefixRows * 128) + ((i ^ (row & 7)) << 4));
            x[4 * i] = v.x;
            x[4 * i + 1] = v.y;
            x[4 * i + 2] = v.z;
            x[4 * i + 3] = v.w;
          }
          tmem_st32(tm + Cfg::kQCol + c / 2, x);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full);
      }
      const float to_cap = A.cap > 0.f ? fminf(qscale / A.cap, 3e38f) : 0.f;
      const float from_cap = A.cap * kLog2e;
      const float x2 = A.cap > 0.f ? 1.f : qscale * kLog2e;
      float m = -INFINITY, l = 0.f;    // l is a sum for the reference m
      const int start = n, end = n + p.n;
      // this warpgroup's columns of its tiles
      constexpr int COLS = Cfg::kShared ? KT / 2 : KT;
      const int c0 = Cfg::kShared ? w * COLS : 0, c1 = c0 + COLS;
      for (int t = Cfg::kShared ? n : n + ((n ^ w) & 1); t < end; t += Cfg::kShared ? 1 : 2) {
        const int b = t % NT;
        const uint32_t S = tm + (uint32_t)(b * PC);
        warp_wait(&sh.s_full[b], (t / NT) & 1);
        tc_fence_after();
        const uint32_t* seen = &sh.seen[t % 8].x;
        const uint32_t all = seen[0] & seen[1] & seen[2] & seen[3];
        // The loops over columns stay loops, and what few tiles need stands apart: with all of
        // it unrolled a tile's code is some 50 KB, and both warpgroups wait for instructions
        // (32768 keys, 1024 rows a head, bf16: 686 us instead of 440)
        float mx = -INFINITY;
        if (all != 0xffffffffu || A.cap > 0.f) {
          // ---- keys that are not there become minus infinity, scores cap tanh(score / cap) log2 e
#pragma unroll 1
          for (int c = c0; c < c1; c += 32) {
            uint32_t v[32];
            tmem_get32(S + c, v);
            tmem_wait_ld(v);
            const uint32_t bits = seen[c / 32];
            float big = 0.f;           // what is not there picks no form of tanh
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (!((bits >> k) & 1u)) v[k] = A.cap > 0.f ? 0u : 0xff800000u;
              big = fmaxf(big, fabsf(__uint_as_float(v[k])));
            }
            if (A.cap > 0.f) {
              if (__any_sync(0xffffffffu, !(big * to_cap < 0.5f))) {
#pragma unroll
                for (int k = 0; k < 32; ++k)
                  v[k] = __float_as_uint(from_cap * tanhf(__uint_as_float(v[k]) * to_cap));
              } else {
                // Lambert's continued fraction, off by less than 2^-29 of tanh y for |y| < 1/2
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float y = __uint_as_float(v[k]) * to_cap, z = y * y;
                  const float num = fmaf(z, z + 105.f, 945.f);
                  const float den = fmaf(z, fmaf(15.f, z, 420.f), 945.f);
                  v[k] = __float_as_uint(from_cap * __fdividef(y * num, den));
                }
              }
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((bits >> k) & 1u)) v[k] = 0xff800000u;
            }
            tmem_st32(S + c, v);
          }
          tmem_wait_st();
        }
        // ---- the largest score
#pragma unroll 1
        for (int c = c0; c < c1; c += 64) {
          uint32_t v[32], u[32];
          tmem_get32(S + c, v);
          tmem_get32(S + (COLS < 64 ? c : c + 32), u);
          tmem_wait_ld(v);
          tmem_wait_ld(u);
          float top[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int k = 0; k < 32; ++k)
            top[k & 3] = fmaxf(top[k & 3], fmaxf(__uint_as_float(v[k]), __uint_as_float(u[k])));
          mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        }
        mx *= x2;
        // ---- the reference: that of the tile before unless a score is more than 2^8 above it.  Of
        // a shared tile both warpgroups find it from both maxima, else the one before is in the other
        // warpgroup's hands
        float to = mx;
        if (Cfg::kShared) {
          // each warpgroup leaves its maximum where the other one's third parts begin, which will
          // overwrite it itself (shared memory is full)
          const uint32_t third = S + KT;
          tmem_st1(third + (w ^ 1) * (KT / 4), __float_as_uint(mx));
          tmem_wait_st();
          tc_fence_before();
          asm volatile("bar.sync 2, 256;" ::: "memory");
          tc_fence_after();
          to = mx = fmaxf(mx, __uint_as_float(tmem_ld1(third + w * (KT / 4))));
          if (t > start && !(mx > m + 8.f)) to = m;
        } else if (t > start) {
          warp_wait(&sh.m_ready[(t - 1) & 3], ((t - 1) >> 2) & 1);
          const float before = sh.m[(t - 1) & 3][row];
          to = mx > before + 8.f ? mx : before;
        }
        if (to != m) {
          l *= ex2(m - to);
          m = to;
        }
        if (!Cfg::kShared || w == 0) sh.m[t & 3][row] = m;
        if (!Cfg::kShared) mbar_arrive(&sh.m_ready[t & 3]);
        const float shift = kPShift - (m == -INFINITY ? 0.f : m);
        // ---- probabilities: 32 keys' hi parts in 16 columns, then their second parts
        const uint64_t x22 = pack2(x2, x2), shift2 = pack2(shift, shift);
        uint64_t sum0 = 0, sum1 = 0;
#pragma unroll 1
        for (int c = c0; c < c1; c += 32) {
          uint32_t v[32], x[32], y[16];
          tmem_get32(S + c, v);
          tmem_wait_ld(v);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            float a, b;
            unpack2(fma2(pack2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), x22, shift2), a, b);
            a = ex2(a);
            b = ex2(b);
            const uint64_t ab = pack2(a, b);
            if (k & 2) sum1 = add2(sum1, ab);
            else sum0 = add2(sum0, ab);
            uint32_t part[Cfg::kParts];
            split2<BF, Cfg::kParts>(a, b, part);
            x[k / 2] = part[0];
            x[16 + k / 2] = part[1];
            y[k / 2] = part[Cfg::kParts - 1];
          }
          tmem_st32(S + c, x);
          if (Cfg::kParts == 3) tmem_st16(S + KT + c / 2, y);
        }
        float s0, s1;
        unpack2(add2(sum0, sum1), s0, s1);
        l += s0 + s1;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.p_full[b]);
      }
      n = end;
      if (p.ru / Cfg::kHalves * kPrefixRows + row < A.rows)
        A.part_ml[((int64_t)p.slot * 2 + w) * kPrefixRows + row] = make_float2(m, l);
    }
  } else if (warp < 12) {
    // ---- the sums of O, a row to a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSum));
    const int row = (warp & 3) * 32 + lane;
    const uint32_t O = tmem + ((uint32_t)((warp & 3) * 32) << 16) + Cfg::kOCol;
    while (run.next(p)) {
      float o[DV], m = -INFINITY;
#pragma unroll
      for (int c = 0; c < DV; ++c) o[c] = 0.f;
      const int start = n;
      for (const int end = n + p.n; n < end; ++n) {
        warp_wait(&sh.o_full, n & 1);
        tc_fence_after();
        const float to = sh.m[n & 3][row];
        if (n > start && __any_sync(0xffffffffu, to != m)) {
          const float f = to != m ? ex2(m - to) : 1.f;
#pragma unroll
          for (int c = 0; c < DV; ++c) o[c] *= f;
        }
        m = to;
#pragma unroll
        for (int c = 0; c < DV; c += 32) {
          uint32_t v[32];
          tmem_get32(O + c, v);
          tmem_wait_ld(v);
          if (c + 32 == DV) {
            tc_fence_before();
            mbar_arrive(&sh.o_empty);
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) o[c + k] += __uint_as_float(v[k]);
        }
      }
      if (p.ru / Cfg::kHalves * kPrefixRows + row < A.rows) {
        float* to = A.part_o + ((int64_t)p.slot * kPrefixRows + row) * DV;
#pragma unroll
        for (int c = 0; c < DV; c += 4)
          *reinterpret_cast<float4*>(to + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
      }
    }
  } else if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsIssue));
    // descriptors: rows of 128 bytes, 8 of them 1024 bytes on; of V (MN-major) 64 columns in
    // a row, the next 64 BLK on
    const uint32_t desc_hi = (uint32_t)(sw128_desc(smem) >> 32);
    if (warp == 12) {
      // ---- S.  A thread of its own: between a tile's products the issuing thread is busy with
      // barriers for some 700 cycles, in which the other one's products run (a tile of
      // bf16 4600 cycles with both in one thread, 4000 in two)
      if (lane == 0) {
        const uint32_t q_lo = (uint32_t)sw128_desc(smem), k_lo = (uint32_t)sw128_desc(ks);
        const uint32_t is = tc_idesc(128, KT) | Cfg::kIdesc16;
        uint32_t pieces = 0;
        while (run.next(p)) {
          wait(&sh.q_full, pieces++ & 1);
          for (const int end = n + p.n; n < end; ++n) {
            const int st = n % NS, b = n % NT;
            wait(&sh.k_full[st], (n / NS) & 1);
            if (n >= NT) wait(&sh.p_read[b], (n / NT - 1) & 1);
            if (*(volatile int*)&sh.dead) break;
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(b * PC);
            const uint32_t kb = k_lo + (uint32_t)(st * Cfg::kK >> 4);
#pragma unroll
            for (int k = Cfg::kParts - 1; k >= 0; --k)
#pragma unroll
              for (int c = 0; c < DQ / 16; ++c) {
                const uint32_t kc = kb + (uint32_t)(((c >> 2) * BLK + (c & 3) * 32) >> 4);
                const uint32_t more = k < Cfg::kParts - 1 || c > 0;
                if (Cfg::kTmemQ && k == 2)
                  tc_mma_ts(d, tmem + Cfg::kQCol + 8 * c, kc, desc_hi, is, more);
                else
                  tc_mma_lo(d, q_lo + (uint32_t)((k * Cfg::kQPart + (c >> 2) * kPrefixRows * 128 +
                                                  (c & 3) * 32) >> 4), kc, desc_hi, is, more);
              }
            mbar_arrive(&sh.s_full[b]);
            tc_commit(&sh.s_full[b]);
            tc_commit(&sh.k_empty[st]);
          }
          // (Not by k_empty: a parity tells a phase from the next only, and the loads of e4m3 may be
          // further ahead of these products than its stages)
          tc_commit(&sh.q_empty);
        }
        tc_commit(&sh.drain[0]);       // nothing is in flight when the tensor memory goes
        mbar_wait(&sh.drain[0], 0);
      }
    } else if (warp == 15) {
      // ---- O
      const uint32_t v_lo = ((smem_u32(vs) >> 4) & 0x3FFF) | (uint32_t)(BLK >> 4) << 16;
      const uint32_t io = tc_idesc(128, DV) | Cfg::kIdesc16 | (1u << 16);
      while (run.next(p)) {
        for (const int end = n + p.n; n < end; ++n) {
          const int st = n % NV, b = n % NT;
          warp_wait(&sh.v_full[st], (n / NV) & 1);
          warp_wait(&sh.p_full[b], (n / NT) & 1);
          const uint4 seen = sh.seen[n % 8];
          if ((seen.x & seen.y & seen.z & seen.w) != 0xffffffffu) {
            // nothing of a row that is not seen counts
            const uint32_t word[4] = {seen.x, seen.y, seen.z, seen.w};
#pragma unroll
            for (int j = 0; j < KT / 32; ++j)
              if (!((word[j] >> lane) & 1u))
                for (int c = 0; c < DV / 64 * 8; ++c)
                  *reinterpret_cast<uint4*>(vs + st * Cfg::kV + (c >> 3) * BLK +
                                            (32 * j + lane) * 128 + (c & 7) * 16) =
                      make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
          }
          __syncwarp();                // all lanes have read `seen`
          if (lane == 0) {
            if (n > 0) wait(&sh.o_empty, (n - 1) & 1);
            if (!*(volatile int*)&sh.dead) {
              tc_fence_after();
              const uint32_t a = tmem + (uint32_t)(b * PC), d = tmem + Cfg::kOCol;
              const uint32_t vb = v_lo + (uint32_t)(st * Cfg::kV >> 4);
#pragma unroll
              for (int k = Cfg::kParts - 1; k >= 0; --k)
#pragma unroll
                for (int c = 0; c < KT / 16; ++c)
                  tc_mma_ts(d, a + (k < 2 ? 32 * (c >> 1) + 16 * k + 8 * (c & 1) : KT + 8 * c),
                            vb + (uint32_t)(c * 2048 >> 4), desc_hi, io,
                            k < Cfg::kParts - 1 || c > 0);
              mbar_arrive(&sh.o_full);           // the reference is there too
              tc_commit(&sh.o_full);
              tc_commit(&sh.p_read[b]);
              tc_commit(&sh.v_empty[st]);
            }
          }
          __syncwarp();
        }
      }
      if (lane == 0) {
        tc_commit(&sh.drain[1]);
        mbar_wait(&sh.drain[1], 0);
      }
    } else {
      // ---- loads: keys, values
      const bool keys = warp == 13;
      constexpr int LINE = E4 ? 128 : 64;                  // elements of a line
      const int RING = E4 ? RS : keys ? NS : NV;
      uint64_t* full = E4 ? (keys ? sh.rk_full : sh.rv_full) : keys ? sh.k_full : sh.v_full;
      uint64_t* empty = E4 ? (keys ? sh.rk_empty : sh.rv_empty) : keys ? sh.k_empty : sh.v_empty;
      const CUtensorMap* map = keys ? &kmap : &vmap;
      const int bytes = keys ? (E4 ? Cfg::kRawK : Cfg::kK) : E4 ? Cfg::kRawV : Cfg::kV;
      const int lines = bytes / BLK;
      uint8_t* const ring = keys ? (E4 ? rk : ks) : E4 ? rv : vs;
      const uint32_t ps = A.c.page_size, shift = A.map.box_shift;
      const int boxes = KT >> shift;
      uint32_t pieces = 0;
      while (run.next(p)) {
        const int x0 = keys ? 0 : p.ru % Cfg::kHalves * 128;     // this unit's columns of V
        // pages of this lane's boxes (lane, lane + 32, ...), fetched a tile ahead
        int page[4];
        uint32_t slot[4];
        auto fetch = [&](int tile) {
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint32_t key = (uint32_t)tile * KT + ((uint32_t)(lane + 32 * b) << shift);
            page[b] = -1;
            slot[b] = 0xffffffffu;     // no such box
            if (lane + 32 * b < boxes && key < (uint32_t)A.keys) {
              const uint32_t pg = key / ps;
              page[b] = A.pages[pg];
              slot[b] = key - pg * ps;
            }
          }
        };
        fetch(p.t0);
        for (int i = 0; i < p.n; ++i, ++n) {
          const int st = n % RING;
          const uint32_t round = n / RING;
          if (round > 0) warp_wait(&empty[st], (round - 1) & 1);
          if (__any_sync(0xffffffffu, *(volatile int*)&sh.dead)) break;
          uint32_t count = 0, ok[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const bool there = page[b] >= 0 && page[b] < A.c.pages;
            if (keys && !there && slot[b] != 0xffffffffu) set_status(A.status, MOE_STATUS_BAD_PAGE);
            ok[b] = __ballot_sync(0xffffffffu, there);
            count += __popc(ok[b]);
            if (!there) page[b] = -1;
          }
          if (keys && lane < 4) {      // keys of the tile that are there
            uint32_t bits = 0xffffffffu;
            if (count != (uint32_t)boxes && 32 * lane < KT)
              for (int k = 0; k < 32; ++k) {
                const int box = (32 * lane + k) >> shift;
                const uint32_t word = box < 32 ? ok[0] : box < 64 ? ok[1] : box < 96 ? ok[2] : ok[3];
                if (!((word >> (box & 31)) & 1u)) bits &= ~(1u << k);
              }
            (&sh.seen[n % 8].x)[lane] = bits;
          }
          __syncwarp();
          if (lane == 0) mbar_expect_tx(&full[st], (count << shift) * 128u * (uint32_t)lines);
          __syncwarp();
          const uint32_t to = smem_u32(ring) + st * bytes;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (page[b] >= 0)
              for (int c = 0; c < lines; ++c)
                tma_load_3d(to + c * BLK + ((lane + 32 * b) << shift) * 128, map, x0 + c * LINE,
                            page[b] * A.map.page_units + p.head * A.map.head_units, (int)slot[b],
                            &full[st]);
          __syncwarp();
          if (keys && i == 0) {        // q, once the products of the piece before are done
            if (pieces > 0) warp_wait(&sh.q_empty, (pieces - 1) & 1);
            else pdl_wait();
            ++pieces;
            if (lane == 0 && !*(volatile int*)&sh.dead) {
              const int64_t tile = (int64_t)p.head * A.row_tiles + p.ru / Cfg::kHalves;
              mbar_expect_tx(&sh.q_full, Cfg::kQ);
#pragma unroll 1
              for (int c = 0; c < Cfg::kQ; c += 16384)
                bulk_g2s_plain(smem + c, A.q + tile * Cfg::kParts * Cfg::kQPart + c, 16384, &sh.q_full);
            }
            __syncwarp();
          }
          if (i + 1 < p.n) fetch(p.t0 + i + 1);
        }
      }
      // after a timeout copies may still be under way: give them time to land
      if (*(volatile int*)&sh.dead)
        for (int k = 0; k < 2; ++k) {
          for (int s = 0; s < RING; ++s) mbar_wait(&full[s], k);
          if (keys) mbar_wait(&sh.q_full, k);
        }
    }
  } else if (E4) {
    // ---- e4m3 -> fp16, rows of 128 bytes swizzled on both sides
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsWiden));
    constexpr int R = RS ? RS : 1;
    const int id = tid - 512;
    auto widen = [&](const uint8_t* from, uint8_t* to, int columns) {
      constexpr int SHARE = 128 / KT;  // threads of a row
      const int r = id % KT, c0 = id / KT;
#pragma unroll 2
      for (int c = c0; c < columns / 16; c += SHARE) {
        const uint4 v = *reinterpret_cast<const uint4*>(from + (c >> 3) * BLK + r * 128 +
                                                        (((c & 7) ^ (r & 7)) << 4));
        uint4 a, b;
        e4m3x4_f16x2(v.x, a.x, a.y);
        e4m3x4_f16x2(v.y, a.z, a.w);
        e4m3x4_f16x2(v.z, b.x, b.y);
        e4m3x4_f16x2(v.w, b.z, b.w);
        uint8_t* row = to + (c >> 2) * BLK + r * 128;
        const int ch = 2 * (c & 3);
        *reinterpret_cast<uint4*>(row + ((ch ^ (r & 7)) << 4)) = a;
        *reinterpret_cast<uint4*>(row + (((ch + 1) ^ (r & 7)) << 4)) = b;
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    auto widen_keys = [&](int t) {
      const int rs = t % R, st = t % NS, round = t / NS;
      warp_wait(&sh.rk_full[rs], (t / R) & 1);
      if (round > 0) warp_wait(&sh.k_empty[st], (round - 1) & 1);
      widen(rk + rs * Cfg::kRawK, ks + st * Cfg::kK, DQ);
      if (lane == 0) {
        mbar_arrive(&sh.k_full[st]);
        mbar_arrive(&sh.rk_empty[rs]);
      }
    };
    auto widen_values = [&](int t) {
      const int rs = t % R, st = t % NV, round = t / NV;
      warp_wait(&sh.rv_full[rs], (t / R) & 1);
      if (round > 0) warp_wait(&sh.v_empty[st], (round - 1) & 1);
      widen(rv + rs * Cfg::kRawV, vs + st * Cfg::kV, DV);
      if (lane == 0) {
        mbar_arrive(&sh.v_full[st]);
        mbar_arrive(&sh.rv_empty[rs]);
      }
    };
    while (run.next(p)) {
      // keys run a tile ahead of values
      for (int i = 0; i <= p.n; ++i) {
        if (i < p.n && (i == 0 || NS > 1)) widen_keys(n + i);
        if (i > 0) widen_values(n + i - 1);
        if (i > 0 && i < p.n && NS == 1) widen_keys(n + i);
        if (*(volatile int*)&sh.dead) break;
      }
      n += p.n;
    }
  }
  tc_dealloc_all(tmem, warp);
}

// ---------------------------------------------------------------------------
// The join: a warp per row of the output.
// ---------------------------------------------------------------------------
struct PrefixJoinArgs {
  const float2* part_ml;
  const float* part_o;
  const int32_t* seq_lens;
  const float2* own;                   // (maximum, sum) of a sequence's own keys
  float *out, *lse;
  int seqs, hq, G, d, DV, halves, keys;
  int RU, m, RG, tiles, quota, parts;
  float v_scale;
};

__global__ void __launch_bounds__(256) prefix_join_kernel(const PrefixJoinArgs A) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (id >= (int64_t)A.seqs * A.hq) return;
  const int s = (int)(id / A.hq), h = (int)(id - (int64_t)s * A.hq), head = h / A.G;
  float* out = A.out + id * A.d;
  // Own keys' maximum and sum come apart, as the parts' do: one logarithm of both, rounded, would
  // leave an error of |lse| 2^-23 in the weight of own keys against the prefix
  const float2 own = A.own[id];
  if (A.seq_lens[s] < A.keys) {        // not behind this prefix: all of its keys are its own
    if (lane == 0 && A.lse) A.lse[id] = (own.x + (log2f(own.y) - kPShift)) * kLn2;
    return;
  }
  const int r = s * A.G + h - head * A.G;
  for (int half = 0; half < A.halves; ++half) {
    const int ru = r / kPrefixRows * A.halves + half, row = r % kPrefixRows;
    const int rg = ru / A.m, unit = head * A.RG + rg;
    const int first = unit * A.tiles / A.quota;
    const int n = ((unit + 1) * A.tiles - 1) / A.quota - first + 1;
    const int64_t slot = (int64_t)(unit * A.m + ru - rg * A.m) * A.parts;
    const float2* ml = A.part_ml + slot * 2 * kPrefixRows + row;
    const float* po = A.part_o + (slot * kPrefixRows + row) * A.DV;
    float M = own.x;
    for (int j = lane; j < 2 * n; j += 32) M = fmaxf(M, ml[(int64_t)j * kPrefixRows].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ms = M == -INFINITY ? 0.f : M;
    const float wo = own.y * ex2(own.x - ms - kPShift);
    const int c = 4 * lane, col = half * A.DV + c;
    const bool mine = c < A.DV && col < A.d;
    float L = wo;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    if (mine) {
      const float4 v = *reinterpret_cast<const float4*>(out + col);
      y = make_float4(v.x * wo, v.y * wo, v.z * wo, v.w * wo);
    }
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float2 p = ml[(int64_t)(2 * j) * kPrefixRows], q = ml[(int64_t)(2 * j + 1) * kPrefixRows];
      const float wp = ex2(p.x - ms - kPShift), wq = ex2(q.x - ms - kPShift);
      const float wv = fmaxf(wp, wq) * A.v_scale;
      L = fmaf(p.y, wp, fmaf(q.y, wq, L));
      if (mine) {
        const float4 v = *reinterpret_cast<const float4*>(po + (int64_t)j * kPrefixRows * A.DV + c);
        y.x = fmaf(v.x, wv, y.x);
        y.y = fmaf(v.y, wv, y.y);
        y.z = fmaf(v.z, wv, y.z);
        y.w = fmaf(v.w, wv, y.w);
      }
    }
    const float norm = L == 0.f ? 0.f : 1.f / L;
    if (mine)
      *reinterpret_cast<float4*>(out + col) =
          make_float4(y.x * norm, y.y * norm, y.z * norm, y.w * norm);
    if (half == 0 && lane == 0 && A.lse) A.lse[id] = (M + log2f(L)) * kLn2;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct PrefixPlan {
  int dq, dv, halves, kt, RU, m, RG, teams;
  int64_t units, slots;                // (head, row group)s, parts at most
};

static PrefixPlan prefix_plan(int seqs, int q_heads, int kv_heads, int head_dim) {
  PrefixPlan p;
  p.dq = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
  p.dv = std::min(p.dq, 128);
  p.halves = p.dq / p.dv;
  p.kt = p.dq == 256 ? 64 : 128;
  const int64_t rows = (int64_t)std::max(seqs, 1) * (q_heads / kv_heads);
  p.RU = (int)((rows + kPrefixRows - 1) / kPrefixRows) * p.halves;
  p.RG = (p.RU + kTeamMost - 1) / kTeamMost;
  p.m = (p.RU + p.RG - 1) / p.RG;
  p.teams = std::max(1, sm_count() / p.m);
  p.units = (int64_t)kv_heads * p.RG;
  // a unit in (tiles - 1) / quota + 2 <= teams / units + 2 parts.  (Of all CTAs, not of those in
  // teams, so that a workspace for more sequences is never smaller)
  p.slots = sm_count() + 2 * p.m * p.units;
  return p;
}

struct PrefixSpace {
  float2* own;
  float2* ml;
  float *o, *qscale;
  uint8_t* q;
  size_t own_bytes;                    // of the attention behind the prefix, in front
};

static int prefix_workspace(const PrefixPlan& p, int seqs, int q_heads, int kv_heads, int head_dim,
                            void* ws, PrefixSpace* out, size_t* bytes) {
  Carve cv = {static_cast<uint8_t*>(ws), 0, 0};
  size_t own = 0;                      // starts with the status
  MOE_CHECK(moe_paged_attention_workspace_bytes(seqs, q_heads, kv_heads, head_dim, &own));
  cv.take<uint8_t>(own);
  float2* stats = cv.take<float2>((size_t)seqs * q_heads);
  float2* ml = cv.take<float2>((size_t)p.slots * 2 * kPrefixRows);
  float* o = cv.take<float>((size_t)p.slots * kPrefixRows * p.dv);
  const size_t rows = (size_t)kv_heads * (p.RU / p.halves) * kPrefixRows;
  float* qscale = cv.take<float>(rows);
  uint8_t* q = cv.take<uint8_t>(rows * p.dq * 3 * 2);    // three parts at most
  if (out) *out = {stats, ml, o, qscale, q, own};
  *bytes = align_up(cv.used, 256);
  return MOE_OK;
}

// Whether the products over all rows take less time than the paged attention of each sequence over
// the prefix, microseconds.  Fitted to both at 2 to 128 sequences behind 256 to 16384 tokens, heads of 64,
// 128 and 256 of all types: the paged attention reads (mostly from L2) 7.5 MB a microsecond, 4.6 of e4m3; the
// kernels here take 13 (28 at 256 columns) for their launches and starts and 3 (5) a tile.
// 32 / 8 heads of 128, fp16: 8 x 4096 tokens 25.5 each, 28 together; 32 x 4096 73 and 31; 2 x 1024 10 and 22.
// bf16: 26 and 30, 74 and 33, 11 and 24.
static bool together_pays(const moe_paged_cache& c, const PrefixPlan& p, int keys, int quota) {
  const double bytes = 2.0 * cache_elem_bytes(c.dtype) * c.seqs * c.kv_heads * c.head_dim * keys;
  const double each = bytes / (c.dtype == MOE_CACHE_E4M3 ? 4.6e6 : 7.5e6);
  return (p.dq == 256 ? 28.0 + 5.0 * quota : 13.0 + 3.0 * quota) < each;
}

template <int DT, int DQ>
static int launch_prefix(PrefixArgs& a, const PrefixRowsArgs& rows, int grid, cudaStream_t s) {
  using Cfg = PrefixCfg<DT, DQ>;
  static std::atomic<uint64_t> ready{0};
  auto kern = prefix_kernel<DT, DQ>;
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((ready.load() >> dev) & 1)) {
    MOE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    // the warpgroups' shares come out of what the block is launched with
    cudaFuncAttributes fa;
    MOE_CUDA(cudaFuncGetAttributes(&fa, kern));
    MOE_REQUIRE(fa.numRegs * (Cfg::kThreads / 128) >= Cfg::kRegsAll, MOE_ERR_CUDA,
                "the kernel was built with %d registers", fa.numRegs);
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  CUtensorMap kmap, vmap;
  MOE_CHECK(make_cache_map(&kmap, a.c, a.c.k, Cfg::kKT, &a.map));
  MOE_CHECK(make_cache_map(&vmap, a.c, a.c.v, Cfg::kKT, &a.map));
  const int64_t blocks = (int64_t)rows.heads * rows.row_tiles * (kPrefixRows / 8);
  MOE_REQUIRE(blocks <= 0x7fffffff, MOE_ERR_UNSUPPORTED, "%d rows are too many", rows.rows);
  MOE_CUDA(launch_pdl(prefix_rows_kernel<Cfg::kBf, DQ>, dim3((unsigned)blocks), dim3(256), 0, s,
                      rows));
  MOE_CUDA(launch_pdl(kern, dim3((unsigned)grid), dim3(Cfg::kThreads), Cfg::kSmem, s, kmap, vmap, a));
  return MOE_OK;
}

template <int DT>
static int launch_prefix_dt(PrefixArgs& a, const PrefixRowsArgs& r, int dq, int grid,
                            cudaStream_t s) {
  return dq == 64    ? launch_prefix<DT, 64>(a, r, grid, s)
         : dq == 128 ? launch_prefix<DT, 128>(a, r, grid, s)
                     : launch_prefix<DT, 256>(a, r, grid, s);
}

}  // namespace moe

extern "C" {

int moe_prefix_attention_workspace_bytes(int seqs, int q_heads, int kv_heads, int head_dim,
                                         size_t* bytes) {
  MOE_REQUIRE(bytes, MOE_ERR_INVALID, "null output pointer");
  MOE_REQUIRE(seqs >= 0 && kv_heads > 0 && head_dim > 0 && head_dim <= moe::kMaxHeadDim,
              MOE_ERR_INVALID, "bad attention shape");
  MOE_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0, MOE_ERR_INVALID,
              "%d query heads for %d key heads", q_heads, kv_heads);
  return moe::prefix_workspace(moe::prefix_plan(seqs, q_heads, kv_heads, head_dim), seqs, q_heads,
                               kv_heads, head_dim, nullptr, nullptr, bytes);
}

int moe_prefix_attention_record(const moe_prefix_attention_args* r) {
  MOE_REQUIRE(r, MOE_ERR_INVALID, "null arguments");
  const moe_paged_attention_args& t = r->attention;
  moe::PrefixArgs a = {};
  MOE_CHECK(moe::check_attention(t, a.c));
  MOE_REQUIRE(r->prefix_pages >= 0 && r->prefix_pages <= a.c.table_width, MOE_ERR_INVALID,
              "a prefix of %d pages in tables of %d", r->prefix_pages, a.c.table_width);
  MOE_REQUIRE(t.window == 0, MOE_ERR_UNSUPPORTED, "a window does not go with a shared prefix");
  if (a.c.seqs == 0) return MOE_OK;
  MOE_REQUIRE(r->prefix || r->prefix_pages == 0, MOE_ERR_INVALID, "null pointer");
  // (whatever form the sizes choose; the paged attention alone takes any)
  MOE_REQUIRE((uintptr_t)t.out % 16 == 0 || r->prefix_pages == 0 || r->form == MOE_PREFIX_EACH,
              MOE_ERR_INVALID, "out must be 16-byte aligned");
  MOE_REQUIRE(r->form >= MOE_PREFIX_AUTO && r->form <= MOE_PREFIX_TOGETHER, MOE_ERR_INVALID,
              "form %d not known", r->form);
  const int S = a.c.seqs, d = a.c.head_dim, P = r->prefix_pages * a.c.page_size;
  const moe::PrefixPlan p = moe::prefix_plan(S, t.q_heads, a.c.kv_heads, d);
  moe::PrefixSpace ws;
  size_t need = 0;
  MOE_CHECK(moe::prefix_workspace(p, S, t.q_heads, a.c.kv_heads, d, t.workspace, &ws, &need));
  MOE_REQUIRE(t.workspace_bytes >= need, MOE_ERR_WORKSPACE, "workspace %zu < %zu bytes",
              t.workspace_bytes, need);
  const int G = t.q_heads / a.c.kv_heads;
  a.q = ws.q;
  a.qscale = ws.qscale;
  a.pages = r->prefix;
  a.status = static_cast<int*>(t.workspace);
  a.part_ml = ws.ml;
  a.part_o = ws.o;
  a.rows = S * G;
  a.row_tiles = p.RU / p.halves;
  a.keys = P;
  a.RU = p.RU;
  a.m = p.m;
  a.RG = p.RG;
  a.tiles = (P + p.kt - 1) / p.kt;
  const int64_t total = p.units * a.tiles;
  const int64_t quota = std::max<int64_t>(1, (total + p.teams - 1) / p.teams);
  MOE_REQUIRE(total < (1ll << 30) && (int64_t)S * G < (1ll << 30) && p.slots < (1ll << 30),
              MOE_ERR_UNSUPPORTED, "%d sequences behind a prefix of %d tokens are too many", S, P);
  a.total = (uint32_t)total;
  a.quota = (int)quota;
  a.parts = (a.tiles - 1) / a.quota + 2;
  MOE_REQUIRE(p.units * p.m * a.parts <= p.slots, MOE_ERR_INVALID, "parts %d", a.parts);
  const int grid = (int)((total + quota - 1) / quota) * p.m;
  if (P == 0 || r->form == MOE_PREFIX_EACH ||
      (r->form == MOE_PREFIX_AUTO && !moe::together_pays(a.c, p, P, a.quota)))
    return moe::attention_from(t, 0);
  a.cap = t.softcap;
  const int vec = (uintptr_t)t.q % 16 == 0 && (S == 1 || t.q_seq_stride % 4 == 0) &&
                  (t.q_heads == 1 || t.q_head_stride % 4 == 0);
  const moe::PrefixRowsArgs rows = {t.q, t.q_seq_stride, t.q_head_stride, ws.q, ws.qscale, G,
                                    a.rows, a.row_tiles, a.c.kv_heads, d, vec, t.scale, a.c.k_scale};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(t.stream);
  // the keys behind the prefix: checks q and out, and writes out
  moe_paged_attention_args own = t;
  own.workspace_bytes = ws.own_bytes;
  {
    ::moe::ProfScope _prof(MOE_K_PREFIX, s);
    MOE_CHECK(a.c.dtype == MOE_CACHE_F16 ? moe::launch_prefix_dt<MOE_CACHE_F16>(a, rows, p.dq, grid, s)
              : a.c.dtype == MOE_CACHE_BF16
                  ? moe::launch_prefix_dt<MOE_CACHE_BF16>(a, rows, p.dq, grid, s)
                  : moe::launch_prefix_dt<MOE_CACHE_E4M3>(a, rows, p.dq, grid, s));
  }
  MOE_CHECK(moe::attention_from(own, P, ws.own));
  const moe::PrefixJoinArgs j = {ws.ml, ws.o, t.seq_lens, ws.own, t.out, t.lse,
                                 S, t.q_heads, G, d, p.dv, p.halves, P, a.RU, a.m, a.RG,
                                 a.tiles, a.quota, a.parts, a.c.v_scale};
  {
    ::moe::ProfScope _prof(MOE_K_PREFIX, s);
    const int64_t blocks = ((int64_t)S * t.q_heads + 7) / 8;
    MOE_CUDA(moe::launch_pdl(moe::prefix_join_kernel, dim3((unsigned)blocks), dim3(256), 0, s, j));
  }
  return moe::check_launch("prefix_attention");
}

}  // extern "C"
