// Attention of one new token per sequence over a paged cache, in one launch.
//
//   s_j = scale q.k_j,  o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m)
//
// Up to 8 query heads that share a key head meet each of its keys and values at
// one reading (more heads are groups of 8, each of which reads them again), so the
// bound is memory; the arithmetic goes to mma.sync (m16n8k16), of which the heads
// fill the M side in two parts each: a CUDA-core form needs 2 FMAs per head and
// element and would be issue-bound from 4 heads on.  (A tcgen05 form would take
// keys as M and q as N; its products would come back through tensor memory.)
//
// Work.  A unit is one (sequence, key head, group of up to 8 query heads); it
// is cut into rounds of one tile of KEYS keys per warp.  All units in order, each at the
// cost of its rounds and kUnitCost more for its start and end, are dealt out in equal
// contiguous runs to the CTAs of one resident grid, whatever the lengths.  Each
// CTA finds its run by a scan of the lengths, so one captured launch serves
// every later length.  A unit that ends up in several CTAs is joined by the last of
// them to finish, from f32 partials in the workspace, in the order of its
// keys; the arrival counters return to zero.  The join comes behind the loop over
// the pieces, and the first piece's arrival does not stop the other warps: in the
// loop both cost registers and time (ragged e4m3 batch 119 instead of 111 us).
//
// A warp takes every NW-th tile of KEYS keys through a ring of its own, keys
// and values in slots of their own; the warps meet only at the end of a unit.
// Slots are filled by TMA in boxes of as many rows as are sure to lie in one
// page (the largest power of two up to KEYS that divides the page size) and 128
// bytes, swizzled so that ldmatrix meets no bank twice: two instructions per
// box instead of two per 16 bytes, without which a tile's copies cost more
// instructions than its arithmetic.  The load cursor runs ahead across the ends
// of units; page ids are fetched one tile ahead of the rows they lead to.
//
// Precision.  q has f32 rows, so it enters the products in parts: hi + lo fp16
// (22 bits) for fp16 and e4m3 caches, three bf16 parts for bf16 caches.  With
// at most 8 heads per 16-row operand the rows below them are free: row g holds
// the hi part of head g, row g + 8 the lo part, and the two results, which meet
// in one thread, are added.  Probabilities are split the same way (times 2^7, so
// that with a reference up to 2^8 below the maximum they fill fp16's range and
// the lo parts of small ones stay above its end).  The tensor core truncates
// where it adds, so no accumulator takes more than four (scores) or eight
// (values) k16 steps; from there on sums are f32 adds.
//
// Measured on a B200 (copy bandwidth 6.55 TB/s): 592 sequences of 1024 keys, 8 key
// heads of 128, fp16 382 us (2.5 GB, 100 %); one of 131071 keys 93 us (0.54 GB,
// 88 %: 4 us until the first tile, then CTAs that end between 74 and 86 us after the
// start with equal work, then the join of 37 parts); e4m3 256 x 2048 keys 184 us
// (1.1 GB, 90 %: bound by the latency of conversion, product and exponentials in
// eight warps); one sequence of 37 keys 5.1 us, of 512 keys 8.7 us.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <numeric>

#include "attention_frag.cuh"
#include "tc_common.cuh"

namespace moe {

constexpr int kAttCtasMost = 3;       // CTAs of an SM

struct AttArgs {
  moe_paged_cache c;
  CacheMap map;
  const float* q;
  int64_t q_ss, q_hs;
  const int32_t* seq_lens;
  float *out, *lse;
  float2* stats;                      // (maximum, sum) in the place of lse, as a part's
  int* status;
  int* arrivals;                      // one per CTA
  float2* part_ml;                    // [2 * grid][kAttHeads] (maximum, sum)
  float* part_o;                      // [2 * grid][kAttHeads][DP]
  int hq, window, from;               // sequences of `from` keys or more: without the first `from`
  float scale, cap;
};

// ---------------------------------------------------------------------------
// shapes: DP = head_dim rounded up to 64, 128 or 256.  A ring slot holds the
// keys or the values of a tile; an odd number of slots makes the slot freed
// by keys the next one that keys go to.  At 256 columns two warps share a tile,
// half of the columns each, and add their halves of the scores: the registers
// of one warp do not hold the accumulators of 256 columns, and without them
// every tile would be folded.
// ---------------------------------------------------------------------------
template <int DT, int DP, bool PACK> struct AttCfg {
  static constexpr bool kBf = DT == MOE_CACHE_BF16;
  using Frag = AFrag<kBf, PACK>;
  static constexpr int kElem = DT == MOE_CACHE_E4M3 ? 1 : 2;
  static constexpr int kSplit = DP > 128 ? 2 : 1;           // warps of a tile
  static constexpr int kDh = DP / kSplit;                   // columns of a warp
  static constexpr int kRow = kDh * kElem < kLine ? kLine : kDh * kElem;   // bytes in the ring
  static constexpr int kWarps = 4;
  static constexpr int kTiles = kWarps / kSplit;            // tiles of a round
  static constexpr int kKeys = kRow <= 128 ? 32 : 16;       // keys of a tile
  static constexpr int kSlot = kKeys * kRow;
  // heads of 64 leave registers for a third CTA, in exchange for the fourth and
  // fifth slot (256 sequences of up to 1024 keys, 8 heads, fp16 60 -> 56 us, e4m3
  // 59 -> 49 us); 128 columns of e4m3 would spill (111 -> 136 us)
  static constexpr int kCtas = DP == 64 ? 3 : 2;
  static constexpr int kSlots = kCtas == 3 ? 3 : 5;
  static constexpr int kRound = kTiles * kKeys;
  static constexpr int kRing = kWarps * kSlots * kSlot;
  static constexpr int kMergeRow = DP + 8;                  // floats
  static constexpr int kMerge = 4 * kAttHeads * kTiles * kMergeRow;   // a row per tile and head
  static constexpr int kQ = DP / 16 * Frag::kBytes;
  static constexpr int kX = kSplit > 1 ? kWarps * 32 * (kKeys / 4) * 4 : 0;   // halves of scores
  static constexpr int kSmem = kRing + kMerge + kQ + kX;
  static constexpr int kFold = 128 / kKeys;                 // tiles between folds
};

// What the start and the end of a unit cost, in rounds.  Without it a CTA with many
// short sequences takes longest: 48 sequences of 1 .. 2500 keys, 16 heads of 64, two
// CTAs of an SM, 60 us with one round, 56 us with two, 58 us with three; 256
// sequences of up to 2048 e4m3 keys 121, 111 and 114 us.
constexpr int kUnitCost = 2;
constexpr int kWholeRounds = 2;        // units of so many rounds are not split if they need not be

// byte offset of 16-byte chunk c of row r in a slot: blocks of KEYS lines,
// swizzled as TMA swizzles them
template <int KEYS>
__device__ __forceinline__ uint32_t slot_at(int r, int c) {
  return (uint32_t)((c >> 3) * KEYS * kLine + r * kLine + (((c & 7) ^ (r & 7)) << 4));
}

// A cursor over a CTA's pieces: rounds r0 .. r1 of R of unit u of a sequence.
struct Cursor {
  int seq, u, head, group;           // unit: key head and group of query heads
  int at, r0, r1, R;                 // `at`: cost at which the unit's rounds begin
  int len, first, from;              // the sequence's keys first .. len, rounds from `from` on
};

struct AttShared {
  Cursor first;                      // a piece that waits for its join
  long long base, scan[4];
  int seq, dead, join[2];            // join: of the last piece, of the first
  uint64_t bars[4][5];               // a barrier per ring slot
  uint64_t joined;                   // of the copies of other CTAs' parts
  float m[4][kAttHeads], l[4][kAttHeads], qmax[4][kAttHeads], qscale[kAttHeads];
};

template <int DT, int DP, bool PACK>
__global__ void __launch_bounds__(AttCfg<DT, DP, PACK>::kWarps * 32, (AttCfg<DT, DP, PACK>::kCtas))
attention_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const AttArgs A) {
  using Cfg = AttCfg<DT, DP, PACK>;
  using Frag = typename Cfg::Frag;
  constexpr int NW = Cfg::kWarps, NT = NW * 32, KEYS = Cfg::kKeys, NS = Cfg::kSlots;
  constexpr int LINE = kLine, RK = Cfg::kRound, SP = Cfg::kSplit, DH = Cfg::kDh, NG = Cfg::kTiles;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ AttShared sh;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int S = A.c.seqs, D = A.c.head_dim, G = A.hq / A.c.kv_heads;
  const int NHT = (G + kAttHeads - 1) / kAttHeads, HU = A.c.kv_heads * NHT;
  const int most = A.c.table_width * A.c.page_size;
  if (lane < NS) {
    mbar_init(&sh.bars[warp][lane], 1);
    fence_mbar_init();
  }
  if (tid == 0) {
    mbar_init(&sh.joined, 1);
    fence_mbar_init();
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  pdl_trigger();
  pdl_wait();

  // ---- this CTA's run of rounds
  auto keys_of = [&](int s, int& first) {
    const int n = min(max(A.seq_lens[s], 0), most);
    first = A.window > 0 && n > A.window ? n - A.window
            : n >= A.from                ? A.from
                                         : 0;
    return n;
  };
  // rounds start at a multiple of KEYS, so that no box crosses a page's end;
  // an empty sequence has one too, which writes its zeros
  auto rounds_of = [&](int s) {
    int first;
    const int n = keys_of(s, first);
    return max(1, (n - first / KEYS * KEYS + RK - 1) / RK);
  };
  const int per = (S + NT - 1) / NT, s0 = min(S, tid * per), s1 = min(S, s0 + per);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) {
    mine += (long long)(rounds_of(s) + kUnitCost) * HU;
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
  for (int w = 0; w < NW; ++w) {
    if (w < warp) before += sh.scan[w];
    total += sh.scan[w];
  }
  if (tid == 0) sh.dead = sh.join[0] = sh.join[1] = 0;
  const int quota = (int)((total + gridDim.x - 1) / gridDim.x);
  const long long start = (long long)blockIdx.x * quota;
  if (start >= total) return;
  const int end = (int)min(total - start, (long long)quota);   // costs count from `start` on
  if (mine > 0 && before <= start && start < before + mine) {
    int s = s0;
    for (;;) {
      const long long n = (long long)(rounds_of(s) + kUnitCost) * HU;
      if (start < before + n) break;
      before += n;
      ++s;
    }
    sh.seq = s;
    sh.base = before;
  }
  __syncthreads();
  const int seq0 = sh.seq, base0 = (int)(sh.base - start);

  auto open_seq = [&](Cursor& c) {
    c.len = keys_of(c.seq, c.first);
    c.from = c.first / KEYS * KEYS;
    c.R = max(1, (c.len - c.from + RK - 1) / RK);
  };
  auto next_piece = [&](Cursor& c) {             // false: that was the CTA's last
    c.at += c.R + kUnitCost;
    if (c.at >= end) return false;
    if (++c.u == HU) {
      c.u = c.head = c.group = 0;
      ++c.seq;
      open_seq(c);
    } else if (++c.group == NHT) {
      c.group = 0;
      ++c.head;
    }
    c.r0 = 0;
    c.r1 = min(c.R, end - c.at);
    return true;
  };
  Cursor C;                                      // of the arithmetic
  C.seq = seq0;
  open_seq(C);
  C.u = -base0 / (C.R + kUnitCost);
  C.head = C.u / NHT;
  C.group = C.u - C.head * NHT;
  C.at = base0 + C.u * (C.R + kUnitCost) + kUnitCost;
  if (C.at >= end) return;                       // the run ends before the unit's rounds
  C.r0 = max(0, -C.at);
  C.r1 = min(C.R, end - C.at);
  // tiles of this warp in a piece: first key, end of the keys, number
  auto tile0 = [&](const Cursor& c) { return c.from + c.r0 * RK + warp / SP * KEYS; };
  auto keys_end = [&](const Cursor& c) { return min(c.len, c.from + c.r1 * RK); };
  auto tiles = [&](const Cursor& c) {
    const int n = keys_end(c) - tile0(c);
    return n > 0 ? (n + RK - 1) / RK : 0;
  };

  // ---- q: this thread's values of the next piece's operand (k16 steps warp,
  // warp + NW, ...), fetched a piece ahead; columns 2t, 2t+1, 2t+8, 2t+9 of a
  // step, but for e4m3 keys, which are read four bytes per lane: 4t .. 4t+3
  constexpr int QK = DP / 16 / NW;
  uint8_t* const qs = smem + Cfg::kRing + Cfg::kMerge;
  float* const mo = reinterpret_cast<float*>(smem + Cfg::kRing);
  const uint8_t* const qw = qs + warp % SP * (DH / 16) * Frag::kBytes;   // this warp's columns
  float4* const xs = reinterpret_cast<float4*>(smem + Cfg::kRing + Cfg::kMerge + Cfg::kQ);
  float qn[QK][4];
  auto first_head = [&](const Cursor& c) { return c.head * G + c.group * kAttHeads; };
  auto heads = [&](const Cursor& c) { return min(kAttHeads, G - c.group * kAttHeads); };
  auto q_fetch = [&](const Cursor& c) {
    const int head = PACK ? g & 3 : g, nh = heads(c);
    const float* q = A.q + (int64_t)c.seq * A.q_ss + (int64_t)(first_head(c) + head) * A.q_hs;
#pragma unroll
    for (int i = 0; i < QK; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 16 * (warp + i * NW) +
                      (Cfg::kElem == 1 ? 4 * t + j : 2 * t + (j & 1) + 8 * (j >> 1));
        qn[i][j] = head < nh && e < D ? q[e] : 0.f;
      }
  };
  auto q_max = [&]() {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < QK; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = fmaxf(mx, fabsf(qn[i][j]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    if (t == 0) sh.qmax[warp][g] = mx;
  };
  auto q_split = [&]() {                         // scaled by a power of two to [2^10, 2^11)
    float mx = sh.qmax[0][g];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, sh.qmax[w][g]);
    // 2^e in two factors, since e may lie outside the exponents of a float
    const int ex = (int)(__float_as_uint(mx) >> 23);           // 0 .. 255
    const int e = mx > 0.f && ex < 255 ? 137 - max(ex, 1) : 0;
    const int e1 = e / 2, e2 = e - e1;
    const float f1 = __uint_as_float((uint32_t)(127 + e1) << 23);
    const float f2 = __uint_as_float((uint32_t)(127 + e2) << 23);
    // a negative scale turns q; one that vanishes stays above zero, so that it
    // leaves the minus infinity of a key that is not seen what it is
    const float sign = A.scale < 0.f ? -1.f : 1.f;
    if (warp == 0 && t == 0)
      sh.qscale[g] = fmaxf(ldexpf(fabsf(A.scale) * A.c.k_scale, -e), 1e-30f);
#pragma unroll
    for (int i = 0; i < QK; ++i) {
      Frag f;
      const float f0 = f1 * sign;
      f.set(qn[i][0] * f0 * f2, qn[i][1] * f0 * f2, qn[i][2] * f0 * f2, qn[i][3] * f0 * f2,
            g);
      f.store(qs + (warp + i * NW) * Frag::kBytes, lane);
    }
  };

  // the first q before the ring's copies: behind them it would arrive last
  q_fetch(C);

  // ---- loads: a cursor of its own that runs ahead of the arithmetic, across
  // the ends of units
  const uint32_t ring_a = smem_u32(smem) + warp * NS * Cfg::kSlot;
  constexpr int BLOCKS = Cfg::kRow / LINE;
  const int box = 1 << A.map.box_shift, boxes = KEYS >> A.map.box_shift, ps = A.c.page_size;
  const int step_pages = RK / ps, step_slots = RK - step_pages * ps;   // from tile to tile
  Cursor W = C;                                  // of the loads
  int wtiles = tiles(W), wend = keys_end(W), wkey = tile0(W), li = 0, lslot = 0;
  bool wmore = true;
  // of this lane's box of tile li: number in the sequence's pages and slot,
  // row of the tensor map
  int pidx = 0, pslot = 0, row = 0, key = 0, page = 0;
  bool in = false;
  auto enter = [&]() {                           // first tile of a piece
    li = 0;
    wtiles = tiles(W);
    wend = keys_end(W);
    wkey = tile0(W);
    key = wkey + (lane << A.map.box_shift);
    pidx = (int)((unsigned)key / (unsigned)ps);
    pslot = key - pidx * ps;
  };
  auto settle = [&]() {                          // to the next piece that has a tile li
    while (li >= wtiles) {
      wmore = next_piece(W);
      if (!wmore) break;
      enter();
    }
  };
  auto fetch = [&]() {                           // page of this lane's box of tile li
    in = wmore && lane < boxes && key < wend && key + box > W.first;
    if (in) page = A.c.block_table[(int64_t)W.seq * A.c.table_stride + pidx];
  };
  uint32_t bytes = 0;                            // of the tile's boxes that exist
  auto copy = [&](const CUtensorMap* map) {
    uint64_t* bar = &sh.bars[warp][lslot];
    if (lane == 0) mbar_expect_tx(bar, bytes);
    __syncwarp();
    if (in) {
      const uint32_t dst = ring_a + lslot * Cfg::kSlot + (lane << A.map.box_shift) * LINE;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
        tma_load_3d(dst + b * KEYS * LINE, map, warp % SP * DH + b * (LINE / Cfg::kElem), row, pslot,
                    bar);
    }
    lslot = lslot + 1 == NS ? 0 : lslot + 1;
  };
  auto issue_keys = [&]() -> uint32_t {          // which keys of the tile are valid
    if (!wmore) return 0u;
    if (in && (page < 0 || page >= A.c.pages)) {
      set_status(A.status, MOE_STATUS_BAD_PAGE);
      in = false;
    }
    row = page * A.map.page_units + W.head * A.map.head_units;
    const uint32_t ok = __ballot_sync(0xffffffffu, in);
    const int n = __popc(ok);
    uint32_t seen = 0xffffffffu;
    if (n != boxes || wkey < W.first || wkey + KEYS > wend) {
      const int r = lane & (KEYS - 1);
      seen = __ballot_sync(0xffffffffu, wkey + r >= W.first && wkey + r < wend &&
                                            ((ok >> (r >> A.map.box_shift)) & 1u));
    }
    bytes = (uint32_t)(n * BLOCKS * LINE) << A.map.box_shift;
    copy(&kmap);
    return seen;
  };
  auto issue_values = [&]() {
    if (!wmore) return;
    copy(&vmap);
    ++li;
    key += RK;
    wkey += RK;
    pidx += step_pages;
    pslot += step_slots;
    if (pslot >= ps) {
      pslot -= ps;
      ++pidx;
    }
    settle();
    fetch();
  };
  // Waits for the slot that is due.  Bounded; after a timeout anywhere in the
  // CTA no wait takes long any more, so that the kernel ends.
  int cslot = 0;
  uint32_t cphase = 0;
  auto wait_slot = [&]() {
    uint64_t* bar = &sh.bars[warp][cslot];
    if (!mbar_test(bar, cphase) && !*(volatile int*)&sh.dead && !mbar_wait(bar, cphase)) {
      sh.dead = 1;
      set_status(A.status, MOE_STATUS_TIMEOUT);
    }
    __syncwarp();
    const uint32_t a = ring_a + cslot * Cfg::kSlot;
    if (++cslot == NS) {
      cslot = 0;
      cphase ^= 1u;
    }
    return a;
  };
  enter();
  settle();
  fetch();
  constexpr int AHEAD = (NS - 1) / 2;            // tiles under way
  uint32_t seen_of[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    seen_of[i] = issue_keys();
    issue_values();
  }

  q_max();
  __syncthreads();
  q_split();
  __syncthreads();

  // lane constants of the fragment addresses: row, and for each of the four
  // chunk pairs of a line the swizzled offset
  const int krow = Cfg::kElem == 2 ? (lane >> 4) * 8 + (lane & 7)
                                   : ((lane >> 3) & 1) * 8 + (lane & 7);
  const int kch = Cfg::kElem == 2 ? (lane >> 3) & 1 : lane >> 4;
  const int vrow = ((lane >> 3) & 1) * 8 + (lane & 7), vch = lane >> 4;
  uint32_t kof[LINE / 32], vof[LINE / 32];
#pragma unroll
  for (int j = 0; j < LINE / 32; ++j) {
    kof[j] = slot_at<KEYS>(krow, 2 * j + kch);
    vof[j] = slot_at<KEYS>(vrow, 2 * j + vch);
  }
  // chunk pair j of a row block of 16: offset beyond kof / vof
  constexpr int PPL = LINE / 32;                 // chunk pairs of a line
  auto beyond = [](int j, int kb) { return (uint32_t)((j / PPL) * KEYS * LINE + kb * 16 * LINE); };

  // The piece's unit: its rounds begin in CTA c0 and go on in n - 1 more
  auto spread = [&](const Cursor& c, int& c0) {
    const int back = c.at < 0 ? (quota - 1 - c.at) / quota : 0;
    c0 = blockIdx.x - back;
    return (c.at + back * quota + c.R - 1) / quota + 1;
  };
  auto arrive = [&](const Cursor& c) {           // true: the last of its unit
    int c0, arrived;
    const int n = spread(c, c0);
    // releases this CTA's partials, acquires those of the others
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;"
                 : "=r"(arrived)
                 : "l"(A.arrivals + c0)
                 : "memory");
    if (arrived != n - 1) return false;
    A.arrivals[c0] = 0;
    return true;
  };

  for (;;) {
    // the piece after this one, and its q
    Cursor N = C;
    const bool more = next_piece(N);
    if (more) q_fetch(N);
    const int ntile = tiles(C);

    const float qscale = sh.qscale[g];           // score = product * qscale
    const float to_cap = A.cap > 0.f ? fminf(qscale / A.cap, 3e38f) : 0.f;
    const float from_cap = A.cap * kLog2e;
    const float x2 = A.cap > 0.f ? 1.f : qscale * kLog2e;
    float o[DH / 8][2];                          // head g, two columns of each 8-wide block
    float acc[DH / 8][4];
#pragma unroll
    for (int c = 0; c < DH / 8; ++c) {
      o[c][0] = o[c][1] = 0.f;
      acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
    }
    // m: reference of the exponentials, 2^8 below the maximum at most (it moves
    // up seldom, so a tile's maximum is not shared between lanes until it has to);
    // l: sum over this lane's keys
    float m = -INFINITY, l = 0.f;
    auto fold = [&](float f) {                   // o = (o + acc) * f
#pragma unroll
      for (int c = 0; c < DH / 8; ++c) {
        o[c][0] = (o[c][0] + (acc[c][0] + acc[c][2])) * f;
        o[c][1] = (o[c][1] + (acc[c][1] + acc[c][3])) * f;
        acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
      }
    };

    for (int i = 0; i < ntile; ++i) {
      const uint32_t ka = wait_slot();
      const uint32_t seen = seen_of[0];
#pragma unroll
      for (int k = 0; k + 1 < AHEAD; ++k) seen_of[k] = seen_of[k + 1];
      seen_of[AHEAD - 1] = issue_keys();

      // scores: keys 8b + 2t, 8b + 2t + 1 of head g in this lane.  Columns past
      // head_dim are zeros in the ring and in q
      float x[KEYS / 8][2];
#pragma unroll
      for (int k4 = 0; k4 < DH / 64; ++k4) {
        float a[KEYS / 8][4];
#pragma unroll
        for (int kk = 4 * k4; kk < 4 * k4 + 4; kk += 3 - Cfg::kElem) {
          Frag q0, q1;
          q0.load(qw + kk * Frag::kBytes, lane);
          if (Cfg::kElem == 1) q1.load(qw + (kk + 1) * Frag::kBytes, lane);
#pragma unroll
          for (int kb = 0; kb < KEYS / 16; ++kb) {
            uint32_t b[4];
            const int j = Cfg::kElem == 2 ? kk : kk / 2;
            ldsm4(b, ka + kof[j % PPL] + beyond(j, kb));
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
        for (int b = 0; b < KEYS / 8; ++b) {
          x[b][0] = (k4 ? x[b][0] : 0.f) + (a[b][0] + a[b][2]);
          x[b][1] = (k4 ? x[b][1] : 0.f) + (a[b][1] + a[b][3]);
        }
      }
      if (PACK) {                                // the third part of q, in the other lanes
#pragma unroll
        for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) x[b][h] += __shfl_xor_sync(0xffffffffu, x[b][h], 16);
      }
      if (SP > 1) {
        // the other half of the columns: both warps get the same sums
        constexpr int V = KEYS / 16;
        float4* mine = xs + warp * 32 * V + lane;
        const float4* other = xs + (warp ^ 1) * 32 * V + lane;
#pragma unroll
        for (int v = 0; v < V; ++v)
          mine[v * 32] = make_float4(x[2 * v][0], x[2 * v][1], x[2 * v + 1][0], x[2 * v + 1][1]);
        asm volatile("bar.sync %0, 64;" ::"r"(1 + warp / SP) : "memory");
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float4 y = other[v * 32];
          x[2 * v][0] += y.x;
          x[2 * v][1] += y.y;
          x[2 * v + 1][0] += y.z;
          x[2 * v + 1][1] += y.w;
        }
        asm volatile("bar.sync %0, 64;" ::"r"(1 + warp / SP) : "memory");
      }
      auto hide = [&](float value) {             // lanes past KEYS repeat the first ones
        if (seen != 0xffffffffu)
#pragma unroll
          for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (!((seen >> (8 * b + 2 * t + h)) & 1u)) x[b][h] = value;
      };
      if (A.cap > 0.f) {                         // x = cap tanh(score / cap) log2 e
        hide(0.f);                               // what the ring holds there picks no form of tanh
        float big = 0.f;
#pragma unroll
        for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            x[b][h] *= to_cap;
            big = fmaxf(big, fabsf(x[b][h]));
          }
        if (__any_sync(0xffffffffu, !(big < 0.5f))) {
#pragma unroll
          for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[b][h] = from_cap * tanhf(x[b][h]);
        } else {
          // Lambert's continued fraction y / (1 + y^2 / (3 + y^2 / (5 + y^2 / (7 + y^2 / 9)))),
          // off by less than 2^-29 of tanh y for |y| < 1/2
#pragma unroll
          for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float y = x[b][h], z = y * y;
              const float num = fmaf(z, z + 105.f, 945.f), den = fmaf(z, fmaf(15.f, z, 420.f), 945.f);
              x[b][h] = from_cap * __fdividef(y * num, den);
            }
        }
      }
      hide(-INFINITY);

      // reference and sum
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < KEYS / 8; ++b) mx = fmaxf(mx, fmaxf(x[b][0], x[b][1]));
      if (__any_sync(0xffffffffu, mx * x2 > m + 8.f)) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * x2;
        const float to = mx > m + 8.f ? mx : m;
        const float f = to == -INFINITY ? 1.f : ex2(m - to);
        fold(f);
        l *= f;
        m = to;
      }
      const float shift = kPShift - (m == -INFINITY ? 0.f : m);
#pragma unroll
      for (int b = 0; b < KEYS / 8; ++b)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[b][h] = ex2(fmaf(x[b][h], x2, shift));
          l += x[b][h];
        }
      Frag pf[KEYS / 16];
#pragma unroll
      for (int kb = 0; kb < KEYS / 16; ++kb)
        pf[kb].set(x[2 * kb][0], x[2 * kb][1], x[2 * kb + 1][0], x[2 * kb + 1][1], g);

      const uint32_t va = wait_slot();
      issue_values();
      if (seen != 0xffffffffu) {                 // nothing of a row that is not seen counts
        for (int r = 0; r < KEYS; ++r)
          if (!((seen >> r) & 1u) && lane < Cfg::kRow / 16) {
            const uint32_t to = va + slot_at<KEYS>(r, lane);
            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to), "r"(0) : "memory");
          }
        fence_proxy_async_smem();
        __syncwarp();
      }

      // p v.  e4m3: a 16-byte chunk holds 16 columns; transposed in pairs of
      // bytes, a register has columns (2g, 2g + 1) of two keys, which become
      // the B registers of the even and of the odd columns.  The accumulators
      // take kFold tiles (eight k16 steps) before they are added up
      constexpr int CPB = Cfg::kElem == 2 ? 2 : 4;      // 8-wide blocks of two chunks
#pragma unroll
      for (int c = 0; c < DH / 8; c += CPB) {
#pragma unroll
        for (int kb = 0; kb < KEYS / 16; ++kb) {
          uint32_t b[4];
          const int pair = Cfg::kElem == 2 ? c / 2 : c / 4;
          ldsm4_t(b, va + vof[pair % PPL] + beyond(pair, kb));
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            if (Cfg::kElem == 2) {
              pf[kb].mul(acc[c + j], b[2 * j], b[2 * j + 1]);
            } else {
              uint32_t e0, o0, e1, o1;           // even and odd columns, keys 0-7 and 8-15
              e4m3x4_f16x2(prmt(b[2 * j], 0u, 0x3120u), e0, o0);
              e4m3x4_f16x2(prmt(b[2 * j + 1], 0u, 0x3120u), e1, o1);
              pf[kb].mul(acc[c + 2 * j], e0, e1);
              pf[kb].mul(acc[c + 2 * j + 1], o0, o1);
            }
          }
        }
      }
      if (i % Cfg::kFold == Cfg::kFold - 1) fold(1.f);
    }
    fold(1.f);
    if (PACK) {
#pragma unroll
      for (int c = 0; c < DH / 8; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) o[c][h] += __shfl_xor_sync(0xffffffffu, o[c][h], 16);
    }

    // ---- the warps' parts meet in shared memory
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0 && warp % SP == 0) {
      sh.m[warp / SP][g] = m;
      sh.l[warp / SP][g] = l;
    }
    {
      float* row = mo + (warp / SP * kAttHeads + g) * Cfg::kMergeRow + warp % SP * DH;
#pragma unroll
      for (int c = 0; c < DH / 8; c += 3 - Cfg::kElem) {
        if (Cfg::kElem == 2)
          *reinterpret_cast<float2*>(row + 8 * c + 2 * t) = make_float2(o[c][0], o[c][1]);
        else                                     // block c: even columns 4t, 4t + 2; c + 1: odd
          *reinterpret_cast<float4*>(row + 8 * c + 4 * t) =
              make_float4(o[c][0], o[c + 1][0], o[c][1], o[c + 1][1]);
      }
    }
    if (more) q_max();
    __syncthreads();
    const bool whole = C.r0 == 0 && C.r1 == C.R;
    const int my_slot = 2 * blockIdx.x + (C.r0 == 0 ? 1 : 0);
    const int nh = heads(C);
    const int64_t row0 = (int64_t)C.seq * A.hq + first_head(C);
    const float unit = A.c.v_scale;
    for (int h = warp; h < nh; h += NW) {
      float M = sh.m[0][h];
#pragma unroll
      for (int w = 1; w < NG; ++w) M = fmaxf(M, sh.m[w][h]);
      const float ms = M == -INFINITY ? 0.f : M;
      float L = 0.f, f[NG];
#pragma unroll
      for (int w = 0; w < NG; ++w) {
        f[w] = ex2(sh.m[w][h] - ms);
        L = fmaf(sh.l[w][h], f[w], L);
      }
      if (whole) {
        const float norm = L == 0.f ? 0.f : unit / L;
#pragma unroll
        for (int w = 0; w < NG; ++w) f[w] *= norm;
        if (lane == 0 && A.stats) A.stats[row0 + h] = make_float2(M, L);
        else if (lane == 0 && A.lse) A.lse[row0 + h] = (M + (log2f(L) - kPShift)) * kLn2;
      } else if (lane == 0) {
        A.part_ml[my_slot * kAttHeads + h] = make_float2(M, L);
      }
      float* to = whole ? A.out + (row0 + h) * D : A.part_o + ((int64_t)my_slot * kAttHeads + h) * DP;
#pragma unroll
      for (int c = lane; c < DP; c += 32) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < NG; ++w)
          y = fmaf(mo[(w * kAttHeads + h) * Cfg::kMergeRow + c], f[w], y);
        if (c < D) to[c] = y;
      }
    }
    if (!whole) fence_proxy_async();             // a part may be fetched by a bulk copy
    if (more) q_split();
    __syncthreads();                             // q of the next piece; mo and sh are free
    // Parts of units are announced as they are written; units that turn out to
    // be complete are joined behind the loop.  Only a CTA's first piece and its
    // last can be parts.
    if (!whole && tid == 0) {
      const bool last = arrive(C);
      if (last && more) sh.first = C;
      sh.join[more] = last;
    }
    if (!more) break;
    C = N;
  }
  // Joins: the parts come into the ring, which has been read out, by one bulk copy
  // for each part's sums and one for its values, and are added in order.  The
  // loops are short because this code runs once: unrolled over 16 loads to
  // registers it took 11600 cycles for 37 parts, most of them instruction fetches.
  __syncthreads();
  uint32_t jphase = 0;
  for (int k = 0; k < 2; ++k) {
    if (!sh.join[k]) continue;
    if (k) C = sh.first;
    int c0;
    const int n = spread(C, c0), nh = heads(C);
    const int64_t row0 = (int64_t)C.seq * A.hq + first_head(C);
    constexpr int ML = kAttHeads * 8, CT = DP / 4;
    const int OB = nh * DP * 4;
    const int most_parts = Cfg::kRing / (ML + OB);         // in the ring at a time
    const float2* ml = reinterpret_cast<const float2*>(smem);
    const float4* po = reinterpret_cast<const float4*>(smem + most_parts * ML);
    // items: four columns of a head; M, L, y: maximum, sum and values so far
    constexpr int ITEMS = kAttHeads * CT / NT > 0 ? kAttHeads * CT / NT : 1;
    float M[ITEMS], L[ITEMS];
    float4 y[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      M[j] = -INFINITY;
      L[j] = 0.f;
      y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int i0 = 0; i0 < n; i0 += most_parts) {
      const int cnt = min(most_parts, n - i0);
      if (k || i0) __syncthreads();              // the parts before have been added
      if (warp == 0) {
        fence_proxy_async();
        if (lane == 0) mbar_expect_tx(&sh.joined, cnt * (ML + OB));
        __syncwarp();
        for (int i = lane; i < cnt; i += 32) {
          const int64_t slot = 2 * (int64_t)(c0 + i0 + i) + (i0 + i == 0);
          bulk_g2s_plain(smem + i * ML, A.part_ml + slot * kAttHeads, ML, &sh.joined);
          bulk_g2s_plain(smem + most_parts * ML + i * OB, A.part_o + slot * kAttHeads * DP, OB,
                         &sh.joined);
        }
      }
      if (!mbar_wait(&sh.joined, jphase)) {
        sh.dead = 1;
        set_status(A.status, MOE_STATUS_TIMEOUT);
      }
      jphase ^= 1u;
#pragma unroll
      for (int j = 0; j < ITEMS; ++j) {
        const int e = tid + j * NT, h = e / CT, col = e % CT;
        if (h >= nh) break;
        float m = M[j];
#pragma unroll 4
        for (int i = 0; i < cnt; ++i) m = fmaxf(m, ml[i * kAttHeads + h].x);
        const float ms = m == -INFINITY ? 0.f : m, f = ex2(M[j] - ms);
        M[j] = m;
        L[j] *= f;
        y[j] = make_float4(y[j].x * f, y[j].y * f, y[j].z * f, y[j].w * f);
#pragma unroll 4
        for (int i = 0; i < cnt; ++i) {
          const float2 p = ml[i * kAttHeads + h];
          const float4 v = po[(i * nh + h) * CT + col];
          const float w = ex2(p.x - ms);
          L[j] = fmaf(p.y, w, L[j]);
          y[j].x = fmaf(v.x, w, y[j].x);
          y[j].y = fmaf(v.y, w, y[j].y);
          y[j].z = fmaf(v.z, w, y[j].z);
          y[j].w = fmaf(v.w, w, y[j].w);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      const int e = tid + j * NT, h = e / CT, col = e % CT;
      if (h >= nh) break;
      const float norm = L[j] == 0.f ? 0.f : A.c.v_scale / L[j];
      float* to = A.out + (row0 + h) * D + 4 * col;
      if (4 * col < D)
        to[0] = y[j].x * norm, to[1] = y[j].y * norm, to[2] = y[j].z * norm, to[3] = y[j].w * norm;
      if (col == 0 && A.stats) A.stats[row0 + h] = make_float2(M[j], L[j]);
      else if (col == 0 && A.lse) A.lse[row0 + h] = (M[j] + (log2f(L[j]) - kPShift)) * kLn2;
    }
  }
  // after a timeout copies may still be under way: give them time to land
  if (*(volatile int*)&sh.dead)
    for (int i = 0; i < NS; ++i) {
      mbar_wait(&sh.bars[warp][i], 0);
      mbar_wait(&sh.bars[warp][i], 1);
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// The cache as a 3-D tensor for TMA: elements of a row; rows one common unit of
// the strides apart (a page and a head lead to a row number); tokens of a page.
int make_cache_map(CUtensorMap* map, const moe_paged_cache& c, void* base, int keys,
                   CacheMap* at) {
  const int eb = cache_elem_bytes(c.dtype);
  const int64_t row = (int64_t)c.head_dim;
  int64_t unit = std::gcd(std::gcd(c.page_stride, c.token_stride), c.head_stride);
  if (unit == 0) unit = row;
  MOE_REQUIRE(unit >= row, MOE_ERR_UNSUPPORTED,
              "cache strides (%lld, %lld, %lld) are not multiples of one row of at least head_dim "
              "elements",
              (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride);
  const int64_t rows = ((c.pages - 1) * c.page_stride + (c.kv_heads - 1) * c.head_stride) / unit + 1;
  MOE_REQUIRE(rows <= 0x7fffffff && unit * eb < (1ll << 40) && c.token_stride * eb < (1ll << 40),
              MOE_ERR_UNSUPPORTED, "cache of %lld rows is too large", (long long)rows);
  at->page_units = (int)(c.page_stride / unit);
  at->head_units = (int)(c.head_stride / unit);
  const int rows_of_box = std::min(keys, c.page_size & -c.page_size);
  at->box_shift = 31 - __builtin_clz((unsigned)rows_of_box);
  const cuuint64_t dims[3] = {(cuuint64_t)row, (cuuint64_t)rows, (cuuint64_t)c.page_size};
  const cuuint64_t strides[2] = {(cuuint64_t)(unit * eb),
                                 (cuuint64_t)(std::max(c.token_stride, unit) * eb)};
  const cuuint32_t box[3] = {(cuuint32_t)(kLine / eb), 1, (cuuint32_t)rows_of_box};
  const cuuint32_t each[3] = {1, 1, 1};
  EncodeTiledFn fn = encode_fn();
  MOE_REQUIRE(fn, MOE_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const CUresult r =
      fn(map, eb == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base,
         dims, strides, box, each, CU_TENSOR_MAP_INTERLEAVE_NONE,
         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  MOE_REQUIRE(r == CUDA_SUCCESS, MOE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return MOE_OK;
}

inline int padded_head_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

static int attention_workspace(int head_dim, AttArgs* a, void* ws, size_t* bytes) {
  Carve cv = {static_cast<uint8_t*>(ws), 0, 0};
  const int slots = kAttCtasMost * sm_count();
  cv.take<uint8_t>(256);
  int* arrivals = cv.take<int>(slots);
  float2* ml = cv.take<float2>((size_t)2 * slots * kAttHeads);
  float* o = cv.take<float>((size_t)2 * slots * kAttHeads * padded_head_dim(head_dim));
  if (a) {
    a->arrivals = arrivals;
    a->part_ml = ml;
    a->part_o = o;
  }
  *bytes = align_up(cv.used, 256);
  return MOE_OK;
}

template <int DT, int DP, bool PACK>
static int launch_attention(AttArgs& a, int max_len, cudaStream_t s) {
  using Cfg = AttCfg<DT, DP, PACK>;
  static_assert(Cfg::kSlots % 2 == 1 && Cfg::kSlots <= 5 && Cfg::kWarps == 4 &&
                    Cfg::kCtas <= kAttCtasMost,
                "");
  static std::atomic<uint64_t> ready{0};
  auto kern = attention_kernel<DT, DP, PACK>;
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((ready.load() >> dev) & 1)) {
    MOE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  CUtensorMap kmap, vmap;
  MOE_CHECK(make_cache_map(&kmap, a.c, a.c.k, Cfg::kKeys, &a.map));
  MOE_CHECK(make_cache_map(&vmap, a.c, a.c.v, Cfg::kKeys, &a.map));
  const int G = a.hq / a.c.kv_heads;
  const int64_t units = (int64_t)a.c.seqs * a.c.kv_heads * ((G + kAttHeads - 1) / kAttHeads);
  const int64_t keys = a.window > 0 ? std::min(a.window, max_len) : std::max(0, max_len - a.from);
  // A round costs about 1 us, a unit in parts about 3 us for their joining: short
  // sequences get a CTA per unit (one of 100 keys 6.3 us instead of 8.0; with three
  // rounds ragged batches lose more than that: their units are split all the same)
  const int64_t rounds = std::max<int64_t>(1, (keys + Cfg::kRound - 1) / Cfg::kRound);
  const int64_t ctas = rounds <= kWholeRounds ? units : units * (rounds + kUnitCost);
  const int grid = (int)std::min<int64_t>(ctas, (int64_t)Cfg::kCtas * sm_count());
  // a CTA counts its costs, and a sequence's, in 32 bits
  const int64_t most = (int64_t)a.c.table_width * a.c.page_size / Cfg::kRound + 2 + kUnitCost;
  MOE_REQUIRE(units / a.c.seqs * most < (1ll << 30) && units * most / grid < (1ll << 30),
              MOE_ERR_UNSUPPORTED, "%d sequences of up to %d pages are too many", a.c.seqs,
              a.c.table_width);
  MOE_CUDA(launch_pdl(kern, dim3((unsigned)grid), dim3(Cfg::kWarps * 32), Cfg::kSmem, s, kmap, vmap,
                      a));
  return MOE_OK;
}

template <int DT, bool PACK>
static int launch_attention_dt(AttArgs& a, int max_len, cudaStream_t s) {
  switch (padded_head_dim(a.c.head_dim)) {
    case 64: return launch_attention<DT, 64, PACK>(a, max_len, s);
    case 128: return launch_attention<DT, 128, PACK>(a, max_len, s);
    default: return launch_attention<DT, 256, PACK>(a, max_len, s);
  }
}

// Refuses what the attention cannot take; c: the cache as the kernels take it.
int check_attention(const moe_paged_attention_args& r, moe_paged_cache& c) {
  const float* q = r.q;
  float* out = r.out;
  MOE_CHECK(take_cache(&r.cache, c));
  MOE_REQUIRE(r.q_heads > 0 && r.q_heads % c.kv_heads == 0, MOE_ERR_INVALID,
              "%d query heads for %d key heads", r.q_heads, c.kv_heads);
  MOE_REQUIRE(r.max_len >= 0 && r.window >= 0, MOE_ERR_INVALID, "negative length or window");
  MOE_REQUIRE(isfinite(r.scale) && isfinite(r.softcap) && r.softcap >= 0.f, MOE_ERR_INVALID,
              "scale and softcap must be finite, softcap >= 0");
  if (c.seqs == 0) return MOE_OK;
  MOE_REQUIRE(q && r.seq_lens && out && r.workspace, MOE_ERR_INVALID, "null pointer");
  // parts in it are fetched by bulk copies
  MOE_REQUIRE((uintptr_t)r.workspace % 16 == 0, MOE_ERR_INVALID, "workspace must be 16-byte aligned");
  {
    // A unit's rows of out are written behind the last read of its rows of q, so out
    // may be q itself, but over other rows it would be read when it is written already.
    const int64_t S = c.seqs, d = c.head_dim, n = S * r.q_heads * d;
    const bool same = (uintptr_t)out == (uintptr_t)q && (S == 1 || r.q_seq_stride == r.q_heads * d) &&
                      (r.q_heads == 1 || r.q_head_stride == d);
    const int64_t ss = (S - 1) * r.q_seq_stride, hs = (r.q_heads - 1) * r.q_head_stride;
    const int64_t lo = std::min<int64_t>(ss, 0) + std::min<int64_t>(hs, 0);
    const int64_t hi = std::max<int64_t>(ss, 0) + std::max<int64_t>(hs, 0) + d;
    const int64_t at = (int64_t)((uintptr_t)out - (uintptr_t)q);         // bytes
    MOE_REQUIRE(same || at >= 4 * hi || at + 4 * n <= 4 * lo, MOE_ERR_INVALID,
                "q and out overlap, and are not the same rows");
  }
  return MOE_OK;
}

// The attention without the first `from` keys of each sequence that has so many; with stats (seqs,
// q_heads) the maxima (powers of two) and sums times 2^kPShift go there, and lse is not written.
int attention_from(const moe_paged_attention_args& r, int from, float2* stats) {
  AttArgs a = {};
  MOE_CHECK(check_attention(r, a.c));
  if (a.c.seqs == 0) return MOE_OK;
  a.q = r.q;
  a.q_ss = r.q_seq_stride;
  a.q_hs = r.q_head_stride;
  a.seq_lens = r.seq_lens;
  a.out = r.out;
  a.lse = r.lse;
  a.stats = stats;
  a.status = static_cast<int*>(r.workspace);
  a.hq = r.q_heads;
  a.window = r.window;
  a.scale = r.scale;
  a.cap = r.softcap;
  a.from = from;
  size_t need = 0;
  MOE_CHECK(attention_workspace(a.c.head_dim, &a, r.workspace, &need));
  MOE_REQUIRE(r.workspace_bytes >= need, MOE_ERR_WORKSPACE, "workspace %zu < %zu bytes",
              r.workspace_bytes, need);
  const int most = a.c.table_width * a.c.page_size;
  const int longest = r.max_len > 0 && r.max_len < most ? r.max_len : most;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r.stream);
  {
    ProfScope _prof(MOE_K_ATTENTION, s);
    if (a.c.dtype == MOE_CACHE_F16)
      MOE_CHECK((launch_attention_dt<MOE_CACHE_F16, false>(a, longest, s)));
    else if (a.c.dtype == MOE_CACHE_E4M3)
      MOE_CHECK((launch_attention_dt<MOE_CACHE_E4M3, false>(a, longest, s)));
    else if (r.q_heads / a.c.kv_heads <= 4)
      MOE_CHECK((launch_attention_dt<MOE_CACHE_BF16, true>(a, longest, s)));
    else
      MOE_CHECK((launch_attention_dt<MOE_CACHE_BF16, false>(a, longest, s)));
  }
  return check_launch("paged_attention");
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
  return moe::attention_workspace(head_dim, nullptr, nullptr, bytes);
}

int moe_paged_attention_record(const moe_paged_attention_args* a) {
  MOE_REQUIRE(a, MOE_ERR_INVALID, "null arguments");
  return moe::attention_from(*a, 0);
}

int moe_paged_attention(const moe_paged_cache* cache, const float* q, int64_t q_seq_stride,
                        int64_t q_head_stride, const int32_t* seq_lens, int q_heads, int max_len,
                        int window, float scale, float softcap, float* out, float* lse,
                        void* workspace, size_t workspace_bytes, moe_stream_t stream) {
  MOE_REQUIRE(cache, MOE_ERR_INVALID, "null cache");
  const moe_paged_attention_args a = {*cache, q, q_seq_stride, q_head_stride, seq_lens, out, lse,
                                      workspace, workspace_bytes, stream, q_heads, max_len, window,
                                      scale, softcap};
  return moe::attention_from(a, 0);
}

}  // extern "C"
