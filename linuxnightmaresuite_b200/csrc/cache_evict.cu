// Eviction from a paged cache by accumulated attention weight.
//
// Of the n slots of a (sequence, key head) `keep` stay: those whose token is among the last
// `recent` positions, then those of the largest mass (of equals the lowest slot).  Attention
// does not care for the order of its keys, so nothing is compacted: the survivors that sit
// in slots >= keep, ascending, move into the slots < keep that are given up, ascending.  A
// step that gives up one slot moves one row, where compaction would move half of the cache.
//
// A cluster of up to 8 CTAs owns a (sequence, head); CTA r has the slots r sl .. (r + 1) sl in
// shared memory, as 32-bit keys whose order is that of the masses (kept in any case: all ones).
// The keep-th largest key comes from a radix select of four digits: counts in
// shared memory, added up across the cluster, and the digit found by a scan.  Then the movers'
// numbers are prefix sums; CTA k % C gets mover k in a list and copies its rows, 16 bytes a
// lane.  Where few slots leave, by the longest length that the call allows, one CTA takes them one
// by one.
//
// Bound by latency where few slots leave (128 sequences, one slot of 1025 each, 8 heads: 9.1 us on
// the device, about the host's time for the call; by radix select 30), by memory where long prompts
// are cut: 6 of up to 32768 tokens to 4096, 8 heads of 128, fp16, 73 us, 40 of them the rows that
// move, 256 bytes each at random, read and written once at 4.3 TB/s; the rest the digits' barriers
// across the cluster.  Digits of 11 bits took 204: counts of a cluster are 64 KB a digit through its
// network.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged_cache.cuh"

namespace moe {
namespace cg = cooperative_groups;

constexpr int kEvictThreads = 256;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictCluster = 8;
constexpr int kEvictSlots = 20480;     // of a CTA at most: 8 bytes each in shared memory
constexpr int kBins = 256;             // a thread each
// Slots that leave one by one, of sequences of so many slots at most.  Device time in place, 8 heads,
// one by one and by radix select, us, one slot of n + 1 (eight of 4100 in the last column):
//                  n = 1024    4096      8192      16384     32767      4100
//   1 sequence    4.6 / 10   6.1 / 14  8.3 / 16   12 / 17    20 / 19   9.2 / 15
//   16 sequences  5.4 / 11   6.4 / 28  8.9 / 49   13 / 53    21 / 63   9.9 / 30
//   64 sequences  6.1 / 20   7.9 / 43   12 / 56   25 / 78  134 / 288    14 / 45
// With results apart one CTA of a head copies its ledger too, which costs more than the select from 8192
// slots of up to 4 sequences on (1 x 16384 34 / 20, 1 x 32767 65 / 24).
constexpr int kFew = 8;
constexpr int kFewSlots = 32768;

struct EvictArgs {
  moe_paged_cache c;
  const int32_t* seq_lens;
  const float* mass;
  const int32_t* held;
  float* mass_out;
  int32_t *held_out, *lens_out;
  int64_t row, row_out;                // slots of a (sequence, head) in the ledgers
  int* status;
  int keep, recent, most, apart;       // apart: lens_out is not seq_lens
};

struct EvictShared {
  int bins[4][kBins];
  int scan[33];
  int newest, digit, above;
  int movers, freed;                   // of this CTA
  int of_warp[3][kEvictWarps];
};

// f32 -> u32 of the same order; +-0 are equal, NaN is last
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// What the CTAs of a (sequence, head) need to know of it.
struct EvictUnit {
  const float* mass;
  const int32_t *held, *table;
  float* mass_out;
  int32_t* held_out;
  int n;                               // 0: nothing to do
  __device__ EvictUnit(const EvictArgs& A, int unit, int rank) {
    const int seq = unit / A.c.kv_heads, head = unit - seq * A.c.kv_heads;
    const int told = max(A.seq_lens[seq], 0);
    n = told > A.most ? 0 : told;
    if (head == 0 && rank == 0 && threadIdx.x == 0) {
      if (told > A.most) set_status(A.status, MOE_STATUS_BAD_PAGE);     // left as it is
      if (A.apart) A.lens_out[seq] = told > A.most ? told : min(n, A.keep);
    }
    mass = A.mass + (int64_t)unit * A.row;
    held = A.held + (int64_t)unit * A.row;
    mass_out = A.mass_out + (int64_t)unit * A.row_out;
    held_out = A.held_out + (int64_t)unit * A.row_out;
    table = A.c.block_table + (int64_t)seq * A.c.table_stride;
  }
  // entries that stay where they are, where the result is another ledger
  __device__ void copy(int i) const {
    if (mass_out != mass) mass_out[i] = mass[i];
    if (held_out != held) held_out[i] = held[i];
  }
};

// The rows of up to 32 moves, (from, to) of one in each lane (-1: none), by a warp: 16 bytes a
// lane, of keys and values, B loads under way.
struct EvictRows {
  uint8_t* k;
  int64_t v_less_k;
  int lines;                           // 16-byte lines of a row, at most 32
  uint32_t per_line;                   // i / lines = i * per_line >> 16 for i < 2048
  __device__ EvictRows(const EvictArgs& A, int head) {
    const int eb = A.c.dtype == MOE_CACHE_E4M3 ? 1 : 2;
    k = static_cast<uint8_t*>(A.c.k) + (int64_t)head * A.c.head_stride * eb;
    v_less_k = (int64_t)((uintptr_t)A.c.v - (uintptr_t)A.c.k);
    lines = A.c.head_dim * eb / 16;
    per_line = 65536u / (uint32_t)lines + 1;
  }
  // byte offset of a slot's row, -1: its page does not exist
  __device__ static int64_t at(const EvictArgs& A, const int32_t* table, int slot) {
    const int p = slot / A.c.page_size, page = table[p];
    if (page < 0 || page >= A.c.pages) return -1;
    return ((int64_t)page * A.c.page_stride + (int64_t)(slot - p * A.c.page_size) * A.c.token_stride) *
           (A.c.dtype == MOE_CACHE_E4M3 ? 1 : 2);
  }
  template <int B> __device__ void move(int64_t from, int64_t to, int count, int lane) const {
    const int items = 2 * count * lines;
    for (int i0 = lane; i0 - lane < items; i0 += 32 * B) {
      uint4 v[B];
      int64_t dst[B];
#pragma unroll
      for (int b = 0; b < B; ++b) {
        const int i = i0 + 32 * b, row = (int)((uint32_t)i * per_line >> 16);
        const int64_t off = (row & 1 ? v_less_k : 0) + 16 * (i - row * lines);
        const int64_t f = __shfl_sync(0xffffffffu, from, row / 2 & 31);
        const int64_t d = __shfl_sync(0xffffffffu, to, row / 2 & 31);
        dst[b] = i < items && f >= 0 ? d + off : -1;
        if (dst[b] != -1) v[b] = *reinterpret_cast<const uint4*>(k + f + off);
      }
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (dst[b] != -1) *reinterpret_cast<uint4*>(k + dst[b]) = v[b];
    }
  }
};

// ---------------------------------------------------------------------------
// Few slots leave (a decode step at the limit): one CTA of a (sequence, head) takes away the
// smallest key so often.  Registers 40, no spills; the form for any number spills 28 bytes.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kEvictThreads, 6) evict_few_kernel(const EvictArgs A) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint64_t least[2][kEvictWarps];
  __shared__ int top[kEvictWarps];
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  const EvictUnit U(A, blockIdx.x, 0);
  const int n = U.n, drop = n - A.keep;
  int newest = INT32_MIN;
#pragma unroll 4
  for (int i = tid; i < n; i += kEvictThreads) {
    keys[i] = order_key(U.mass[i]);
    newest = max(newest, U.held[i]);
  }
  if (drop <= 0) {
    for (int i = tid; i < n; i += kEvictThreads) U.copy(i);
    return;
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) top[warp] = newest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kEvictWarps; ++w) newest = max(newest, top[w]);
  const int64_t since = (int64_t)newest - A.recent;
  // smallest key, of equals the largest slot: the smallest (key, ~slot).  Kept in any case: all
  // ones, which only slots that are all kept so can be; taken away: never again
  auto mine = [&]() {
    uint64_t m = ~0ull;
#pragma unroll 4
    for (int i = tid; i < n; i += kEvictThreads) {
      const uint64_t k = (uint64_t)keys[i] << 32 | (uint32_t)~i;
      m = k < m ? k : m;
    }
    return m;
  };
  if (A.recent > 0) {
#pragma unroll 4
    for (int i = tid; i < n; i += kEvictThreads)
      if (U.held[i] > since) keys[i] = 0xffffffffu;
  }
  uint64_t m = mine();
  int gone[kFew];
#pragma unroll
  for (int r = 0; r < kFew; ++r) {
    gone[r] = -1;
    if (r < drop) {
      const uint32_t hi = __reduce_min_sync(0xffffffffu, (uint32_t)(m >> 32));
      const uint32_t lo = __reduce_min_sync(0xffffffffu, (uint32_t)(m >> 32) == hi ? (uint32_t)m : ~0u);
      if (lane == 0) least[r & 1][warp] = (uint64_t)hi << 32 | lo;
      __syncthreads();
      uint64_t all = ~0ull;
#pragma unroll
      for (int w = 0; w < kEvictWarps; ++w) all = least[r & 1][w] < all ? least[r & 1][w] : all;
      gone[r] = (int)~(uint32_t)all;
      if (gone[r] % kEvictThreads == tid) {      // its thread looks for its next one
        uint64_t next = ~0ull;
        for (int i = tid; i < n; i += kEvictThreads) {
          const uint64_t k = (uint64_t)keys[i] << 32 | (uint32_t)~i;
          if (k > all && k < next) next = k;
        }
        m = next;
      }
    }
  }
  if (U.mass_out != U.mass || U.held_out != U.held)
    for (int i = tid; i < A.keep; i += kEvictThreads) {
      bool left = false;
#pragma unroll
      for (int r = 0; r < kFew; ++r) left |= gone[r] == i;
      if (!left) U.copy(i);
    }
  if (warp != 0) return;
  // lane j: the j-th slot from `keep` on that stays and the j-th below it that leaves
  int from = -1, to = -1, survivors = 0;
  for (int i = A.keep; i < n; ++i) {
    bool left = false;
#pragma unroll
    for (int r = 0; r < kFew; ++r) left |= gone[r] == i;
    if (!left && survivors++ == lane) from = i;
  }
#pragma unroll
  for (int r = 0; r < kFew; ++r) {
    int rank = 0;                      // of this slot among those that leave below `keep`
#pragma unroll
    for (int q = 0; q < kFew; ++q) rank += gone[q] >= 0 && gone[q] < gone[r];
    if (gone[r] >= 0 && gone[r] < A.keep && rank == lane) to = gone[r];
  }
  int64_t src = -1, dst = -1;
  if (from >= 0) {
    U.mass_out[to] = U.mass[from];
    U.held_out[to] = U.held[from];
    src = EvictRows::at(A, U.table, from);
    dst = EvictRows::at(A, U.table, to);
    if (src < 0 || dst < 0) {
      set_status(A.status, MOE_STATUS_BAD_PAGE);
      src = dst = -1;
    }
  }
  EvictRows(A, blockIdx.x % A.c.kv_heads).move<2>(src, dst, survivors, lane);
}

// ---------------------------------------------------------------------------
// Any number of slots.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kEvictThreads, 3) evict_kernel(const EvictArgs A) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ EvictShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int unit = blockIdx.x / C;
  const int tid = threadIdx.x, NT = kEvictThreads, lane = tid & 31, warp = tid >> 5;
  auto meet = [&]() {                  // a CTA alone needs no cluster's barrier
    if (C > 1) cluster.sync();
    else __syncthreads();
  };
  pdl_trigger();
  pdl_wait();
  const EvictUnit U(A, unit, rank);
  const int n = U.n;
  if (n <= A.keep) {                   // the same for the whole cluster
    for (int i = rank * NT + tid; i < n; i += C * NT) U.copy(i);
    return;
  }
  const int sl = (n + C - 1) / C, s0 = min(n, rank * sl), cnt = min(n, s0 + sl) - s0;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  int2* list = reinterpret_cast<int2*>(smem + ((4u * (uint32_t)sl + 15u) & ~15u));

  // ---- keys
  if (tid == 0) {
    sh.newest = INT32_MIN;
    sh.movers = sh.freed = 0;
  }
#pragma unroll
  for (int d = 0; d < 4; ++d) sh.bins[d][tid] = 0;
  __syncthreads();
  int newest = INT32_MIN;
#pragma unroll 8
  for (int i = tid; i < cnt; i += NT) {
    newest = max(newest, U.held[s0 + i]);
    keys[i] = order_key(U.mass[s0 + i]);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (lane == 0) atomicMax(&sh.newest, newest);
  meet();
  for (int r = 0; r < C; ++r) newest = max(newest, *cluster.map_shared_rank(&sh.newest, r));
  const int64_t since = (int64_t)newest - A.recent;
  if (A.recent > 0)
#pragma unroll 8
    for (int i = tid; i < cnt; i += NT)
      if (U.held[s0 + i] > since) keys[i] = 0xffffffffu;

  // ---- the keep-th largest key: digits of 8 bits, `want` of those that match so far.  (Digits of
  // 11 bits take one round less, but every CTA reads the others' counts, and 64 KB of those
  // through the cluster's network took 10 us a round)
  uint32_t limit = 0, mask = 0;
  int want = A.keep;
#pragma unroll 1
  for (int d = 0; d < 4; ++d) {
    const int shift = 24 - 8 * d;
    int* bins = sh.bins[d];
#pragma unroll 4
    for (int i = tid; i < cnt; i += NT)
      if ((keys[i] & mask) == limit) atomicAdd(&bins[(keys[i] >> shift) & 255u], 1);
    meet();
    const int digit = kBins - 1 - tid;           // thread 0: the largest
    int mine = 0;
#pragma unroll
    for (int r = 0; r < kEvictCluster; ++r)
      if (r < C) mine += *cluster.map_shared_rank(&bins[digit], r);
    int total;
    const int above = block_excl_scan(mine, sh.scan, total);
    if (above < want && above + mine >= want) {
      sh.digit = digit;
      sh.above = above;
    }
    __syncthreads();
    limit |= (uint32_t)sh.digit << shift;
    mask |= 255u << shift;
    want -= sh.above;
    __syncthreads();
  }
  // kept: keys above the limit, and the first `want` of those equal to it.  A warp takes
  // a contiguous part of the slice, so that its counts need no barrier
  auto count = [&](bool p) { return __popc(__ballot_sync(0xffffffffu, p)); };
  auto before = [&](bool p) {
    return __popc(__ballot_sync(0xffffffffu, p) & ((1u << lane) - 1));
  };
  const int seg = (cnt + NT - 1) / NT * 32, w0 = min(cnt, warp * seg), w1 = min(cnt, w0 + seg);
  int equals = 0;
  for (int i = w0 + lane; i - lane < w1; i += 32) equals += count(i < w1 && keys[i] == limit);
  if (lane == 0) sh.of_warp[0][warp] = equals;
  __syncthreads();
  int equal = 0;                       // in the slices before this one: the last digit's counts
  for (int r = 0; r < rank; ++r) equal += *cluster.map_shared_rank(&sh.bins[3][limit & 255u], r);
  for (int w = 0; w < warp; ++w) equal += sh.of_warp[0][w];
  // keys become what happens to a slot: 0 it is given up, 1 moves away, 2 is filled, 3 stays
  int mv = 0, fr = 0;
#pragma unroll 2
  for (int i = w0 + lane; i - lane < w1; i += 32) {
    const bool in = i < w1;
    const uint32_t k = in ? keys[i] : 0u;
    const bool eq = in && k == limit;
    const int nth = equal + before(eq);          // every lane votes
    const bool kept = in && (k > limit || (eq && nth < want));
    equal += count(eq);
    const bool moves = kept && s0 + i >= A.keep, freed = in && !kept && s0 + i < A.keep;
    if (in) keys[i] = moves ? 1u : freed ? 2u : kept ? 3u : 0u;
    mv += count(moves);
    fr += count(freed);
  }
  if (lane == 0) {
    sh.of_warp[1][warp] = mv;
    sh.of_warp[2][warp] = fr;
    if (mv) atomicAdd(&sh.movers, mv);
    if (fr) atomicAdd(&sh.freed, fr);
  }
  meet();
  int movers = 0, freed = 0, all = 0;
  for (int r = 0; r < C; ++r) {
    const int m = *cluster.map_shared_rank(&sh.movers, r);
    if (r < rank) {
      movers += m;
      freed += *cluster.map_shared_rank(&sh.freed, r);
    }
    all += m;
  }
  for (int w = 0; w < warp; ++w) {
    movers += sh.of_warp[1][w];
    freed += sh.of_warp[2][w];
  }
  if (U.mass_out != U.mass || U.held_out != U.held)
#pragma unroll 4
    for (int i = w0 + lane; i < w1; i += 32)
      if (keys[i] == 3u) U.copy(s0 + i);
  // ---- mover k and freed slot k meet in the list of CTA k % C (a power of two)
  const int shift = 31 - __clz(C);
  for (int i = w0 + lane; i - lane < w1; i += 32) {
    const uint32_t what = i < w1 ? keys[i] : 0u;
    const int m = movers + before(what == 1u), f = freed + before(what == 2u);
    if (what == 1u) cluster.map_shared_rank(list, m & (C - 1))[m >> shift].x = s0 + i;
    if (what == 2u) cluster.map_shared_rank(list, f & (C - 1))[f >> shift].y = s0 + i;
    movers += count(what == 1u);
    freed += count(what == 2u);
  }
  meet();
  // no CTA's shared memory is read or written by others from here on

  // ---- a warp takes 32 moves: a lane each finds the rows of one, then the rows go over
  const EvictRows rows(A, unit % A.c.kv_heads);
  const int mine = all > rank ? (all - rank + C - 1) / C : 0;
  constexpr int MOVES = 32;
  for (int m0 = warp * MOVES; m0 < mine; m0 += kEvictWarps * MOVES) {
    int64_t from = -1, to = -1;
    if (m0 + lane < mine) {
      const int2 m = list[m0 + lane];
      U.mass_out[m.y] = U.mass[m.x];
      U.held_out[m.y] = U.held[m.x];
      from = EvictRows::at(A, U.table, m.x);
      to = EvictRows::at(A, U.table, m.y);
      if (from < 0 || to < 0) {
        set_status(A.status, MOE_STATUS_BAD_PAGE);
        from = to = -1;
      }
    }
    rows.move<8>(from, to, min(MOVES, mine - m0), lane);
  }
}

__global__ void evict_lens_kernel(int32_t* lens, int seqs, int keep, int most) {
  pdl_trigger();
  pdl_wait();
  const int s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s < seqs && lens[s] <= most) lens[s] = min(max(lens[s], 0), keep);
}

// Whether [a, a + n) and [b, b + m) share bytes.
static bool overlap(const void* a, int64_t n, const void* b, int64_t m) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}

static int launch_evict(EvictArgs& a, cudaStream_t s) {
  const int64_t blocks = (int64_t)a.c.seqs * a.c.kv_heads;
  // what sequences of max_len slots lose at most
  if (a.most - a.keep <= kFew && a.most <= kFewSlots) {
    MOE_REQUIRE(blocks <= 0x7fffffff, MOE_ERR_UNSUPPORTED, "%d sequences are too many", a.c.seqs);
    const size_t bytes = (size_t)std::max(4 * a.most, 16);
    if (bytes > 40 * 1024)
      MOE_CUDA(cudaFuncSetAttribute(evict_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    4 * kFewSlots));
    MOE_CUDA(launch_pdl(evict_few_kernel, dim3((unsigned)blocks), dim3(kEvictThreads), bytes, s, a));
    return MOE_OK;
  }
  // More CTAs for a head while the GPU is not full and a CTA would have a thousand
  // slots or more (the barriers of a cluster cost more than counting fewer)
  const int64_t units = (int64_t)a.c.seqs * a.c.kv_heads;
  int C = 1;
  while (C < kEvictCluster &&
         (a.most / C > kEvictSlots || (a.most / C >= 2048 && units * C < 4 * sm_count())))
    C *= 2;
  const int64_t sl = (a.most + C - 1) / C;
  MOE_REQUIRE(sl <= kEvictSlots, MOE_ERR_UNSUPPORTED,
              "sequences of %d slots: eviction takes up to %d", a.most, kEvictSlots * kEvictCluster);
  MOE_REQUIRE(units * C <= 0x7fffffff, MOE_ERR_UNSUPPORTED, "%d sequences are too many", a.c.seqs);
  const size_t smem = (size_t)(8 * sl + 64);
  MOE_CUDA(cudaFuncSetAttribute(evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                8 * kEvictSlots + 64));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * C));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, evict_kernel, a));
  return MOE_OK;
}

}  // namespace moe

extern "C" {

int moe_cache_evict_record(const moe_cache_evict_args* r) {
  MOE_REQUIRE(r, MOE_ERR_INVALID, "null arguments");
  moe::EvictArgs a = {};
  MOE_CHECK(moe::take_cache(&r->cache, a.c));
  MOE_CHECK(moe::check_cache_rows_apart(a.c));
  MOE_REQUIRE(r->keep > 0 && r->recent >= 0 && r->recent <= r->keep, MOE_ERR_INVALID,
              "keep %d, recent %d: 0 <= recent <= keep and keep > 0 are needed", r->keep, r->recent);
  MOE_REQUIRE(r->max_len >= 0, MOE_ERR_INVALID, "negative length");
  MOE_REQUIRE(r->ledger_slots > 0 && r->out_slots > 0, MOE_ERR_INVALID, "bad ledger");
  const int64_t most = std::min<int64_t>((int64_t)a.c.table_width * a.c.page_size, r->ledger_slots);
  a.most = (int)(r->max_len > 0 ? std::min<int64_t>(r->max_len, most) : most);
  MOE_REQUIRE(r->out_slots >= std::min(r->keep, a.most), MOE_ERR_INVALID,
              "%lld slots in the ledgers of the result, %d are kept", (long long)r->out_slots, r->keep);
  if (a.c.seqs == 0) return MOE_OK;
  MOE_REQUIRE(r->seq_lens && r->mass && r->held && r->mass_out && r->held_out && r->lens_out,
              MOE_ERR_INVALID, "null pointer");
  const int64_t units = (int64_t)a.c.seqs * a.c.kv_heads, in = 4 * units * r->ledger_slots,
                out = 4 * units * r->out_slots;
  const bool same = r->ledger_slots == r->out_slots;
  MOE_REQUIRE(((const void*)r->mass_out == r->mass && same) ||
                  !moe::overlap(r->mass, in, r->mass_out, out),
              MOE_ERR_INVALID, "mass and mass_out overlap, and are not the same");
  MOE_REQUIRE(((const void*)r->held_out == r->held && same) ||
                  !moe::overlap(r->held, in, r->held_out, out),
              MOE_ERR_INVALID, "held and held_out overlap, and are not the same");
  MOE_REQUIRE(!moe::overlap(r->mass, in, r->held_out, out) &&
                  !moe::overlap(r->held, in, r->mass_out, out) &&
                  !moe::overlap(r->mass_out, out, r->held_out, out),
              MOE_ERR_INVALID, "mass and held overlap");
  const bool in_place = r->lens_out == r->seq_lens;
  MOE_REQUIRE(in_place || !moe::overlap(r->seq_lens, 4ll * a.c.seqs, r->lens_out, 4ll * a.c.seqs),
              MOE_ERR_INVALID, "seq_lens and lens_out overlap, and are not the same");
  a.seq_lens = r->seq_lens;
  a.mass = r->mass;
  a.held = r->held;
  a.mass_out = r->mass_out;
  a.held_out = r->held_out;
  a.lens_out = r->lens_out;
  a.row = r->ledger_slots;
  a.row_out = r->out_slots;
  a.status = r->status;
  a.keep = r->keep;
  a.recent = r->recent;
  a.apart = !in_place;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(r->stream);
  {
    ::moe::ProfScope _prof(MOE_K_CACHE_EVICT, s);
    MOE_CHECK(moe::launch_evict(a, s));
  }
  if (in_place) {                      // other heads of a sequence read its length until then
    ::moe::ProfScope _prof(MOE_K_CACHE_EVICT, s);
    MOE_CUDA(moe::launch_pdl(moe::evict_lens_kernel, dim3((a.c.seqs + 255) / 256), dim3(256), 0, s,
                             r->lens_out, a.c.seqs, a.keep, a.most));
  }
  return moe::check_launch("cache_evict");
}

}  // extern "C"
