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
// The keep-th largest key comes from a radix select, 11 + 11 + 10 bits: counts in
// shared memory, added up across the cluster, and the digit found by a scan.  (The first
// digit holds sign, exponent and two bits: masses differ by powers of two, and 8-bit digits
// would put nearly all of them into four counters.)  Then the movers' numbers are
// prefix sums; CTA k % C gets mover k in a list and copies its rows, 16 bytes a lane.
//
// Bound by latency where few slots leave (the digits' three rounds), by memory where long
// prompts are cut: the rows that move, read and written once.
#include <cooperative_groups.h>

#include <algorithm>

#include "paged_cache.cuh"

namespace moe {
namespace cg = cooperative_groups;

constexpr int kEvictThreads = 256;
constexpr int kEvictCluster = 8;
constexpr int kEvictSlots = 20480;     // of a CTA at most: 8 bytes each in shared memory
constexpr int kDigit = 11;
constexpr int kBins = 1 << kDigit;

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
  int bins[kBins];
  int scan[33];
  int newest, digit, above;
  int equal, movers, freed;            // of this CTA: keys equal to the limit, movers, slots given up
};

// f32 -> u32 of the same order; +-0 are equal, NaN is last
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(kEvictThreads) evict_kernel(const EvictArgs A) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ EvictShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int unit = blockIdx.x / C, seq = unit / A.c.kv_heads, head = unit - seq * A.c.kv_heads;
  const int tid = threadIdx.x, NT = kEvictThreads;
  pdl_trigger();
  pdl_wait();
  const int told = max(A.seq_lens[seq], 0), n = told > A.most ? 0 : told;
  const bool first = head == 0 && rank == 0 && tid == 0;
  if (first) {
    if (told > A.most) set_status(A.status, MOE_STATUS_BAD_PAGE);   // left as it is
    if (A.apart) A.lens_out[seq] = told > A.most ? told : min(n, A.keep);
  }
  const float* mass = A.mass + (int64_t)unit * A.row;
  const int32_t* held = A.held + (int64_t)unit * A.row;
  float* mass_out = A.mass_out + (int64_t)unit * A.row_out;
  int32_t* held_out = A.held_out + (int64_t)unit * A.row_out;
  if (n <= A.keep) {                   // the same for the whole cluster
    if (mass_out != mass)
      for (int i = rank * NT + tid; i < n; i += C * NT) mass_out[i] = mass[i];
    if (held_out != held)
      for (int i = rank * NT + tid; i < n; i += C * NT) held_out[i] = held[i];
    return;
  }
  const int sl = (n + C - 1) / C, s0 = min(n, rank * sl), cnt = min(n, s0 + sl) - s0;
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  int2* list = reinterpret_cast<int2*>(smem + ((4u * (uint32_t)sl + 15u) & ~15u));

  // ---- keys
  if (tid == 0) sh.newest = INT32_MIN;
  __syncthreads();
  int newest = INT32_MIN;
  for (int i = tid; i < cnt; i += NT) {
    newest = max(newest, held[s0 + i]);
    keys[i] = order_key(mass[s0 + i]);
  }
  newest = __reduce_max_sync(0xffffffffu, newest);
  if (tid % 32 == 0) atomicMax(&sh.newest, newest);
  cluster.sync();
  newest = INT32_MIN;
  for (int r = 0; r < C; ++r) newest = max(newest, *cluster.map_shared_rank(&sh.newest, r));
  const int64_t since = (int64_t)newest - A.recent;
  if (A.recent > 0)
    for (int i = tid; i < cnt; i += NT)
      if (held[s0 + i] > since) keys[i] = 0xffffffffu;

  // ---- the keep-th largest key: digits from the top, `want` of those that match so far
  uint32_t limit = 0, mask = 0;
  int want = A.keep;
  for (int shift = 32 - kDigit; ; shift = max(0, shift - kDigit)) {
    // digits of 11, 11 and 10 bits
    const int bits = mask == 0 ? kDigit : min(kDigit, __ffs(mask) - 1);
    const uint32_t low = (1u << bits) - 1;
    for (int b = tid; b < kBins; b += NT) sh.bins[b] = 0;
    __syncthreads();
    for (int i = tid; i < cnt; i += NT)
      if ((keys[i] & mask) == limit) atomicAdd(&sh.bins[(keys[i] >> shift) & low], 1);
    cluster.sync();
    // thread tid: 8 digits, from the largest down
    constexpr int PER = kBins / kEvictThreads;
    int sums[PER], mine = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) sums[j] = 0;
    for (int r = 0; r < C; ++r) {
      const int4* bins =
          reinterpret_cast<const int4*>(cluster.map_shared_rank(&sh.bins[0], r) + kBins - PER * (tid + 1));
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) {
        const int4 v = bins[j];
        sums[4 * j] += v.x;
        sums[4 * j + 1] += v.y;
        sums[4 * j + 2] += v.z;
        sums[4 * j + 3] += v.w;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) mine += sums[j];
    int total;
    int above = block_excl_scan(mine, sh.scan, total);
    if (above < want && above + mine >= want) {
      bool found = false;
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        if (!found && above + sums[j] >= want) {
          found = true;
          sh.digit = kBins - PER * (tid + 1) + j;
          sh.above = above;
        }
        above += sums[j];
      }
    }
    cluster.sync();                    // the counts have been read; digit and above are there
    limit |= (uint32_t)sh.digit << shift;
    mask |= low << shift;
    want -= sh.above;
    if (shift == 0) break;
  }
  // kept: keys above the limit, and the first `want` of those equal to it

  // ---- equals in the slices before this one
  auto count = [&](bool p) { return __popc(__ballot_sync(0xffffffffu, p)); };
  if (tid == 0) sh.equal = sh.movers = sh.freed = 0;
  __syncthreads();
  const int rounds = (cnt + NT - 1) / NT;
  for (int j = 0; j < rounds; ++j) {
    const int i = tid + j * NT;
    const int e = count(i < cnt && keys[i] == limit);
    if (tid % 32 == 0 && e) atomicAdd(&sh.equal, e);
  }
  cluster.sync();
  int equal = 0;
  for (int r = 0; r < rank; ++r) equal += *cluster.map_shared_rank(&sh.equal, r);
  // keys become what happens to a slot: 0 nothing, 1 moves away, 2 is filled
  for (int j = 0; j < rounds; ++j) {
    const int i = tid + j * NT;
    const uint32_t k = i < cnt ? keys[i] : 0u;
    const bool eq = i < cnt && k == limit;
    int total;
    const int before = block_excl_scan(eq ? 1 : 0, sh.scan, total);
    const bool kept = i < cnt && (k > limit || (eq && equal + before < want));
    equal += total;
    const bool moves = kept && s0 + i >= A.keep, freed = i < cnt && !kept && s0 + i < A.keep;
    if (i < cnt) keys[i] = moves ? 1u : freed ? 2u : 0u;
    if (i < cnt && kept && !moves) {
      if (mass_out != mass) mass_out[s0 + i] = mass[s0 + i];
      if (held_out != held) held_out[s0 + i] = held[s0 + i];
    }
    const int m = count(moves), f = count(freed);
    if (tid % 32 == 0) {
      if (m) atomicAdd(&sh.movers, m);
      if (f) atomicAdd(&sh.freed, f);
    }
  }
  cluster.sync();
  int movers = 0, freed = 0, all = 0;
  for (int r = 0; r < C; ++r) {
    const int m = *cluster.map_shared_rank(&sh.movers, r);
    if (r < rank) {
      movers += m;
      freed += *cluster.map_shared_rank(&sh.freed, r);
    }
    all += m;
  }
  // ---- mover k and freed slot k meet in the list of CTA k % C
  for (int j = 0; j < rounds; ++j) {
    const int i = tid + j * NT;
    const uint32_t what = i < cnt ? keys[i] : 0u;
    int total;
    const int k = block_excl_scan(what == 1u ? 1 : what == 2u ? 1 << 16 : 0, sh.scan, total);
    if (what == 1u) {
      const int at = movers + (k & 0xffff);
      cluster.map_shared_rank(list, at % C)[at / C].x = s0 + i;
    } else if (what == 2u) {
      const int at = freed + (k >> 16);
      cluster.map_shared_rank(list, at % C)[at / C].y = s0 + i;
    }
    movers += total & 0xffff;
    freed += total >> 16;
  }
  cluster.sync();

  // ---- rows: 16 bytes a lane, keys and values
  const int eb = A.c.dtype == MOE_CACHE_E4M3 ? 1 : 2, ps = A.c.page_size;
  const int lines = A.c.head_dim * eb / 16;                  // of a row, at most 32
  const int32_t* table = A.c.block_table + (int64_t)seq * A.c.table_stride;
  const int mine = all > rank ? (all - rank + C - 1) / C : 0;
  uint8_t* kc = static_cast<uint8_t*>(A.c.k) + (int64_t)head * A.c.head_stride * eb;
  const int64_t v_less_k = (int64_t)((uintptr_t)A.c.v - (uintptr_t)A.c.k);
  const uint32_t per_line = 65536u / (uint32_t)lines + 1;    // i / lines = i * per_line >> 16, i < 2048
  auto row_of = [&](int slot) -> int64_t {
    const int p = slot / ps, page = table[p];
    if (page < 0 || page >= A.c.pages) return -1;
    return ((int64_t)page * A.c.page_stride + (int64_t)(slot - p * ps) * A.c.token_stride) * eb;
  };
  // a warp takes 32 moves: each lane finds the rows of one, then the rows go over
  // several at a time
  const int lane = tid % 32, warps = NT / 32;
  for (int m0 = tid / 32 * 32; m0 < mine; m0 += warps * 32) {
    int64_t from = -1, to = -1;
    if (m0 + lane < mine) {
      const int2 mv = list[m0 + lane];
      mass_out[mv.y] = mass[mv.x];
      held_out[mv.y] = held[mv.x];
      from = row_of(mv.x);
      to = row_of(mv.y);
      if (from < 0 || to < 0) {
        set_status(A.status, MOE_STATUS_BAD_PAGE);
        from = to = -1;
      }
    }
    const int items = 2 * min(32, mine - m0) * lines;
    constexpr int B = 8;                                     // loads under way
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
        if (dst[b] != -1) v[b] = *reinterpret_cast<const uint4*>(kc + f + off);
      }
#pragma unroll
      for (int b = 0; b < B; ++b)
        if (dst[b] != -1) *reinterpret_cast<uint4*>(kc + dst[b]) = v[b];
    }
  }
  // no CTA ends while others may still read its shared memory: the last such
  // reads and writes were before the barrier in front of the rows
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
