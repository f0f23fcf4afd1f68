// y = W x (+ residual) for a few rows, W in packed Q4_0 / Q8_0 tiles.
//
// Each weight is read once for up to 16 rows, so the bound is memory up to
// about 8 rows, and mma.sync issue beyond.  As in the experts' GEMVs the quants
// themselves are the (exact fp16) A operand, x enters as fp16 hi + lo columns (4
// rows fill the 8 columns of an MMA), and a 32-weight block is scaled in f32 after
// its sum.  The quants are made signed: as subnormals with their offset in the
// accumulator, the experts' form, they take 8 half-precision operations per
// 512 weights less (262144 x 2816 for one row 75 us instead of 83 then), but the
// tensor core aligns the subnormals' products to exponents 7 bits too large, and
// the result was off by up to 1.1e-6 of its norm instead of 1e-7.
//
// One CTA of 16 warps per SM stays resident.  It turns its columns of x into
// fragments in shared memory once, while the first weights are under way, and
// then its warps stream W: a warp owns pairs of 16-row strips (two strips share
// each fragment read) and 1 / ks of their columns, through a ring of bulk
// copies.  Where x is too wide for one SM's shared memory (or W has few rows) a
// cluster of cs CTAs splits the columns, so that each converts only its part of
// x; each CTA then stores its sums in the shared memory of the one that adds them.
// The split (cs, ks) is the one with the least estimated time; sums are in a fixed
// order.
//
// Measured on a B200 (copy bandwidth 6.55 TB/s): 262144 x 2816 Q4_0 for one row 70
// us in a short run (416 MB, 90 %), 77 to 83 us in calls that go on and on (77 to 82
// %: the load lowers the clock, and instructions come next), 65536 x 2816 for 1, 4,
// 8, 16 rows 22.4, 24.5, 35.6, 53 us (floor 15.9), 6144 x 2816 for one row 6.0 us, of which 4 are launch, fragments and
// the meeting of the warps, 4096 x 8192 for 16 rows 17.1 us (fragments 4.4, weights
// 8.5 where the MMAs alone take 4.3, meetings 3.3).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "packed_tiles.cuh"

namespace moe {

constexpr int kLinWarps = 16;
constexpr int kLinMaxStages = 8;      // barriers of a warp
constexpr int kLinHead = 2048;         // barriers, row maxima and scales
constexpr int kLinSmem = 226 * 1024;

struct LinArgs {
  const uint8_t* w;
  const float *x, *residual;
  float* y;
  int64_t xs, rs, ys;
  int rows, cols, T;
  int kt;                              // tiles of a strip
  int pairs;                           // pairs of strips
  int cs, ks, tps, nst, rounds, vec;   // tps: tiles of a CTA's columns
};

__device__ __forceinline__ float pow2f(int e) {   // -126 <= e <= 127
  return __uint_as_float((uint32_t)(127 + e) << 23);
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

// The eight columns of an MMA are four pairs (hi part, lo part).  With 3 rows of
// x or more a pair is a row, and G column groups hold up to 4 G rows.  With one
// or two rows the pairs are NBG = 4 or 2 consecutive 32-weight blocks of a row
// (the fragment of a block is zero in the other blocks' columns): one
// accumulator then serves NBG blocks, and a lane scales its own block only.
template <int NBG, int G> struct LinCfg {
  static constexpr int kTok = 4 / NBG;           // rows of a column group
  static constexpr int kRows = kTok * G;         // rows of a pass
  static constexpr int kRed = 2 * G * 2 * 32;    // floats of a pair of strips
  static constexpr int kTileBytes = G * 2 * 512; // fragments of a tile's two blocks
};

// x columns [64 t0, 64 t1) of n rows -> fragments `rec` ([block][column group] of
// 512 bytes); a row times 2^ex has its largest finite |x| in [2^14, 2^15).
template <int QT, int NBG, int G>
__device__ __forceinline__ void build_fragments(const LinArgs& A, uint8_t* rec, int rec_blocks,
                                                int* ex, uint32_t* smax, int row0, int n, int t0,
                                                int t1) {
  constexpr int TOK = LinCfg<NBG, G>::kTok, ROWS = LinCfg<NBG, G>::kRows;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  const int nb = 2 * (t1 - t0), real = min(nb, A.cols / 32 - 2 * t0);   // blocks, with columns
  const int P = n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16;
  const int wpr = kLinWarps / P, row = warp / wpr, part = warp % wpr;   // warps of a row
  const bool on = row < n;
  const float* x = A.x + (int64_t)(row0 + (on ? row : 0)) * A.xs + (int64_t)t0 * 64;
  auto values = [&](int b, float (&v)[8]) {
    const int c0 = 32 * b + (QT == MOE_Q4_0 ? 4 * t : 8 * t), c1 = c0 + (QT == MOE_Q4_0 ? 16 : 4);
    if (A.vec) {
      const float4 a = *reinterpret_cast<const float4*>(x + c0);
      const float4 c = *reinterpret_cast<const float4*>(x + c1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = c.x; v[5] = c.y; v[6] = c.z; v[7] = c.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = x[c0 + i];
        v[4 + i] = x[c1 + i];
      }
    }
  };
  if (tid < ROWS) ex[tid] = 0;
  if (NBG > 1 || n < ROWS || real < rec_blocks)  // else every place is written below
    for (int i = tid; i < G * rec_blocks * 32; i += kLinWarps * 32)
      reinterpret_cast<uint4*>(rec)[i] = make_uint4(0, 0, 0, 0);
  // with 16 rows the first loads of a lane stay in registers for the second pass;
  // with fewer the code costs more than the second load (first use of an
  // instruction line: 4096 columns of one row 4.8 -> 5.3 us)
  constexpr int KEEP = G == 4 ? 8 : 0;
  const int b0 = part * 8 + (lane >> 2), step = wpr * 8;
  float kept[KEEP + 1][8];
  uint32_t mx = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (on && b0 + i * step < real) values(b0 + i * step, kept[i]);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (on && b0 + i * step < real)
#pragma unroll
      for (int k = 0; k < 8; ++k) mx = max(mx, __float_as_uint(fabsf(kept[i][k])));
  if (on)
#pragma unroll 4
    for (int b = b0 + KEEP * step; b < real; b += step) {
      float v[8];
      values(b, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) mx = max(mx, __float_as_uint(fabsf(v[k])));
    }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (lane == 0) smax[warp] = mx;
  __syncthreads();
  if (!on) return;
  mx = 0;
  for (int i = 0; i < wpr; ++i) mx = max(mx, smax[row * wpr + i]);
  const bool special = mx >= 0x7f800000u;        // Inf or NaN: the scale goes by the others,
  if (special) {                                 // which each warp of the row looks up for itself
    mx = 0;
    for (int b = lane >> 2; b < real; b += 8) {
      float v[8];
      values(b, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t u = __float_as_uint(fabsf(v[k]));
        if (u < 0x7f800000u) mx = max(mx, u);
      }
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
  }
  const int eb = (int)(mx >> 23);                // biased exponent
  const int e = mx == 0 ? 0 : 141 - max(eb, 1);
  const float f1 = pow2f(e / 2), f2 = pow2f(e - e / 2);
  if (part == 0 && lane == 0) ex[row] = e;
  const int cg = row / TOK;
  auto put = [&](int b, const float (&v)[8], auto inf) {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      // register slots i, i + 1 hold elements 0, 2 | 1, 3 of each four (Q4_0)
      const int p = QT == MOE_Q4_0 ? (i & 4) + ((i & 2) ? 1 : 0) : i;
      const int q = QT == MOE_Q4_0 ? p + 2 : i + 1;
      const float a = v[p] * f1 * f2, c = v[q] * f1 * f2;
      const __half2 h = __floats2half2_rn(a, c);
      float al = a - __low2float(h), cl = c - __high2float(h);
      if (inf.value) {                           // an infinity is its hi part alone
        if (isinf(a)) al = 0.f;
        if (isinf(c)) cl = 0.f;
      }
      const __half2 l = __floats2half2_rn(al, cl);
      hi[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
      lo[i / 2] = *reinterpret_cast<const uint32_t*>(&l);
    }
    const int pair = (b % NBG) * TOK + row % TOK;
    uint8_t* r = rec + (size_t)(b * G + cg) * 512 + pair * 128 + t * 16;
    // blocks lie on the same banks: the odd ones write their lo half first
    const bool odd = b & 1;
    *reinterpret_cast<uint4*>(r + (odd ? 64 : 0)) =
        odd ? make_uint4(lo[0], lo[1], lo[2], lo[3]) : make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(r + (odd ? 0 : 64)) =
        odd ? make_uint4(hi[0], hi[1], hi[2], hi[3]) : make_uint4(lo[0], lo[1], lo[2], lo[3]);
  };
  if (special) {
    for (int b = b0; b < real; b += step) {
      float v[8];
      values(b, v);
      put(b, v, std::true_type());
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (b0 + i * step < real) put(b0 + i * step, kept[i], std::false_type());
#pragma unroll 2
  for (int b = b0 + KEEP * step; b < real; b += step) {
    float v[8];
    values(b, v);
    put(b, v, std::false_type());
  }
}

template <int QT, int NBG, int G, int U>
__global__ void __launch_bounds__(kLinWarps * 32, 1) linear_kernel(const LinArgs A) {
  using Tr = QTraits<QT>;
  using Cfg = LinCfg<NBG, G>;
  constexpr int TB = Tr::kTileBytes, STAGE = 2 * U * TB, NRED = Cfg::kRed;
  constexpr int TOK = Cfg::kTok;
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* const bars_all = reinterpret_cast<uint64_t*>(smem);
  uint32_t* const smax = reinterpret_cast<uint32_t*>(smem + 1024);
  int* const ex = reinterpret_cast<int*>(smem + 1024 + 64);
  volatile int* const dead = reinterpret_cast<volatile int*>(smem + 1024 + 128);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % A.cs, cluster = blockIdx.x / A.cs, nclusters = gridDim.x / A.cs;
  const int groups = kLinWarps / A.ks, group = warp / A.ks, kq = warp % A.ks;
  const int row0 = blockIdx.y * Cfg::kRows, n = min(Cfg::kRows, A.T - row0);
  // columns: this CTA's tiles, this warp's (an even number: whole stages)
  const int tps = A.tps, t0 = min(A.kt, rank * tps), t1 = min(A.kt, t0 + tps);
  const int wps = ((t1 - t0 + A.ks - 1) / A.ks + 1) / 2 * 2;
  const int wt0 = min(t1, t0 + kq * wps), wt1 = min(t1, wt0 + wps), nt = wt1 - wt0;
  const int rec_blocks = 2 * tps;                // tps is even
  uint8_t* const rec = smem + kLinHead;
  // Sums of the warps: in their rings, which are read out when the only round
  // ends, or in places of their own
  const bool own_red = A.ks > 1 && A.rounds > 1;
  float* const red0 = reinterpret_cast<float*>(rec + (size_t)tps * Cfg::kTileBytes);
  float* const part = red0 + (own_red ? kLinWarps * NRED : 0);
  // sums of a round in rows of 32, dealt out to the CTAs of the cluster
  const int red_rows = groups * (NRED / 32), own_rows = (red_rows + A.cs - 1) / A.cs;
  uint8_t* const rings = reinterpret_cast<uint8_t*>(
      part + (A.cs > 1 ? (A.rounds > 1 ? 2 : 1) * A.cs * own_rows * 32 : 0));
  uint8_t* const ring = rings + warp * A.nst * STAGE;
  float* const red = own_red ? red0 : reinterpret_cast<float*>(rings);
  const int red_step = own_red ? NRED : A.nst * STAGE / 4;   // floats from warp to warp
  uint64_t* const bars = bars_all + warp * kLinMaxStages;

  if (lane < A.nst) {
    mbar_init(&bars[lane], 1);
    fence_mbar_init();
  }
  if (tid == 0) *dead = 0;                       // seen by all after build_fragments
  if (A.cs > 1) cluster_arrive();                // waited for before the first store to another CTA
  __syncwarp();
  pdl_trigger();

  // ---- weights: stage q of this warp is tiles [wt0 + j U, ..) of pair `p`
  const int nsr = (nt + U - 1) / U;              // stages of a pair
  // pairs go round the clusters, so that few of them still use every SM
  const int p0 = group * nclusters + cluster, pstep = nclusters * groups;
  const int mine = p0 < A.pairs ? (A.pairs - p0 + pstep - 1) / pstep : 0;
  const int total = mine * nsr;
  const uint64_t pol = evict_first_policy();
  const int strips = (A.rows + 15) / 16;
  int ip = p0, ij = 0, islot = 0, issued = 0;
  const int64_t strip = (int64_t)A.kt * TB;      // bytes from strip to strip
  // lanes 0 and 1 copy a strip each
  const uint8_t* src = A.w + (2 * ip + (lane & 1)) * strip + (int64_t)wt0 * TB;
  const int last = (nt - (nsr - 1) * U) * TB;    // bytes of a pair's last stage
  auto issue = [&]() {                           // stage `issued`
    const uint32_t bytes = ij == nsr - 1 ? last : U * TB;
    const int n = 2 * ip + 1 < strips ? 2 : 1;
    if (lane == 0) mbar_expect_tx(&bars[islot], n * bytes);
    if (lane < n) bulk_g2s(ring + islot * STAGE + lane * U * TB, src, bytes, &bars[islot], pol);
    ++issued;
    src += U * TB;
    islot = islot + 1 == A.nst ? 0 : islot + 1;
    if (++ij == nsr) {
      ij = 0;
      ip += pstep;
      src += 2 * pstep * strip - (int64_t)nsr * U * TB;
    }
  };
  pdl_wait();
  for (int q = 0; q < A.nst && q < total; ++q) issue();
  build_fragments<QT, NBG, G>(A, rec, rec_blocks, ex, smax, row0, n, t0, t1);
  __syncthreads();

  // ---- stream
  int slot = 0;
  uint32_t phase = 0;
  // fragments of this warp's columns
  const uint8_t* const xl = rec + lane * 16 + (size_t)2 * (wt0 - t0) * G * 512;
  // value k = 2 (s G + cg) + i of lane l: row g + 8 i of strip s of pair p, row of x
  // of column group cg
  auto place = [&](int p, int k, int l, int& tok, int& row) {
    tok = TOK * (k / 2 % G) + (l & 3);
    row = 32 * p + 16 * (k / (2 * G)) + (l >> 2) + 8 * (k % 2);
    return (l & 3) < TOK && tok < n && row < A.rows;
  };
  auto residual_at = [&](int tok, int row) {
    return A.residual ? A.residual[(int64_t)(row0 + tok) * A.rs + row] : 0.f;
  };
  auto store = [&](int tok, int row, float y) { A.y[(int64_t)(row0 + tok) * A.ys + row] = y; };
  for (int r = 0; r < A.rounds; ++r) {
    const int p = p0 + r * pstep;
    float v[2][G][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int cg = 0; cg < G; ++cg) v[s][cg][0] = v[s][cg][1] = 0.f;
    if (p < A.pairs) {
      for (int j = 0; j < nsr; ++j) {
        // bounded; after a timeout anywhere in the CTA no wait takes long any more
        if (!mbar_test(&bars[slot], phase) && !*dead && !mbar_wait(&bars[slot], phase)) *dead = 1;
        __syncwarp();
        const uint8_t* st = ring + slot * STAGE;
        const uint8_t* xq = xl + j * (U * 2 * G * 512);
        const int left = nt - j * U;             // tiles of the stage, U or more: all
        float c[2][G][4];
        auto begin = [&]() {                     // of a group of blocks
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cg = 0; cg < G; ++cg) c[s][cg][0] = c[s][cg][1] = c[s][cg][2] = c[s][cg][3] = 0.f;
        };
        auto finish = [&](int tile, int half, bool valid) {   // scales of this lane's block
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const __half* d = reinterpret_cast<const __half*>(st + (s * U + tile) * TB +
                                                              Tr::kTileQuant + g * 8) + half;
            const float d0 = valid ? __half2float(d[0]) : 0.f;
            const float d8 = valid ? __half2float(d[2]) : 0.f;
#pragma unroll
            for (int cg = 0; cg < G; ++cg) {
              v[s][cg][0] = fmaf(d0, c[s][cg][0] + c[s][cg][1], v[s][cg][0]);
              v[s][cg][1] = fmaf(d8, c[s][cg][2] + c[s][cg][3], v[s][cg][1]);
            }
          }
        };
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u == 0 || u < left) {
            if (NBG == 4 && u % 2 == 0) begin();
            TileRegs<QT> w[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) lds_quants<QT>(w[s], st + (s * U + u) * TB, lane);
            if (NBG == 2) begin();
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              if (NBG == 1) begin();
              uint32_t a0[2][4], a1[2][4];
#pragma unroll
              for (int s = 0; s < 2; ++s) tile_quants<QT, false>(w[s], b, a0[s], a1[s]);
#pragma unroll
              for (int cg = 0; cg < G; ++cg) {
                const uint4 xf =
                    *reinterpret_cast<const uint4*>(xq + ((2 * u + b) * G + cg) * 512);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                  mma_16816(c[s][cg], a0[s][0], a0[s][1], a0[s][2], a0[s][3], xf.x, xf.y, c[s][cg]);
                  mma_16816(c[s][cg], a1[s][0], a1[s][1], a1[s][2], a1[s][3], xf.z, xf.w, c[s][cg]);
                }
              }
              if (NBG == 1) finish(u, b, true);
            }
            if (NBG == 2) finish(u, t >> 1, true);
          }
          // four blocks: the lane's is in tile t / 2 of the two
          if (NBG == 4 && u % 2 == 1 && u - 1 < left)
            finish(u - 1 + (t >> 1), t & 1, u - 1 + (t >> 1) < left);
        }
        __syncwarp();                            // the stage has been read
        if (issued < total && !*dead) issue();
        if (++slot == A.nst) {
          slot = 0;
          phase ^= 1u;
        }
      }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int cg = 0; cg < G; ++cg)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (NBG >= 2) v[s][cg][i] += __shfl_xor_sync(0xffffffffu, v[s][cg][i], 2);
          if (NBG == 4) v[s][cg][i] += __shfl_xor_sync(0xffffffffu, v[s][cg][i], 1);
        }
    float rv[2][G][2];                           // residuals, on the way while the warps meet
    if (A.cs == 1 && kq == 0)
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int cg = 0; cg < G; ++cg)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            int tok, row;
            const bool here = place(p, (s * G + cg) * 2 + i, lane, tok, row);
            rv[s][cg][i] = here ? residual_at(tok, row) : 0.f;
          }
    if (A.ks > 1) {
      // the column parts of a pair meet in the group's first warp
      if (r > 0) asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * A.ks) : "memory");
      if (kq > 0)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int cg = 0; cg < G; ++cg)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              red[warp * red_step + ((s * G + cg) * 2 + i) * 32 + lane] = v[s][cg][i];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * A.ks) : "memory");
      if (kq == 0)
        for (int k = 1; k < A.ks; ++k)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cg = 0; cg < G; ++cg)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                v[s][cg][i] += red[(warp + k) * red_step + ((s * G + cg) * 2 + i) * 32 + lane];
    }
    if (*dead)                                   // a wait ran out: NaN
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int cg = 0; cg < G; ++cg) v[s][cg][0] = v[s][cg][1] = __uint_as_float(0x7fffffffu);
    const bool lead = kq == 0 && p < A.pairs;
    if (lead) {
#pragma unroll
      for (int cg = 0; cg < G; ++cg) {
        const int e = ex[TOK * cg + (t < TOK ? t : 0)];
        const float f1 = pow2f(-(e / 2)), f2 = pow2f(-(e - e / 2));
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) v[s][cg][i] = v[s][cg][i] * f1 * f2;
      }
    }
    if (A.cs == 1) {
      if (lead) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int cg = 0; cg < G; ++cg)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              int tok, row;
              if (place(p, (s * G + cg) * 2 + i, lane, tok, row))
                store(tok, row, v[s][cg][i] + rv[s][cg][i]);
            }
      }
    } else {
      // The CTAs' parts: row c goes to CTA c % cs, which adds up the rows that
      // it gets.  A buffer is used again two rounds later, behind the barrier of
      // the round between.
      float* mine_p = part + (size_t)(r & 1) * A.cs * own_rows * 32;
      const uint32_t to = smem_u32(mine_p);
      if (r == 0) cluster_wait();
      if (kq == 0)
#pragma unroll
        for (int k = 0; k < NRED / 32; ++k) {
          const int c = group * (NRED / 32) + k, own = c / A.cs;
          st_cluster(to + ((rank * own_rows + own) * 32 + lane) * 4, c - own * A.cs,
                     v[k / (2 * G)][k / 2 % G][k % 2]);
        }
      // this warp's first row, and its residual on the way meanwhile
      int tok = 0, row = 0;
      auto find = [&](int own) {
        const int c = own * A.cs + rank, gr = c / (NRED / 32);
        const int pe = gr * nclusters + cluster + r * pstep;
        return c < red_rows && pe < A.pairs && place(pe, c - gr * (NRED / 32), lane, tok, row);
      };
      bool here = warp < own_rows && find(warp);
      float y = here ? residual_at(tok, row) : 0.f;
      cluster_sync();
      for (int own = warp; own < own_rows; own += kLinWarps) {
        if (own != warp) {
          here = find(own);
          y = here ? residual_at(tok, row) : 0.f;
        }
        float sum = 0.f;
        for (int c = 0; c < A.cs; ++c) sum += mine_p[(c * own_rows + own) * 32 + lane];
        if (here) store(tok, row, sum + y);
      }
    }
  }
  // after a timeout the copies already issued are still waited for (bounded)
  if (*dead)
    for (int i = 0; i < A.nst; ++i) {
      mbar_wait(&bars[i], 0);
      mbar_wait(&bars[i], 1);
    }
}

// Tiles of a CTA's columns: an even number, so that a stage is two of them.
inline int linear_tps(int kt, int cs) { return ((kt + cs - 1) / cs + 1) / 2 * 2; }

// Shared memory of a split in so many rounds with nst ring stages.
template <int QT, int NBG, int G, int U>
static size_t linear_smem(int kt, int cs, int ks, int rounds, int nst) {
  using Cfg = LinCfg<NBG, G>;
  const size_t own_rows = (kLinWarps / ks * (Cfg::kRed / 32) + cs - 1) / cs;
  static_assert(Cfg::kRed * 4 <= 2 * 2 * U * QTraits<QT>::kTileBytes, "sums in a ring");
  return kLinHead + (size_t)linear_tps(kt, cs) * Cfg::kTileBytes +
         (ks > 1 && rounds > 1 ? kLinWarps * Cfg::kRed * 4 : 0) +
         (cs > 1 ? (rounds > 1 ? 2 : 1) * 128 * cs * own_rows : 0) +
         (size_t)kLinWarps * nst * 2 * U * QTraits<QT>::kTileBytes;
}

// Clusters of cs CTAs that are resident at once (a cluster stays inside one GPC:
// 148 SMs hold 74, 33 and 15 clusters of 2, 4 and 8).
static int resident_clusters(const void* kern, int cs, int dev) {
  static std::atomic<int> known[64][4];
  const int k = cs == 2 ? 1 : cs == 4 ? 2 : 3;
  if (cs == 1) return sm_count();
  int n = dev < 64 ? known[dev][k].load() : 0;
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(cs * 148));
    cfg.blockDim = dim3(kLinWarps * 32);
    cfg.dynamicSmemBytes = kLinSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cs;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = std::max(1, sm_count() / (2 * cs));
    }
    if (dev < 64) known[dev][k].store(n);
  }
  return n;
}

template <int QT, int NBG, int G, int U>
static int linear_ready(int& dev) {
  static std::atomic<uint64_t> ready{0};
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((ready.load() >> dev) & 1)) {
    MOE_CUDA(cudaFuncSetAttribute(linear_kernel<QT, NBG, G, U>,
                                  cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmem));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  return MOE_OK;
}

// The split (cs, ks) of a size with the least estimated time.
struct LinPlan {
  int dev = -1, kt, pairs, cs, ks, nst, clusters, rounds;
  double time;
};
template <int QT, int NBG, int G, int U>
static const LinPlan& linear_plan(const LinArgs& a, int dev) {
  using Cfg = LinCfg<NBG, G>;
  // the plans of a few sizes are remembered, for calls that repeat them
  static thread_local LinPlan plans[16];
  LinPlan& plan = plans[(a.kt * 31 + a.pairs) & 15];
  if (plan.dev == dev && plan.kt == a.kt && plan.pairs == a.pairs) return plan;
  plan = {dev, a.kt, a.pairs, 0, 0, 2, 0, 0, 0};
  // Microseconds: rounds x (tiles of a warp, the meetings of warps and of a
  // cluster), the tiles again by the share of the warps that have work, and the
  // fragments of the CTA's columns.  Fitted to all splits of 15 sizes with 1, 4, 8
  // and 16 rows; the split that it takes is 0.6 % slower than the best one on
  // average (8 % at worst).
  const double g = G - 1;
  const double tile = 0.13 + 0.06 * g + (QT == MOE_Q8_0 ? 0.18 : 0) + (U == 1 ? 0.06 : 0);
  const double share = 0.1 + 0.05 * g, frag = 0.018 * G + 0.003 * Cfg::kRows;
  const double warps_meet = 0.46 + 0.04 * g, ctas_meet = 1.36 + 0.56 * g;
  for (int cs = 1; cs <= 8; cs *= 2) {
    const int resident =
        resident_clusters((const void*)linear_kernel<QT, NBG, G, U>, cs, dev);
    for (int ks = 1; ks <= kLinWarps; ks *= 2) {
      const int tps = linear_tps(a.kt, cs), wt = ((tps + ks - 1) / ks + 1) / 2 * 2;
      const int slots = resident * (kLinWarps / ks);   // pairs of a round
      const int rounds = (a.pairs + slots - 1) / slots;
      if (linear_smem<QT, NBG, G, U>(a.kt, cs, ks, rounds, 2) > kLinSmem) continue;
      const double t =
          rounds * (wt * tile + (ks > 1 ? warps_meet : 0) + (cs > 1 ? ctas_meet : 0)) +
          (double)a.pairs / slots * wt * share + tps * frag;
      if (plan.cs == 0 || t < plan.time) {
        plan.time = t;
        plan.cs = cs;
        plan.ks = ks;
        plan.clusters = std::min(resident, a.pairs);
        plan.rounds = rounds;
      }
    }
  }
  while (plan.cs > 0 && plan.nst < (U > 1 ? 4 : kLinMaxStages) &&
         linear_smem<QT, NBG, G, U>(a.kt, plan.cs, plan.ks, plan.rounds, plan.nst + 1) <= kLinSmem)
    ++plan.nst;
  return plan;
}

template <int QT, int NBG, int G, int U>
static int launch_linear(LinArgs& a, cudaStream_t s, bool& fits) {
  using Cfg = LinCfg<NBG, G>;
  int dev = 0;
  MOE_CHECK((linear_ready<QT, NBG, G, U>(dev)));
  const LinPlan& plan = linear_plan<QT, NBG, G, U>(a, dev);
  fits = plan.cs > 0;
  if (!fits) return MOE_OK;
  a.cs = plan.cs;
  a.ks = plan.ks;
  a.nst = plan.nst;
  a.tps = linear_tps(a.kt, a.cs);
  a.rounds = plan.rounds;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(plan.clusters * a.cs), (unsigned)((a.T + Cfg::kRows - 1) / Cfg::kRows));
  cfg.blockDim = dim3(kLinWarps * 32);
  cfg.dynamicSmemBytes = linear_smem<QT, NBG, G, U>(a.kt, a.cs, a.ks, a.rounds, a.nst);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.cs;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.cs > 1 ? 2 : 1;
  MOE_CUDA(cudaLaunchKernelEx(&cfg, linear_kernel<QT, NBG, G, U>, a));
  return MOE_OK;
}

// 16 rows, whose fragments take most of the shared memory: one tile per wait needs
// half the ring, which lets splits over fewer CTAs fit (Q8_0 4096 x 8192 18.6 us
// instead of 21.9).
template <int QT>
static int launch_linear_16(LinArgs& a, cudaStream_t s, bool& fits) {
  int dev = 0;
  MOE_CHECK((linear_ready<QT, 1, 4, 2>(dev)));
  MOE_CHECK((linear_ready<QT, 1, 4, 1>(dev)));
  const LinPlan &two = linear_plan<QT, 1, 4, 2>(a, dev), &one = linear_plan<QT, 1, 4, 1>(a, dev);
  if (one.cs > 0 && (two.cs == 0 || one.time < two.time))
    return launch_linear<QT, 1, 4, 1>(a, s, fits);
  return launch_linear<QT, 1, 4, 2>(a, s, fits);
}

// Rows of a pass: as many as T needs (1, 2, 4, 8 or 16), fewer where x is so wide
// that their fragments do not fit.  Up to 4 rows of 4-bit weights are bound by
// instructions, so four tiles are taken per wait where the ring fits (65536 x
// 2816: 1 row 25.7 -> 22.9 us, 4 rows 28.1 -> 24.9 us when it was done; 8 rows,
// nearer the MMAs' bound, 36.5 -> 37.4 us).
template <int QT>
static int launch_linear_qt(LinArgs& a, cudaStream_t s) {
  constexpr int U = QT == MOE_Q4_0 ? 4 : 2;
  bool fits = false;
  if (a.T > 8) MOE_CHECK((launch_linear_16<QT>(a, s, fits)));
  if (!fits && a.T > 4) MOE_CHECK((launch_linear<QT, 1, 2, 2>(a, s, fits)));
  if (!fits && a.T > 2) MOE_CHECK((launch_linear<QT, 1, 1, U>(a, s, fits)));
  if (!fits && a.T > 2 && U > 2) MOE_CHECK((launch_linear<QT, 1, 1, 2>(a, s, fits)));
  if (!fits && a.T == 2) MOE_CHECK((launch_linear<QT, 2, 1, U>(a, s, fits)));
  if (!fits && a.T == 2 && U > 2) MOE_CHECK((launch_linear<QT, 2, 1, 2>(a, s, fits)));
  if (!fits && a.T == 1) MOE_CHECK((launch_linear<QT, 4, 1, U>(a, s, fits)));
  if (!fits && a.T == 1 && U > 2) MOE_CHECK((launch_linear<QT, 4, 1, 2>(a, s, fits)));
  MOE_REQUIRE(fits, MOE_ERR_UNSUPPORTED, "cols %d: rows of x this wide do not fit", a.cols);
  return MOE_OK;
}

// n rows of f32 at a pointer, `width` elements each, `stride` apart.
struct Rows {
  const float* p;
  int64_t stride, width, n;
};

// Whether a row of a shares memory with a row of b.  Side by side in one buffer
// their spans may meet although no rows do, so rows are compared then.
static bool rows_overlap(Rows a, Rows b) {
  auto upward = [](Rows& r) {                    // the same rows in rising order
    if (r.stride < 0) {
      r.p += (r.n - 1) * r.stride;
      r.stride = -r.stride;
    }
  };
  upward(a);
  upward(b);
  const int64_t d = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p);   // bytes, as all from here on
  const int64_t as = 4 * a.stride, aw = 4 * a.width, bs = 4 * b.stride, bw = 4 * b.width;
  if (d >= (a.n - 1) * as + aw || d + (b.n - 1) * bs + bw <= 0) return false;
  for (int64_t i = 0; i < a.n; ++i) {
    const int64_t lo = i * as - bw - d, hi = i * as + aw - d;      // lo < offset of b's row < hi
    if (bs == 0 ? lo < 0 && 0 < hi
                : std::max<int64_t>(0, lo < 0 ? 0 : lo / bs + 1) <=
                      std::min(b.n - 1, hi <= 0 ? -1 : (hi - 1) / bs))
      return true;
  }
  return false;
}

}  // namespace moe

extern "C" int moe_linear(const uint8_t* w, int qtype, int rows, int cols, const float* x,
                          int64_t x_stride, int T, const float* residual, int64_t residual_stride,
                          float* y, int64_t y_stride, moe_stream_t stream) {
  MOE_REQUIRE(moe::qtype_ok(qtype), MOE_ERR_UNSUPPORTED, "quant type %d not supported", qtype);
  MOE_REQUIRE(rows > 0 && cols > 0 && T >= 0, MOE_ERR_INVALID, "bad shape");
  MOE_REQUIRE(cols % 32 == 0, MOE_ERR_UNSUPPORTED, "cols %d is not a multiple of 32", cols);
  MOE_REQUIRE(rows <= 0x7ffffff0 - 32, MOE_ERR_UNSUPPORTED, "%d rows are too many", rows);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(w && x && y, MOE_ERR_INVALID, "null pointer");
  MOE_REQUIRE((uintptr_t)w % 16 == 0, MOE_ERR_INVALID, "w must be 16-byte aligned");
  MOE_REQUIRE(T <= 65535 * 4, MOE_ERR_UNSUPPORTED, "%d rows of x are too many", T);
  MOE_REQUIRE(T == 1 || y_stride >= rows || -y_stride >= rows, MOE_ERR_INVALID,
              "rows of y overlap");
  const moe::Rows yr = {y, y_stride, rows, T};
  MOE_REQUIRE(!moe::rows_overlap({x, x_stride, cols, T}, yr), MOE_ERR_INVALID, "x and y overlap");
  MOE_REQUIRE(!residual || (residual == y && (T == 1 || residual_stride == y_stride)) ||
                  !moe::rows_overlap({residual, residual_stride, rows, T}, yr),
              MOE_ERR_INVALID, "residual and y overlap, and are not the same rows");
  moe::LinArgs a = {};
  a.w = w;
  a.x = x;
  a.residual = residual;
  a.y = y;
  a.xs = x_stride;
  a.rs = residual_stride;
  a.ys = y_stride;
  a.rows = rows;
  a.cols = cols;
  a.T = T;
  a.kt = (cols + 63) / 64;
  a.pairs = ((rows + 15) / 16 + 1) / 2;
  a.vec = (uintptr_t)x % 16 == 0 && (T == 1 || x_stride % 4 == 0);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  {
    ::moe::ProfScope _prof(MOE_K_LINEAR, s);
    MOE_CHECK(qtype == MOE_Q4_0 ? moe::launch_linear_qt<MOE_Q4_0>(a, s)
                                : moe::launch_linear_qt<MOE_Q8_0>(a, s));
  }
  return moe::check_launch("linear");
}

extern "C" int moe_linear_record(const moe_linear_args* a) {
  MOE_REQUIRE(a, MOE_ERR_INVALID, "null arguments");
  return moe_linear(a->w, a->qtype, a->rows, a->cols, a->x, a->x_stride, a->T, a->residual,
                    a->residual_stride, a->y, a->y_stride, a->stream);
}
