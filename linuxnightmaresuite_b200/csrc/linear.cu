// y = W x (+ residual) for a few rows, W in packed Q4_0 / Q8_0 tiles.
//
// Each weight is read once for up to 16 rows, so the bound is memory up to
// about 8 rows, and mma.sync issue beyond.  As in the experts' GEMVs the quants
// themselves are the (exact fp16) A operand, x enters as fp16 hi + lo columns (4
// rows fill the 8 columns of an MMA), and a 32-weight block is scaled in f32 after
// its sum.  The quants are made signed: as subnormals with their offset in the
// accumulator, the experts' form, they take 8 half-precision operations per
// 512 weights less (262144 x 2816 for one row 75 us instead of 83), but the
// tensor core aligns the subnormals' products to exponents 7 bits too large, and
// the result was off by up to 1.1e-6 of its norm instead of 1e-7.
//
// One CTA of 16 warps per SM stays resident.  It turns its columns of x into
// fragments in shared memory once, while the first weights are under way, and
// then its warps stream W: a warp owns pairs of 16-row strips (two strips share
// each fragment read) and 1 / ks of their columns, through a ring of bulk
// copies.  Where x is too wide for one SM's shared memory (or W has few rows) a
// cluster of cs CTAs splits the columns, so that each converts only its part of
// x; their sums meet in distributed shared memory.  The split (cs, ks) is the
// one with the least estimated time; sums are in a fixed order.
//
// Measured on a B200 (copy bandwidth 6.55 TB/s): 262144 x 2816 Q4_0 for one row 72
// us (416 MB, 88 %), 65536 x 2816 for 1, 4, 8, 16 rows 22.6, 24.8, 35, 54 us (floor
// 15.9), 6144 x 2816 for one row 6.3 us, of which 4 are launch, fragments and the
// meeting of the warps.
#include <algorithm>
#include <atomic>

#include "packed_tiles.cuh"

namespace moe {

constexpr int kLinWarps = 16;
constexpr int kLinMaxStages = 4;
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
__device__ __forceinline__ float ld_cluster(uint32_t addr, int rank) {
  uint32_t a;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
  return v;
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
// 512 bytes); a row times 2^ex has its largest |x| in [2^14, 2^15).
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
  uint32_t mx = 0;
  if (on)
#pragma unroll 4
    for (int b = part * 8 + (lane >> 2); b < real; b += wpr * 8) {
      float v[8];
      values(b, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = max(mx, __float_as_uint(fabsf(v[i])));
    }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if (lane == 0) smax[warp] = mx;
  if (tid < ROWS) ex[tid] = 0;
  for (int i = tid; i < G * rec_blocks * 32; i += kLinWarps * 32)
    reinterpret_cast<uint4*>(rec)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (!on) return;
  mx = 0;
  for (int i = 0; i < wpr; ++i) mx = max(mx, smax[row * wpr + i]);
  const int eb = (int)(mx >> 23);                // biased exponent; 255: Inf or NaN
  const int e = mx == 0 || eb == 255 ? 0 : 141 - max(eb, 1);
  const float f1 = pow2f(e / 2), f2 = pow2f(e - e / 2);
  if (part == 0 && lane == 0) ex[row] = e;
  const int cg = row / TOK;
  for (int b = part * 8 + (lane >> 2); b < real; b += wpr * 8) {
    uint32_t hi[4], lo[4];
    float v[8];
    values(b, v);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      // register slots i, i + 1 hold elements 0, 2 | 1, 3 of each four (Q4_0)
      const int p = QT == MOE_Q4_0 ? (i & 4) + ((i & 2) ? 1 : 0) : i;
      const int q = QT == MOE_Q4_0 ? p + 2 : i + 1;
      const float a = v[p] * f1 * f2, c = v[q] * f1 * f2;
      const __half2 h = __floats2half2_rn(a, c);
      const __half2 l = __floats2half2_rn(a - __low2float(h), c - __high2float(h));
      hi[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
      lo[i / 2] = *reinterpret_cast<const uint32_t*>(&l);
    }
    const int pair = (b % NBG) * TOK + row % TOK;
    uint8_t* r = rec + (size_t)(b * G + cg) * 512 + pair * 128 + t * 16;
    *reinterpret_cast<uint4*>(r) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4*>(r + 64) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
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
  float* const red = reinterpret_cast<float*>(rec + (size_t)tps * Cfg::kTileBytes);
  float* const part = red + (A.ks > 1 ? kLinWarps * NRED : 0);
  uint8_t* const ring =
      reinterpret_cast<uint8_t*>(part + (A.cs > 1 ? 2 * groups * NRED : 0)) + warp * A.nst * STAGE;
  uint64_t* const bars = bars_all + warp * kLinMaxStages;

  if (lane < A.nst) {
    mbar_init(&bars[lane], 1);
    fence_mbar_init();
  }
  if (tid == 0) *dead = 0;                       // seen by all after build_fragments
  __syncwarp();
  pdl_trigger();
  pdl_wait();

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
  for (int q = 0; q < A.nst && q < total; ++q) issue();
  build_fragments<QT, NBG, G>(A, rec, rec_blocks, ex, smax, row0, n, t0, t1);
  __syncthreads();

  // ---- stream
  int slot = 0;
  uint32_t phase = 0;
  // fragments of this warp's columns
  const uint8_t* const xl = rec + lane * 16 + (size_t)2 * (wt0 - t0) * G * 512;
  // value i (row g + 8 i) of strip s, column group cg in lane l
  auto put = [&](int p, int s, int cg, int i, int l, float y) {
    const int tok = TOK * cg + (l & 3), row = 32 * p + 16 * s + (l >> 2) + 8 * i;
    if ((l & 3) < TOK && tok < n && row < A.rows) {
      if (A.residual) y += A.residual[(int64_t)(row0 + tok) * A.rs + row];
      A.y[(int64_t)(row0 + tok) * A.ys + row] = y;
    }
  };
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
          if (*dead) v[s][cg][i] = __uint_as_float(0x7fffffffu);   // a wait ran out: NaN
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
              red[warp * NRED + ((s * G + cg) * 2 + i) * 32 + lane] = v[s][cg][i];
      asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(32 * A.ks) : "memory");
      if (kq == 0)
        for (int k = 1; k < A.ks; ++k)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int cg = 0; cg < G; ++cg)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                v[s][cg][i] += red[(warp + k) * NRED + ((s * G + cg) * 2 + i) * 32 + lane];
    }
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
            for (int i = 0; i < 2; ++i) put(p, s, cg, i, lane, v[s][cg][i]);
      }
    } else {
      // the CTAs' parts: every thread of the cluster adds up its places
      float* mine_p = part + (size_t)(r & 1) * groups * NRED;
      if (kq == 0)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int cg = 0; cg < G; ++cg)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              mine_p[group * NRED + ((s * G + cg) * 2 + i) * 32 + lane] = v[s][cg][i];
      cluster_sync();
      for (int e = rank * kLinWarps * 32 + tid; e < groups * NRED; e += A.cs * kLinWarps * 32) {
        const int pe = e / NRED * nclusters + cluster + r * pstep, k = e % NRED / 32;
        const uint32_t a = smem_u32(mine_p + e);
        float f[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) f[c] = c < A.cs ? ld_cluster(a, c) : 0.f;
        float y = f[0];
#pragma unroll
        for (int c = 1; c < 8; ++c) y += f[c];
        if (pe < A.pairs) put(pe, k / (2 * G), k / 2 % G, k % 2, e % 32, y);
      }
    }
  }
  // after a timeout the copies already issued are still waited for (bounded)
  if (*dead)
    for (int i = 0; i < A.nst; ++i) {
      mbar_wait(&bars[i], 0);
      mbar_wait(&bars[i], 1);
    }
  if (A.cs > 1) cluster_sync();                  // nobody reads this CTA's parts any more
}

// Tiles of a CTA's columns: an even number, so that a stage is two of them.
inline int linear_tps(int kt, int cs) { return ((kt + cs - 1) / cs + 1) / 2 * 2; }

// Shared memory of a split; nst ring stages take what is left.
template <int QT, int NBG, int G, int U>
static size_t linear_smem(int kt, int cs, int ks, int nst) {
  using Cfg = LinCfg<NBG, G>;
  const size_t nred = (size_t)Cfg::kRed * 4;
  return kLinHead + (size_t)linear_tps(kt, cs) * Cfg::kTileBytes + (ks > 1 ? kLinWarps * nred : 0) +
         (cs > 1 ? 2 * (kLinWarps / ks) * nred : 0) +
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
static int launch_linear(LinArgs& a, cudaStream_t s, bool& fits) {
  using Cfg = LinCfg<NBG, G>;
  auto kern = linear_kernel<QT, NBG, G, U>;
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  MOE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !((ready.load() >> dev) & 1)) {
    MOE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kLinSmem));
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  // The splits of a few sizes are remembered, for calls that repeat them.
  struct Plan { int dev = -1, kt, pairs, cs, ks, nst, clusters; };
  static thread_local Plan plans[16];
  Plan& plan = plans[(a.kt * 31 + a.pairs) & 15];
  if (plan.dev != dev || plan.kt != a.kt || plan.pairs != a.pairs)
    plan = {dev, a.kt, a.pairs, 0, 0, 0, 0};
  if (plan.nst == 0) {
    // Estimated time of a split, in the time all warps of an SM take for one tile
    // of two strips each (about 800 cycles of HBM): rounds x (tiles of a warp, and
    // the meetings of warps, 3, and of a cluster, 8), and the fragments of the
    // CTA's columns (28 cycles per group and tile).
    double best = 0;
    for (int cs = 1; cs <= 8; cs *= 2) {
      const int resident = resident_clusters((const void*)kern, cs, dev);
      for (int ks = 1; ks <= kLinWarps; ks *= 2) {
        if (linear_smem<QT, NBG, G, U>(a.kt, cs, ks, 2) > kLinSmem) continue;
        const int tps = linear_tps(a.kt, cs), wt = ((tps + ks - 1) / ks + 1) / 2 * 2;
        const int slots = resident * (kLinWarps / ks);
        const int rounds = (a.pairs + slots - 1) / slots;
        const double t = rounds * (wt * (1 + 0.25 * (G - 1)) + (ks > 1 ? 3 : 0) + (cs > 1 ? 8 : 0)) +
                         0.035 * G * tps;
        if (plan.cs == 0 || t < best) {
          best = t;
          plan.cs = cs;
          plan.ks = ks;
          plan.clusters = resident;
        }
      }
    }
    plan.nst = 2;
    while (plan.cs > 0 && plan.nst < kLinMaxStages &&
           linear_smem<QT, NBG, G, U>(a.kt, plan.cs, plan.ks, plan.nst + 1) <= kLinSmem)
      ++plan.nst;
  }
  fits = plan.cs > 0;
  if (!fits) return MOE_OK;
  a.cs = plan.cs;
  a.ks = plan.ks;
  a.nst = plan.nst;
  a.tps = linear_tps(a.kt, a.cs);
  const int per = kLinWarps / a.ks;                  // pairs of a cluster's round
  const int clusters = std::min(plan.clusters, a.pairs);
  a.rounds = (a.pairs + clusters * per - 1) / (clusters * per);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * a.cs), (unsigned)((a.T + Cfg::kRows - 1) / Cfg::kRows));
  cfg.blockDim = dim3(kLinWarps * 32);
  cfg.dynamicSmemBytes = linear_smem<QT, NBG, G, U>(a.kt, a.cs, a.ks, a.nst);
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
  MOE_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return MOE_OK;
}

// Rows of a pass: as many as T needs (1, 2, 4, 8 or 16), fewer where x is so wide
// that their fragments do not fit.  Up to 4 rows of 4-bit weights are bound by
// instructions, so four tiles are taken per wait where the ring fits (65536 x
// 2816: 1 row 25.7 -> 22.9 us, 4 rows 28.1 -> 24.9 us; 8 rows, nearer the MMAs'
// bound, 36.5 -> 37.4 us).
template <int QT>
static int launch_linear_qt(LinArgs& a, cudaStream_t s) {
  constexpr int U = QT == MOE_Q4_0 ? 4 : 2;
  bool fits = false;
  if (a.T > 8) MOE_CHECK((launch_linear<QT, 1, 4, 2>(a, s, fits)));
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
