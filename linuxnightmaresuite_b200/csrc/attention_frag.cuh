// What the attention kernels share: the cache as a tensor for TMA, operands split into
// 16-bit parts, and the mma.sync products with query heads as the 16 rows of M and keys as N.
#pragma once

#include <cuda.h>

#include "paged_cache.cuh"

namespace moe {

constexpr int kAttHeads = 8;          // query heads of a unit at most
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kPShift = 7.f;        // probabilities enter sums and products times 2^7
constexpr int kLine = 128;            // bytes of a row in one TMA box

// A cache as the rows of a tensor map: row page * page_units + head * head_units, boxes of
// 2^box_shift tokens.
struct CacheMap {
  int page_units, head_units, box_shift;
};
int make_cache_map(CUtensorMap* map, const moe_paged_cache& c, void* base, int keys, CacheMap* at);
int check_attention(const moe_paged_attention_args& r, moe_paged_cache& c);
int attention_from(const moe_paged_attention_args& r, int from, float2* stats = nullptr);

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// d = a b (+ d unless FIRST)
template <bool BF, bool FIRST>
__device__ __forceinline__ void mma_acc(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  const float c0 = FIRST ? 0.f : d[0], c1 = FIRST ? 0.f : d[1], c2 = FIRST ? 0.f : d[2],
              c3 = FIRST ? 0.f : d[3];
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
        "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// two adjacent values -> NP packed parts that add up to them (22 bits of fp16,
// 24 of bf16); the lower value sits in the lower half
template <bool BF, int NP>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&r)[NP]) {
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (BF) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      r[i] = *reinterpret_cast<const uint32_t*>(&h);
      x -= __low2float(h);
      y -= __high2float(h);
    } else {
      const __half2 h = __floats2half2_rn(x, y);
      r[i] = *reinterpret_cast<const uint32_t*>(&h);
      x -= __low2float(h);
      y -= __high2float(h);
    }
  }
}

// four e4m3 -> two fp16x2, exact
__device__ __forceinline__ void e4m3x4_f16x2(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
      " cvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

// A operand of one k16 step: one 16-row tile of {hi rows, lo rows}.  bf16 has a
// second tile {third part, zero} that goes into the same accumulators, unless a
// unit has at most four heads (PACK): then rows 4 to 7 hold the third parts, and
// lanes g and g + 4 add up their results.
template <bool BF, bool PACK> struct AFrag {
  static constexpr int kParts = BF ? 3 : 2;
  static constexpr bool kTwo = BF && !PACK;      // a second tile
  static constexpr int kRegs = kTwo ? 3 : 2;
  uint32_t lo[kRegs], hi[kRegs];      // k columns 2t, 2t+1 and 2t+8, 2t+9
  __device__ __forceinline__ static void parts(float x, float y, int g, uint32_t (&r)[kRegs]) {
    if (BF && PACK) {
      uint32_t all[3];
      split2<true, 3>(x, y, all);
      r[0] = g < 4 ? all[0] : all[2];
      r[1] = g < 4 ? all[1] : 0u;
    } else {
      split2<BF, kRegs>(x, y, r);
    }
  }
  __device__ __forceinline__ void set(float x0, float x1, float x2, float x3, int g) {
    parts(x0, x1, g, lo);
    parts(x2, x3, g, hi);
  }
  template <bool FIRST = false>
  __device__ __forceinline__ void mul(float (&d)[4], uint32_t b0, uint32_t b1) const {
    mma_acc<BF, FIRST>(d, lo[0], lo[1], hi[0], hi[1], b0, b1);
    if (kTwo) mma_acc<BF, false>(d, lo[kRegs - 1], 0u, hi[kRegs - 1], 0u, b0, b1);
  }
  // in shared memory: 16 bytes per lane, then for a second tile 8 more
  static constexpr int kBytes = 32 * 8 * kRegs;
  __device__ __forceinline__ void store(uint8_t* at, int lane) const {
    *reinterpret_cast<uint4*>(at + lane * 16) = make_uint4(lo[0], lo[1], hi[0], hi[1]);
    if (kTwo) *reinterpret_cast<uint2*>(at + 512 + lane * 8) =
        make_uint2(lo[kRegs - 1], hi[kRegs - 1]);
  }
  __device__ __forceinline__ void load(const uint8_t* at, int lane) {
    const uint4 v = *reinterpret_cast<const uint4*>(at + lane * 16);
    lo[0] = v.x;
    lo[1] = v.y;
    hi[0] = v.z;
    hi[1] = v.w;
    if (kTwo) {
      const uint2 w = *reinterpret_cast<const uint2*>(at + 512 + lane * 8);
      lo[kRegs - 1] = w.x;
      hi[kRegs - 1] = w.y;
    }
  }
};

}  // namespace moe
