// Packed weight tiles as MMA operands, shared by the mma.sync GEMVs (experts.cu,
// linear.cu): a tile's fragments from shared memory, the dequantisers, one
// 32-weight block's product.
#pragma once

#include "moe_common.cuh"

namespace moe {

constexpr float kSubUnit = 16777216.0f;   // 2^24: one fp16 subnormal step
// Activation block record in shared memory: 512 B of fragments, then the
// offset corrections as one f32x4 accumulator quad per lane column t
// ({C[2t], C[2t+1], C[2t], C[2t+1]}), then 16 B of padding so that records of
// consecutive blocks start on different banks.
constexpr int kXRec = 592;

// quant offset removed by the subnormal dequantisation
template <int QT>
__host__ __device__ constexpr float quant_offset() { return QT == MOE_Q4_0 ? 8.f : 128.f; }
__device__ __forceinline__ float half_lo(uint32_t v) {
  return __half2float(__ushort_as_half((unsigned short)(v & 0xFFFFu)));
}
__device__ __forceinline__ float half_hi(uint32_t v) {
  return __half2float(__ushort_as_half((unsigned short)(v >> 16)));
}

// element of a 32-block held at register slot i (0..7) of lane-column t
template <int QT>
__device__ __forceinline__ constexpr int frag_elem_c(int t, int i) {
  return QT == MOE_Q4_0 ? ((i < 4 ? 0 : 16) + 4 * t + ((i & 3) == 1 ? 2 : ((i & 3) == 2 ? 1 : (i & 3))))
                        : 8 * t + i;
}
// inverse: element e -> (t, i)
template <int QT>
__device__ __forceinline__ void frag_pos(int e, int& t, int& i) {
  if (QT == MOE_Q4_0) {
    int hi = e >= 16;
    int r = e & 15;
    t = r >> 2;
    int m = r & 3;                       // 0,1,2,3 -> slot 0,2,1,3
    i = (hi ? 4 : 0) + (m == 1 ? 2 : (m == 2 ? 1 : m));
  } else {
    t = e >> 3;
    i = e & 7;
  }
}

// ---------------------------------------------------------------------------
// tile fragments
// ---------------------------------------------------------------------------
template <int QT>
struct TileRegs {
  uint4 q[QT == MOE_Q4_0 ? 1 : 2];
  uint2 sc;
};

// fragment registers of one staged tile (shared memory, lane-contiguous)
template <int QT>
__device__ __forceinline__ void lds_quants(TileRegs<QT>& r, const uint8_t* tile, int lane) {
  const uint8_t* qp = tile + lane * QTraits<QT>::kLaneBytes;
  r.q[0] = *reinterpret_cast<const uint4*>(qp);
  if (QT == MOE_Q8_0) r.q[QT == MOE_Q4_0 ? 0 : 1] = *reinterpret_cast<const uint4*>(qp + 16);
}
template <int QT>
__device__ __forceinline__ void lds_tile(TileRegs<QT>& r, const uint8_t* tile, int lane) {
  using Tr = QTraits<QT>;
  lds_quants<QT>(r, tile, lane);
  r.sc = *reinterpret_cast<const uint2*>(tile + Tr::kTileQuant + (lane >> 2) * 8);
}

// Q4_0 quant word -> four fp16x2 subnormals: low nibbles n * 2^-24, high
// nibbles 16 n * 2^-24 (paired with activations stored / 16).
__device__ __forceinline__ void dequant_q4_sub(uint32_t w, uint32_t& lo01, uint32_t& lo23,
                                               uint32_t& hi01, uint32_t& hi23) {
  const uint32_t w8 = w >> 8;
  lo01 = w & 0x000F000Fu;
  lo23 = w8 & 0x000F000Fu;
  hi01 = w & 0x00F000F0u;
  hi23 = w8 & 0x00F000F0u;
}

// Q8_0 quant word -> two fp16x2 subnormals (q + 128) * 2^-24.
__device__ __forceinline__ void dequant_q8_sub(uint32_t w, uint32_t& h01, uint32_t& h23) {
  const uint32_t u = w ^ 0x80808080u;
  h01 = prmt(u, 0u, 0x4140u);
  h23 = prmt(u, 0u, 0x4342u);
}

// A fragments of both k16 steps for block b (rows g and g+8).
// SUB: subnormal quants (offset handled by the accumulator's initial value);
// otherwise exact signed fp16 integers.
template <int QT, bool SUB>
__device__ __forceinline__ void tile_quants(const TileRegs<QT>& r, int b, uint32_t (&a0)[4],
                                            uint32_t (&a1)[4]) {
  if (QT == MOE_Q4_0) {
    uint32_t wg = b ? r.q[0].y : r.q[0].x;
    uint32_t w8 = b ? r.q[0].w : r.q[0].z;
    uint32_t l01, l23, h01, h23, m01, m23, n01, n23;
    if (SUB) {
      dequant_q4_sub(wg, l01, l23, h01, h23);
      dequant_q4_sub(w8, m01, m23, n01, n23);
    } else {
      dequant_q4(wg, l01, l23, h01, h23);
      dequant_q4(w8, m01, m23, n01, n23);
    }
    a0[0] = l01; a0[1] = m01; a0[2] = l23; a0[3] = m23;
    a1[0] = h01; a1[1] = n01; a1[2] = h23; a1[3] = n23;
  } else {
    const uint4& qa = r.q[0];
    const uint4& qb = r.q[QT == MOE_Q4_0 ? 0 : 1];
    uint32_t g0 = b ? qa.z : qa.x, g1 = b ? qa.w : qa.y;
    uint32_t e0 = b ? qb.z : qb.x, e1 = b ? qb.w : qb.y;
    uint32_t x01, x23, y01, y23;
    if (SUB) {
      dequant_q8_sub(g0, x01, x23);
      dequant_q8_sub(e0, y01, y23);
    } else {
      dequant_q8(g0, x01, x23);
      dequant_q8(e0, y01, y23);
    }
    a0[0] = x01; a0[1] = y01; a0[2] = x23; a0[3] = y23;
    if (SUB) {
      dequant_q8_sub(g1, x01, x23);
      dequant_q8_sub(e1, y01, y23);
    } else {
      dequant_q8(g1, x01, x23);
      dequant_q8(e1, y01, y23);
    }
    a1[0] = x01; a1[1] = y01; a1[2] = x23; a1[3] = y23;
  }
}

// The same with the block's scales.
template <int QT, bool SUB>
__device__ __forceinline__ void tile_afrags(const TileRegs<QT>& r, int b, uint32_t (&a0)[4],
                                            uint32_t (&a1)[4], float2& dg, float2& dg8) {
  tile_quants<QT, SUB>(r, b, a0, a1);
  const float s0 = b ? half_hi(r.sc.x) : half_lo(r.sc.x);
  const float s8 = b ? half_hi(r.sc.y) : half_lo(r.sc.y);
  dg = make_float2(s0, s0);
  dg8 = make_float2(s8, s8);
}

// One 32-weight block: two k16 MMAs into an accumulator that starts at c0
// (zero, or the offset corrections of the lane's two columns for rows g and
// g+8), then acc += scale * block (packed f32x2 FMA).  acc[0]: row g,
// acc[1]: row g+8.
__device__ __forceinline__ void block_mma(float2 (&acc)[2], const uint32_t (&a0)[4],
                                          const uint32_t (&a1)[4], uint4 xf, float4 c0, float2 dg,
                                          float2 dg8) {
  const float init[4] = {c0.x, c0.y, c0.z, c0.w};
  float tmp[4];
  mma_16816(tmp, a0[0], a0[1], a0[2], a0[3], xf.x, xf.y, init);
  mma_16816(tmp, a1[0], a1[1], a1[2], a1[3], xf.z, xf.w, tmp);
  acc[0] = __ffma2_rn(dg, make_float2(tmp[0], tmp[1]), acc[0]);
  acc[1] = __ffma2_rn(dg8, make_float2(tmp[2], tmp[3]), acc[1]);
}

}  // namespace moe
