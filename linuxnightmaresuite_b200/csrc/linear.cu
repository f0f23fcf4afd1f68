// y = W x (+ residual) for a few rows, W in packed Q4_0 / Q8_0 tiles.
//
// First form: one warp per (row of W, row of x), decoding its weights from the
// packed tiles.
#include "moe_common.cuh"

namespace moe {

struct LinArgs {
  const uint8_t* w;
  const float *x, *residual;
  float* y;
  int64_t xs, rs, ys;
  int rows, cols, T;
};

template <int QT>
__global__ void __launch_bounds__(256) linear_kernel(const LinArgs A) {
  using Tr = QTraits<QT>;
  constexpr int SL = Tr::kLaneBytes / 4;
  pdl_trigger();
  pdl_wait();
  const int64_t unit = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (unit >= (int64_t)A.rows * A.T) return;
  const int row = (int)(unit % A.rows), t = (int)(unit / A.rows);
  const int kt = (A.cols + 63) / 64, g = row & 7, half = (row >> 3) & 1;
  float acc = 0.f;
  for (int b = 0; b < A.cols / 32; ++b) {
    const uint8_t* tile = A.w + ((int64_t)(row >> 4) * kt + (b >> 1)) * Tr::kTileBytes;
    const int sub = half * 2 + (b & 1);
    const float d =
        __half2float(*reinterpret_cast<const __half*>(tile + Tr::kTileQuant + 8 * g + 2 * sub));
    const int i = QT == MOE_Q4_0 ? lane & 15 : lane;
    const uint8_t byte = tile[(4 * g + i / SL) * Tr::kLaneBytes + sub * SL + i % SL];
    const int v = QT == MOE_Q4_0 ? (lane < 16 ? byte & 15 : byte >> 4) - 8 : (int)(int8_t)byte;
    acc = fmaf(d * (float)v, A.x[t * A.xs + 32 * b + lane], acc);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0) {
    if (A.residual) acc += A.residual[t * A.rs + row];
    A.y[t * A.ys + row] = acc;
  }
}

}  // namespace moe

extern "C" int moe_linear(const uint8_t* w, int qtype, int rows, int cols, const float* x,
                          int64_t x_stride, int T, const float* residual, int64_t residual_stride,
                          float* y, int64_t y_stride, moe_stream_t stream) {
  MOE_REQUIRE(moe::qtype_ok(qtype), MOE_ERR_UNSUPPORTED, "quant type %d not supported", qtype);
  MOE_REQUIRE(rows > 0 && cols > 0 && T >= 0, MOE_ERR_INVALID, "bad shape");
  MOE_REQUIRE(cols % 32 == 0, MOE_ERR_UNSUPPORTED, "cols %d is not a multiple of 32", cols);
  if (T == 0) return MOE_OK;
  MOE_REQUIRE(w && x && y, MOE_ERR_INVALID, "null pointer");
  MOE_REQUIRE((uintptr_t)w % 16 == 0, MOE_ERR_INVALID, "w must be 16-byte aligned");
  moe::LinArgs a = {w, x, residual, y, x_stride, residual_stride, y_stride, rows, cols, T};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t units = (int64_t)rows * T;
  {
    ::moe::ProfScope _prof(MOE_K_LINEAR, s);
    auto kern = qtype == MOE_Q4_0 ? moe::linear_kernel<MOE_Q4_0> : moe::linear_kernel<MOE_Q8_0>;
    MOE_CUDA(moe::launch_pdl(kern, dim3((unsigned)((units + 7) / 8)), dim3(256), 0, s, a));
  }
  return moe::check_launch("linear");
}
