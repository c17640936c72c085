// Activation quantisation with separate outputs: E4M3 codes and one scale per
// row and 128 columns (act_quant, inplace=False; npu_ops.py:73-104).
//
// The arithmetic is in fp8_quant.cuh.
//
// Bound: HBM, (bytes of x + 1) per element.  A half warp holds a block, eight
// columns per lane, so a lane loads 16 bytes (two loads for fp32) and stores
// 8; a warp has eight blocks in flight before the first reduction.  Rows that
// do not start on 16 bytes take one element per load, neighbours across the
// lanes.  Measured: 8192 x 4096 bf16 with E8M0 scales 17.2 us (5.9 TB/s, 91 %
// of the copy rate), 4095 x 2008 fp32 with fp32 scales 11.8 us
// (8.4 without the remainder of 0.875 x and the look at ties; half the blocks
// in flight, with fewer registers, took 12.0).
#include "capi_internal.h"
#include "common.cuh"
#include "fp8_quant.cuh"

#include <cuda_fp16.h>

namespace dsv4 {
namespace {

constexpr int QB = 128;          // columns per scale
constexpr int Q_STEPS = 4;       // blocks per half warp in flight
constexpr int Q_THREADS = 128;

template <int DT>
struct In;
template <>
struct In<DSV4_DT_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float f(T v) { return bf16_from_bits(v); }
};
template <>
struct In<DSV4_DT_FP16> {
  using T = __half;
  static __device__ __forceinline__ float f(T v) { return __half2float(v); }
};
template <>
struct In<DSV4_DT_FP32> {
  using T = float;
  static __device__ __forceinline__ float f(T v) { return v; }
};

// VEC: rows of x start on 16 bytes, rows of q on 8, and cols % 8 == 0.
template <int DT, int SC, bool VEC>
__global__ void __launch_bounds__(Q_THREADS)
    act_quant_fp8_kernel(const typename In<DT>::T* __restrict__ x, int64_t rows, int64_t cols, int64_t ldx,
                         uint8_t* __restrict__ q, int64_t ldq, void* __restrict__ scale) {
  using T = typename In<DT>::T;
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, half = lane >> 4, hl = lane & 15;
  const int64_t nb = (cols + QB - 1) / QB;
  const int64_t segs = (nb + 2 * Q_STEPS - 1) / (2 * Q_STEPS);
  const int64_t w = ((int64_t)blockIdx.x * Q_THREADS + threadIdx.x) >> 5;
  const int64_t row = w / segs;
  if (row >= rows) return;
  const int64_t b0 = (w - row * segs) * (2 * Q_STEPS) + half;
  const T* xr = x + row * ldx;
  uint8_t* qr = q + row * ldq;
  float v[Q_STEPS][8];
#pragma unroll
  for (int i = 0; i < Q_STEPS; ++i) {
    const int64_t c = (b0 + 2 * i) * QB + (VEC ? hl * 8 : hl);
    if constexpr (VEC) {
      uint4 raw[sizeof(T) / 2] = {};
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; ++j)
          raw[j] = __ldcg(reinterpret_cast<const uint4*>(xr + c) + j);
      }
      const T* e = reinterpret_cast<const T*>(raw);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = In<DT>::f(e[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = c + j * 16 < cols ? In<DT>::f(__ldcg(xr + c + j * 16)) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < Q_STEPS; ++i) {
    const float a = fp8_amax(v[i]);
    const int64_t b = b0 + 2 * i;
    uint2 o;
    if constexpr (SC == DSV4_SCALE_FP32) {
      o = fp8_codes_fp32<DT == DSV4_DT_FP32>(v[i], a);
      if (hl == 0 && b < nb) static_cast<float*>(scale)[row * nb + b] = fp8_scale_fp32(a);
    } else {
      const int e = scale_exp_448(a);
      o = fp8_codes_pow2(v[i], e);
      if (hl == 0 && b < nb) {
        if constexpr (SC == DSV4_SCALE_E8M0) static_cast<uint8_t*>(scale)[row * nb + b] = (uint8_t)(e + 127);
        else static_cast<float*>(scale)[row * nb + b] = pow2i(e);
      }
    }
    const int64_t c = b * QB + (VEC ? hl * 8 : hl);
    if constexpr (VEC) {
      if (c < cols) *reinterpret_cast<uint2*>(qr + c) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j * 16 < cols) qr[c + j * 16] = (uint8_t)((j < 4 ? o.x : o.y) >> (8 * (j & 3)));
    }
  }
}

template <int DT, int SC>
cudaError_t launch_quant(const void* x, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q, int64_t ldq, void* scale,
                         cudaStream_t st) {
  using T = typename In<DT>::T;
  const bool vec = cols % 8 == 0 && (uintptr_t)x % 16 == 0 && (ldx * (int64_t)sizeof(T)) % 16 == 0 &&
                   (uintptr_t)q % 8 == 0 && ldq % 8 == 0;
  const int64_t nb = (cols + QB - 1) / QB, segs = (nb + 2 * Q_STEPS - 1) / (2 * Q_STEPS);
  const int64_t warps = rows * segs, per = Q_THREADS / 32;
  const dim3 grid((unsigned)((warps + per - 1) / per));
  return launch_k(vec ? act_quant_fp8_kernel<DT, SC, true> : act_quant_fp8_kernel<DT, SC, false>, grid,
                  dim3(Q_THREADS), 0, st, pdl_enabled(), static_cast<const T*>(x), rows, cols, ldx, q, ldq, scale);
}

template <int DT>
cudaError_t launch_quant_s(int sc, const void* x, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q, int64_t ldq,
                           void* scale, cudaStream_t st) {
  if (sc == DSV4_SCALE_E8M0) return launch_quant<DT, DSV4_SCALE_E8M0>(x, rows, cols, ldx, q, ldq, scale, st);
  if (sc == DSV4_SCALE_FP32) return launch_quant<DT, DSV4_SCALE_FP32>(x, rows, cols, ldx, q, ldq, scale, st);
  return launch_quant<DT, DSV4_SCALE_FP32_POW2>(x, rows, cols, ldx, q, ldq, scale, st);
}

}  // namespace

int act_quant_fp8_launch(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q, int64_t ldq,
                         void* scale, int scale_type, cudaStream_t st) {
  cudaError_t e;
  if (x_dtype == DSV4_DT_BF16) e = launch_quant_s<DSV4_DT_BF16>(scale_type, x, rows, cols, ldx, q, ldq, scale, st);
  else if (x_dtype == DSV4_DT_FP16) e = launch_quant_s<DSV4_DT_FP16>(scale_type, x, rows, cols, ldx, q, ldq, scale, st);
  else e = launch_quant_s<DSV4_DT_FP32>(scale_type, x, rows, cols, ldx, q, ldq, scale, st);
  if (e != cudaSuccess) return fail(DSV4_ECUDA, std::string("act_quant_fp8: ") + cudaGetErrorString(e));
  return DSV4_OK;
}

}  // namespace dsv4

using namespace dsv4;

extern "C" int dsv4_act_quant_fp8(const void* x, int32_t x_dtype, int64_t rows, int64_t cols, int64_t ldx, uint8_t* q,
                                  int64_t ldq, void* scale, int32_t scale_type, void* stream) {
  DSV4_API_BEGIN
  DSV4_CHECK_ARG(x_dtype == DSV4_DT_BF16 || x_dtype == DSV4_DT_FP16 || x_dtype == DSV4_DT_FP32,
                 "x must be bf16, fp16 or fp32");
  DSV4_CHECK_ARG(scale_type == DSV4_SCALE_E8M0 || scale_type == DSV4_SCALE_FP32 || scale_type == DSV4_SCALE_FP32_POW2,
                 "unknown scale type");
  DSV4_CHECK_ARG(rows >= 0 && cols > 0, "rows must be >= 0 and cols > 0");
  DSV4_CHECK_ARG(ldx >= cols && ldq >= cols, "a row stride is smaller than the row");
  if (rows == 0) return DSV4_OK;
  DSV4_CHECK_ARG(x && q && scale, "null pointer");
  DSV4_CHECK_ARG((uintptr_t)x % (x_dtype == DSV4_DT_FP32 ? 4 : 2) == 0, "misaligned x");
  DSV4_CHECK_ARG(scale_type == DSV4_SCALE_E8M0 || (uintptr_t)scale % 4 == 0, "misaligned scale");
  const int64_t segs = ((cols + QB - 1) / QB + 2 * Q_STEPS - 1) / (2 * Q_STEPS);
  DSV4_CHECK_ARG(rows <= (INT64_C(1) << 32) / segs, "too many rows");
  DeviceScope dev;
  if (int rc = dev.enter(x)) return rc;
  if (int rc = act_quant_fp8_launch(x, x_dtype, rows, cols, ldx, q, ldq, scale, scale_type, (cudaStream_t)stream))
    return rc;
  DSV4_API_END
}
