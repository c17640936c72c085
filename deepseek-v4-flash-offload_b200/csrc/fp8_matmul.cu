// Product of E4M3 matrices with a scale per row and 128 of K on the left and
// per 128 x 128 block on the right:
//
//   y[m, n] = sum_kb as[m, kb] * bs(kb, n / 128) * sum_{k in kb} a[m, k] b(n, k)
//
// (dequant_fp8_weight followed by a linear layer, npu_ops.py:161-167, without
// the dequantised matrix).  b is [N, K] (trans_b) or [K, N]: the tensor cores
// read either major order from shared memory, so the gradient of a linear
// layer's input uses the same stored weight.
//
// Weights are the M side of the MMA (128 of N per CTA), tokens its N side (BN
// of M, 16 to 128), so that one token still feeds whole 128-row MMAs.
// E8M0 scales: tcgen05 kind::mxf8f6f4 applies them.  Its four scale bytes per
//   row (32 of K each) hold the scales of four consecutive 128-blocks instead,
//   and the four MMAs of a k-tile all name byte (kt % 4): one 4-byte word per
//   row and 512 of K, the bytes as they lie in memory.
// fp32 scales: kind::f8f6f4 into a ring of TMEM accumulators, one k-tile each;
//   the epilogue warps add as * bs times each partial sum to fp32 registers.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

namespace dsv4 {
namespace {

constexpr int F_BK = 128;              // k-tile = one scale block, one 128-byte swizzle row
constexpr int F_BM = 128;              // of N (weight rows) per CTA
constexpr int F_GROUP = 4;             // k-tiles per scale group
constexpr int F_SLOTS = 4;             // scale groups in flight
constexpr int F_EPI_WARP0 = 4;

// Set by a kernel whose bounded wait ran out; read by dsv4_fp8_status.
__device__ int g_fp8_status;

struct Fp8Params {
  const void* as;      // [M, kb] bytes or floats
  const void* bs;      // element (kb, nb) at kb * bs_k + nb * bs_n
  int64_t bs_k, bs_n;
  void* y;
  int64_t ldy, M, N;
  int kb;              // scale blocks along K = k-tiles
};

template <int BN, bool E8>
struct FCfg {
  static constexpr int A_BYTES = F_BM * F_BK;
  static constexpr int B_BYTES = BN * F_BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // two CTAs share an SM: their rings stay within half of its shared memory
  static constexpr int STAGES = BN == 128 ? 3 : (BN == 64 ? 4 : 5);
  static constexpr int SLOT_BYTES = E8 ? 1024 : F_GROUP * BN * 4;
  static constexpr int EPI_WARPS = BN == 128 ? 8 : 4;
  static constexpr int COLS = BN / (EPI_WARPS / 4);      // accumulator columns per epilogue warp
  static constexpr int THREADS = (F_EPI_WARP0 + EPI_WARPS) * 32;
  static constexpr int NACC = E8 ? 1 : (BN == 128 ? 2 : 4);
  static constexpr int SF_COL = BN;                      // E8M0: 8 columns of scales, twice
  static constexpr uint32_t TMEM_COLS = E8 ? (BN == 128 ? 256 : (BN == 64 ? 128 : (BN == 32 ? 64 : 32))) : NACC * BN;
  static constexpr int BARS = 2 * STAGES + 2 * F_SLOTS + 2 * NACC + 1;
  static constexpr int SMEM = STAGES * STAGE_BYTES + F_SLOTS * SLOT_BYTES + BARS * 8 + 16 + 1024;
};

__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor of kind::f8f6f4 with E4M3 A and B, fp32 D.
__host__ __device__ __forceinline__ uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | (((uint32_t)(n >> 3) & 63u) << 17) | (((uint32_t)(m >> 4) & 31u) << 24);
}
constexpr uint32_t IDESC_A_MN = 1u << 15;   // operand A stored along M (both kinds)

// Scale bytes / floats of four k-tiles from k-tile kt (past the end: byte 127
// = 1, float 0; their operand bytes are zero).
// Read past L1: the kernel just before may have written them.
__device__ __forceinline__ uint32_t sf_word(const uint8_t* p, int64_t stride, int kt, int kb) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < F_GROUP; ++i) w |= (kt + i < kb ? (uint32_t)__ldcg(p + (int64_t)i * stride) : 127u) << (8 * i);
  return w;
}

template <int BN, bool E8, bool A_MN>
__global__ void __launch_bounds__(FCfg<BN, E8>::THREADS, 1)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const Fp8Params p, const int out_f32) {
  using C = FCfg<BN, E8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + F_SLOTS * C::SLOT_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* sfull = empty + C::STAGES;
  uint64_t* sempty = sfull + F_SLOTS;
  uint64_t* accfull = sempty + F_SLOTS;
  uint64_t* accempty = accfull + C::NACC;
  uint64_t* drain = accempty + C::NACC;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  int* err = reinterpret_cast<int*>(tmem_holder + 1);   // this CTA's waits; copied to g_fp8_status at the end
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * F_BM;
  const int64_t m0 = (int64_t)blockIdx.y * BN;
  const int nkt = p.kb;
  const int ngr = (nkt + F_GROUP - 1) / F_GROUP;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < F_SLOTS; ++s) {
      mbar_init(&sfull[s], 1);
      mbar_init(&sempty[s], E8 ? 1 : C::EPI_WARPS);
    }
    for (int s = 0; s < C::NACC; ++s) {
      mbar_init(&accfull[s], 1);
      mbar_init(&accempty[s], C::EPI_WARPS);
    }
    mbar_init(drain, 1);
    *err = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmW);
    prefetch_tensormap(&tmX);
  }
  if (warp == 3) {
    tmem_alloc(tmem_holder, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  griddep_wait();
  griddep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------- producer
    if (lane == 0) {
      const uint64_t pol = policy_evict_normal();
      int issued = 0;
      for (int kt = 0; kt < nkt; ++kt) {
        const int s = kt % C::STAGES;
        if (kt >= C::STAGES && !mbar_wait(&empty[s], (uint32_t)(kt / C::STAGES - 1) & 1u, err)) break;
        uint8_t* st = smem + s * C::STAGE_BYTES;
        mbar_expect_tx(&full[s], C::STAGE_BYTES);
        if constexpr (A_MN) tma_load_2d(st, &tmW, &full[s], n0, kt * F_BK, pol);
        else tma_load_2d(st, &tmW, &full[s], kt * F_BK, n0, pol);
        tma_load_2d(st + C::A_BYTES, &tmX, &full[s], kt * F_BK, (int)m0, pol);
        mbar_arrive(&full[s]);
        ++issued;
      }
      // copies still in flight (after a wait that ran out) land before the CTA exits
      for (int c = issued - C::STAGES < 0 ? 0 : issued - C::STAGES; c < issued; ++c) {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(&full[c % C::STAGES], (uint32_t)(c / C::STAGES) & 1u) &&
               globaltimer_ns() - t0 < DSV4_WAIT_NS) {
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issuer
    if (lane == 0) {
      const uint32_t mn = A_MN ? IDESC_A_MN : 0u;
      constexpr uint32_t A_STEP = A_MN ? (32 * 128) >> 4 : 2u;   // 32 of K: 32 rows of 128 B, or 32 B of a row
      bool ok = true;
      for (int kt = 0; kt < nkt; ++kt) {
        const int s = kt % C::STAGES, gr = kt / F_GROUP, slot = gr % F_SLOTS;
        if (!(ok = mbar_wait(&full[s], (uint32_t)(kt / C::STAGES) & 1u, err))) break;
        const uint32_t aA = smem_u32(smem + s * C::STAGE_BYTES);
        const uint64_t dA = desc_sw128(aA), dB = desc_sw128(aA + C::A_BYTES);
        if constexpr (E8) {
          // tcgen05 operations of one thread run in issue order, so a copy
          // into columns that earlier MMAs read waits for them
          const uint32_t sfa = tmem + C::SF_COL + 8 * (gr & 1), sfb = sfa + 4;
          if (kt % F_GROUP == 0) {
            if (!(ok = mbar_wait(&sfull[slot], (uint32_t)(gr / F_SLOTS) & 1u, err))) break;
            tc_fence_after();
            const uint32_t sl = smem_u32(slots + slot * C::SLOT_BYTES);
            tc_cp_sf(sfa, desc_sf(sl));
            tc_cp_sf(sfb, desc_sf(sl + 512));
            tc_commit(&sempty[slot]);
          }
          tc_fence_after();
          const uint32_t id = kt % F_GROUP, sel = id << 30;
          const uint32_t idesc = idesc_mxf8f6f4(BN, false, id, true) | mn;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_mxf8f6f4(tmem, dA + A_STEP * j, dB + 2u * j, idesc, (kt | j) != 0 ? 1u : 0u, sfa | sel, sfb | sel);
          tc_commit(&empty[s]);
        } else {
          const int ab = kt % C::NACC;
          if (kt >= C::NACC && !(ok = mbar_wait(&accempty[ab], (uint32_t)(kt / C::NACC - 1) & 1u, err))) break;
          tc_fence_after();
          const uint32_t idesc = idesc_f8(F_BM, BN) | mn;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_f8(tmem + ab * BN, dA + A_STEP * j, dB + 2u * j, idesc, j != 0 ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(&accfull[ab]);
        }
      }
      if constexpr (E8) tc_commit(&accfull[0]);
      // the MMAs issued (also before a wait that ran out) complete before TMEM is freed
      tc_commit(drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < DSV4_WAIT_NS) {
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------------------------------------------------------- scales
    for (int gr = 0; gr < ngr; ++gr) {
      const int slot = gr % F_SLOTS, kt0 = gr * F_GROUP;
      uint8_t* sl = slots + slot * C::SLOT_BYTES;
      if constexpr (E8) {
        const uint8_t* bs = static_cast<const uint8_t*>(p.bs) + (int64_t)kt0 * p.bs_k + (n0 / F_BK) * p.bs_n;
        const uint32_t wa = sf_word(bs, p.bs_k, kt0, nkt);
        uint32_t wb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          wb[j] = (lane + 32 * j < BN && m < p.M)
                      ? sf_word(static_cast<const uint8_t*>(p.as) + m * nkt + kt0, 1, kt0, nkt)
                      : 0x7f7f7f7fu;
        }
        bool ok = true;
        if (gr >= F_SLOTS) ok = __all_sync(0xffffffffu, mbar_wait(&sempty[slot], (uint32_t)(gr / F_SLOTS - 1) & 1u, err));
        if (!ok) break;
        *reinterpret_cast<uint4*>(sl + lane * 16) = make_uint4(wa, wa, wa, wa);
        *reinterpret_cast<uint4*>(sl + 512 + lane * 16) = make_uint4(wb[0], wb[1], wb[2], wb[3]);
        fence_proxy_async_smem();   // read by tcgen05.cp
      } else {
        float sb[F_GROUP], v[F_GROUP][(BN + 31) / 32];
        const float* bs = static_cast<const float*>(p.bs) + (int64_t)kt0 * p.bs_k + (n0 / F_BK) * p.bs_n;
#pragma unroll
        for (int i = 0; i < F_GROUP; ++i) {
          sb[i] = kt0 + i < nkt ? __ldcg(bs + (int64_t)i * p.bs_k) : 0.f;
#pragma unroll
          for (int j = 0; j < (BN + 31) / 32; ++j) {
            const int64_t m = m0 + lane + 32 * j;
            v[i][j] = (lane + 32 * j < BN && m < p.M && kt0 + i < nkt)
                          ? __ldcg(static_cast<const float*>(p.as) + m * nkt + kt0 + i)
                          : 0.f;
          }
        }
        bool ok = true;
        if (gr >= F_SLOTS) ok = __all_sync(0xffffffffu, mbar_wait(&sempty[slot], (uint32_t)(gr / F_SLOTS - 1) & 1u, err));
        if (!ok) break;
        float* f = reinterpret_cast<float*>(sl);
#pragma unroll
        for (int i = 0; i < F_GROUP; ++i)
#pragma unroll
          for (int j = 0; j < (BN + 31) / 32; ++j)
            if (lane + 32 * j < BN) f[i * BN + lane + 32 * j] = v[i][j] * sb[i];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sfull[slot]);
    }
  } else if (warp >= F_EPI_WARP0) {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, c0 = ((warp - F_EPI_WARP0) >> 2) * C::COLS;
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0;
    float acc[C::COLS];
    bool ok = true;
    if constexpr (E8) {
      ok = __all_sync(0xffffffffu, mbar_wait(&accfull[0], 0, err) && read_status(err) == 0);
      tc_fence_after();
      if (ok) {
#pragma unroll
        for (int c = 0; c < C::COLS; c += 16) tmem_ld16(trow + c, acc + c);
        tc_wait_ld();
      }
    } else {
#pragma unroll
      for (int c = 0; c < C::COLS; ++c) acc[c] = 0.f;
      for (int kt = 0; kt < nkt; ++kt) {
        const int ab = kt % C::NACC, gr = kt / F_GROUP, slot = gr % F_SLOTS;
        const bool mine = (kt % F_GROUP != 0 || mbar_wait(&sfull[slot], (uint32_t)(gr / F_SLOTS) & 1u, err)) &&
                          mbar_wait(&accfull[ab], (uint32_t)(kt / C::NACC) & 1u, err);
        if (!(ok = __all_sync(0xffffffffu, mine))) break;
        tc_fence_after();
        const float* f = reinterpret_cast<const float*>(slots + slot * C::SLOT_BYTES) + (kt % F_GROUP) * BN + c0;
#pragma unroll
        for (int c = 0; c < C::COLS; c += 16) {
          float v[16];
          tmem_ld16(trow + ab * BN + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float4 s = *reinterpret_cast<const float4*>(f + c + j);
            acc[c + j] = fmaf(v[j], s.x, acc[c + j]);
            acc[c + j + 1] = fmaf(v[j + 1], s.y, acc[c + j + 1]);
            acc[c + j + 2] = fmaf(v[j + 2], s.z, acc[c + j + 2]);
            acc[c + j + 3] = fmaf(v[j + 3], s.w, acc[c + j + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&accempty[ab]);
          if (kt % F_GROUP == F_GROUP - 1 || kt == nkt - 1) mbar_arrive(&sempty[slot]);
        }
      }
    }
    const int64_t n = (int64_t)n0 + q * 32 + lane;
    if (ok && n < p.N) {
#pragma unroll
      for (int c = 0; c < C::COLS; ++c) {
        const int64_t m = m0 + c0 + c;
        if (m < p.M) {
          if (out_f32) static_cast<float*>(p.y)[m * p.ldy + n] = acc[c];
          else static_cast<uint16_t*>(p.y)[m * p.ldy + n] = bf16_bits(acc[c]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *err) set_status(&g_fp8_status, *err);
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int BN, bool E8, bool A_MN>
int launch_small(const CUtensorMap& tw, const CUtensorMap& tx, const Fp8Params& p, int out_f32, cudaStream_t st) {
  using C = FCfg<BN, E8>;
  auto k = fp8_matmul_kernel<BN, E8, A_MN>;
  DSV4_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
  const dim3 grid((unsigned)((p.N + F_BM - 1) / F_BM), (unsigned)((p.M + BN - 1) / BN));
  DSV4_CUDA_CHECK(launch_k(k, grid, dim3(C::THREADS), C::SMEM, st, pdl_enabled(), tw, tx, p, out_f32));
  return DSV4_OK;
}

template <int BN>
int launch_small_v(bool e8, bool a_mn, const CUtensorMap& tw, const CUtensorMap& tx, const Fp8Params& p, int out_f32,
                   cudaStream_t st) {
  if (e8) return a_mn ? launch_small<BN, true, true>(tw, tx, p, out_f32, st) : launch_small<BN, true, false>(tw, tx, p, out_f32, st);
  return a_mn ? launch_small<BN, false, true>(tw, tx, p, out_f32, st) : launch_small<BN, false, false>(tw, tx, p, out_f32, st);
}

}  // namespace

static int fp8_matmul_run(const uint8_t* a, int64_t lda, const void* as, const uint8_t* b, int64_t ldb, const void* bs,
                          int scale_type, bool trans_b, int64_t m, int64_t n, int64_t k, void* y, int64_t ldy,
                          int out_dtype, cudaStream_t st) {
  const int64_t kb = (k + F_BK - 1) / F_BK, nb = (n + F_BK - 1) / F_BK;
  Fp8Params p{as, bs, trans_b ? 1 : nb, trans_b ? kb : 1, y, ldy, m, n, (int)kb};
  const int bn = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128));
  CUtensorMap tw, tx;
  const uint64_t dw[2] = {(uint64_t)(trans_b ? k : n), (uint64_t)(trans_b ? n : k)}, sw[1] = {(uint64_t)ldb};
  const uint32_t bw[2] = {128, 128};
  if (int rc = make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)b, dw, sw, bw, "fp8_matmul b")) return rc;
  const uint64_t dx[2] = {(uint64_t)k, (uint64_t)m}, sx[1] = {(uint64_t)lda};
  const uint32_t bx[2] = {128, (uint32_t)bn};
  if (int rc = make_map(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)a, dx, sx, bx, "fp8_matmul a")) return rc;
  const bool e8 = scale_type == DSV4_SCALE_E8M0;
  const int f32 = out_dtype == DSV4_DT_FP32;
  switch (bn) {
    case 16: return launch_small_v<16>(e8, !trans_b, tw, tx, p, f32, st);
    case 32: return launch_small_v<32>(e8, !trans_b, tw, tx, p, f32, st);
    case 64: return launch_small_v<64>(e8, !trans_b, tw, tx, p, f32, st);
    default: return launch_small_v<128>(e8, !trans_b, tw, tx, p, f32, st);
  }
}

}  // namespace dsv4

using namespace dsv4;

extern "C" int dsv4_fp8_matmul(const uint8_t* a, int64_t lda, const void* a_scale, const uint8_t* b, int64_t ldb,
                               const void* b_scale, int32_t scale_type, int32_t trans_b, int64_t m, int64_t n,
                               int64_t k, void* y, int64_t ldy, int32_t out_dtype, void* stream) {
  DSV4_API_BEGIN
  DSV4_CHECK_ARG(scale_type == DSV4_SCALE_E8M0 || scale_type == DSV4_SCALE_FP32, "scales must be E8M0 or fp32");
  DSV4_CHECK_ARG(out_dtype == DSV4_DT_BF16 || out_dtype == DSV4_DT_FP32, "the output is bf16 or fp32");
  DSV4_CHECK_ARG(m >= 0 && n >= 0 && k > 0, "m and n must be >= 0 and k > 0");
  DSV4_CHECK_ARG(m <= 65535LL * 16 && n <= 0x7fffff00 && k <= 0x7fffff00, "a size is too large");
  DSV4_CHECK_ARG(lda >= k && ldb >= (trans_b ? k : n) && ldy >= n, "a row stride is smaller than the row");
  if (m == 0 || n == 0) return DSV4_OK;
  DSV4_CHECK_ARG(a && a_scale && b && b_scale && y, "null pointer");
  DSV4_CHECK_ARG((uintptr_t)a % 16 == 0 && lda % 16 == 0 && (uintptr_t)b % 16 == 0 && ldb % 16 == 0,
                 "a and b must start on 16 bytes, with row strides a multiple of 16");
  DSV4_CHECK_ARG((uintptr_t)y % (out_dtype == DSV4_DT_FP32 ? 4 : 2) == 0, "misaligned output");
  DSV4_CHECK_ARG(scale_type == DSV4_SCALE_E8M0 || ((uintptr_t)a_scale % 4 == 0 && (uintptr_t)b_scale % 4 == 0),
                 "misaligned scales");
  DeviceScope dev;
  if (int rc = dev.enter(a)) return rc;
  if (int rc = fp8_matmul_run(a, lda, a_scale, b, ldb, b_scale, scale_type, trans_b != 0, m, n, k, y, ldy, out_dtype,
                              (cudaStream_t)stream))
    return rc;
  DSV4_API_END
}

extern "C" int dsv4_fp8_status(int32_t device, void* stream) {
  DSV4_API_BEGIN
  int prev = -1, word = 0;
  DSV4_CUDA_CHECK(cudaGetDevice(&prev));
  DSV4_CUDA_CHECK(cudaSetDevice(device));
  cudaError_t e = cudaMemcpyFromSymbolAsync(&word, g_fp8_status, sizeof(int), 0, cudaMemcpyDeviceToHost,
                                            (cudaStream_t)stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
  if (e == cudaSuccess && word) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_fp8_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize((cudaStream_t)stream);
  }
  cudaSetDevice(prev);
  DSV4_CUDA_CHECK(e);
  if (word) return fail(word, "fp8_matmul: a device-side wait ran out");
  DSV4_API_END
}
