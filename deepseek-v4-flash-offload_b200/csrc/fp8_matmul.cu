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

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0u;
}
// Bounded wait on a barrier that CTAs of the cluster may arrive on.  The clock
// is read once in 1024 tries, since reading %globaltimer costs more than the
// k-tile a role waits for.  False once a wait of this CTA has run out.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, int* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    if (i % 64 == 0 && read_status(status) == DSV4_ETIMEOUT) return false;
    if (i % 1024 == 0) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > DSV4_WAIT_NS) {
        set_status(status, DSV4_ETIMEOUT);
        return false;
      }
    }
  }
}

// bar_wait of a whole warp: every lane gets the same answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, status));
}
// One lane of a converged warp, always the same one.  The roles that issue TMA
// and tcgen05 operations run warp-uniformly and elect a lane for the issue:
// their descriptors then stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(p));
  return p != 0u;
}

struct Fp8Params {
  const void* as;      // [M, kb] bytes or floats
  const void* bs;      // element (kb, nb) at kb * bs_k + nb * bs_n
  int64_t bs_k, bs_n;
  void* y;
  int64_t ldy, M, N;
  int kb;              // scale blocks along K = k-tiles
  int vec;             // access width of a row of `as` (scale_vec)
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

// Scales of F_CHUNK k-tiles at a time.  Rows of `as` are loaded with the widest
// access that their start allows, and the loads of a chunk are all in flight
// together (one byte-wise load per k-tile kept the tensor cores waiting: 0.8 us
// a k-tile instead of 0.3).  Read past L1: the kernel just before may have
// written them.  Past the end of K: byte 127 (= 1) or float 0; the operand
// bytes there are zero.
constexpr int F_CHUNK = 16;
// Access width of the rows of `as`, in elements: 16, 4 or 1 bytes, 4 or 1 floats.
__host__ __device__ __forceinline__ int scale_vec(const void* as, int kb, bool e8) {
  if (!e8) return kb % 4 == 0 && (uintptr_t)as % 16 == 0 ? 4 : 1;
  return kb % 16 == 0 && (uintptr_t)as % 16 == 0 ? 16 : (kb % 4 == 0 && (uintptr_t)as % 4 == 0 ? 4 : 1);
}
// Words w[g] = bytes of k-tiles kt + 4 g ..+ 3 of the row at p.
__device__ __forceinline__ void sf_row(const uint8_t* p, int kt, int kb, int vec, bool in, uint32_t w[4]) {
  if (in && vec == 16) {   // kb % 16 == 0: a chunk never runs past the end
    const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p + kt));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    return;
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    w[g] = 0x7f7f7f7fu;
    if (!in) continue;
    if (vec == 4) {
      if (kt + 4 * g < kb) w[g] = __ldcg(reinterpret_cast<const uint32_t*>(p + kt + 4 * g));
    } else {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = kt + 4 * g + i < kb ? (uint32_t)__ldcg(p + kt + 4 * g + i) : 127u;
      w[g] = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
    }
  }
}
// The byte of one of 32 k-tiles from kt, a lane each (a block column of bs).
__device__ __forceinline__ uint32_t sf_lane(const uint8_t* p, int64_t stride, int kt, int kb, bool in) {
  return in && kt < kb ? (uint32_t)__ldcg(p + (int64_t)kt * stride) : 127u;
}
// Word of the four k-tiles whose bytes lanes l0 .. l0 + 3 hold.
__device__ __forceinline__ uint32_t sf_gather(uint32_t b, int l0) {
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) w |= __shfl_sync(0xffffffffu, b, l0 + i) << (8 * i);
  return w;
}
// f[i] = float of k-tile kt + i of the row at p, N a multiple of 4.
template <int N>
__device__ __forceinline__ void scale_row(const float* p, int kt, int kb, int vec, bool in, float f[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    if (vec == 4) {
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && kt + i < kb) v = __ldcg(reinterpret_cast<const float4*>(p + kt + i));
      f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[i + j] = in && kt + i + j < kb ? __ldcg(p + kt + i + j) : 0.f;
    }
  }
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
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp-uniform
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
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);
  griddep_wait();
  griddep_launch();

  if (warp == 0) {
    // ------------------------------------------------------------- producer
    const uint64_t pol = policy_evict_normal();
    int issued = 0;
    for (int kt = 0; kt < nkt; ++kt) {
      const int s = kt % C::STAGES;
      if (kt >= C::STAGES && !warp_wait(&empty[s], (uint32_t)(kt / C::STAGES - 1) & 1u, err)) break;
      uint8_t* st = smem + s * C::STAGE_BYTES;
      if (elect_one()) {
        mbar_expect_tx(&full[s], C::STAGE_BYTES);
        if constexpr (A_MN) tma_load_2d(st, &tmW, &full[s], n0, kt * F_BK, pol);
        else tma_load_2d(st, &tmW, &full[s], kt * F_BK, n0, pol);
        tma_load_2d(st + C::A_BYTES, &tmX, &full[s], kt * F_BK, (int)m0, pol);
        mbar_arrive(&full[s]);
      }
      __syncwarp();
      ++issued;
    }
    // copies still in flight (after a wait that ran out) land before the CTA exits
    for (int c = issued - C::STAGES < 0 ? 0 : issued - C::STAGES; c < issued; ++c) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&full[c % C::STAGES], (uint32_t)(c / C::STAGES) & 1u) &&
             globaltimer_ns() - t0 < DSV4_WAIT_NS) {
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issuer
    const uint32_t mn = A_MN ? IDESC_A_MN : 0u;
    constexpr uint32_t A_STEP = A_MN ? (32 * 128) >> 4 : 2u;   // 32 of K: 32 rows of 128 B, or 32 B of a row
    for (int kt = 0; kt < nkt; ++kt) {
      const int s = kt % C::STAGES, gr = kt / F_GROUP, slot = gr % F_SLOTS;
      if (!warp_wait(&full[s], (uint32_t)(kt / C::STAGES) & 1u, err)) break;
      const uint32_t aA = smem_u32(smem + s * C::STAGE_BYTES);
      const uint64_t dA = desc_sw128(aA), dB = desc_sw128(aA + C::A_BYTES);
      if constexpr (E8) {
        // tcgen05 operations of one thread run in issue order, so a copy
        // into columns that earlier MMAs read waits for them
        const uint32_t sfa = tmem + C::SF_COL + 8 * (gr & 1), sfb = sfa + 4;
        const bool fresh = kt % F_GROUP == 0;
        if (fresh && !warp_wait(&sfull[slot], (uint32_t)(gr / F_SLOTS) & 1u, err)) break;
        tc_fence_after();
        const uint32_t id = kt % F_GROUP, sel = id << 30;
        const uint32_t idesc = idesc_mxf8f6f4(BN, false, id, true) | mn;
        if (elect_one()) {
          if (fresh) {
            const uint32_t sl = smem_u32(slots + slot * C::SLOT_BYTES);
            tc_cp_sf(sfa, desc_sf(sl));
            tc_cp_sf(sfb, desc_sf(sl + 512));
            tc_commit(&sempty[slot]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_mxf8f6f4(tmem, dA + A_STEP * j, dB + 2u * j, idesc, (kt | j) != 0 ? 1u : 0u, sfa | sel, sfb | sel);
          tc_commit(&empty[s]);
        }
      } else {
        const int ab = kt % C::NACC;
        if (kt >= C::NACC && !warp_wait(&accempty[ab], (uint32_t)(kt / C::NACC - 1) & 1u, err)) break;
        tc_fence_after();
        const uint32_t idesc = idesc_f8(F_BM, BN) | mn;
        if (elect_one()) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            tc_mma_f8(tmem + ab * BN, dA + A_STEP * j, dB + 2u * j, idesc, j != 0 ? 1u : 0u);
          tc_commit(&empty[s]);
          tc_commit(&accfull[ab]);
        }
      }
      __syncwarp();
    }
    if (elect_one()) {
      if constexpr (E8) tc_commit(&accfull[0]);
      tc_commit(drain);
    }
    __syncwarp();
    // the MMAs issued (also before a wait that ran out) complete before TMEM is freed
    const uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < DSV4_WAIT_NS) {
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---------------------------------------------------------------- scales
    constexpr int ROWS = (BN + 31) / 32;   // token rows per lane
    if constexpr (E8) {
      const uint8_t* bs = static_cast<const uint8_t*>(p.bs) + (int64_t)(n0 / F_BK) * p.bs_n;
      uint32_t cur[ROWS][4], nxt[ROWS][4], wbyte = 0;
      auto load = [&](int kt, uint32_t (&w)[ROWS][4]) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          const bool in = lane + 32 * j < BN && m < p.M;
          sf_row(static_cast<const uint8_t*>(p.as) + (in ? m * nkt : 0), kt, nkt, p.vec, in, w[j]);
        }
      };
      load(0, nxt);
      bool ok = true;
      for (int gr = 0; gr < ngr && ok; gr += 4) {
        if (gr % 8 == 0) wbyte = sf_lane(bs, p.bs_k, gr * F_GROUP + lane, nkt, true);
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) cur[j][g] = nxt[j][g];
        if (gr + 4 < ngr) load((gr + 4) * F_GROUP, nxt);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (gr + g >= ngr) break;
          const int slot = (gr + g) % F_SLOTS;
          uint8_t* sl = slots + slot * C::SLOT_BYTES;
          const uint32_t wa = sf_gather(wbyte, (gr + g) % 8 * 4);
          uint32_t wb[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) wb[j] = j < ROWS ? cur[j < ROWS ? j : 0][g] : 0x7f7f7f7fu;
          if (gr + g >= F_SLOTS && !(ok = warp_wait(&sempty[slot], (uint32_t)((gr + g) / F_SLOTS - 1) & 1u, err))) break;
          *reinterpret_cast<uint4*>(sl + lane * 16) = make_uint4(wa, wa, wa, wa);
          *reinterpret_cast<uint4*>(sl + 512 + lane * 16) = make_uint4(wb[0], wb[1], wb[2], wb[3]);
          fence_proxy_async_smem();   // read by tcgen05.cp
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[slot]);
        }
      }
    } else {
      const float* bs = static_cast<const float*>(p.bs) + (int64_t)(n0 / F_BK) * p.bs_n;
      float cur[ROWS][F_GROUP], nxt[ROWS][F_GROUP], sb = 0.f;
      auto load = [&](int kt, float (&f)[ROWS][F_GROUP]) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          const bool in = lane + 32 * j < BN && m < p.M;
          scale_row<F_GROUP>(static_cast<const float*>(p.as) + (in ? m * nkt : 0), kt, nkt, p.vec, in, f[j]);
        }
      };
      load(0, nxt);
      for (int gr = 0; gr < ngr; ++gr) {
        const int slot = gr % F_SLOTS, kt0 = gr * F_GROUP;
        if (gr % 8 == 0) sb = kt0 + lane < nkt ? __ldcg(bs + (int64_t)(kt0 + lane) * p.bs_k) : 0.f;
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
#pragma unroll
          for (int i = 0; i < F_GROUP; ++i) cur[j][i] = nxt[j][i];
        if (gr + 1 < ngr) load(kt0 + F_GROUP, nxt);
        if (gr >= F_SLOTS && !warp_wait(&sempty[slot], (uint32_t)(gr / F_SLOTS - 1) & 1u, err)) break;
        float* f = reinterpret_cast<float*>(slots + slot * C::SLOT_BYTES);
#pragma unroll
        for (int i = 0; i < F_GROUP; ++i) {
          const float s = __shfl_sync(0xffffffffu, sb, gr % 8 * 4 + i);
#pragma unroll
          for (int j = 0; j < ROWS; ++j)
            if (lane + 32 * j < BN) f[i * BN + lane + 32 * j] = cur[j][i] * s;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfull[slot]);
      }
    }
  } else if (warp >= F_EPI_WARP0) {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, c0 = ((warp - F_EPI_WARP0) >> 2) * C::COLS;
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0;
    float acc[C::COLS];
    bool ok = true;
    if constexpr (E8) {
      ok = __all_sync(0xffffffffu, bar_wait(&accfull[0], 0, err) && read_status(err) == 0);
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
        const bool mine = (kt % F_GROUP != 0 || bar_wait(&sfull[slot], (uint32_t)(gr / F_SLOTS) & 1u, err)) &&
                          bar_wait(&accfull[ab], (uint32_t)(kt / C::NACC) & 1u, err);
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


// ---------------------------------------------------------------------------
// Large products: CTA pairs.  Tokens are the M side (128 rows per CTA, 256 per
// pair), weights the N side (256, half of them in each CTA's shared memory):
// tcgen05.mma.cta_group::2 reads both halves, so a CTA loads 32 KB per k-tile
// for 128 x 256 x 128 products and the pair's tile has half the operand
// traffic of two separate 128 x 256 tiles.  Persistent: one pair per two SMs
// walks the tiles, with the ring running ahead into the next tile.
//   warp 0: TMA producer (each CTA its own halves, into the leader's barrier)
//   warp 1: MMA issuer (leader CTA only)
//   warp 2: E8M0 scale words (tokens' rows of this CTA, the weights' blocks)
//   warps 4-11: epilogue, 32 rows x 128 columns each
// E8M0: one 256-column accumulator, released as soon as the epilogue has it in
// registers.  fp32 scales: two accumulators, a k-tile each; an epilogue thread
// holds one row of one 128-block, so a partial sum takes one multiply-add.
// ---------------------------------------------------------------------------
constexpr int L_TM = 256, L_TN = 256;
constexpr int L_STAGES = 6;
constexpr int L_STAGE_BYTES = 2 * 128 * F_BK;
constexpr int L_SLOT_BYTES = 3 * 512;            // scale atoms: 128 rows of a, two blocks of b
constexpr int L_SF_COL = 256;                    // 12 columns of scales, twice
constexpr int L_EPI_WARPS = 8;
constexpr int L_THREADS = (F_EPI_WARP0 + L_EPI_WARPS) * 32;
constexpr int L_RASTER = 8;                      // m-tiles walked together: their operands meet in L2
constexpr int L_SMEM = L_STAGES * L_STAGE_BYTES + F_SLOTS * L_SLOT_BYTES + 512 + 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this CTA's shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Into this CTA's shared memory, the bytes counted by a barrier of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1,
                                                 uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "l"(policy)
      : "memory");
}
// Arrival on the same barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void tc_cp_sf_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                               uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tc_mma_mxf8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                                 uint32_t accumulate, uint32_t sfa_tmem, uint32_t sfb_tmem) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa_tmem), "r"(sfb_tmem)
      : "memory");
}
constexpr uint32_t IDESC_B_MN = 1u << 16;   // operand B stored along N
// kind::mxf8f6f4 descriptor (E4M3 both) with M = 256 instead of 128.
__device__ __forceinline__ uint32_t idesc_mxf8_pair(uint32_t sf_id) {
  return (idesc_mxf8f6f4(L_TN, false, sf_id, true) & ~(31u << 24)) | ((256u >> 4) << 24);
}

struct LTile {
  int64_t m0;
  int n0;
};
__device__ __forceinline__ LTile large_tile(int t, int mt, int nt) {
  const int per = L_RASTER * nt, g = t / per, r = t - g * per;
  const int gm = min(L_RASTER, mt - g * L_RASTER);
  LTile o;
  o.m0 = (int64_t)(g * L_RASTER + r % gm) * L_TM;
  o.n0 = (r / gm) * L_TN;
  return o;
}

// 128 columns of a row from n0, columns >= N left alone; vec: 16-byte stores.
__device__ __forceinline__ void store_row(const float (&acc)[128], const Fp8Params& p, int64_t m, int64_t n0,
                                          int out_f32, bool vec) {
  if (out_f32) {
    float* y = static_cast<float*>(p.y) + m * p.ldy + n0;
#pragma unroll
    for (int c = 0; c < 128; c += 4) {
      if (vec && n0 + c + 4 <= p.N) {
        *reinterpret_cast<float4*>(y + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n0 + c + j < p.N) y[c + j] = acc[c + j];
      }
    }
  } else {
    uint16_t* y = static_cast<uint16_t*>(p.y) + m * p.ldy + n0;
#pragma unroll
    for (int c = 0; c < 128; c += 8) {
      if (vec && n0 + c + 8 <= p.N) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = bf16_bits(acc[c + 2 * j]) | ((uint32_t)bf16_bits(acc[c + 2 * j + 1]) << 16);
        *reinterpret_cast<uint4*>(y + c) = make_uint4(o[0], o[1], o[2], o[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (n0 + c + j < p.N) y[c + j] = bf16_bits(acc[c + j]);
      }
    }
  }
}

template <bool E8, bool B_MN>
__global__ void __launch_bounds__(L_THREADS, 1)
    fp8_matmul_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const Fp8Params p, const int mt, const int nt, const int out_f32, const int vec) {
  constexpr int NACC = E8 ? 1 : 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* slots = smem + L_STAGES * L_STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + F_SLOTS * L_SLOT_BYTES);   // leader's: both CTAs' bytes
  uint64_t* empty = full + L_STAGES;
  uint64_t* sfull = empty + L_STAGES;       // leader's: one arrival per CTA
  uint64_t* sempty = sfull + F_SLOTS;
  uint64_t* accfull = sempty + F_SLOTS;
  uint64_t* accempty = accfull + NACC;      // leader's: the epilogue warps of both CTAs
  uint64_t* drain = accempty + NACC;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  int* err = reinterpret_cast<int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp-uniform
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int nkt = p.kb, ngr = (nkt + F_GROUP - 1) / F_GROUP, tiles = mt * nt;
  if (threadIdx.x == 0) {
    for (int s = 0; s < L_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < F_SLOTS; ++s) {
      mbar_init(&sfull[s], 2);
      mbar_init(&sempty[s], 1);
    }
    for (int s = 0; s < NACC; ++s) {
      mbar_init(&accfull[s], 1);
      mbar_init(&accempty[s], 2 * L_EPI_WARPS);
    }
    mbar_init(drain, 1);
    *err = 0;
    fence_barrier_init();
    prefetch_tensormap(&tmW);
    prefetch_tensormap(&tmX);
  }
  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's barriers are initialised too
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_holder, 0);
  griddep_wait();
  griddep_launch();

  if (warp == 0) {
    const uint64_t pol = policy_evict_normal();
    int it = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const LTile tl = large_tile(t, mt, nt);
      const int m0 = (int)(tl.m0 + rank * 128), n0 = tl.n0 + (int)rank * 128;
      for (int kt = 0; kt < nkt; ++kt, ++it) {
        const int s = it % L_STAGES;
        if (it >= L_STAGES && !(ok = warp_wait(&empty[s], (uint32_t)(it / L_STAGES - 1) & 1u, err))) break;
        uint8_t* st = smem + s * L_STAGE_BYTES;
        const uint32_t bar = map_rank(&full[s], 0);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&full[s], 2 * L_STAGE_BYTES);
          tma_load_2d_pair(st, &tmX, bar, kt * F_BK, m0, pol);
          if constexpr (B_MN) tma_load_2d_pair(st + 128 * F_BK, &tmW, bar, n0, kt * F_BK, pol);
          else tma_load_2d_pair(st + 128 * F_BK, &tmW, bar, kt * F_BK, n0, pol);
          if (rank == 0) mbar_arrive(&full[s]);
        }
        __syncwarp();
      }
    }
    if (!ok) {
      // a wait ran out: the copies still in flight land (microseconds) before the CTA exits
      const uint64_t t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 10000000ull) {
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t mn = B_MN ? IDESC_B_MN : 0u;
      constexpr uint32_t B_STEP = B_MN ? (32 * 128) >> 4 : 2u;
      int it = 0, grp = 0, ti = 0;
      bool ok = true;
      for (int t = pair; t < tiles && ok; t += pairs, ++ti) {
        if constexpr (E8) {
          if (ti > 0 && !(ok = warp_wait(&accempty[0], (uint32_t)(ti - 1) & 1u, err))) break;
        }
        for (int kt = 0; kt < nkt; ++kt, ++it) {
          const int s = it % L_STAGES;
          if (!(ok = warp_wait(&full[s], (uint32_t)(it / L_STAGES) & 1u, err))) break;
          const uint32_t aA = smem_u32(smem + s * L_STAGE_BYTES);
          const uint64_t dA = desc_sw128(aA), dB = desc_sw128(aA + 128 * F_BK);
          if constexpr (E8) {
            if (kt % F_GROUP == 0 && kt > 0) ++grp;
            const int slot = grp % F_SLOTS;
            const uint32_t sfa = tmem + L_SF_COL + 16 * (grp & 1), sfb = sfa + 4;
            const bool fresh = kt % F_GROUP == 0;
            if (fresh && !(ok = warp_wait(&sfull[slot], (uint32_t)(grp / F_SLOTS) & 1u, err))) break;
            tc_fence_after();
            const uint32_t id = kt % F_GROUP, sel = id << 30;
            const uint32_t idesc = idesc_mxf8_pair(id) | mn;
            if (elect_one()) {
              if (fresh) {
                const uint32_t sl = smem_u32(slots + slot * L_SLOT_BYTES);
                tc_cp_sf_pair(sfa, desc_sf(sl));
                tc_cp_sf_pair(sfb, desc_sf(sl + 512));
                tc_cp_sf_pair(sfb + 4, desc_sf(sl + 1024));
                tc_commit_pair(&sempty[slot]);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma_mxf8_pair(tmem, dA + 2u * j, dB + B_STEP * j, idesc, (kt | j) != 0 ? 1u : 0u, sfa | sel,
                                 sfb | sel);
              tc_commit_pair(&empty[s]);
              if (kt == nkt - 1) tc_commit_pair(&accfull[0]);
            }
          } else {
            const int ab = it & 1;
            if (it >= 2 && !(ok = warp_wait(&accempty[ab], (uint32_t)(it / 2 - 1) & 1u, err))) break;
            tc_fence_after();
            const uint32_t idesc = idesc_f8(256, L_TN) | mn;
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma_f8_pair(tmem + ab * 256, dA + 2u * j, dB + B_STEP * j, idesc, j != 0 ? 1u : 0u);
              tc_commit_pair(&empty[s]);
              tc_commit_pair(&accfull[ab]);
            }
          }
          __syncwarp();
        }
        if constexpr (E8) ++grp;
      }
      if (elect_one()) tc_commit_pair(drain);
      __syncwarp();
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < DSV4_WAIT_NS) {
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    if constexpr (E8) {
      int grp = 0;
      bool ok = true;
      uint32_t cur[4][4], nxt[4][4], wbyte[2] = {};
      auto load = [&](int t, int kt) {
        const int64_t m0 = large_tile(t, mt, nt).m0 + rank * 128;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          sf_row(static_cast<const uint8_t*>(p.as) + (m < p.M ? m * nkt : 0), kt, nkt, p.vec, m < p.M, nxt[j]);
        }
      };
      if (pair < tiles) load(pair, 0);
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int nb0 = large_tile(t, mt, nt).n0 / 128;
        for (int gr = 0; gr < ngr && ok; gr += 4) {
          if (gr % 8 == 0) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
              wbyte[j] = sf_lane(static_cast<const uint8_t*>(p.bs) + (int64_t)(nb0 + j) * p.bs_n, p.bs_k,
                                 gr * F_GROUP + lane, nkt, (nb0 + j) * 128 < p.N);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) cur[j][g] = nxt[j][g];
          if (gr + 4 < ngr) load(t, (gr + 4) * F_GROUP);
          else if (t + pairs < tiles) load(t + pairs, 0);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            if (gr + g >= ngr) break;
            const int slot = grp % F_SLOTS;
            uint8_t* sl = slots + slot * L_SLOT_BYTES;
            const uint32_t wb0 = sf_gather(wbyte[0], (gr + g) % 8 * 4), wb1 = sf_gather(wbyte[1], (gr + g) % 8 * 4);
            if (grp >= F_SLOTS && !(ok = warp_wait(&sempty[slot], (uint32_t)(grp / F_SLOTS - 1) & 1u, err))) break;
            *reinterpret_cast<uint4*>(sl + lane * 16) = make_uint4(cur[0][g], cur[1][g], cur[2][g], cur[3][g]);
            *reinterpret_cast<uint4*>(sl + 512 + lane * 16) = make_uint4(wb0, wb0, wb0, wb0);
            *reinterpret_cast<uint4*>(sl + 1024 + lane * 16) = make_uint4(wb1, wb1, wb1, wb1);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(map_rank(&sfull[slot], 0));
            ++grp;
          }
        }
      }
    }
  } else if (warp >= F_EPI_WARP0) {
    const int q = warp & 3, c0 = ((warp - F_EPI_WARP0) >> 2) * 128;
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0;
    int it = 0, ti = 0;
    bool ok = true;
    for (int t = pair; t < tiles && ok; t += pairs, ++ti) {
      const LTile tl = large_tile(t, mt, nt);
      const int64_t m = tl.m0 + rank * 128 + q * 32 + lane, n0 = tl.n0 + c0;
      float acc[128];
      if constexpr (E8) {
        ok = warp_wait(&accfull[0], (uint32_t)ti & 1u, err);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 128; c += 16) tmem_ld16(trow + c, acc + c);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(map_rank(&accempty[0], 0));
      } else {
#pragma unroll
        for (int c = 0; c < 128; ++c) acc[c] = 0.f;
        const bool inm = m < p.M, inn = n0 < p.N;
        const float* as = static_cast<const float*>(p.as) + (inm ? m * nkt : 0);
        const float* bs = static_cast<const float*>(p.bs) + (inn ? n0 / 128 * p.bs_n : 0);
        float sa[F_GROUP], na[F_GROUP], sb = 0.f;
        scale_row<F_GROUP>(as, 0, nkt, p.vec, inm, na);
        for (int kt = 0; kt < nkt; ++kt, ++it) {
          if (kt % 32 == 0) sb = inn && kt + lane < nkt ? __ldcg(bs + (int64_t)(kt + lane) * p.bs_k) : 0.f;
          if (kt % F_GROUP == 0) {
#pragma unroll
            for (int i = 0; i < F_GROUP; ++i) sa[i] = na[i];
            if (kt + F_GROUP < nkt) scale_row<F_GROUP>(as, kt + F_GROUP, nkt, p.vec, inm, na);
          }
          const float s = sa[0] * __shfl_sync(0xffffffffu, sb, kt % 32);
          sa[0] = sa[1], sa[1] = sa[2], sa[2] = sa[3];
          const int ab = it & 1;
          ok = warp_wait(&accfull[ab], (uint32_t)(it / 2) & 1u, err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            float v[16];
            tmem_ld16(trow + ab * 256 + c, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(v[j], s, acc[c + j]);
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(map_rank(&accempty[ab], 0));
        }
        if (!ok) break;
      }
      if (m < p.M) store_row(acc, p, m, n0, out_f32, vec != 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // the other CTA's MMAs into this CTA's TMEM and its arrivals here are done
  if (threadIdx.x == 0 && *err) set_status(&g_fp8_status, *err);
  if (warp == 3) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <bool E8, bool B_MN>
int launch_pair(const CUtensorMap& tx, const CUtensorMap& tw, const Fp8Params& p, int out_f32, int sms,
                cudaStream_t st) {
  auto k = fp8_matmul_pair_kernel<E8, B_MN>;
  DSV4_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, L_SMEM));
  const int64_t mt = (p.M + L_TM - 1) / L_TM, nt = (p.N + L_TN - 1) / L_TN;
  const int pairs = (int)std::min<int64_t>(mt * nt, sms / 2);
  const int al = out_f32 ? 4 : 8;
  const int vec = p.ldy % al == 0 && (uintptr_t)p.y % 16 == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs));
  cfg.blockDim = dim3(L_THREADS);
  cfg.dynamicSmemBytes = L_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  DSV4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, tx, tw, p, (int)mt, (int)nt, out_f32, vec));
  return DSV4_OK;
}

}  // namespace

static int fp8_matmul_run(const uint8_t* a, int64_t lda, const void* as, const uint8_t* b, int64_t ldb, const void* bs,
                          int scale_type, bool trans_b, int64_t m, int64_t n, int64_t k, void* y, int64_t ldy,
                          int out_dtype, cudaStream_t st) {
  const int64_t kb = (k + F_BK - 1) / F_BK, nb = (n + F_BK - 1) / F_BK;
  Fp8Params p{as, bs, trans_b ? 1 : nb, trans_b ? kb : 1, y, ldy, m, n, (int)kb,
              scale_vec(as, (int)kb, scale_type == DSV4_SCALE_E8M0)};
  const bool large = m > 128 && n > 128;
  const int bn = large ? 128 : m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128));
  CUtensorMap tw, tx;
  const uint64_t dw[2] = {(uint64_t)(trans_b ? k : n), (uint64_t)(trans_b ? n : k)}, sw[1] = {(uint64_t)ldb};
  const uint32_t bw[2] = {128, 128};
  if (int rc = make_map(&tw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)b, dw, sw, bw, "fp8_matmul b")) return rc;
  const uint64_t dx[2] = {(uint64_t)k, (uint64_t)m}, sx[1] = {(uint64_t)lda};
  const uint32_t bx[2] = {128, (uint32_t)bn};
  if (int rc = make_map(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)a, dx, sx, bx, "fp8_matmul a")) return rc;
  const bool e8 = scale_type == DSV4_SCALE_E8M0;
  const int f32 = out_dtype == DSV4_DT_FP32;
  if (large) {
    int dev = 0, sms = 0;
    DSV4_CUDA_CHECK(cudaGetDevice(&dev));
    DSV4_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    if (e8) return trans_b ? launch_pair<true, false>(tx, tw, p, f32, sms, st) : launch_pair<true, true>(tx, tw, p, f32, sms, st);
    return trans_b ? launch_pair<false, false>(tx, tw, p, f32, sms, st) : launch_pair<false, true>(tx, tw, p, f32, sms, st);
  }
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
