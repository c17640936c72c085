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
// E8M0 scales: tcgen05 kind::mxf8f6f4 applies them.  Its four scale bytes per
//   row (32 of K each) hold the scales of four consecutive 128-blocks instead,
//   and the four MMAs of a k-tile all name byte (kt % 4): one 4-byte word per
//   row and 512 of K, the bytes as they lie in memory.
// fp32 scales: kind::f8f6f4 into a ring of TMEM accumulators, one k-tile each;
//   the epilogue warps add as * bs times each partial sum to fp32 registers.
//   Handing an accumulator over (commit, load, release) takes about as long as
//   three k-tiles' MMAs: four of them with few rows, two wider ones in the
//   pair kernel.
//
// Measured (device, graph replay): 1 x 2048 x 4096 5.0 us, 64 x 4096 x 4096 7.4
// us, 2048 x 4096 x 4096 29 us, 8192 x 8192 x 4096 206 us (2.67 PFLOP/s) with
// E8M0 scales, 288 us (1.91 PFLOP/s) with fp32 scales; the same inputs in every
// replay, so the small ones stay in L2.  Few rows are bound by
// latency (the weights alone would take 1.3 us of HBM time for the first), many
// by the tensor cores and L2 (64 B per clock and SM), fp32 scales by the
// epilogue's multiply-adds.
//
// Two kernels share the roles (TMA producer, MMA issuer, scale loader,
// epilogue): a CTA per 128 of N and up to 128 rows of a whose K a cluster
// splits (few rows: latency, HBM), and a persistent one of CTA pairs (many
// rows: tensor cores, L2).  fp8_shape() chooses.
#include <algorithm>
#include <atomic>

#include "capi_internal.h"
#include "common.cuh"
#include "fp8_quant.cuh"

namespace dsv4 {
namespace {

constexpr int F_BK = 128;              // k-tile = one scale block, one 128-byte swizzle row
constexpr int F_BM = 128;              // of N (weight rows) per CTA
constexpr int F_GROUP = 4;             // k-tiles per scale group
constexpr int F_SLOTS = 4;             // scale groups in flight
constexpr int F_EPI_WARP0 = 4;
constexpr int F_MAX_SMEM = 227 * 1024;        // a CTA's opt-in limit
constexpr int F_SM_SMEM = 228 * 1024;         // an SM's, 1 KB of which each CTA takes beside its own
constexpr int F_MIN_SMEM = 92 * 1024;         // every kernel here takes more
// Whether two CTAs of these kernels, one of `smem` bytes and any other, never
// share an SM; else each may take half of the SM's 512 TMEM columns.
constexpr bool alone_on_sm(int smem) { return smem + F_MIN_SMEM + 2 * 1024 > F_SM_SMEM; }
constexpr int64_t F_MAX_M = 65535LL * 128;   // grid y, in tiles of 128 rows

// Set by a kernel whose bounded wait ran out; read by dsv4_fp8_status.
__device__ int g_fp8_status;

struct Fp8Params {
  const void* as;      // [M, kb] bytes or floats
  const void* bs;      // element (kb, nb) at kb * bs_k + nb * bs_n
  int64_t bs_k, bs_n;
  void* y;
  int64_t ldy, M, N;
  int kb;              // scale blocks along K = k-tiles
  int vec;             // access width of a row of `as` (scale_vec)
  int out_f32;         // y is fp32, else bf16
  // rows to quantise (FUSE): bf16 on 16 bytes, K a multiple of 8
  const uint16_t* x;
  int64_t ldx, K;
  int vec_y;           // rows of y take vector stores
};

// ---------------------------------------------------------------------------
// waits, cluster and issue helpers
// ---------------------------------------------------------------------------
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
// Bounded wait of a whole warp; every lane gets the same answer.  False once a
// wait of this CTA has run out.  CLUSTER: what another CTA wrote before its
// arrival is read after the wait (the fence that this takes is not free).
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status) {
  uint64_t t0 = 0;
  bool ok = true;
  for (uint32_t i = 1;; ++i) {
    if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) break;
    if (i % 64 == 0 && read_status(status) == DSV4_ETIMEOUT) {
      ok = false;
      break;
    }
    if (i % 1024 == 0) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > DSV4_WAIT_NS) {
        set_status(status, DSV4_ETIMEOUT);
        ok = false;
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
// Whether the phase has completed, for a later `__all_sync(~0u, ...) ||
// warp_wait(...)`: a look ahead whose latency hides behind other work.
__device__ __forceinline__ uint32_t bar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok;
}
// Position in a ring of N stages: the stage, and the parity of its current
// round.  (Kept by counting: quotients by five on the way to every wait cost
// the fp32-scale epilogue 0.1 us per k-tile.)
template <int N>
struct Ring {
  int s = 0;
  uint32_t ph = 0;
  __device__ __forceinline__ void next() {
    if (++s == N) {
      s = 0;
      ph ^= 1u;
    }
  }
};
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
// Arrival that publishes nothing in memory (an accumulator has been read: its
// values are in registers).  What it orders, the loads from TMEM before the
// leader's next MMA into it, the tcgen05 fences on both sides of each wait and
// arrival order; a release at cluster scope here, and an acquire in the wait
// for it, cost 1.1 us per k-tile together.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// ---------------------------------------------------------------------------
// tcgen05
// ---------------------------------------------------------------------------
__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
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
__device__ __forceinline__ void tc_cp_sf_pair(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
}
// Arrival on the same barrier of both CTAs once the MMAs issued so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// Instruction descriptors: kind::f8f6f4 with E4M3 A and B, fp32 D; either
// kind's bits for an operand stored along M / N; kind::mxf8f6f4 with M = 256.
__device__ __forceinline__ uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | (((uint32_t)(n >> 3) & 63u) << 17) | (((uint32_t)(m >> 4) & 31u) << 24);
}
constexpr uint32_t IDESC_A_MN = 1u << 15;
constexpr uint32_t IDESC_B_MN = 1u << 16;
__device__ __forceinline__ uint32_t idesc_mxf8_pair(int n, uint32_t sf_id) {
  return (idesc_mxf8f6f4(n, false, sf_id, true) & ~(31u << 24)) | ((256u >> 4) << 24);
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

// ---------------------------------------------------------------------------
// Scales of 16 (E8M0) or 4 (fp32) k-tiles at a time, a chunk ahead of their
// use.  Rows of `as` are loaded with the widest access that their start
// allows, and the loads of a chunk are all in flight together (one byte-wise
// load per k-tile kept the tensor cores waiting: 0.8 us a k-tile instead of
// 0.28).  Read past L1: the kernel just before may have written them.  Past
// the end of K: byte 127 (= 1) or float 0; the operand bytes there are zero.
// ---------------------------------------------------------------------------
// Access width of the rows of `as`, in elements: 16, 4 or 1 bytes, 4 or 1 floats.
inline int scale_vec(const void* as, int kb, bool e8) {
  if (!e8) return kb % 4 == 0 && (uintptr_t)as % 16 == 0 ? 4 : 1;
  return kb % 16 == 0 && (uintptr_t)as % 16 == 0 ? 16 : (kb % 4 == 0 && (uintptr_t)as % 4 == 0 ? 4 : 1);
}
// Words w[g] = bytes of k-tiles kt + 4 g ..+ 3 of the row at p.
__device__ __forceinline__ void sf_row(const uint8_t* p, int kt, int kb, int vec, bool in, uint32_t (&w)[4]) {
  if (in && vec == 16) {   // rows are multiples of 16 bytes: a chunk never leaves its row
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
// The byte of k-tile kt of a block column, a lane each of 32.
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
// f[i] = float of k-tile kt + i of the row at p.
__device__ __forceinline__ void scale_row(const float* p, int kt, int kb, int vec, bool in, float (&f)[F_GROUP]) {
  if (vec == 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (in && kt < kb) v = __ldcg(reinterpret_cast<const float4*>(p + kt));
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else {
#pragma unroll
    for (int j = 0; j < F_GROUP; ++j) f[j] = in && kt + j < kb ? __ldcg(p + kt + j) : 0.f;
  }
}

// ---------------------------------------------------------------------------
// Few rows: weights are the M side of the MMA (128 of N per CTA), rows of a
// its N side (BN), so that one row still feeds whole 128-row MMAs.  The CTAs
// of a cluster take a share of K each; at the end every CTA adds one slice of
// the tile over the others' shared memory, in rank order.
//   warp 0: TMA producer, warp 1: MMA issuer, warp 2: scales, warp 3: TMEM
//   warps 4..: epilogue, 32 of N each (lane = weight row, columns = rows of a)
// FUSE (a linear layer on up to 64 rows): a's tiles are not loaded but made
// from the bf16 rows by further warps, a half warp per row and k-tile, codes
// and scales as act_quant gives them.  One launch instead of two; every CTA
// quantises its share of K again, out of L2.
// ---------------------------------------------------------------------------
template <int BN, bool E8, bool FUSE = false>
struct FCfg {
  static constexpr int A_BYTES = F_BM * F_BK;
  static constexpr int B_BYTES = BN * F_BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // Two CTAs share an SM: their rings stay within half of its shared memory.
  static constexpr int STAGES = BN == 128 ? (E8 ? 3 : 4) : (BN == 64 ? 4 : 5);
  static constexpr int SLOT_BYTES = E8 ? 1024 : F_GROUP * BN * 4;
  static constexpr int EPI_WARPS = BN >= 64 ? 8 : 4;
  static constexpr int COLS = BN / (EPI_WARPS / 4);      // accumulator columns per epilogue warp
  static constexpr int QUANT_WARPS = FUSE ? (BN == 64 ? 8 : 4) : 0;
  static constexpr int QUANT_WARP0 = F_EPI_WARP0 + EPI_WARPS;
  static constexpr int THREADS = (QUANT_WARP0 + QUANT_WARPS) * 32;
  static constexpr int RESIDENT = BN <= 32 || (E8 && !FUSE) ? 2 : 1;   // CTAs per SM (registers)
  static constexpr int NACC = E8 ? 1 : 4;
  static constexpr int SF_COL = BN;                      // E8M0: 8 columns of scales, twice
  static constexpr uint32_t TMEM_COLS = E8 ? (BN == 128 ? 256 : (BN == 64 ? 128 : (BN == 32 ? 64 : 32))) : NACC * BN;
  static constexpr int BARS = 2 * STAGES + 2 * F_SLOTS + 2 * NACC + 1;
  static constexpr int RED_BYTES = BN * F_BM * 4;        // fp32 results, in the ring after the last MMA
  static constexpr int SMEM = STAGES * STAGE_BYTES + F_SLOTS * SLOT_BYTES + BARS * 8 + 16 + 1024;
  static_assert(RED_BYTES <= STAGES * STAGE_BYTES, "the ring holds the results");
  // The CTAs of a cluster wait for one another, so a CTA that is resident must
  // get its TMEM without waiting for another resident one: at most two of
  // these CTAs fit an SM (shared memory), and either both take at most half
  // of the 512 columns or one leaves no room for the other.  (The routed
  // layer's kernels with TMEM take 176 KB or more: none shares an SM with these.)
  static_assert(SMEM >= F_MIN_SMEM && 3 * (F_MIN_SMEM + 1024) > F_SM_SMEM, "at most two CTAs per SM");
  static_assert(TMEM_COLS <= 256 || alone_on_sm(SMEM), "two CTAs share an SM's TMEM");
};

// Eight columns of a row of x from column c (zeros past the end of K).
__device__ __forceinline__ uint4 x_load(const Fp8Params& p, int64_t m, int64_t c) {
  return m < p.M && c < p.K ? __ldcg(reinterpret_cast<const uint4*>(p.x + m * p.ldx + c)) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ void x_floats(const uint4& o, float (&v)[8]) {
  const uint32_t d[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = bf16_from_bits((d[j >> 1] >> (16 * (j & 1))) & 0xffffu);
}

template <int BN, bool E8, bool A_MN, bool FUSE>
__global__ void __launch_bounds__(FCfg<BN, E8, FUSE>::THREADS, FCfg<BN, E8, FUSE>::RESIDENT)
    fp8_matmul_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                      const Fp8Params p, const int per) {
  using C = FCfg<BN, E8, FUSE>;
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
  // this CTA's k-tiles: kbeg .. kbeg + nkt - 1 (`per`, a multiple of 4, per CTA of the cluster)
  const int split = gridDim.z, rank = blockIdx.z;
  const int kbeg = rank * per, nkt = min(per, p.kb - kbeg);
  const int ngr = (nkt + F_GROUP - 1) / F_GROUP;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1 + C::QUANT_WARPS);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < F_SLOTS; ++s) {
      mbar_init(&sfull[s], FUSE && !E8 ? C::QUANT_WARPS : 1);
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
    if constexpr (!FUSE) prefetch_tensormap(&tmX);
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
    Ring<C::STAGES> ring;
    for (int kt = 0; kt < nkt; ++kt, ring.next()) {
      const int s = ring.s;
      if (kt >= C::STAGES && !warp_wait(&empty[s], ring.ph ^ 1u, err)) break;
      uint8_t* st = smem + s * C::STAGE_BYTES;
      const int k0 = (kbeg + kt) * F_BK;
      if (elect_one()) {
        mbar_expect_tx(&full[s], FUSE ? C::A_BYTES : C::STAGE_BYTES);
        if constexpr (A_MN) tma_load_2d(st, &tmW, &full[s], n0, k0, pol);
        else tma_load_2d(st, &tmW, &full[s], k0, n0, pol);
        if constexpr (!FUSE) tma_load_2d(st + C::A_BYTES, &tmX, &full[s], k0, (int)m0, pol);
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
    Ring<C::STAGES> ring;
    for (int kt = 0; kt < nkt; ++kt, ring.next()) {
      const int s = ring.s, gr = kt / F_GROUP, slot = gr % F_SLOTS;
      if (!warp_wait(&full[s], ring.ph, err)) break;
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
          const uint32_t sl = smem_u32(slots + slot * C::SLOT_BYTES);
          if (fresh) tc_cp_sf(sfa, desc_sf(sl));
          // FUSE: the bytes of a's words come one k-tile after the other
          if (FUSE || fresh) tc_cp_sf(sfb, desc_sf(sl + 512));
          if (FUSE ? kt % F_GROUP == F_GROUP - 1 || kt == nkt - 1 : fresh) tc_commit(&sempty[slot]);
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
          tc_commit(&empty[s]);   // the stage is free and the accumulator is full
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
    constexpr int ROWS = (BN + 31) / 32;                       // rows of a per lane
    const int vec = kbeg % 16 == 0 ? p.vec : min(p.vec, 4);
    if constexpr (E8) {
      const uint8_t* bs = static_cast<const uint8_t*>(p.bs) + (int64_t)(n0 / F_BK) * p.bs_n + (int64_t)kbeg * p.bs_k;
      uint32_t cur[ROWS][4], nxt[ROWS][4], wbyte = 0;
      auto load = [&](int kt) {
        if constexpr (FUSE) return;   // the quantising warps write a's bytes
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          const bool in = lane + 32 * j < BN && m < p.M;
          sf_row(static_cast<const uint8_t*>(p.as) + (in ? m * p.kb + kbeg : 0), kt, nkt, vec, in, nxt[j]);
        }
      };
      load(0);
      bool ok = true;
      for (int gr = 0; gr < ngr && ok; gr += 4) {
        if (gr % 8 == 0) wbyte = sf_lane(bs, p.bs_k, gr * F_GROUP + lane, nkt, true);
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
#pragma unroll
          for (int g = 0; g < 4; ++g) cur[j][g] = nxt[j][g];
        if (gr + 4 < ngr) load((gr + 4) * F_GROUP);
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
          if constexpr (!FUSE) *reinterpret_cast<uint4*>(sl + 512 + lane * 16) = make_uint4(wb[0], wb[1], wb[2], wb[3]);
          fence_proxy_async_smem();   // read by tcgen05.cp
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[slot]);
        }
      }
    } else if constexpr (!FUSE) {
      const float* bs = static_cast<const float*>(p.bs) + (int64_t)(n0 / F_BK) * p.bs_n + (int64_t)kbeg * p.bs_k;
      float cur[ROWS][F_GROUP], nxt[ROWS][F_GROUP], sb = 0.f;
      auto load = [&](int kt) {
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          const bool in = lane + 32 * j < BN && m < p.M;
          scale_row(static_cast<const float*>(p.as) + (in ? m * p.kb + kbeg : 0), kt, nkt, vec, in, nxt[j]);
        }
      };
      load(0);
      for (int gr = 0; gr < ngr; ++gr) {
        const int slot = gr % F_SLOTS, kt0 = gr * F_GROUP;
        if (gr % 8 == 0) sb = kt0 + lane < nkt ? __ldcg(bs + (int64_t)(kt0 + lane) * p.bs_k) : 0.f;
#pragma unroll
        for (int j = 0; j < ROWS; ++j)
#pragma unroll
          for (int i = 0; i < F_GROUP; ++i) cur[j][i] = nxt[j][i];
        if (gr + 1 < ngr) load(kt0 + F_GROUP);
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
  } else if (FUSE && warp >= C::QUANT_WARP0) {
    // ------------------------------------------------------------- quantising
    constexpr int QW = FUSE ? C::QUANT_WARPS : 1, PASS = FUSE ? BN / (2 * QW) : 1;
    const int hl = lane & 15, row0 = (warp - C::QUANT_WARP0) * 2 + (lane >> 4);   // rows row0 + i * 2 QW
    const float* bs = E8 ? nullptr
                         : static_cast<const float*>(p.bs) + (int64_t)(n0 / F_BK) * p.bs_n + (int64_t)kbeg * p.bs_k;
    uint4 nxt[PASS];
    float sb = 0.f;
    auto load = [&](int kt) {
#pragma unroll
      for (int i = 0; i < PASS; ++i) nxt[i] = x_load(p, m0 + row0 + i * 2 * QW, (int64_t)(kbeg + kt) * F_BK + hl * 8);
      if constexpr (!E8) sb = __ldcg(bs + (int64_t)kt * p.bs_k);
    };
    load(0);
    Ring<C::STAGES> ring;
    for (int kt = 0; kt < nkt; ++kt, ring.next()) {
      uint2 code[PASS];
      float sc[PASS];   // E8M0: the exponent byte
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        float v[8];
        x_floats(nxt[i], v);
        const float a = fp8_amax(v);
        if constexpr (E8) {
          const int e = scale_exp_448(a);
          code[i] = fp8_codes_pow2(v, e);
          sc[i] = __int_as_float(e + 127);
        } else {
          code[i] = fp8_codes_fp32<false>(v, a);
          sc[i] = fp8_scale_fp32(a) * sb;
        }
      }
      if (kt + 1 < nkt) load(kt + 1);
      const int gr = kt / F_GROUP, slot = E8 ? gr % F_SLOTS : kt % F_SLOTS;
      if (kt >= C::STAGES && !warp_wait(&empty[ring.s], ring.ph ^ 1u, err)) break;
      if constexpr (E8) {
        if (kt % F_GROUP == 0 && gr >= F_SLOTS && !warp_wait(&sempty[slot], (uint32_t)(gr / F_SLOTS - 1) & 1u, err)) break;
      } else {
        if (kt >= F_SLOTS && !warp_wait(&sempty[slot], (uint32_t)(kt / F_SLOTS - 1) & 1u, err)) break;
      }
      uint8_t* tile = smem + ring.s * C::STAGE_BYTES + C::A_BYTES;
      uint8_t* sl = slots + slot * C::SLOT_BYTES;
#pragma unroll
      for (int i = 0; i < PASS; ++i) {
        // rows of 128 bytes, 16-byte units swizzled by row as TMA would
        const int r = row0 + i * 2 * QW;
        *reinterpret_cast<uint2*>(tile + r * 128 + (((hl >> 1) ^ (r & 7)) << 4) + (hl & 1) * 8) = code[i];
        if (hl == 0) {
          if constexpr (E8) sl[512 + (r & 31) * 16 + (r >> 5) * 4 + kt % F_GROUP] = (uint8_t)__float_as_int(sc[i]);
          else reinterpret_cast<float*>(sl)[r] = sc[i];
        }
      }
      fence_proxy_async_smem();   // read by the tensor cores
      __syncwarp();
      if (lane == 0) {
        if constexpr (!E8) mbar_arrive(&sfull[slot]);
        mbar_arrive(&full[ring.s]);
      }
    }
    __syncwarp();
  } else if (warp >= F_EPI_WARP0) {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, c0 = ((warp - F_EPI_WARP0) >> 2) * C::COLS;
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0;
    float* red = reinterpret_cast<float*>(smem) + c0 * F_BM + q * 32 + lane;   // [row of a][128 of N]
    if constexpr (E8) {
      if (warp_wait(&accfull[0], 0, err)) {
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::COLS; c += 16) {
          float v[16];
          tmem_ld16(trow + c, v);
          tc_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) red[(c + j) * F_BM] = v[j];
        }
      }
    } else {
      float acc[C::COLS];
#pragma unroll
      for (int c = 0; c < C::COLS; ++c) acc[c] = 0.f;
      bool ok = true;
      Ring<C::STAGES> ring;
      for (int kt = 0; kt < nkt; ++kt, ring.next()) {
        // a slot holds the scales of four k-tiles; FUSE: of one
        constexpr int SPAN = FUSE ? 1 : F_GROUP;
        const int ab = kt % C::NACC, gr = kt / SPAN, slot = gr % F_SLOTS;
        if (kt % SPAN == 0 && !(ok = warp_wait(&sfull[slot], (uint32_t)(gr / F_SLOTS) & 1u, err))) break;
        if (!(ok = warp_wait(&empty[ring.s], ring.ph, err))) break;
        tc_fence_after();
        float v[C::COLS];
#pragma unroll
        for (int c = 0; c < C::COLS; c += 16) tmem_ld16(trow + ab * BN + c, v + c);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&accempty[ab]);
        const float* f = reinterpret_cast<const float*>(slots + slot * C::SLOT_BYTES) + (kt % SPAN) * BN + c0;
#pragma unroll
        for (int c = 0; c < C::COLS; c += 4) {
          const float4 s = *reinterpret_cast<const float4*>(f + c);
          acc[c] = fmaf(v[c], s.x, acc[c]);
          acc[c + 1] = fmaf(v[c + 1], s.y, acc[c + 1]);
          acc[c + 2] = fmaf(v[c + 2], s.z, acc[c + 2]);
          acc[c + 3] = fmaf(v[c + 3], s.w, acc[c + 3]);
        }
        __syncwarp();
        if (lane == 0 && (kt % SPAN == SPAN - 1 || kt == nkt - 1)) mbar_arrive(&sempty[slot]);
      }
      // the last accumulator is full: no MMA reads the ring any more
      if (ok) {
#pragma unroll
        for (int c = 0; c < C::COLS; ++c) red[c * F_BM] = acc[c];
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  // the cluster's partial results, each CTA a slice, added in rank order
  if (split > 1) cluster_sync();
  else __syncthreads();
  const int rows = (int)min((int64_t)BN, p.M - m0), units = rows * (F_BM / 4);   // of four columns
  const int u1 = (int)((int64_t)units * (rank + 1) / split);
  for (int u = (int)((int64_t)units * rank / split) + (int)threadIdx.x; u < u1; u += C::THREADS) {
    const float* src = reinterpret_cast<const float*>(smem) + u * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (split == 1) {
      a = *reinterpret_cast<const float4*>(src);
    } else {
      for (int r = 0; r < split; ++r) {
        const float4 v = ld_cluster_f4(map_rank(src, r));
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
      }
    }
    const int64_t n = (int64_t)n0 + u % (F_BM / 4) * 4, at = (m0 + u / (F_BM / 4)) * p.ldy + n;
    const float o[4] = {a.x, a.y, a.z, a.w};
    if (p.out_f32) {
      float* y = static_cast<float*>(p.y) + at;
      if (p.vec_y && n + 4 <= p.N) {
        *reinterpret_cast<float4*>(y) = a;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) y[j] = o[j];
      }
    } else {
      uint16_t* y = static_cast<uint16_t*>(p.y) + at;
      if (p.vec_y && n + 4 <= p.N) {
        *reinterpret_cast<uint2*>(y) = make_uint2(bf16_bits(a.x) | ((uint32_t)bf16_bits(a.y) << 16),
                                                  bf16_bits(a.z) | ((uint32_t)bf16_bits(a.w) << 16));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) y[j] = bf16_bits(o[j]);
      }
    }
  }
  __syncwarp();
  if (split > 1) cluster_sync();   // the others have read this CTA's part
  if (threadIdx.x == 0 && *err) set_status(&g_fp8_status, *err);
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// ---------------------------------------------------------------------------
// Many rows: CTA pairs.  Rows of a are the M side (128 per CTA, 256 per pair),
// weights the N side, half of them in each CTA's shared memory:
// tcgen05.mma.cta_group::2 reads both halves, so the pair's tile has half the
// operand traffic of two separate ones.  Persistent: one pair per two SMs
// walks the tiles, the ring running ahead into the next tile.
//   warp 0: TMA producer (each CTA its own halves, into the leader's barrier)
//   warp 1: MMA issuer (leader CTA), or passing free accumulators on to it
//   warp 2: scales (the rows of this CTA, the weights' blocks)
//   warps 4-11: epilogue, 32 rows x 128 columns each
// E8M0: one accumulator of 256 columns, released as soon as the epilogue has it
// in registers.  fp32 scales: two of 256 columns, a k-tile each; an epilogue
// thread has one row of one 128-block of N, so a partial sum takes one
// multiply-add.  (Four accumulators of 128 columns, whose MMAs read a's tile
// from shared memory twice as often, took 0.67 us per k-tile of 256 x 256; two
// of 256 first took 0.66 and take 0.54 with the waits tested ahead.)
// ---------------------------------------------------------------------------
constexpr int L_TM = 256;
constexpr int L_SF_COL = 256;                    // 12 columns of scales, twice
constexpr int L_RASTER = 8;                      // m-tiles walked together: their operands meet in L2
constexpr int L_OUT_BYTES = 32 * 128;            // per epilogue warp: 32 rows x 128 bytes

constexpr int L_TN = 256;
constexpr int L_A_BYTES = 128 * F_BK;
constexpr int L_STAGE_BYTES = L_A_BYTES + L_TN / 2 * F_BK;

template <bool E8>
struct LCfg {
  static constexpr int EPI_WARPS = 8;
  static constexpr int COLS = L_TN / (EPI_WARPS / 4);       // accumulator columns per epilogue warp
  static constexpr int THREADS = (F_EPI_WARP0 + EPI_WARPS) * 32;
  static constexpr int NACC = E8 ? 1 : 2;
  static constexpr int STAGES = 5;
  // E8M0: scale atoms of 128 rows of a and two blocks of b; fp32: as * bs of
  // four k-tiles, two blocks of N and 128 rows
  static constexpr int SLOT_BYTES = E8 ? 3 * 512 : F_GROUP * 2 * 128 * 4;
  static constexpr int BARS = 2 * STAGES + 2 * F_SLOTS + 2 * NACC + 1;
  static constexpr int SMEM =
      STAGES * L_STAGE_BYTES + EPI_WARPS * L_OUT_BYTES + F_SLOTS * SLOT_BYTES + BARS * 8 + 16 + 1024;
  // fp32: the four issuing warps give registers to the epilogue (128 sums and
  // 64 values on their way from TMEM per thread); the shares add up to no more
  // than the block is launched with
  static constexpr int REGS_ISSUE = 56, REGS_EPI = 224, REGS_LAUNCH = 168;
  static_assert(REGS_ISSUE * 128 + REGS_EPI * EPI_WARPS * 32 <= REGS_LAUNCH * THREADS, "register split");
  static_assert(SMEM >= F_MIN_SMEM && alone_on_sm(SMEM), "takes all 512 TMEM columns");
};

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

// The 32 x COLS results of an epilogue warp, a lane per row, to rows m0 .. of y
// and columns n0 .., 128 bytes of each row at a time through the warp's staging
// buffer (16-byte units swizzled by row): every store then covers whole
// 128-byte lines of four rows instead of 16 bytes of 32.
template <int COLS>
__device__ __forceinline__ void store_tile(const float (&acc)[COLS], uint8_t* buf, const Fp8Params& p, int64_t m0,
                                           int64_t n0, int lane) {
  const int esz = p.out_f32 ? 4 : 2, per = 128 / esz;   // columns per pass
#pragma unroll
  for (int pass = 0; pass < COLS / 32; ++pass) {
    if (pass >= COLS / 64 && !p.out_f32) break;
    const int64_t nc = n0 + pass * per;
    if (nc >= p.N) break;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      uint4 o;
      if (p.out_f32) {
        const int c = pass * 32 + u * 4;
        o = make_uint4(__float_as_uint(acc[c]), __float_as_uint(acc[c + 1]), __float_as_uint(acc[c + 2]),
                       __float_as_uint(acc[c + 3]));
      } else {
        const int c = pass * 64 % COLS + u * 8;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = bf16_bits(acc[c + 2 * j]) | ((uint32_t)bf16_bits(acc[c + 2 * j + 1]) << 16);
        o = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(buf + lane * 128 + ((u ^ (lane & 7)) << 4)) = o;
    }
    __syncwarp();
    if (p.vec_y && nc + per <= p.N) {
      uint8_t* y = static_cast<uint8_t*>(p.y) + nc * esz + (lane & 7) * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        const uint4 o = *reinterpret_cast<const uint4*>(buf + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        if (m0 + r < p.M) *reinterpret_cast<uint4*>(y + (m0 + r) * p.ldy * esz) = o;
      }
    } else {
      for (int r = 0; r < 32 && m0 + r < p.M; ++r) {
        for (int c = lane; c < per && nc + c < p.N; c += 32) {
          const uint8_t* o = buf + r * 128 + (((c * esz >> 4) ^ (r & 7)) << 4) + (c * esz & 15);
          if (p.out_f32) static_cast<float*>(p.y)[(m0 + r) * p.ldy + nc + c] = *reinterpret_cast<const float*>(o);
          else static_cast<uint16_t*>(p.y)[(m0 + r) * p.ldy + nc + c] = *reinterpret_cast<const uint16_t*>(o);
        }
      }
    }
    __syncwarp();
  }
}

template <bool E8, bool B_MN>
__global__ void __launch_bounds__(LCfg<E8>::THREADS, 1)
    fp8_matmul_pair_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                           const Fp8Params p, const int mt, const int nt) {
  using C = LCfg<E8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* outs = smem + C::STAGES * L_STAGE_BYTES;
  uint8_t* slots = outs + C::EPI_WARPS * L_OUT_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(slots + F_SLOTS * C::SLOT_BYTES);   // leader's: both CTAs' bytes
  uint64_t* empty = full + C::STAGES;
  uint64_t* sfull = empty + C::STAGES;      // E8M0, leader's: one arrival per CTA
  uint64_t* sempty = sfull + F_SLOTS;
  uint64_t* accfull = sempty + F_SLOTS;
  uint64_t* accempty = accfull + C::NACC;   // this CTA's epilogue warps; leader's: and the other CTA's warp 1
  uint64_t* drain = accempty + C::NACC;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  int* err = reinterpret_cast<int*>(tmem_holder + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp-uniform
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int nkt = p.kb, ngr = (nkt + F_GROUP - 1) / F_GROUP, tiles = mt * nt;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < F_SLOTS; ++s) {
      mbar_init(&sfull[s], E8 ? 2 : 1);
      mbar_init(&sempty[s], E8 ? 1 : C::EPI_WARPS);
    }
    for (int s = 0; s < C::NACC; ++s) {
      mbar_init(&accfull[s], 1);
      mbar_init(&accempty[s], C::EPI_WARPS + (rank == 0 ? 1 : 0));
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

  if constexpr (!E8) {
    if (warp < F_EPI_WARP0) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_ISSUE));
  }
  if (warp == 0) {
    const uint64_t pol = policy_evict_normal();
    int it = 0;
    bool ok = true;
    Ring<C::STAGES> ring;
    for (int t = pair; t < tiles && ok; t += pairs) {
      const LTile tl = large_tile(t, mt, nt);
      const int m0 = (int)(tl.m0 + rank * 128), n0 = tl.n0 + (int)rank * 128;
      for (int kt = 0; kt < nkt; ++kt, ++it, ring.next()) {
        const int s = ring.s;
        if (it >= C::STAGES && !(ok = warp_wait(&empty[s], ring.ph ^ 1u, err))) break;
        uint8_t* st = smem + s * L_STAGE_BYTES;
        const uint32_t bar = map_rank(&full[s], 0);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(&full[s], 2 * L_STAGE_BYTES);
          tma_load_2d_pair(st, &tmX, bar, kt * F_BK, m0, pol);
          if constexpr (B_MN) tma_load_2d_pair(st + L_A_BYTES, &tmW, bar, n0, kt * F_BK, pol);
          else tma_load_2d_pair(st + L_A_BYTES, &tmW, bar, kt * F_BK, n0, pol);
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
      constexpr uint32_t B_STEP = B_MN ? (32 * 128) >> 4 : 2u;   // 32 of K: 32 rows of 128 B, or 32 B of a row
      int it = 0, grp = 0, ti = 0;
      bool ok = true;
      Ring<C::STAGES> ring;
      for (int t = pair; t < tiles && ok; t += pairs, ++ti) {
        if constexpr (E8) {
          if (ti > 0 && !(ok = warp_wait(&accempty[0], (uint32_t)(ti - 1) & 1u, err))) break;
        }
        for (int kt = 0; kt < nkt; ++kt, ++it, ring.next()) {
          const int s = ring.s;
          if (!(ok = warp_wait(&full[s], ring.ph, err))) break;
          const uint32_t aA = smem_u32(smem + s * L_STAGE_BYTES);
          const uint64_t dA = desc_sw128(aA), dB = desc_sw128(aA + L_A_BYTES);
          if constexpr (E8) {
            const bool fresh = kt % F_GROUP == 0;
            if (fresh && kt > 0) ++grp;
            const int slot = grp % F_SLOTS;
            const uint32_t sfa = tmem + L_SF_COL + 16 * (grp & 1), sfb = sfa + 4;
            if (fresh && !(ok = warp_wait<true>(&sfull[slot], (uint32_t)(grp / F_SLOTS) & 1u, err))) break;
            tc_fence_after();
            const uint32_t id = kt % F_GROUP, sel = id << 30;
            const uint32_t idesc = idesc_mxf8_pair(L_TN, id) | mn;
            if (elect_one()) {
              if (fresh) {
                const uint32_t sl = smem_u32(slots + slot * C::SLOT_BYTES);
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
            const uint32_t idesc = idesc_f8(L_TM, L_TN) | mn;
            if (elect_one()) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                tc_mma_f8_pair(tmem + ab * L_TN, dA + 2u * j, dB + B_STEP * j, idesc, j != 0 ? 1u : 0u);
              tc_commit_pair(&empty[s]);   // the stage is free and the accumulator is full
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
    } else {
      // passes this CTA's free accumulators on to the leader: the epilogue
      // warps then only arrive at home (a remote arrival holds its warp up)
      const int mine = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0, uses = E8 ? mine : mine * nkt;
      for (int u = 0; u < uses; ++u) {
        const int ab = u % C::NACC;
        if (!warp_wait(&accempty[ab], (uint32_t)(u / C::NACC) & 1u, err)) break;
        // the epilogue's tcgen05.ld -> fence, arrival | wait, fence -> fence,
        // arrival | wait, fence -> the leader's MMA: every link has its fences
        tc_fence_after();
        tc_fence_before();
        if (lane == 0) mbar_arrive_cluster_relaxed(map_rank(&accempty[ab], 0));
        __syncwarp();
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
                                 gr * F_GROUP + lane, nkt, (int64_t)(nb0 + j) * 128 < p.N);
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
            uint8_t* sl = slots + slot * C::SLOT_BYTES;
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
    } else {
      int grp = 0;
      bool ok = true;
      float cur[4][F_GROUP], nxt[4][F_GROUP], sb[2] = {};
      auto load = [&](int t, int kt) {
        const int64_t m0 = large_tile(t, mt, nt).m0 + rank * 128;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t m = m0 + lane + 32 * j;
          scale_row(static_cast<const float*>(p.as) + (m < p.M ? m * nkt : 0), kt, nkt, p.vec, m < p.M, nxt[j]);
        }
      };
      if (pair < tiles) load(pair, 0);
      for (int t = pair; t < tiles && ok; t += pairs) {
        const int nb0 = large_tile(t, mt, nt).n0 / 128;
        for (int gr = 0; gr < ngr; ++gr, ++grp) {
          const int slot = grp % F_SLOTS, kt0 = gr * F_GROUP;
          if (gr % 8 == 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              sb[h] = (int64_t)(nb0 + h) * 128 < p.N && kt0 + lane < nkt
                          ? __ldcg(static_cast<const float*>(p.bs) + (int64_t)(kt0 + lane) * p.bs_k +
                                   (int64_t)(nb0 + h) * p.bs_n)
                          : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < F_GROUP; ++i) cur[j][i] = nxt[j][i];
          if (gr + 1 < ngr) load(t, kt0 + F_GROUP);
          else if (t + pairs < tiles) load(t + pairs, 0);
          if (grp >= F_SLOTS && !(ok = warp_wait(&sempty[slot], (uint32_t)(grp / F_SLOTS - 1) & 1u, err))) break;
          float* f = reinterpret_cast<float*>(slots + slot * C::SLOT_BYTES) + lane;   // [k-tile][block][row]
#pragma unroll
          for (int i = 0; i < F_GROUP; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float s = __shfl_sync(0xffffffffu, sb[h], gr % 8 * 4 + i);
#pragma unroll
              for (int j = 0; j < 4; ++j) f[(i * 2 + h) * 128 + 32 * j] = cur[j][i] * s;
            }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sfull[slot]);
        }
      }
    }
  } else if (warp >= F_EPI_WARP0) {
    if constexpr (!E8) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_EPI));
    const int q = warp & 3, c0 = ((warp - F_EPI_WARP0) >> 2) * C::COLS;
    const uint32_t trow = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c0;
    uint8_t* buf = outs + (warp - F_EPI_WARP0) * L_OUT_BYTES;
    int it = 0, ti = 0, grp = 0;
    bool ok = true;
    Ring<C::STAGES> ring;
    for (int t = pair; t < tiles && ok; t += pairs, ++ti) {
      const LTile tl = large_tile(t, mt, nt);
      const int64_t m0 = tl.m0 + rank * 128 + q * 32, n0 = tl.n0 + c0;
      float acc[C::COLS];
      if constexpr (E8) {
        if (!(ok = warp_wait(&accfull[0], (uint32_t)ti & 1u, err))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < C::COLS; c += 16) tmem_ld16(trow + c, acc + c);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&accempty[0]);
      } else {
#pragma unroll
        for (int c = 0; c < C::COLS; ++c) acc[c] = 0.f;
        bool ready = false;
        const float* sc = reinterpret_cast<const float*>(slots) + (c0 / 128) * 128 + q * 32 + lane;
        for (int kt = 0; kt < nkt; ++kt, ++it) {
          const int ab = it & 1, slot = grp % F_SLOTS;
          if (kt % F_GROUP == 0 && !(ok = warp_wait(&sfull[slot], (uint32_t)(grp / F_SLOTS) & 1u, err))) break;
          const float s = sc[slot * (C::SLOT_BYTES / 4) + kt % F_GROUP * 256];
          if (!ready && !(ok = warp_wait(&empty[ring.s], ring.ph, err))) break;
          ring.next();
          tc_fence_after();
          uint32_t next = 0;
          const uint32_t src = trow + (uint32_t)(ab * L_TN);
#pragma unroll
          for (int c = 0; c < C::COLS; c += 64) {
            float v[64];
#pragma unroll
            for (int j = 0; j < 64; j += 16) tmem_ld16(src + (uint32_t)(c + j), v + j);
            tc_wait_ld();
            if (c == C::COLS - 64) {   // the accumulator is in registers
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&accempty[ab]);
              next = bar_test(&empty[ring.s], ring.ph);
            }
#pragma unroll
            for (int j = 0; j < 64; ++j) acc[c + j] = fmaf(v[j], s, acc[c + j]);
          }
          ready = __all_sync(0xffffffffu, next != 0u);
          if (kt % F_GROUP == F_GROUP - 1 || kt == nkt - 1) {
            if (lane == 0) mbar_arrive(&sempty[slot]);
            ++grp;
          }
        }
        if (!ok) break;
      }
      store_tile(acc, buf, p, m0, n0, lane);
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

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// What a kernel needs once per device: its shared memory opt-in and, with
// setmaxnreg (regs > 0), a look at the registers it is launched with:
// setmaxnreg.inc waits for registers that a smaller launch would not have.
template <typename K>
int prepare_kernel(K k, int smem, int regs, int dev, std::atomic<uint64_t>& done) {
  const uint64_t bit = dev < 64 ? UINT64_C(1) << dev : 0;
  if (done.load(std::memory_order_acquire) & bit) return DSV4_OK;
  DSV4_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (regs) {
    cudaFuncAttributes fa;
    DSV4_CUDA_CHECK(cudaFuncGetAttributes(&fa, k));
    if ((fa.numRegs + 7) / 8 * 8 < regs) return fail(DSV4_ECUDA, "fp8_matmul: built with too few registers per thread");
  }
  done.fetch_or(bit, std::memory_order_release);
  return DSV4_OK;
}
int sm_count(int dev) {
  static std::atomic<int> known[64];
  int n = dev < 64 ? known[dev].load(std::memory_order_relaxed) : 0;
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && dev < 64)
    known[dev].store(n, std::memory_order_relaxed);
  return n;
}
// k-tiles per CTA of a cluster of `want`: a multiple of four, a word of E8M0 scales.
int k_share(int kb, int want) { return ((kb + want - 1) / want + 3) / 4 * 4; }

template <typename K, typename... Args>
int launch_cluster(K k, dim3 grid, int threads, int smem, dim3 cluster, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster.x;
  attr[1].val.clusterDim.y = cluster.y;
  attr[1].val.clusterDim.z = cluster.z;
  cfg.attrs = attr;
  cfg.numAttrs = cluster.x * cluster.z > 1 ? 2 : 1;
  DSV4_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, args...));
  return DSV4_OK;
}

// The largest number of CTAs per cluster, up to `want`, with which all `tiles`
// clusters are on the GPU at once, `resident` CTAs per SM.  (The CTAs of a
// cluster share a GPC: at one CTA per SM, 15 clusters of 8 fit 148 SMs, and the
// 16th doubled the time of 64 x 2048 x 4096 with fp32 scales, 7.5 to 12 us.)
// The occupancy query answers for one CTA per SM: it is asked with the largest
// shared memory.
template <typename K>
int fitting_cluster(K k, int threads, int resident, int64_t tiles, int want, int dev, std::atomic<int> (&known)[64][9]) {
  for (; want > 1; --want) {
    int n = dev < 64 ? known[dev][want].load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, 1, (unsigned)want);
      cfg.blockDim = dim3(threads);
      cfg.dynamicSmemBytes = F_MAX_SMEM;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = (unsigned)want;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&n, k, &cfg) != cudaSuccess) {
        cudaGetLastError();
        n = 0;
      }
      if (n == 0) n = -1;
      if (dev < 64) known[dev][want].store(n, std::memory_order_relaxed);
    }
    if ((int64_t)n * resident >= tiles) break;
  }
  return want;
}
// The few-row kernel made ready on `dev`, and *cluster reduced to the size that fits.
template <int BN, bool E8, bool A_MN, bool FUSE>
int fit_small(int64_t tiles, int dev, int* cluster) {
  using C = FCfg<BN, E8, FUSE>;
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> fits[64][9];
  auto k = fp8_matmul_kernel<BN, E8, A_MN, FUSE>;
  if (int rc = prepare_kernel(k, F_MAX_SMEM, 0, dev, done)) return rc;
  *cluster = fitting_cluster(k, C::THREADS, C::RESIDENT, tiles, *cluster, dev, fits);
  return DSV4_OK;
}
template <int BN>
int fit_fused(bool e8, bool a_mn, int64_t tiles, int dev, int* cluster) {
  if (e8) return a_mn ? fit_small<BN, true, true, true>(tiles, dev, cluster) : fit_small<BN, true, false, true>(tiles, dev, cluster);
  return a_mn ? fit_small<BN, false, true, true>(tiles, dev, cluster) : fit_small<BN, false, false, true>(tiles, dev, cluster);
}
template <int BN, bool E8, bool A_MN, bool FUSE>
int launch_small(const CUtensorMap& tw, const CUtensorMap& tx, const Fp8Params& p, int want, int dev, cudaStream_t st) {
  using C = FCfg<BN, E8, FUSE>;
  auto k = fp8_matmul_kernel<BN, E8, A_MN, FUSE>;
  const int64_t nt = (p.N + F_BM - 1) / F_BM, mt = (p.M + BN - 1) / BN;
  if (int rc = fit_small<BN, E8, A_MN, FUSE>(nt * mt, dev, &want)) return rc;
  const int per = k_share(p.kb, want);
  const unsigned split = (unsigned)((p.kb + per - 1) / per);
  return launch_cluster(k, dim3((unsigned)nt, (unsigned)mt, split), C::THREADS, C::SMEM, dim3(1, 1, split), st, tw, tx,
                        p, per);
}
template <int BN, bool FUSE>
int launch_small(bool e8, bool a_mn, const CUtensorMap& tw, const CUtensorMap& tx, const Fp8Params& p, int want,
                 int dev, cudaStream_t st) {
  if (e8) return a_mn ? launch_small<BN, true, true, FUSE>(tw, tx, p, want, dev, st) : launch_small<BN, true, false, FUSE>(tw, tx, p, want, dev, st);
  return a_mn ? launch_small<BN, false, true, FUSE>(tw, tx, p, want, dev, st) : launch_small<BN, false, false, FUSE>(tw, tx, p, want, dev, st);
}
template <bool E8, bool B_MN>
int launch_pair(const CUtensorMap& tx, const CUtensorMap& tw, const Fp8Params& p, int sms, int dev, cudaStream_t st) {
  using C = LCfg<E8>;
  static std::atomic<uint64_t> done{0};
  if (int rc = prepare_kernel(fp8_matmul_pair_kernel<E8, B_MN>, C::SMEM, E8 ? 0 : C::REGS_LAUNCH, dev, done)) return rc;
  const int64_t mt = (p.M + L_TM - 1) / L_TM, nt = (p.N + L_TN - 1) / L_TN;
  const unsigned pairs = (unsigned)std::min<int64_t>(mt * nt, sms / 2);
  return launch_cluster(fp8_matmul_pair_kernel<E8, B_MN>, dim3(2 * pairs), C::THREADS, C::SMEM, dim3(2, 1, 1), st, tx,
                        tw, p, (int)mt, (int)nt);
}

// Kernel and tile of a product.
struct Fp8Shape {
  bool pair;
  int bn;     // rows of a per CTA's load
  int split;  // CTAs that share K
};
// Few rows while the 128 x 128 tiles fit the SMs once: the cluster size then
// fills the SMs with shares of K.  Measured (us, few rows | pairs), E8M0:
// 300 x 1001 x 2000: 8.0 | 21.3, 512 x 4096 x 2048 (128 tiles): 10.9 | 11.3,
// 1024 x 4096 x 4096 (256 tiles): 23.1 | 18.5, 2048^3: 14.6 | 12.7; fp32
// scales: 8.1 | 23.8, 12.2 | 14.5, 35.9 | 24.7, 22.9 | 16.0.  Up to 128 of N a
// pair's 256-wide tile would be half empty.
Fp8Shape fp8_shape(int64_t m, int64_t n, int sms) {
  Fp8Shape c = {};
  c.bn = m <= 16 ? 16 : (m <= 32 ? 32 : (m <= 64 ? 64 : 128));
  const int64_t tiles = ((n + F_BM - 1) / F_BM) * ((m + c.bn - 1) / c.bn);
  c.pair = n > 128 && m > 128 && tiles > sms;
  c.split = (int)std::max<int64_t>(1, std::min<int64_t>(8, sms / tiles));
  return c;
}

}  // namespace

static int weight_map(CUtensorMap* m, const uint8_t* b, int64_t ldb, bool trans_b, int64_t n, int64_t k) {
  const uint64_t d[2] = {(uint64_t)(trans_b ? k : n), (uint64_t)(trans_b ? n : k)}, s[1] = {(uint64_t)ldb};
  const uint32_t box[2] = {128, 128};
  return make_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)b, d, s, box, "fp8 weight");
}

static int fp8_matmul_run(const uint8_t* a, int64_t lda, const void* as, const uint8_t* b, int64_t ldb, const void* bs,
                          int scale_type, bool trans_b, int64_t m, int64_t n, int64_t k, void* y, int64_t ldy,
                          int out_dtype, int dev, cudaStream_t st) {
  const int64_t kb = (k + F_BK - 1) / F_BK, nb = (n + F_BK - 1) / F_BK;
  const bool e8 = scale_type == DSV4_SCALE_E8M0, f32 = out_dtype == DSV4_DT_FP32;
  const int sms = sm_count(dev);
  if (sms <= 0) return fail(DSV4_ECUDA, "fp8_matmul: no SM count");
  const Fp8Shape c = fp8_shape(m, n, sms);
  Fp8Params p = {};
  p.as = as, p.bs = bs, p.bs_k = trans_b ? 1 : nb, p.bs_n = trans_b ? kb : 1;
  p.y = y, p.ldy = ldy, p.M = m, p.N = n, p.kb = (int)kb;
  p.vec = scale_vec(as, (int)kb, e8);
  p.out_f32 = f32;
  // 16-byte stores of the pair kernel, four elements of the other
  const int al = c.pair ? 16 : (f32 ? 16 : 8);
  p.vec_y = (uintptr_t)y % al == 0 && ldy * (f32 ? 4 : 2) % al == 0;
  CUtensorMap tw, tx;
  if (int rc = weight_map(&tw, b, ldb, trans_b, n, k)) return rc;
  const uint64_t dx[2] = {(uint64_t)k, (uint64_t)m}, sx[1] = {(uint64_t)lda};
  const uint32_t bx[2] = {F_BK, (uint32_t)(c.pair ? 128 : c.bn)};
  if (int rc = make_map(&tx, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)a, dx, sx, bx, "fp8_matmul a")) return rc;
  if (c.pair) {
    if (e8) return trans_b ? launch_pair<true, false>(tx, tw, p, sms, dev, st) : launch_pair<true, true>(tx, tw, p, sms, dev, st);
    return trans_b ? launch_pair<false, false>(tx, tw, p, sms, dev, st) : launch_pair<false, true>(tx, tw, p, sms, dev, st);
  }
  switch (c.bn) {
    case 16: return launch_small<16, false>(e8, !trans_b, tw, tx, p, c.split, dev, st);
    case 32: return launch_small<32, false>(e8, !trans_b, tw, tx, p, c.split, dev, st);
    case 64: return launch_small<64, false>(e8, !trans_b, tw, tx, p, c.split, dev, st);
    default: return launch_small<128, false>(e8, !trans_b, tw, tx, p, c.split, dev, st);
  }
}

// Whether a linear layer quantises its rows in the product's launch.  Every
// CTA then quantises its share of K again, so that share has to be short: the
// second launch costs about 2 us, a k-tile 0.15 us (16 rows) to 0.4 us (64
// rows), more with fp32 scales.  Measured (us, one launch | two; E8M0): 1 x
// 4096 x 4096: 6.4 | 8.2, 64 x 4096 x 2048 (4 k-tiles): 7.7 | 8.1, 64 x 8192 x
// 8192 (32 k-tiles): 28 | 17; fp32: 1 x 2048 x 4096: 6.3 | 6.6, 64 x 4096 x
// 2048: 10.4 | 8.5.
// Only where the fused kernel's clusters fit at the full size: the other one,
// of which as many CTAs or more share an SM, then splits K the same way, and
// the sums have the same order.
static bool linear_fuses(const void* x, int x_dtype, int64_t ldx, int64_t m, int64_t n, int64_t k, bool e8, bool a_mn,
                         int dev) {
  const int sms = sm_count(dev);
  if (sms <= 0 || m > 64 || x_dtype != DSV4_DT_BF16 || k % 8 || (uintptr_t)x % 16 || ldx % 8) return false;
  const Fp8Shape c = fp8_shape(m, n, sms);
  const int per = k_share((int)((k + F_BK - 1) / F_BK), c.split);
  // above 32 rows one CTA fits an SM, and few clusters of more than four do
  if (m <= 16 ? per > (e8 ? 8 : 4) : !(e8 && per <= 4 && (m <= 32 || c.split <= 4))) return false;
  const int64_t tiles = (n + F_BM - 1) / F_BM;
  int fits = c.split;
  const int rc = c.bn == 16   ? fit_fused<16>(e8, a_mn, tiles, dev, &fits)
                 : c.bn == 32 ? fit_fused<32>(e8, a_mn, tiles, dev, &fits)
                              : fit_fused<64>(e8, a_mn, tiles, dev, &fits);
  return rc == DSV4_OK && fits == c.split;
}
static int fp8_linear_fused(const void* x, int64_t ldx, const uint8_t* w, int64_t ldw, const void* ws,
                            int scale_type, bool trans_w, int64_t m, int64_t n, int64_t k, void* y, int64_t ldy,
                            int dev, cudaStream_t st) {
  const int64_t kb = (k + F_BK - 1) / F_BK, nb = (n + F_BK - 1) / F_BK;
  const bool e8 = scale_type == DSV4_SCALE_E8M0;
  const int sms = sm_count(dev);
  if (sms <= 0) return fail(DSV4_ECUDA, "fp8_linear: no SM count");
  const Fp8Shape c = fp8_shape(m, n, sms);
  Fp8Params p = {};
  p.bs = ws, p.bs_k = trans_w ? 1 : nb, p.bs_n = trans_w ? kb : 1;
  p.y = y, p.ldy = ldy, p.M = m, p.N = n, p.kb = (int)kb;
  p.vec_y = (uintptr_t)y % 8 == 0 && ldy % 4 == 0;
  p.x = static_cast<const uint16_t*>(x), p.ldx = ldx, p.K = k;
  CUtensorMap tw;
  if (int rc = weight_map(&tw, w, ldw, trans_w, n, k)) return rc;
  switch (c.bn) {
    case 16: return launch_small<16, true>(e8, !trans_w, tw, tw, p, c.split, dev, st);
    case 32: return launch_small<32, true>(e8, !trans_w, tw, tw, p, c.split, dev, st);
    default: return launch_small<64, true>(e8, !trans_w, tw, tw, p, c.split, dev, st);
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
  DSV4_CHECK_ARG(m <= F_MAX_M && n <= 0x7fffff00 && k <= 0x7fffff00 &&
                     ((m + 127) / 128) * ((n + 127) / 128) <= 0x7fffffff,
                 "a size is too large");
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
                              dev.device, (cudaStream_t)stream))
    return rc;
  DSV4_API_END
}

// Codes (rows of k bytes, padded to 16), then the scales.
static int64_t linear_scale_offset(int64_t m, int64_t k) { return m * ((k + 15) / 16 * 16); }
static int64_t linear_workspace(int64_t m, int64_t k, int scale_type) {
  return linear_scale_offset(m, k) + m * ((k + 127) / 128) * (scale_type == DSV4_SCALE_E8M0 ? 1 : 4);
}

extern "C" int64_t dsv4_fp8_linear_workspace_bytes(int64_t m, int64_t k, int32_t scale_type) {
  if (m < 0 || k <= 0 || k > 0x7fffff00 || m > F_MAX_M ||
      (scale_type != DSV4_SCALE_E8M0 && scale_type != DSV4_SCALE_FP32))
    return DSV4_EINVAL;
  return linear_workspace(m, k, scale_type);
}

extern "C" int dsv4_fp8_linear(const void* x, int32_t x_dtype, int64_t ldx, const uint8_t* w, int64_t ldw,
                               const void* w_scale, int32_t scale_type, int32_t trans_w, int64_t m, int64_t n,
                               int64_t k, void* y, int64_t ldy, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  DSV4_API_BEGIN
  DSV4_CHECK_ARG(x_dtype == DSV4_DT_BF16 || x_dtype == DSV4_DT_FP32, "x must be bf16 or fp32");
  DSV4_CHECK_ARG(scale_type == DSV4_SCALE_E8M0 || scale_type == DSV4_SCALE_FP32, "scales must be E8M0 or fp32");
  DSV4_CHECK_ARG(m >= 0 && n >= 0 && k > 0, "m and n must be >= 0 and k > 0");
  DSV4_CHECK_ARG(m <= F_MAX_M && n <= 0x7fffff00 && k <= 0x7fffff00 &&
                     ((m + 127) / 128) * ((n + 127) / 128) <= 0x7fffffff,
                 "a size is too large");
  DSV4_CHECK_ARG(ldx >= k && ldw >= (trans_w ? k : n) && ldy >= n, "a row stride is smaller than the row");
  if (m == 0 || n == 0) return DSV4_OK;
  DSV4_CHECK_ARG(x && w && w_scale && y && workspace, "null pointer");
  DSV4_CHECK_ARG((uintptr_t)w % 16 == 0 && ldw % 16 == 0, "w must start on 16 bytes, with a row stride a multiple of 16");
  DSV4_CHECK_ARG((uintptr_t)x % (x_dtype == DSV4_DT_FP32 ? 4 : 2) == 0 &&
                     (uintptr_t)y % (x_dtype == DSV4_DT_FP32 ? 4 : 2) == 0 &&
                     (scale_type == DSV4_SCALE_E8M0 || (uintptr_t)w_scale % 4 == 0),
                 "misaligned x, y or scales");
  DSV4_CHECK_ARG((uintptr_t)workspace % 16 == 0 && workspace_bytes >= linear_workspace(m, k, scale_type),
                 "the workspace is too small or not 16-byte aligned");
  DeviceScope dev;
  if (int rc = dev.enter(x)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (linear_fuses(x, x_dtype, ldx, m, n, k, scale_type == DSV4_SCALE_E8M0, trans_w == 0, dev.device))
    return fp8_linear_fused(x, ldx, w, ldw, w_scale, scale_type, trans_w != 0, m, n, k, y, ldy, dev.device, st);
  uint8_t* q = static_cast<uint8_t*>(workspace);
  uint8_t* s = q + linear_scale_offset(m, k);
  const int64_t ldq = (k + 15) / 16 * 16;
  if (int rc = act_quant_fp8_launch(x, x_dtype, m, k, ldx, q, ldq, s, scale_type, st)) return rc;
  if (int rc = fp8_matmul_run(q, ldq, s, w, ldw, w_scale, scale_type, trans_w != 0, m, n, k, y, ldy, x_dtype,
                              dev.device, st))
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
