// Load balance loss of a router, the per-expert counts and the gradient of the
// logits (no counterpart in the reference, whose router only serves; the score
// functions are those of OffloadDeepseekV4MoE._route, deepseek_v4.py:126-131).
//
// With scores s = score(logits), p = s / sum_e s, and per sequence q its
// tokens n_q, picks c_q[e] of expert e, and f_q[e] = c_q[e] E / sum_e c_q[e]:
//   loss = alpha / Q * sum_q sum_e f_q[e] * mean_t p[t, e]      (Q sequences with tokens)
//   dlogit_j = up * alpha / Q * p_j r_j (g_j - d_t),   g = f_q / n_q,  d_t = sum_e g_e p_e
//   r = 1 (softmax), 1 - s (sigmoid), sigma / (2 softplus) (sqrtsoftplus).
// The counts depend on the picks alone, so they come first and the loss is
// then the sum of one number per token, d_t: no [sequence, expert] sums of
// probabilities are kept.  The forward stores (row maximum, 1 / sum, d_t) per
// token, and the backward is one pass without reductions.
//
// Counts are integer atomics (any order gives the same numbers), the d_t are
// added in double in a fixed order, so results do not depend on scheduling.
// Bound: HBM, the logits once forward, once backward, the gradient once.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

namespace dsv4 {
namespace {

constexpr int BL_THREADS = 256;          // 8 warps
constexpr int BL_WARPS = BL_THREADS / 32;
constexpr int BL_TOK = 8;                // tokens per warp: g stays in registers
constexpr int BL_SMALL_THREADS = 512;    // the one-CTA forward
constexpr int BL_MAX_E = 1024;
constexpr int64_t BL_ONE_CTA_TOKENS = 256;   // one launch up to here

// Saved state of one forward (the caller's buffer), then scratch.
struct BalanceLayout {
  int64_t head;      // int[4]: sequences with tokens, CTAs done, unused, unused
  int64_t info;      // int[S][2]: tokens, picks
  int64_t hist;      // int[S][E]
  int64_t rows;      // float4[T]: row maximum, 1 / sum (< 0: no part in the loss), d_t, sequence bits
  int64_t part;      // double[CTAs]
  int64_t bytes;
};
__host__ __device__ inline int64_t al16(int64_t v) { return (v + 15) / 16 * 16; }
inline int64_t bl_ctas(int64_t T) { return (T + BL_WARPS * BL_TOK - 1) / (BL_WARPS * BL_TOK); }
inline BalanceLayout bl_layout(int64_t T, int64_t E, int64_t S) {
  BalanceLayout l;
  l.head = 0;
  l.info = 16;
  l.hist = l.info + al16(S * 8);
  l.rows = l.hist + al16(S * E * 4);
  l.part = l.rows + T * 16;
  l.bytes = l.part + al16(std::max<int64_t>(bl_ctas(T), BL_SMALL_THREADS / 32) * 8);
  return l;
}

struct BalanceParams {
  const void* logits;
  int64_t T;
  int E, k, S, score;
  const int32_t* idx;
  const int32_t* off;     // [S + 1] or null (one sequence)
  float alpha;
  float* loss;
  int32_t* counts;
  int* head;
  int2* info;
  int* hist;
  float4* rows;
  double* part;
  int* status;
  const float* up;
  void* dlogits;
};

// The sequence of row t, -1 for a row in none (binary search).
__device__ __forceinline__ int seq_of(const BalanceParams& p, int64_t t) {
  if (!p.off) return 0;
  int lo = 0, hi = p.S + 1;   // number of offsets <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)p.off[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1 < p.S ? lo - 1 : -1;
}

// Offsets that descend or leave [0, T] are reported (every row still finds
// some sequence in [0, S), so nothing is read or written out of range).
__device__ void check_offsets(const BalanceParams& p) {
  if (!p.off) return;
  for (int i = threadIdx.x; i <= p.S; i += blockDim.x) {
    const int32_t v = __ldcg(&p.off[i]);
    if (v < 0 || v > p.T || (i > 0 && v < __ldcg(&p.off[i - 1]))) set_status(p.status, DSV4_EINVAL);
  }
}

// Counts of the picks of rows [t0, t1) by one CTA, one thread per token,
// straight into the global histogram.
__device__ void count_rows(const BalanceParams& p, int64_t t0, int64_t t1) {
  const int lane = threadIdx.x & 31;
  for (int64_t t = t0 + threadIdx.x; t - lane < t1; t += blockDim.x) {
    const bool in = t < t1;
    const int s = in ? seq_of(p, t) : -1;
    int picks = 0;
    for (int j = 0; j < p.k; ++j) {
      int e = -1;
      if (s >= 0) {
        e = __ldcg(&p.idx[t * p.k + j]);
        if (e < -1 || e >= p.E) {
          set_status(p.status, DSV4_EINVAL);
          e = -1;
        }
      }
      if (e >= 0) {
        atomicAdd(&p.hist[(int64_t)s * p.E + e], 1);
        ++picks;
      }
    }
    // tokens and picks per sequence: one add per group of lanes with the same sequence
    const int key = picks ? s : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, key);
    int sum = 0;
    for (uint32_t r = same; r; r &= r - 1) sum += __shfl_sync(same, picks, __ffs(r) - 1);
    if (key >= 0 && lane == __ffs(same) - 1) {
      atomicAdd(&p.info[s].x, __popc(same));
      atomicAdd(&p.info[s].y, sum);
    }
  }
}

__device__ __forceinline__ float ld_logit(const float* p) { return __ldcg(p); }
__device__ __forceinline__ float ld_logit(const uint16_t* p) { return bf16_from_bits(__ldcg(p)); }

// Four consecutive logits of a row from column c; columns >= E give `pad`.
template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* row, int c, int E, float pad, float v[4]) {
  if constexpr (VEC) {
    if (c < E) {
      if constexpr (sizeof(T) == 4) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(row + c));
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
      } else {
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(row + c));
        v[0] = bf16_from_bits(u.x & 0xffffu), v[1] = bf16_from_bits(u.x >> 16);
        v[2] = bf16_from_bits(u.y & 0xffffu), v[3] = bf16_from_bits(u.y >> 16);
      }
    } else {
      v[0] = v[1] = v[2] = v[3] = pad;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i < E ? ld_logit(row + c + i) : pad;
  }
}

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Score of a logit (softmax: relative to the row maximum) and, for the
// gradient, r with dscore/dlogit = score * r.
template <int SF>
__device__ __forceinline__ float score_of(float l, float mx) {
  if constexpr (SF == DSV4_SCORE_SOFTMAX) return expf(l - mx);
  else if constexpr (SF == DSV4_SCORE_SIGMOID) return 1.f / (1.f + expf(-l));
  else return sqrtf(fmaxf(l, 0.f) + log1pf(expf(-fabsf(l))));
}
template <int SF>
__device__ __forceinline__ float score_grad(float l, float mx, float* r) {
  if constexpr (SF == DSV4_SCORE_SOFTMAX) {
    *r = 1.f;
    return expf(l - mx);
  } else if constexpr (SF == DSV4_SCORE_SIGMOID) {
    const float s = 1.f / (1.f + expf(-l));
    *r = 1.f / (1.f + expf(l));   // 1 - s without cancellation
    return s;
  } else {
    const float e = expf(-fabsf(l));
    const float sp = fmaxf(l, 0.f) + log1pf(e);
    const float sg = (l >= 0.f ? 1.f : e) / (1.f + e);
    *r = sp > 0.f ? 0.5f * sg / sp : 0.5f;   // sg / sp -> 1 far below zero
    return sqrtf(sp);
  }
}

// Per-sequence part of g held by a warp: lane's four columns of each chunk.
template <int NV>
struct GRow {
  int seq = -2;
  float g[NV][4];
  // atomics of another kernel (or of this CTA before a barrier) wrote the
  // histogram: read it past L1
  __device__ __forceinline__ void load(const BalanceParams& p, int s, int lane) {
    if (s == seq) return;
    seq = s;
    const int2 in = __ldcg(&p.info[s]);
    const float c = in.y > 0 ? (float)((double)p.E / ((double)in.x * (double)in.y)) : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = i * 128 + lane * 4 + j;
        g[i][j] = e < p.E ? c * (float)__ldcg(&p.hist[(int64_t)s * p.E + e]) : 0.f;
      }
  }
};

// Whether row t has a pick (its lanes look at the k picks together).
__device__ __forceinline__ bool row_live(const BalanceParams& p, int64_t t, int lane) {
  bool any = false;
  for (int j = lane; j < p.k; j += 32) {
    const int e = __ldcg(&p.idx[t * p.k + j]);
    any |= e >= 0 && e < p.E;
  }
  return __any_sync(0xffffffffu, any);
}

// d_t of the rows [t0, t1) of one warp, their sum in double.
template <typename T, bool VEC, int SF, int NV>
__device__ double forward_rows(const BalanceParams& p, int64_t t0, int64_t t1) {
  const int lane = threadIdx.x & 31;
  const T* base = static_cast<const T*>(p.logits);
  GRow<NV> gr;
  double sum = 0.0;
  int s = t0 < t1 ? seq_of(p, t0) : -1;
  for (int64_t t = t0; t < t1; ++t) {
    if (p.off) s = seq_of(p, t);
    if (s < 0 || !row_live(p, t, lane)) {
      if (lane == 0) p.rows[t] = make_float4(0.f, -1.f, 0.f, 0.f);
      continue;
    }
    const T* row = base + t * p.E;
    float v[NV][4];
#pragma unroll
    for (int i = 0; i < NV; ++i) load4<T, VEC>(row, i * 128 + lane * 4, p.E, -INFINITY, v[i]);
    gr.load(p, s, lane);
    float mx = 0.f;
    if constexpr (SF == DSV4_SCORE_SOFTMAX) {
      mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx = fmaxf(mx, v[i][j]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (mx == -INFINITY) mx = 0.f;   // every score is 0
    }
    float z = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = i * 128 + lane * 4 + j;
        const float sc = e < p.E ? score_of<SF>(v[i][j], mx) : 0.f;
        z += sc;
        u = fmaf(sc, gr.g[i][j], u);
      }
    z = warp_sum_f(z);
    u = warp_sum_f(u);
    // a row whose scores are all zero has no probabilities: no part in the loss
    const bool none = z == 0.f;
    const float zi = none ? -1.f : 1.f / z, d = none ? 0.f : u / z;
    if (lane == 0) p.rows[t] = make_float4(mx, zi, d, __int_as_float(s));
    sum += (double)d;
  }
  return sum;
}

// Sum of the partial sums, number of sequences, loss, by one CTA.
__device__ void finish(const BalanceParams& p, int n_part, double* red, int* redi) {
  double a = 0.0;
  for (int i = threadIdx.x; i < n_part; i += blockDim.x) a += __ldcg(&p.part[i]);
  int q = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) q += __ldcg(&p.info[i]).x > 0;
  red[threadIdx.x] = a;
  redi[threadIdx.x] = q;
  __syncthreads();
  for (int h = blockDim.x / 2; h > 0; h >>= 1) {
    if ((int)threadIdx.x < h) {
      red[threadIdx.x] += red[threadIdx.x + h];
      redi[threadIdx.x] += redi[threadIdx.x + h];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.head[0] = redi[0];
    *p.loss = redi[0] ? (float)((double)p.alpha * red[0] / redi[0]) : 0.f;
  }
}

__global__ void __launch_bounds__(BL_THREADS) balance_zero_kernel(int4* __restrict__ z, int64_t n16) {
  griddep_wait();
  griddep_launch();
  for (int64_t i = blockIdx.x * (int64_t)BL_THREADS + threadIdx.x; i < n16; i += (int64_t)gridDim.x * BL_THREADS)
    z[i] = make_int4(0, 0, 0, 0);
}

__global__ void __launch_bounds__(BL_THREADS) balance_count_kernel(const BalanceParams p) {
  griddep_wait();
  griddep_launch();
  const int64_t t0 = (int64_t)blockIdx.x * BL_THREADS;
  if (blockIdx.x == 0) check_offsets(p);
  count_rows(p, t0, min(t0 + BL_THREADS, p.T));
}

template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_THREADS) balance_forward_kernel(const BalanceParams p) {
  __shared__ double red[BL_THREADS];
  __shared__ int redi[BL_THREADS];
  __shared__ int last;
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * BL_WARPS + warp) * BL_TOK;
  const double d = forward_rows<T, VEC, SF, NV>(p, min(t0, p.T), min(t0 + BL_TOK, p.T));
  for (int64_t i = blockIdx.x * (int64_t)BL_THREADS + threadIdx.x; i < (int64_t)p.S * p.E;
       i += (int64_t)gridDim.x * BL_THREADS)
    p.counts[i] = __ldcg(&p.hist[i]);
  if (lane == 0) red[warp] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    double a = 0.0;
    for (int w = 0; w < BL_WARPS; ++w) a += red[w];
    p.part[blockIdx.x] = a;
    __threadfence();
    last = atomicAdd(&p.head[1], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  finish(p, gridDim.x, red, redi);
}

// Small batches: counts, loss and row statistics in one CTA and one launch.
template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_SMALL_THREADS) balance_forward_small_kernel(const BalanceParams p) {
  __shared__ double red[BL_SMALL_THREADS];
  __shared__ int redi[BL_SMALL_THREADS];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  for (int64_t i = threadIdx.x; i < (int64_t)p.S * p.E; i += blockDim.x) p.hist[i] = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) p.info[i] = make_int2(0, 0);
  __threadfence();
  __syncthreads();
  check_offsets(p);
  count_rows(p, 0, p.T);
  __threadfence();
  __syncthreads();
  for (int64_t i = threadIdx.x; i < (int64_t)p.S * p.E; i += blockDim.x) p.counts[i] = __ldcg(&p.hist[i]);
  const int64_t per = (p.T + nw - 1) / nw, t0 = warp * per;
  const double d = forward_rows<T, VEC, SF, NV>(p, min(t0, p.T), min(t0 + per, p.T));
  if (lane == 0) p.part[warp] = d;
  __threadfence();
  __syncthreads();
  finish(p, nw, red, redi);
}

template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_THREADS) balance_backward_kernel(const BalanceParams p) {
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * BL_WARPS + warp) * BL_TOK, t1 = min(t0 + BL_TOK, p.T);
  const int q = __ldcg(&p.head[0]);
  const float c = q ? p.alpha / (float)q * __ldcg(p.up) : 0.f;
  GRow<NV> gr;
  for (int64_t t = t0; t < t1; ++t) {
    const float4 st = __ldcg(&p.rows[t]);
    const bool live = st.y >= 0.f || st.y != st.y;
    float o[NV][4];
    if (live) {
      const T* row = static_cast<const T*>(p.logits) + t * p.E;
      float v[NV][4];
#pragma unroll
      for (int i = 0; i < NV; ++i) load4<T, VEC>(row, i * 128 + lane * 4, p.E, 0.f, v[i]);
      gr.load(p, __float_as_int(st.w), lane);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float r;
          const float s = score_grad<SF>(v[i][j], st.x, &r);
          o[i][j] = c * (s * st.y) * r * (gr.g[i][j] - st.z);
        }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }
    T* dst = static_cast<T*>(p.dlogits) + t * p.E;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = i * 128 + lane * 4;
      if constexpr (VEC) {
        if (e < p.E) {
          if constexpr (sizeof(T) == 4)
            *reinterpret_cast<float4*>(dst + e) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
          else
            *reinterpret_cast<uint2*>(dst + e) = make_uint2(bf16_bits(o[i][0]) | ((uint32_t)bf16_bits(o[i][1]) << 16),
                                                            bf16_bits(o[i][2]) | ((uint32_t)bf16_bits(o[i][3]) << 16));
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (e + j < p.E) {
            if constexpr (sizeof(T) == 4) dst[e + j] = o[i][j];
            else dst[e + j] = bf16_bits(o[i][j]);
          }
      }
    }
  }
}

enum Pass { FORWARD, FORWARD_SMALL, BACKWARD };

template <typename T, bool VEC, int SF, int NV>
cudaError_t launch_pass(Pass pass, const BalanceParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)std::max<int64_t>(bl_ctas(p.T), 1));
  if (pass == FORWARD)
    return launch_k(balance_forward_kernel<T, VEC, SF, NV>, grid, dim3(BL_THREADS), 0, st, pdl_enabled(), p);
  if (pass == FORWARD_SMALL)
    return launch_k(balance_forward_small_kernel<T, VEC, SF, NV>, dim3(1), dim3(BL_SMALL_THREADS), 0, st, pdl_enabled(), p);
  return launch_k(balance_backward_kernel<T, VEC, SF, NV>, grid, dim3(BL_THREADS), 0, st, pdl_enabled(), p);
}
template <typename T, bool VEC, int SF>
cudaError_t launch_nv(Pass pass, const BalanceParams& p, cudaStream_t st) {
  if (p.E <= 256) return launch_pass<T, VEC, SF, 2>(pass, p, st);
  if (p.E <= 512) return launch_pass<T, VEC, SF, 4>(pass, p, st);
  return launch_pass<T, VEC, SF, 8>(pass, p, st);
}
template <typename T, bool VEC>
cudaError_t launch_sf(Pass pass, const BalanceParams& p, cudaStream_t st) {
  if (p.score == DSV4_SCORE_SOFTMAX) return launch_nv<T, VEC, DSV4_SCORE_SOFTMAX>(pass, p, st);
  if (p.score == DSV4_SCORE_SIGMOID) return launch_nv<T, VEC, DSV4_SCORE_SIGMOID>(pass, p, st);
  return launch_nv<T, VEC, DSV4_SCORE_SQRTSOFTPLUS>(pass, p, st);
}
// 16-byte (fp32) / 8-byte (bf16) accesses where every row starts on them.
cudaError_t launch(Pass pass, int dtype, const BalanceParams& p, cudaStream_t st) {
  const uintptr_t al = dtype == DSV4_DT_FP32 ? 16 : 8;
  const bool vec = p.E % 4 == 0 && (uintptr_t)p.logits % al == 0 && (uintptr_t)p.dlogits % al == 0;
  if (dtype == DSV4_DT_FP32) return vec ? launch_sf<float, true>(pass, p, st) : launch_sf<float, false>(pass, p, st);
  return vec ? launch_sf<uint16_t, true>(pass, p, st) : launch_sf<uint16_t, false>(pass, p, st);
}

const char* bad_sizes(int64_t T, int32_t E, int32_t S) {
  if (T < 0 || T > 0x7fffffff) return "n_tokens must be in [0, 2^31)";
  if (E < 1 || E > BL_MAX_E) return "n_experts must be in [1, 1024]";
  if (S < 1 || (int64_t)S * E > 0x7fffffff) return "n_seqs must be positive, n_seqs * n_experts below 2^31";
  return nullptr;
}

BalanceParams bl_params(void* ws, int64_t T, int E, int S) {
  const BalanceLayout l = bl_layout(T, E, S);
  uint8_t* w = static_cast<uint8_t*>(ws);
  BalanceParams p = {};
  p.T = T, p.E = E, p.S = S;
  p.head = reinterpret_cast<int*>(w + l.head);
  p.info = reinterpret_cast<int2*>(w + l.info);
  p.hist = reinterpret_cast<int*>(w + l.hist);
  p.rows = reinterpret_cast<float4*>(w + l.rows);
  p.part = reinterpret_cast<double*>(w + l.part);
  return p;
}

}  // namespace
}  // namespace dsv4

using namespace dsv4;

extern "C" int64_t dsv4_balance_workspace_bytes(int64_t n_tokens, int32_t n_experts, int32_t n_seqs) {
  if (bad_sizes(n_tokens, n_experts, n_seqs)) return DSV4_EINVAL;
  return bl_layout(n_tokens, n_experts, n_seqs).bytes;
}

extern "C" int dsv4_balance_forward(const void* logits, int32_t dtype, int64_t n_tokens, int32_t n_experts,
                                    const int32_t* indices, int32_t topk, const int32_t* seq_offsets, int32_t n_seqs,
                                    int32_t score_func, float alpha, float* loss, int32_t* counts, void* workspace,
                                    int64_t workspace_bytes, int* status, void* stream) {
  DSV4_API_BEGIN
  const char* bad = bad_sizes(n_tokens, n_experts, n_seqs);
  DSV4_CHECK_ARG(!bad, bad);
  DSV4_CHECK_ARG(dtype == DSV4_DT_FP32 || dtype == DSV4_DT_BF16, "logits must be fp32 or bf16");
  DSV4_CHECK_ARG(topk >= 1, "topk must be positive");
  DSV4_CHECK_ARG(score_func >= DSV4_SCORE_SOFTMAX && score_func <= DSV4_SCORE_SQRTSOFTPLUS, "unknown score function");
  DSV4_CHECK_ARG(seq_offsets || n_seqs == 1, "several sequences need their offsets");
  DSV4_CHECK_ARG(loss && counts && workspace && (n_tokens == 0 || (logits && indices)), "null pointer");
  DSV4_CHECK_ARG((uintptr_t)workspace % 16 == 0, "the workspace must be 16-byte aligned");
  DSV4_CHECK_ARG(workspace_bytes >= bl_layout(n_tokens, n_experts, n_seqs).bytes, "workspace too small");
  DeviceScope dev;
  if (int rc = dev.enter(workspace)) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  BalanceParams p = bl_params(workspace, n_tokens, n_experts, n_seqs);
  p.logits = logits, p.idx = indices, p.k = topk, p.off = seq_offsets, p.score = score_func, p.alpha = alpha;
  p.loss = loss, p.counts = counts, p.status = status;
  if (n_tokens <= BL_ONE_CTA_TOKENS && (int64_t)n_seqs * n_experts <= 16384) {
    DSV4_CUDA_CHECK(launch(FORWARD_SMALL, dtype, p, st));
    return DSV4_OK;
  }
  const int64_t n16 = bl_layout(n_tokens, n_experts, n_seqs).rows / 16;   // head, info, histogram
  const unsigned zc = (unsigned)std::min<int64_t>((n16 + BL_THREADS - 1) / BL_THREADS, 148 * 4);
  DSV4_CUDA_CHECK(launch_k(balance_zero_kernel, dim3(zc), dim3(BL_THREADS), 0, st, pdl_enabled(),
                           static_cast<int4*>(workspace), n16));
  if (n_tokens > 0)
    DSV4_CUDA_CHECK(launch_k(balance_count_kernel, dim3((unsigned)((n_tokens + BL_THREADS - 1) / BL_THREADS)),
                             dim3(BL_THREADS), 0, st, pdl_enabled(), p));
  DSV4_CUDA_CHECK(launch(FORWARD, dtype, p, st));
  DSV4_API_END
}

extern "C" int dsv4_balance_backward(const void* logits, int32_t dtype, int64_t n_tokens, int32_t n_experts,
                                     int32_t n_seqs, int32_t score_func, float alpha, const float* grad_loss,
                                     void* dlogits, const void* workspace, int64_t workspace_bytes, void* stream) {
  DSV4_API_BEGIN
  const char* bad = bad_sizes(n_tokens, n_experts, n_seqs);
  DSV4_CHECK_ARG(!bad, bad);
  DSV4_CHECK_ARG(dtype == DSV4_DT_FP32 || dtype == DSV4_DT_BF16, "logits must be fp32 or bf16");
  DSV4_CHECK_ARG(score_func >= DSV4_SCORE_SOFTMAX && score_func <= DSV4_SCORE_SQRTSOFTPLUS, "unknown score function");
  if (n_tokens == 0) return DSV4_OK;
  DSV4_CHECK_ARG(logits && grad_loss && dlogits && workspace, "null pointer");
  DSV4_CHECK_ARG((uintptr_t)workspace % 16 == 0, "the workspace must be 16-byte aligned");
  DSV4_CHECK_ARG(workspace_bytes >= bl_layout(n_tokens, n_experts, n_seqs).bytes, "workspace too small");
  DeviceScope dev;
  if (int rc = dev.enter(workspace)) return rc;
  BalanceParams p = bl_params(const_cast<void*>(workspace), n_tokens, n_experts, n_seqs);
  p.logits = logits, p.score = score_func, p.alpha = alpha, p.up = grad_loss, p.dlogits = dlogits;
  DSV4_CUDA_CHECK(launch(BACKWARD, dtype, p, (cudaStream_t)stream));
  DSV4_API_END
}
