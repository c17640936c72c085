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
// probabilities are kept.  The forward stores (row maximum, 1 / sum, d_t,
// sequence) per token, and the backward is one pass without reductions.
//
// Counts are integer atomics (any order gives the same numbers), the d_t are
// added in a fixed order, in double beyond a warp's rows, so results
// do not depend on scheduling.
// Bound: HBM, the logits once forward, once backward, the gradient once.
// While a warp computes its rows, the next ones are on their way.  Measured
// (65536 x 256 fp32, 24 sequences, sigmoid): 63 us forward (three launches)
// and backward together; 64 rows: 10.3 us.
#include <algorithm>

#include "capi_internal.h"
#include "common.cuh"

namespace dsv4 {
namespace {

constexpr int BL_THREADS = 256;          // 8 warps
constexpr int BL_WARPS = BL_THREADS / 32;
constexpr int BL_CTAS = 4;               // per SM (64 registers a thread)
constexpr int BL_TOK = 32;               // rows per warp at most: a lane keeps each one's state
constexpr int BL_MAX_E = 1024;
constexpr int BL_COUNT_TOK = 256;        // rows per CTA of the counts
constexpr int BL_OFFS = 1024;            // sequence offsets kept in shared memory
constexpr int BL_SEG = 64;               // shorter pieces of a sequence count straight in global memory
// One CTA and one launch up to here: its counts live in shared memory.
constexpr int BL_SMALL_THREADS = 1024;
constexpr int BL_SMALL_TOKENS = 256;
constexpr int BL_SMALL_COUNTS = 8192;

// Saved state of one forward (the caller's buffer), then scratch.
struct BalanceLayout {
  int64_t head;      // int[4]: sequences with tokens, CTAs done, unused, unused
  int64_t info;      // int[S][2]: tokens, picks
  int64_t hist;      // int[S][E]
  int64_t rows;      // float4[T]: row maximum, 1 / sum, d_t, sequence (int bits, -1: no part in the loss)
  int64_t part;      // double[CTAs]
  int64_t bytes;
};
inline int64_t al16(int64_t v) { return (v + 15) / 16 * 16; }
// Rows per warp: all CTAs on the GPU at once, up to 32 rows.
inline int bl_tok(int64_t T) {
  const int64_t warps = (int64_t)148 * BL_CTAS * BL_WARPS;
  return (int)std::max<int64_t>(1, std::min<int64_t>(BL_TOK, (T + warps - 1) / warps));
}
inline int64_t bl_ctas(int64_t T) {
  const int64_t rows = (int64_t)BL_WARPS * bl_tok(T);
  return (T + rows - 1) / rows;
}
inline BalanceLayout bl_layout(int64_t T, int64_t E, int64_t S) {
  BalanceLayout l;
  l.head = 0;
  l.info = 16;
  l.hist = l.info + al16(S * 8);
  l.rows = l.hist + al16(S * E * 4);
  l.part = l.rows + T * 16;
  l.bytes = l.part + al16(std::max<int64_t>(bl_ctas(T), 1) * 8);
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

// The sequence of row t, -1 for a row in none (binary search); off: the
// offsets, or their copy in shared memory.
__device__ __forceinline__ int seq_of(const int32_t* off, int S, int64_t t) {
  if (!off) return 0;
  int lo = 0, hi = S + 1;   // number of offsets <= t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)off[mid] <= t) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1 < S ? lo - 1 : -1;
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

// Adds the picks of row t of sequence s to hist[e]; returns how many count.
__device__ __forceinline__ int count_row(const BalanceParams& p, int64_t t, int* hist) {
  int picks = 0;
  const int32_t* row = p.idx + t * p.k;
  for (int j = 0; j < p.k; j += 4) {
    int e[4] = {-1, -1, -1, -1};
    if (p.k % 4 == 0 && (uintptr_t)p.idx % 16 == 0) {
      const int4 v = __ldcg(reinterpret_cast<const int4*>(row + j));
      e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j + i < p.k) e[i] = __ldcg(row + j + i);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e[i] >= 0 && e[i] < p.E) {
        atomicAdd(&hist[e[i]], 1);
        ++picks;
      } else if (e[i] != -1) {
        set_status(p.status, DSV4_EINVAL);
      }
    }
  }
  return picks;
}

// Tokens and picks of the lanes' rows added to their sequences' totals, one
// add per group of lanes with the same sequence.
__device__ __forceinline__ void add_info(int2* info, int s, int picks) {
  const int lane = threadIdx.x & 31, key = picks ? s : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, key);
  const int sum = __reduce_add_sync(same, picks);
  if (key >= 0 && lane == __ffs(same) - 1) {
    atomicAdd(&info[s].x, __popc(same));
    atomicAdd(&info[s].y, sum);
  }
}

__global__ void __launch_bounds__(BL_THREADS) balance_zero_kernel(int4* __restrict__ z, int64_t n16) {
  griddep_wait();
  griddep_launch();
  for (int64_t i = blockIdx.x * (int64_t)BL_THREADS + threadIdx.x; i < n16; i += (int64_t)gridDim.x * BL_THREADS)
    z[i] = make_int4(0, 0, 0, 0);
}

// Counts of BL_COUNT_TOK rows per CTA; every row's sequence goes to its row
// state.  A long piece of one sequence is counted in shared memory first
// (straight into 256 global counters, one sequence of 65536 rows took 70 us
// more); where sequences are short, BL_SEG rows at a time go straight to
// global memory.
__global__ void __launch_bounds__(BL_THREADS) balance_count_kernel(const BalanceParams p) {
  __shared__ int hist[BL_MAX_E];
  __shared__ int32_t offs[BL_OFFS];
  griddep_wait();
  griddep_launch();
  if (blockIdx.x == 0) check_offsets(p);
  const int32_t* off = p.off;
  if (off && p.S < BL_OFFS) {   // a search in global memory costs a microsecond
    for (int i = threadIdx.x; i <= p.S; i += BL_THREADS) offs[i] = __ldcg(&p.off[i]);
    __syncthreads();
    off = offs;
  }
  const int64_t t0 = (int64_t)blockIdx.x * BL_COUNT_TOK, t1 = min(t0 + BL_COUNT_TOK, p.T);
  for (int64_t a = t0; a < t1;) {   // all threads agree on the pieces
    const int s = seq_of(off, p.S, a);
    int64_t b = t1;
    if (s >= 0 && off) b = max(a + 1, min((int64_t)off[s + 1], t1));
    const bool local = s >= 0 && b - a >= BL_SEG;
    if (local) {
      for (int i = threadIdx.x; i < p.E; i += BL_THREADS) hist[i] = 0;
      __syncthreads();
    } else {
      b = min(a + BL_SEG, t1);
    }
    for (int64_t t = a + threadIdx.x; t - (threadIdx.x & 31) < b; t += BL_THREADS) {
      const int st = t >= b ? -1 : (local ? s : seq_of(off, p.S, t));
      const int picks = st >= 0 ? count_row(p, t, local ? hist : p.hist + (int64_t)st * p.E) : 0;
      if (t < b) p.rows[t] = make_float4(0.f, 0.f, 0.f, __int_as_float(picks ? st : -1));
      add_info(p.info, st, picks);
    }
    if (local) {
      __syncthreads();
      for (int i = threadIdx.x; i < p.E; i += BL_THREADS)
        if (hist[i]) atomicAdd(&p.hist[(int64_t)s * p.E + i], hist[i]);
      __syncthreads();
    }
    a = b;
  }
}

// ---------------------------------------------------------------------------
// rows
// ---------------------------------------------------------------------------
// Lane's column j of chunk i (128 columns): four neighbours where rows take
// vector accesses, else neighbours across the lanes.
template <bool VEC>
__device__ __forceinline__ int col(int i, int j) {
  const int lane = threadIdx.x & 31;
  return VEC ? i * 128 + lane * 4 + j : i * 128 + j * 32 + lane;
}
// A row's logits; columns >= E give -inf, whose score is 0.
template <typename T, bool VEC, int NV>
__device__ __forceinline__ void load_row(const T* row, int E, float (&v)[NV][4]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if constexpr (VEC) {
      const int c = col<VEC>(i, 0);
      if (c < E) {
        if constexpr (sizeof(T) == 4) {
          const float4 f = __ldcg(reinterpret_cast<const float4*>(row + c));
          v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w;
        } else {
          const uint2 u = __ldcg(reinterpret_cast<const uint2*>(row + c));
          v[i][0] = bf16_from_bits(u.x & 0xffffu), v[i][1] = bf16_from_bits(u.x >> 16);
          v[i][2] = bf16_from_bits(u.y & 0xffffu), v[i][3] = bf16_from_bits(u.y >> 16);
        }
      } else {
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = col<VEC>(i, j);
        if constexpr (sizeof(T) == 4) v[i][j] = c < E ? __ldcg(row + c) : -INFINITY;
        else v[i][j] = c < E ? bf16_from_bits(__ldcg(row + c)) : -INFINITY;
      }
    }
  }
}

// exp(x) = 2^(x log2 e), the rounding error of the product put back (log2 e in
// two parts, Cody and Waite 1980): within 6 2^-24 for results between 2^-126
// and 2^126.  The hardware's 2^t of the product alone is off by up to 60 2^-24
// at x = -86.  Beyond, 2^t as it is: 0, infinity or NaN have no error to put back.
__device__ __forceinline__ float exp_fast(float x) {
  const float t = x * 1.4426950216f;
  const float lo = fmaf(x, 1.9259629911e-8f, fmaf(x, 1.4426950216f, -t));
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return fabsf(t) < 126.f ? fmaf(r, lo * 0.69314718056f, r) : r;
}
// sqrt(softplus(l)) = h sqrt(u): for l < 0, h = exp(l / 2) and u = log1p(e) / e
// with e = h^2; for l >= 0, h = 1 and u = l + log1p(e), e = exp(-l).  So a score
// keeps its digits down to exp(l / 2) = 2^-126, where softplus(l) itself has
// long left the range of fp32.  log1p(e) = 2 atanh(z), z = e / (2 + e) <= 1/3,
// by its power series in z^2 <= 1/9: the first term left out is below 1.5e-8 of
// the sum, and unlike log(1 + e) it keeps its digits as e goes to 0.
__device__ __forceinline__ float softplus_root(float l, float* u, float* e_out) {
  const float h = exp_fast(-0.5f * fabsf(l)), e = h * h;
  const float w = __fdividef(1.f, 2.f + e), z = e * w, q = z * z;
  float s = 1.f / 13.f;
  s = fmaf(s, q, 1.f / 11.f);
  s = fmaf(s, q, 1.f / 9.f);
  s = fmaf(s, q, 1.f / 7.f);
  s = fmaf(s, q, 1.f / 5.f);
  s = fmaf(s, q, 1.f / 3.f);
  s = fmaf(s, q, 1.f);
  const float ratio = 2.f * w * s;
  *e_out = e;
  *u = l >= 0.f ? fmaf(e, ratio, l) : ratio;
  return l >= 0.f ? 1.f : h;   // a NaN stays one in h
}
// Score of a logit (softmax: relative to the row maximum mx).  The exponential,
// the fast quotient and the root are each within a few 2^-23; the library's
// exact ones made the kernel compute-bound.
template <int SF>
__device__ __forceinline__ float score_of(float l, float mx) {
  if constexpr (SF == DSV4_SCORE_SOFTMAX) {
    return exp_fast(l - mx);
  } else if constexpr (SF == DSV4_SCORE_SIGMOID) {
    return __fdividef(1.f, 1.f + exp_fast(-l));
  } else {
    float u, e;
    const float h = softplus_root(l, &u, &e);
    return h * (u * rsqrtf(u));
  }
}
// dscore / dlogit.
template <int SF>
__device__ __forceinline__ float score_slope(float l, float mx) {
  if constexpr (SF == DSV4_SCORE_SOFTMAX) {
    return exp_fast(l - mx);
  } else if constexpr (SF == DSV4_SCORE_SIGMOID) {
    const float e = exp_fast(-fabsf(l)), d = 1.f + e;   // s (1 - s) = e / (1 + e)^2, either sign of l
    return __fdividef(e, d * d);
  } else {
    float u, e;   // sigma / (2 score), sigma = h^2 / (1 + e)
    const float h = softplus_root(l, &u, &e);
    return __fdividef(0.5f * h, 1.f + e) * rsqrtf(u);
  }
}

// g of one sequence, a warp's columns, from its counts.  Atomics of another
// kernel (or of this CTA before a barrier) wrote them: global ones are read
// past L1.
__device__ __forceinline__ float g_factor(int2 info, int E) {
  return info.y > 0 ? (float)E / ((float)info.x * (float)info.y) : 0.f;
}
template <bool VEC, int NV>
struct GRow {
  int seq = -1;
  float g[NV][4];
  __device__ __forceinline__ void from_counts(int s, int2 info, const int* hist, bool global, int E, float scale) {
    seq = s;
    const float c = scale * g_factor(info, E);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = col<VEC>(i, j);
        g[i][j] = e < E ? c * (float)(global ? __ldcg(hist + e) : hist[e]) : 0.f;
      }
  }
  __device__ __forceinline__ void from_shared(int s, const float* gs, int E) {
    seq = s;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = col<VEC>(i, j);
        g[i][j] = e < E ? gs[e] : 0.f;
      }
  }
};
// g of the sequence of the CTA's first row that counts, in shared memory for
// all its warps (each warp reading it from L2 made the 1 KB of a batch's only
// sequence the limit: 59 us instead of 31).  Returns that sequence.  `state`:
// lanes 0 .. tok - 1 hold the sequences of the warp's rows.
__device__ __forceinline__ int share_g(const BalanceParams& p, int mine, float* gs, int* first, float scale) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t some = __ballot_sync(0xffffffffu, mine >= 0);
  const int s = __shfl_sync(0xffffffffu, mine, some ? __ffs(some) - 1 : 0);
  if (lane == 0) first[warp] = some ? s : -1;
  __syncthreads();
  int s0 = -1;
  for (int w = 0; w < BL_WARPS; ++w)
    if (s0 < 0) s0 = first[w];
  if (s0 >= 0) {
    const float c = scale * g_factor(__ldcg(&p.info[s0]), p.E);
    for (int e = threadIdx.x; e < p.E; e += BL_THREADS) gs[e] = c * (float)__ldcg(&p.hist[(int64_t)s0 * p.E + e]);
  }
  __syncthreads();
  return s0;
}

// d_t, row maximum and 1 / sum of R rows of the sequence in gr (together, so
// that their reductions overlap).
template <int SF, bool VEC, int NV, int R>
__device__ __forceinline__ void rows_forward(float (*v)[NV][4], const GRow<VEC, NV>& gr, float (&mx)[R], float (&zi)[R],
                                             float (&d)[R]) {
  float z[R], u[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    mx[r] = 0.f;
    if constexpr (SF == DSV4_SCORE_SOFTMAX) {
      mx[r] = -INFINITY;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx[r] = fmaxf(mx[r], v[r][i][j]);
    }
  }
  if constexpr (SF == DSV4_SCORE_SOFTMAX) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], o));
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (mx[r] == -INFINITY) mx[r] = 0.f;   // every score is 0
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    z[r] = u[r] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float sc = score_of<SF>(v[r][i][j], mx[r]);
        z[r] += sc;
        u[r] = fmaf(sc, gr.g[i][j], u[r]);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      z[r] += __shfl_xor_sync(0xffffffffu, z[r], o);
      u[r] += __shfl_xor_sync(0xffffffffu, u[r], o);
    }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // a row whose scores are all zero has no probabilities: p = 0
    zi[r] = z[r] == 0.f ? 0.f : 1.f / z[r];
    d[r] = z[r] == 0.f ? 0.f : u[r] / z[r];
  }
}

// Sum of the partial sums, number of sequences, loss, by one CTA.
__device__ void finish(const BalanceParams& p, const double* part, int n_part, const int2* info, double* red,
                       int* redi) {
  double a = 0.0;
  for (int i = threadIdx.x; i < n_part; i += blockDim.x) a += __ldcg(&part[i]);
  int q = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) q += __ldcg(&info[i].x) > 0;
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

template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_THREADS, NV <= 2 ? BL_CTAS : 1) balance_forward_kernel(const BalanceParams p, const int tok) {
  __shared__ double red[BL_THREADS];
  __shared__ int redi[BL_THREADS];
  __shared__ float gs[BL_MAX_E];
  __shared__ int last;
  constexpr int BATCH = NV == 1 ? 4 : (NV == 2 ? 2 : 1);   // rows computed together
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * BL_WARPS + warp) * tok;
  const int n = (int)max((int64_t)0, min((int64_t)tok, p.T - t0));
  const T* rows = static_cast<const T*>(p.logits) + t0 * p.E;
  float v[BATCH][NV][4], nx[BATCH][NV][4];
  // Before the wait: the kernel just before is this call's count kernel, which
  // does not write logits, and it starts its successor only after its own wait,
  // when whatever wrote them is complete.
#pragma unroll
  for (int r = 0; r < BATCH; ++r)
    if (r < n) load_row<T, VEC, NV>(rows + (int64_t)r * p.E, p.E, nx[r]);
  griddep_wait();
  griddep_launch();
  const int mine = lane < n ? __float_as_int(__ldcg(&p.rows[t0 + lane].w)) : -1;
  const int s0 = share_g(p, mine, gs, redi, 1.f);
  GRow<VEC, NV> gr;
  float sum = 0.f;
  float4 state = make_float4(0.f, 0.f, 0.f, __int_as_float(mine));   // lane i: row t0 + i
#pragma unroll 1
  for (int b = 0; b < n; b += BATCH) {
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[r][i][j] = nx[r][i][j];
      if (b + BATCH + r < n) load_row<T, VEC, NV>(rows + (int64_t)(b + BATCH + r) * p.E, p.E, nx[r]);
    }
    int s[BATCH];
    bool other = false;
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
      s[r] = b + r < n ? __shfl_sync(0xffffffffu, mine, (b + r) & 31) : -1;
      other |= s[r] >= 0 && s[r] != gr.seq;
    }
    float mx[BATCH], zi[BATCH], d[BATCH];
    if (!other) {
      rows_forward<SF, VEC, NV, BATCH>(v, gr, mx, zi, d);
    } else {
#pragma unroll
      for (int r = 0; r < BATCH; ++r) {
        if (s[r] < 0) continue;
        if (s[r] != gr.seq) {
          if (s[r] == s0) gr.from_shared(s[r], gs, p.E);
          else gr.from_counts(s[r], __ldcg(&p.info[s[r]]), p.hist + (int64_t)s[r] * p.E, true, p.E, 1.f);
        }
        float m1[1], z1[1], d1[1];
        rows_forward<SF, VEC, NV, 1>(v + r, gr, m1, z1, d1);
        mx[r] = m1[0], zi[r] = z1[0], d[r] = d1[0];
      }
    }
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
      if (s[r] < 0) continue;
      if (lane == b + r) state = make_float4(mx[r], zi[r], d[r], __int_as_float(s[r]));
      sum += d[r];
    }
  }
  if (lane < n) p.rows[t0 + lane] = state;
  for (int64_t i = blockIdx.x * (int64_t)BL_THREADS + threadIdx.x; i < (int64_t)p.S * p.E;
       i += (int64_t)gridDim.x * BL_THREADS)
    p.counts[i] = __ldcg(&p.hist[i]);
  __syncthreads();
  if (lane == 0) red[warp] = (double)sum;
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
  finish(p, p.part, gridDim.x, p.info, red, redi);
}

// Small batches: counts, loss and row statistics in one CTA and one launch.
template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_SMALL_THREADS) balance_forward_small_kernel(const BalanceParams p) {
  extern __shared__ int hist[];            // [S][E] counts, then [S] (tokens, picks)
  __shared__ int row_seq[BL_SMALL_TOKENS];
  __shared__ double red[BL_SMALL_THREADS];
  __shared__ int redi[BL_SMALL_THREADS];
  griddep_wait();
  griddep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int n = p.S * p.E, T_ = (int)p.T;
  int2* info = reinterpret_cast<int2*>(hist + (n + 1) / 2 * 2);
  // the first row of this warp is on its way while the picks are counted
  float v[NV][4];
  if (warp < T_) load_row<T, VEC, NV>(static_cast<const T*>(p.logits) + (int64_t)warp * p.E, p.E, v);
  for (int i = threadIdx.x; i < n; i += blockDim.x) hist[i] = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) info[i] = make_int2(0, 0);
  __syncthreads();
  check_offsets(p);
  if (threadIdx.x < BL_SMALL_TOKENS) {
    const int t = threadIdx.x, s = t < T_ ? seq_of(p.off, p.S, t) : -1;
    const int picks = s >= 0 ? count_row(p, t, hist + s * p.E) : 0;
    row_seq[t] = picks ? s : -1;
    add_info(info, s, picks);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) p.counts[i] = p.hist[i] = hist[i];
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) p.info[i] = info[i];
  GRow<VEC, NV> gr;
  float sum = 0.f;
  for (int t = warp; t < T_; t += nw) {
    if (t != warp) load_row<T, VEC, NV>(static_cast<const T*>(p.logits) + (int64_t)t * p.E, p.E, v);
    const int s = row_seq[t];
    float mx = 0.f, zi = 0.f, d = 0.f;
    if (s >= 0) {
      if (s != gr.seq) gr.from_counts(s, info[s], hist + s * p.E, false, p.E, 1.f);
      float m1[1], z1[1], d1[1];
      rows_forward<SF, VEC, NV, 1>(&v, gr, m1, z1, d1);
      mx = m1[0], zi = z1[0], d = d1[0];
    }
    if (lane == 0) p.rows[t] = make_float4(mx, zi, d, __int_as_float(s));
    sum += d;
  }
  __syncthreads();
  red[threadIdx.x] = lane == 0 ? (double)sum : 0.0;
  int q = 0;
  for (int i = threadIdx.x; i < p.S; i += blockDim.x) q += info[i].x > 0;
  redi[threadIdx.x] = q;
  __syncthreads();
  if (warp == 0) {
    double a = red[lane * 32];             // warp w's sum is at 32 w
    q = 0;
    for (int i = lane; i < (int)blockDim.x; i += 32) q += redi[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      a += __shfl_xor_sync(0xffffffffu, a, o);
      q += __shfl_xor_sync(0xffffffffu, q, o);
    }
    if (lane == 0) {
      p.head[0] = q;
      *p.loss = q ? (float)((double)p.alpha * a / q) : 0.f;
    }
  }
}

template <typename T, bool VEC, int SF, int NV>
__global__ void __launch_bounds__(BL_THREADS, NV <= 2 ? BL_CTAS : 1) balance_backward_kernel(const BalanceParams p, const int tok) {
  __shared__ float gs[BL_MAX_E];
  __shared__ int first[BL_WARPS];
  constexpr int BATCH = NV == 1 ? 4 : (NV == 2 ? 2 : 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t0 = ((int64_t)blockIdx.x * BL_WARPS + warp) * tok;
  const int n = (int)max((int64_t)0, min((int64_t)tok, p.T - t0));
  const T* rows = static_cast<const T*>(p.logits) + t0 * p.E;
  griddep_wait();
  griddep_launch();
  float v[BATCH][NV][4], nx[BATCH][NV][4];
#pragma unroll
  for (int r = 0; r < BATCH; ++r)
    if (r < n) load_row<T, VEC, NV>(rows + (int64_t)r * p.E, p.E, nx[r]);
  const float4 state = lane < n ? __ldcg(&p.rows[t0 + lane]) : make_float4(0.f, 0.f, 0.f, __int_as_float(-1));
  const int q = __ldcg(&p.head[0]);
  const float c = q ? p.alpha / (float)q * __ldcg(p.up) : 0.f;
  const int s0 = share_g(p, __float_as_int(state.w), gs, first, c);
  GRow<VEC, NV> gr;
#pragma unroll 1
  for (int b = 0; b < n; b += BATCH) {
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[r][i][j] = nx[r][i][j];
      if (b + BATCH + r < n) load_row<T, VEC, NV>(rows + (int64_t)(b + BATCH + r) * p.E, p.E, nx[r]);
    }
#pragma unroll
    for (int r = 0; r < BATCH; ++r) {
      if (b + r >= n) break;
      const float mx = __shfl_sync(0xffffffffu, state.x, (b + r) & 31);
      // c goes with g and d: c / sum would leave fp32 where a row's scores are small
      const float zi = __shfl_sync(0xffffffffu, state.y, (b + r) & 31);
      const float d = c * __shfl_sync(0xffffffffu, state.z, (b + r) & 31);
      const int s = __float_as_int(__shfl_sync(0xffffffffu, state.w, (b + r) & 31));
      if (s >= 0) {
        if (s != gr.seq) {
          if (s == s0) gr.from_shared(s, gs, p.E);
          else gr.from_counts(s, __ldcg(&p.info[s]), p.hist + (int64_t)s * p.E, true, p.E, c);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) v[r][i][j] = zi * score_slope<SF>(v[r][i][j], mx) * (gr.g[i][j] - d);
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[r][i][0] = v[r][i][1] = v[r][i][2] = v[r][i][3] = 0.f;
      }
      T* dst = static_cast<T*>(p.dlogits) + (t0 + b + r) * p.E;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const float* o = v[r][i];
        if constexpr (VEC) {
          const int e = col<VEC>(i, 0);
          if (e < p.E) {
            if constexpr (sizeof(T) == 4)
              *reinterpret_cast<float4*>(dst + e) = make_float4(o[0], o[1], o[2], o[3]);
            else
              *reinterpret_cast<uint2*>(dst + e) =
                  make_uint2(bf16_bits(o[0]) | ((uint32_t)bf16_bits(o[1]) << 16),
                             bf16_bits(o[2]) | ((uint32_t)bf16_bits(o[3]) << 16));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int e = col<VEC>(i, j);
            if (e < p.E) {
              if constexpr (sizeof(T) == 4) dst[e] = o[j];
              else dst[e] = bf16_bits(o[j]);
            }
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
enum Pass { FORWARD, FORWARD_SMALL, BACKWARD };

template <typename T, bool VEC, int SF, int NV>
cudaError_t launch_pass(Pass pass, const BalanceParams& p, cudaStream_t st) {
  const dim3 grid((unsigned)std::max<int64_t>(bl_ctas(p.T), 1));
  if (pass == FORWARD)
    return launch_k(balance_forward_kernel<T, VEC, SF, NV>, grid, dim3(BL_THREADS), 0, st, pdl_enabled(), p,
                    bl_tok(p.T));
  if (pass == FORWARD_SMALL) {
    const size_t smem = ((size_t)p.S * p.E + 1) / 2 * 8 + (size_t)p.S * 8;
    return launch_k(balance_forward_small_kernel<T, VEC, SF, NV>, dim3(1), dim3(BL_SMALL_THREADS), smem, st,
                    pdl_enabled(), p);
  }
  return launch_k(balance_backward_kernel<T, VEC, SF, NV>, grid, dim3(BL_THREADS), 0, st, pdl_enabled(), p,
                  bl_tok(p.T));
}
template <typename T, bool VEC, int SF>
cudaError_t launch_nv(Pass pass, const BalanceParams& p, cudaStream_t st) {
  if (p.E <= 128) return launch_pass<T, VEC, SF, 1>(pass, p, st);
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
  DSV4_CHECK_ARG(n_tokens <= 0x7fffffff / topk, "n_tokens * topk must be below 2^31: picks are counted in 32 bits");
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
  if (n_tokens <= BL_SMALL_TOKENS && (int64_t)n_seqs * (n_experts + 2) <= BL_SMALL_COUNTS) {
    DSV4_CUDA_CHECK(launch(FORWARD_SMALL, dtype, p, st));
    return DSV4_OK;
  }
  const int64_t n16 = bl_layout(n_tokens, n_experts, n_seqs).rows / 16;   // head, info, histogram
  const unsigned zc = (unsigned)std::min<int64_t>((n16 + BL_THREADS - 1) / BL_THREADS, 148 * 4);
  DSV4_CUDA_CHECK(launch_k(balance_zero_kernel, dim3(zc), dim3(BL_THREADS), 0, st, pdl_enabled(),
                           static_cast<int4*>(workspace), n16));
  if (n_tokens > 0)
    DSV4_CUDA_CHECK(launch_k(balance_count_kernel, dim3((unsigned)((n_tokens + BL_COUNT_TOK - 1) / BL_COUNT_TOK)),
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
