// Log probabilities of given tokens, with the entropy and the best alternatives of every row, and the gradient.
//
//   s = beta x    M = max x    R = sum over all j but the (first) largest of exp(beta (x_j - M))    logZ = log(1 + R)
//   log p_j = beta (x_j - M) - logZ          H = logZ - sum_j p_j beta (x_j - M)
//   d x_j = beta (g ([j = t] - p_j) - g_H p_j (log p_j + H))
//
// The largest element's own exp(0) = 1 stays out of the running sum R, so a row that is nearly certain keeps its
// digits (log1p instead of log); its maximum goes to the caller beside logZ instead of their sum, so that large
// logits keep theirs in the gradient.  A row in which every element is -inf has log p = -inf, H = 0 and no
// gradient; a row with a NaN or +inf has NaN everywhere but in top_ids, whose order takes NaN as the largest.
//
// Forward: bound by reading the logits once.  A block (for few rows a cluster of 2 to 8 blocks that meet in the
// first one's shared memory) streams a row with 16-byte loads and keeps, per thread, the running maximum, R and
// A = sum e d of the elements it saw, d = log2(e) beta (x - m).  The branch that moves the maximum is rare, so an
// element costs a widening, a compare, a subtraction, a product, ex2 and two accumulations.  The best `top`
// alternatives cost no second pass over the row: the `top`-th largest of the threads' maxima is a lower bound of the
// row's `top`-th largest element, and only the threads above it (about `top` of them) have anything to offer; their
// elements are read again by whole warps.  The few candidates are ranked by counting (value first, then the
// lower index).  Rows of at most 1024 elements go to one warp each.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>

#include "fv_ops.h"

namespace cg = cooperative_groups;

namespace fvo {
namespace {

constexpr int LP_MAX_TOP = 64;
constexpr int LP_CAND = 1024;      // candidates a block can hold at once
constexpr int LP_SMALL = 1024;     // rows up to here: one warp
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

typedef unsigned long long u64;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Order of the elements as unsigned integers: NaN above +inf, -0 equal to +0, 0 below everything.
__device__ __forceinline__ unsigned key_of(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) {
  if (k == 0xffffffffu) return CUDART_NAN_F;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// larger value first, then the lower index
__device__ __forceinline__ u64 cand_of(unsigned key, unsigned idx) { return (u64)key << 32 | (unsigned)~idx; }

// What a set of elements contributes: its maximum m (-inf: none above -inf), R and A relative to m, A in units of
// log 2.  A NaN or +inf among them leaves r = NaN and stays in m.
struct Part {
  float m, r, a;
};
__device__ __forceinline__ Part merge(Part p, Part q, float bl2) {
  if (q.m > p.m) {
    const Part t = p;
    p = q;
    q = t;
  }
  if (q.m == -CUDART_INF_F) {  // nothing in q but possibly a NaN
    p.r += q.r;
    return p;
  }
  const float delta = (q.m - p.m) * bl2, e = ex2(delta), t = 1.0f + q.r;
  p.r = fmaf(e, t, p.r);
  if (e > 0.f) p.a += e * fmaf(delta, t, q.a);
  return p;
}
__device__ __forceinline__ Part warp_merge(Part p, float bl2) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Part q;
    q.m = __shfl_xor_sync(FULL, p.m, o);
    q.r = __shfl_xor_sync(FULL, p.r, o);
    q.a = __shfl_xor_sync(FULL, p.a, o);
    // both sides take the same operand first, so that all lanes end with the same bits
    p = (threadIdx.x & o) ? merge(q, p, bl2) : merge(p, q, bl2);
  }
  return p;
}

// One access's elements into a thread's part.
template <int N>
__device__ __forceinline__ void take(Part& p, const float (&x)[N], float bl2) {
  float big = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) big = max_nan(big, x[i]);
  if (!(big <= p.m) || big == -CUDART_INF_F) {
    if (big == -CUDART_INF_F) return;
    if (p.m != p.m) return;
    if (!(big < CUDART_INF_F)) {  // NaN or +inf: the row has no probabilities
      p.m = big;
      p.r = CUDART_NAN_F;
      return;
    }
    // the maximum moves: what was seen so far, its old maximum included, is scaled to the new one
    if (p.m != -CUDART_INF_F) {
      const float delta = (p.m - big) * bl2, e = ex2(delta), t = 1.0f + p.r;
      p.a = e > 0.f ? e * fmaf(delta, t, p.a) : 0.f;
      p.r = e * t;
    }
    p.m = big;
    bool own = true;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (own && x[i] == big) {
        own = false;
      } else {
        const float d = max_nan((x[i] - big) * bl2, -200.f), e = ex2(d);
        p.r += e;
        p.a = fmaf(e, d, p.a);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = max_nan((x[i] - p.m) * bl2, -200.f), e = ex2(d);  // below 2^-126 e is 0 and d stays finite
    p.r += e;
    p.a = fmaf(e, d, p.a);
  }
}

struct RowOut {
  float *log_prob, *entropy, *row_max, *log_z, *top_lp;
  int32_t* top_ids;
};

// The row's scalars from its part, and the token's log probability.
struct RowScalars {
  float m, log_z;
  bool empty;
};
__device__ __forceinline__ RowScalars finish(const Part& p) {
  RowScalars s;
  const bool bad = p.r != p.r;
  s.empty = !bad && p.m == -CUDART_INF_F;
  s.m = bad ? CUDART_NAN_F : p.m;
  s.log_z = bad ? CUDART_NAN_F : s.empty ? -CUDART_INF_F : log1pf(p.r);
  return s;
}
__device__ __forceinline__ float log_p(const RowScalars& s, float x, float beta) {
  if (s.empty) return -CUDART_INF_F;
  return beta * (x - s.m) - s.log_z;
}
template <typename T>
__device__ __forceinline__ float value_at(const T* x, int64_t V, long long t) {
  return t >= 0 && t < V ? to_f<T>(x[t]) : CUDART_NAN_F;
}
__device__ __forceinline__ void write_row(const RowOut& o, int64_t row, const Part& p, const RowScalars& s, float xt, long long t,
                                          int64_t V, float beta) {
  o.row_max[row] = s.m;
  o.log_z[row] = s.log_z;
  o.entropy[row] = s.empty ? 0.f : s.log_z - p.a * LN2 / (1.0f + p.r);
  // -1 marks padding; any other id outside the vocabulary has no probability
  o.log_prob[row] = t == -1 ? 0.f : t < 0 || t >= V ? CUDART_NAN_F : log_p(s, xt, beta);
}
__device__ __forceinline__ long long target_of(const void* t, int is64, int64_t row) {
  return is64 ? static_cast<const long long*>(t)[row] : (long long)static_cast<const int*>(t)[row];
}

// How a row's elements are dealt to threads: up to 15 single elements before the first and after the last 16-byte
// boundary (one to each of the first threads), whole vectors between them.
template <typename T>
struct Row {
  static constexpr int VEC = 16 / (int)sizeof(T);
  const T* x;
  int head, ends;   // single elements before the vectors, and altogether
  int64_t nvec, V;
  __device__ Row(const T* p, int64_t v) : x(p), V(v) {
    const int off = (int)(((uintptr_t)p & 15) / sizeof(T));
    head = (int)min((int64_t)((VEC - off) % VEC), v);
    nvec = (v - head) / VEC;
    ends = (int)(v - nvec * VEC);
  }
  __device__ int64_t vec_at(int64_t i) const { return head + i * VEC; }
  __device__ int64_t end_at(int i) const { return i < head ? i : nvec * VEC + i; }
};

// ---- forward, one block or one cluster per row ------------------------------------------------------
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
    k_log_probs(const T* __restrict__ logits, int64_t xs, int64_t V, const void* __restrict__ targets, int t64, float beta, int top,
                int parts, RowOut out) {
  constexpr int VEC = Row<T>::VEC, WARPS = THREADS / 32, PER = THREADS / 32;
  __shared__ Part warp_part[WARPS];
  __shared__ Part all_part[8];
  __shared__ unsigned keys[THREADS];
  __shared__ u64 cand[LP_CAND];
  __shared__ u64 best[LP_MAX_TOP];
  __shared__ u64 gathered[8 * LP_MAX_TOP];
  __shared__ unsigned count, tau_s, warp_n[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / parts;
  const int rank = (int)(blockIdx.x - row * parts);
  const Row<T> rw(logits + row * xs, V);
  const float bl2 = beta * LOG2E;
  // this block's vectors [v0, v1); the first block of a cluster also has the single elements
  const int64_t v0 = rw.nvec * rank / parts, v1 = rw.nvec * (rank + 1) / parts;
  const int ends = rank == 0 ? rw.ends : 0;
  cg::cluster_group cluster = cg::this_cluster();
  if (parts > 1) cluster.barrier_arrive();
  long long t = -1;
  float xt = 0.f;
  if (tid == 0 && rank == 0) {
    t = target_of(targets, t64, row);
    xt = value_at(rw.x, V, t);
  }
  Part p{-CUDART_INF_F, 0.f, 0.f};
  if (tid < ends) {
    const float x[1] = {to_f<T>(rw.x[rw.end_at(tid)])};
    take<1>(p, x, bl2);
  }
  constexpr int U = 4;  // loads in flight per thread
  int64_t i = v0 + tid;
  for (; i + (U - 1) * THREADS < v1; i += U * THREADS) {
    Pack<T, VEC> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = load_pack<T, VEC>(rw.x + rw.vec_at(i + u * THREADS));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[k] = to_f<T>(w[u].e[k]);
      take<VEC>(p, x, bl2);
    }
  }
  for (; i < v1; i += THREADS) {
    const Pack<T, VEC> w = load_pack<T, VEC>(rw.x + rw.vec_at(i));
    float x[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) x[k] = to_f<T>(w.e[k]);
    take<VEC>(p, x, bl2);
  }
  // largest key this thread saw; 0 if it saw nothing
  const bool saw = tid < ends || v0 + tid < v1;
  const unsigned my_key = saw ? key_of(p.m) : 0u;
  keys[tid] = my_key;
  p = warp_merge(p, bl2);
  if (lane == 0) warp_part[warp] = p;
  if (tid == 0) count = 0;
  __syncthreads();
  if (warp == 0) {
    Part q{-CUDART_INF_F, 0.f, 0.f};
    if (lane < WARPS) q = warp_part[lane];
    q = warp_merge(q, bl2);
    if (lane == 0) warp_part[0] = q;
    if (top > 0) {  // a lower bound of the top-th largest of the threads' maxima, exact in its leading bits
      unsigned k[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) k[j] = keys[lane + 32 * j];
      unsigned tau = 0;
      constexpr int LOW = sizeof(T) == 2 ? 13 : 8;
      for (int b = 31; b >= LOW; --b) {
        const unsigned c = tau | 1u << b;
        unsigned n = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) n += k[j] >= c;
        if (__reduce_add_sync(FULL, n) >= (unsigned)top) tau = c;
      }
      if (lane == 0) tau_s = max(tau, 1u);
    }
  }
  __syncthreads();
  p = warp_part[0];
  int mine = 0;  // how many of the row's best this block has to offer, in best[]
  if (top > 0) {
    const int64_t have = (v1 - v0) * VEC + ends;
    mine = (int)min((int64_t)top, have);
    unsigned tau = tau_s;
    bool strict = false, ties = false;
    for (;;) {
      // offer: elements with key >= tau (strict: > tau); whole warps read the elements of one thread after another
      const u64 floor_key = (u64)tau + (strict ? 1 : 0);
      unsigned holders = __ballot_sync(FULL, my_key >= floor_key);
      while (holders) {
        const int owner = warp * 32 + __ffs(holders) - 1;
        holders &= holders - 1;
        auto offer = [&](float x, int64_t at) {
          const unsigned k = key_of(x);
          if (k >= floor_key) {
            const unsigned slot = atomicAdd(&count, 1u);
            if (slot < LP_CAND) cand[slot] = cand_of(k, (unsigned)at);
          }
        };
        if (lane == 0 && owner < ends) offer(to_f<T>(rw.x[rw.end_at(owner)]), rw.end_at(owner));
        for (int64_t v = v0 + owner + (int64_t)lane * THREADS; v < v1; v += 32 * THREADS) {
          const Pack<T, VEC> w = load_pack<T, VEC>(rw.x + rw.vec_at(v));
#pragma unroll
          for (int k = 0; k < VEC; ++k) offer(to_f<T>(w.e[k]), rw.vec_at(v) + k);
        }
      }
      __syncthreads();
      const unsigned n = count;
      __syncthreads();
      if (n <= LP_CAND) {
        // ties at tau that did not fit are taken below in the order of their indices
        ties = strict && n < (unsigned)mine;
        break;
      }
      if (tid == 0) count = 0;
      if (!strict) {
        strict = true;
      } else {  // more than fit lie above tau: the top-th largest of those held is a higher bound
        for (int c = tid; c < LP_CAND; c += THREADS) {
          const u64 me = cand[c];
          int above = 0;
          for (int j = 0; j < LP_CAND; ++j) above += cand[j] > me;
          if (above == mine - 1) tau_s = (unsigned)(me >> 32);
        }
        strict = false;
      }
      __syncthreads();
      tau = tau_s;
    }
    const int n = (int)count;
    for (int c = tid; c < n; c += THREADS) {
      const u64 me = cand[c];
      int above = 0;
      for (int j = 0; j < n; ++j) above += cand[j] > me;
      if (above < mine) best[above] = me;
    }
    if (ties) {  // the first elements equal to tau, by index: the single ones at the front, the vectors', those at the end
      int got = n;
      const int64_t lo = rank == 0 ? 0 : rw.vec_at(v0), hi = rw.vec_at(v1);
      for (int phase = 0; phase < 2 && got < mine; ++phase) {
        const int64_t from = phase == 0 ? lo : rw.nvec * VEC + rw.head, to = phase == 0 ? hi : (rank == 0 ? V : 0);
        for (int64_t base = from; base < to && got < mine; base += THREADS) {
          const int64_t at = base + tid;
          const bool eq = at < to && key_of(to_f<T>(rw.x[at])) == tau;
          const unsigned votes = __ballot_sync(FULL, eq);
          if (lane == 0) warp_n[warp] = __popc(votes);
          __syncthreads();
          int before = got, all = 0;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += warp_n[w];
            all += warp_n[w];
          }
          const int slot = before + __popc(votes & ((1u << lane) - 1));
          if (eq && slot < mine) best[slot] = cand_of(tau, (unsigned)at);
          got += all;
          __syncthreads();
        }
      }
    }
    __syncthreads();
  }
  if (parts > 1) {  // everything to the cluster's first block
    cluster.barrier_wait();  // the first block runs: its shared memory may be written
    if (tid == 0) cluster.map_shared_rank(all_part, 0)[rank] = p;
    u64* far = cluster.map_shared_rank(gathered, 0);
    for (int c = tid; c < top; c += THREADS) far[rank * LP_MAX_TOP + c] = c < mine ? best[c] : 0ull;
    cluster.sync();
    if (rank != 0) return;
    p = all_part[0];
    for (int k = 1; k < parts; ++k) p = merge(p, all_part[k], bl2);
    // the lists are sorted: an element's place is the number of larger ones in every list
    const int total = parts * top;
    for (int c = tid; c < total; c += THREADS) {
      const u64 me = gathered[(c / top) * LP_MAX_TOP + c % top];
      if (!me) continue;
      int above = 0;
      for (int k = 0; k < parts; ++k)
        for (int j = 0; j < top; ++j) above += gathered[k * LP_MAX_TOP + j] > me;
      if (above < top) best[above] = me;
    }
    __syncthreads();
  }
  const RowScalars s = finish(p);
  if (tid == 0) write_row(out, row, p, s, xt, t, V, beta);
  for (int c = tid; c < top; c += THREADS) {
    const u64 me = best[c];
    out.top_ids[row * top + c] = (int32_t)~(unsigned)me;
    out.top_lp[row * top + c] = log_p(s, value_of((unsigned)(me >> 32)), beta);
  }
}

// ---- forward, one warp per row ----------------------------------------------------------------------
template <typename T, int E>  // V <= 32 * E
__global__ void __launch_bounds__(128)
    k_log_probs_warp(const T* __restrict__ logits, int64_t xs, int64_t rows, int V, const void* __restrict__ targets, int t64,
                     float beta, int top, RowOut out) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const T* xr = logits + row * xs;
  const float bl2 = beta * LOG2E;
  const long long t = target_of(targets, t64, row);
  const float xt = value_at(xr, V, t);
  float x[E];
  float m = -CUDART_INF_F, bad = 0.f;
  unsigned big = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = lane + 32 * e;
    x[e] = c < V ? to_f<T>(xr[c]) : -CUDART_INF_F;
    m = fmaxf(m, x[e]);
    if (!(x[e] < CUDART_INF_F)) bad = CUDART_NAN_F;
    if (c < V) big = max(big, key_of(x[e]));
  }
  float wm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULL, wm, o));
  // the first element equal to the maximum stays out of the sum
  const unsigned at_max = __ballot_sync(FULL, m == wm);
  bool own = lane == __ffs(at_max) - 1;
  Part p{wm, bad, 0.f};
  if (wm != -CUDART_INF_F) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (own && x[e] == wm) {
        own = false;
      } else {
        const float d = max_nan((x[e] - wm) * bl2, -200.f), z = ex2(d);
        p.r += z;
        p.a = fmaf(z, d, p.a);
      }
    }
  }
  p.r = warp_sum(p.r);
  p.a = warp_sum(p.a);
  const RowScalars s = finish(p);
  if (lane == 0) write_row(out, row, p, s, xt, t, V, beta);
  // the best `top`: each lane holds its best not yet taken
  unsigned taken = 0;
  for (int k = 0; k < top; ++k) {
    const unsigned best = __reduce_max_sync(FULL, big);
    int where = 0x7fffffff;
    if (big == best) {
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (!(taken >> e & 1) && lane + 32 * e < V && key_of(x[e]) == best) where = lane + 32 * e;
    }
    const int at = __reduce_min_sync(FULL, where);
    if (lane == 0) {
      out.top_ids[row * top + k] = at;
      out.top_lp[row * top + k] = log_p(s, value_of(best), beta);
    }
    if (at == where) {
      taken |= 1u << (at >> 5);
      big = 0;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(taken >> e & 1) && lane + 32 * e < V) big = max(big, key_of(x[e]));
    }
  }
}

// ---- backward ---------------------------------------------------------------------------------------
struct GradRow {
  float m, log_z, h, g, gh, beta;
  bool empty;
};
// every element but the token's own
__device__ __forceinline__ float grad_of(const GradRow& r, float x) {
  if (r.empty) return 0.f;
  const float lp = max_nan(fmaf(r.beta, x - r.m, -r.log_z), -200.f);  // below exp(-87) p is 0 and lp stays finite
  return r.beta * -ex2(lp * LOG2E) * fmaf(r.gh, lp + r.h, r.g);
}
// the token's: 1 - p by expm1, which keeps its digits where p is nearly 1
__device__ __forceinline__ float grad_at_token(const GradRow& r, float x) {
  if (r.empty) return 0.f;
  const float d = fmaf(r.beta, x - r.m, -r.log_z), lp = max_nan(d, -200.f);
  return -r.beta * (r.g * expm1f(d) + r.gh * ex2(lp * LOG2E) * (lp + r.h));
}
__device__ __forceinline__ GradRow grad_row(int64_t row, long long t, int64_t V, const float* row_max, const float* log_z,
                                            const float* entropy, const float* g, const float* gh, float beta) {
  GradRow r;
  r.m = row_max[row];
  r.log_z = log_z[row];
  r.h = gh ? entropy[row] : 0.f;
  r.g = t == -1 ? 0.f : t < 0 || t >= V ? CUDART_NAN_F : g[row];
  r.gh = gh ? gh[row] : 0.f;
  r.beta = beta;
  r.empty = r.log_z == -CUDART_INF_F;
  return r;
}
// A block takes `chunk` columns of one row; the vectors are aligned to the gradient, which is dense.
template <typename T>
__global__ void __launch_bounds__(256)
    k_log_probs_grad(const T* __restrict__ logits, int64_t xs, int64_t V, int chunks, const void* __restrict__ targets, int t64,
                     const float* __restrict__ row_max, const float* __restrict__ log_z, const float* __restrict__ entropy,
                     const float* __restrict__ g, const float* __restrict__ gh, float beta, T* __restrict__ dx) {
  constexpr int VEC = Row<T>::VEC, U = 4;
  const int64_t row = blockIdx.x / chunks;
  const int part = (int)(blockIdx.x - row * chunks);
  const T* xr = logits + row * xs;
  T* dr = dx + row * V;
  const Row<T> rw(dr, V);
  const long long t = target_of(targets, t64, row);
  const GradRow r = grad_row(row, t, V, row_max, log_z, entropy, g, gh, beta);
  const int64_t v0 = rw.nvec * part / chunks, v1 = rw.nvec * (part + 1) / chunks;
  const bool same = (((uintptr_t)xr ^ (uintptr_t)dr) & 15) == 0;
  if (part == 0 && (int)threadIdx.x < rw.ends) {
    const int64_t at = rw.end_at(threadIdx.x);
    const float x = to_f<T>(xr[at]);
    dr[at] = from_f<T>(at == t ? grad_at_token(r, x) : grad_of(r, x));
  }
  for (int64_t i0 = v0 + threadIdx.x; i0 < v1; i0 += U * 256) {
    Pack<T, VEC> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * 256;
      if (i < v1) {
        const int64_t at = rw.vec_at(i);
        if (same) {
          w[u] = load_pack_stream<T, VEC>(xr + at);
        } else {
#pragma unroll
          for (int k = 0; k < VEC; ++k) w[u].e[k] = xr[at + k];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i = i0 + u * 256;
      if (i < v1) {
        const int64_t at = rw.vec_at(i);
        const int64_t ahead = t - at;
        Pack<T, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.e[k] = from_f<T>(grad_of(r, to_f<T>(w[u].e[k])));
        if (ahead >= 0 && ahead < VEC) {
#pragma unroll
          for (int k = 0; k < VEC; ++k)
            if (k == ahead) o.e[k] = from_f<T>(grad_at_token(r, to_f<T>(w[u].e[k])));
        }
        store_pack<T, VEC>(dr + at, o);
      }
    }
  }
}
// Short rows: one warp each.
template <typename T>
__global__ void __launch_bounds__(128)
    k_log_probs_grad_warp(const T* __restrict__ logits, int64_t xs, int64_t rows, int V, const void* __restrict__ targets, int t64,
                          const float* __restrict__ row_max, const float* __restrict__ log_z, const float* __restrict__ entropy,
                          const float* __restrict__ g, const float* __restrict__ gh, float beta, T* __restrict__ dx) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const long long t = target_of(targets, t64, row);
  const GradRow r = grad_row(row, t, V, row_max, log_z, entropy, g, gh, beta);
#pragma unroll 4
  for (int c = threadIdx.x & 31; c < V; c += 32) {
    const float x = to_f<T>(logits[row * xs + c]);
    dx[row * V + c] = from_f<T>(c == t ? grad_at_token(r, x) : grad_of(r, x));
  }
}

template <typename T, int THREADS>
cudaError_t launch_rows(int parts, int64_t rows, cudaStream_t st, const T* x, int64_t xs, int64_t V, const void* targets, int t64,
                        float beta, int top, RowOut out) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k_log_probs<T, THREADS>, x, xs, V, targets, t64, beta, top, parts, out);
}

}  // namespace
}  // namespace fvo

using namespace fvo;

extern "C" {

int fv_token_log_probs(int device, void* stream, const void* logits, int64_t stride, int64_t rows, int64_t vocab, int dtype,
                       const void* targets, int targets_int64, float beta, int top, float* log_prob, float* entropy, float* row_max,
                       float* log_z, int32_t* top_ids, float* top_log_prob) {
  FV_CHECK_DTYPE(dtype, "fv_token_log_probs");
  FV_REQUIRE(rows >= 0 && rows < (1ll << 28) && vocab >= 1 && vocab < (1ll << 31) && stride >= 0, FV_ERR_INVALID,
             "fv_token_log_probs: bad shape [%lld][%lld], stride %lld", (long long)rows, (long long)vocab, (long long)stride);
  FV_REQUIRE(beta > 0.f && std::isfinite(beta), FV_ERR_INVALID, "fv_token_log_probs: beta must be positive and finite");
  FV_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, FV_ERR_INVALID,
             "fv_token_log_probs: top must be in [0, min(%d, vocabulary size)], got %d", LP_MAX_TOP, top);
  if (rows == 0) return FV_OK;
  FV_REQUIRE(logits && targets && log_prob && entropy && row_max && log_z && (top == 0 || (top_ids && top_log_prob)), FV_ERR_INVALID,
             "fv_token_log_probs: NULL argument");
  fv::DeviceGuard guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const RowOut out{log_prob, entropy, row_max, log_z, top_log_prob, top_ids};
  cudaError_t e = cudaSuccess;
  FV_DTYPE_SWITCH(dtype, T, {
    const T* x = static_cast<const T*>(logits);
    if (vocab <= LP_SMALL) {
      const unsigned grid = (unsigned)((rows + 3) / 4);
      const int V = (int)vocab;
      if (vocab <= 128)
        k_log_probs_warp<T, 4><<<grid, 128, 0, st>>>(x, stride, rows, V, targets, targets_int64, beta, top, out);
      else if (vocab <= 512)
        k_log_probs_warp<T, 16><<<grid, 128, 0, st>>>(x, stride, rows, V, targets, targets_int64, beta, top, out);
      else
        k_log_probs_warp<T, 32><<<grid, 128, 0, st>>>(x, stride, rows, V, targets, targets_int64, beta, top, out);
      e = cudaGetLastError();
    } else {
      // few rows: a cluster per row, as long as every block keeps two vectors a thread
      int parts = 1;
      while (parts < 8 && rows * parts * 2 <= 2 * sms && vocab / (parts * 2) >= 2 * 256 * Row<T>::VEC) parts *= 2;
      e = launch_rows<T, 256>(parts, rows, st, x, stride, vocab, targets, targets_int64, beta, top, out);
    }
  });
  FV_CUDA(e);
  return FV_OK;
}

int fv_token_log_probs_backward(int device, void* stream, const float* grad_log_prob, const float* grad_entropy, const void* logits,
                                int64_t stride, int64_t rows, int64_t vocab, int dtype, const void* targets, int targets_int64,
                                const float* row_max, const float* log_z, const float* entropy, float beta, void* dlogits) {
  FV_CHECK_DTYPE(dtype, "fv_token_log_probs_backward");
  FV_REQUIRE(rows >= 0 && rows < (1ll << 28) && vocab >= 1 && vocab < (1ll << 31) && stride >= 0, FV_ERR_INVALID,
             "fv_token_log_probs_backward: bad shape [%lld][%lld], stride %lld", (long long)rows, (long long)vocab, (long long)stride);
  FV_REQUIRE(beta > 0.f && std::isfinite(beta), FV_ERR_INVALID, "fv_token_log_probs_backward: beta must be positive and finite");
  if (rows == 0) return FV_OK;
  FV_REQUIRE(grad_log_prob && logits && targets && row_max && log_z && (!grad_entropy || entropy) && dlogits, FV_ERR_INVALID,
             "fv_token_log_probs_backward: NULL argument");
  fv::DeviceGuard guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FV_DTYPE_SWITCH(dtype, T, {
    const T* x = static_cast<const T*>(logits);
    T* dx = static_cast<T*>(dlogits);
    if (vocab <= LP_SMALL) {
      k_log_probs_grad_warp<T><<<(unsigned)((rows + 3) / 4), 128, 0, st>>>(x, stride, rows, (int)vocab, targets, targets_int64, row_max,
                                                                           log_z, entropy, grad_log_prob, grad_entropy, beta, dx);
    } else {
      // 1024 vectors a block: each thread has its four loads in flight once
      const int chunks = (int)std::min<int64_t>((vocab / Row<T>::VEC + 1023) / 1024, (1ll << 31) / rows - 1);
      k_log_probs_grad<T><<<(unsigned)(rows * std::max(chunks, 1)), 256, 0, st>>>(x, stride, vocab, std::max(chunks, 1), targets,
                                                                                  targets_int64, row_max, log_z, entropy, grad_log_prob,
                                                                                  grad_entropy, beta, dx);
    }
  });
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // extern "C"
