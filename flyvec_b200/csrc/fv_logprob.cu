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
// first one's shared memory) streams a row with 16-byte loads, four in flight per thread.  A thread takes the maximum of
// the four words first and rescales its sums once for all their elements, without a branch; an element then costs a
// widening, half a compare, half a subtraction and product (packed), a clamp, ex2 and half of each accumulation.  The
// largest element's 1 is taken out afterwards: one warp reads the words of the thread that saw it once more.  The best
// `top` alternatives cost no second pass over the row either: the threads' maxima give a lower bound of the row's
// top-th largest element, only the threads whose maximum reaches it (about 2 top of 256) have anything to offer, and
// their words are read again (L2).  The few candidates are ranked by counting (value first, then the lower index).
// Rows of at most 1024 elements go to one warp each.
//
// 10000 x 20000 bf16: 73 us (5.5 TB/s) without alternatives, bound by the issue of ex2 and the arithmetic around it; 97 us with
// ten, whose search (two more barriers, a second trip to L2) hides only in part behind the other blocks' rows.  4096 x 50000
// float: 131 us (6.2 TB/s) and 158 us with twenty.  1280 threads per SM: 1024 are 5 % slower, 1536 spill.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "fv_ops.h"

namespace cg = cooperative_groups;

namespace fvo {
namespace {

constexpr int LP_MAX_TOP = 64;
constexpr int LP_CAND = 1024;      // candidates a block can hold at once
constexpr int LP_SMALL = 1024;     // rows up to here: one warp
constexpr int LP_THREADS = 256;    // largest block, and that of every cluster
constexpr int LP_SLOTS = 16;       // batches of a thread whose maxima are kept apart
constexpr int LP_LIST = 256;       // batches that can be listed for their candidates
constexpr float LP_MAX_BETA = 0x1p127f; // its product with log2(e) is still a float
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

typedef unsigned long long u64;

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

// A thread's running sums while it streams its elements: m their maximum (NaN once there was one), s the sum of
// exp(beta (x - m)) and a the sum of exp(.) times the exponent, both over ALL elements including the largest.  The
// accumulators are pairs, so that the packed float instructions do two elements at a time.
struct Stream {
  float m;
  float2 s, a;
};
// largest element (NaN if there is one) of N 16-byte words
template <typename T, int N>
__device__ __forceinline__ float words_max(const uint4 (&q)[N]) {
  if constexpr (sizeof(T) == 4) {
    float m = -CUDART_INF_F;
#pragma unroll
    for (int u = 0; u < N; ++u)
      m = max_nan(m, max_nan(max_nan(__uint_as_float(q[u].x), __uint_as_float(q[u].y)), max_nan(__uint_as_float(q[u].z), __uint_as_float(q[u].w))));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    auto two = [](unsigned w) { return *reinterpret_cast<T2*>(&w); };
    T2 m = two(q[0].x);
#pragma unroll
    for (int u = 0; u < N; ++u) m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(two(q[u].x), two(q[u].y)), __hmax2_nan(two(q[u].z), two(q[u].w))));
    const float2 f = widen2<T>(*reinterpret_cast<unsigned*>(&m));
    return max_nan(f.x, f.y);
  }
}
// log2(e) beta (x - m) of a pair, kept finite: below -200 its exp is 0, and 0 times it has to stay 0
__device__ __forceinline__ float2 exponents(float2 x, float minus_m, float bl2) {
  float2 d = mul2(add2(x, make_float2(minus_m, minus_m)), make_float2(bl2, bl2));
  d.x = max_nan(d.x, -200.f);
  d.y = max_nan(d.y, -200.f);
  return d;
}
// the same from the i-th pair of a word: 16-bit elements are widened by the subtraction itself
template <typename T>
__device__ __forceinline__ float2 exponents_of(const uint4& q, int i, float minus_m, float bl2) {
  float2 x;
  if constexpr (sizeof(T) == 4) {
    x = add2(pair_of<T>(q, i), both(minus_m));
  } else {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
    const unsigned short lo = (unsigned short)w[i], hi = (unsigned short)(w[i] >> 16);
    if constexpr (std::is_same<T, __half>::value) {
      asm("add.f32.f16 %0, %1, %2;" : "=f"(x.x) : "h"(lo), "f"(minus_m));
      asm("add.f32.f16 %0, %1, %2;" : "=f"(x.y) : "h"(hi), "f"(minus_m));
    } else {
      asm("add.f32.bf16 %0, %1, %2;" : "=f"(x.x) : "h"(lo), "f"(minus_m));
      asm("add.f32.bf16 %0, %1, %2;" : "=f"(x.y) : "h"(hi), "f"(minus_m));
    }
  }
  float2 d = mul2(x, both(bl2));
  d.x = max_nan(d.x, -200.f);
  d.y = max_nan(d.y, -200.f);
  return d;
}
// the k-th element of a word in registers
template <typename T>
__device__ __forceinline__ float element_of(const uint4& q, int k) {
  constexpr int PER = 4 / (int)sizeof(T);
  const int i = k / PER;
  const unsigned w = i < 2 ? (i == 0 ? q.x : q.y) : (i == 2 ? q.z : q.w);
  if constexpr (PER == 1)
    return __uint_as_float(w);
  else
    return k & 1 ? widen2<T>(w).y : widen2<T>(w).x;
}
// N words of elements: one rescaling for all of them, without a branch, then two elements per step.  Returns their
// maximum.
template <typename T, int N>
__device__ __forceinline__ float take(Stream& t, const uint4 (&q)[N], float bl2) {
  const float big = words_max<T, N>(q), m = max_nan(t.m, big), m0 = m == -CUDART_INF_F ? 0.f : m;
  const float delta = max_nan((t.m - m0) * bl2, -200.f), e = ex2(delta);
  const float2 e2 = make_float2(e, e);
  t.a = mul2(fma2(make_float2(delta, delta), t.s, t.a), e2);
  t.s = mul2(t.s, e2);
  t.m = m;
#pragma unroll
  for (int u = 0; u < N; ++u)
#pragma unroll
    for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
      const float2 d = exponents_of<T>(q[u], i, -m0, bl2), z = make_float2(ex2(d.x), ex2(d.y));
      t.s = add2(t.s, z);
      t.a = fma2(z, d, t.a);
    }
  return big;
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
// A warp's r-th largest of its lanes' keys (0 if fewer lanes hold anything).
__device__ __forceinline__ unsigned warp_rth(unsigned key, int r) {
  unsigned best = 0;
  for (int k = 0; k < r; ++k) {
    best = __reduce_max_sync(FULL, key);
    if ((threadIdx.x & 31) == __ffs(__ballot_sync(FULL, key == best)) - 1) key = 0;
  }
  return best;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1280 / THREADS)
    k_log_probs(const T* __restrict__ logits, int64_t xs, int64_t V, const void* __restrict__ targets, int t64, float beta, int top,
                int parts, RowOut out) {
  constexpr int VEC = Row<T>::VEC, WARPS = THREADS / 32;
  __shared__ unsigned warp_key[WARPS], warp_tau[WARPS];
  __shared__ float2 warp_sum2[WARPS];
  __shared__ Part all_part[8];
  __shared__ u64 cand[LP_CAND];
  __shared__ u64 best[LP_MAX_TOP];
  __shared__ u64 gathered[THREADS == LP_THREADS ? 8 * LP_MAX_TOP : 1];  // clusters have blocks of LP_THREADS
  __shared__ float slot_max[LP_SLOTS][THREADS];
  __shared__ unsigned short listed[LP_LIST];
  __shared__ unsigned count, n_listed, tau_s, warp_n[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = parts == 1 ? (int64_t)blockIdx.x : blockIdx.x / parts;
  const int rank = (int)(blockIdx.x - row * parts);
  const Row<T> rw(logits + row * xs, V);
  const float bl2 = beta * LOG2E;
  // this block's vectors [v0, v0 + nv); the first block of a cluster also has the single elements
  const int64_t v0 = parts == 1 ? 0 : rw.nvec * rank / parts;
  const int nv = (int)((parts == 1 ? rw.nvec : rw.nvec * (rank + 1) / parts) - v0);
  const uint4* __restrict__ vecs = reinterpret_cast<const uint4*>(rw.x + rw.vec_at(v0));
  const int ends = rank == 0 ? rw.ends : 0;
  cg::cluster_group cluster = cg::this_cluster();
  if (parts > 1) cluster.barrier_arrive();
  long long t = -1;
  float xt = 0.f;
  if (tid == 0) {
    count = n_listed = 0;
    if (rank == 0) {
      t = target_of(targets, t64, row);
      xt = value_at(rw.x, V, t);
    }
  }
  Stream st{-CUDART_INF_F, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  constexpr int U = 4;  // loads in flight per thread
  int i = tid, batch = 0;
  // the largest element of each batch of U words, for finding the candidates again
  auto note = [&](float big) {
    if (top > 0) {
      float* at = &slot_max[batch % LP_SLOTS][tid];
      *at = batch < LP_SLOTS ? big : max_nan(*at, big);
      ++batch;
    }
  };
  for (; i + (U - 1) * THREADS < nv; i += U * THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = vecs[i + u * THREADS];
    note(take<T, U>(st, q, bl2));
  }
  if (i < nv) {  // the last words together; what is missing reads as masked
    uint4 q[U - 1];
    const unsigned none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int u = 0; u < U - 1; ++u) q[u] = i + u * THREADS < nv ? vecs[i + u * THREADS] : make_uint4(none, none, none, none);
    note(take<T, U - 1>(st, q, bl2));
  }
  if (tid < ends) {  // a single element, as if the others of its word were masked
    const float x = to_f<T>(rw.x[rw.end_at(tid)]);
    const float m = max_nan(st.m, x), m0 = m == -CUDART_INF_F ? 0.f : m;
    const float delta = max_nan((st.m - m0) * bl2, -200.f), e = ex2(delta);
    const float d = max_nan((x - m0) * bl2, -200.f), z = ex2(d);
    st.a = make_float2(fmaf(z, d, fmaf(delta, st.s.x, st.a.x) * e), fmaf(delta, st.s.y, st.a.y) * e);
    st.s = make_float2(fmaf(st.s.x, e, z), st.s.y * e);
    st.m = m;
  }
  // largest key this thread saw; 0 if it saw nothing
  const unsigned my_key = tid < ends || tid < nv ? key_of(st.m) : 0u;
  const unsigned wk = __reduce_max_sync(FULL, my_key);
  if (lane == 0) warp_key[warp] = wk;
  if (top > 0) {
    // A lower bound of the top-th largest element: the warps whose lanes all hold elements have, between them, `top`
    // lanes whose maxima reach the smallest of the warps' r-th largest, r = top / warps.
    const int full = min(WARPS, nv >> 5);
    const int r = full ? (top + full - 1) / full : 33;
    unsigned rth = 0;
    if (r <= 32) rth = warp_rth(my_key, r);
    const bool many = __popc(__ballot_sync(FULL, my_key == rth)) > 16;
    if (lane == 0) {
      warp_tau[warp] = warp < full ? rth : r <= 32 ? 0xffffffffu : 0u;
      warp_n[warp] = many;
    }
  }
  __syncthreads();
  unsigned block_key = 0, tau = 0xffffffffu;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    block_key = max(block_key, warp_key[w]);
    if (top > 0) tau = min(tau, warp_tau[w]);
  }
  // Half a warp's maxima equal to the bound: a masked or constant row.  Only what lies above it is offered then, and
  // its equals are taken in the order of their indices.
  bool strict = false;
  if (top > 0) {
#pragma unroll
    for (int w = 0; w < WARPS; ++w) strict = strict || (warp_tau[w] == tau && warp_n[w]);
  }
  tau = max(tau, 1u);
  // The sums relative to the block's maximum, without the largest element's own 1: its thread (the first of the first
  // warp that holds it) leaves its sum out, and its warp reads that thread's elements again.
  const float M = value_of(block_key), M0 = M == -CUDART_INF_F ? 0.f : M;
  float r_sum, a_sum;
  {
    const float delta = max_nan((st.m - M0) * bl2, -200.f), e = ex2(delta), s = st.s.x + st.s.y;
    r_sum = s * e;
    a_sum = fmaf(delta, s, st.a.x + st.a.y) * e;
  }
  bool first = wk == block_key && block_key != 0u && M < CUDART_INF_F && M > -CUDART_INF_F;
#pragma unroll
  for (int w = 0; w < WARPS; ++w)
    if (w < warp && warp_key[w] == block_key) first = false;
  if (first) {
    const int owner_lane = __ffs(__ballot_sync(FULL, my_key == block_key)) - 1, owner = warp * 32 + owner_lane;
    if (lane == owner_lane) r_sum = 0.f;
    bool taken = false;  // the largest element itself has been left out
    if (owner < ends) {
      const float x = to_f<T>(rw.x[rw.end_at(owner)]);
      taken = x == M;
      if (!taken && lane == 0) r_sum += ex2(max_nan((x - M0) * bl2, -200.f));
    }
    for (int base = owner; base < nv; base += 32 * THREADS) {
      const int v = base + lane * THREADS;
      uint4 q = make_uint4(0, 0, 0, 0);
      const bool live = v < nv;
      if (live) q = vecs[v];
      bool has = false;
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 x = pair_of<T>(q, k);
        has = has || (live && (x.x == M || x.y == M));
      }
      const unsigned who = __ballot_sync(FULL, has);
      bool skip = !taken && who && lane == __ffs(who) - 1;
      taken = taken || who;
      if (live) {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const float2 x = pair_of<T>(q, k), d = exponents(x, -M0, bl2);
          if (skip && x.x == M)
            skip = false;
          else
            r_sum += ex2(d.x);
          if (skip && x.y == M)
            skip = false;
          else
            r_sum += ex2(d.y);
        }
      }
    }
  }
  r_sum = warp_sum(r_sum);
  a_sum = warp_sum(a_sum);
  if (lane == 0) warp_sum2[warp] = make_float2(r_sum, a_sum);
  int mine = 0;  // how many of the row's best this block has to offer
  unsigned n_cand = 0;
  bool ties = false;
  if (top > 0) {
    mine = (int)min((int64_t)top, (int64_t)nv * VEC + ends);
    for (bool again = false;; again = true) {
      // offer: elements with key >= tau (strict: > tau)
      const u64 floor_key = (u64)tau + (strict ? 1 : 0);
      const float floor_value = value_of(tau);
      auto offer = [&](float x, int64_t at) {
        const unsigned k = key_of(x);
        if (k >= floor_key) {
          const unsigned slot = atomicAdd(&count, 1u);
          if (slot < LP_CAND) cand[slot] = cand_of(k, (unsigned)at);
        }
      };
      auto offer_word = [&](int v) {
        const uint4 one[1] = {vecs[v]};
        if (words_max<T, 1>(one) < floor_value) return;
        unsigned hits = 0;
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
          const float2 x = pair_of<T>(one[0], k);
          hits |= (x.x < floor_value ? 0u : 1u << 2 * k) | (x.y < floor_value ? 0u : 2u << 2 * k);
        }
        for (; hits; hits &= hits - 1) {
          const int k = __ffs(hits) - 1;
          offer(element_of<T>(one[0], k), rw.vec_at(v0 + v) + k);
        }
      };
      if (tid < ends) offer(to_f<T>(rw.x[rw.end_at(tid)]), rw.end_at(tid));
      if (!again) {
        // the batches that reach the bound are listed, then their words are dealt to all threads
        if (my_key >= floor_key) {
          for (int b = 0; b < min(batch, LP_SLOTS); ++b)
            if (!(slot_max[b][tid] < floor_value) && key_of(slot_max[b][tid]) >= floor_key) {
              const unsigned place = atomicAdd(&n_listed, 1u);
              if (place < LP_LIST) listed[place] = (unsigned short)(tid * LP_SLOTS + b);
            }
        }
        __syncthreads();
        const int n = (int)n_listed;
        if (n <= LP_LIST) {
          for (int w = tid; w < n * U; w += THREADS) {
            const int e = listed[w / U];
            for (int v = e / LP_SLOTS + (e % LP_SLOTS * U + w % U) * THREADS; v < nv; v += LP_SLOTS * U * THREADS) offer_word(v);
          }
        }
      } else {
        unsigned holds = __ballot_sync(FULL, my_key >= floor_key);
        for (; holds; holds &= holds - 1)
          for (int v = warp * 32 + __ffs(holds) - 1 + lane * THREADS; v < nv; v += 32 * THREADS) offer_word(v);
      }
      __syncthreads();
      n_cand = count;
      if (!again && n_listed > LP_LIST) {  // not all were listed: again, all words of the threads that reach the bound
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
        continue;
      }
      if (n_cand <= LP_CAND) {
        // ties at tau that did not fit are taken below in the order of their indices
        ties = strict && n_cand < (unsigned)mine;
        break;
      }
      __syncthreads();
      if (tid == 0) count = 0;
      if (strict) {  // more than fit lie above tau: the top-th largest of those held is a higher bound
        for (int c = tid; c < LP_CAND; c += THREADS) {
          const u64 me = cand[c];
          int above = 0;
          for (int j = 0; j < LP_CAND; ++j) above += cand[j] > me;
          if (above == mine - 1) tau_s = (unsigned)(me >> 32);
        }
      }
      __syncthreads();
      if (strict) tau = tau_s;
      strict = !strict;
    }
    if (ties || parts > 1) {
      for (int c = tid; c < (int)n_cand; c += THREADS) {
        const u64 me = cand[c];
        int above = 0;
        for (int j = 0; j < (int)n_cand; ++j) above += cand[j] > me;
        if (above < mine) best[above] = me;
      }
    }
    if (ties) {  // the first elements equal to tau, by index: the single ones at the front, the vectors', those at the end
      int got = (int)n_cand;
      const int64_t lo = rank == 0 ? 0 : rw.vec_at(v0), hi = rw.vec_at(v0 + nv);
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
    if (ties || parts > 1) __syncthreads();
  } else {
    __syncthreads();
  }
  Part p{M, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    p.r += warp_sum2[w].x;
    p.a += warp_sum2[w].y;
  }
  if (!(M < CUDART_INF_F)) p.r = CUDART_NAN_F;
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
      for (int k = 0; k < parts; ++k) {  // how many of list k are larger: halving
        int lo = 0, hi = top;
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (gathered[k * LP_MAX_TOP + mid] > me)
            lo = mid + 1;
          else
            hi = mid;
        }
        above += lo;
      }
      if (above < top) best[above] = me;
    }
    __syncthreads();
  }
  if (tid != 0 && tid >= (ties || parts > 1 ? top : (int)n_cand)) return;
  const RowScalars s = finish(p);
  if (tid == 0) write_row(out, row, p, s, xt, t, V, beta);
  auto write_top = [&](int place, u64 me) {
    out.top_ids[row * top + place] = (int32_t)~(unsigned)me;
    out.top_lp[row * top + place] = log_p(s, value_of((unsigned)(me >> 32)), beta);
  };
  if (ties || parts > 1) {
    for (int c = tid; c < top; c += THREADS) write_top(c, best[c]);
  } else {
    for (int c = tid; c < (int)n_cand; c += THREADS) {
      const u64 me = cand[c];
      int above = 0;
      for (int j = 0; j < (int)n_cand; ++j) above += cand[j] > me;
      if (above < top) write_top(above, me);
    }
  }
}

// ---- forward, one warp per row ----------------------------------------------------------------------
// The row stays in registers, element lane + 32 e in x[e].  The top-th largest key is found bit by bit with warp
// counts; what lies above it, and as many elements equal to it as are needed in the order of their indices, are the
// candidates, exactly `top` of them.
template <typename T, int E>  // V <= 32 * E
__global__ void __launch_bounds__(128)
    k_log_probs_warp(const T* __restrict__ logits, int64_t xs, int64_t rows, int V, const void* __restrict__ targets, int t64,
                     float beta, int top, RowOut out) {
  __shared__ u64 cand_all[4][LP_MAX_TOP];
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  u64* cand = cand_all[threadIdx.x >> 5];
  const T* xr = logits + row * xs;
  const float bl2 = beta * LOG2E;
  const long long t = target_of(targets, t64, row);
  const float xt = value_at(xr, V, t);
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = lane + 32 * e;
    x[e] = c < V ? to_f<T>(xr[c]) : -CUDART_INF_F;
  }
  float m = -CUDART_INF_F, bad = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    m = fmaxf(m, x[e]);
    if (!(x[e] < CUDART_INF_F)) bad = CUDART_NAN_F;
  }
  float wm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(FULL, wm, o));
  // the first element equal to the maximum stays out of the sum
  bool own = lane == __ffs(__ballot_sync(FULL, m == wm)) - 1;
  Part p{wm, bad, 0.f};
  if (wm != -CUDART_INF_F) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = max_nan((x[e] - wm) * bl2, -200.f);
      float z = ex2(d);
      if (own && x[e] == wm) {
        own = false;
        z = 0.f;
      }
      p.r += z;
      p.a = fmaf(z, d, p.a);
    }
  }
  p.r = warp_sum(p.r);
  p.a = warp_sum(p.a);
  const RowScalars s = finish(p);
  if (lane == 0) write_row(out, row, p, s, xt, t, V, beta);
  if (top == 0) return;
  // 16-bit elements differ in the leading bits of their keys alone
  constexpr int DROP = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  unsigned key[E];
#pragma unroll
  for (int e = 0; e < E; ++e) key[e] = lane + 32 * e < V ? key_of(x[e]) >> DROP : 0u;
  unsigned tau = 0;
  for (int b = 31 - DROP; b >= 0; --b) {
    const unsigned c = tau | 1u << b;
    unsigned n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) n += key[e] >= c;
    n = __reduce_add_sync(FULL, n);
    if (n >= (unsigned)top) tau = c;
    if (n == (unsigned)top) break;  // exactly these
  }
  const unsigned below = (1u << lane) - 1;
  int n = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool take = key[e] > tau;
    const unsigned v = __ballot_sync(FULL, take);
    if (take) cand[n + __popc(v & below)] = cand_of(key_of(x[e]), (unsigned)(lane + 32 * e));
    n += __popc(v);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool take = key[e] == tau;
    const unsigned v = __ballot_sync(FULL, take);
    const int slot = n + __popc(v & below);
    if (take && slot < top) cand[slot] = cand_of(key_of(x[e]), (unsigned)(lane + 32 * e));
    n += __popc(v);
  }
  __syncwarp();
  for (int c = lane; c < top; c += 32) {
    const u64 me = cand[c];
    int above = 0;
    for (int j = 0; j < top; ++j) above += cand[j] > me;
    out.top_ids[row * top + above] = (int32_t)~(unsigned)me;
    out.top_lp[row * top + above] = log_p(s, value_of((unsigned)(me >> 32)), beta);
  }
}

// ---- backward ---------------------------------------------------------------------------------------
struct GradRow {
  float m, log_z, h, g, gh, beta, bl2, lz2, c0, c1;
  bool empty;  // nothing but -inf: no gradient
};
// Every element but the token's own, two at a time, in powers of two: l = log2 p, d = p (c0 + c1 l) with
// c0 = -beta (g + g_H H) and c1 = -beta g_H log(2).  Below 2^-200 p is 0 and l stays finite.
__device__ __forceinline__ float2 grad_of(const GradRow& r, float2 x) {
  float2 l = fma2(add2(x, make_float2(-r.m, -r.m)), make_float2(r.bl2, r.bl2), make_float2(-r.lz2, -r.lz2));
  l.x = max_nan(l.x, -200.f);
  l.y = max_nan(l.y, -200.f);
  const float2 p = make_float2(ex2(l.x), ex2(l.y));
  return mul2(p, fma2(make_float2(r.c1, r.c1), l, make_float2(r.c0, r.c0)));
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
  r.bl2 = beta * LOG2E;
  r.lz2 = r.empty ? 0.f : r.log_z * LOG2E;
  if (r.empty) r.m = 0.f;
  r.c0 = r.empty ? 0.f : -beta * fmaf(r.gh, r.h, r.g);
  r.c1 = r.empty ? 0.f : -beta * r.gh * LN2;
  return r;
}
// A block takes some 1024 words of one row, four to a thread; they are aligned to the gradient, which is dense.  Bound by
// memory: 4096 x 50000, bf16 130 us (6.3 TB/s read and written), float 258 us (6.4 TB/s); half as many words a block 170 us.  float16
// costs more instructions to convert, and the issue slots are 86 % full with bf16: 10000 x 20000 157 us where bf16 takes 133.
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
    dr[at] = from_f<T>(at == t ? grad_at_token(r, x) : grad_of(r, make_float2(x, x)).x);
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
        float2 d[VEC / 2];
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) d[k] = grad_of(r, pair_of<T>(w[u].w, k));
        o.w = word_of<T>(d);
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
    dx[row * V + c] = from_f<T>(c == t ? grad_at_token(r, x) : grad_of(r, make_float2(x, x)).x);
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
  FV_REQUIRE(beta > 0.f && beta <= LP_MAX_BETA, FV_ERR_INVALID, "fv_token_log_probs: beta must be positive and at most 2^127");
  FV_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, FV_ERR_INVALID,
             "fv_token_log_probs: top must be in [0, min(%d, vocabulary size)], got %d", LP_MAX_TOP, top);
  if (rows == 0) return FV_OK;
  FV_REQUIRE(logits && targets && log_prob && entropy && row_max && log_z && (top == 0 || (top_ids && top_log_prob)), FV_ERR_INVALID,
             "fv_token_log_probs: NULL argument");
  OnDevice guard(device);
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
      // a warp's share of the fixed work per row (reductions, candidates) weighs more the shorter the row
      const int64_t words = vocab / Row<T>::VEC;
      e = parts > 1 || words > 4096      ? launch_rows<T, LP_THREADS>(parts, rows, st, x, stride, vocab, targets, targets_int64, beta, top, out)
          : words <= 512 && top <= 16 ? launch_rows<T, 64>(1, rows, st, x, stride, vocab, targets, targets_int64, beta, top, out)
                                      : launch_rows<T, 128>(1, rows, st, x, stride, vocab, targets, targets_int64, beta, top, out);
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
  FV_REQUIRE(beta > 0.f && beta <= LP_MAX_BETA, FV_ERR_INVALID, "fv_token_log_probs_backward: beta must be positive and at most 2^127");
  if (rows == 0) return FV_OK;
  FV_REQUIRE(grad_log_prob && logits && targets && row_max && log_z && (!grad_entropy || entropy) && dlogits, FV_ERR_INVALID,
             "fv_token_log_probs_backward: NULL argument");
  OnDevice guard(device);
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
