// Layer norm over the last axis, forward and backward.
//
//   forward   mean = sum x / D     rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)     y = (x - mean) rstd w + b
//   backward  h = (x - mean) rstd, u = dy w:
//             dx = rstd (u - sum u / D - h sum (u h) / D)      dw = sum_rows dy h      db = sum_rows dy
//
// Both passes are bound by memory: a row is read once and written once.  A group of threads (a warp for short rows, a
// block for longer ones) walks over rows; bulk asynchronous copies bring the next rows into a ring in shared memory
// while it works on one, so that the loads never wait for the reductions.  All sums are float.  The variance is formed
// together with the mean, in one pass about a pivot (the mean of eight of the row's elements), so that a large common
// offset does not cancel it; should the pivot lie more than a standard deviation from the mean (where at most one bit is
// lost) the row is summed again about the mean.
//
// Rows need not start on 16-byte boundaries: the copies take whole 16-byte words around a row, and a thread's columns
// are aligned to the words, not to the row's start.  A group's rows are a multiple of 8 apart, so all of them start
// at the same place in a word and a thread's columns, its weights and its gradient sums stay the same.  Only where dy
// or the output starts at another place in a word than x is that array accessed element by element.
//
// The weight's and the bias's gradients are sums over rows.  A thread keeps the running sums of its columns in
// registers; a block leaves one partial row in the workspace and a second kernel adds the partials in a fixed order (no
// atomics: the same inputs give the same bits).  Rows of more than 32 KB (64 KB in the float forward pass) are read
// again from L2 instead of being held.
//
// 16384 x 4096: forward 16-bit 55 us (4.9 TB/s), float 90 us (6.0 TB/s); backward bf16 82 us and float16 85 us (4.9 and 4.7 TB/s), float
// 132 us (6.1 TB/s).  float is bound by memory.  16-bit rows have twice the elements to a byte, and neither memory nor the issue
// slots are full (55 and 52 % of them issue): the 16 warps an SM that the registers allow wait on fixed latencies, on reads
// of shared memory and, backward, at the barrier of the row's sums.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "fv_ops.h"

namespace fvo {

int sm_count(int device) {
  static int cached[64] = {0};  // written with the same value by every thread that gets here first
  if (device < 0 || device >= 64) return 0;
  if (!cached[device]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 0;
    cached[device] = n;
  }
  return cached[device];
}

long long wait_limit(long long set) {
  static std::atomic<long long> limit{WAIT_LIMIT};
  if (set >= -1) limit.store(set == -1 ? WAIT_LIMIT : set, std::memory_order_relaxed);
  return limit.load(std::memory_order_relaxed);
}

namespace {

constexpr int NORM_WARPS = 4;         // rows a block of the one-warp-per-row form holds
constexpr int NORM_MAX_THREADS = 512; // of the one-block-per-row form
constexpr size_t NORM_SMEM = 208 << 10; // what the blocks of an SM share for their rings

// Sum over the group that owns a row: a warp, or a block through `red` ([2][16][2], the two halves used in turn, so
// that one barrier per sum is enough).
template <bool BLOCK>
__device__ __forceinline__ float2 group_sum2(float a, float b, float (*red)[2], int nwarps) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(FULL, a, o);
    b += __shfl_xor_sync(FULL, b, o);
  }
  if (BLOCK) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) {
      red[threadIdx.x >> 5][0] = a;
      red[threadIdx.x >> 5][1] = b;
    }
    __syncthreads();
    // every thread adds the warps' sums in the same order: two per load, no shuffles
    const float4* all = reinterpret_cast<const float4*>(red);
    a = b = 0.f;
    for (int k = 0; k < (nwarps + 1) / 2; ++k) {
      const float4 f = all[k];
      a += f.x;
      b += f.y;
      if (2 * k + 1 < nwarps) {
        a += f.z;
        b += f.w;
      }
    }
  }
  return make_float2(a, b);
}

template <bool BLOCK>
__device__ __forceinline__ float group_sum(float a, float (*red)[2], int nwarps) {
  return group_sum2<BLOCK>(a, 0.f, red, nwarps).x;
}

template <int VEC>
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t at, const float (&v)[VEC]) {
  if (dtype == FV_F32) {
    float* q = static_cast<float*>(p) + at;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(q + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) q[i] = v[i];
    }
  } else if constexpr (VEC % 4 == 0) {
    unsigned w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const float2 f = make_float2(v[2 * i], v[2 * i + 1]);
      w[i] = dtype == FV_BF16 ? join2<__nv_bfloat16>(f) : join2<__half>(f);
    }
    unsigned char* q = static_cast<unsigned char*>(p) + at * 2;
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
    else
      *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (dtype == FV_BF16)
        static_cast<__nv_bfloat16*>(p)[at + i] = __float2bfloat16_rn(v[i]);
      else
        static_cast<__half*>(p)[at + i] = __float2half_rn(v[i]);
    }
  }
}
__device__ __forceinline__ void store_one(void* p, int dtype, int64_t at, float v) {
  const float one[1] = {v};
  store_as<1>(p, dtype, at, one);
}

// ---- the ring -----------------------------------------------------------------------------------------
__device__ unsigned g_norm_status = 0;

constexpr int RING_MOST = 8;  // stages at most
// Rows as they come into shared memory: `arrays` rows to a stage, each in `pitch` bytes, starting at the row's place in its
// first 16-byte word.
struct Ring {
  unsigned char* base;
  uint64_t* bars;
  int stages, pitch;
};
__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ring_copy(unsigned char* dst, const void* row, int bytes, uint64_t* bar) {
  const uintptr_t from = (uintptr_t)row & ~(uintptr_t)15, to = ((uintptr_t)row + bytes + 15) & ~(uintptr_t)15;
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_addr(dst)), "l"(from),
               "r"((uint32_t)(to - from)), "r"(shared_addr(bar))
               : "memory");
}
__device__ __forceinline__ uint32_t ring_bytes(const void* row, int bytes) {
  return (uint32_t)((((uintptr_t)row + bytes + 15) & ~(uintptr_t)15) - ((uintptr_t)row & ~(uintptr_t)15));
}
__device__ __forceinline__ void ring_expect(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_addr(bar)), "r"(bytes) : "memory");
}
// Bounded wait for a stage.  A thread whose wait ran out is `late`: it goes on without waiting or copying, so that all
// threads of its group keep meeting at the same barriers, and outlasts the copies in flight before it ends; the results
// are invalid.  A limit of 0 cycles makes every thread late from the start.
__device__ __forceinline__ void ring_wait(uint64_t* bar, int parity, long long limit, bool& late) {
  for (long long t0 = 0;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(shared_addr(bar)), "r"(parity)
        : "memory");
    if (ok || late) return;
    const long long now = clock64();
    if (t0 == 0) t0 = now;
    if (now - t0 > limit) {
      atomicOr(&g_norm_status, 1u);
      late = true;
    }
  }
}
// A group's place: its threads, its first row and the distance to its next.
template <bool BLOCK>
struct Group {
  int size, t, warps;
  int64_t first, step;
  __device__ Group() {
    size = BLOCK ? blockDim.x : 32;
    t = BLOCK ? threadIdx.x : threadIdx.x & 31;
    warps = BLOCK ? blockDim.x >> 5 : 1;
    first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * NORM_WARPS + (threadIdx.x >> 5);
    step = (int64_t)gridDim.x * (BLOCK ? 1 : NORM_WARPS);
  }
};
template <bool BLOCK>
__device__ __forceinline__ Ring make_ring(unsigned char* smem, int stages, int pitch, int arrays, int t) {
  Ring r;
  const int w = BLOCK ? 0 : threadIdx.x >> 5;
  r.bars = reinterpret_cast<uint64_t*>(smem) + w * RING_MOST;
  r.base = smem + (BLOCK ? 1 : NORM_WARPS) * RING_MOST * 8 + (size_t)w * stages * pitch * arrays;
  r.stages = stages;
  r.pitch = pitch;
  if (t == 0) {
    for (int s = 0; s < stages; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_addr(r.bars + s)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (BLOCK)
    __syncthreads();
  else
    __syncwarp();
  return r;
}

// A thread's columns: NV words of VEC elements, word t + j size of the row's words; `off` elements of the first word
// precede the row.
template <int VEC, int NV>
struct Columns {
  int off, D, t, size;
  __device__ __forceinline__ int at(int j) const { return (t + j * size) * VEC - off; }  // column of the word's first element
  __device__ __forceinline__ bool any(int j) const { return at(j) < D; }
  __device__ __forceinline__ bool whole(int j) const { return at(j) >= 0 && at(j) + VEC <= D; }
  __device__ __forceinline__ bool has(int j, int i) const { return (unsigned)(at(j) + i) < (unsigned)D; }
};
// a vector of D elements at a thread's columns, as pairs of floats; `none` outside or without a vector
template <typename T, int VEC, int NV>
__device__ __forceinline__ void load_columns(const Columns<VEC, NV>& c, const T* v, float none, float2 (&out)[NV][VEC / 2]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      out[j][i].x = v && c.has(j, 2 * i) ? to_f<T>(v[c.at(j) + 2 * i]) : none;
      out[j][i].y = v && c.has(j, 2 * i + 1) ? to_f<T>(v[c.at(j) + 2 * i + 1]) : none;
    }
}
// the words a thread holds of a row in shared memory; `none` in place of what lies outside the row
template <typename T, int VEC, int NV, bool EDGE>
__device__ __forceinline__ void word_pairs(const Columns<VEC, NV>& c, int j, const Pack<T, VEC>& p, float none, float2 (&out)[VEC / 2]) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) {
    out[i] = pair_of<T>(p.w, i);
    if (EDGE) {
      if (!c.has(j, 2 * i)) out[i].x = none;
      if (!c.has(j, 2 * i + 1)) out[i].y = none;
    }
  }
}

// y in the type `ydt`; EDGE: a row's first or last word may be partial.
template <typename T, int NV, bool BLOCK, bool EDGE>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 32 * NORM_WARPS)
    k_norm(const T* __restrict__ x, int64_t xs, int64_t rows, int D, const T* __restrict__ w, const T* __restrict__ b, float eps,
           void* __restrict__ y, int ydt, float* __restrict__ mean_out, float* __restrict__ rstd_out, int stages, int pitch, long long limit) {
  constexpr int VEC = 16 / (int)sizeof(T);
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float red[2][16][2];
  const Group<BLOCK> g;
  const Ring ring = make_ring<BLOCK>(smem, stages, pitch, 1, g.t);
  const int bytes = D * (int)sizeof(T);
  bool late = false;
  auto fetch = [&](int64_t r, int s) {
    if (r < rows && !late) {
      const T* row = x + r * xs;
      ring_expect(ring.bars + s, ring_bytes(row, bytes));
      ring_copy(ring.base + (size_t)s * pitch, row, bytes, ring.bars + s);
    }
  };
  if (g.t == 0)
    for (int s = 0; s < stages; ++s) fetch(g.first + s * g.step, s);
  if (limit == 0) {
    late = true;
    atomicOr(&g_norm_status, 1u);
  }
  const int off = EDGE ? (int)(((uintptr_t)(x + g.first * xs) & 15) / sizeof(T)) : 0;
  const Columns<VEC, NV> col{off, D, g.t, g.size};
  int turn = 0;
  float2 pw[NV][VEC / 2], pb[NV][VEC / 2];
  load_columns(col, w, 1.f, pw);
  load_columns(col, b, 0.f, pb);
  const int yes = ydt == FV_F32 ? 4 : 2;
  const float inv_n = 1.0f / (float)D;
  // where the words of the group's first row go; the next row's are `hop` further
  unsigned char* out = static_cast<unsigned char*>(y) + (g.first * D + col.at(0)) * yes;
  const int64_t hop = g.step * D * yes;
  const bool aligned = !EDGE || ((uintptr_t)y + (uintptr_t)(g.first * D - off) * yes) % (VEC * yes < 16 ? VEC * yes : 16) == 0;
  // The pivot: mean of a word, or the first element of a row that has no whole word
  const bool wide = !EDGE || D >= 2 * VEC;
  const int pivot_at = EDGE ? (wide ? VEC : off) : 0;
  int s = 0, parity = 0;
  for (int64_t r = g.first; r < rows; r += g.step, out += hop) {
    ring_wait(ring.bars + s, parity, limit, late);
    const T* stage = reinterpret_cast<const T*>(ring.base + (size_t)s * pitch);
    float pivot;
    if (wide) {
      const Pack<T, VEC> p = load_pack<T, VEC>(stage + pivot_at);
      float h[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = to_f<T>(p.e[i]);
#pragma unroll
      for (int k = VEC / 2; k; k /= 2)
#pragma unroll
        for (int i = 0; i < k; ++i) h[i] += h[i + k];
      pivot = h[0] * (1.0f / VEC);
    } else {
      pivot = to_f<T>(stage[pivot_at]);
    }
    float2 v[NV][VEC / 2];
    float shift, var;
    for (bool again = false;; again = true) {
      float2 sum = both(0.f), q = both(0.f);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (col.any(j)) {
          word_pairs<T, VEC, NV, EDGE>(col, j, load_pack<T, VEC>(stage + (g.t + j * g.size) * VEC), pivot, v[j]);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            v[j][i] = add2(v[j][i], both(-pivot));
            sum = add2(sum, v[j][i]);
            q = fma2(v[j][i], v[j][i], q);
          }
        }
      const float2 sums = group_sum2<BLOCK>(sum.x + sum.y, q.x + q.y, red[turn], g.warps);
      turn ^= 1;
      shift = sums.x * inv_n;
      var = fmaf(-shift, shift, sums.y * inv_n);
      if (again || !(shift * shift > var)) break;
      pivot += shift;  // it lay far out: again about the mean
    }
    if (!BLOCK) __syncwarp();
    if (g.t == 0) fetch(r + stages * g.step, s);  // every thread has its part of the stage in registers
    const float rstd = rsqrtf(max_nan(var, 0.f) + eps), minus = -shift * rstd;
    if (g.t == 0) {
      if (mean_out) mean_out[r] = pivot + shift;
      if (rstd_out) rstd_out[r] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col.any(j)) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float2 u = fma2(fma2(v[j][i], both(rstd), both(minus)), pw[j][i], pb[j][i]);
          o[2 * i] = u.x;
          o[2 * i + 1] = u.y;
        }
        unsigned char* to = out + j * g.size * VEC * yes;
        if (!EDGE || (aligned && col.whole(j))) {
          store_as<VEC>(to, ydt, 0, o);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (col.has(j, i)) store_one(to, ydt, i, o[i]);
        }
      }
    if (++s == stages) {
      s = 0;
      parity ^= 1;
    }
  }
  if (late) outlast_copies();
}

// Rows too long for registers: three passes, the second and third out of L2.
template <typename T>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
    k_norm_long(const T* __restrict__ x, int64_t xs, int64_t rows, int64_t D, const T* __restrict__ w, const T* __restrict__ b,
                float eps, void* __restrict__ y, int ydt, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ __align__(16) float red[2][16][2];
  const int nw = blockDim.x >> 5;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) s += to_f<T>(xr[c]);
    const float mean = group_sum<true>(s, red[0], nw) / (float)D;
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) {
      const float d = to_f<T>(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(group_sum<true>(q, red[1], nw) / (float)D + eps);
    if (threadIdx.x == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) {
      float o[1] = {(to_f<T>(xr[c]) - mean) * rstd};
      if (w) o[0] *= to_f<T>(w[c]);
      if (b) o[0] += to_f<T>(b[c]);
      store_as<1>(y, ydt, r * D + c, o);
    }
  }
}

// dx, and with a weight the block's partial sums of dw and db in part[blockIdx.x][2][D].  16-bit rows of at most two words
// a thread keep h and u in registers between the sums and dx (16384 x 4096: 84 us; formed again from shared memory 106 us);
// with four words, and for float, the registers cost more than the second reading.
template <typename T, int NV, bool BLOCK, bool EDGE>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 32 * NORM_WARPS)
    k_norm_grad(const T* __restrict__ dy, int64_t gs, const T* __restrict__ x, int64_t xs, int64_t rows, int D,
                const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ w, T* __restrict__ dx,
                float* __restrict__ part, int stages, int pitch, long long limit) {
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr bool KEEP = sizeof(T) == 2 && NV <= 2;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(16) float red[2][16][2];
  const Group<BLOCK> g;
  const Ring ring = make_ring<BLOCK>(smem, stages, pitch, 2, g.t);
  const int bytes = D * (int)sizeof(T);
  bool late = false;
  auto fetch = [&](int64_t r, int s) {
    if (r < rows && !late) {
      const T *xr = x + r * xs, *gr = dy + r * gs;
      unsigned char* to = ring.base + (size_t)s * 2 * pitch;
      ring_expect(ring.bars + s, ring_bytes(xr, bytes) + ring_bytes(gr, bytes));
      ring_copy(to, xr, bytes, ring.bars + s);
      ring_copy(to + pitch, gr, bytes, ring.bars + s);
    }
  };
  if (g.t == 0)
    for (int s = 0; s < stages; ++s) fetch(g.first + s * g.step, s);
  if (limit == 0) {
    late = true;
    atomicOr(&g_norm_status, 1u);
  }
  const int off = EDGE ? (int)(((uintptr_t)(x + g.first * xs) & 15) / sizeof(T)) : 0;
  const int goff = EDGE ? (int)(((uintptr_t)(dy + g.first * gs) & 15) / sizeof(T)) : 0;
  const Columns<VEC, NV> col{off, D, g.t, g.size};
  float2 pw[NV][VEC / 2];
  load_columns(col, w, 1.f, pw);
  const float inv_n = 1.0f / (float)D;
  T* out_row = dx + g.first * D + col.at(0);
  const int64_t hop = g.step * D;
  const bool aligned = !EDGE || (uintptr_t)(dx + g.first * D - off) % 16 == 0;
  float2 dw[NV][VEC / 2], db[NV][VEC / 2];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) dw[j][i] = db[j][i] = both(0.f);
  int s = 0, parity = 0, turn = 0;
  float next_mu = 0.f, next_rs = 0.f;
  if (g.first < rows) {
    next_mu = mean[g.first];
    next_rs = rstd[g.first];
  }
  for (int64_t r = g.first; r < rows; r += g.step, turn ^= 1, out_row += hop) {
    const float mu = next_mu, rs = next_rs;
    if (r + g.step < rows) {
      next_mu = mean[r + g.step];
      next_rs = rstd[r + g.step];
    }
    ring_wait(ring.bars + s, parity, limit, late);
    const T* sx = reinterpret_cast<const T*>(ring.base + (size_t)s * 2 * pitch);
    const T* sg = reinterpret_cast<const T*>(ring.base + (size_t)s * 2 * pitch + pitch);
    // h and dy of word j, 0 outside the row
    auto row_values = [&](int j, float2 (&h)[VEC / 2], float2 (&gv)[VEC / 2]) {
      word_pairs<T, VEC, NV, EDGE>(col, j, load_pack<T, VEC>(sx + (g.t + j * g.size) * VEC), mu, h);
      Pack<T, VEC> q;
      if (!EDGE || goff == off) {
        q = load_pack<T, VEC>(sg + (g.t + j * g.size) * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) q.e[i] = col.has(j, i) ? sg[goff + col.at(j) + i] : from_f<T>(0.f);
      }
      word_pairs<T, VEC, NV, EDGE>(col, j, q, 0.f, gv);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) h[i] = mul2(add2(h[i], both(-mu)), both(rs));
    };
    float2 a = both(0.f), q = both(0.f);
    float2 hk[NV][VEC / 2], uk[NV][VEC / 2];
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col.any(j)) {
        float2 (&h)[VEC / 2] = hk[j];
        float2 gv[VEC / 2];
        row_values(j, h, gv);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float2 u = uk[j][i] = mul2(gv[i], pw[j][i]);
          a = add2(a, u);
          q = fma2(u, h[i], q);
          dw[j][i] = fma2(gv[i], h[i], dw[j][i]);
          db[j][i] = add2(db[j][i], gv[i]);
        }
      }
    const float2 sums = group_sum2<BLOCK>(a.x + a.y, q.x + q.y, red[turn], g.warps);
    if (!BLOCK) __syncwarp();
    // all threads are past the row before this one: its stage is free
    if (g.t == 0 && r != g.first) fetch(r + (stages - 1) * g.step, s == 0 ? stages - 1 : s - 1);
    const float ma = sums.x * inv_n, mq = sums.y * inv_n;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col.any(j)) {
        if constexpr (!KEEP) {
          float2 gv[VEC / 2];
          row_values(j, hk[j], gv);
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) uk[j][i] = mul2(gv[i], pw[j][i]);
        }
        float2 d[VEC / 2];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) d[i] = mul2(both(rs), fma2(hk[j][i], both(-mq), add2(uk[j][i], both(-ma))));
        Pack<T, VEC> o;
        o.w = word_of<T>(d);
        T* to = out_row + j * g.size * VEC;
        if (!EDGE || (aligned && col.whole(j))) {
          store_pack<T, VEC>(to, o);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (col.has(j, i)) to[i] = o.e[i];
        }
      }
    if (++s == stages) {
      s = 0;
      parity ^= 1;
    }
  }
  if (late) outlast_copies();
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * D;
  if (BLOCK) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (col.has(j, i)) {
          out[col.at(j) + i] = i & 1 ? dw[j][i / 2].y : dw[j][i / 2].x;
          out[D + col.at(j) + i] = i & 1 ? db[j][i / 2].y : db[j][i / 2].x;
        }
  } else {  // the block's warps one after the other, a fixed order; their copies have all arrived
    float* cols = reinterpret_cast<float*>(smem + NORM_WARPS * RING_MOST * 8);
    for (int k = 0; k < NORM_WARPS; ++k) {
      __syncthreads();
      if ((threadIdx.x >> 5) == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (col.has(j, i)) {
              const int c = col.at(j) + i;
              cols[c] = (k ? cols[c] : 0.f) + (i & 1 ? dw[j][i / 2].y : dw[j][i / 2].x);
              cols[D + c] = (k ? cols[D + c] : 0.f) + (i & 1 ? db[j][i / 2].y : db[j][i / 2].x);
            }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      out[c] = cols[c];
      out[D + c] = cols[D + c];
    }
  }
}

// Long rows: dx alone, then the column sums by k_norm_grad_cols.
template <typename T>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
    k_norm_grad_long(const T* __restrict__ dy, int64_t gs, const T* __restrict__ x, int64_t xs, int64_t rows, int64_t D,
                     const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ w, T* __restrict__ dx) {
  __shared__ __align__(16) float red[2][16][2];
  const int nw = blockDim.x >> 5;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x, turn ^= 1) {
    const T *xr = x + r * xs, *gr = dy + r * gs;
    const float mu = mean[r], rs = rstd[r];
    float a = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) {
      const float u = to_f<T>(gr[c]) * (w ? to_f<T>(w[c]) : 1.f);
      a += u;
      q = fmaf(u, (to_f<T>(xr[c]) - mu) * rs, q);
    }
    const float2 sums = group_sum2<true>(a, q, red[turn], nw);
    const float ma = sums.x / (float)D, mq = sums.y / (float)D;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) {
      const float u = to_f<T>(gr[c]) * (w ? to_f<T>(w[c]) : 1.f);
      dx[r * D + c] = from_f<T>(rs * (u - ma - (to_f<T>(xr[c]) - mu) * rs * mq));
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
    k_norm_grad_cols(const T* __restrict__ dy, int64_t gs, const T* __restrict__ x, int64_t xs, int64_t rows, int64_t D,
                     const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= D) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
    const float g = to_f<T>(dy[r * gs + c]);
    dw = fmaf(g, (to_f<T>(x[r * xs + c]) - mean[r]) * rstd[r], dw);
    db += g;
  }
  part[(int64_t)blockIdx.y * 2 * D + c] = dw;
  part[(int64_t)blockIdx.y * 2 * D + D + c] = db;
}

// out[c] = sum of part[p][c] over p in a fixed order; c runs over dw's and then db's columns.  A block takes 32 columns, four
// to a thread, and 64 partial rows at a time.
template <typename T>
__global__ void __launch_bounds__(512)
    k_norm_grad_reduce(const float* __restrict__ part, int64_t P, int64_t D, T* __restrict__ dw, T* __restrict__ db) {
  column_sums(part, P, 2 * D, [&](int64_t c, float v) {
    if (c < D)
      dw[c] = from_f<T>(v);
    else
      db[c - D] = from_f<T>(v);
  });
}

struct NormPlan {
  bool is_long, block, edge;
  int words;           // 16-byte words per thread
  int threads, stages, pitch;
  int64_t grid;
  size_t smem;
};

// One warp per row while a row fits one (64 bytes a lane at most) and there are rows enough to fill the GPU with warps; else
// one block per row.  Threads hold one or two words each as long as 512 threads suffice.  The ring takes what shared memory
// leaves to the blocks that run side by side.
NormPlan plan_norm(int64_t rows, int64_t D, int dtype, bool grad, bool edge, int sms) {
  NormPlan p{};
  const int64_t es = (int64_t)elem_size(dtype), bytes = D * es;
  const int64_t words = (bytes + 15) / 16 + (edge ? 1 : 0);
  p.edge = edge;
  p.is_long = words > (!grad && dtype == FV_F32 ? 8 : 4) * NORM_MAX_THREADS;
  if (p.is_long) {
    p.block = true;
    p.threads = NORM_MAX_THREADS;
    p.grid = std::min<int64_t>(rows, (int64_t)sms * 4);
    return p;
  }
  const int arrays = grad ? 2 : 1;
  p.pitch = (int)(words * 16 + 15) / 16 * 16;
  p.block = !(words <= 32 || (words <= 128 && rows >= 4 * sms));
  int per_sm, groups = 1;
  if (!p.block) {
    p.words = words <= 32 ? 1 : words <= 64 ? 2 : 4;
    p.threads = 32 * NORM_WARPS;
    groups = NORM_WARPS;
    per_sm = !grad ? 8 : p.words == 4 ? 3 : 6;  // 8192 x 1024 bf16, gradient: 3 blocks 84 us, 4 103 us; 256 columns: 6 91 us, 3 102 us
  } else {
    // 16384 x 4096, forward: bf16 with 4 words 55 us, with 2 60 us; float with 2 words 92 us, with 4 101 us
    p.words = !grad && dtype != FV_F32 ? 4 : 2;
    while (words > (int64_t)p.words * NORM_MAX_THREADS) p.words *= 2;
    p.threads = (int)(((words + p.words - 1) / p.words + 31) / 32 * 32);
    per_sm = std::max(1, std::min(16, (!grad ? 1024 : dtype == FV_F32 ? 768 : 512) / p.threads));
  }
  const int64_t fixed = (int64_t)groups * RING_MOST * 8, stage = (int64_t)groups * arrays * p.pitch;
  while (per_sm > 1 && (int64_t)NORM_SMEM / per_sm < fixed + 2 * stage) --per_sm;
  p.stages = (int)std::max<int64_t>(2, std::min<int64_t>(RING_MOST, ((int64_t)NORM_SMEM / per_sm - fixed) / stage));
  const int64_t all = (rows + groups - 1) / groups;
  p.grid = std::min<int64_t>(all, (int64_t)sms * per_sm);
  // a block's partial sums cost as much as a row or two: four rows to a block at least
  if (grad) p.grid = std::min<int64_t>(p.grid, std::max<int64_t>(std::min<int64_t>(all, sms), all / 4));
  // a group's rows start at the same place in a word when they are a multiple of 8 apart
  if (p.edge && p.grid < all) p.grid = std::max<int64_t>(8, p.grid / 8 * 8);
  p.smem = (size_t)(fixed + stage * p.stages);
  if (grad && !p.block) p.smem = std::max(p.smem, (size_t)(fixed + 2 * D * 4));
  return p;
}

template <typename T, int NV, bool BLOCK, bool EDGE>
cudaError_t launch_norm(const NormPlan& p, cudaStream_t st, const T* x, int64_t xs, int64_t rows, int D, const T* w, const T* b, float eps,
                        void* y, int ydt, float* mean, float* rstd) {
  const auto kernel = k_norm<T, NV, BLOCK, EDGE>;
  static std::atomic<bool> given[64];
  if (cudaError_t e = fv::allow_smem((const void*)kernel, given, p.smem, NORM_SMEM)) return e;
  kernel<<<(unsigned)p.grid, p.threads, p.smem, st>>>(x, xs, rows, D, w, b, eps, y, ydt, mean, rstd, p.stages, p.pitch, wait_limit());
  return cudaGetLastError();
}
template <typename T, int NV, bool BLOCK, bool EDGE>
cudaError_t launch_norm_grad(const NormPlan& p, cudaStream_t st, const T* dy, int64_t gs, const T* x, int64_t xs, int64_t rows, int D,
                             const float* mean, const float* rstd, const T* w, T* dx, float* part) {
  const auto kernel = k_norm_grad<T, NV, BLOCK, EDGE>;
  static std::atomic<bool> given[64];
  if (cudaError_t e = fv::allow_smem((const void*)kernel, given, p.smem, NORM_SMEM)) return e;
  kernel<<<(unsigned)p.grid, p.threads, p.smem, st>>>(dy, gs, x, xs, rows, D, mean, rstd, w, dx, part, p.stages, p.pitch, wait_limit());
  return cudaGetLastError();
}

// The forms that plan_norm chooses: a warp's threads hold one, two or four words; a block's two or four of a gradient, four of a
// 16-bit forward row, two, four or eight of a float one.
template <typename T, bool EDGE, typename... A>
cudaError_t launch_norm_form(const NormPlan& p, A... a) {
  if (!p.block)
    return p.words == 1   ? launch_norm<T, 1, false, EDGE>(p, a...)
           : p.words == 2 ? launch_norm<T, 2, false, EDGE>(p, a...)
                          : launch_norm<T, 4, false, EDGE>(p, a...);
  if constexpr (sizeof(T) == 4) {
    if (p.words == 2) return launch_norm<T, 2, true, EDGE>(p, a...);
    if (p.words == 8) return launch_norm<T, 8, true, EDGE>(p, a...);
  }
  return launch_norm<T, 4, true, EDGE>(p, a...);
}
template <typename T, bool EDGE, typename... A>
cudaError_t launch_norm_grad_form(const NormPlan& p, A... a) {
  if (!p.block)
    return p.words == 1   ? launch_norm_grad<T, 1, false, EDGE>(p, a...)
           : p.words == 2 ? launch_norm_grad<T, 2, false, EDGE>(p, a...)
                          : launch_norm_grad<T, 4, false, EDGE>(p, a...);
  return p.words == 2 ? launch_norm_grad<T, 2, true, EDGE>(p, a...) : launch_norm_grad<T, 4, true, EDGE>(p, a...);
}

int64_t grad_parts(const NormPlan& p, int64_t rows, int64_t D, int sms) {
  if (!p.is_long) return p.grid;
  const int64_t blocks = (D + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)sms * 8 / blocks));
}

// Whole words only: every row of every array starts and ends on a 16-byte boundary.
bool norm_even(int64_t D, size_t es, std::initializer_list<std::pair<const void*, int64_t>> arrays) {
  bool ok = D * (int64_t)es % 16 == 0;
  for (const auto& a : arrays) ok = ok && vec_ok(a.first, a.second, es, 16);
  return ok;
}

}  // namespace
}  // namespace fvo

namespace fvo {
__device__ unsigned g_taken;
__global__ void k_take_status(unsigned* bits) { g_taken = atomicExch(bits, 0u); }
cudaError_t take_status(unsigned* bits, uint32_t* word) {
  cudaError_t e = cudaMemcpy(word, bits, sizeof(uint32_t), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess || !*word) return e;
  k_take_status<<<1, 1>>>(bits);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  return cudaMemcpyFromSymbol(word, g_taken, sizeof(uint32_t));
}
cudaError_t norm_status(uint32_t* word) {
  void* bits = nullptr;
  const cudaError_t e = cudaGetSymbolAddress(&bits, g_norm_status);
  return e != cudaSuccess ? e : take_status(static_cast<unsigned*>(bits), word);
}
}  // namespace fvo

using namespace fvo;

extern "C" {

int fv_layer_norm(int device, void* stream, const void* x, int64_t x_stride, int64_t rows, int64_t cols, int dtype, const void* weight,
                  const void* bias, float eps, void* y, int y_dtype, float* mean, float* rstd) {
  FV_CHECK_DTYPE(dtype, "fv_layer_norm");
  FV_CHECK_DTYPE(y_dtype, "fv_layer_norm");
  FV_REQUIRE(rows >= 0 && cols >= 1 && cols < (1ll << 31), FV_ERR_INVALID, "fv_layer_norm: bad shape [%lld][%lld]", (long long)rows,
             (long long)cols);
  FV_REQUIRE(x_stride >= 0, FV_ERR_INVALID, "fv_layer_norm: negative row stride");
  FV_REQUIRE(eps >= 0.f && std::isfinite(eps), FV_ERR_INVALID, "fv_layer_norm: eps must be finite and not negative");
  FV_REQUIRE(!bias || weight, FV_ERR_INVALID, "fv_layer_norm: a bias needs a weight");
  if (rows == 0) return FV_OK;
  FV_REQUIRE(x && y, FV_ERR_INVALID, "fv_layer_norm: NULL argument");
  OnDevice guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  const size_t es = elem_size(dtype);
  // y is dense; its words (of as many elements as x's) must start on boundaries too
  const bool even = norm_even(cols, es, {{x, x_stride}}) && (uintptr_t)y % 16 == 0;
  const NormPlan p = plan_norm(rows, cols, dtype, false, !even, sms);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  FV_DTYPE_SWITCH(dtype, T, {
    const T *px = static_cast<const T*>(x), *pw = static_cast<const T*>(weight), *pb = static_cast<const T*>(bias);
    if (p.is_long) {
      k_norm_long<T><<<(unsigned)p.grid, p.threads, 0, st>>>(px, x_stride, rows, cols, pw, pb, eps, y, y_dtype, mean, rstd);
      e = cudaGetLastError();
    } else {
      e = p.edge ? launch_norm_form<T, true>(p, st, px, x_stride, rows, (int)cols, pw, pb, eps, y, y_dtype, mean, rstd)
                 : launch_norm_form<T, false>(p, st, px, x_stride, rows, (int)cols, pw, pb, eps, y, y_dtype, mean, rstd);
    }
  });
  FV_CUDA(e);
  return FV_OK;
}

static int norm_grad_plan(int device, const void* dy, int64_t gs, const void* x, int64_t xs, int64_t rows, int64_t cols, int dtype,
                          const void* dx, NormPlan* p, int64_t* parts) {
  const int sms = sm_count(device);
  FV_REQUIRE(sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  *p = plan_norm(rows, cols, dtype, true, !norm_even(cols, elem_size(dtype), {{dy, gs}, {x, xs}, {dx, 0}}), sms);
  *parts = grad_parts(*p, rows, cols, sms);
  return FV_OK;
}

int fv_layer_norm_backward_workspace(int device, int64_t rows, int64_t cols, int dtype, size_t* bytes) {
  FV_CHECK_DTYPE(dtype, "fv_layer_norm_backward_workspace");
  FV_REQUIRE(bytes && rows >= 0 && cols >= 1 && cols < (1ll << 31), FV_ERR_INVALID, "fv_layer_norm_backward_workspace: bad argument");
  // the plan for aligned rows and the one for others may differ in their number of blocks
  const int sms = sm_count(device);
  FV_REQUIRE(sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  int64_t parts = 0;
  for (bool edge : {false, true}) parts = std::max(parts, grad_parts(plan_norm(rows, cols, dtype, true, edge, sms), rows, cols, sms));
  *bytes = (size_t)std::max<int64_t>(parts, 1) * 2 * (size_t)cols * sizeof(float);
  return FV_OK;
}

int fv_layer_norm_backward(int device, void* stream, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int64_t rows,
                           int64_t cols, int dtype, const float* mean, const float* rstd, const void* weight, void* dx, void* dweight,
                           void* dbias, void* workspace, size_t workspace_bytes) {
  FV_CHECK_DTYPE(dtype, "fv_layer_norm_backward");
  FV_REQUIRE(rows >= 0 && cols >= 1 && cols < (1ll << 31), FV_ERR_INVALID, "fv_layer_norm_backward: bad shape [%lld][%lld]",
             (long long)rows, (long long)cols);
  FV_REQUIRE(dy_stride >= 0 && x_stride >= 0, FV_ERR_INVALID, "fv_layer_norm_backward: negative row stride");
  FV_REQUIRE(!weight == !dweight && !weight == !dbias, FV_ERR_INVALID,
             "fv_layer_norm_backward: dweight and dbias go with a weight and not without one");
  FV_REQUIRE(rows == 0 || (dy && x && mean && rstd && dx), FV_ERR_INVALID, "fv_layer_norm_backward: NULL argument");
  if (rows == 0 && !weight) return FV_OK;
  OnDevice guard(device);
  FV_REQUIRE(guard.ok, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    FV_CUDA(cudaMemsetAsync(dweight, 0, (size_t)cols * elem_size(dtype), st));
    FV_CUDA(cudaMemsetAsync(dbias, 0, (size_t)cols * elem_size(dtype), st));
    return FV_OK;
  }
  NormPlan p{};
  int64_t parts = 0;
  if (int rc = norm_grad_plan(device, dy, dy_stride, x, x_stride, rows, cols, dtype, dx, &p, &parts)) return rc;
  const size_t need = (size_t)parts * 2 * (size_t)cols * sizeof(float);
  FV_REQUIRE(!weight || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), FV_ERR_INVALID,
             "fv_layer_norm_backward: the workspace must be 16-byte aligned and hold %llu bytes, got %llu", (unsigned long long)need,
             (unsigned long long)workspace_bytes);
  float* part = weight ? static_cast<float*>(workspace) : nullptr;
  cudaError_t e = cudaSuccess;
  FV_DTYPE_SWITCH(dtype, T, {
    const T *pg = static_cast<const T*>(dy), *px = static_cast<const T*>(x), *pw = static_cast<const T*>(weight);
    T* pd = static_cast<T*>(dx);
    if (p.is_long) {
      k_norm_grad_long<T><<<(unsigned)p.grid, p.threads, 0, st>>>(pg, dy_stride, px, x_stride, rows, cols, mean, rstd, pw, pd);
      if (part)
        k_norm_grad_cols<T><<<dim3((unsigned)((cols + 255) / 256), (unsigned)parts), 256, 0, st>>>(pg, dy_stride, px, x_stride, rows, cols,
                                                                                                  mean, rstd, part);
    } else {
      e = p.edge ? launch_norm_grad_form<T, true>(p, st, pg, dy_stride, px, x_stride, rows, (int)cols, mean, rstd, pw, pd, part)
                 : launch_norm_grad_form<T, false>(p, st, pg, dy_stride, px, x_stride, rows, (int)cols, mean, rstd, pw, pd, part);
    }
    if (part)
      k_norm_grad_reduce<T><<<(unsigned)((2 * cols + 31) / 32), 512, 0, st>>>(part, parts, cols, static_cast<T*>(dweight),
                                                                                       static_cast<T*>(dbias));
  });
  FV_CUDA(e);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // extern "C"
