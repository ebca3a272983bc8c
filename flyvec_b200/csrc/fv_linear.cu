// Matrix product with bias, activation and residual in its epilogue, and its gradients.
//
//   forward    z = x w^T + b     y = act(z) + residual           x [rows][inner], w [outer][inner]
//   backward   dz = dy act'(z)   dx = dz w     dw = dz^T x     db = sum_rows dz     (the residual's gradient is dy)
//
// All three products are one kernel, k_gemm: D[m][n] = sum_k A[m][k] B[n][k] in 16-bit operands with float accumulators.
// An operand may be stored with k contiguous ("k-major") or with its row index contiguous ("mn-major"), so the
// gradients and transposed weights need no transposition: only the shape of the TMA boxes, the strides in the
// shared-memory descriptor and two bits of the instruction descriptor differ.
//
// k_gemm: one persistent block per SM.  One thread issues TMA loads into a ring of 64-deep k-blocks (192 KB of
// shared memory, 128-byte swizzle), one thread issues tcgen05.mma on them (128 x BN tile, BN = 64, 128 or 256; the
// accumulator sits in TMEM twice, so that the next tile's products run under the previous tile's epilogue), eight
// warps take the accumulator through bias, activation and residual and out by way of shared memory, so that rows
// leave in full 32-byte sectors.  Edges cost nothing extra: TMA fills zeros beyond the tensor, stores are guarded.
// When there are fewer tiles than SMs, 2 to 8 blocks of a cluster share a tile's k range and add their partial
// tiles over distributed shared memory, in rank order (no atomics, no workspace: the same bits every time).
//
// With at most 64 rows (serving) the product is bound by reading w.  One or two rows (up to four where the sums are short)
// are done by plain loads and float FMAs (k_gemv), more by k_gemm with the roles exchanged: w's rows fill the 128-row side of the tile and the few
// rows of x its narrow side.
//
// TMA needs 16-byte aligned rows.  Operands without them are copied once into rows of a multiple of 8 elements
// (k_pack) in the caller's workspace; everything else is read where it lies.
//
// What bounds it: large products the tensor cores under the power limit (8192 x 8192 x 2048, bf16: 178 us, 1.55 PFLOP/s,
// cuBLAS 177 us); with pre-activation, gelu and residual the epilogue (235 us: eight warps take 17 us a tile where the products
// take 13); small ones launch, set-up and drain (about 5 us) and 0.16 us per k-block, the rate at which one thread
// issues loads.  256 x 256 pairs halve what a block reads of B: 0.36 instead of 0.42 us per k-block with all SMs at work.
//
// Roundings to 16 bits: the outputs, and dz before it enters the two products (as tensor-core operands have to be; db
// is formed from the unrounded dz).
//
// Every wait is bounded: a wait that runs out raises a flag (fv_ops_status), the block outlasts what it has in
// flight, frees its TMEM and returns.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "fv_ops.h"

namespace fvo {
namespace {

// ---- activations ------------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;
// exp(-z^2 / 2) and the tail Phi(-|z|) of the normal distribution, by Abramowitz and Stegun's formula 7.1.26 for erfc
// (|error of erf| <= 1.5e-7, shrinking with exp(-z^2 / 2)): two special-function calls a value, the rest two values at a
// time.  az = |z|.  z Phi(z) is off by 2.1e-7 at most (near |z| = 3), by 6e-5 of its value at z = -3 and 5e-4 at -4: nothing beside a
// rounding to 16 bits where the value is large, and no worse at -4 than z (1 + erf) / 2 in floats.
__device__ __forceinline__ float2 normal_tail(float2 z, float2 az, float2& e) {
  const float2 d = fma2(both(0.3275911f * 0.70710678f), az, both(1.0f)), t = make_float2(rcp(d.x), rcp(d.y));
  const float2 l = mul2(mul2(z, z), both(-0.5f * LOG2E));
  e = make_float2(ex2(l.x), ex2(l.y));
  float2 q = fma2(both(0.5f * 1.061405429f), t, both(0.5f * -1.453152027f));
  q = fma2(q, t, both(0.5f * 1.421413741f));
  q = fma2(q, t, both(0.5f * -0.284496736f));
  q = fma2(q, t, both(0.5f * 0.254829592f));
  return mul2(mul2(q, t), e);
}
// |z|, kept finite so that 0 times it stays 0
__device__ __forceinline__ float2 magnitude(float2 z) { return make_float2(min_nan(fabsf(z.x), 1e30f), min_nan(fabsf(z.y), 1e30f)); }
// 1 / (1 + exp(-x))
__device__ __forceinline__ float2 logistic(float2 x) {
  const float2 l = mul2(x, both(-LOG2E)), d = add2(make_float2(ex2(l.x), ex2(l.y)), both(1.0f));
  return make_float2(rcp(d.x), rcp(d.y));
}
constexpr float TANH_A = 0.7978845608f, TANH_B = 0.044715f;  // (1 + tanh u) / 2 = 1 / (1 + exp(-2 u)), u = A (z + B z^3)

template <int ACT>
__device__ __forceinline__ float2 act_value(float2 z) {
  if constexpr (ACT == FV_ACT_RELU) return make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f));
  if constexpr (ACT == FV_ACT_GELU) {  // z Phi(z) = max(z, 0) - |z| Phi(-|z|)
    const float2 az = magnitude(z);
    float2 e;
    const float2 q = normal_tail(z, az, e);
    return fma2(make_float2(-az.x, -az.y), q, make_float2(max_nan(z.x, 0.f), max_nan(z.y, 0.f)));
  }
  if constexpr (ACT == FV_ACT_GELU_TANH)
    return mul2(z, logistic(mul2(z, fma2(mul2(z, z), both(2.0f * TANH_A * TANH_B), both(2.0f * TANH_A)))));
  if constexpr (ACT == FV_ACT_SILU) return mul2(z, logistic(z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float2 act_slope(float2 z) {
  if constexpr (ACT == FV_ACT_RELU)  // NaN for a NaN
    return make_float2(z.x > 0.f ? 1.f : z.x <= 0.f ? 0.f : z.x, z.y > 0.f ? 1.f : z.y <= 0.f ? 0.f : z.y);
  if constexpr (ACT == FV_ACT_GELU) {  // Phi(z) + z phi(z)
    float2 e;
    const float2 q = normal_tail(z, magnitude(z), e);
    const float2 side = make_float2(copysignf(0.5f - q.x, z.x), copysignf(0.5f - q.y, z.y));
    return add2(side, fma2(mul2(make_float2(max_nan(min_nan(z.x, 1e30f), -1e30f), max_nan(min_nan(z.y, 1e30f), -1e30f)), e),
                           both(0.3989422804f), both(0.5f)));
  }
  if constexpr (ACT == FV_ACT_GELU_TANH) {
    // beyond 16 the slope is 0 or 1 to the last bit, and z z would overflow at last
    const float2 y = make_float2(max_nan(min_nan(z.x, 16.f), -16.f), max_nan(min_nan(z.y, 16.f), -16.f)), y2 = mul2(y, y);
    const float2 s = logistic(mul2(y, fma2(y2, both(2.0f * TANH_A * TANH_B), both(2.0f * TANH_A))));
    const float2 r = make_float2(1.0f - s.x, 1.0f - s.y);  // s + y s (1 - s) 2 A (1 + 3 B y^2)
    return fma2(mul2(mul2(y, s), r), fma2(y2, both(6.0f * TANH_A * TANH_B), both(2.0f * TANH_A)), s);
  }
  if constexpr (ACT == FV_ACT_SILU) {
    const float2 y = make_float2(max_nan(z.x, -1e30f), max_nan(z.y, -1e30f)), s = logistic(y);
    return mul2(s, fma2(y, make_float2(1.0f - s.x, 1.0f - s.y), both(1.0f)));
  }
  return both(1.0f);
}
template <int ACT, int N>
__device__ __forceinline__ void act_each(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 y = act_value<ACT>(make_float2(v[i], v[i + 1]));
    v[i] = y.x;
    v[i + 1] = y.y;
  }
}
template <int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
  if (act == FV_ACT_RELU) act_each<FV_ACT_RELU>(v);
  if (act == FV_ACT_GELU) act_each<FV_ACT_GELU>(v);
  if (act == FV_ACT_GELU_TANH) act_each<FV_ACT_GELU_TANH>(v);
  if (act == FV_ACT_SILU) act_each<FV_ACT_SILU>(v);
}

// ---- device-side status -----------------------------------------------------------------------------
__device__ unsigned g_status = 0;

// ---- PTX --------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Waits for the phase of the given parity; false when the limit ran out here or elsewhere in the block.
__device__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* stop, long long limit) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    if (mbar_try(bar, parity)) return true;
    if (*stop) return false;
    if (clock64() - t0 > limit) {
      *stop = 1;
      atomicOr(&g_status, 1u);
      return false;
    }
  }
}
// One thread of a converged warp, in a form that the compiler knows to be one thread: the loads and products below
// take their operands from uniform registers, and under a plain lane == 0 each would be wrapped in a loop over lanes
// (0.285 against 0.199 us per k-block).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {
  uint32_t far;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(addr), "r"(rank));
  return far;
}
__device__ __forceinline__ void mbar_arrive_far(uint32_t far) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(far) : "memory");
}
// PAIR: the copy lands in this block and reports to a barrier of either block of the pair
template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     dst),
                 "l"(map), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(map), "r"(x), "r"(y), "r"(bar)
               : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle; byte offsets in units of 16.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
template <bool PAIR>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// arrives at `bar` (of both blocks of a pair) when the products issued so far are done
template <bool PAIR>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (PAIR)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 lanes (the warp's quarter) x 32 columns
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  uint32_t far;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(addr), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(far) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- the product ------------------------------------------------------------------------------------
constexpr int BM = 128, BK = 64;                 // tile rows, depth of a k-block
constexpr int RING_BYTES = 192 << 10;            // operand ring
constexpr int EPI_WARPS = 8;
constexpr int GEMM_THREADS = 96 + 32 * EPI_WARPS; // loads of A, products, epilogue, loads of B
constexpr int STAGE_OUT = 32 * 128;              // an epilogue warp's staging: 32 rows of 128 bytes
constexpr int GEMM_SMEM = 1024 + RING_BYTES + EPI_WARPS * (STAGE_OUT + 128) + 256;  // + 32 floats of bias a warp

struct GemmParams {
  int64_t m, n;        // rows of A, rows of B
  int kblocks, tiles_m, tiles_n;
  int a_mn, b_mn;      // operand stored with its row index contiguous
  uint32_t idesc;
  int act, out_f32, swap;  // swap: D is stored transposed, out[n][m]; bias runs along m
  int vec_y, vec_z, vec_r; // rows of y, z, residual start on 16-byte boundaries
  const void *bias, *residual;
  void *y, *z;
  int64_t ldr, ldy, ldz;
};
// One launch: one product, or two of the same tile shape whose tiles follow one another (a backward pass's dx and dw, so
// that the second fills the SMs the first leaves idle).
struct GemmMaps {
  CUtensorMap a[2], b[2], y[2];
};
struct GemmJob {
  GemmParams p[2];
  int tiles0, tiles;  // of the first product (the one with the longer sums), of both
  int splits;
  int spare;          // tiles of the second product that cost as much as one of the first
  long long limit;    // cycles of a wait
};
// The k-th tile of place c of `places` (blocks, pairs or clusters); -1 after the last.  The first product's tiles go round
// the places; those that get none in the last round take `spare` tiles of the second product meanwhile, whose other
// tiles go round all places.
__device__ __forceinline__ int tile_of(const GemmJob& j, int c, int k, int places) {
  const int rounds = j.tiles0 / places, rest = j.tiles0 - rounds * places, idle = places - rest;
  if (k < rounds) return c + k * places;
  k -= rounds;
  int i;
  if (c < rest) {
    if (k == 0) return rounds * places + c;
    i = j.spare * idle + c + (k - 1) * places;
  } else {
    i = k < j.spare ? c - rest + k * idle : j.spare * idle + c + (k - j.spare) * places;
  }
  return j.tiles0 + i < j.tiles ? j.tiles0 + i : -1;
}

// Where a tile lies.  Tiles are taken in bands of 16 row tiles, column by column within a band, so that the blocks
// at work at one time share operand tiles in L2.
__device__ __forceinline__ void tile_at(const GemmParams& p, int t, int& tm, int& tn) {
  constexpr int BAND = 16;
  const int per = BAND * p.tiles_n, band = t / per, in = t - band * per;
  const int rows = min(BAND, p.tiles_m - band * BAND);
  tn = in / rows;
  tm = band * BAND + in - tn * rows;
}

// An epilogue warp's staging: 32 rows of 128 bytes, the 16-byte words of row r swizzled with r % 8 as TMA's 128-byte
// swizzle does (so that lanes writing one word of eight rows hit all banks).  A slice of the output is 128 bytes wide: 64
// columns of 16 bits in two halves, or 32 of float.
template <typename T>
__device__ __forceinline__ void stage_row(uint8_t* stage, int row, const float (&v)[32], int half) {
  uint8_t* base = stage + row * 128;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float2 q[4] = {make_float2(v[8 * c], v[8 * c + 1]), make_float2(v[8 * c + 2], v[8 * c + 3]), make_float2(v[8 * c + 4], v[8 * c + 5]),
                         make_float2(v[8 * c + 6], v[8 * c + 7])};
    *reinterpret_cast<uint4*>(base + (((c + 4 * half) ^ (row & 7)) << 4)) = word_of<T>(q);
  }
}
__device__ __forceinline__ void stage_row_f32(uint8_t* stage, int row, const float (&v)[32]) {
  uint8_t* base = stage + row * 128;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(base + ((c ^ (row & 7)) << 4)) = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
}
// The staged rows as a 128-byte wide box of the output; what lies outside the output is not written.
__device__ __forceinline__ void stage_store(const uint8_t* stage, const CUtensorMap* map, int64_t r0, int64_t c0) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"((int)c0), "r"((int)r0),
                 "r"(smem_u32(stage))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}
// before the staging rows are written again
__device__ __forceinline__ void stage_free() {
  if ((threadIdx.x & 31) == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
}
// The same for outputs whose rows do not start on 16-byte boundaries: 32 columns, element by element.
__device__ __forceinline__ void stage_out(const uint8_t* stage, void* out, int64_t ld, int es, int half, int64_t r0, int64_t c0, int64_t rows,
                                          int64_t cols) {
  const int lane = threadIdx.x & 31, at = lane * es + (es == 2 ? 64 * half : 0);
  __syncwarp();
  if (c0 + lane < cols) {
    uint8_t* d = static_cast<uint8_t*>(out) + (r0 * ld + c0 + lane) * es;
    const int n = (int)min((int64_t)32, rows - r0);
#pragma unroll 4
    for (int r = 0; r < n; ++r, d += ld * es) {
      const uint8_t* s = stage + r * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 15);
      if (es == 4)
        *reinterpret_cast<uint32_t*>(d) = *reinterpret_cast<const uint32_t*>(s);
      else
        *reinterpret_cast<uint16_t*>(d) = *reinterpret_cast<const uint16_t*>(s);
    }
  }
  __syncwarp();
}
// One staged half (32 columns of 16 bits) to an array by plain stores; unlike the asynchronous copy it is done with the
// staging rows when it returns.
__device__ __forceinline__ void copy_out(const uint8_t* stage, void* out, int64_t ld, bool vec, int half, int64_t r0, int64_t c0, int64_t rows,
                                         int64_t cols) {
  if (!vec || c0 + 32 > cols) {
    stage_out(stage, out, ld, 2, half, r0, c0, rows, cols);
    return;
  }
  const int lane = threadIdx.x & 31, c = (lane & 3) + 4 * half;
  __syncwarp();
  uint8_t* base = static_cast<uint8_t*>(out) + ((r0 + lane / 4) * ld + c0) * 2 + (lane & 3) * 16;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = lane / 4 + 8 * k;
    if (r0 + r < rows) *reinterpret_cast<uint4*>(base + 16 * k * ld) = *reinterpret_cast<const uint4*>(stage + r * 128 + ((c ^ (r & 7)) << 4));
  }
  __syncwarp();
}
// 32 x 64 16-bit elements of an array: fetched early into registers (eight 16-byte words a lane; rows that do not admit
// them are fetched late, element by element), then put into the staging rows.  What lies outside reads as 0.
__device__ __forceinline__ void fetch_in(uint4 (&w)[8], const void* in, int64_t ld, bool vec, int64_t r0, int64_t c0, int64_t rows,
                                         int64_t cols) {
  const int lane = threadIdx.x & 31;
  if (!vec || c0 + 64 > cols) return;
  const uint8_t* base = static_cast<const uint8_t*>(in) + ((r0 + lane / 8) * ld + c0) * 2 + (lane & 7) * 16;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w[k] = make_uint4(0, 0, 0, 0);
    if (r0 + lane / 8 + 4 * k < rows) w[k] = __ldcs(reinterpret_cast<const uint4*>(base + 8 * k * ld));
  }
}
__device__ __forceinline__ void stage_in(uint8_t* stage, const uint4 (&w)[8], const void* in, int64_t ld, bool vec, int64_t r0, int64_t c0,
                                         int64_t rows, int64_t cols) {
  const int lane = threadIdx.x & 31;
  if (vec && c0 + 64 <= cols) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int r = lane / 8 + 4 * k;
      *reinterpret_cast<uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = w[k];
    }
  } else {
    const uint8_t* base = static_cast<const uint8_t*>(in);
#pragma unroll 4
    for (int r = 0; r < 32; ++r)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c = lane + 32 * h;
        uint16_t v = 0;
        if (r0 + r < rows && c0 + c < cols) v = __ldg(reinterpret_cast<const uint16_t*>(base + ((r0 + r) * ld + c0 + c) * 2));
        *reinterpret_cast<uint16_t*>(stage + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2) = v;
      }
  }
  __syncwarp();
}

template <typename T>
__device__ __forceinline__ void store_one(const GemmParams& p, int64_t r, int64_t c, float v) {  // r, c: row and column of y
  if (p.z) static_cast<T*>(p.z)[r * p.ldz + c] = from_f<T>(v);
  float one[2] = {v, v};
  act_values(one, p.act);
  v = one[0];
  if (p.residual) v += to_f<T>(static_cast<const T*>(p.residual)[r * p.ldr + c]);
  if (p.out_f32)
    static_cast<float*>(p.y)[r * p.ldy + c] = v;
  else
    static_cast<T*>(p.y)[r * p.ldy + c] = from_f<T>(v);
}

// N consecutive rows of column c (the exchanged roles), each lane of a warp a column: the steps one after the other over
// all rows, so that each is a short loop
template <typename T, int N>
__device__ __forceinline__ void store_column(const GemmParams& p, int64_t r, int64_t c, float (&v)[N]) {
  const int n = (int)min((int64_t)N, p.n - r);  // p.n: rows of x
  if (p.bias) {
    const float b = to_f<T>(static_cast<const T*>(p.bias)[c]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += b;
  }
  if (p.z) {
    T* z = static_cast<T*>(p.z) + r * p.ldz + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) z[i * p.ldz] = from_f<T>(v[i]);
  }
  act_values(v, p.act);
  if (p.residual) {
    const T* q = static_cast<const T*>(p.residual) + r * p.ldr + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) v[i] += to_f<T>(q[i * p.ldr]);
  }
  if (p.out_f32) {
    float* y = static_cast<float*>(p.y) + r * p.ldy + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) y[i * p.ldy] = v[i];
  } else {
    T* y = static_cast<T*>(p.y) + r * p.ldy + c;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) y[i * p.ldy] = from_f<T>(v[i]);
  }
}
// four consecutive columns of row r; c is a multiple of 4
template <typename T>
__device__ __forceinline__ void store_four(const GemmParams& p, int64_t r, int64_t c, float (&v)[4]) {
  if (c + 4 > p.n || !p.vec_y || (p.z && !p.vec_z) || (p.residual && !p.vec_r)) {
#pragma unroll 1
    for (int j = 0; j < 4; ++j)
      if (c + j < p.n)
        store_one<T>(p, r, c + j, (j < 2 ? (j ? v[1] : v[0]) : (j == 2 ? v[2] : v[3])) +
                                      (p.bias ? to_f<T>(static_cast<const T*>(p.bias)[c + j]) : 0.f));
    return;
  }
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += to_f<T>(static_cast<const T*>(p.bias)[c + j]);
  }
  Pack<T, 4> o;
  if (p.z) {
#pragma unroll
    for (int j = 0; j < 4; ++j) o.e[j] = from_f<T>(v[j]);
    store_pack<T, 4>(static_cast<T*>(p.z) + r * p.ldz + c, o);
  }
  act_values(v, p.act);
  if (p.residual) {
    const Pack<T, 4> q = load_pack<T, 4>(static_cast<const T*>(p.residual) + r * p.ldr + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += to_f<T>(q.e[j]);
  }
  if (p.out_f32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.y) + r * p.ldy + c) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) o.e[j] = from_f<T>(v[j]);
    store_pack<T, 4>(static_cast<T*>(p.y) + r * p.ldy + c, o);
  }
}

// PAIR: two neighbouring blocks (a cluster) work on one 256 x BN tile: each loads its 128 rows of A and half of B's rows, the
// first one's thread issues the products of both (they read both blocks' shared memory), and each takes its own 128 rows of
// the accumulator through the epilogue.
template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(GEMM_THREADS, 1)
    k_gemm(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmJob job) {
  constexpr int BROWS = PAIR ? BN / 2 : BN;  // rows of B this block loads
  constexpr int A_BYTES = BM * BK * 2, B_BYTES = BROWS * BK * 2, STAGE = A_BYTES + B_BYTES, STAGES = RING_BYTES / STAGE;
  constexpr int TMEM_COLS = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = smem + RING_BYTES;
  float* bias_slices = reinterpret_cast<float*>(staging + EPI_WARPS * STAGE_OUT);
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + EPI_WARPS * (STAGE_OUT + 128));
  volatile int* stop = reinterpret_cast<volatile int*>(bars + 2 * STAGES + 5);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 6);
  const uint32_t ring = smem_u32(smem), bar0 = smem_u32(bars);
  auto full = [&](int s) { return bar0 + 8 * s; };
  auto empty = [&](int s) { return bar0 + 8 * (STAGES + s); };
  auto acc_full = [&](int a) { return bar0 + 8 * (2 * STAGES + a); };
  auto acc_empty = [&](int a) { return bar0 + 8 * (2 * STAGES + 2 + a); };
  const uint32_t drained = bar0 + 8 * (2 * STAGES + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int side = PAIR ? blockIdx.x & 1 : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(acc_full(a), 1);
      mbar_init(acc_empty(a), PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    mbar_init(drained, 1);
    *stop = job.limit == 0;  // waits that last no longer than a look
    if (*stop) atomicOr(&g_status, 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(TMEM_COLS) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  __syncwarp();
  if constexpr (PAIR) cluster_barrier();  // the other block's barriers are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // blocks of one cluster (splits > 1) share a tile and divide its k-blocks; otherwise a block walks over its tiles
  const int rank = !PAIR && job.splits > 1 ? blockIdx.x % job.splits : 0;
  const int group = PAIR ? 2 : job.splits, first = blockIdx.x / group, step = gridDim.x / group;
  // tile t: its product, place and k-blocks
  auto locate = [&](int t, int& tm, int& tn) {
    const int which = t >= job.tiles0;
    tile_at(job.p[which], which ? t - job.tiles0 : t, tm, tn);
    return which;
  };
  auto first_k = [&](const GemmParams& p) { return (int)((int64_t)p.kblocks * rank / job.splits); };
  auto last_k = [&](const GemmParams& p) { return (int)((int64_t)p.kblocks * (rank + 1) / job.splits); };

  if (warp == 0 || warp == 2 + EPI_WARPS) {
    // loads: one thread for A and one for B, because one alone issues a load every 0.09 us
    const bool is_a = warp == 0;
    if (elect_one()) {
      int s = 0, phase = 0;
      bool ok = true;
      for (int i = 0, t; ok && (t = tile_of(job, first, i, step)) >= 0; ++i) {
        int tm, tn;
        const int which = locate(t, tm, tn);
        const GemmParams& p = job.p[which];
        const CUtensorMap* map = is_a ? &maps.a[which] : &maps.b[which];
        const bool mn = is_a ? p.a_mn : p.b_mn;
        const int kb1 = last_k(p), row = is_a ? (PAIR ? tm * 2 + side : tm) * BM : tn * BN + side * BROWS;
        for (int kb = first_k(p); kb < kb1; ++kb) {
          if (!(ok = mbar_wait(empty(s), phase ^ 1, stop, job.limit))) break;
          const uint32_t to = ring + s * STAGE + (is_a ? 0 : A_BYTES);
          const uint32_t bar = PAIR ? cluster_addr(full(s), 0) : full(s);  // a pair's loads report to its first block
          if (is_a && side == 0) mbar_expect(full(s), PAIR ? 2 * STAGE : STAGE);
          if (mn) {
            const int panels = (is_a ? BM : BROWS) / 64;
            for (int j = 0; j < panels; ++j) tma_load<PAIR>(to + j * 8192, map, row + j * 64, kb * BK, bar);
          } else {
            tma_load<PAIR>(to, map, kb * BK, row, bar);
          }
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) outlast_copies();  // of a stage that only one of the two threads has started no phase ends
    }
  } else if (warp == 1) {
    if (side == 0 && elect_one()) {  // products
      int s = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (int i = 0, t; ok && (t = tile_of(job, first, i, step)) >= 0; ++i) {
        const GemmParams& p = job.p[t >= job.tiles0];
        // one 16-deep step inside a 64-deep k-block: 32 bytes along k-major rows, 16 rows of 128 bytes otherwise
        const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
        const uint32_t a_lead = p.a_mn ? 8192 : 16, b_lead = p.b_mn ? 8192 : 16;
        const uint32_t idesc = p.idesc;
        const int kb0 = first_k(p), kb1 = last_k(p);
        if (!(ok = mbar_wait(acc_empty(acc), acc_phase ^ 1, stop, job.limit))) break;
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait(full(s), phase, stop, job.limit))) break;
          tc_fence_after();
          const uint32_t a = ring + s * STAGE, b = a + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            mma_f16<PAIR>(tmem + acc * BN, smem_desc(a + k * a_step, a_lead, 1024), smem_desc(b + k * b_step, b_lead, 1024), idesc,
                    kb != kb0 || k != 0);
          mma_commit<PAIR>(empty(s));
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit<PAIR>(acc_full(acc));
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      if (!ok) {  // products in flight must end before TMEM is freed
        volatile int never = 0;
        mma_commit<PAIR>(drained);
        mbar_wait(drained, 0, &never, WAIT_LIMIT);
      }
    }
  } else {
    // epilogue: warp w reads the TMEM lanes of its quarter; two warps share a quarter and take 64-column slices in turn
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    uint8_t* stage = staging + (warp - 2) * STAGE_OUT;
    float* bias_slice = bias_slices + (warp - 2) * 32;
    int acc = 0, acc_phase = 0;
    // The residual is fetched a slice ahead and the bias a tile ahead, over the tile's end: their latency would be waited
    // for with the accumulator ready otherwise.
    uint4 early[8];
    float bias_reg[4], bias_next[4];  // of this warp's two slices, a column a lane
    auto fetch_ahead = [&](int t, bool of_residual) {
      if (t < 0 || job.splits > 1) return;
      int tm, tn;
      const int which = locate(t, tm, tn);
      const GemmParams& p = job.p[which];
      if (p.swap) return;
      if (of_residual) {
        if (p.residual && half * 64 < BN)
          fetch_in(early, p.residual, p.ldr, p.vec_r, (int64_t)(PAIR ? tm * 2 + side : tm) * BM + quarter * 32, (int64_t)tn * BN + half * 64, p.m,
                   p.n);
      } else if (p.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t c = (int64_t)tn * BN + half * 64 + (j >> 1) * 128 + (j & 1) * 32 + lane;
          bias_next[j] = c < p.n ? to_f<T>(static_cast<const T*>(p.bias)[c]) : 0.f;
        }
      }
    };
    int t_next = tile_of(job, first, 0, step);
    fetch_ahead(t_next, true);
    fetch_ahead(t_next, false);
    for (int i = 0, t; (t = t_next) >= 0; ++i) {
      int tm, tn;
      const int which = locate(t, tm, tn);
      const GemmParams& p = job.p[which];
      const T* bias = static_cast<const T*>(p.bias);
      const int64_t r0 = (int64_t)(PAIR ? tm * 2 + side : tm) * BM + quarter * 32;
      t_next = tile_of(job, first, i + 1, step);
#pragma unroll
      for (int j = 0; j < 4; ++j) bias_reg[j] = bias_next[j];
      fetch_ahead(t_next, false);
      bool ahead = false;  // the next tile's first residual slice is on its way
      mbar_wait(acc_full(acc), acc_phase, stop, job.limit);  // if it runs out the warp goes on, together, with what there is
      tc_fence_after();
      const uint32_t src = tmem + acc * BN + ((uint32_t)(quarter * 32) << 16);
      if (!PAIR && job.splits > 1) {  // to shared memory (the ring is free: every load was consumed before acc_full)
        float* part = reinterpret_cast<float*>(smem);
        for (int c = half * 32; c < BN; c += 64) {
          float v[32];
          tmem_load32(src + c, v);
          float4* d = reinterpret_cast<float4*>(part + (quarter * 32 + lane) * (BN + 4) + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        break;  // one tile per cluster
      }
      if (p.swap) {
        const int64_t o = r0 + lane;
        for (int c = half * 32; c < BN; c += 64) {
          const int64_t c0 = (int64_t)tn * BN + c;
          if (c0 >= p.n || r0 >= p.m) continue;  // nothing of this slice exists (uniform over the warp)
          float v[32];
          tmem_load32(src + c, v);
          if (o < p.m) store_column<T, 32>(p, c0, o, v);
        }
      } else {
        for (int c = half * 64; c < BN; c += 128) {
          const int64_t c0 = (int64_t)tn * BN + c;
          if (c0 >= p.n || r0 >= p.m) continue;
          // A lane's staging row holds the residual's words, then in their place the pre-activation's on their way out, then the
          // result's (a float result fills the whole row: the residual is staged again for the second half).
          uint8_t* mine = stage + lane * 128;
          auto word = [&](int k) { return reinterpret_cast<uint4*>(mine + ((k ^ (lane & 7)) << 4)); };
#pragma unroll 1  // half the code: the instruction cache is short of it
          for (int h = 0; h < 2; ++h) {
            const int64_t ch = c0 + 32 * h;
            if (ch >= p.n) break;
            if (h == 0 || p.out_f32) {
              stage_free();
              if (p.residual) {
                stage_in(stage, early, p.residual, p.ldr, p.vec_r, r0, c0, p.m, p.n);
                if (h == 1 || !p.out_f32 || c0 + 32 >= p.n) {  // no longer needed
                  if (c + 128 < BN && c0 + 128 < p.n) {
                    fetch_in(early, p.residual, p.ldr, p.vec_r, r0, c0 + 128, p.m, p.n);
                  } else {
                    fetch_ahead(t_next, true);
                    ahead = true;
                  }
                }
              }
            }
            float v[32];
            if (bias) bias_slice[lane] = c >= 128 ? (h ? bias_reg[3] : bias_reg[2]) : (h ? bias_reg[1] : bias_reg[0]);
            tmem_load32(src + c + 32 * h, v);
            if (bias) {
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 b4 = reinterpret_cast<const float4*>(bias_slice)[i];
                const float2 lo = add2(make_float2(v[4 * i], v[4 * i + 1]), make_float2(b4.x, b4.y));
                const float2 hi = add2(make_float2(v[4 * i + 2], v[4 * i + 3]), make_float2(b4.z, b4.w));
                v[4 * i] = lo.x;
                v[4 * i + 1] = lo.y;
                v[4 * i + 2] = hi.x;
                v[4 * i + 3] = hi.y;
              }
              __syncwarp();  // the slice may be written again
            }
            uint4 res[4];
            if (p.residual) {
#pragma unroll
              for (int k = 0; k < 4; ++k) res[k] = *word(4 * h + k);
            }
            if (p.z) {
              stage_row<T>(stage, lane, v, h);
              copy_out(stage, p.z, p.ldz, p.vec_z, h, r0, ch, p.m, p.n);
            }
            act_values(v, p.act);
            if (p.residual) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                  const float2 u = add2(make_float2(v[8 * k + i], v[8 * k + i + 1]), pair_of<T>(res[k], i / 2));
                  v[8 * k + i] = u.x;
                  v[8 * k + i + 1] = u.y;
                }
              }
            }
            if (p.out_f32) {
              __syncwarp();  // the other lanes have read their residual
              stage_row_f32(stage, lane, v);
              if (p.vec_y)
                stage_store(stage, &maps.y[which], r0, ch);
              else
                stage_out(stage, p.y, p.ldy, 4, 0, r0, ch, p.m, p.n);
            } else {
              stage_row<T>(stage, lane, v, h);
              if (!p.vec_y) stage_out(stage, p.y, p.ldy, 2, h, r0, ch, p.m, p.n);
            }
          }
          if (!p.out_f32 && p.vec_y) stage_store(stage, &maps.y[which], r0, c0);
        }
      }
      if (!ahead) fetch_ahead(t_next, true);  // a tile without a slice for this warp
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_far(cluster_addr(acc_empty(acc), 0));
        else
          mbar_arrive(acc_empty(acc));
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // shared memory outlives the stores that read it
  }
  __syncwarp();
  if (!PAIR && job.splits > 1) {
    __syncthreads();
    __syncwarp();
    cluster_barrier();
    // this block finishes 128 / splits rows of the tile from all blocks' partial tiles
    if (!*stop && first < job.tiles) {
      const GemmParams& p = job.p[0];
      int tm, tn;
      tile_at(p, first, tm, tn);
      const int rows = BM / job.splits, row0 = rank * rows;
      constexpr int QUADS = BN / 4;
      for (int i = threadIdx.x; i < rows * QUADS; i += GEMM_THREADS) {
        // consecutive threads along the output's contiguous axis
        const int r = row0 + (p.swap ? i % rows : i / QUADS), c = 4 * (p.swap ? i / rows : i % QUADS);
        const int64_t m = (int64_t)tm * BM + r, n = (int64_t)tn * BN + c;
        if (m >= p.m || n >= p.n) continue;
        const uint32_t at = ring + (r * (BN + 4) + c) * 4;
        float4 q[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < job.splits) q[k] = ld_cluster4(at, k);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < job.splits) {
            v[0] += q[k].x;
            v[1] += q[k].y;
            v[2] += q[k].z;
            v[3] += q[k].w;
          }
        if (p.swap) {
          store_column<T, 4>(p, n, m, v);
        } else {
          store_four<T>(p, m, n, v);
        }
      }
    }
    __syncwarp();
    cluster_barrier();  // nobody leaves while others read its shared memory
  }
  __syncthreads();
  __syncwarp();
  if constexpr (PAIR) cluster_barrier();  // the pair's loads, products and arrivals are done on both sides
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM_COLS) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(TMEM_COLS) : "memory");
  }
}

// ---- up to four rows --------------------------------------------------------------------------------
// G lanes share C output columns: each reads VEC elements of the columns' weight rows at a time and multiplies them with the
// rows of x, which lie in shared memory in their own type (a 16-byte read per row and VEC elements, no bank conflicts).  Bound
// by reading w once: 20000 columns of 400, one row: 4.4 us; 4096 of 4096: 6.1 us (both out of L2).
constexpr int GEMV_THREADS = 256, GEMV_CHUNK = 4096;
template <typename T, int VEC, int G, int MT, int C>
__global__ void __launch_bounds__(GEMV_THREADS)
    k_gemv(const T* __restrict__ x, int64_t ldx, const T* __restrict__ w, int64_t ldw, int64_t inner, int64_t outer,
           const __grid_constant__ GemmParams p) {
  extern __shared__ __align__(16) unsigned char xraw[];
  T* xs = reinterpret_cast<T*>(xraw);  // [MT][pitch]
  const int lane = threadIdx.x & (G - 1);
  const int64_t o = ((int64_t)blockIdx.x * GEMV_THREADS + threadIdx.x) / G * C;
  const T* wr[C];
#pragma unroll
  for (int c = 0; c < C; ++c) wr[c] = w + min(o + c, outer - 1) * ldw;  // a column beyond the last is computed and not written
  const int chunk = (int)min(inner, (int64_t)GEMV_CHUNK), pitch = (chunk + 7) / 8 * 8;
  float2 acc[MT][C];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < C; ++c) acc[m][c] = both(0.f);
  for (int64_t k0 = 0; k0 < inner; k0 += chunk) {
    const int n = (int)min((int64_t)chunk, inner - k0);
    if (k0) __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m)
      for (int k = threadIdx.x; k < n; k += GEMV_THREADS) xs[m * pitch + k] = x[m * ldx + k0 + k];
    __syncthreads();
#pragma unroll 4
    for (int k = lane * VEC; k < n; k += G * VEC) {
      Pack<T, VEC> q[C];
#pragma unroll
      for (int c = 0; c < C; ++c) q[c] = load_pack_stream<T, VEC>(wr[c] + k0 + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const Pack<T, VEC> v = load_pack<T, VEC>(xs + m * pitch + k);
        if constexpr (VEC == 1) {
#pragma unroll
          for (int c = 0; c < C; ++c) acc[m][c].x = fmaf(to_f<T>(q[c].e[0]), to_f<T>(v.e[0]), acc[m][c].x);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float2 f = make_float2(to_f<T>(v.e[i]), to_f<T>(v.e[i + 1]));
#pragma unroll
            for (int c = 0; c < C; ++c) acc[m][c] = fma2(make_float2(to_f<T>(q[c].e[i]), to_f<T>(q[c].e[i + 1])), f, acc[m][c]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float mine = 0.f;  // lane m keeps row m's sum
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float s = acc[m][c].x + acc[m][c].y;
#pragma unroll
      for (int d = G / 2; d; d >>= 1) s += __shfl_xor_sync(FULL, s, d);
      if (lane == m) mine = s;
    }
    if (lane < MT && o + c < outer) store_one<T>(p, lane, o + c, mine + (p.bias ? to_f<T>(static_cast<const T*>(p.bias)[o + c]) : 0.f));
  }
}

// ---- copies, gradients' first step ------------------------------------------------------------------
// src [rows][cols] with any row stride to dst with rows of `pitch` (a multiple of 8) elements, for up to two operands.
struct PackJob {
  struct {
    const uint16_t* src;
    uint16_t* dst;
    int64_t ld, rows, cols, pitch;
  } one[2];
  int count;
  int64_t rows, cols;  // the most of either
  unsigned across;     // blocks along x that take the columns; as many again take further rows
};
__device__ __forceinline__ void pack_rows(const PackJob& job, int which) {
  const auto& j = job.one[which];
  const unsigned times = gridDim.x / job.across, turn = blockIdx.x / job.across;
  const int64_t c0 = ((int64_t)(blockIdx.x - turn * job.across) * 32 + (threadIdx.x & 31)) * 8;
  if (c0 >= j.cols || turn >= times) return;
#pragma unroll 2
  for (int64_t r = ((int64_t)turn * gridDim.y + blockIdx.y) * 8 + (threadIdx.x >> 5); r < j.rows; r += (int64_t)times * gridDim.y * 8) {
    uint16_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c0 + i < j.cols ? __ldg(j.src + r * j.ld + c0 + i) : (uint16_t)0;
    *reinterpret_cast<uint4*>(j.dst + r * j.pitch + c0) =
        make_uint4(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16, v[4] | (uint32_t)v[5] << 16, v[6] | (uint32_t)v[7] << 16);
  }
}
__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackJob job) { pack_rows(job, blockIdx.z); }

// dz = dy act'(z) (if dz) and the column sums: partial ones to part[blockIdx.y][outer], or, when the blocks of one range of
// columns form a cluster (few rows), the whole ones to db.  A warp takes every eighth row of the block's range, a lane VEC
// columns, ROWS rows in flight.  Further planes of the grid copy operands, so that few rows need one launch for all of it.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(256)
    k_act_grad(const T* __restrict__ dy, int64_t ldg, const T* __restrict__ z, int64_t ldz, int64_t rows, int64_t outer,
               T* __restrict__ dz, int64_t pitch, float* __restrict__ part, T* __restrict__ db, const __grid_constant__ PackJob job) {
  if (blockIdx.z) {
    pack_rows(job, blockIdx.z - 1);
    return;
  }
  constexpr int ROWS = ACT == FV_ACT_NONE ? 4 : 2;  // with an activation four rows cost registers and 5 % of the time
  __shared__ float sum[8][32 * VEC];
  __shared__ __align__(16) float total[32 * VEC];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = ((int64_t)blockIdx.x * 32 + lane) * VEC;
  const int64_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s[i] = 0.f;
  if (c < outer) {
    for (int64_t r = r0 + warp; r < r1; r += 8 * ROWS) {
      Pack<T, VEC> g[ROWS], q[ROWS];
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (r + 8 * k < r1) {
          g[k] = load_pack_stream<T, VEC>(dy + (r + 8 * k) * ldg + c);
          if (ACT != FV_ACT_NONE) q[k] = load_pack_stream<T, VEC>(z + (r + 8 * k) * ldz + c);
        }
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
        if (r + 8 * k < r1) {
          if constexpr (VEC == 8) {
            float2 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[i] = pair_of<T>(g[k].w, i);
              if (ACT != FV_ACT_NONE) v[i] = mul2(v[i], act_slope<ACT>(pair_of<T>(q[k].w, i)));
              const float2 t = add2(make_float2(s[2 * i], s[2 * i + 1]), v[i]);
              s[2 * i] = t.x;
              s[2 * i + 1] = t.y;
            }
            g[k].w = word_of<T>(v);
          } else {
            float2 v = both(to_f<T>(g[k].e[0]));
            if (ACT != FV_ACT_NONE) v = mul2(v, act_slope<ACT>(both(to_f<T>(q[k].e[0]))));
            s[0] += v.x;
            g[k].e[0] = from_f<T>(v.x);
          }
          if (dz) store_pack<T, VEC>(dz + (r + 8 * k) * pitch + c, g[k]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) sum[warp][lane * VEC + i] = s[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const int64_t col = (int64_t)blockIdx.x * 32 * VEC + i;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sum[w][i];
    if (db)
      total[i] = v;
    else if (col < outer)
      part[(int64_t)blockIdx.y * outer + col] = v;
  }
  if (!db) return;
  __syncwarp();
  cluster_barrier();
  if (blockIdx.y == 0 && threadIdx.x < 8 * VEC) {  // the cluster's blocks in their order
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (unsigned k = 0; k < gridDim.y; ++k) {
      const float4 q = ld_cluster4(smem_u32(total + 4 * threadIdx.x), k);
      v[0] += q.x;
      v[1] += q.y;
      v[2] += q.z;
      v[3] += q.w;
    }
    const int64_t col = (int64_t)blockIdx.x * 32 * VEC + 4 * threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (col + i < outer) db[col + i] = from_f<T>(v[i]);
  }
  __syncwarp();
  cluster_barrier();  // nobody leaves while its sums are read
}
template <typename T, int VEC>
cudaError_t launch_act_grad(cudaStream_t st, const T* dy, int64_t ldg, const T* z, int64_t ldz, int64_t rows, int64_t outer, int act, T* dz,
                            int64_t pitch, float* part, T* db, int64_t chunks, const PackJob& job) {
  const unsigned gx = (unsigned)((outer + 32 * VEC - 1) / (32 * VEC));
  // the rows to copy may be many more than dy's, by which y goes: blocks along x take them, up to four rows to a warp
  const unsigned px = job.count ? job.across * (unsigned)((job.rows + 32 * chunks - 1) / (32 * chunks)) : 0u;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(std::max(gx, px), (unsigned)chunks, 1u + (unsigned)job.count);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.z = 1;
  attr[0].val.clusterDim.y = (unsigned)chunks;
  cfg.attrs = attr;
  cfg.numAttrs = db ? 1 : 0;
  auto go = [&](auto kernel) { return cudaLaunchKernelEx(&cfg, kernel, dy, ldg, z, ldz, rows, outer, dz, pitch, part, db, job); };
  switch (act) {
    case FV_ACT_RELU: return go(k_act_grad<T, VEC, FV_ACT_RELU>);
    case FV_ACT_GELU: return go(k_act_grad<T, VEC, FV_ACT_GELU>);
    case FV_ACT_GELU_TANH: return go(k_act_grad<T, VEC, FV_ACT_GELU_TANH>);
    case FV_ACT_SILU: return go(k_act_grad<T, VEC, FV_ACT_SILU>);
    default: return go(k_act_grad<T, VEC, FV_ACT_NONE>);
  }
}
template <typename T>
__global__ void __launch_bounds__(512) k_col_sum(const float* __restrict__ part, int64_t P, int64_t n, T* __restrict__ out) {
  column_sums(part, P, n, [&](int64_t c, float v) { out[c] = from_f<T>(v); });
}

// ---- host side --------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                              CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// A matrix as the product sees it: `rows` x `depth`; element (r, k) at p[r * ld + k], or p[k * ld + r] when mn.
struct Operand {
  const void* p;
  int64_t rows, depth, ld;
  bool mn;
  int64_t inner() const { return mn ? rows : depth; }
  int64_t outer() const { return mn ? depth : rows; }
  // TMA: 16-byte aligned rows.  A single row has no stride that matters.
  // Rows that overlap (a broadcast) are copied too.
  bool tma_ok() const { return (uintptr_t)p % 16 == 0 && (outer() == 1 || (ld % 8 == 0 && ld >= inner())); }
};
constexpr size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t pad8(int64_t n) { return (n + 7) / 8 * 8; }
size_t packed_bytes(const Operand& o) { return align256((size_t)o.outer() * (size_t)pad8(o.inner()) * 2); }

struct Workspace {
  uint8_t* base;
  size_t size, used = 0;
  void* take(size_t n) {
    void* r = base + used;
    used += align256(n);
    return r;
  }
};

// Copies of those of two operands that TMA cannot read: the operands afterwards, and the job that fills them.
int plan_pack(Operand& a, Operand& b, Workspace& ws, PackJob* job) {
  *job = PackJob{};
  for (Operand* o : {&a, &b}) {
    if (o->tma_ok()) continue;
    const int64_t pitch = pad8(o->inner());
    uint16_t* dst = static_cast<uint16_t*>(ws.take((size_t)o->outer() * (size_t)pitch * 2));
    job->one[job->count++] = {static_cast<const uint16_t*>(o->p), dst, o->ld, o->outer(), o->inner(), pitch};
    job->rows = std::max(job->rows, o->outer());
    job->cols = std::max(job->cols, o->inner());
    job->across = (unsigned)((job->cols + 255) / 256);
    o->p = dst;
    o->ld = pitch;
  }
  FV_REQUIRE(!job->count || ws.used <= ws.size, FV_ERR_INVALID, "workspace too small: %llu bytes needed so far, got %llu",
             (unsigned long long)ws.used, (unsigned long long)ws.size);
  return FV_OK;
}
int pack_operands(const PackJob& job, cudaStream_t st) {
  if (!job.count) return FV_OK;
  k_pack<<<dim3(job.across, (unsigned)std::min<int64_t>((job.rows + 7) / 8, 4096), (unsigned)job.count), 256, 0, st>>>(job);
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

int make_map(CUtensorMap* map, const Operand& o, int dtype, int box_rows) {
  const EncodeFn enc = encode_fn();
  FV_REQUIRE(enc, FV_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)o.inner(), (cuuint64_t)o.outer()};
  const cuuint64_t strides[1] = {(cuuint64_t)(o.outer() == 1 ? pad8(o.inner()) : o.ld) * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)(o.mn ? 64 : box_rows)};
  const cuuint32_t one[2] = {1, 1};
  const CUresult r = enc(map, dtype == FV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(o.p),
                         dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FV_REQUIRE(r == CUDA_SUCCESS, FV_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d ([%lld][%lld], stride %lld)", (int)r, (long long)o.outer(),
             (long long)o.inner(), (long long)o.ld);
  return FV_OK;
}

// An output [rows][cols], dense, as 128-byte wide boxes of 32 rows.
int make_out_map(CUtensorMap* map, void* out, int64_t rows, int64_t cols, int dtype) {
  const EncodeFn enc = encode_fn();
  FV_REQUIRE(enc, FV_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
  const size_t es = elem_size(dtype);
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)(cols * es)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), 32};
  const cuuint32_t one[2] = {1, 1};
  const CUresult r = enc(map, dtype == FV_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                              : dtype == FV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         2, out, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  FV_REQUIRE(r == CUDA_SUCCESS, FV_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d for an output [%lld][%lld]", (int)r, (long long)rows,
             (long long)cols);
  return FV_OK;
}

struct Shape {
  int bn, splits;
  bool pair;
};
struct Size {
  int64_t m, n, kblocks;
};
// Estimated microseconds of one launch, from measurements on a B200: a k-block costs `few` with a handful of blocks at
// work (bound by the issue of loads up to a width of 128, by the products above) and `many` with all SMs at work (L2, power); a
// tile's epilogue costs `epi` and runs under the next tile's products; launch, set-up and drain cost 3.5.
struct Cost {
  int bn;
  bool pair;
  double few, many, epi;
};
constexpr Cost COSTS[] = {{256, true, 0.28, 0.36, 4.4}, {256, false, 0.28, 0.42, 4.2}, {128, false, 0.165, 0.23, 2.5}, {64, false, 0.165, 0.175, 1.3}};
double estimate(const Cost& c, int splits, const Size* sizes, int count, int sms) {
  const double places = c.pair ? sms / 2 : sms / splits;
  double tiles = 0, work = 0, longest = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t rows = c.pair ? 2 * BM : BM;
    const double t = (double)((sizes[i].m + rows - 1) / rows) * (double)((sizes[i].n + c.bn - 1) / c.bn);
    tiles += t;
  }
  const double busy = std::min(1.0, tiles / places), kb = c.few + (c.many - c.few) * busy;
  for (int i = 0; i < count; ++i) {
    const int64_t rows = c.pair ? 2 * BM : BM;
    const double t = (double)((sizes[i].m + rows - 1) / rows) * (double)((sizes[i].n + c.bn - 1) / c.bn);
    const double one = std::max((double)((sizes[i].kblocks + splits - 1) / splits) * kb, tiles > places ? c.epi : 0.0);
    work += t * one;
    longest = std::max(longest, one);
  }
  const double waves = (double)((int64_t)((tiles + places - 1) / places));
  const double run = tiles <= places ? longest : count == 1 ? waves * longest : std::max(work / places, longest) + 0.1 * longest;
  return 3.5 + run + c.epi + (splits > 1 ? 1.5 + 0.3 * splits + c.epi : 0.0);
}
// Tile shape and split of k with the least estimate.
Shape choose_shape(const Size* sizes, int count, int sms, bool narrow, double* time) {
  Shape best{64, 1, false};
  double least = 1e300;
  for (const Cost& c : COSTS) {
    if (narrow && c.bn > 64) continue;
    for (int s : {1, 2, 4, 8}) {
      if (s > 1) {  // one tile per cluster: all of them at once
        const double tiles = (double)((sizes[0].m + BM - 1) / BM) * (double)((sizes[0].n + c.bn - 1) / c.bn);
        if (c.pair || count > 1 || s > sizes[0].kblocks || tiles * s > sms) break;
      }
      const double t = estimate(c, s, sizes, count, sms);
      if (t < least) {
        least = t;
        best = {c.bn, s, c.pair};
      }
    }
  }
  if (time) *time = least;
  return best;
}

// The two products of a backward pass: in one launch of one shape (answers 1) or in two.
int choose_backward(const Size* sizes, int sms, Shape* shapes) {
  double one = 0, two[2] = {0, 0};
  const Shape joint = choose_shape(sizes, 2, sms, false, &one);
  for (int i = 0; i < 2; ++i) shapes[i] = choose_shape(&sizes[i], 1, sms, false, &two[i]);
  if (one > two[0] + two[1]) return 2;
  shapes[0] = joint;
  return 1;
}

template <typename T, int BN, bool PAIR>
int launch_gemm(const GemmMaps& maps, const GemmJob& job, unsigned grid, int splits, cudaStream_t st) {
  static std::atomic<bool> given[64];
  FV_CUDA(fv::allow_smem((const void*)k_gemm<T, BN, PAIR>, given, GEMM_SMEM, GEMM_SMEM));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(GEMM_THREADS);
  cfg.dynamicSmemBytes = GEMM_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2u : (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR || splits > 1 ? 1 : 0;
  FV_CUDA(cudaLaunchKernelEx(&cfg, k_gemm<T, BN, PAIR>, maps, job));
  return FV_OK;
}

// One product D = A B^T with the epilogue that `p` describes (its output side is filled in by the caller).
struct Product {
  Operand a, b;
  GemmParams p;
};
Size size_of(const Product& d) { return Size{d.a.rows, d.b.rows, (d.a.depth + BK - 1) / BK}; }

int gemm(Product* d, int count, int dtype, const Shape& s, int sms, cudaStream_t st) {
  GemmMaps maps{};
  GemmJob job{};
  job.splits = s.splits;
  job.limit = wait_limit();
  const int rows = s.pair ? 2 * BM : BM;
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    GemmParams& p = d[i].p;
    const Operand &a = d[i].a, &b = d[i].b;
    p.m = a.rows;
    p.n = b.rows;
    p.kblocks = (int)((a.depth + BK - 1) / BK);
    p.tiles_m = (int)((p.m + rows - 1) / rows);
    p.tiles_n = (int)((p.n + s.bn - 1) / s.bn);
    tiles += (int64_t)p.tiles_m * p.tiles_n;
    FV_REQUIRE(tiles < (1ll << 30), FV_ERR_INVALID, "the product is too large");
    if (i == 0) job.tiles0 = (int)tiles;
    p.a_mn = a.mn;
    p.b_mn = b.mn;
    const uint32_t type = dtype == FV_BF16 ? 1u : 0u;
    p.idesc = 1u << 4 | type << 7 | type << 10 | (uint32_t)a.mn << 15 | (uint32_t)b.mn << 16 | (uint32_t)(s.bn / 8) << 17 | (uint32_t)(rows / 16) << 24;
    if (!p.swap && s.splits == 1 && p.vec_y)
      if (int rc = make_out_map(&maps.y[i], p.y, p.m, p.n, p.out_f32 ? FV_F32 : dtype)) return rc;
    if (int rc = make_map(&maps.a[i], a, dtype, BM)) return rc;
    if (int rc = make_map(&maps.b[i], b, dtype, s.pair ? s.bn / 2 : s.bn)) return rc;
    job.p[i] = p;
  }
  job.tiles = (int)tiles;
  // with a remainder round of the first product; an epilogue is worth about a dozen k-blocks
  if (count == 2) job.spare = std::max(job.p[0].kblocks, 12) / std::max(job.p[1].kblocks, 12);
  const unsigned grid = (unsigned)(s.splits > 1 ? tiles * s.splits : std::min<int64_t>(tiles, s.pair ? sms / 2 : sms) * (s.pair ? 2 : 1));
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return s.pair        ? launch_gemm<T, 256, true>(maps, job, grid, 1, st)
           : s.bn == 256 ? launch_gemm<T, 256, false>(maps, job, grid, s.splits, st)
           : s.bn == 128 ? launch_gemm<T, 128, false>(maps, job, grid, s.splits, st)
                         : launch_gemm<T, 64, false>(maps, job, grid, s.splits, st);
  };
  return dtype == FV_BF16 ? go(__nv_bfloat16{}) : go(__half{});
}

template <typename T, int VEC, int G, int C>
void launch_gemv(const T* x, int64_t ldx, const T* w, int64_t ldw, int64_t rows, int64_t inner, int64_t outer, const GemmParams& p,
                 cudaStream_t st) {
  const unsigned grid = (unsigned)(((outer + C - 1) / C * G + GEMV_THREADS - 1) / GEMV_THREADS);
  const size_t smem = (size_t)rows * (std::min<int64_t>(inner, GEMV_CHUNK) + 7) * sizeof(T);  // 32 KB at most
  switch (rows) {
    case 1: k_gemv<T, VEC, G, 1, C><<<grid, GEMV_THREADS, smem, st>>>(x, ldx, w, ldw, inner, outer, p); break;
    case 2: k_gemv<T, VEC, G, 2, C><<<grid, GEMV_THREADS, smem, st>>>(x, ldx, w, ldw, inner, outer, p); break;
    case 3: k_gemv<T, VEC, G, 3, C><<<grid, GEMV_THREADS, smem, st>>>(x, ldx, w, ldw, inner, outer, p); break;
    default: k_gemv<T, VEC, G, 4, C><<<grid, GEMV_THREADS, smem, st>>>(x, ldx, w, ldw, inner, outer, p);
  }
}

constexpr int64_t GEMV_ROWS = 4, NARROW_ROWS = 64, FEW_ROWS = 1024;

// k_gemv needs k-major rows of w (and of x).  Three and four rows go there when the sums are short or when k_gemm would have to
// copy w first (4 rows: 4096 x 4096 12.7 us against k_gemm's 12.0, 400 x 20000 9.1 against 9.4).
bool use_gemv(int64_t rows, const Operand& x, const Operand& w) {
  return !w.mn && !x.mn && (rows <= 2 || (rows <= GEMV_ROWS && (w.depth <= 1024 || !w.tma_ok())));
}

// A matrix given by both strides: k-major when its second axis is contiguous, else its first must be.
bool operand_of(const void* p, int64_t rows, int64_t depth, int64_t rs, int64_t cs, Operand* o) {
  if (cs == 1 || depth == 1) {
    *o = Operand{p, rows, depth, rs, false};
    return rs >= 0;
  }
  if (rs == 1 || rows == 1) {
    *o = Operand{p, rows, depth, cs, true};
    return cs >= 0;
  }
  return false;
}
Operand transposed(const Operand& o) { return Operand{o.p, o.depth, o.rows, o.ld, !o.mn}; }

bool sizes_ok(int64_t rows, int64_t inner, int64_t outer) {
  return rows >= 0 && inner >= 1 && outer >= 1 && rows < (1ll << 31) - 256 && inner < (1ll << 31) - 256 && outer < (1ll << 31) - 256;
}
// Strides past these would not fit a tensor map.
bool stride_ok(int64_t s) { return s >= 0 && s < (1ll << 38); }

int64_t act_grad_chunks(int64_t rows, int64_t outer, int vec, int sms) {
  const int64_t blocks = (outer + 32 * vec - 1) / (32 * vec);
  return std::max<int64_t>(1, std::min<int64_t>((rows + 15) / 16, (int64_t)sms * 8 / blocks));
}

}  // namespace
}  // namespace fvo

using namespace fvo;

extern "C" {

int fv_ops_status(int device, uint32_t* word) {
  FV_REQUIRE(word, FV_ERR_INVALID, "fv_ops_status: NULL argument");
  OnDevice guard(device);
  FV_REQUIRE(guard.ok, FV_ERR_CUDA, "cannot select device %d", device);
  static std::mutex one;
  const std::lock_guard<std::mutex> lock(one);
  FV_CUDA(cudaDeviceSynchronize());  // non-blocking streams too, which the copies below would not wait for
  void* bits = nullptr;
  FV_CUDA(cudaGetSymbolAddress(&bits, g_status));
  FV_CUDA(take_status(static_cast<unsigned*>(bits), word));
  uint32_t more = 0;
  FV_CUDA(norm_status(&more));
  *word |= more;
  return FV_OK;
}

int fv_ops_wait_limit(int64_t cycles) {
  FV_REQUIRE(cycles >= -1, FV_ERR_INVALID, "fv_ops_wait_limit: %lld cycles", (long long)cycles);
  wait_limit(cycles);
  return FV_OK;
}

int fv_linear_shapes(int sms, int64_t rows, int64_t inner, int64_t outer, int backward, int32_t* shapes) {
  FV_REQUIRE(shapes && sms >= 2 && sms <= 1024 && rows >= 1 && sizes_ok(rows, inner, outer), FV_ERR_INVALID, "fv_linear_shapes: bad argument");
  auto blocks = [](int64_t n) { return (n + BK - 1) / BK; };
  Shape s[2];
  int count = 1;
  if (backward) {
    Size sizes[2] = {{rows, inner, blocks(outer)}, {outer, inner, blocks(rows)}};
    if (rows > outer) std::swap(sizes[0], sizes[1]);
    count = choose_backward(sizes, sms, s);
  } else {
    const bool narrow = rows <= NARROW_ROWS;
    const Size size{narrow ? outer : rows, narrow ? rows : outer, blocks(inner)};
    s[0] = choose_shape(&size, 1, sms, narrow, nullptr);
  }
  *shapes++ = count;
  for (int i = 0; i < count; ++i) {
    *shapes++ = s[i].bn;
    *shapes++ = s[i].splits;
    *shapes++ = s[i].pair;
  }
  return FV_OK;
}

int fv_linear_workspace(int64_t rows, int64_t inner, int64_t outer, const void* x, int64_t x_rs, int64_t x_cs, const void* w, int64_t w_rs,
                        int64_t w_cs, size_t* bytes) {
  FV_REQUIRE(bytes && sizes_ok(rows, inner, outer), FV_ERR_INVALID, "fv_linear_workspace: bad argument");
  Operand ox, ow;
  FV_REQUIRE(operand_of(x, rows, inner, x_rs, x_cs, &ox) && operand_of(w, outer, inner, w_rs, w_cs, &ow), FV_ERR_INVALID,
             "fv_linear: one axis of x and of the weight must be contiguous");
  *bytes = 0;
  if (rows == 0 || use_gemv(rows, ox, ow)) return FV_OK;
  if (!ox.tma_ok()) *bytes += packed_bytes(ox);
  if (!ow.tma_ok()) *bytes += packed_bytes(ow);
  return FV_OK;
}

int fv_linear(int device, void* stream, const void* x, int64_t x_rs, int64_t x_cs, const void* w, int64_t w_rs, int64_t w_cs, int64_t rows,
              int64_t inner, int64_t outer, int dtype, const void* bias, int act, const void* residual, int64_t residual_stride, void* y,
              int y_dtype, void* z, void* workspace, size_t workspace_bytes) {
  FV_REQUIRE(dtype == FV_BF16 || dtype == FV_F16, FV_ERR_INVALID, "fv_linear: operands must be bfloat16 or float16");
  FV_REQUIRE(y_dtype == dtype || y_dtype == FV_F32, FV_ERR_INVALID, "fv_linear: the output has the operands' type or is float32");
  FV_REQUIRE(sizes_ok(rows, inner, outer), FV_ERR_INVALID, "fv_linear: bad shape [%lld][%lld] x [%lld][%lld]", (long long)rows,
             (long long)inner, (long long)outer, (long long)inner);
  FV_REQUIRE(act >= FV_ACT_NONE && act <= FV_ACT_SILU, FV_ERR_INVALID, "fv_linear: unknown activation %d", act);
  FV_REQUIRE(stride_ok(x_rs) && stride_ok(x_cs) && stride_ok(w_rs) && stride_ok(w_cs) && stride_ok(residual_stride), FV_ERR_INVALID,
             "fv_linear: bad stride");
  if (rows == 0) return FV_OK;
  FV_REQUIRE(x && w && y, FV_ERR_INVALID, "fv_linear: NULL argument");
  Operand ox, ow;
  FV_REQUIRE(operand_of(x, rows, inner, x_rs, x_cs, &ox) && operand_of(w, outer, inner, w_rs, w_cs, &ow), FV_ERR_INVALID,
             "fv_linear: one axis of x and of the weight must be contiguous");
  FV_REQUIRE(workspace_bytes == 0 || (workspace && (uintptr_t)workspace % 256 == 0), FV_ERR_INVALID,
             "fv_linear: the workspace must be 256-byte aligned");
  OnDevice guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  GemmParams p{};
  p.act = act;
  p.out_f32 = y_dtype == FV_F32;
  p.bias = bias;
  p.residual = residual;
  p.ldr = residual_stride;
  p.y = y;
  p.z = z;
  p.ldy = p.ldz = outer;
  const size_t ys = p.out_f32 ? 4 : 2;
  p.vec_y = vec_ok(y, outer, ys, 16);
  p.vec_z = z && vec_ok(z, outer, 2, 16);
  p.vec_r = residual && vec_ok(residual, residual_stride, 2, 16);
  if (use_gemv(rows, ox, ow)) {
    // Eight lanes to a column when that fills the GPU, else a warp; two columns to a group when there are enough of them.
    // 16-byte loads where the rows of w allow them.
    const int64_t ldw = outer > 1 ? ow.ld : 0;
    const bool wide = vec_ok(w, ldw, 2, 16) && inner % 8 == 0, two = vec_ok(w, ldw, 2, 4) && inner % 2 == 0;
    const bool few = outer * 8 < (int64_t)sms * 1024, pairs = outer * 32 >= (int64_t)sms * 512;
    auto run = [&](auto tag) {
      using T = decltype(tag);
      const T *px = static_cast<const T*>(x), *pw = static_cast<const T*>(w);
      if (wide && !few) launch_gemv<T, 8, 8, 1>(px, ox.ld, pw, ow.ld, rows, inner, outer, p, st);
      else if (wide && pairs) launch_gemv<T, 8, 32, 2>(px, ox.ld, pw, ow.ld, rows, inner, outer, p, st);
      else if (wide) launch_gemv<T, 8, 32, 1>(px, ox.ld, pw, ow.ld, rows, inner, outer, p, st);
      else if (two) launch_gemv<T, 2, 32, 1>(px, ox.ld, pw, ow.ld, rows, inner, outer, p, st);
      else launch_gemv<T, 1, 32, 1>(px, ox.ld, pw, ow.ld, rows, inner, outer, p, st);
    };
    if (dtype == FV_BF16) run(__nv_bfloat16{});
    else run(__half{});
    FV_CUDA(cudaGetLastError());
    return FV_OK;
  }
  Workspace ws{static_cast<uint8_t*>(workspace), workspace_bytes};
  PackJob job;
  if (int rc = plan_pack(ox, ow, ws, &job)) return rc;
  if (int rc = pack_operands(job, st)) return rc;
  const bool narrow = rows <= NARROW_ROWS;  // w's rows on the wide side of the tiles
  p.swap = narrow;
  Product d = narrow ? Product{ow, ox, p} : Product{ox, ow, p};
  const Size size = size_of(d);
  return gemm(&d, 1, dtype, choose_shape(&size, 1, sms, narrow, nullptr), sms, st);
}

// dz is written when there is an activation, or when dy cannot be read by TMA.
static bool needs_dz(const void* dy, int64_t dy_stride, int64_t rows, int64_t outer, int act) {
  return act != FV_ACT_NONE || !Operand{dy, rows, outer, dy_stride, false}.tma_ok();
}

int fv_linear_backward_workspace(int device, int64_t rows, int64_t inner, int64_t outer, const void* dy, int64_t dy_stride, const void* x,
                                 int64_t x_rs, int64_t x_cs, const void* w, int64_t w_rs, int64_t w_cs, int act, size_t* bytes) {
  FV_REQUIRE(bytes && sizes_ok(rows, inner, outer), FV_ERR_INVALID, "fv_linear_backward_workspace: bad argument");
  Operand ox, ow;
  FV_REQUIRE(operand_of(x, rows, inner, x_rs, x_cs, &ox) && operand_of(w, outer, inner, w_rs, w_cs, &ow), FV_ERR_INVALID,
             "fv_linear_backward: one axis of x and of the weight must be contiguous");
  const int sms = sm_count(device);
  FV_REQUIRE(sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  *bytes = 0;
  if (rows == 0) return FV_OK;
  if (needs_dz(dy, dy_stride, rows, outer, act)) *bytes += align256((size_t)rows * (size_t)pad8(outer) * 2);
  *bytes += align256((size_t)act_grad_chunks(rows, outer, 1, sms) * (size_t)outer * sizeof(float)) +
            align256((size_t)act_grad_chunks(rows, outer, 8, sms) * (size_t)outer * sizeof(float));
  if (!ox.tma_ok()) *bytes += packed_bytes(ox);
  if (!ow.tma_ok()) *bytes += packed_bytes(ow);
  return FV_OK;
}

int fv_linear_backward(int device, void* stream, const void* dy, int64_t dy_stride, const void* x, int64_t x_rs, int64_t x_cs, const void* w,
                       int64_t w_rs, int64_t w_cs, int64_t rows, int64_t inner, int64_t outer, int dtype, const void* z, int64_t z_stride,
                       int act, void* dx, void* dw, void* db, void* workspace, size_t workspace_bytes) {
  FV_REQUIRE(dtype == FV_BF16 || dtype == FV_F16, FV_ERR_INVALID, "fv_linear_backward: operands must be bfloat16 or float16");
  FV_REQUIRE(sizes_ok(rows, inner, outer), FV_ERR_INVALID, "fv_linear_backward: bad shape [%lld][%lld] x [%lld][%lld]", (long long)rows,
             (long long)inner, (long long)outer, (long long)inner);
  FV_REQUIRE(act >= FV_ACT_NONE && act <= FV_ACT_SILU, FV_ERR_INVALID, "fv_linear_backward: unknown activation %d", act);
  FV_REQUIRE(stride_ok(dy_stride) && stride_ok(z_stride) && stride_ok(x_rs) && stride_ok(x_cs) && stride_ok(w_rs) && stride_ok(w_cs),
             FV_ERR_INVALID, "fv_linear_backward: bad stride");
  FV_REQUIRE(dw && db, FV_ERR_INVALID, "fv_linear_backward: NULL argument");
  OnDevice guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {  // a sum over nothing
    FV_CUDA(cudaMemsetAsync(dw, 0, (size_t)outer * (size_t)inner * 2, st));
    FV_CUDA(cudaMemsetAsync(db, 0, (size_t)outer * 2, st));
    return FV_OK;
  }
  FV_REQUIRE(dy && x && w && dx && (act == FV_ACT_NONE || z), FV_ERR_INVALID,
             "fv_linear_backward: NULL argument (an activation's gradient needs the pre-activation)");
  Operand ox, ow;
  FV_REQUIRE(operand_of(x, rows, inner, x_rs, x_cs, &ox) && operand_of(w, outer, inner, w_rs, w_cs, &ow), FV_ERR_INVALID,
             "fv_linear_backward: one axis of x and of the weight must be contiguous");
  size_t need = 0;
  if (int rc = fv_linear_backward_workspace(device, rows, inner, outer, dy, dy_stride, x, x_rs, x_cs, w, w_rs, w_cs, act, &need)) return rc;
  FV_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 256 == 0, FV_ERR_INVALID,
             "fv_linear_backward: the workspace must be 256-byte aligned and hold %llu bytes, got %llu", (unsigned long long)need,
             (unsigned long long)workspace_bytes);
  Workspace ws{static_cast<uint8_t*>(workspace), workspace_bytes};
  Operand od{dy, rows, outer, dy_stride, false};
  void* dz = nullptr;
  const int64_t pitch = pad8(outer);
  if (needs_dz(dy, dy_stride, rows, outer, act)) {
    dz = ws.take((size_t)rows * (size_t)pitch * 2);
    od = Operand{dz, rows, outer, pitch, false};
  }
  const bool vec = outer % 8 == 0 && vec_ok(dy, dy_stride, 2, 16) && (act == FV_ACT_NONE || vec_ok(z, z_stride, 2, 16));
  // Few rows: one launch forms dz, its whole column sums (clusters of up to eight blocks) and the copies.  777 x 501 x 1003 17 us
  // instead of 22 with three launches; 2000 rows of 256: 26 us instead of 18, too many rows for eight blocks.
  const bool few = rows <= FEW_ROWS;
  const int64_t chunks = few ? std::min<int64_t>(8, (rows + 63) / 64) : act_grad_chunks(rows, outer, vec ? 8 : 1, sms);
  float* part = few ? nullptr : static_cast<float*>(ws.take((size_t)chunks * (size_t)outer * sizeof(float)));
  PackJob job;
  if (int rc = plan_pack(ox, ow, ws, &job)) return rc;
  const bool together = few && job.rows <= FEW_ROWS;
  auto first = [&](auto tag) {
    using T = decltype(tag);
    const T *pg = static_cast<const T*>(dy), *pz = static_cast<const T*>(z);
    T *pd = static_cast<T*>(dz), *sums = few ? static_cast<T*>(db) : nullptr;
    const PackJob with = together ? job : PackJob{};
    return vec ? launch_act_grad<T, 8>(st, pg, dy_stride, pz, z_stride, rows, outer, act, pd, pitch, part, sums, chunks, with)
               : launch_act_grad<T, 1>(st, pg, dy_stride, pz, z_stride, rows, outer, act, pd, pitch, part, sums, chunks, with);
  };
  FV_CUDA(dtype == FV_BF16 ? first(__nv_bfloat16{}) : first(__half{}));
  if (!few) {
    const unsigned grid = (unsigned)((outer + 31) / 32);
    if (dtype == FV_BF16)
      k_col_sum<__nv_bfloat16><<<grid, 512, 0, st>>>(part, chunks, outer, static_cast<__nv_bfloat16*>(db));
    else
      k_col_sum<__half><<<grid, 512, 0, st>>>(part, chunks, outer, static_cast<__half*>(db));
    FV_CUDA(cudaGetLastError());
  }
  if (!together)
    if (int rc = pack_operands(job, st)) return rc;
  GemmParams px{}, pw{};
  px.y = dx;
  pw.y = dw;
  px.ldy = pw.ldy = inner;
  px.vec_y = vec_ok(dx, inner, 2, 16);
  pw.vec_y = vec_ok(dw, inner, 2, 16);
  Product d[2] = {{od, transposed(ow), px}, {transposed(od), transposed(ox), pw}};
  if (rows > outer) std::swap(d[0], d[1]);  // the one with the longer sums first
  const Size sizes[2] = {size_of(d[0]), size_of(d[1])};
  Shape shapes[2];
  if (choose_backward(sizes, sms, shapes) == 1) return gemm(d, 2, dtype, shapes[0], sms, st);
  for (int i = 0; i < 2; ++i)
    if (int rc = gemm(&d[i], 1, dtype, shapes[i], sms, st)) return rc;
  return FV_OK;
}

}  // extern "C"
