// Layer norm over the last axis, forward and backward.
//
//   forward   mean = sum x / D     rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)     y = (x - mean) rstd w + b
//   backward  h = (x - mean) rstd, u = dy w:
//             dx = rstd (u - sum u / D - h sum (u h) / D)      dw = sum_rows dy h      db = sum_rows dy
//
// Both passes are bound by memory: each row is read once, kept in registers while its sums are formed, and
// written once.  A row of up to 1024 elements belongs to one warp (no barrier), a longer one to a block of up
// to 512 threads with 8, 16 or 32 elements each; rows beyond 16384 elements (8192 for the float gradient,
// whose accumulators would spill) are read again from L2 instead of being held.  All sums are float; the variance
// is formed from the centred values, so a large common offset does not cancel it.
//
// The weight's and the bias's gradients are sums over rows.  Each thread of the backward kernel owns the same
// columns in every row its block visits, so it keeps their running sums in registers; a block leaves one
// partial row in the workspace and a second kernel adds the partials in a fixed order (no atomics: the same
// inputs give the same bits).
#include <algorithm>

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

namespace {

constexpr int NORM_WARPS = 4;         // rows a block of the one-warp-per-row form holds
constexpr int NORM_MAX_THREADS = 512; // of the one-block-per-row form

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
    a = lane < nwarps ? red[lane][0] : 0.f;
    b = lane < nwarps ? red[lane][1] : 0.f;
#pragma unroll
    for (int o = 8; o; o >>= 1) {
      a += __shfl_xor_sync(FULL, a, o);
      b += __shfl_xor_sync(FULL, b, o);
    }
    a = __shfl_sync(FULL, a, 0);
    b = __shfl_sync(FULL, b, 0);
  }
  return make_float2(a, b);
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
  } else if (dtype == FV_BF16) {
    Pack<__nv_bfloat16, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.e[i] = __float2bfloat16_rn(v[i]);
    store_pack<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p) + at, o);
  } else {
    Pack<__half, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.e[i] = __float2half_rn(v[i]);
    store_pack<__half, VEC>(static_cast<__half*>(p) + at, o);
  }
}

// y in the type `ydt`; VEC elements per access, NV accesses per thread.
template <typename T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 32 * NORM_WARPS)
    k_norm(const T* __restrict__ x, int64_t xs, int64_t rows, int D, const T* __restrict__ w, const T* __restrict__ b, float eps,
           void* __restrict__ y, int ydt, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[2][16][2];
  const int G = BLOCK ? blockDim.x : 32, t = BLOCK ? threadIdx.x : threadIdx.x & 31, nw = BLOCK ? blockDim.x >> 5 : 1;
  const int64_t per = BLOCK ? 1 : NORM_WARPS, first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * NORM_WARPS + (threadIdx.x >> 5);
  const float n = (float)D;
  for (int64_t r = first; r < rows; r += (int64_t)gridDim.x * per) {
    const T* xr = x + r * xs;
    float v[NV][VEC];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
        const Pack<T, VEC> p = load_pack_stream<T, VEC>(xr + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[j][i] = to_f<T>(p.e[i]);
          s += v[j][i];
        }
      }
    }
    const float mean = group_sum2<BLOCK>(s, 0.f, red[0], nw).x / n;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if ((t + j * G) * VEC < D) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          v[j][i] -= mean;
          q = fmaf(v[j][i], v[j][i], q);
        }
      }
    const float rstd = 1.0f / sqrtf(group_sum2<BLOCK>(q, 0.f, red[1], nw).x / n + eps);
    if (t == 0) {
      if (mean_out) mean_out[r] = mean;
      if (rstd_out) rstd_out[r] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = v[j][i] * rstd;
        if (w) {
          const Pack<T, VEC> pw = load_pack<T, VEC>(w + c);
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] *= to_f<T>(pw.e[i]);
        }
        if (b) {
          const Pack<T, VEC> pb = load_pack<T, VEC>(b + c);
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i] += to_f<T>(pb.e[i]);
        }
        store_as<VEC>(y, ydt, r * (int64_t)D + c, o);
      }
    }
  }
}

// Rows too long for registers: three passes, the second and third out of L2.
template <typename T>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
    k_norm_long(const T* __restrict__ x, int64_t xs, int64_t rows, int64_t D, const T* __restrict__ w, const T* __restrict__ b,
                float eps, void* __restrict__ y, int ydt, float* __restrict__ mean_out, float* __restrict__ rstd_out) {
  __shared__ float red[2][16][2];
  const int nw = blockDim.x >> 5;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * xs;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) s += to_f<T>(xr[c]);
    const float mean = group_sum2<true>(s, 0.f, red[0], nw).x / (float)D;
    float q = 0.f;
    for (int64_t c = threadIdx.x; c < D; c += blockDim.x) {
      const float d = to_f<T>(xr[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.0f / sqrtf(group_sum2<true>(q, 0.f, red[1], nw).x / (float)D + eps);
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

// dx, and with a weight the block's partial sums of dw and db in part[blockIdx.x][2][D].
template <typename T, int VEC, int NV, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? NORM_MAX_THREADS : 32 * NORM_WARPS)
    k_norm_grad(const T* __restrict__ dy, int64_t gs, const T* __restrict__ x, int64_t xs, int64_t rows, int D,
                const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ w, T* __restrict__ dx,
                float* __restrict__ part) {
  __shared__ float red[2][16][2];
  __shared__ float cols[BLOCK ? 1 : 2 * 32 * NV * VEC];
  const int G = BLOCK ? blockDim.x : 32, t = BLOCK ? threadIdx.x : threadIdx.x & 31, nw = BLOCK ? blockDim.x >> 5 : 1;
  const int64_t per = BLOCK ? 1 : NORM_WARPS, first = BLOCK ? blockIdx.x : (int64_t)blockIdx.x * NORM_WARPS + (threadIdx.x >> 5);
  const int64_t step = (int64_t)gridDim.x * per;
  const float n = (float)D;
  float dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) dw[j][i] = db[j][i] = 0.f;
  Pack<T, VEC> px[NV], pg[NV];
  auto fetch = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
        px[j] = load_pack_stream<T, VEC>(x + r * xs + c);
        pg[j] = load_pack_stream<T, VEC>(dy + r * gs + c);
      }
    }
  };
  if (first < rows) fetch(first);
  int turn = 0;
  for (int64_t r = first; r < rows; r += step, turn ^= 1) {
    const float mu = mean[r], rs = rstd[r];
    float a = 0.f, q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
        Pack<T, VEC> pw;
        if (w) pw = load_pack<T, VEC>(w + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float g = to_f<T>(pg[j].e[i]), h = (to_f<T>(px[j].e[i]) - mu) * rs;
          const float u = w ? g * to_f<T>(pw.e[i]) : g;
          a += u;
          q = fmaf(u, h, q);
          dw[j][i] = fmaf(g, h, dw[j][i]);
          db[j][i] += g;
        }
      }
    }
    const float2 sums = group_sum2<BLOCK>(a, q, red[turn], nw);
    const float ma = sums.x / n, mq = sums.y / n;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
        Pack<T, VEC> pw, o;
        if (w) pw = load_pack<T, VEC>(w + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float g = to_f<T>(pg[j].e[i]), h = (to_f<T>(px[j].e[i]) - mu) * rs;
          const float u = w ? g * to_f<T>(pw.e[i]) : g;
          o.e[i] = from_f<T>(rs * (u - ma - h * mq));
        }
        store_pack<T, VEC>(dx + r * (int64_t)D + c, o);
      }
    }
    if (r + step < rows) fetch(r + step);
  }
  if (!part) return;
  float* out = part + (int64_t)blockIdx.x * 2 * D;
  if (BLOCK) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (t + j * G) * VEC;
      if (c < D) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          out[c + i] = dw[j][i];
          out[D + c + i] = db[j][i];
        }
      }
    }
  } else {  // the block's warps one after the other, a fixed order
    constexpr int W = 32 * NV * VEC;
    for (int k = 0; k < NORM_WARPS; ++k) {
      if ((threadIdx.x >> 5) == k) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const int c = (t + j * G) * VEC + i;
            cols[c] = (k ? cols[c] : 0.f) + dw[j][i];
            cols[W + c] = (k ? cols[W + c] : 0.f) + db[j][i];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < D; c += blockDim.x) {
      out[c] = cols[c];
      out[D + c] = cols[W + c];
    }
  }
}

// Long rows: dx alone, then the column sums by k_norm_grad_cols.
template <typename T>
__global__ void __launch_bounds__(NORM_MAX_THREADS)
    k_norm_grad_long(const T* __restrict__ dy, int64_t gs, const T* __restrict__ x, int64_t xs, int64_t rows, int64_t D,
                     const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ w, T* __restrict__ dx) {
  __shared__ float red[2][16][2];
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

// out[c] = sum of part[p][c] over p in a fixed order; c runs over dw's and then db's columns.
template <typename T>
__global__ void __launch_bounds__(512)
    k_norm_grad_reduce(const float* __restrict__ part, int64_t P, int64_t D, T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float sum[16][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < 2 * D)
    for (int64_t p = threadIdx.y; p < P; p += 16) s += part[p * 2 * D + c];
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < 2 * D) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += sum[k][threadIdx.x];
    if (c < D)
      dw[c] = from_f<T>(s);
    else
      db[c - D] = from_f<T>(s);
  }
}

struct NormPlan {
  bool is_long, block;
  int vec_bytes;   // width of one access
  int elems;       // elements per thread: 8, 16 or 32
  int threads;
  int64_t grid;
};

// One warp per row while a row fits one (32 elements a lane at most) and there are rows enough to fill the
// GPU with warps; else one block per row.
NormPlan plan_norm(int64_t rows, int64_t D, int dtype, bool grad, int vec_bytes, int sms) {
  NormPlan p{};
  const int64_t most = grad && dtype == FV_F32 ? 8192 : 16384;
  p.is_long = D > most;
  p.vec_bytes = vec_bytes;
  if (p.is_long) {
    p.block = true;
    p.threads = NORM_MAX_THREADS;
    p.grid = std::min<int64_t>(rows, (int64_t)sms * 4);
    return p;
  }
  p.block = !(D <= 256 || (D <= 1024 && rows >= 4 * sms));
  if (!p.block) {
    p.elems = D <= 256 ? 8 : D <= 512 ? 16 : 32;
    p.threads = 32 * NORM_WARPS;
    p.grid = std::min<int64_t>((rows + NORM_WARPS - 1) / NORM_WARPS, (int64_t)sms * (grad ? 4 : 16));
  } else {
    p.elems = D <= 8 * NORM_MAX_THREADS ? 8 : D <= 16 * NORM_MAX_THREADS ? 16 : 32;
    p.threads = (int)(((D + p.elems - 1) / p.elems + 31) / 32 * 32);
    p.grid = std::min<int64_t>(rows, grad ? (int64_t)sms * std::max(1, 1024 / p.threads) : (int64_t)sms * (2048 / p.threads) * 4);
  }
  return p;
}

template <typename T, int VEC, int E>
void launch_norm(const NormPlan& p, cudaStream_t st, const T* x, int64_t xs, int64_t rows, int D, const T* w, const T* b, float eps,
                 void* y, int ydt, float* mean, float* rstd) {
  if (p.block)
    k_norm<T, VEC, E / VEC, true><<<(unsigned)p.grid, p.threads, 0, st>>>(x, xs, rows, D, w, b, eps, y, ydt, mean, rstd);
  else
    k_norm<T, VEC, E / VEC, false><<<(unsigned)p.grid, p.threads, 0, st>>>(x, xs, rows, D, w, b, eps, y, ydt, mean, rstd);
}
template <typename T, int VEC, int E>
void launch_norm_grad(const NormPlan& p, cudaStream_t st, const T* dy, int64_t gs, const T* x, int64_t xs, int64_t rows, int D,
                      const float* mean, const float* rstd, const T* w, T* dx, float* part) {
  if (p.block)
    k_norm_grad<T, VEC, E / VEC, true><<<(unsigned)p.grid, p.threads, 0, st>>>(dy, gs, x, xs, rows, D, mean, rstd, w, dx, part);
  else
    k_norm_grad<T, VEC, E / VEC, false><<<(unsigned)p.grid, p.threads, 0, st>>>(dy, gs, x, xs, rows, D, mean, rstd, w, dx, part);
}

#define NORM_ELEMS(p, T, VEC, FN, ...)                             \
  do {                                                             \
    if ((p).elems == 8) FN<T, VEC, 8>(p, __VA_ARGS__);             \
    else if ((p).elems == 16) FN<T, VEC, 16>(p, __VA_ARGS__);      \
    else FN<T, VEC, 32>(p, __VA_ARGS__);                           \
  } while (0)
#define NORM_VEC(p, T, FN, ...)                                                   \
  do {                                                                            \
    constexpr int V16 = 16 / (int)sizeof(T), V4 = 4 / (int)sizeof(T);             \
    if ((p).vec_bytes == 16) NORM_ELEMS(p, T, V16, FN, __VA_ARGS__);              \
    else if (V4 > 1 && (p).vec_bytes == 4) NORM_ELEMS(p, T, V4, FN, __VA_ARGS__);      \
    else NORM_ELEMS(p, T, 1, FN, __VA_ARGS__);                                    \
  } while (0)

int64_t grad_parts(const NormPlan& p, int64_t rows, int64_t D, int sms) {
  if (!p.is_long) return p.grid;
  const int64_t blocks = (D + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>(rows, (int64_t)sms * 8 / blocks));
}

int norm_vec_bytes(int64_t D, size_t es, std::initializer_list<std::pair<const void*, int64_t>> arrays) {
  for (unsigned bytes : {16u, 4u}) {
    if (bytes <= es && bytes != 16u) break;
    bool ok = D % (int64_t)(bytes / es) == 0;
    for (const auto& a : arrays) ok = ok && (!a.first || vec_ok(a.first, a.second, es, bytes));
    if (ok) return (int)bytes;
  }
  return (int)es;
}

}  // namespace
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
  FV_REQUIRE(eps >= 0.f, FV_ERR_INVALID, "fv_layer_norm: eps must not be negative");
  FV_REQUIRE(!bias || weight, FV_ERR_INVALID, "fv_layer_norm: a bias needs a weight");
  if (rows == 0) return FV_OK;
  FV_REQUIRE(x && y, FV_ERR_INVALID, "fv_layer_norm: NULL argument");
  fv::DeviceGuard guard(device);
  const int sms = sm_count(device);
  FV_REQUIRE(guard.ok && sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  const size_t es = elem_size(dtype);
  int vb = norm_vec_bytes(cols, es, {{x, x_stride}, {weight, 0}, {bias, 0}});
  // y is dense and may be wider than x: its rows must admit the same element count per access
  while (vb > (int)es && ((uintptr_t)y % std::min<size_t>(16, vb / es * elem_size(y_dtype)) != 0)) vb = vb == 16 && es == 2 ? 4 : (int)es;
  const NormPlan p = plan_norm(rows, cols, dtype, false, vb, sms);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  FV_DTYPE_SWITCH(dtype, T, {
    const T *px = static_cast<const T*>(x), *pw = static_cast<const T*>(weight), *pb = static_cast<const T*>(bias);
    if (p.is_long)
      k_norm_long<T><<<(unsigned)p.grid, p.threads, 0, st>>>(px, x_stride, rows, cols, pw, pb, eps, y, y_dtype, mean, rstd);
    else
      NORM_VEC(p, T, launch_norm, st, px, x_stride, rows, (int)cols, pw, pb, eps, y, y_dtype, mean, rstd);
  });
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

static int norm_grad_plan(int device, const void* dy, int64_t gs, const void* x, int64_t xs, int64_t rows, int64_t cols, int dtype,
                          const void* weight, const void* dx, NormPlan* p, int64_t* parts) {
  const int sms = sm_count(device);
  FV_REQUIRE(sms > 0, FV_ERR_CUDA, "cannot select device %d", device);
  const int vb = norm_vec_bytes(cols, elem_size(dtype), {{dy, gs}, {x, xs}, {weight, 0}, {dx, 0}});
  *p = plan_norm(rows, cols, dtype, true, vb, sms);
  *parts = grad_parts(*p, rows, cols, sms);
  return FV_OK;
}

int fv_layer_norm_backward_workspace(int device, int64_t rows, int64_t cols, int dtype, size_t* bytes) {
  FV_CHECK_DTYPE(dtype, "fv_layer_norm_backward_workspace");
  FV_REQUIRE(bytes && rows >= 0 && cols >= 1 && cols < (1ll << 31), FV_ERR_INVALID, "fv_layer_norm_backward_workspace: bad argument");
  NormPlan p;
  int64_t parts = 0;
  if (int rc = norm_grad_plan(device, nullptr, 0, nullptr, 0, rows, cols, dtype, nullptr, nullptr, &p, &parts)) return rc;
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
  fv::DeviceGuard guard(device);
  FV_REQUIRE(guard.ok, FV_ERR_CUDA, "cannot select device %d", device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (rows == 0) {
    FV_CUDA(cudaMemsetAsync(dweight, 0, (size_t)cols * elem_size(dtype), st));
    FV_CUDA(cudaMemsetAsync(dbias, 0, (size_t)cols * elem_size(dtype), st));
    return FV_OK;
  }
  NormPlan p;
  int64_t parts = 0;
  if (int rc = norm_grad_plan(device, dy, dy_stride, x, x_stride, rows, cols, dtype, weight, dx, &p, &parts)) return rc;
  const size_t need = (size_t)parts * 2 * (size_t)cols * sizeof(float);
  FV_REQUIRE(!weight || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0), FV_ERR_INVALID,
             "fv_layer_norm_backward: the workspace must be 16-byte aligned and hold %llu bytes, got %llu", (unsigned long long)need,
             (unsigned long long)workspace_bytes);
  float* part = weight ? static_cast<float*>(workspace) : nullptr;
  FV_DTYPE_SWITCH(dtype, T, {
    const T *pg = static_cast<const T*>(dy), *px = static_cast<const T*>(x), *pw = static_cast<const T*>(weight);
    T* pd = static_cast<T*>(dx);
    if (p.is_long) {
      k_norm_grad_long<T><<<(unsigned)p.grid, p.threads, 0, st>>>(pg, dy_stride, px, x_stride, rows, cols, mean, rstd, pw, pd);
      if (part)
        k_norm_grad_cols<T><<<dim3((unsigned)((cols + 255) / 256), (unsigned)parts), 256, 0, st>>>(pg, dy_stride, px, x_stride, rows, cols,
                                                                                                  mean, rstd, part);
    } else {
      NORM_VEC(p, T, launch_norm_grad, st, pg, dy_stride, px, x_stride, rows, (int)cols, mean, rstd, pw, pd, part);
    }
    if (part)
      k_norm_grad_reduce<T><<<(unsigned)((2 * cols + 31) / 32), dim3(32, 16), 0, st>>>(part, parts, cols, static_cast<T*>(dweight),
                                                                                       static_cast<T*>(dbias));
  });
  FV_CUDA(cudaGetLastError());
  return FV_OK;
}

}  // extern "C"
