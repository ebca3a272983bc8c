// Helpers shared by the dense operators (fv_norm.cu, fv_logprob.cu, fv_linear.cu): element types, 16-byte
// vectors of them, reductions.  Nothing here allocates or synchronises.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <math_constants.h>

#include "fv_common.h"

namespace fvo {

constexpr unsigned FULL = 0xffffffffu;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements moved by one access.  VEC * sizeof(T) is 16, 8, 4 or 2 bytes and the address a
// multiple of it.
template <int BYTES>
struct Word;
template <>
struct Word<16> { using type = uint4; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<4> { using type = unsigned; };
template <>
struct Word<2> { using type = unsigned short; };

template <typename T, int VEC>
union Pack {
  typename Word<(int)sizeof(T) * VEC>::type w;
  T e[VEC];
  __device__ __forceinline__ Pack() {}
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  Pack<T, VEC> r;
  r.w = *reinterpret_cast<const decltype(r.w)*>(p);
  return r;
}
// read once: keep it out of L1
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack_stream(const T* p) {
  Pack<T, VEC> r;
  r.w = __ldcs(reinterpret_cast<const decltype(r.w)*>(p));
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<decltype(v.w)*>(p) = v.w;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}

// ---- single instructions ----
__device__ __forceinline__ float ex2(float x) {  // 2^x, to 2^-22; results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {  // 1 / x, to 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// larger and smaller of two, a NaN if either is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
// After a wait that ran out: the asynchronous copies in flight must land before the block's shared memory goes to another.
// They depend on nothing but memory, which this (some 50 ms) outlasts by far.
__device__ __forceinline__ void outlast_copies() {
  const long long t0 = clock64();
  while (clock64() - t0 < 100000000ll) __nanosleep(10000);
}
// two float operations at a time
__device__ __forceinline__ unsigned long long pack2(float2 v) { return *reinterpret_cast<unsigned long long*>(&v); }
__device__ __forceinline__ float2 unpack2(unsigned long long v) { return *reinterpret_cast<float2*>(&v); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x)), "l"(pack2(y)));
  return unpack2(r);
}
__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x)), "l"(pack2(y)));
  return unpack2(r);
}
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(x)), "l"(pack2(y)), "l"(pack2(z)));
  return unpack2(r);
}

// two 16-bit elements of a 32-bit word as floats, and back (one conversion for both)
template <typename T>
__device__ __forceinline__ float2 widen2(unsigned w);
template <>
__device__ __forceinline__ float2 widen2<__nv_bfloat16>(unsigned w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 widen2<__half>(unsigned w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <typename T>
__device__ __forceinline__ unsigned join2(float2 v);
template <>
__device__ __forceinline__ unsigned join2<__nv_bfloat16>(float2 v) {
  const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&r);
}
template <>
__device__ __forceinline__ unsigned join2<__half>(float2 v) {
  const __half2 r = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const unsigned*>(&r);
}
// the i-th pair of elements of a 16-byte word
template <typename T>
__device__ __forceinline__ float2 pair_of(const uint4& q, int i) {
  const unsigned w[4] = {q.x, q.y, q.z, q.w};
  if constexpr (sizeof(T) == 4)
    return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  else
    return widen2<T>(w[i]);
}
// a 16-byte word of pairs
template <typename T>
__device__ __forceinline__ uint4 word_of(const float2 (&v)[8 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
  else
    return make_uint4(join2<T>(v[0]), join2<T>(v[1]), join2<T>(v[2]), join2<T>(v[3]));
}

// Sums of the columns of part[P][n] in a fixed order, 32 columns to a block of 512 threads: four columns to a thread, 64
// rows at a time, then a tree.  `out(c, v)` is called once per column.
template <typename F>
__device__ __forceinline__ void column_sums(const float* __restrict__ part, int64_t P, int64_t n, F out) {
  __shared__ float4 sum[64][8];
  const int q = threadIdx.x & 7, lane = threadIdx.x >> 3;
  const int64_t c = (int64_t)blockIdx.x * 32 + 4 * q;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (n % 4 == 0 && c < n) {
#pragma unroll 8
    for (int64_t p = lane; p < P; p += 64) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(part + p * n + c));
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
  } else {
#pragma unroll 4
    for (int64_t p = lane; p < P; p += 64) {
      const float* v = part + p * n + c;
      if (c < n) s.x += v[0];
      if (c + 1 < n) s.y += v[1];
      if (c + 2 < n) s.z += v[2];
      if (c + 3 < n) s.w += v[3];
    }
  }
  sum[lane][q] = s;
  for (int k = 32; k; k >>= 1) {
    __syncthreads();
    if (lane < k) {
      const float4 v = sum[lane + k][q];
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
      sum[lane][q] = s;
    }
  }
  if (lane == 0) {
    if (c < n) out(c, s.x);
    if (c + 1 < n) out(c + 1, s.y);
    if (c + 2 < n) out(c + 2, s.z);
    if (c + 3 < n) out(c + 3, s.w);
  }
}

inline bool vec_ok(const void* p, int64_t stride_elems, size_t elem, unsigned bytes) {
  return (uintptr_t)p % bytes == 0 && ((uint64_t)stride_elems * elem) % bytes == 0;
}
inline size_t elem_size(int dtype) { return dtype == FV_F32 ? 4 : 2; }

// Makes `device` current for the scope.  Unlike fv::DeviceGuard it leaves the runtime alone when it already is: two calls
// of 0.2 us saved where a whole operator call takes ten.
struct OnDevice {
  int prev = -1;
  bool ok = false;
  explicit OnDevice(int device) {
    int now = -1;
    if (cudaGetDevice(&now) != cudaSuccess) return;
    if (now == device) {
      ok = true;
      return;
    }
    ok = cudaSetDevice(device) == cudaSuccess;
    if (ok) prev = now;
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
};

// Cycles after which a bounded wait inside a kernel gives up, about two seconds; wait_limit answers what the next launches get
// (and sets it first: -1 the default, 0 waits that last no longer than a look).
constexpr long long WAIT_LIMIT = 4000000000ll;
long long wait_limit(long long set = -2);

int sm_count(int device);  // cached per device; 0 after an error

// Reads and clears a word of error bits in device memory in one step, so that a bit raised meanwhile is not lost.  The caller
// (fv_ops_status) has waited for the device and lets no other thread in.
cudaError_t take_status(unsigned* bits, uint32_t* word);
cudaError_t norm_status(uint32_t* word);  // that of fv_norm.cu's kernels

}  // namespace fvo

#define FV_DTYPE_SWITCH(code, T, ...)         \
  switch (code) {                             \
    case FV_F32: {                            \
      using T = float;                        \
      __VA_ARGS__;                            \
      break;                                  \
    }                                         \
    case FV_BF16: {                           \
      using T = __nv_bfloat16;                \
      __VA_ARGS__;                            \
      break;                                  \
    }                                         \
    default: {                                \
      using T = __half;                       \
      __VA_ARGS__;                            \
    }                                         \
  }

#define FV_CHECK_DTYPE(code, what) \
  FV_REQUIRE((code) == FV_F32 || (code) == FV_BF16 || (code) == FV_F16, FV_ERR_INVALID, what ": unknown element type %d", (int)(code))
