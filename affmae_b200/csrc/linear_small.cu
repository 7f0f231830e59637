// Matrix product for a few rows (serving: single tokens).
//
// y[m,n] = sum_k x[m,k] w[n,k] with M <= 8 is bound by reading w once, so
// there is nothing for the tensor cores to reuse: a warp takes a weight row
// (four where there are several rows of x, whose loads and conversions they
// then share), streams it with 16-byte loads, multiplies it with every row of
// x (which stays in L1) in fp32 and reduces across the lanes; the epilogue
// follows in the same launch.
#include "activation.cuh"
#include "linear.cuh"

#include <cuda_fp8.h>

#include <type_traits>

namespace affb {

constexpr int SR_WARPS = 8;

struct e4m3 { uint8_t v; };

// 16 bytes of a row as fp32.
template <typename T> struct Pack16;
template <> struct Pack16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void get(const uint4& u, float* o) {
    o[0] = __uint_as_float(u.x); o[1] = __uint_as_float(u.y); o[2] = __uint_as_float(u.z); o[3] = __uint_as_float(u.w);
  }
};
template <> struct Pack16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float* o) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <> struct Pack16<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void get(const uint4& u, float* o) {
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      o[2 * i] = f.x; o[2 * i + 1] = f.y;
    }
  }
};
__device__ __forceinline__ float2 e4m3x2(uint16_t p) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)p, __NV_E4M3);
  return __half22float2(__half2(h));
}
template <> struct Pack16<e4m3> {
  static constexpr int N = 16;
  static __device__ __forceinline__ void get(const uint4& u, float* o) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = e4m3x2((uint16_t)(w[i] & 0xffffu)), b = e4m3x2((uint16_t)(w[i] >> 16));
      o[4 * i] = a.x; o[4 * i + 1] = a.y; o[4 * i + 2] = b.x; o[4 * i + 3] = b.y;
    }
  }
};
template <typename T> __device__ __forceinline__ float one(const T* p) { return ldf(p); }
template <> __device__ __forceinline__ float one<e4m3>(const e4m3* p) { return e4m3x2((uint16_t)p->v).x; }

__device__ __forceinline__ float small_load(const void* p, int dtype, int64_t i) {
  if (dtype == AFFB_F32) return ((const float*)p)[i];
  if (dtype == AFFB_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void small_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == AFFB_F32) ((float*)p)[i] = v;
  else if (dtype == AFFB_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}

// Element group g of a 16-byte vector as fp32: 4 values of e4m3 or fp32, 8 of
// the 16-bit types, so that a group is unpacked into few registers.
template <typename T> struct Group { static constexpr int N = 8, COUNT = 1; };
template <> struct Group<float> { static constexpr int N = 4, COUNT = 1; };
template <> struct Group<e4m3> { static constexpr int N = 4, COUNT = 4; };
template <typename T>
__device__ __forceinline__ void unpack_group(const uint4& u, int g, float* o) {
  if constexpr (std::is_same<T, e4m3>::value) {
    const uint32_t w = g == 0 ? u.x : g == 1 ? u.y : g == 2 ? u.z : u.w;
    const float2 a = e4m3x2((uint16_t)(w & 0xffffu)), b = e4m3x2((uint16_t)(w >> 16));
    o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
  } else {
    Pack16<T>::get(u, o);
  }
}

__device__ __forceinline__ void small_finish(float v, int m, int64_t n, int64_t N, const LinearEpilogue& e) {
  const int64_t i = (int64_t)m * N + n;
  if (e.row_scale) v *= e.row_scale[m];
  if (e.col_scale) v *= e.col_scale[n];
  if (e.bias) v += small_load(e.bias, e.bias_dtype, n);
  if (e.z) small_store(e.z, e.z_dtype, i, v);
  switch (e.act) {
    case AFFB_ACT_RELU: v = activate<AFFB_ACT_RELU>(v); break;
    case AFFB_ACT_GELU: v = activate<AFFB_ACT_GELU>(v); break;
    case AFFB_ACT_SILU: v = activate<AFFB_ACT_SILU>(v); break;
    default: break;
  }
  if (e.residual) v += small_load(e.residual, e.residual_dtype, i);
  small_store(e.out, e.out_dtype, i, v);
}

// MR: rows of x (M <= MR); NC: weight rows of a warp.
template <typename T, int MR, int NC, bool VEC>
__global__ void __launch_bounds__(SR_WARPS * 32) small_rows_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                   int M, int64_t N, int64_t K, LinearEpilogue e) {
  const int lane = threadIdx.x & 31;
  const int64_t n0 = ((int64_t)blockIdx.x * SR_WARPS + (threadIdx.x >> 5)) * NC;
  if (n0 >= N) return;
  float acc[MR][NC];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[m][c] = 0.f;
  const T* wr[NC];  // past the last row: that row again
#pragma unroll
  for (int c = 0; c < NC; ++c) wr[c] = w + (n0 + c < N ? n0 + c : N - 1) * K;
  if constexpr (VEC) {
    const int64_t kv = K / Pack16<T>::N;
#pragma unroll(MR == 1 ? 4 : 2)
    for (int64_t k = lane; k < kv; k += 32) {
      uint4 a[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) a[c] = __ldg(reinterpret_cast<const uint4*>(wr[c]) + k);
#pragma unroll
      for (int g = 0; g < Group<T>::COUNT; ++g) {
        constexpr int P = Group<T>::N;
        float wv[NC][P];
#pragma unroll
        for (int c = 0; c < NC; ++c) unpack_group<T>(a[c], g, wv[c]);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
          if (m < M) {
            float b[P];
            unpack_group<T>(__ldg(reinterpret_cast<const uint4*>(x + m * K) + k), g, b);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int i = 0; i < P; ++i) acc[m][c] = fmaf(wv[c][i], b[i], acc[m][c]);
          }
        }
      }
    }
  } else {
    for (int64_t k = lane; k < K; k += 32) {
      float a[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) a[c] = one<T>(wr[c] + k);
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        if (m < M) {
          const float b = one<T>(x + m * K + k);
#pragma unroll
          for (int c = 0; c < NC; ++c) acc[m][c] = fmaf(a[c], b, acc[m][c]);
        }
      }
    }
  }
  // lane m * NC + c finishes output (m, n0 + c)
  float v = 0.f;
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float sum = warp_sum(acc[m][c]);
      if (lane == m * NC + c) v = sum;
    }
  const int m = lane / NC, c = lane % NC;
  if (m < MR && m < M && n0 + c < N) small_finish(v, m, n0 + c, N, e);
}

template <typename T, int MR, int NC, bool VEC>
static void small_go(const void* x, const void* w, int M, int64_t N, int64_t K, const LinearEpilogue& e,
                     cudaStream_t st) {
  const unsigned blocks = (unsigned)((N + SR_WARPS * NC - 1) / (SR_WARPS * NC));
  small_rows_kernel<T, MR, NC, VEC><<<blocks, SR_WARPS * 32, 0, st>>>((const T*)x, (const T*)w, M, N, K, e);
}
template <typename T, bool VEC>
static void small_launch(const void* x, const void* w, int M, int64_t N, int64_t K, const LinearEpilogue& e,
                         cudaStream_t st) {
  if (M == 1) small_go<T, 1, 1, VEC>(x, w, M, N, K, e, st);
  else if (M == 2) small_go<T, 2, 4, VEC>(x, w, M, N, K, e, st);
  else if (M <= 4) small_go<T, 4, 4, VEC>(x, w, M, N, K, e, st);
  else small_go<T, 8, 4, VEC>(x, w, M, N, K, e, st);
}

template <typename T>
static void small_align(const void* x, const void* w, int M, int64_t N, int64_t K, const LinearEpilogue& e,
                        cudaStream_t st) {
  const bool vec = K % Pack16<T>::N == 0 && aligned_to(x, 16) && aligned_to(w, 16);
  if (vec) small_launch<T, true>(x, w, M, N, K, e, st);
  else small_launch<T, false>(x, w, M, N, K, e, st);
}

int linear_small(const void* x, const void* w, int dtype, int64_t M, int64_t N, int64_t K, const LinearEpilogue& e,
                 cudaStream_t st) {
  switch (dtype) {
    case AFFB_F32: small_align<float>(x, w, (int)M, N, K, e, st); break;
    case AFFB_F16: small_align<__half>(x, w, (int)M, N, K, e, st); break;
    case AFFB_BF16: small_align<__nv_bfloat16>(x, w, (int)M, N, K, e, st); break;
    default: small_align<e4m3>(x, w, (int)M, N, K, e, st); break;
  }
  AFFB_LAUNCH_CHECK("linear: few rows");
  return AFFB_OK;
}

}  // namespace affb
