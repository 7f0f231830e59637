// Side passes of the matrix product: operand packing for rows that TMA cannot
// address, the fp32 -> 3 x bf16 split, the activation's gradient with the
// bias gradient's column sums, and the sums of partial products.
#include "activation.cuh"
#include "linear.cuh"

#include <type_traits>

namespace affb {

// ------------------------------------------------------------------ pack --
// A warp a row, lanes over its columns.
template <typename U>
__global__ void __launch_bounds__(256) pack_rows_kernel(const U* __restrict__ src, int64_t R, int64_t C,
                                                        U* __restrict__ dst, int64_t ld) {
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < R; r += (int64_t)gridDim.x * 8) {
#pragma unroll 4
    for (int64_t c = threadIdx.x & 31; c < C; c += 32) dst[r * ld + c] = src[r * C + c];
  }
}

int linear_pack(const void* src, int64_t elem, int64_t R, int64_t C, void* dst, int64_t ld, cudaStream_t st) {
  if (R * C == 0) return AFFB_OK;
  const unsigned blocks = (unsigned)imin64((R + 7) / 8, (int64_t)sm_count() * 16);
  if (elem == 1) pack_rows_kernel<uint8_t><<<blocks, 256, 0, st>>>((const uint8_t*)src, R, C, (uint8_t*)dst, ld);
  else pack_rows_kernel<uint16_t><<<blocks, 256, 0, st>>>((const uint16_t*)src, R, C, (uint16_t*)dst, ld);
  AFFB_LAUNCH_CHECK("linear: pack");
  return AFFB_OK;
}

// Three bf16 parts of an fp32 value: each takes the next 8 bits of the
// mantissa, so their sum is the value (up to bf16's exponent range); o[3] is
// the first of a finite value, else 0.
__device__ __forceinline__ void split_value(float v, __nv_bfloat16* o) {
  o[0] = __float2bfloat16_rn(v);
  // the largest fp32 values would round up to infinity
  if (isfinite(v) && !isfinite(__bfloat162float(o[0]))) o[0] = __float2bfloat16_rz(v);
  // an infinity or NaN stays in the first part alone
  const float r1 = isfinite(v) ? v - __bfloat162float(o[0]) : 0.f;
  o[1] = __float2bfloat16_rn(r1);
  o[2] = __float2bfloat16_rn(isfinite(r1) ? r1 - __bfloat162float(o[1]) : 0.f);
  o[3] = isfinite(v) ? o[0] : __float2bfloat16_rn(0.f);
}

// A warp a row of either of two arrays; a lane takes two columns, so that the
// parts are written in words (rows of the parts are 16-byte aligned).
__global__ void __launch_bounds__(256) split_rows_kernel(SplitRows a, SplitRows b) {
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < a.R + b.R; i += (int64_t)gridDim.x * 8) {
    const SplitRows& w = i < a.R ? a : b;
    const int64_t r = i < a.R ? i : i - a.R, part = w.R * w.ld, C = w.C;
    const float* s = w.src + r * C;
    __nv_bfloat16* d = (__nv_bfloat16*)w.dst + r * w.ld;
#pragma unroll 4
    for (int64_t c = (threadIdx.x & 31) * 2; c < C; c += 64) {
      __nv_bfloat16 p[SPLIT_PLANES], q[SPLIT_PLANES];
      split_value(s[c], p);
      split_value(c + 1 < C ? s[c + 1] : 0.f, q);
#pragma unroll
      for (int k = 0; k < SPLIT_PLANES; ++k) *reinterpret_cast<__nv_bfloat162*>(d + c + k * part) = __nv_bfloat162(p[k], q[k]);
    }
  }
}

int linear_split(const SplitRows& a, const SplitRows& b, cudaStream_t st) {
  if (a.R + b.R == 0) return AFFB_OK;
  const unsigned blocks = (unsigned)imin64((a.R + b.R + 7) / 8, (int64_t)sm_count() * 16);
  split_rows_kernel<<<blocks, 256, 0, st>>>(a, b);
  AFFB_LAUNCH_CHECK("linear: split");
  return AFFB_OK;
}

// ---------------------------------------------------- activation gradient --
constexpr int DZ_THREADS = 256;
constexpr int DZ_COLS = 256;   // columns of one block
constexpr int DZ_MIN_ROWS = 64;

int64_t linear_dz_strips(int64_t R, int64_t C) {
  const int64_t cols = (C + DZ_COLS - 1) / DZ_COLS;
  const int64_t want = ((int64_t)sm_count() * 6 + cols - 1) / cols;
  const int64_t most = (R + DZ_MIN_ROWS - 1) / DZ_MIN_ROWS;
  return want < most ? want : (most > 0 ? most : 1);
}

template <typename T, int VEC>
__device__ __forceinline__ void ldn(const T* p, float* o) {
  if constexpr (VEC == 8) {
    ld8(p, o);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[k] = ldf(p + k);
  }
}

// Block: DZ_COLS columns x one strip of rows.  A thread keeps VEC columns and
// walks down the strip; the threads of a column group are summed in order, so
// the sums do not depend on timing (and are of the unrounded gradients).  dz is
// rounded to the operands' type, since the products take operands of one type
// (error of the gradients at 96 -> 192 bf16 GELU 2.3e-3 of their norm, 1.7e-3
// from their own rounding alone).  Bound by HBM, and by what is on the way:
// six blocks an SM, for which the strips are counted (131072 x 768 bf16 ReLU:
// 92 us, 117 with the five that two registers more leave).
template <typename TO, typename T, typename TZ, int ACT, int VEC>
__global__ void __launch_bounds__(DZ_THREADS, 6) dz_kernel(const TO* __restrict__ dout, const TZ* __restrict__ z, int64_t R,
                                                        int64_t C, void* __restrict__ dz, int64_t ld, int64_t strip,
                                                        float* __restrict__ part) {
  constexpr bool SPLIT = std::is_same<T, float>::value;
  __shared__ float red[DZ_THREADS * VEC];
  const int64_t c0 = (int64_t)blockIdx.x * DZ_COLS;
  const int cols = (int)imin64(DZ_COLS, C - c0);
  const int cv = (cols + VEC - 1) / VEC;        // column groups
  const int lanes = DZ_THREADS / cv;            // rows walked side by side
  const int g = threadIdx.x % cv, rl = threadIdx.x / cv;
  const int64_t r0 = (int64_t)blockIdx.y * strip, r1 = imin64(R, r0 + strip);
  const int64_t c = c0 + (int64_t)g * VEC;
  float sum[VEC];
#pragma unroll
  for (int k = 0; k < VEC; ++k) sum[k] = 0.f;
  if (rl < lanes) {
    for (int64_t r = r0 + rl; r < r1; r += lanes) {
      float d[VEC];
      ldn<TO, VEC>(dout + r * C + c, d);
      if constexpr (ACT != AFFB_ACT_NONE) {
        float zz[VEC];
        ldn<TZ, VEC>(z + r * C + c, zz);
#pragma unroll
        for (int k = 0; k < VEC; ++k) d[k] = through_grad<ACT>(d[k], zz[k]);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) sum[k] += d[k];
      if (dz) {
        if constexpr (SPLIT) {
          __nv_bfloat16* o = (__nv_bfloat16*)dz + r * ld + c;
          union { __nv_bfloat16 v[VEC]; uint4 u; } plane[SPLIT_PLANES];
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            __nv_bfloat16 p[SPLIT_PLANES];
            split_value(d[k], p);
#pragma unroll
            for (int i = 0; i < SPLIT_PLANES; ++i) plane[i].v[k] = p[i];
          }
#pragma unroll
          for (int i = 0; i < SPLIT_PLANES; ++i) {
            if constexpr (VEC == 8) *reinterpret_cast<uint4*>(o + i * R * ld) = plane[i].u;
            else o[i * R * ld] = plane[i].v[0];
          }
        } else {
          T* o = (T*)dz + r * ld + c;
          if constexpr (VEC == 8) {
            st8(o, d);
          } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) stf(o + k, d[k]);
          }
        }
      }
    }
  }
  if (!part) return;
#pragma unroll
  for (int k = 0; k < VEC; ++k) red[k * DZ_THREADS + threadIdx.x] = sum[k];
  __syncthreads();
  for (int i = threadIdx.x; i < cols; i += DZ_THREADS) {
    const int gg = i / VEC, k = i % VEC;
    float s = 0.f;
    for (int l = 0; l < lanes; ++l) s += red[k * DZ_THREADS + l * cv + gg];
    part[(int64_t)blockIdx.y * C + c0 + i] = s;
  }
}

template <typename TO, typename T, int ACT>
static int dz_launch(const void* dout, const void* z, int64_t R, int64_t C, void* dz, int64_t ld, float* part,
                     cudaStream_t st) {
  const int64_t strips = linear_dz_strips(R, C);
  const int64_t strip = (R + strips - 1) / strips;
  const dim3 grid((unsigned)((C + DZ_COLS - 1) / DZ_COLS), (unsigned)strips);
  const bool vec = C % 8 == 0 && aligned_to(dout, 16) && aligned_to(z, 16) && aligned_to(dz, 16) && ld % 8 == 0;
  // the type that z_type() names
  using TZ = typename std::conditional<std::is_same<T, __nv_bfloat16>::value &&
                                           (ACT == AFFB_ACT_GELU || ACT == AFFB_ACT_SILU),
                                       __half, T>::type;
  if (vec)
    dz_kernel<TO, T, TZ, ACT, 8><<<grid, DZ_THREADS, 0, st>>>((const TO*)dout, (const TZ*)z, R, C, dz, ld, strip, part);
  else
    dz_kernel<TO, T, TZ, ACT, 1><<<grid, DZ_THREADS, 0, st>>>((const TO*)dout, (const TZ*)z, R, C, dz, ld, strip, part);
  AFFB_LAUNCH_CHECK("linear: activation gradient");
  return AFFB_OK;
}

template <typename TO, typename T>
static int dz_act(int act, const void* dout, const void* z, int64_t R, int64_t C, void* dz, int64_t ld, float* part,
                  cudaStream_t st) {
  switch (act) {
    case AFFB_ACT_RELU: return dz_launch<TO, T, AFFB_ACT_RELU>(dout, z, R, C, dz, ld, part, st);
    case AFFB_ACT_GELU: return dz_launch<TO, T, AFFB_ACT_GELU>(dout, z, R, C, dz, ld, part, st);
    case AFFB_ACT_SILU: return dz_launch<TO, T, AFFB_ACT_SILU>(dout, z, R, C, dz, ld, part, st);
    default: return dz_launch<TO, T, AFFB_ACT_NONE>(dout, z, R, C, dz, ld, part, st);
  }
}

int linear_dz(const void* dout, int dout_dtype, const void* z, int act, int dtype, int64_t R, int64_t C, void* dz,
              int64_t ld, float* part, cudaStream_t st) {
  if (dtype == AFFB_F32) return dz_act<float, float>(act, dout, z, R, C, dz, ld, part, st);
  if (dtype == AFFB_BF16)
    return dout_dtype == AFFB_F32 ? dz_act<float, __nv_bfloat16>(act, dout, z, R, C, dz, ld, part, st)
                                  : dz_act<__nv_bfloat16, __nv_bfloat16>(act, dout, z, R, C, dz, ld, part, st);
  return dout_dtype == AFFB_F32 ? dz_act<float, __half>(act, dout, z, R, C, dz, ld, part, st)
                                : dz_act<__half, __half>(act, dout, z, R, C, dz, ld, part, st);
}

// ------------------------------------------------------- sums of partials --
__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
  if (dtype == AFFB_F32) return ((const float*)p)[i];
  if (dtype == AFFB_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
  if (dtype == AFFB_F32) ((float*)p)[i] = v;
  else if (dtype == AFFB_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}
__device__ __forceinline__ float activate_code(int act, float z) {
  switch (act) {
    case AFFB_ACT_RELU: return activate<AFFB_ACT_RELU>(z);
    case AFFB_ACT_GELU: return activate<AFFB_ACT_GELU>(z);
    case AFFB_ACT_SILU: return activate<AFFB_ACT_SILU>(z);
    default: return z;
  }
}

// Block: 32 consecutive elements x L lanes of parts, summed in a fixed order.
template <int L>
__global__ void __launch_bounds__(32 * L) sum_parts_kernel(const float* __restrict__ part, int S, int64_t M, int64_t N,
                                                           int64_t ld, LinearEpilogue e) {
  __shared__ float red[L][33];
  const int x = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int64_t n = M * N, plane = M * ld;
  for (int64_t i0 = (int64_t)blockIdx.x * 32; i0 < n; i0 += (int64_t)gridDim.x * 32) {
    const int64_t i = i0 + x;
    const int64_t m = i < n ? i / N : 0, c = i < n ? i - m * N : 0;
    float s = 0.f;
    if (i < n) {
      const float* p = part + m * ld + c;
#pragma unroll 8
      for (int k = l; k < S; k += L) s += __ldg(p + k * plane);
    }
    red[l][x] = s;
    __syncthreads();
    if (l == 0 && i < n) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < L; ++k) v += red[k][x];
      if (e.row_scale) v *= e.row_scale[m];
      if (e.col_scale) v *= e.col_scale[c];
      if (e.bias) v += load_as(e.bias, e.bias_dtype, c);
      if (e.z) store_as(e.z, e.z_dtype, i, v);
      v = activate_code(e.act, v);
      if (e.residual) v += load_as(e.residual, e.residual_dtype, i);
      store_as(e.out, e.out_dtype, i, v);
    }
    __syncthreads();
  }
}

// Few parts: a thread sums one element's in order.
__global__ void __launch_bounds__(256) sum_few_parts_kernel(const float* __restrict__ part, int S, int64_t M, int64_t N,
                                                            int64_t ld, LinearEpilogue e) {
  const int64_t n = M * N, plane = M * ld;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / N, c = i - m * N;
    const float* p = part + m * ld + c;
    float v = 0.f;
#pragma unroll 8
    for (int k = 0; k < S; ++k) v += __ldg(p + k * plane);
    if (e.row_scale) v *= e.row_scale[m];
    if (e.col_scale) v *= e.col_scale[c];
    if (e.bias) v += load_as(e.bias, e.bias_dtype, c);
    if (e.z) store_as(e.z, e.z_dtype, i, v);
    v = activate_code(e.act, v);
    if (e.residual) v += load_as(e.residual, e.residual_dtype, i);
    store_as(e.out, e.out_dtype, i, v);
  }
}

int linear_sum(const float* part, int64_t S, int64_t M, int64_t N, int64_t ld, const LinearEpilogue& e,
               cudaStream_t st) {
  if (M * N == 0) return AFFB_OK;
  // Lanes over the parts until the threads fill the GPU: a thread an element
  // streams 12 parts of 768 x 384 in 7 us (with 32 lanes 107), eight lanes sum
  // 74 parts of 192 x 96 in 5.5 us (23 without), 32 lanes 888 parts of 192 in
  // 9 us (24 with eight).
  const int64_t n = M * N, fill = (int64_t)sm_count() * 1024;
  const unsigned blocks = (unsigned)imin64((n + 31) / 32, (int64_t)sm_count() * 32);
  if (n >= fill || S < 8)
    sum_few_parts_kernel<<<(unsigned)imin64((n + 255) / 256, (int64_t)sm_count() * 8), 256, 0, st>>>(part, (int)S, M, N,
                                                                                                     ld, e);
  else if (n * 8 >= fill / 2 || S < 32)
    sum_parts_kernel<8><<<blocks, 256, 0, st>>>(part, (int)S, M, N, ld, e);
  else
    sum_parts_kernel<32><<<blocks, 1024, 0, st>>>(part, (int)S, M, N, ld, e);
  AFFB_LAUNCH_CHECK("linear: sum of partial products");
  return AFFB_OK;
}

}  // namespace affb
