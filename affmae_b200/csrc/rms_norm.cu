// Root-mean-square norm with the residual's addition over rows of C channels:
//   s = x + f delta          (f: factor of the row's group, or 1; delta optional)
//   y = s rstd w,  rstd = (mean(s^2) + eps)^-1/2
// y in fp32 / 16 bits, or as e4m3 values with one fp32 scale per row:
//   scale = max|y| / 448 (1 for a zero row),  q = e4m3(y / scale).
// The statistics use the unrounded fp32 sum.  Backward, with g = dy w:
//   dx = ds + rstd (g - s rstd^2 mean(g s)),  ddelta = f dx,
//   dw = sum over rows of dy s rstd.
//
// Bound by HBM: every tensor is read and written once.  A row of up to
// 32 * 8 * 4 channels is held by one warp in registers, a longer one by a
// block of eight warps (up to 8192 channels in registers, beyond that the row
// is read again for the second pass).  dw is summed per block in row order and
// then over blocks in order, so it does not depend on timing.
#include "common.cuh"

#include <cuda_fp8.h>

namespace affb {

constexpr float E4M3_MAX = 448.f;

struct RmsArgs {
  const void* x;
  const void* delta;       // or null
  const float* row_scale;  // [R / rows_per_scale] or null
  int64_t rows_per_scale;
  const float* w;          // null: rows are quantised as they are, without the norm
  float eps;
  int64_t R;
  int C;
  void* s;                 // x's dtype; null without delta
  float* rstd;             // or null
  void* y;                 // y_dtype, or null
  int y_dtype;
  uint8_t* q;              // e4m3 values, or null
  float* scale;
};

template <typename T, int VEC>
__device__ __forceinline__ void rms_load(const T* p, float* o) {
  if constexpr (VEC == 8) {
    ld8(p, o);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) o[k] = ldf(p + k);
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void rms_store(T* p, const float* v) {
  if constexpr (VEC == 8) {
    st8(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) stf(p + k, v[k]);
  }
}
template <int VEC>
__device__ __forceinline__ void rms_store_as(void* p, int dtype, int64_t i, const float* v) {
  if (dtype == AFFB_F32) rms_store<float, VEC>((float*)p + i, v);
  else if (dtype == AFFB_BF16) rms_store<__nv_bfloat16, VEC>((__nv_bfloat16*)p + i, v);
  else rms_store<__half, VEC>((__half*)p + i, v);
}
template <int VEC>
__device__ __forceinline__ void rms_load_as(const void* p, int dtype, int64_t i, float* v) {
  if (dtype == AFFB_F32) rms_load<float, VEC>((const float*)p + i, v);
  else if (dtype == AFFB_BF16) rms_load<__nv_bfloat16, VEC>((const __nv_bfloat16*)p + i, v);
  else rms_load<__half, VEC>((const __half*)p + i, v);
}
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float* v) {
  if constexpr (VEC == 8) {
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * j], v[4 * j + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * j + 2], v[4 * j + 3]), __NV_SATFINITE, __NV_E4M3);
      o[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(o[0], o[1]);
  } else {
#pragma unroll
    for (int k = 0; k < VEC; ++k) p[k] = __nv_cvt_float_to_fp8(v[k], __NV_SATFINITE, __NV_E4M3);
  }
}

__device__ __forceinline__ float rms_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
struct AddOp { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct MaxOp { __device__ __forceinline__ float operator()(float a, float b) const { return rms_max_nan(a, b); } };

// Reduction over the THREADS / 32 warps that share a row (all lanes get it).
template <int WARPS, typename Op>
__device__ __forceinline__ float row_reduce(float v, float* red, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (WARPS > 1) {
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // red may still be read by the reduction before
    if ((threadIdx.x & 31) == 0) red[warp] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < WARPS; ++i) v = op(v, red[i]);
  }
  return v;
}

// W warps share a row; NV chunks of VEC channels a lane are kept in registers
// (NV == 0: none, the row is read again).
template <typename TX, typename TD, int W, int NV, int VEC>
__global__ void __launch_bounds__(256) rms_fwd_kernel(RmsArgs a) {
  __shared__ float red[8];
  constexpr int ROWS = 8 / W;
  constexpr int KEEP = NV > 0 ? NV : 1;
  const int t = threadIdx.x % (W * 32);
  const int C = a.C;
  const int steps = NV > 0 ? NV : (C + W * 32 * VEC - 1) / (W * 32 * VEC);
  for (int64_t r = (int64_t)blockIdx.x * ROWS + threadIdx.x / (W * 32); r < a.R; r += (int64_t)gridDim.x * ROWS) {
    const float f = a.row_scale ? a.row_scale[r / a.rows_per_scale] : 1.f;
    const TX* x = (const TX*)a.x + r * C;
    const TD* d = (const TD*)a.delta + r * C;
    float v[KEEP][VEC];
    auto row_chunk = [&](int c, float* o) {
      rms_load<TX, VEC>(x + c, o);
      if (a.delta) {
        float dd[VEC];
        rms_load<TD, VEC>(d + c, dd);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = a.row_scale ? fmaf(f, dd[k], o[k]) : o[k] + dd[k];
      }
    };
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * W * 32 + t) * VEC;
      float* o = v[NV > 0 ? i : 0];
#pragma unroll
      for (int k = 0; k < VEC; ++k) o[k] = 0.f;
      if (c < C) {
        row_chunk(c, o);
        if (a.s) rms_store<TX, VEC>((TX*)a.s + r * C + c, o);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) sq = fmaf(o[k], o[k], sq);
    }
    const float rstd = a.w ? 1.f / sqrtf(row_reduce<W>(sq, red, AddOp()) / (float)C + a.eps) : 1.f;
    if (a.rstd && t == 0) a.rstd[r] = rstd;
    float top = 0.f;
    if (a.q) {
#pragma unroll
      for (int i = 0; i < steps; ++i) {
        const int c = (i * W * 32 + t) * VEC;
        if (c < C) {
          float* o = v[NV > 0 ? i : 0];
          if (NV == 0) row_chunk(c, o);
#pragma unroll
          for (int k = 0; k < VEC; ++k) top = rms_max_nan(top, fabsf(a.w ? o[k] * rstd * a.w[c + k] : o[k]));
        }
      }
      top = row_reduce<W>(top, red, MaxOp());
    }
    const float scale = top == 0.f ? 1.f : top / E4M3_MAX;
    if (a.q && t == 0) a.scale[r] = scale;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * W * 32 + t) * VEC;
      if (c < C) {
        float* o = v[NV > 0 ? i : 0];
        if (NV == 0) row_chunk(c, o);
        float y[VEC], wv[VEC];
        if (a.w) rms_load<float, VEC>(a.w + c, wv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) y[k] = a.w ? o[k] * rstd * wv[k] : o[k];
        if (a.q) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) y[k] = y[k] / scale;
          store_e4m3<VEC>(a.q + r * C + c, y);
        } else {
          rms_store_as<VEC>(a.y, a.y_dtype, r * C + c, y);
        }
      }
    }
  }
}

struct RmsBwdArgs {
  const void* dy;          // y_dtype, or null
  int y_dtype;
  const void* ds;          // x's dtype, or null
  const void* s;           // x's dtype: the saved sum (x itself without delta)
  const float* rstd;
  const float* w;
  const float* row_scale;
  int64_t rows_per_scale;
  int64_t R;
  int C;
  void* dx;                // x's dtype, or null
  void* ddelta;            // TD, or null
  float* part;             // [blocks][C] sums of dy s rstd, or null
};

template <typename TX, typename TD, int W, int NV, int VEC>
__global__ void __launch_bounds__(256) rms_bwd_kernel(RmsBwdArgs a) {
  extern __shared__ float dws[];  // [ROWS][C]: sums of each row slot of the block
  __shared__ float red[8];
  constexpr int ROWS = 8 / W;
  constexpr int KEEP = NV > 0 ? NV : 1;
  const int t = threadIdx.x % (W * 32), slot = threadIdx.x / (W * 32);
  const int C = a.C;
  const int steps = NV > 0 ? NV : (C + W * 32 * VEC - 1) / (W * 32 * VEC);
  // the sums of a long row stay in the block's own row of `part`
  float* sums = NV > 0 ? dws + slot * C : (a.part ? a.part + (int64_t)blockIdx.x * C : nullptr);
  if (a.part)
    for (int i = 0; i < steps; ++i) {
      const int c = (i * W * 32 + t) * VEC;
      if (c < C)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sums[c + k] = 0.f;
    }
  for (int64_t r = (int64_t)blockIdx.x * ROWS + slot; r < a.R; r += (int64_t)gridDim.x * ROWS) {
    const float rstd = a.rstd[r];
    float sv[KEEP][VEC], gv[KEEP][VEC];
    auto chunk = [&](int c, float* s, float* g) {
      rms_load<TX, VEC>((const TX*)a.s + r * C + c, s);
#pragma unroll
      for (int k = 0; k < VEC; ++k) g[k] = 0.f;
      if (a.dy) rms_load_as<VEC>(a.dy, a.y_dtype, r * C + c, g);
    };
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * W * 32 + t) * VEC;
      float *s = sv[NV > 0 ? i : 0], *g = gv[NV > 0 ? i : 0];
      if (c < C) {
        chunk(c, s, g);
        float wv[VEC];
        rms_load<float, VEC>(a.w + c, wv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          if (a.part) sums[c + k] += g[k] * s[k] * rstd;
          g[k] *= wv[k];
          dot = fmaf(g[k], s[k], dot);
        }
      }
    }
    if (!a.dx && !a.ddelta) continue;
    const float coef = row_reduce<W>(dot, red, AddOp()) / (float)C * rstd * rstd;
    const float f = a.row_scale ? a.row_scale[r / a.rows_per_scale] : 1.f;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * W * 32 + t) * VEC;
      if (c < C) {
        float *s = sv[NV > 0 ? i : 0], *g = gv[NV > 0 ? i : 0], o[VEC];
        if (NV == 0) {
          chunk(c, s, g);
          float wv[VEC];
          rms_load<float, VEC>(a.w + c, wv);
#pragma unroll
          for (int k = 0; k < VEC; ++k) g[k] *= wv[k];
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = rstd * (g[k] - s[k] * coef);
        if (a.ds) {
          float d[VEC];
          rms_load<TX, VEC>((const TX*)a.ds + r * C + c, d);
#pragma unroll
          for (int k = 0; k < VEC; ++k) o[k] += d[k];
        }
        if (a.dx) rms_store<TX, VEC>((TX*)a.dx + r * C + c, o);
        if (a.ddelta) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) o[k] *= f;
          rms_store<TD, VEC>((TD*)a.ddelta + r * C + c, o);
        }
      }
    }
  }
  if (a.part && NV > 0) {
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) {
      float v = 0.f;
      for (int k = 0; k < ROWS; ++k) v += dws[k * C + c];
      a.part[(int64_t)blockIdx.x * C + c] = v;
    }
  }
}

// dw[c] = sum over blocks of part[block][c], in block order.
__global__ void __launch_bounds__(256) rms_dw_kernel(const float* __restrict__ part, int64_t blocks, int C,
                                                     float* __restrict__ dw) {
  __shared__ float red[8][33];
  const int x = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < C) {
#pragma unroll 4
    for (int64_t b = l; b < blocks; b += 8) v += part[b * C + c];
  }
  red[l][x] = v;
  __syncthreads();
  if (l == 0 && c < C) {
    v = 0.f;
    for (int k = 0; k < 8; ++k) v += red[k][x];
    dw[c] = v;
  }
}

constexpr int RMS_BWD_BLOCKS_PER_SM = 4;
static int64_t rms_bwd_blocks(int64_t R, int rows) {
  return imin64((R + rows - 1) / rows, (int64_t)sm_count() * RMS_BWD_BLOCKS_PER_SM);
}
// Rows a block takes side by side (the kernels' ROWS).
static int rms_rows(int C, bool vec) { return C <= 32 * (vec ? 8 : 1) * 4 ? 8 : 1; }

template <typename TX, typename TD, int VEC>
static void rms_fwd_launch(const RmsArgs& a, cudaStream_t st) {
  const int64_t sms = sm_count();
  const int C = a.C;
#define RMS_FWD(W, NV)                                                                                \
  rms_fwd_kernel<TX, TD, W, NV, VEC>                                                                  \
      <<<(unsigned)imin64((a.R + 8 / W - 1) / (8 / W), sms * 8), 256, 0, st>>>(a)
  if (C <= 32 * VEC) RMS_FWD(1, 1);
  else if (C <= 64 * VEC) RMS_FWD(1, 2);
  else if (C <= 128 * VEC) RMS_FWD(1, 4);
  else if (C <= 256 * VEC) RMS_FWD(8, 1);
  else if (C <= 512 * VEC) RMS_FWD(8, 2);
  else if (C <= 1024 * VEC) RMS_FWD(8, 4);
  else RMS_FWD(8, 0);
#undef RMS_FWD
}

template <typename TX, typename TD, int VEC>
static void rms_bwd_launch(const RmsBwdArgs& a, cudaStream_t st) {
  const int C = a.C;
#define RMS_BWD(W, NV)                                                                                        \
  rms_bwd_kernel<TX, TD, W, NV, VEC><<<(unsigned)rms_bwd_blocks(a.R, 8 / W), 256,                             \
                                       a.part && NV > 0 ? (size_t)(8 / W) * C * 4 : 0, st>>>(a)
  if (C <= 32 * VEC) RMS_BWD(1, 1);
  else if (C <= 64 * VEC) RMS_BWD(1, 2);
  else if (C <= 128 * VEC) RMS_BWD(1, 4);
  else if (C <= 256 * VEC) RMS_BWD(8, 1);
  else if (C <= 512 * VEC) RMS_BWD(8, 2);
  else if (C <= 1024 * VEC) RMS_BWD(8, 4);
  else RMS_BWD(8, 0);
#undef RMS_BWD
}

static bool rms_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

static int rms_check(int x_dtype, int delta_dtype, bool has_delta, int64_t R, int64_t C, const float* row_scale,
                     int64_t groups) {
  const auto ok = [](int d) { return d == AFFB_F32 || d == AFFB_F16 || d == AFFB_BF16; };
  AFFB_REQUIRE(ok(x_dtype) && (!has_delta || ok(delta_dtype)), "rms_norm: inputs must be fp32, fp16 or bf16");
  AFFB_REQUIRE(R >= 0 && C >= 1 && C < (1ll << 30), "rms_norm: needs rows >= 0 and 1 <= channels < 2^30");
  AFFB_REQUIRE(!row_scale || (has_delta && groups >= 1 && R % groups == 0),
               "rms_norm: row_scale needs delta and a group count that divides the rows");
  return AFFB_OK;
}

#define RMS_DISPATCH(xd, dd, TX, TD, ...)                                       \
  AFFB_DISPATCH(xd, TX, {                                                       \
    switch (dd) {                                                               \
      case AFFB_F32: { using TD = float; __VA_ARGS__; break; }                  \
      case AFFB_F16: { using TD = __half; __VA_ARGS__; break; }                 \
      default: { using TD = __nv_bfloat16; __VA_ARGS__; break; }                \
    }                                                                           \
  })

}  // namespace affb

using namespace affb;

extern "C" int affb_rms_norm_fwd(const void* x, int x_dtype, const void* delta, int delta_dtype,
                                 const float* row_scale, int64_t groups, const float* weight, float eps, int64_t R,
                                 int64_t C, void* s, float* rstd, void* y, int y_dtype, void* q, float* q_scale,
                                 void* stream) {
  int rc = rms_check(x_dtype, delta_dtype, delta != nullptr, R, C, row_scale, groups);
  if (rc) return rc;
  AFFB_REQUIRE((y != nullptr) != (q != nullptr) || R == 0, "rms_norm: exactly one of y and q is written");
  AFFB_REQUIRE(!y || y_dtype == AFFB_F32 || y_dtype == AFFB_F16 || y_dtype == AFFB_BF16,
               "rms_norm: y must be fp32, fp16 or bf16");
  AFFB_REQUIRE(!q || q_scale, "rms_norm: q needs q_scale");
  AFFB_REQUIRE(!s || delta, "rms_norm: the sum is written only with delta");
  if (R == 0) return AFFB_OK;
  AFFB_REQUIRE(x && weight, "rms_norm: null pointer");
  RmsArgs a{x, delta, row_scale, row_scale ? R / groups : 1, weight, eps, R, (int)C, s, rstd, y, y_dtype,
            (uint8_t*)q, q_scale};
  const bool vec = C % 8 == 0 && rms_aligned(x) && rms_aligned(delta) && rms_aligned(weight) && rms_aligned(s) &&
                   rms_aligned(y) && ((uintptr_t)q & 7) == 0;
  cudaStream_t st = as_stream(stream);
  const int dd = delta ? delta_dtype : x_dtype;
  RMS_DISPATCH(x_dtype, dd, TX, TD, {
    if (vec) rms_fwd_launch<TX, TD, 8>(a, st);
    else rms_fwd_launch<TX, TD, 1>(a, st);
  });
  AFFB_LAUNCH_CHECK("affb_rms_norm_fwd");
  return AFFB_OK;
}

extern "C" int affb_quantize_e4m3(const void* x, int dtype, int64_t R, int64_t C, void* q, float* q_scale,
                                  void* stream) {
  int rc = rms_check(dtype, dtype, false, R, C, nullptr, 0);
  if (rc) return rc;
  if (R == 0) return AFFB_OK;
  AFFB_REQUIRE(x && q && q_scale, "quantize_e4m3: null pointer");
  RmsArgs a{x, nullptr, nullptr, 1, nullptr, 0.f, R, (int)C, nullptr, nullptr, nullptr, AFFB_F32, (uint8_t*)q, q_scale};
  const bool vec = C % 8 == 0 && rms_aligned(x) && ((uintptr_t)q & 7) == 0;
  cudaStream_t st = as_stream(stream);
  AFFB_DISPATCH(dtype, TX, {
    if (vec) rms_fwd_launch<TX, TX, 8>(a, st);
    else rms_fwd_launch<TX, TX, 1>(a, st);
  });
  AFFB_LAUNCH_CHECK("affb_quantize_e4m3");
  return AFFB_OK;
}

extern "C" int64_t affb_rms_norm_bwd_workspace_bytes(int64_t R, int64_t C) {
  if (R < 1 || C < 1) return 0;
  // sized for either row layout
  return rms_bwd_blocks(R, 1) * C * 4;
}

extern "C" int affb_rms_norm_bwd(const void* dy, int y_dtype, const void* ds, const void* s, int x_dtype,
                                 const float* rstd, const float* weight, const float* row_scale, int64_t groups,
                                 int64_t R, int64_t C, void* dx, void* ddelta, int delta_dtype, float* dweight,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = rms_check(x_dtype, delta_dtype, ddelta != nullptr, R, C, ddelta ? row_scale : nullptr, groups);
  if (rc) return rc;
  AFFB_REQUIRE(!dy || y_dtype == AFFB_F32 || y_dtype == AFFB_F16 || y_dtype == AFFB_BF16,
               "rms_norm: dy must be fp32, fp16 or bf16");
  cudaStream_t st = as_stream(stream);
  if (R == 0) {
    if (dweight && cudaMemsetAsync(dweight, 0, (size_t)C * 4, st) != cudaSuccess) {
      set_error("rms_norm: cannot clear dweight");
      return AFFB_ERR_CUDA;
    }
    return AFFB_OK;
  }
  AFFB_REQUIRE(s && rstd && weight, "rms_norm: null pointer");
  const bool vec = C % 8 == 0 && rms_aligned(dy) && rms_aligned(ds) && rms_aligned(s) && rms_aligned(weight) &&
                   rms_aligned(dx) && rms_aligned(ddelta);
  const int64_t blocks = rms_bwd_blocks(R, rms_rows((int)C, vec));
  AFFB_REQUIRE(!dweight || (workspace && workspace_bytes >= blocks * C * 4), "rms_norm: workspace too small");
  RmsBwdArgs a{dy, y_dtype, ds, s, rstd, weight, row_scale, row_scale ? R / groups : 1, R, (int)C, dx, ddelta,
               dweight ? (float*)workspace : nullptr};
  const int dd = ddelta ? delta_dtype : x_dtype;
  RMS_DISPATCH(x_dtype, dd, TX, TD, {
    if (vec) rms_bwd_launch<TX, TD, 8>(a, st);
    else rms_bwd_launch<TX, TD, 1>(a, st);
  });
  if (dweight) rms_dw_kernel<<<(unsigned)((C + 31) / 32), 256, 0, st>>>((const float*)workspace, blocks, (int)C, dweight);
  AFFB_LAUNCH_CHECK("affb_rms_norm_bwd");
  return AFFB_OK;
}
