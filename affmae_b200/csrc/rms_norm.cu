// Root-mean-square norm with the residual's addition over rows of C channels:
//   s = x + f delta          (f: factor of the row's group, or 1; delta optional)
//   y = s rstd w,  rstd = (mean(s^2) + eps)^-1/2
// y in fp32 / 16 bits, or as e4m3 values with one fp32 scale per row:
//   scale = max|y| / 448 (1 where that is zero),  q = e4m3(y / scale).
// The statistics use the unrounded fp32 sum.  Backward, with g = dy w:
//   dx = ds + rstd (g - s rstd^2 mean(g s)),  ddelta = f dx,
//   dw = sum over rows of dy s rstd.
//
// Bound by HBM: every tensor is read and written once.  A row is shared by
// TPR threads that hold it in registers, NV chunks of VEC channels each; TPR
// is the smallest of 8, 16, 32 and a whole block whose chunks cover the row
// with few idle lanes (96 channels: 16 threads of one chunk; 384: 16 of
// three).  Rows beyond 4 chunks a thread of a block are read again for the
// second pass.  Where there are several rounds of rows a block brings them in
// by bulk copies, two to four rounds ahead (the rows of a round are
// contiguous): registers alone keep too few bytes on the way.  dw is summed per block in row order and then over blocks in
// order, so it does not depend on timing.
#include "tcgen05.cuh"

#include <cuda_fp8.h>

#include <type_traits>

namespace affb {

constexpr float E4M3_MAX = 448.f;

struct RmsArgs {
  const void* x;
  const void* delta;       // or null
  int delta_dtype;
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

// Reduction over the TPR threads that share a row (all of them get it).  A
// block-wide one goes through `red` with one barrier between its writes and
// its reads, so the block's next one may have begun before the last warp has
// read: it must not use the same `red`.
template <int TPR, typename Op>
__device__ __forceinline__ float row_reduce(float v, float* red, Op op) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 32; ++i) v = op(v, red[i]);
  }
  return v;
}

// Rounds of rows on their way into shared memory: up to four arrays with the
// same rows, stage after stage.
struct RowPipe {
  const void* src[4];
  int row_bytes[4];   // 0: no such array
  int rows;           // of a round
  int stages;
  int stage_bytes;
  int* failed;        // the device's failure word
};
constexpr int PIPE_HEAD = 128;  // barriers and the failure flag, before the stages

template <int ROWS>
struct PipeReader {
  const RowPipe& p;
  unsigned char* base;
  uint32_t bars;
  volatile int* failed;
  int64_t R;
  int stage;
  uint32_t phase;

  __device__ __forceinline__ PipeReader(const RowPipe& pipe, unsigned char* smem, int64_t rows) : p(pipe), R(rows) {
    base = smem + PIPE_HEAD;
    bars = tc5::smem_addr(smem);
    failed = reinterpret_cast<volatile int*>(smem + 64);
    stage = 0;
    phase = 0;
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) tc5::bar_init(bars + 8 * i, 1);
      tc5::bar_init_fence();
      *failed = 0;
    }
    __syncthreads();
    if (threadIdx.x == 0)
      for (int i = 0; i < p.stages; ++i) issue(i, i);
  }
  // One thread: the copies of this block's round `it` into stage `st`.
  __device__ __forceinline__ void issue(int64_t it, int st) {
    const int64_t r0 = ((int64_t)blockIdx.x + it * gridDim.x) * ROWS;
    if (r0 >= R) return;
    const int n = (int)imin64(ROWS, R - r0);
    tc5::bar_expect(bars + 8 * st, (uint32_t)(n * (p.row_bytes[0] + p.row_bytes[1] + p.row_bytes[2] + p.row_bytes[3])));
    uint32_t to = tc5::smem_addr(base + st * p.stage_bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.row_bytes[i]) {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                     "l"((const unsigned char*)p.src[i] + r0 * p.row_bytes[i]), "r"(n * p.row_bytes[i]),
                     "r"(bars + 8 * st)
                     : "memory");
        to += ROWS * p.row_bytes[i];
      }
    }
  }
  // All threads: the round has landed; false (for all) when a wait ran out.
  __device__ __forceinline__ bool wait() {
    return !__syncthreads_or(!tc5::bar_wait(bars + 8 * stage, phase, failed));
  }
  // Row `slot` of array i of the current round.
  __device__ __forceinline__ const unsigned char* row(int i, int slot) const {
    const unsigned char* q = base + stage * p.stage_bytes;
    for (int j = 0; j < i; ++j) q += ROWS * p.row_bytes[j];
    return q + slot * p.row_bytes[i];
  }
  // All threads are done with the round `it`: its stage takes round it + stages.
  __device__ __forceinline__ void next(int64_t it) {
    __syncthreads();
    if (threadIdx.x == 0) issue(it + p.stages, stage);
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
  }
  // After a wait that ran out: what is still on its way has to land.
  __device__ __forceinline__ void give_up(int64_t it) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < p.stages; ++i) {
        const int st = (stage + i) % p.stages;
        if (((int64_t)blockIdx.x + (it + i) * gridDim.x) * ROWS < R)
          tc5::bar_drain(bars + 8 * st, stage + i >= p.stages ? phase ^ 1 : phase);
      }
      report_failure(p.failed);
    }
  }
};

template <bool PIPE, typename T, int VEC>
__device__ __forceinline__ void row_load(const T* global, const unsigned char* staged, int c, float* o) {
  if constexpr (PIPE) ld8_shared(reinterpret_cast<const T*>(staged) + c, o);
  else rms_load<T, VEC>(global + c, o);
}
template <bool PIPE, int VEC>
__device__ __forceinline__ void row_load_as(const void* global, int dtype, int64_t i, const unsigned char* staged, int c,
                                            float* o) {
  if constexpr (PIPE) {
    if (dtype == AFFB_F32) ld8_shared(reinterpret_cast<const float*>(staged) + c, o);
    else if (dtype == AFFB_BF16) ld8_shared(reinterpret_cast<const __nv_bfloat16*>(staged) + c, o);
    else ld8_shared(reinterpret_cast<const __half*>(staged) + c, o);
  } else {
    rms_load_as<VEC>(global, dtype, i + c, o);
  }
}

template <bool PIPE, int ROWS>
__device__ __forceinline__ auto make_reader(const RowPipe& p, unsigned char* smem, int64_t R) {
  if constexpr (PIPE) return PipeReader<ROWS>(p, smem, R);
  else return char(0);
}

__device__ __forceinline__ float group_scale(const float* row_scale, int64_t r, int64_t rows_per_scale) {
  // 32-bit division where it fits: a 64-bit one costs as much as a narrow row
  const int64_t g = (r | rows_per_scale) >> 31 ? r / rows_per_scale : (int64_t)((uint32_t)r / (uint32_t)rows_per_scale);
  return row_scale[g];
}

// NV == 0: the row is read again instead of kept.  PIPE: rows come through
// shared memory (x, delta).
template <typename TX, int TPR, int NV, int VEC, bool PIPE>
__global__ void __launch_bounds__(256) rms_fwd_kernel(const __grid_constant__ RmsArgs a,
                                                      const __grid_constant__ RowPipe pipe) {
  extern __shared__ __align__(128) unsigned char staged[];
  // sums of squares and maxima, two rows of each in turn: without the norm the maximum is a row's only reduction
  __shared__ float red[4][8];
  constexpr int ROWS = 256 / TPR;
  constexpr int KEEP = NV > 0 ? NV : 1;
  const int t = threadIdx.x % TPR;
  const int C = a.C;
  const float inv_c = 1.f / (float)C;
  int flip = 0;
  const int steps = NV > 0 ? NV : (C + TPR * VEC - 1) / (TPR * VEC);
  const int slot = threadIdx.x / TPR;
  PipeReader<ROWS>* reader = nullptr;
  typename std::conditional<PIPE, PipeReader<ROWS>, char>::type store = make_reader<PIPE, ROWS>(pipe, staged, a.R);
  if constexpr (PIPE) reader = &store;
  int64_t it = 0;
  // the threads of a warp stay together (shuffles): rows past the end are computed on nothing
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.R; r0 += (int64_t)gridDim.x * ROWS, ++it) {
    if constexpr (PIPE) {
      if (!reader->wait()) {
        reader->give_up(it);
        break;
      }
    }
    const int64_t r = r0 + slot;
    const bool in = r < a.R;
    const float f = a.row_scale && in ? group_scale(a.row_scale, r, a.rows_per_scale) : 1.f;
    const TX* x = (const TX*)a.x + r * C;
    float v[KEEP][VEC];
    auto row_chunk = [&](int c, float* o) {
      row_load<PIPE, TX, VEC>(x, PIPE ? reader->row(0, slot) : nullptr, c, o);
      if (a.delta) {
        float dd[VEC];
        row_load_as<PIPE, VEC>(a.delta, a.delta_dtype, r * C, PIPE ? reader->row(1, slot) : nullptr, c, dd);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = a.row_scale ? fmaf(f, dd[k], o[k]) : o[k] + dd[k];
      }
    };
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * TPR + t) * VEC;
      float* o = v[NV > 0 ? i : 0];
#pragma unroll
      for (int k = 0; k < VEC; ++k) o[k] = 0.f;
      if (in && c < C) {
        row_chunk(c, o);
        if (a.s) rms_store<TX, VEC>((TX*)a.s + r * C + c, o);
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) sq = fmaf(o[k], o[k], sq);
    }
    float rstd = 1.f;
    if (a.w) {
      rstd = rsqrtf(row_reduce<TPR>(sq, red[flip], AddOp()) * inv_c + a.eps);
      if (a.rstd && in && t == 0) a.rstd[r] = rstd;
    }
    // y: kept in place of the row
    auto normed = [&](int c, float* o) {
      if (a.w) {
        float wv[VEC];
        rms_load<float, VEC>(a.w + c, wv);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = o[k] * rstd * wv[k];
      }
    };
    float top = 0.f, scale = 1.f, inv = 0.f;
    if (a.q) {
#pragma unroll
      for (int i = 0; i < steps; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (in && c < C) {
          float* o = v[NV > 0 ? i : 0];
          if (NV == 0) row_chunk(c, o);
          normed(c, o);
#pragma unroll
          for (int k = 0; k < VEC; ++k) top = rms_max_nan(top, fabsf(o[k]));
        }
      }
      top = row_reduce<TPR>(top, red[2 + flip], MaxOp());
      scale = top / E4M3_MAX;
      if (scale == 0.f) scale = 1.f;  // a row of zeros, or of values whose scale would be less than 2^-150
      if (in && t == 0) a.scale[r] = scale;
      // y is off by a few units in the last place, next to which the reciprocal's rounding is nothing (16384 x 4096
      // bf16: 93 us, 107 with divisions); rows that are quantised as they are, and those whose scale has no
      // reciprocal, are divided, since values that lie at a tie would move by a step
      if (a.w) inv = 1.f / scale;
      if (isinf(inv)) inv = 0.f;
    }
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (in && c < C) {
        float* o = v[NV > 0 ? i : 0];
        if (NV == 0) row_chunk(c, o);
        if (NV == 0 || !a.q) normed(c, o);
        if (a.q) {
          if (inv != 0.f) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) o[k] *= inv;
          } else {
            for (int k = 0; k < VEC; ++k) o[k] /= scale;
          }
          store_e4m3<VEC>(a.q + r * C + c, o);
        } else {
          rms_store_as<VEC>(a.y, a.y_dtype, r * C + c, o);
        }
      }
    }
    flip ^= 1;
    if constexpr (PIPE) reader->next(it);
  }
}

struct RmsBwdArgs {
  const void* dy;          // y_dtype, or null
  int y_dtype;
  const void* ds;          // x's dtype, or null
  const void* s;           // x's dtype: the saved sum, or x where delta is given
  const void* delta;       // delta_dtype: the sum is x + f delta again (a 16-bit sum is not what was normed), or null
  const float* rstd;
  const float* w;
  const float* row_scale;
  int64_t rows_per_scale;
  int64_t R;
  int C;
  void* dx;                // x's dtype, or null
  void* ddelta;            // or null
  int delta_dtype;
  float* part;             // [blocks][C] sums of dy s rstd, or null
};

// PIPE: rows come through shared memory (s, dy, ds, delta).
template <typename TX, int TPR, int NV, int VEC, bool PIPE>
__global__ void __launch_bounds__(256) rms_bwd_kernel(const __grid_constant__ RmsBwdArgs a,
                                                      const __grid_constant__ RowPipe pipe) {
  extern __shared__ __align__(128) unsigned char staged[];
  float* dws = reinterpret_cast<float*>(staged);  // at the end: [ROWS][C], sums of each row slot of the block
  __shared__ float red[2][8];
  constexpr int ROWS = 256 / TPR;
  constexpr int KEEP = NV > 0 ? NV : 1;
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int C = a.C;
  const float inv_c = 1.f / (float)C;
  const int steps = NV > 0 ? NV : (C + TPR * VEC - 1) / (TPR * VEC);
  float sums[KEEP][VEC], wv[KEEP][VEC];
  // the sums of a row too long for registers stay in the block's own row of `part`
  float* far = NV == 0 && a.part ? a.part + (int64_t)blockIdx.x * C : nullptr;
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    const int c = (i * TPR + t) * VEC;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
      sums[NV > 0 ? i : 0][k] = 0.f;
      if (far && c < C) far[c + k] = 0.f;
    }
    if (NV > 0 && c < C) rms_load<float, VEC>(a.w + c, wv[NV > 0 ? i : 0]);
  }
  int flip = 0;
  PipeReader<ROWS>* reader = nullptr;
  typename std::conditional<PIPE, PipeReader<ROWS>, char>::type store = make_reader<PIPE, ROWS>(pipe, staged, a.R);
  if constexpr (PIPE) reader = &store;
  int64_t it = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * ROWS; r0 < a.R; r0 += (int64_t)gridDim.x * ROWS, ++it) {
    const int64_t r = r0 + slot;
    const bool in = r < a.R;
    if constexpr (PIPE) {
      if (!reader->wait()) {
        reader->give_up(it);
        break;
      }
    }
    const float rstd = in ? a.rstd[r] : 0.f;
    const float f = a.row_scale && in ? group_scale(a.row_scale, r, a.rows_per_scale) : 1.f;
    float sv[KEEP][VEC], gv[KEEP][VEC];
    auto chunk = [&](int c, float* s, float* g) {
      row_load<PIPE, TX, VEC>((const TX*)a.s + r * C, PIPE ? reader->row(0, slot) : nullptr, c, s);
      if (a.delta) {
        float dd[VEC];
        row_load_as<PIPE, VEC>(a.delta, a.delta_dtype, r * C, PIPE ? reader->row(3, slot) : nullptr, c, dd);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s[k] = a.row_scale ? fmaf(f, dd[k], s[k]) : s[k] + dd[k];
      }
#pragma unroll
      for (int k = 0; k < VEC; ++k) g[k] = 0.f;
      if (a.dy) row_load_as<PIPE, VEC>(a.dy, a.y_dtype, r * C, PIPE ? reader->row(1, slot) : nullptr, c, g);
      if (NV == 0) rms_load<float, VEC>(a.w + c, wv[0]);
    };
    float dot = 0.f;
    float dv[KEEP][VEC];  // ds, requested with the rest of the row
    if (NV > 0 && !PIPE && a.ds && in) {
#pragma unroll
      for (int i = 0; i < steps; ++i) {
        const int c = (i * TPR + t) * VEC;
        if (c < C) rms_load<TX, VEC>((const TX*)a.ds + r * C + c, dv[NV > 0 ? i : 0]);
      }
    }
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * TPR + t) * VEC, n = NV > 0 ? i : 0;
      if (in && c < C) {
        chunk(c, sv[n], gv[n]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const float gs = gv[n][k] * sv[n][k];
          if (far) far[c + k] += gs * rstd;
          else sums[n][k] = fmaf(gs, rstd, sums[n][k]);
          dot = fmaf(gs, wv[n][k], dot);
        }
      }
    }
    if (!a.dx && !a.ddelta) {
      if constexpr (PIPE) reader->next(it);
      continue;
    }
    const float coef = row_reduce<TPR>(dot, red[flip], AddOp()) * inv_c * rstd * rstd;
    flip ^= 1;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int c = (i * TPR + t) * VEC, n = NV > 0 ? i : 0;
      if (in && c < C) {
        float o[VEC];
        if (NV == 0) chunk(c, sv[0], gv[0]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) o[k] = rstd * (gv[n][k] * wv[n][k] - sv[n][k] * coef);
        if (a.ds) {
          if (NV == 0 || PIPE)
            row_load<PIPE, TX, VEC>((const TX*)a.ds + r * C, PIPE ? reader->row(2, slot) : nullptr, c, dv[n]);
#pragma unroll
          for (int k = 0; k < VEC; ++k) o[k] += dv[n][k];
        }
        if (a.dx) rms_store<TX, VEC>((TX*)a.dx + r * C + c, o);
        if (a.ddelta) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) o[k] *= f;
          rms_store_as<VEC>(a.ddelta, a.delta_dtype, r * C + c, o);
        }
      }
    }
    if constexpr (PIPE) reader->next(it);
  }
  if (a.part && NV > 0) {
    if constexpr (PIPE) __syncthreads();  // the stages' memory is used again
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (c < C)
#pragma unroll
        for (int k = 0; k < VEC; ++k) dws[slot * C + c + k] = sums[i][k];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) {
      float v = 0.f;
      for (int k = 0; k < ROWS; ++k) v += dws[k * C + c];
      a.part[(int64_t)blockIdx.x * C + c] = v;
    }
  }
}

// dw[c] = sum over blocks of part[block][c], in a fixed order: 32 channels x
// 32 lanes of blocks.
__global__ void __launch_bounds__(1024) rms_dw_kernel(const float* __restrict__ part, int64_t blocks, int C,
                                                      float* __restrict__ dw) {
  __shared__ float red[32][33];
  const int x = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + x;
  float v = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int64_t b = l; b < blocks; b += 32) v += __ldg(part + b * C + c);
  }
  red[l][x] = v;
  __syncthreads();
  v = warp_sum(red[x][l]);
  if (x == 0 && blockIdx.x * 32 + l < C) dw[blockIdx.x * 32 + l] = v;
}

constexpr int PIPE_BYTES = 54 * 1024;  // of a block: four on an SM
constexpr int PIPE_MOST = 200 * 1024;  // or one, for the widest rows

// Threads that share a row, and chunks each holds (0: more than fit).  In the
// backward, which keeps four or five arrays of a row, rows of 33 to 48 chunks
// are shared by 32 threads instead of 16 (83888 x 384: fp32 138 -> 115 us,
// bf16 101 -> 92) and rows of 65 to 128 by the block instead of a warp
// (16384 x 1024: fp32 83 -> 57 us, bf16 134 -> 55).
struct RowLayout {
  int tpr, nv;
};
static RowLayout rms_layout(int64_t C, int vec, bool backward) {
  const int64_t n = (C + vec - 1) / vec;  // chunks of a row
  if (vec == 8) {
    if (n <= 8) return {8, 1};
    if (n <= 16) return {16, 1};
    if (n <= 32) return {32, 1};
    if (n <= 48 && !backward) return {16, 3};
    if (n <= 64) return {32, 2};
    if (n <= 128 && !backward) return {32, 4};
  } else {
    if (n <= 32) return {32, 1};
    if (n <= 128) return {32, 4};
  }
  return {256, n <= 256 ? 1 : n <= 512 ? 2 : n <= 1024 ? 4 : 0};
}

constexpr int RMS_BWD_BLOCKS_PER_SM = 4;
static int64_t rms_bwd_blocks(int64_t R, int64_t rows) {
  return imin64((R + rows - 1) / rows, (int64_t)sm_count() * RMS_BWD_BLOCKS_PER_SM);
}

#define RMS_LAYOUTS(VEC, L, GO)                      \
  if (VEC == 8 && L.tpr == 8) GO(8, 1)               \
  else if (VEC == 8 && L.tpr == 16 && L.nv == 1) GO(16, 1) \
  else if (VEC == 8 && L.tpr == 16) GO(16, 3)        \
  else if (L.tpr == 32 && L.nv == 1) GO(32, 1)       \
  else if (VEC == 8 && L.tpr == 32 && L.nv == 2) GO(32, 2) \
  else if (L.tpr == 32) GO(32, 4)                    \
  else if (L.nv == 1) GO(256, 1)                     \
  else if (L.nv == 2) GO(256, 2)                     \
  else if (L.nv == 4) GO(256, 4)                     \
  else GO(256, 0)

// The pipe of a kernel whose blocks of `rows` rows a round take `blocks`
// blocks: stages 0 where a block has fewer than three rounds (nothing to
// prefetch), or two stages do not fit beside a second block.
static RowPipe rms_pipe(const RowLayout& l, int64_t R, int64_t blocks, const void* a, int64_t a_bytes, const void* b,
                        int64_t b_bytes, const void* c = nullptr, int64_t c_bytes = 0, const void* d = nullptr,
                        int64_t d_bytes = 0) {
  RowPipe p{{a, b, c, d},
            {(int)a_bytes, b ? (int)b_bytes : 0, c ? (int)c_bytes : 0, d ? (int)d_bytes : 0},
            256 / l.tpr,
            0,
            0,
            failure_word()};
  if (l.nv == 0 || R < 3 * blocks * p.rows) return p;
  p.stage_bytes = p.rows * (p.row_bytes[0] + p.row_bytes[1] + p.row_bytes[2] + p.row_bytes[3]);
  p.stage_bytes = (p.stage_bytes + 127) / 128 * 128;
  p.stages = PIPE_BYTES / p.stage_bytes;
  if (p.stages > 4) p.stages = 4;
  if (p.stages < 2) p.stages = 2 * p.stage_bytes <= PIPE_MOST ? 2 : 0;
  return p;
}
static int rms_pipe_smem(const RowPipe& p) { return PIPE_HEAD + p.stages * p.stage_bytes; }
// Blocks of it that an SM holds (228 KB, 1 KB of its own and some statics a block).
static int64_t rms_pipe_blocks(const RowPipe& p) { return imin64(4, 228 * 1024 / (rms_pipe_smem(p) + 1536)); }

template <typename K, typename A>
static cudaError_t rms_go(K kernel, unsigned blocks, int smem, const A& a, const RowPipe& p, cudaStream_t st) {
  const cudaError_t e = allow_dynamic_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  kernel<<<blocks, 256, smem, st>>>(a, p);
  return cudaGetLastError();
}

template <typename TX, int VEC>
static cudaError_t rms_fwd_launch(const RmsArgs& a, cudaStream_t st) {
  const RowLayout l = rms_layout(a.C, VEC, false);
  const int64_t rows = 256 / l.tpr, rounds = (a.R + rows - 1) / rows;
  // fp32 rows keep enough bytes on the way without the pipe (16384 x 4096: 129 us, 146 with it; bf16: 121 and 90)
  RowPipe p{};
  if (VEC == 8 && sizeof(TX) == 2)
    p = rms_pipe(l, a.R, (int64_t)sm_count() * 4, a.x, a.C * (int64_t)sizeof(TX), a.delta,
                 a.C * (a.delta_dtype == AFFB_F32 ? 4 : 2));
  const unsigned blocks = (unsigned)imin64(rounds, (int64_t)sm_count() * (p.stages ? rms_pipe_blocks(p) : 8));
#define RMS_GO(TPR, NV)                                                                                          \
  {                                                                                                              \
    if constexpr (VEC == 8 && NV > 0)                                                                            \
      if (p.stages) return rms_go(rms_fwd_kernel<TX, TPR, NV, VEC, true>, blocks, rms_pipe_smem(p), a, p, st);   \
    return rms_go(rms_fwd_kernel<TX, TPR, NV, VEC, false>, blocks, 0, a, p, st);                                 \
  }
  RMS_LAYOUTS(VEC, l, RMS_GO)
#undef RMS_GO
}

template <typename TX, int VEC>
static cudaError_t rms_bwd_launch(const RmsBwdArgs& a, int64_t* part_rows, cudaStream_t st) {
  const int64_t sx = a.C * (int64_t)sizeof(TX), sy = a.C * (a.y_dtype == AFFB_F32 ? 4 : 2);
  const int64_t sd = a.C * (a.delta_dtype == AFFB_F32 ? 4 : 2);
  const RowLayout l = rms_layout(a.C, VEC, true);
  const int64_t rows = 256 / l.tpr;
  int64_t blocks = rms_bwd_blocks(a.R, rows);
  const int sums = a.part && l.nv > 0 ? (int)(rows * a.C * 4) : 0;  // at most 32 KB
  RowPipe p{};
  if (VEC == 8) p = rms_pipe(l, a.R, blocks, a.s, sx, a.dy, sy, a.ds, sx, a.delta, sd);
  if (p.stages) blocks = imin64(blocks, sm_count() * rms_pipe_blocks(p));
  *part_rows = blocks;
#define RMS_GO(TPR, NV)                                                                                         \
  {                                                                                                             \
    if constexpr (VEC == 8 && NV > 0)                                                                           \
      if (p.stages)                                                                                             \
        return rms_go(rms_bwd_kernel<TX, TPR, NV, VEC, true>, (unsigned)blocks,                                 \
                      rms_pipe_smem(p) > sums ? rms_pipe_smem(p) : sums, a, p, st);                             \
    return rms_go(rms_bwd_kernel<TX, TPR, NV, VEC, false>, (unsigned)blocks, sums, a, p, st);                   \
  }
  RMS_LAYOUTS(VEC, l, RMS_GO)
#undef RMS_GO
}
static int rms_status(cudaError_t e) {
  if (e == cudaSuccess) return AFFB_OK;
  set_error("rms_norm: launch failed: %s", cudaGetErrorString(e));
  return AFFB_ERR_CUDA;
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
  if ((rc = take_failure())) return rc;
  RmsArgs a{x, delta, delta_dtype, row_scale, row_scale ? R / groups : 1, weight, eps, R, (int)C, s, rstd, y, y_dtype,
            (uint8_t*)q, q_scale};
  const bool vec = C % 8 == 0 && rms_aligned(x) && rms_aligned(delta) && rms_aligned(weight) && rms_aligned(s) &&
                   rms_aligned(y) && ((uintptr_t)q & 7) == 0;
  cudaStream_t st = as_stream(stream);
  AFFB_DISPATCH(x_dtype, TX, return rms_status(vec ? rms_fwd_launch<TX, 8>(a, st) : rms_fwd_launch<TX, 1>(a, st)));
}

extern "C" int affb_quantize_e4m3(const void* x, int dtype, int64_t R, int64_t C, void* q, float* q_scale,
                                  void* stream) {
  int rc = rms_check(dtype, dtype, false, R, C, nullptr, 0);
  if (rc) return rc;
  if (R == 0) return AFFB_OK;
  AFFB_REQUIRE(x && q && q_scale, "quantize_e4m3: null pointer");
  if ((rc = take_failure())) return rc;
  RmsArgs a{x, nullptr, AFFB_F32, nullptr, 1, nullptr, 0.f, R, (int)C, nullptr, nullptr, nullptr, AFFB_F32, (uint8_t*)q, q_scale};
  const bool vec = C % 8 == 0 && rms_aligned(x) && ((uintptr_t)q & 7) == 0;
  cudaStream_t st = as_stream(stream);
  AFFB_DISPATCH(dtype, TX, return rms_status(vec ? rms_fwd_launch<TX, 8>(a, st) : rms_fwd_launch<TX, 1>(a, st)));
}

extern "C" int64_t affb_rms_norm_bwd_workspace_bytes(int64_t R, int64_t C) {
  if (R < 1 || C < 1) return 0;
  // sized for either row layout
  return rms_bwd_blocks(R, 1) * C * 4;
}

extern "C" int affb_rms_norm_bwd(const void* dy, int y_dtype, const void* ds, const void* s, int x_dtype,
                                 const void* delta, const float* rstd, const float* weight, const float* row_scale, int64_t groups,
                                 int64_t R, int64_t C, void* dx, void* ddelta, int delta_dtype, float* dweight,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = rms_check(x_dtype, delta_dtype, ddelta || delta, R, C, ddelta || delta ? row_scale : nullptr, groups);
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
                   rms_aligned(dx) && rms_aligned(ddelta) && rms_aligned(delta);
  AFFB_REQUIRE(!dweight || (workspace && workspace_bytes >= affb_rms_norm_bwd_workspace_bytes(R, C)),
               "rms_norm: workspace too small");
  if ((rc = take_failure())) return rc;
  int64_t blocks = 0;
  RmsBwdArgs a{dy, y_dtype, ds, s, delta, rstd, weight, row_scale, row_scale ? R / groups : 1, R, (int)C, dx, ddelta, delta_dtype,
               dweight ? (float*)workspace : nullptr};
  AFFB_DISPATCH(x_dtype, TX,
                if ((rc = rms_status(vec ? rms_bwd_launch<TX, 8>(a, &blocks, st) : rms_bwd_launch<TX, 1>(a, &blocks, st))))
                  return rc);
  if (dweight) rms_dw_kernel<<<(unsigned)((C + 31) / 32), 1024, 0, st>>>((const float*)workspace, blocks, (int)C, dweight);
  AFFB_LAUNCH_CHECK("affb_rms_norm_bwd");
  return AFFB_OK;
}
