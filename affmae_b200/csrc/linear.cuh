// Matrix product with bias, activation and residual in its epilogue: the
// pieces shared by linear.cu (tensor-core product and the C entry points),
// linear_small.cu (few rows) and linear_aux.cu (operand packing, the
// activation's gradient, sums of partial results).
#pragma once

#include "common.cuh"

namespace affb {

inline int64_t dtype_size(int dtype) { return dtype == AFFB_F32 ? 4 : dtype == AFFB_E4M3 ? 1 : 2; }
inline bool is_float_dtype(int dtype) { return dtype == AFFB_F32 || dtype == AFFB_F16 || dtype == AFFB_BF16; }
inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline bool aligned_to(const void* p, int64_t a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }

// What follows the sums x . w of an output: scales (e4m3 operands), bias,
// activation, residual, and where they go.
struct LinearEpilogue {
  const float* row_scale;  // [M] or null
  const float* col_scale;  // [N] or null
  const void* bias;        // [N] or null
  int bias_dtype;
  const void* residual;    // [M,N] or null
  int residual_dtype;
  int act;                 // AFFB_ACT_*
  void* out;               // [M,N]
  int out_dtype;
  void* z;                 // [M,N] pre-activation sums, or null
  int z_dtype;
};

// linear_small.cu: out = epilogue(x w^T) for M <= small_rows(dtype) <= 8 rows,
// one launch.  K = 4096, N = 8192 against the tensor-core product: bf16 4 rows
// 22 us (28), 8 rows 37 (28); e4m3 2 rows 11.5 (16), 4 rows 17.6 (16); fp32
// (K = 1024, N = 4096) 8 rows 15 (35, six products of parts).
inline int64_t small_rows(int dtype) { return dtype == AFFB_F32 ? 8 : dtype == AFFB_E4M3 ? 3 : 4; }
int linear_small(const void* x, const void* w, int dtype, int64_t M, int64_t N, int64_t K, const LinearEpilogue& e,
                 cudaStream_t st);

// linear_aux.cu
// rows [R,C] -> [R,ld] of the same element size (the tail of a row is not written)
int linear_pack(const void* src, int64_t elem, int64_t R, int64_t C, void* dst, int64_t ld, cudaStream_t st);
// fp32 rows [R,C] -> three bf16 parts [3][R][ld] whose sum is the fp32 value
int linear_split(const float* src, int64_t R, int64_t C, void* dst, int64_t ld, cudaStream_t st);
// dz = dout * act'(z): dz (null: not wanted) [R,ld] of `dtype`, or the three
// bf16 parts of it when dtype is fp32; column sums into part [strips][C] fp32
// (null: not wanted).  strips = linear_dz_strips(R, C).
int64_t linear_dz_strips(int64_t R, int64_t C);
int linear_dz(const void* dout, int dout_dtype, const void* z, int act, int dtype, int64_t R, int64_t C, void* dz,
              int64_t ld, float* part, cudaStream_t st);
// out[e] = epilogue(sum_s part[s][row][ld]) over S parts of [M,N] (row pitch ld)
int linear_sum(const float* part, int64_t S, int64_t M, int64_t N, int64_t ld, const LinearEpilogue& e,
               cudaStream_t st);

}  // namespace affb
