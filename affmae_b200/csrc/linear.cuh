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

// Type of the pre-activation sums kept for the backward: fp16 in place of bf16
// where the activation is smooth (its gradient wants absolute accuracy: with
// bf16 sums the GELU layer's dx is off by 1.45 times its own rounding, with
// fp16 ones by 1.35), the operands' own for the sign that ReLU needs.
inline int z_type(int dtype, int act) {
  return dtype == AFFB_BF16 && (act == AFFB_ACT_GELU || act == AFFB_ACT_SILU) ? AFFB_F16 : dtype;
}

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

// linear_small.cu: out = epilogue(x w^T) for few rows (at most 8), one launch.
// Against the tensor-core product (in brackets; us, weights out of DRAM), bf16:
// w [512,1024] 1 row 2.3 (7.3), 4 rows 6.6 (7.5); [4096,1024] 2 rows 6.7 (8.9),
// 4 rows 8.6 (8.9); [4096,4096] 1 row 11.5 (14.6), 2 rows 19.8 (14.8), 4 rows
// 28 (15); [16384,8192] 1 row 49 (64), 2 rows 90 (65).  e4m3: [4096,1024]
// 4 rows 6.5 (6.9); [4096,4096] 1 row 7.7 (12), 2 rows 13.4 (12); [8192,4096]
// 2 rows 14.9 (18.4), 4 rows 21.8 (18.1); [16384,8192] 1 row 29 (35), 2 rows 57
// (35).  fp32, whose operands are split for six products: 8 rows 17 (22), 19
// (30), 69 (97), 467 (605) with the same weights as bf16, 1 row 3.9 (22) to 85
// (675).
inline bool few_rows(int dtype, int64_t M, int64_t N, int64_t K) {
  if (dtype == AFFB_F32) return M <= 8;
  return M == 1 || (M <= 4 && M * N * K <= (16ll << 20));
}
int linear_small(const void* x, const void* w, int dtype, int64_t M, int64_t N, int64_t K, const LinearEpilogue& e,
                 cudaStream_t st);

// linear_aux.cu
// rows [R,C] -> [R,ld] of the same element size (the tail of a row is not written)
int linear_pack(const void* src, int64_t elem, int64_t R, int64_t C, void* dst, int64_t ld, cudaStream_t st);
// fp32 rows [R,C] -> three bf16 parts [R][ld] whose sum is the fp32 value, and
// a fourth plane: the first part, or 0 where the value is not finite; for one
// or two arrays (R = 0: none) in one launch
constexpr int SPLIT_PLANES = 4;
struct SplitRows {
  const float* src;
  int64_t R, C;
  void* dst;
  int64_t ld;
};
int linear_split(const SplitRows& a, const SplitRows& b, cudaStream_t st);
// dz = dout * act'(z): dz (null: not wanted) [R,ld] of `dtype`, or the four
// bf16 planes of it when dtype is fp32; column sums into part [strips][C] fp32
// (null: not wanted).  strips = linear_dz_strips(R, C).
int64_t linear_dz_strips(int64_t R, int64_t C);
int linear_dz(const void* dout, int dout_dtype, const void* z, int act, int dtype, int64_t R, int64_t C, void* dz,
              int64_t ld, float* part, cudaStream_t st);
// out[e] = epilogue(sum_s part[s][row][ld]) over S parts of [M,N] (row pitch ld)
int linear_sum(const float* part, int64_t S, int64_t M, int64_t N, int64_t ld, const LinearEpilogue& e,
               cudaStream_t st);

}  // namespace affb
