// Learned relative-position bias by buckets, and the gradient of its table.
//
// With ascending edges 1 <= e_1 < ... < e_k a distance n falls into bucket
// c(n) = #{j : e_j <= n}.  Along one axis the offset d = round(kpos - qpos)
// has index k + sign(d) c(|d|) (both sides apart, 2k + 1 values) or, one
// sided, c(max(-d, 0)) (k + 1 values; keys after the query share index 0).
// Two axes (positions x, y) combine as index(y) * n + index(x).
//   bias[b,h,i,m] = table[index, h],   dtable[index, h] = sum of dbias.
// Keys are those of member_idx [B,Nq,M], or all Nk of the sequence.
//
// Forward: bound by the bytes of the lists read and the biases written; a
// thread takes eight consecutive pairs, so that every access is 16 bytes or
// more, and finds buckets by a byte table in shared memory.
//
// Backward: bins in shared memory.  Float atomics would make the sums depend
// on timing, so a block takes 2048 pairs at a time, scales their gradients by
// a power of two of the tile's largest (19 bits are kept, an error below
// 2^-20 of that largest value per term), adds them as integers, and then adds
// the tile's sums to fp32 bins.  The blocks' bins are summed in block order.
#include "common.cuh"

namespace affb {

constexpr int BB_THREADS = 256;
constexpr int BB_VEC = 8;
constexpr int BB_TILE = BB_THREADS * BB_VEC;
constexpr int BB_HEADS = 4;          // heads of one backward block
constexpr int BB_MAX_EDGES = 64;
constexpr int BB_MAX_ROWS = 4225;    // 65 x 65
constexpr int BB_LUT = 8192;         // distances answered by the byte table
constexpr int BB_BITS = 19;          // 2^19 * 2048 terms stay below 2^31
constexpr int BB_NO_ROW = 0xFFFF;
constexpr int BB_BLOCKS_PER_SM = 4;

struct BucketArgs {
  int edges[BB_MAX_EDGES];
  int k;                // number of edges
  int lut;              // entries of the byte table (last edge + 1), or 0: search the edges
  int one_sided;
  int axes;
  int per_axis;         // index values of one axis
  int rows;             // rows of the table
  const void* q_pos;    // [B,Nq,axes]
  const void* k_pos;    // [B,Nk,axes]
  const int* member;    // [B,Nq,M] or null (M = Nk)
  int B, H;
  int64_t Nq, Nk, M, NM;
};

__device__ __forceinline__ int offset_of(float k, float q) {
  const int d = __float2int_rn(k - q);  // saturates; NaN counts as 0
  return max(-(1 << 30), min(1 << 30, d));
}
__device__ __forceinline__ int offset_of(int k, int q) {
  const int64_t d = (int64_t)k - q;
  return (int)(d < -(1 << 30) ? -(1 << 30) : d > (1 << 30) ? (1 << 30) : d);
}
__device__ __forceinline__ int offset_of(int64_t k, int64_t q) {
  // the difference of two 64-bit positions may itself pass 64 bits
  if ((k < 0) != (q < 0)) {
    if (k < 0) return (uint64_t)q - (uint64_t)k > (1u << 30) ? -(1 << 30) : (int)(k - q);
    return (uint64_t)k - (uint64_t)q > (1u << 30) ? (1 << 30) : (int)(k - q);
  }
  const int64_t d = k - q;
  return (int)(d < -(1 << 30) ? -(1 << 30) : d > (1 << 30) ? (1 << 30) : d);
}

// c(n) by binary search of the edges.
__device__ __forceinline__ int search_edges(const BucketArgs& a, int n) {
  int lo = 0, hi = a.k;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.edges[mid] <= n) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ void fill_lut(const BucketArgs& a, uint8_t* lut) {
  for (int i = threadIdx.x; i < a.lut; i += BB_THREADS) lut[i] = (uint8_t)search_edges(a, i);
}
__device__ __forceinline__ int axis_index(const BucketArgs& a, const uint8_t* lut, int d) {
  const int n = a.one_sided ? max(-d, 0) : abs(d);
  const int c = a.lut ? lut[min(n, a.lut - 1)] : search_edges(a, n);
  return a.one_sided ? c : d < 0 ? a.k - c : a.k + c;
}
// Table row of the pair (query qi, key ki) of one batch element.
template <typename P>
__device__ __forceinline__ int pair_row(const BucketArgs& a, const uint8_t* lut, const P* q, const P* kp, int64_t ki) {
  if (ki < 0 || ki >= a.Nk) return BB_NO_ROW;
  if (a.axes == 1) return axis_index(a, lut, offset_of(kp[ki], q[0]));
  const P* p = kp + 2 * ki;
  return axis_index(a, lut, offset_of(p[1], q[1])) * a.per_axis + axis_index(a, lut, offset_of(p[0], q[0]));
}

// Rows of BB_VEC consecutive pairs of batch element b starting at nm.
template <typename P, bool VEC>
__device__ __forceinline__ void pair_rows(const BucketArgs& a, const uint8_t* lut, int b, int64_t nm, int* row) {
  const P* qb = (const P*)a.q_pos + (int64_t)b * a.Nq * a.axes;
  const P* kb = (const P*)a.k_pos + (int64_t)b * a.Nk * a.axes;
  if constexpr (VEC) {  // M % 8 == 0: one query
    const int64_t i = nm / a.M, m = nm - i * a.M;
    const P* q = qb + i * a.axes;
    if (a.member) {
      const int4* mp = reinterpret_cast<const int4*>(a.member + (int64_t)b * a.NM + nm);
      const int4 u = __ldg(mp), v = __ldg(mp + 1);
      const int id[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < BB_VEC; ++j) row[j] = pair_row(a, lut, q, kb, (int64_t)id[j]);
    } else {
#pragma unroll
      for (int j = 0; j < BB_VEC; ++j) row[j] = pair_row(a, lut, q, kb, m + j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < BB_VEC; ++j) {
      row[j] = BB_NO_ROW;
      if (nm + j < a.NM) {
        const int64_t i = (nm + j) / a.M, m = nm + j - i * a.M;
        const int64_t ki = a.member ? (int64_t)a.member[(int64_t)b * a.NM + nm + j] : m;
        row[j] = pair_row(a, lut, qb + i * a.axes, kb, ki);
      }
    }
  }
}

template <typename T, typename TB, typename P, bool VEC>
__global__ void __launch_bounds__(BB_THREADS) bucket_fwd_kernel(const __grid_constant__ BucketArgs a,
                                                                const TB* __restrict__ table, int in_smem,
                                                                T* __restrict__ out) {
  extern __shared__ unsigned char sm[];
  uint8_t* lut = sm;
  float* tab = reinterpret_cast<float*>(sm + BB_LUT);  // [H][rows]
  fill_lut(a, lut);
  if (in_smem)
    for (int i = threadIdx.x; i < a.rows * a.H; i += BB_THREADS) tab[(i % a.H) * a.rows + i / a.H] = ldf(table + i);
  __syncthreads();
  const int64_t per = (a.NM + BB_VEC - 1) / BB_VEC, total = per * a.B;
  for (int64_t v = (int64_t)blockIdx.x * BB_THREADS + threadIdx.x; v < total; v += (int64_t)gridDim.x * BB_THREADS) {
    const int b = (int)(v / per);
    const int64_t nm = (v - b * per) * BB_VEC;
    int row[BB_VEC];
    pair_rows<P, VEC>(a, lut, b, nm, row);
    for (int h = 0; h < a.H; ++h) {
      float o[BB_VEC];
#pragma unroll
      for (int j = 0; j < BB_VEC; ++j) {
        if (row[j] == BB_NO_ROW) o[j] = 0.f;
        else o[j] = in_smem ? tab[h * a.rows + row[j]] : ldf(table + (int64_t)row[j] * a.H + h);
      }
      T* p = out + ((int64_t)b * a.H + h) * a.NM + nm;
      if constexpr (VEC) {
        st8(p, o);
      } else {
#pragma unroll
        for (int j = 0; j < BB_VEC; ++j)
          if (nm + j < a.NM) stf(p + j, o[j]);
      }
    }
  }
}

__device__ __forceinline__ float bb_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Block (x: tiles taken in turn, y: group of BB_HEADS heads).
template <typename T, typename P, bool VEC>
__global__ void __launch_bounds__(BB_THREADS) bucket_bwd_kernel(const __grid_constant__ BucketArgs a,
                                                                const T* __restrict__ dout,
                                                                float* __restrict__ part) {
  extern __shared__ unsigned char sm[];
  __shared__ float wmax[BB_HEADS][BB_THREADS / 32];
  __shared__ float raw[BB_TILE];
  __shared__ uint16_t raw_row[BB_TILE];
  uint8_t* lut = sm;
  float* acc = reinterpret_cast<float*>(sm + BB_LUT);                   // [BB_HEADS][rows]
  int* bins = reinterpret_cast<int*>(acc + BB_HEADS * a.rows);          // [BB_HEADS][rows]
  const int h0 = blockIdx.y * BB_HEADS, nh = min(BB_HEADS, a.H - h0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  fill_lut(a, lut);
  for (int i = threadIdx.x; i < BB_HEADS * a.rows; i += BB_THREADS) {
    acc[i] = 0.f;
    bins[i] = 0;
  }
  __syncthreads();
  const int64_t per = (a.NM + BB_TILE - 1) / BB_TILE, total = per * a.B;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int b = (int)(t / per);
    const int64_t nm = (t - b * per) * BB_TILE + threadIdx.x * BB_VEC;
    const bool in = nm < a.NM;
    int row[BB_VEC];
#pragma unroll
    for (int j = 0; j < BB_VEC; ++j) row[j] = BB_NO_ROW;
    if (in) pair_rows<P, VEC>(a, lut, b, nm, row);
    float g[BB_HEADS][BB_VEC];
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
#pragma unroll
      for (int j = 0; j < BB_VEC; ++j) g[h][j] = 0.f;
      if (in && h < nh) {
        const T* p = dout + ((int64_t)b * a.H + h0 + h) * a.NM + nm;
        if constexpr (VEC) {
          ld8(p, g[h]);
        } else {
#pragma unroll
          for (int j = 0; j < BB_VEC; ++j)
            if (nm + j < a.NM) g[h][j] = ldf(p + j);
        }
      }
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < BB_VEC; ++j)
        if (row[j] != BB_NO_ROW) top = bb_max_nan(top, fabsf(g[h][j]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = bb_max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) wmax[h][warp] = top;
    }
    __syncthreads();
    float down[BB_HEADS];  // 2^-(t / 2) of the scale 2^t, 0: nothing to add
    float rest[BB_HEADS];  // 2^-(t - t / 2)
    bool odd = false;      // an infinity or NaN among the tile's gradients
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < BB_THREADS / 32; ++w) top = bb_max_nan(top, wmax[h][w]);
      down[h] = 0.f;
      if (!isfinite(top)) {
        odd = true;
      } else if (top > 0.f) {
        // top < 2^e: values times 2^(BITS - e) stay below 2^BITS.  The power is
        // applied in two halves, as it may itself pass the range of fp32.
        const int t = BB_BITS - (((__float_as_int(top) >> 23) & 255) - 126), t1 = t / 2;
        const float up = __int_as_float((127 + t1) << 23), up2 = __int_as_float((127 + t - t1) << 23);
        down[h] = __int_as_float((127 - t1) << 23);
        rest[h] = __int_as_float((127 - t + t1) << 23);
#pragma unroll
        for (int j = 0; j < BB_VEC; ++j)
          if (row[j] != BB_NO_ROW) atomicAdd(bins + h * a.rows + row[j], __float2int_rn(g[h][j] * up * up2));
      }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
      if (down[h] != 0.f) {
        for (int i = threadIdx.x; i < a.rows; i += BB_THREADS) {
          const int s = bins[h * a.rows + i];
          if (s != 0) {
            acc[h * a.rows + i] += (float)s * down[h] * rest[h];
            bins[h * a.rows + i] = 0;
          }
        }
      }
    }
    if (odd) {  // those heads: a thread per bin adds the tile's values in order
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h) {
        float top = 0.f;
        for (int w = 0; w < BB_THREADS / 32; ++w) top = bb_max_nan(top, wmax[h][w]);
        if (!isfinite(top)) {
          __syncthreads();
#pragma unroll
          for (int j = 0; j < BB_VEC; ++j) {
            raw[threadIdx.x * BB_VEC + j] = g[h][j];
            raw_row[threadIdx.x * BB_VEC + j] = (uint16_t)row[j];
          }
          __syncthreads();
          for (int i = threadIdx.x; i < a.rows; i += BB_THREADS)
            for (int j = 0; j < BB_TILE; ++j)
              if (raw_row[j] == i) acc[h * a.rows + i] += raw[j];
        }
      }
    }
    __syncthreads();
  }
  float* o = part + ((int64_t)blockIdx.x * a.H + h0) * a.rows;
  for (int i = threadIdx.x; i < nh * a.rows; i += BB_THREADS) o[i] = acc[i];
}

// dtable[row, h] = sum over blocks of part[block][h][row], in block order.
template <typename TB>
__global__ void __launch_bounds__(256) bucket_table_kernel(const float* __restrict__ part, int64_t blocks, int rows,
                                                           int H, TB* __restrict__ dtable) {
  __shared__ float red[8][33];
  const int x = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int64_t n = (int64_t)rows * H, i = (int64_t)blockIdx.x * 32 + x;
  float v = 0.f;
  if (i < n) {
#pragma unroll 4
    for (int64_t b = l; b < blocks; b += 8) v += part[b * n + i];
  }
  red[l][x] = v;
  __syncthreads();
  if (l == 0 && i < n) {
    v = 0.f;
    for (int k = 0; k < 8; ++k) v += red[k][x];
    const int64_t h = i / rows, r = i - h * rows;
    stf(dtable + r * H + h, v);
  }
}

static int64_t bucket_bwd_blocks(int64_t B, int64_t H, int64_t NM) {
  const int64_t tiles = (NM + BB_TILE - 1) / BB_TILE * B, groups = (H + BB_HEADS - 1) / BB_HEADS;
  const int64_t want = ((int64_t)sm_count() * BB_BLOCKS_PER_SM + groups - 1) / groups;
  return tiles < want ? tiles : want;
}

static int bucket_args(const int32_t* edges, int n_edges, int one_sided, const void* q_pos, const void* k_pos,
                       int pos_type, int axes, const int32_t* member, int64_t B, int64_t H, int64_t Nq, int64_t Nk,
                       int64_t M, BucketArgs* a) {
  AFFB_REQUIRE(axes == 1 || axes == 2, "bucket_bias: positions have 1 or 2 axes");
  AFFB_REQUIRE(edges && n_edges >= 1 && n_edges <= (axes == 1 ? BB_MAX_EDGES : 32),
               "bucket_bias: needs 1 to 64 edges (32 with two axes)");
  for (int i = 0; i < n_edges; ++i) {
    AFFB_REQUIRE(edges[i] >= 1 && edges[i] <= (1 << 30) && (i == 0 || edges[i] > edges[i - 1]),
                 "bucket_bias: edges must ascend within [1, 2^30]");
    a->edges[i] = edges[i];
  }
  AFFB_REQUIRE(pos_type >= AFFB_POS_F32 && pos_type <= AFFB_POS_I64, "bucket_bias: unknown position type");
  AFFB_REQUIRE(B >= 0 && H >= 1 && Nq >= 0 && Nk >= 0 && M >= 0, "bucket_bias: negative size or no head");
  AFFB_REQUIRE(member || M == Nk || B * Nq * M == 0, "bucket_bias: without member_idx every key is taken (M = Nk)");
  AFFB_REQUIRE(B < (1ll << 31) && H < (1 << 18) && Nq < (1ll << 40) && Nk < (1ll << 40), "bucket_bias: size too large");
  a->k = n_edges;
  a->lut = edges[n_edges - 1] < BB_LUT ? edges[n_edges - 1] + 1 : 0;
  a->one_sided = one_sided != 0;
  a->axes = axes;
  a->per_axis = one_sided ? n_edges + 1 : 2 * n_edges + 1;
  a->rows = axes == 1 ? a->per_axis : a->per_axis * a->per_axis;
  a->q_pos = q_pos;
  a->k_pos = k_pos;
  a->member = member;
  a->B = (int)B;
  a->H = (int)H;
  a->Nq = Nq;
  a->Nk = Nk;
  a->M = M;
  a->NM = Nq * M;
  if (B * a->NM > 0) AFFB_REQUIRE(q_pos && k_pos, "bucket_bias: null positions");
  return AFFB_OK;
}

static bool bb_vec(const BucketArgs& a, const void* t) {
  return a.M % BB_VEC == 0 && ((uintptr_t)t & 15) == 0 && ((uintptr_t)a.member & 15) == 0;
}

#define BB_POS(pos_type, P, ...)                                   \
  switch (pos_type) {                                              \
    case AFFB_POS_F32: { using P = float; __VA_ARGS__; break; }    \
    case AFFB_POS_I32: { using P = int; __VA_ARGS__; break; }      \
    default: { using P = int64_t; __VA_ARGS__; break; }            \
  }

constexpr int BB_TABLE_SMEM = 96 * 1024;  // larger tables are read through L1 instead

template <typename T, typename TB, typename P, bool VEC>
static cudaError_t bucket_fwd_launch(const BucketArgs& a, const void* table, void* out, cudaStream_t st) {
  const int64_t bytes = (int64_t)a.rows * a.H * 4;
  const int in_smem = bytes <= BB_TABLE_SMEM;
  const int smem = BB_LUT + (in_smem ? (int)bytes : 0);
  auto* k = bucket_fwd_kernel<T, TB, P, VEC>;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, BB_LUT + BB_TABLE_SMEM);
    if (e != cudaSuccess) return e;
  }
  const int64_t threads = (a.NM + BB_VEC - 1) / BB_VEC * a.B;
  const unsigned blocks = (unsigned)imin64((threads + BB_THREADS - 1) / BB_THREADS, (int64_t)sm_count() * 8);
  k<<<blocks, BB_THREADS, smem, st>>>(a, (const TB*)table, in_smem, (T*)out);
  return cudaGetLastError();
}

template <typename T, typename P, bool VEC>
static cudaError_t bucket_bwd_launch(const BucketArgs& a, const void* dout, float* part, int64_t blocks,
                                     cudaStream_t st) {
  const int smem = BB_LUT + 2 * BB_HEADS * a.rows * 4;
  auto* k = bucket_bwd_kernel<T, P, VEC>;
  if (smem > 32 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid((unsigned)blocks, (unsigned)((a.H + BB_HEADS - 1) / BB_HEADS));
  k<<<grid, BB_THREADS, smem, st>>>(a, (const T*)dout, part);
  return cudaGetLastError();
}

static int bb_status(cudaError_t e) {
  if (e == cudaSuccess) return AFFB_OK;
  set_error("bucket_bias: launch failed: %s", cudaGetErrorString(e));
  return AFFB_ERR_CUDA;
}

}  // namespace affb

using namespace affb;

extern "C" int affb_bucket_bias_fwd(const void* table, int table_dtype, const int32_t* edges, int n_edges,
                                    int one_sided, const void* q_pos, const void* k_pos, int pos_type, int axes,
                                    const int32_t* member_idx, int64_t B, int64_t H, int64_t Nq, int64_t Nk, int64_t M,
                                    void* out, int out_dtype, void* stream) {
  BucketArgs a{};
  int rc = bucket_args(edges, n_edges, one_sided, q_pos, k_pos, pos_type, axes, member_idx, B, H, Nq, Nk, M, &a);
  if (rc) return rc;
  AFFB_REQUIRE(out_dtype == AFFB_F32 || out_dtype == AFFB_F16 || out_dtype == AFFB_BF16,
               "bucket_bias: the output must be fp32, fp16 or bf16");
  if (B * a.NM == 0) return AFFB_OK;
  AFFB_REQUIRE(table && out, "bucket_bias: null pointer");
  const bool vec = bb_vec(a, out);
  cudaStream_t st = as_stream(stream);
  cudaError_t e = cudaSuccess;
  AFFB_DISPATCH(table_dtype, TB, {
    AFFB_DISPATCH(out_dtype, T, {
      BB_POS(pos_type, P, {
        if (vec) e = bucket_fwd_launch<T, TB, P, true>(a, table, out, st);
        else e = bucket_fwd_launch<T, TB, P, false>(a, table, out, st);
      })
    })
  });
  return bb_status(e);
}

extern "C" int64_t affb_bucket_bias_bwd_workspace_bytes(int n_edges, int one_sided, int axes, int64_t B, int64_t H,
                                                        int64_t Nq, int64_t M) {
  if (B * Nq * M <= 0 || H < 1) return 0;
  const int64_t n = one_sided ? n_edges + 1 : 2 * n_edges + 1;
  return bucket_bwd_blocks(B, H, Nq * M) * H * (axes == 1 ? n : n * n) * 4;
}

extern "C" int affb_bucket_bias_bwd(const void* dout, int dout_dtype, const int32_t* edges, int n_edges, int one_sided,
                                    const void* q_pos, const void* k_pos, int pos_type, int axes,
                                    const int32_t* member_idx, int64_t B, int64_t H, int64_t Nq, int64_t Nk, int64_t M,
                                    void* dtable, int table_dtype, void* workspace, int64_t workspace_bytes,
                                    void* stream) {
  BucketArgs a{};
  int rc = bucket_args(edges, n_edges, one_sided, q_pos, k_pos, pos_type, axes, member_idx, B, H, Nq, Nk, M, &a);
  if (rc) return rc;
  AFFB_REQUIRE(dout_dtype == AFFB_F32 || dout_dtype == AFFB_F16 || dout_dtype == AFFB_BF16,
               "bucket_bias: the gradient must be fp32, fp16 or bf16");
  AFFB_REQUIRE(dtable, "bucket_bias: null pointer");
  cudaStream_t st = as_stream(stream);
  const int64_t n = (int64_t)a.rows * H;
  int64_t blocks = 0;
  if (B * a.NM > 0) {
    AFFB_REQUIRE(dout, "bucket_bias: null pointer");
    blocks = bucket_bwd_blocks(B, H, a.NM);
    AFFB_REQUIRE(workspace && workspace_bytes >= blocks * n * 4, "bucket_bias: workspace too small");
    const bool vec = bb_vec(a, dout);
    cudaError_t e = cudaSuccess;
    AFFB_DISPATCH(dout_dtype, T, {
      BB_POS(pos_type, P, {
        if (vec) e = bucket_bwd_launch<T, P, true>(a, dout, (float*)workspace, blocks, st);
        else e = bucket_bwd_launch<T, P, false>(a, dout, (float*)workspace, blocks, st);
      })
    });
    if ((rc = bb_status(e))) return rc;
  }
  AFFB_DISPATCH(table_dtype, TB,
                bucket_table_kernel<TB><<<(unsigned)((n + 31) / 32), 256, 0, st>>>((const float*)workspace, blocks,
                                                                                   a.rows, (int)H, (TB*)dtable));
  AFFB_LAUNCH_CHECK("affb_bucket_bias_bwd");
  return AFFB_OK;
}
