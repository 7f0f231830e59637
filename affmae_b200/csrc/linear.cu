// Matrix product with bias, activation and residual in its epilogue:
//   z = x w^T + b,  y = act(z) + residual,
// its backward (dx = dz w, dw = dz^T x with dz = dy act'(z)) and its form for
// e4m3 operands with one scale per row of each.
//
// One kernel computes D[m,n] = sum_k A[m,k] B[n,k] for all of them.  A and B
// are brought in by TMA as 128-byte-swizzled tiles, K-major (rows of k) or
// MN-major (rows of m or n, for the two products of the backward, which
// contract over the other index of the stored matrices), and multiplied by
// tcgen05.mma with the accumulator in tensor memory.  A block is persistent
// and split by role: one warp issues the loads, one the products, sixteen take
// the finished accumulator (two are in flight) through the epilogue into
// shared memory, from where TMA stores write it.
//
// An SM takes in about 50 bytes a cycle, so a block that multiplies 128 x 256
// tiles waits for its 48 KB of operands twice as long as the products take.
// Two blocks of a cluster therefore share a 256 x 256 tile (cta_group::2):
// each loads half of either operand, 32 KB, and keeps half of the rows.
//
// fp32 operands are split into three bf16 parts (8 mantissa bits each) and
// the six leading products of parts are summed into the same accumulator,
// smallest first; what is left out is of the order of 2^-24.  A fourth plane
// holds the first part with zeros for what is not finite: the products of an
// infinity with the other operand's small parts, of either sign or zero, would
// make NaN of it.
//
// Long contractions with few output tiles (the weight gradient sums over all
// tokens) are split over blocks; partial products go to a workspace and are
// summed in a fixed order, so results do not depend on timing.
#include "activation.cuh"
#include "linear.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace affb {

using namespace tc5;

constexpr int TILE_M = 128;
constexpr int EPI_WARPS = 16;
constexpr int LIN_THREADS = 64 + EPI_WARPS * 32;
constexpr int A_BYTES = TILE_M * 128;   // a block's rows of a tile
constexpr int SMEM_MAX = 232448;     // 227 KB of a block
constexpr int MAX_STAGES = 8;
constexpr int WARP_ROWS = 32;        // a warp's part of a tile: 32 rows x 64 columns
constexpr int WARP_COLS = 64;
constexpr int CHUNK = 32;            // worked on at a time
constexpr int BUF_BYTES = WARP_ROWS * 128;  // staged rows of 128 bytes: 64 columns of 16 bits or 32 of fp32
constexpr int BAR_BYTES = 512;
constexpr int COLS_BYTES = EPI_WARPS * 2 * WARP_COLS * 4;  // each epilogue warp's bias and column scales

struct GemmArgs {
  int M, N, bn, mt, nt, splits;
  int kblocks;       // 128-byte blocks of the contraction
  int parts;         // pairs of operand parts summed (1, or 6 for fp32)
  int stages;
  int a_mn, b_mn, f8;
  int a_blocks, b_blocks;  // MN-major: one load of that many 64-column blocks (0: a load each)
  int b_bytes;       // a block's part of B
  uint32_t idesc;    // without the width
  int direct;        // outputs not addressable by TMA: plain stores
  int res_rows;      // rows of the residual are 16-byte aligned
  int res_tma;       // the residual is brought into the second staging buffer while the products run
  int bufs;          // staging buffers of a warp: out, and z where it is wanted
  int* failed;       // the device's failure word
  LinearEpilogue e;
};

// Parts of A and B of product i of an fp32 contraction, smallest first
// (0: leading 8 bits, 1: next, 2: last, 3: leading ones of what is finite).
__device__ __forceinline__ int part_a(int i) { return (0x013123 >> (4 * i)) & 15; }
__device__ __forceinline__ int part_b(int i) { return (0x031132 >> (4 * i)) & 15; }

// The units of work of a block or pair: (split, row tile, column tile), column
// tiles fastest, every step-th.  Divides once, then steps by additions.
struct Units {
  int s, mi, ni, step_m, step_n;
  __device__ __forceinline__ Units(const GemmArgs& p, int first, int step) {
    const int tiles = p.mt * p.nt, t = first % tiles;
    s = first / tiles;
    mi = t / p.nt;
    ni = t - mi * p.nt;
    step_m = step / p.nt;
    step_n = step - step_m * p.nt;
  }
  // Columns multiplied: the last tile's are rounded up to 32 (unless B comes in
  // blocks of 64, which a narrower tile would not begin at).
  __device__ __forceinline__ int width(const GemmArgs& p) const {
    const int left = (p.N - ni * p.bn + 31) & ~31;
    return p.b_blocks || left > p.bn ? p.bn : left;
  }
  __device__ __forceinline__ bool more(const GemmArgs& p) const { return s < p.splits; }
  __device__ __forceinline__ void next(const GemmArgs& p) {
    mi += step_m;
    ni += step_n;
    if (ni >= p.nt) {
      ni -= p.nt;
      ++mi;
    }
    while (mi >= p.mt) {
      mi -= p.mt;
      ++s;
    }
  }
  __device__ __forceinline__ int first_k(int total_k, const GemmArgs& p) const {
    return p.splits == 1 ? 0 : (int)((int64_t)total_k * s / p.splits);
  }
  __device__ __forceinline__ int last_k(int total_k, const GemmArgs& p) const {
    return p.splits == 1 ? total_k : (int)((int64_t)total_k * (s + 1) / p.splits);
  }
};

// 32 columns of one row into a warp's staging buffer, in the 128-byte swizzle
// that the TMA store undoes: half 0 or 1 of a row of 16-bit values, or all of
// a row of fp32.
template <typename T>
__device__ __forceinline__ void stage_row(unsigned char* buf, int lane, int half, const float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      st8(reinterpret_cast<T*>(buf + lane * 128 + (((4 * half + j) ^ (lane & 7)) << 4)), v + 8 * j);
  }
}
// Plain accesses where TMA cannot address the rows (their pitch or start is
// not a multiple of 16 bytes): the warp goes through a staging buffer, so that
// its lanes write or read neighbouring columns of one row after the other.
template <typename T>
__device__ __forceinline__ void store_rows(unsigned char* buf, int lane, const float* v, T* p, int64_t ld, int rows,
                                           int n) {
  stage_row<T>(buf, lane, 0, v);
  __syncwarp();
  constexpr int PER = 16 / sizeof(T);
#pragma unroll 4
  for (int r = 0; r < rows; ++r)
    if (lane < n)
      p[r * ld + lane] = *reinterpret_cast<const T*>(buf + r * 128 + (((lane / PER) ^ (r & 7)) << 4) +
                                                     (lane % PER) * sizeof(T));
  __syncwarp();
}
__device__ __forceinline__ float load_float(const void* p, int dtype, int64_t i) {
  if (dtype == AFFB_F32) return ((const float*)p)[i];
  if (dtype == AFFB_BF16) return __bfloat162float(((const __nv_bfloat16*)p)[i]);
  return __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void add_rows(unsigned char* buf, int lane, float* v, const void* p, int dtype, int64_t first,
                                         int64_t ld, int rows, int n) {
#pragma unroll 4
  for (int r = 0; r < rows; ++r)
    if (lane < n)
      *reinterpret_cast<float*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) =
          load_float(p, dtype, first + r * ld + lane);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 w = *reinterpret_cast<const float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4));
    v[4 * j] += w.x;
    v[4 * j + 1] += w.y;
    v[4 * j + 2] += w.z;
    v[4 * j + 3] += w.w;
  }
  __syncwarp();
}
// stage_row's counterpart: 32 columns of a staged row added to v.
template <typename T>
__device__ __forceinline__ void add_staged(const unsigned char* buf, int lane, int half, float* v) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 w = *reinterpret_cast<const float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4));
      v[4 * j] += w.x;
      v[4 * j + 1] += w.y;
      v[4 * j + 2] += w.z;
      v[4 * j + 3] += w.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float w[8];
      ld8_shared(reinterpret_cast<const T*>(buf + lane * 128 + (((4 * half + j) ^ (lane & 7)) << 4)), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * j + i] += w[i];
    }
  }
}
// 32 columns of a row of the residual added to v, 16-byte aligned.
template <typename T>
__device__ __forceinline__ void add_row(const T* p, float* v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float r[8];
    ld8(p + 8 * j, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * j + i] += r[i];
  }
}

// One k block: four products of 32 bytes along k.
template <int CG, bool F8>
__device__ __forceinline__ void mma_block(uint32_t d, uint64_t a, uint64_t b, uint64_t sa, uint64_t sb, uint32_t idesc,
                                          bool accumulate) {
#pragma unroll
  for (int k = 0; k < 4; ++k) mma<CG, F8>(d, a + k * sa, b + k * sb, idesc, accumulate || k > 0);
}

// CG: blocks that share a tile of CG * 128 rows.
template <typename TO, int ACT, int CG>
__global__ void __launch_bounds__(LIN_THREADS, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_2,
                const __grid_constant__ GemmArgs p) {  // map_2: z, or the residual
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const int stage_bytes = A_BYTES + p.b_bytes;
  unsigned char* staging = smem + p.stages * stage_bytes;
  float* cols = reinterpret_cast<float*>(staging + EPI_WARPS * p.bufs * BUF_BYTES);
  unsigned char* bars = reinterpret_cast<unsigned char*>(cols) + COLS_BYTES;
  const uint32_t full = smem_addr(bars), empty = full + 8 * MAX_STAGES;
  const uint32_t acc_full = empty + 8 * MAX_STAGES, acc_empty = acc_full + 16, drain = acc_empty + 16;
  volatile int* failed = reinterpret_cast<volatile int*>(bars + 200);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 208);

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      bar_init(full + 8 * i, 1);
      bar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(acc_full + 8 * i, 1);
      bar_init(acc_empty + 8 * i, EPI_WARPS * CG);
    }
    bar_init(drain, 1);
    for (int i = 0; i < EPI_WARPS; ++i) bar_init(full + 256 + 8 * i, 1);
    bar_init_fence();
    *failed = 0;
    tma_prefetch(&map_a);
    tma_prefetch(&map_b);
  }
  if (warp == 1) tmem_alloc<CG>(smem_addr(tmem_slot));
  fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);

  const int total_k = p.kblocks * p.parts;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (warp == 0) {
    const bool leads = elect_one();
    const int ke = p.f8 ? 128 : 64;  // elements of one k block
    int st = 0, count = 0;
    uint32_t phase = 1;
    bool ok = true;
    const uint32_t base = smem_addr(smem);
    // both blocks' loads complete on the first block's barrier, where the products are issued
    const uint32_t full_at = CG == 2 ? peer_addr(full, 0) : full;
    for (Units u(p, first, step); u.more(p) && ok; u.next(p)) {
      const int m0 = (u.mi * CG + (int)rank) * TILE_M, n0 = u.ni * p.bn + (int)rank * (u.width(p) / CG);
      const int kb0 = u.first_k(total_k, p), kb1 = u.last_k(total_k, p);
      int part = p.parts > 1 ? kb0 / p.kblocks : 0;
      int kk = kb0 - part * p.kblocks;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = warp_wait(empty + 8 * st, phase, failed))) break;
        const int k0 = kk * ke;
        const int za = p.parts > 1 ? part_a(part) : 0, zb = p.parts > 1 ? part_b(part) : 0;
        const uint32_t bar = full_at + 8 * st, a = base + st * stage_bytes, b = a + A_BYTES;
        if (leads) {
          if (rank == 0) bar_expect(full + 8 * st, stage_bytes * CG);
          if (p.a_blocks) {
            tma_load4<CG>(a, &map_a, 0, k0, m0 >> 6, za, bar);
          } else if (p.a_mn) {
            tma_load<CG>(a, &map_a, m0, k0, za, bar);
            tma_load<CG>(a + 8192, &map_a, m0 + 64, k0, za, bar);
          } else {
            tma_load<CG>(a, &map_a, k0, m0, za, bar);
          }
          if (p.b_blocks) {
            tma_load4<CG>(b, &map_b, 0, k0, n0 >> 6, zb, bar);
          } else if (p.b_mn) {
            for (int j = 0; j * 8192 < p.b_bytes; ++j) tma_load<CG>(b + j * 8192, &map_b, n0 + 64 * j, k0, zb, bar);
          } else {
            tma_load<CG>(b, &map_b, k0, n0, zb, bar);
          }
        }
        ++count;
        if (++kk == p.kblocks) {
          kk = 0;
          ++part;
        }
        if (++st == p.stages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    if (!ok) {  // loads still in flight must land before the block's memory is given back
      if (CG == 2) settle();
      else
        for (int i = count > p.stages ? count - p.stages : 0; i < count; ++i)
          bar_drain(full + 8 * (i % p.stages), (i / p.stages) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const bool leads = elect_one();
      int st = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 1;
      bool ok = true;
      // advance of 32 bytes along k (K-major) or of 16 k rows (MN-major)
      const uint64_t sa = p.a_mn ? 2048 >> 4 : 32 >> 4, sb = p.b_mn ? 2048 >> 4 : 32 >> 4;
      const uint32_t base = smem_addr(smem);
      const uint64_t da0 = smem_desc(base, p.a_mn ? 8192 : 0, 1024);
      const uint64_t db0 = smem_desc(base + A_BYTES, p.b_mn ? 8192 : 0, 1024);
      for (Units u(p, first, step); u.more(p) && ok; u.next(p)) {
        const int n_k = u.last_k(total_k, p) - u.first_k(total_k, p);
        const uint32_t idesc = p.idesc | ((uint32_t)u.width(p) >> 3 << 17);
        if (!(ok = warp_wait(acc_empty + 8 * acc, acc_phase, failed))) break;
        fence_after();
        const uint32_t d = tmem + acc * 256;
        for (int kb = 0; kb < n_k; ++kb) {
          if (!(ok = warp_wait(full + 8 * st, phase, failed))) break;
          fence_after();
          const uint64_t off = (uint64_t)((uint32_t)(st * stage_bytes) >> 4);
          if (leads) {
            if (p.f8) mma_block<CG, true>(d, da0 + off, db0 + off, sa, sb, idesc, kb > 0);
            else mma_block<CG, false>(d, da0 + off, db0 + off, sa, sb, idesc, kb > 0);
            mma_commit<CG>(empty + 8 * st);
          }
          if (++st == p.stages) {
            st = 0;
            phase ^= 1;
          }
        }
        if (ok && leads) mma_commit<CG>(acc_full + 8 * acc);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      if (!ok) {
        if (leads) mma_commit<CG>(drain);
        bar_drain(drain, 0);
      }
    }
    __syncwarp();
  } else {
    const int ew = warp - 2, quad = warp & 3, group = ew >> 2;
    const uint32_t done_at = CG == 2 ? peer_addr(acc_empty, 0) : acc_empty;  // where the products wait
    const auto read_all = [&](int acc) {  // this warp has read its part of the accumulator
      fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 2) bar_arrive_cluster(done_at + 8 * acc);
        else bar_arrive(done_at + 8 * acc);
      }
    };
    unsigned char* buf = staging + ew * p.bufs * BUF_BYTES;
    unsigned char* zbuf = buf + BUF_BYTES;
    const uint32_t res_bar = full + 256 + 8 * ew;
    uint32_t res_phase = 0;
    const auto fetch_residual = [&](int n, int m) {  // one box: 32 rows of 128 bytes
      if (lane == 0) {
        bar_expect(res_bar, BUF_BYTES);
        tma_load<1>(smem_addr(zbuf), &map_2, n, m, 0, res_bar);
      }
    };
    float* bias = cols + ew * 2 * WARP_COLS;
    const bool per_col = p.e.bias || p.e.col_scale;
    const int z_bytes = p.e.z_dtype == AFFB_F32 ? 4 : 2;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (Units u(p, first, step); u.more(p); u.next(p)) {
      const int s = u.s, m0 = (u.mi * CG + (int)rank) * TILE_M + quad * WARP_ROWS;
      const int c0 = group * WARP_COLS, n0 = u.ni * p.bn + c0;
      const int ncols = min(min(p.bn - c0, p.N - n0), WARP_COLS);  // <= 0: nothing for this warp in a narrow tile
      const int m = m0 + lane;
      if (per_col) {
        __syncwarp();  // the tile before has been read
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = h * CHUNK + lane, n = n0 + c;
          if (c < ncols) {
            float b = 0.f;
            if (p.e.bias) {
              if (p.e.bias_dtype == AFFB_F32) b = ((const float*)p.e.bias)[n];
              else if (p.e.bias_dtype == AFFB_BF16) b = __bfloat162float(((const __nv_bfloat16*)p.e.bias)[n]);
              else b = __half2float(((const __half*)p.e.bias)[n]);
            }
            bias[c] = b;
            if (p.e.col_scale) bias[WARP_COLS + c] = p.e.col_scale[n];
          }
        }
        __syncwarp();
      }
      if (p.res_tma && ncols > 0) fetch_residual(n0, m0);
      const float rs = (p.e.row_scale && m < p.M) ? p.e.row_scale[m] : 1.f;
      // all lanes of the warp leave together
      if (!warp_wait(acc_full + 8 * acc, acc_phase, failed)) break;
      fence_after();
      if (ncols <= 0) read_all(acc);
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        const int c = h * CHUNK;
        if (c >= ncols) break;
        uint32_t r[32];
        tmem_load32(tmem + acc * 256 + c0 + c + ((uint32_t)(quad * 32) << 16), r);
        tmem_wait_load();
        if (c + CHUNK >= ncols) read_all(acc);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (p.e.col_scale) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 w = *reinterpret_cast<const float2*>(bias + WARP_COLS + c + i);
            unpack2(mul2(pack2(v[i], v[i + 1]), mul2(both(rs), pack2(w.x, w.y))), v[i], v[i + 1]);
          }
        }
        if (per_col) {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 w = *reinterpret_cast<const float4*>(bias + c + i);
            unpack2(add2(pack2(v[i], v[i + 1]), pack2(w.x, w.y)), v[i], v[i + 1]);
            unpack2(add2(pack2(v[i + 2], v[i + 3]), pack2(w.z, w.w)), v[i + 2], v[i + 3]);
          }
        }
        const int n = min(CHUNK, ncols - c);
        // first element of the warp's rows, and how many there are
        const int64_t off = ((int64_t)s * p.M + m0) * p.N + n0 + c;
        const int rows = min(WARP_ROWS, p.M - m0);
        // the buffers' last stores have been read (those of the tile before, or of fp32's first half)
        if (!p.direct && (h == 0 || sizeof(TO) == 4 || (p.e.z && z_bytes == 4))) {
          if (lane == 0) store_wait_read<0>();
          __syncwarp();
        }
        if (p.e.z) {
          if (p.direct) {
            if (p.e.z_dtype == AFFB_F32) store_rows(buf, lane, v, (float*)p.e.z + off, p.N, rows, n);
            else if (p.e.z_dtype == AFFB_BF16) store_rows(buf, lane, v, (__nv_bfloat16*)p.e.z + off, p.N, rows, n);
            else store_rows(buf, lane, v, (__half*)p.e.z + off, p.N, rows, n);
          } else {
            if (p.e.z_dtype == AFFB_F32) stage_row<float>(zbuf, lane, h, v);
            else if (p.e.z_dtype == AFFB_BF16) stage_row<__nv_bfloat16>(zbuf, lane, h, v);
            else stage_row<__half>(zbuf, lane, h, v);
          }
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) activate_pair<ACT>(v[i], v[i + 1]);
        if (p.res_tma) {
          const bool wide = p.e.residual_dtype == AFFB_F32;
          if (h == 0 || wide) {
            if (!warp_wait(res_bar, res_phase, failed)) break;
            res_phase ^= 1;
          }
          if (wide) {
            add_staged<float>(zbuf, lane, h, v);
            __syncwarp();
            if (h == 0 && CHUNK < ncols) fetch_residual(n0 + CHUNK, m0);
          } else if (p.e.residual_dtype == AFFB_BF16) {
            add_staged<__nv_bfloat16>(zbuf, lane, h, v);
          } else {
            add_staged<__half>(zbuf, lane, h, v);
          }
          if (!wide) __syncwarp();
        } else if (p.e.residual) {
          if (p.direct || !p.res_rows || n < CHUNK) {
            if (p.direct) {
              add_rows(buf, lane, v, p.e.residual, p.e.residual_dtype, off, p.N, rows, n);
            } else if (m < p.M) {
#pragma unroll
              for (int i = 0; i < CHUNK; ++i)
                if (i < n) v[i] += load_float(p.e.residual, p.e.residual_dtype, off + (int64_t)lane * p.N + i);
            }
          } else if (m < p.M) {
            const int64_t o = off + (int64_t)lane * p.N;
            if (p.e.residual_dtype == AFFB_F32) add_row((const float*)p.e.residual + o, v);
            else if (p.e.residual_dtype == AFFB_BF16) add_row((const __nv_bfloat16*)p.e.residual + o, v);
            else add_row((const __half*)p.e.residual + o, v);
          }
        }
        if (p.direct) {
          store_rows(buf, lane, v, (TO*)p.e.out + off, p.N, rows, n);
        } else {
          stage_row<TO>(buf, lane, h, v);
          const bool last = c + CHUNK >= ncols;
          const bool out_now = sizeof(TO) == 4 || last, z_now = p.e.z && (z_bytes == 4 || last);
          if (out_now || z_now) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (out_now) tma_store(&map_out, smem_addr(buf), n0 + (sizeof(TO) == 4 ? c : 0), m0, s);
              if (z_now) tma_store(&map_2, smem_addr(zbuf), n0 + (z_bytes == 4 ? c : 0), m0, s);
              store_commit();
            }
          }
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) store_wait_all();
    if (p.res_tma && *failed) settle();  // a residual on its way
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // nothing of the other block's is on its way here any more
  if (warp == 1) {
    fence_after();
    tmem_free<CG>(tmem);
  }
  if (threadIdx.x == 0 && *failed) report_failure(p.failed);
}

// ------------------------------------------------------------------ host --
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// A [planes][rows][cols] array with row pitch `ld` (elements); `blocks`: seen
// as [planes][cols / 64][rows][64], boxes of that many blocks of 64 columns.
static int make_map(CUtensorMap* map, int dtype, const void* base, int64_t cols, int64_t rows, int64_t planes,
                    int64_t ld, int box_cols, int box_rows, CUtensorMapSwizzle swizzle, int blocks = 0) {
  const CUtensorMapDataType t = dtype == AFFB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : dtype == AFFB_F16  ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                : dtype == AFFB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const int64_t es = dtype_size(dtype);
  cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes, 1};
  cuuint64_t strides[3] = {(cuuint64_t)(ld * es), (cuuint64_t)(rows * ld * es), 0};
  cuuint32_t box[4] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  if (blocks) {
    dims[0] = 64;
    dims[2] = (cuuint64_t)(cols / 64);
    dims[3] = (cuuint64_t)planes;
    strides[1] = (cuuint64_t)(64 * es);
    strides[2] = (cuuint64_t)(rows * ld * es);
    box[2] = (cuuint32_t)blocks;
  }
  EncodeFn fn = encode_fn();
  AFFB_REQUIRE(fn, "linear: the driver has no tensor-map encoder");
  const auto encode = [&] {
    return fn(map, t, blocks ? 4 : 3, const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  // a thread that has made no runtime call yet (autograd's, say) has no context; this call gives it one
  if (rc == CUDA_ERROR_INVALID_CONTEXT && cudaFree(nullptr) == cudaSuccess) rc = encode();
  AFFB_REQUIRE(rc == CUDA_SUCCESS, "linear: tensor map refused (code %d)", (int)rc);
  return AFFB_OK;
}

// One operand of a product: [planes][rows][cols], contracted over cols
// (K-major) or over rows (MN-major).
struct Operand {
  const void* p;
  int64_t rows, cols, ld;
  bool mn;
};

constexpr int PAIR_K = 6;
constexpr int WIDEST_TWO_BUFFERS = 192;

struct Shape {
  int cg, bn, nt, mt, splits;
};

// Tile and split of the contraction; `step`: multiple that the width of tiles
// beside one another has to be (what one store covers); `widest`: of a single
// block's tile (two staging buffers a warp leave no room for two stages of 256
// columns).
//
// Pairs of blocks (256-row tiles up to 256 columns wide) where there are
// enough tiles, or enough k blocks to split, for all of them, and a tile's
// contraction is long enough to be worth the pair's handshakes; else single
// blocks.  524288 rows of bf16 to 192, 384 and 768 columns, us by pairs against
// single blocks: two k blocks 105, 180, 257 (74, 116, 173); three 119, 203, 293
// (90, 146, 224); four 125, 212, 296 (100, 169, 257); five 131, 219, 291 (121,
// 199, 311); six 123, 205, 305 (122, 207, 334); eight 133, 217, 364 (152, 263,
// 405); e4m3 8192 x 4096 -> 8192, 32 blocks: 190 (215).
// Tiles that leave SMs idle are split along the contraction, at least 4 k
// blocks a part.  The width is the one that costs least, a k block of a tile
// taken as its columns and 64 more for what does not depend on them, and a
// split as SPLIT_COST for the launch that sums the parts (13107 x 771 in fp32:
// three rounds of 208 columns instead of 256, 95 -> 91 us; 5243 x 384: 63
// pairs of 128 columns instead of 42 of 192, 11.8 -> 10.9 us).
constexpr int64_t SPLIT_COST = 2000;  // about 3 us

static Shape choose_shape(int64_t M, int64_t N, int64_t total_k, int step, int widest) {
  const int64_t sms = sm_count();
  Shape s;
  const int64_t wide = (N + 255) / 256;
  const int64_t pair_tiles = (M + 255) / 256 * wide;
  const int64_t most_splits = total_k >= 8 ? total_k / 4 : 1;
  s.cg = M > TILE_M && total_k >= PAIR_K && pair_tiles * most_splits >= sms / 2 ? 2 : 1;
  const int64_t teams = sms / s.cg;
  s.mt = (int)((M + TILE_M * s.cg - 1) / (TILE_M * s.cg));
  const int64_t most_bn = s.cg == 1 ? widest : 256;
  int64_t best = 0;
  for (int64_t nt = wide; nt <= 4 * wide + 3; ++nt) {
    const int64_t per = (N + nt - 1) / nt;
    const int64_t bn = round_up(per, nt > 1 ? step : s.cg == 1 ? 16 : 32);
    if (bn > most_bn || (nt > wide && bn < 64 && best)) continue;
    const int64_t tiles = s.mt * ((N + bn - 1) / bn);
    int64_t sp = teams / tiles < most_splits ? teams / tiles : most_splits;
    if (sp < 2) sp = 1;
    for (int64_t splits = 1; splits <= sp; splits += sp > 1 ? sp - 1 : 1) {  // none, or as many as fit
      const int64_t cost = (tiles * splits + teams - 1) / teams * ((total_k + splits - 1) / splits) * (bn + 64) +
                           (splits > 1 ? SPLIT_COST : 0);
      if (best == 0 || cost < best) {
        best = cost;
        s.bn = (int)bn;
        s.nt = (int)((N + bn - 1) / bn);
        s.splits = (int)splits;
      }
    }
  }
  return s;
}
// Columns that one store of the epilogue covers: 128 bytes by TMA.
static int store_step(bool direct, int out_dtype) { return direct || out_dtype == AFFB_F32 ? 32 : 64; }

static int64_t partial_bytes(int64_t M, int64_t N, int64_t total_k) {
  int64_t most = 0;
  for (int i = 0; i < 4; ++i) {
    const Shape s = choose_shape(M, N, total_k, i & 1 ? 32 : 64, i & 2 ? 256 : WIDEST_TWO_BUFFERS);
    if (s.splits > 1) {
      const int64_t b = round_up((int64_t)s.splits * M * round_up(N, 4) * 4, 256);
      if (b > most) most = b;
    }
  }
  return most;
}

// K blocks of a contraction of length K (all part pairs).
static int64_t k_blocks(int dtype, int64_t K) {
  const int64_t ke = dtype == AFFB_E4M3 ? 128 : 64;
  return (K + ke - 1) / ke * (dtype == AFFB_F32 ? 6 : 1);
}

template <typename TO, int CG>
static const void* kernel_of(int act) {
  switch (act) {
    case AFFB_ACT_RELU: return (const void*)gemm_kernel<TO, AFFB_ACT_RELU, CG>;
    case AFFB_ACT_GELU: return (const void*)gemm_kernel<TO, AFFB_ACT_GELU, CG>;
    case AFFB_ACT_SILU: return (const void*)gemm_kernel<TO, AFFB_ACT_SILU, CG>;
    default: return (const void*)gemm_kernel<TO, AFFB_ACT_NONE, CG>;
  }
}
template <int CG>
static const void* kernel_of(int out_dtype, int act) {
  return out_dtype == AFFB_F32    ? kernel_of<float, CG>(act)
         : out_dtype == AFFB_BF16 ? kernel_of<__nv_bfloat16, CG>(act)
                                  : kernel_of<__half, CG>(act);
}

// The kernel's shared-memory limit, raised once per device (idempotent, so a
// race between threads is harmless).
static cudaError_t allow_smem(const void* k, int slot) {
  static bool done[64][24];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (dev < 64 && done[dev][slot]) return cudaSuccess;
  err = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX);
  if (err == cudaSuccess && dev < 64) done[dev][slot] = true;
  return err;
}

static bool tma_rows(const void* p, int dtype, int64_t N) {
  return aligned_to(p, 16) && N * dtype_size(dtype) % 16 == 0;
}

// D = A B^T over a contraction of length K, then the epilogue.  `dtype` names
// the operands' type as the caller has them (fp32: four bf16 planes each);
// `ws` holds partial_bytes(...).
static int gemm(int dtype, const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K, LinearEpilogue e,
                unsigned char* ws, cudaStream_t st) {
  const int64_t total_k = k_blocks(dtype, K);
  const bool plain = !(tma_rows(e.out, e.out_dtype, N) && (!e.z || tma_rows(e.z, e.z_dtype, N)));
  const bool res_rows = e.residual && tma_rows(e.residual, e.residual_dtype, N);
  const bool two_buffers = e.z || (res_rows && !plain);
  const Shape s = choose_shape(M, N, total_k, store_step(plain, e.out_dtype == AFFB_F32 && e.z ? e.z_dtype : e.out_dtype),
                               two_buffers ? WIDEST_TWO_BUFFERS : 256);
  const int et = dtype == AFFB_F32 ? AFFB_BF16 : dtype;  // element type in memory
  const int64_t planes = dtype == AFFB_F32 ? SPLIT_PLANES : 1;
  GemmArgs p{};
  p.failed = failure_word();
  AFFB_REQUIRE(p.failed, "linear: no host memory for the device's failure word");
  p.M = (int)M; p.N = (int)N;
  p.bn = s.bn; p.mt = s.mt; p.nt = s.nt; p.splits = s.splits;
  p.parts = dtype == AFFB_F32 ? 6 : 1;
  p.kblocks = (int)(total_k / p.parts);
  p.a_mn = a.mn; p.b_mn = b.mn; p.f8 = dtype == AFFB_E4M3;
  const int half_n = s.bn / s.cg;  // a block's columns of B
  p.b_bytes = b.mn ? (int)round_up(half_n, 64) * 128 : half_n * 128;
  // blocks of 64 columns in one load where no block runs past its row, and the tiles begin at a block
  p.a_blocks = a.mn && a.cols % 64 == 0 ? TILE_M / 64 : 0;
  p.b_blocks = b.mn && b.cols % 64 == 0 && half_n % 64 == 0 ? half_n / 64 : 0;
  p.idesc = instr_desc(et == AFFB_BF16 ? 1 : 0, a.mn, b.mn, (uint32_t)(TILE_M * s.cg), 0);  // n: each tile's own
  LinearEpilogue full = e;
  if (s.splits > 1) {
    e = LinearEpilogue{};
    e.out = ws;
    e.out_dtype = AFFB_F32;
    p.N = (int)round_up(N, 4);  // pitch of the partial products (columns past N hold zeros)
  }
  p.e = e;
  p.direct = s.splits > 1 ? 0 : plain;
  p.res_rows = e.residual && res_rows;  // not where partial products are written
  p.res_tma = p.res_rows && !e.z && !p.direct;
  p.bufs = e.z || p.res_tma ? 2 : 1;
  const int stage = A_BYTES + p.b_bytes;
  const int fixed = 1024 + EPI_WARPS * p.bufs * BUF_BYTES + COLS_BYTES + BAR_BYTES;
  p.stages = (SMEM_MAX - fixed) / stage;
  if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
  AFFB_REQUIRE(p.stages >= 2, "linear: no room for two stages");
  const int smem = fixed + p.stages * stage;

  CUtensorMap ma, mb, mo{}, mz{};
  const int ke = p.f8 ? 128 : 64;
  int rc;
  if ((rc = make_map(&ma, et, a.p, a.cols, a.rows, planes, a.ld, a.mn ? 64 : ke, a.mn ? 64 : TILE_M,
                     CU_TENSOR_MAP_SWIZZLE_128B, p.a_blocks)))
    return rc;
  if ((rc = make_map(&mb, et, b.p, b.cols, b.rows, planes, b.ld, b.mn ? 64 : ke, b.mn ? 64 : half_n,
                     CU_TENSOR_MAP_SWIZZLE_128B, p.b_blocks)))
    return rc;
  if (!p.direct) {
    const auto cols = [](int t) { return t == AFFB_F32 ? 32 : 64; };  // of a staged row of 128 bytes
    if ((rc = make_map(&mo, e.out_dtype, e.out, p.N, M, s.splits, p.N, cols(e.out_dtype), WARP_ROWS,
                       CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
    if (e.z && (rc = make_map(&mz, e.z_dtype, e.z, p.N, M, 1, p.N, cols(e.z_dtype), WARP_ROWS,
                              CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
    if (p.res_tma && (rc = make_map(&mz, e.residual_dtype, e.residual, p.N, M, 1, p.N, cols(e.residual_dtype), WARP_ROWS,
                                    CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
  }
  const void* k = s.cg == 2 ? kernel_of<2>(e.out_dtype, e.act) : kernel_of<1>(e.out_dtype, e.act);
  const int slot = (s.cg - 1) * 12 + (e.out_dtype == AFFB_F32 ? 0 : e.out_dtype == AFFB_BF16 ? 4 : 8) + e.act;
  cudaError_t err = allow_smem(k, slot);
  if (err == cudaSuccess) {
    const int64_t units = (int64_t)s.mt * s.nt * s.splits;
    void* args[] = {&ma, &mb, &mo, &mz, &p};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(imin64(units, sm_count() / s.cg) * s.cg));
    cfg.blockDim = dim3(LIN_THREADS);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)s.cg;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.cg == 2 ? 1 : 0;
    err = cudaLaunchKernelExC(&cfg, k, args);
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_error("linear: launch failed: %s", cudaGetErrorString(err));
    return AFFB_ERR_CUDA;
  }
  if (s.splits > 1) return linear_sum((const float*)ws, s.splits, M, N, p.N, full, st);
  return AFFB_OK;
}

// --------------------------------------------------------------- operands --
// Row pitch of an operand as the product reads it: its own when TMA can
// address it, else that of a packed copy.
static int64_t pitch(int dtype, int64_t cols) { return round_up(cols, dtype == AFFB_E4M3 ? 16 : 8); }
static bool needs_copy(int dtype, const void* p, int64_t cols) {
  return dtype == AFFB_F32 || cols % (dtype == AFFB_E4M3 ? 16 : 8) != 0 || !aligned_to(p, 16);
}
// Bytes of a value in an operand's copy.
static int64_t operand_size(int dtype) { return dtype == AFFB_F32 ? 2 * SPLIT_PLANES : dtype_size(dtype); }
// Bytes of an operand's copy where its shape (or `any`: other reasons) needs one.
static int64_t copy_bytes(int dtype, int64_t rows, int64_t cols, bool any) {
  if (!any && dtype != AFFB_F32 && cols % (dtype == AFFB_E4M3 ? 16 : 8) == 0) return 0;
  return round_up(rows * pitch(dtype, cols) * operand_size(dtype), 256);
}
struct Arena {
  unsigned char* base;
  int64_t used, size;
  void* take(int64_t bytes) {
    void* p = base + used;
    used += round_up(bytes, 256);
    return used <= size ? p : nullptr;
  }
};
// `split`: an fp32 operand's copy is left to the caller's launch.
static int make_operand(int dtype, const void* src, int64_t rows, int64_t cols, bool mn, Arena* ws, Operand* o,
                        SplitRows* split, cudaStream_t st) {
  *o = Operand{src, rows, cols, cols, mn};
  if (!needs_copy(dtype, src, cols)) return AFFB_OK;
  o->ld = pitch(dtype, cols);
  void* dst = ws->take(rows * o->ld * operand_size(dtype));
  AFFB_REQUIRE(dst, "linear: workspace too small (or an operand that is not 16-byte aligned)");
  o->p = dst;
  if (dtype != AFFB_F32) return linear_pack(src, dtype_size(dtype), rows, cols, dst, o->ld, st);
  *split = SplitRows{(const float*)src, rows, cols, dst, o->ld};
  return AFFB_OK;
}

static int check_sizes(int64_t M, int64_t N, int64_t K) {
  AFFB_REQUIRE(M >= 0 && N >= 1 && K >= 1, "linear: needs rows >= 0 and at least one input and one output channel");
  const int64_t most = (1ll << 31) - 1024;
  AFFB_REQUIRE(M < most && N < most && K < most, "linear: a dimension exceeds 2^31");
  const int64_t mt = (M + TILE_M - 1) / TILE_M, nt = (N + 31) / 32, kt = (K + TILE_M - 1) / TILE_M;
  AFFB_REQUIRE(mt * nt < most && mt * ((K + 31) / 32) < most && kt * nt < most, "linear: too many tiles");
  return AFFB_OK;
}

static int forward(const void* x, const void* w, int dtype, int64_t M, int64_t N, int64_t K, const LinearEpilogue& e,
                   void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  int rc = take_failure();
  if (rc) return rc;
  if (few_rows(dtype, M, N, K)) return linear_small(x, w, dtype, M, N, K, e, st);
  Arena ws{(unsigned char*)workspace, 0, workspace ? workspace_bytes : 0};
  Operand a, b;
  SplitRows sx{}, sw{};
  if ((rc = make_operand(dtype, x, M, K, false, &ws, &a, &sx, st))) return rc;
  if ((rc = make_operand(dtype, w, N, K, false, &ws, &b, &sw, st))) return rc;
  if ((rc = linear_split(sx, sw, st))) return rc;
  const int64_t part = partial_bytes(M, N, k_blocks(dtype, K));
  unsigned char* pp = nullptr;
  if (part) AFFB_REQUIRE(pp = (unsigned char*)ws.take(part), "linear: workspace too small");
  return gemm(dtype, a, b, M, N, K, e, pp, st);
}

}  // namespace affb

using namespace affb;

extern "C" int affb_linear_status(int* failed) {
  AFFB_REQUIRE(failed, "affb_linear_status: null pointer");
  *failed = 0;
  const cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    set_error("affb_linear_status: %s", cudaGetErrorString(e));
    return AFFB_ERR_CUDA;
  }
  *failed = take_failure() != AFFB_OK;
  return AFFB_OK;
}

// One thread waits for a barrier that nothing completes, as the products do.
__global__ void wait_probe_kernel(unsigned long long limit_ns, int* word) {
  __shared__ __align__(8) unsigned long long bar;
  __shared__ int failed;
  failed = 0;
  bar_init(smem_addr(&bar), 1);
  bar_init_fence();
  if (!bar_wait(smem_addr(&bar), 0, &failed, limit_ns)) report_failure(word);
}

extern "C" int affb_linear_wait_probe(int limit_ms, void* stream) {
  AFFB_REQUIRE(limit_ms >= 1 && limit_ms <= 2000, "affb_linear_wait_probe: a limit of 1 to 2000 ms");
  int* word = failure_word();
  AFFB_REQUIRE(word, "affb_linear_wait_probe: no host memory for the device's failure word");
  wait_probe_kernel<<<1, 1, 0, as_stream(stream)>>>(limit_ms * 1000000ull, word);
  AFFB_LAUNCH_CHECK("affb_linear_wait_probe");
  return AFFB_OK;
}

extern "C" int64_t affb_linear_fwd_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (N < 1 || K < 1 || few_rows(dtype, M, N, K)) return 0;
  return copy_bytes(dtype, M, K, false) + copy_bytes(dtype, N, K, false) + partial_bytes(M, N, k_blocks(dtype, K));
}

extern "C" int64_t affb_linear_bwd_workspace_bytes(int dtype, int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  const int64_t strips = linear_dz_strips(M, N);
  int64_t b = copy_bytes(dtype, M, N, true) + copy_bytes(dtype, N, K, false) + copy_bytes(dtype, M, K, false);
  b += round_up(strips * N * 4, 256);
  const int64_t p1 = partial_bytes(M, K, k_blocks(dtype, N)), p2 = partial_bytes(N, K, k_blocks(dtype, M));
  return b + (p1 > p2 ? p1 : p2);
}

extern "C" int affb_linear_fwd(const void* x, const void* weight, const void* bias, int bias_dtype,
                               const void* residual, int residual_dtype, int act, int dtype, int64_t M, int64_t N,
                               int64_t K, void* out, int out_dtype, void* z, void* workspace, int64_t workspace_bytes,
                               void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc) return rc;
  AFFB_REQUIRE(is_float_dtype(dtype), "linear: operands must be fp32, fp16 or bf16");
  AFFB_REQUIRE(act >= AFFB_ACT_NONE && act <= AFFB_ACT_SILU, "linear: unknown activation %d", act);
  AFFB_REQUIRE(out_dtype == dtype || out_dtype == AFFB_F32, "linear: the output is of the operands' type or fp32");
  AFFB_REQUIRE(!bias || is_float_dtype(bias_dtype), "linear: unsupported bias dtype");
  AFFB_REQUIRE(!residual || is_float_dtype(residual_dtype), "linear: unsupported residual dtype");
  if (M == 0) return AFFB_OK;
  AFFB_REQUIRE(x && weight && out, "linear: null pointer");
  AFFB_REQUIRE(workspace || affb_linear_fwd_workspace_bytes(dtype, M, N, K) == 0, "linear: workspace missing");
  LinearEpilogue e{nullptr, nullptr, bias, bias_dtype, residual, residual_dtype, act, out, out_dtype, z, z_type(dtype, act)};
  return forward(x, weight, dtype, M, N, K, e, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int64_t affb_linear_e4m3_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  return affb_linear_fwd_workspace_bytes(AFFB_E4M3, M, N, K);
}

extern "C" int affb_linear_e4m3(const void* x, const float* x_scale, const void* weight, const float* weight_scale,
                                const float* bias, const void* residual, int residual_dtype, int act, int64_t M,
                                int64_t N, int64_t K, void* out, int out_dtype, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc) return rc;
  AFFB_REQUIRE(act >= AFFB_ACT_NONE && act <= AFFB_ACT_SILU, "linear_e4m3: unknown activation %d", act);
  AFFB_REQUIRE(is_float_dtype(out_dtype), "linear_e4m3: the output must be fp32, fp16 or bf16");
  AFFB_REQUIRE(!residual || is_float_dtype(residual_dtype), "linear_e4m3: unsupported residual dtype");
  if (M == 0) return AFFB_OK;
  AFFB_REQUIRE(x && x_scale && weight && weight_scale && out, "linear_e4m3: null pointer");
  AFFB_REQUIRE(workspace || affb_linear_e4m3_workspace_bytes(M, N, K) == 0, "linear_e4m3: workspace missing");
  LinearEpilogue e{x_scale, weight_scale, bias, AFFB_F32, residual, residual_dtype, act, out, out_dtype, nullptr, 0};
  return forward(x, weight, AFFB_E4M3, M, N, K, e, workspace, workspace_bytes, as_stream(stream));
}

extern "C" int affb_linear_bwd(const void* dout, int dout_dtype, const void* z, const void* x, const void* weight,
                               int act, int dtype, int64_t M, int64_t N, int64_t K, void* dx, void* dweight,
                               void* dbias, int dbias_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_sizes(M, N, K);
  if (rc) return rc;
  AFFB_REQUIRE(is_float_dtype(dtype), "linear: operands must be fp32, fp16 or bf16");
  AFFB_REQUIRE(act >= AFFB_ACT_NONE && act <= AFFB_ACT_SILU, "linear: unknown activation %d", act);
  AFFB_REQUIRE(dout_dtype == dtype || dout_dtype == AFFB_F32, "linear: the gradient is of the operands' type or fp32");
  AFFB_REQUIRE(!dbias || is_float_dtype(dbias_dtype), "linear: unsupported bias dtype");
  cudaStream_t st = as_stream(stream);
  if (M == 0) {  // sums over no rows
    cudaError_t err = cudaSuccess;
    if (dweight) err = cudaMemsetAsync(dweight, 0, (size_t)(N * K * dtype_size(dtype)), st);
    if (dbias && err == cudaSuccess) err = cudaMemsetAsync(dbias, 0, (size_t)(N * dtype_size(dbias_dtype)), st);
    if (err != cudaSuccess) {
      set_error("linear: %s", cudaGetErrorString(err));
      return AFFB_ERR_CUDA;
    }
    return AFFB_OK;
  }
  AFFB_REQUIRE(dout && (act == AFFB_ACT_NONE || z) && (!dx || weight) && (!dweight || x), "linear: null pointer");
  AFFB_REQUIRE(workspace, "linear: workspace missing");
  if ((rc = take_failure())) return rc;
  Arena ws{(unsigned char*)workspace, 0, workspace_bytes};

  // dz: the output gradient itself when nothing changes it
  Operand dz{dout, M, N, N, false};
  const bool want_dz = dx || dweight;
  const bool as_is = act == AFFB_ACT_NONE && dout_dtype == dtype && !needs_copy(dtype, dout, N);
  void* dzp = nullptr;
  if (want_dz && !as_is) {
    dz.ld = pitch(dtype, N);
    dzp = ws.take(M * dz.ld * operand_size(dtype));
    AFFB_REQUIRE(dzp, "linear: workspace too small");
    dz.p = dzp;
  }
  float* part = nullptr;
  const int64_t strips = linear_dz_strips(M, N);
  if (dbias) AFFB_REQUIRE(part = (float*)ws.take(strips * N * 4), "linear: workspace too small");
  if (dzp || part) {
    if ((rc = linear_dz(dout, dout_dtype, z, act, dtype, M, N, dzp, dz.ld, part, st))) return rc;
  }
  if (dbias) {
    LinearEpilogue e{};
    e.out = dbias;
    e.out_dtype = dbias_dtype;
    if ((rc = linear_sum(part, strips, 1, N, N, e, st))) return rc;
  }
  LinearEpilogue e{};
  e.out_dtype = dtype;
  const int64_t p1 = dx ? partial_bytes(M, K, k_blocks(dtype, N)) : 0;
  const int64_t p2 = dweight ? partial_bytes(N, K, k_blocks(dtype, M)) : 0;
  unsigned char* pp = nullptr;
  if (p1 || p2) AFFB_REQUIRE(pp = (unsigned char*)ws.take(p1 > p2 ? p1 : p2), "linear: workspace too small");
  Operand w{}, xo{};
  SplitRows sx{}, sw{};
  if (dx && (rc = make_operand(dtype, weight, N, K, true, &ws, &w, &sw, st))) return rc;
  if (dweight && (rc = make_operand(dtype, x, M, K, true, &ws, &xo, &sx, st))) return rc;
  if ((rc = linear_split(sx, sw, st))) return rc;
  if (dx) {  // dx[m,k] = sum_n dz[m,n] w[n,k]
    dz.mn = false;
    e.out = dx;
    if ((rc = gemm(dtype, dz, w, M, K, N, e, pp, st))) return rc;
  }
  if (dweight) {  // dw[n,k] = sum_m dz[m,n] x[m,k]
    dz.mn = true;
    e.out = dweight;
    if ((rc = gemm(dtype, dz, xo, N, K, M, e, pp, st))) return rc;
  }
  return AFFB_OK;
}
