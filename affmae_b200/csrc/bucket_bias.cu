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
// The bytes that have to move are the lists and the biases; what bounds the
// kernels is the load/store unit.  A lane takes two consecutive pairs (one
// where rows of the output are not aligned for two), so that the lists, the
// positions of a run of keys and the biases are read and written by
// neighbouring lanes, and four such steps are in flight.  The table lies in
// shared memory with four heads side by side (one access a pair and four
// heads).  Where the distances up to the last edge are few it is expanded to
// one entry per offset, so no bucket is looked up at all.
//
// Backward: bins in shared memory.  Float atomics would make the sums depend
// on timing, so a block takes 2048 pairs at a time, scales their gradients by
// a power of two of the tile's largest, adds the nearest integers (of 19
// bits), adds what that rounding leaves in units 2^20 times as fine (few
// 16-bit gradients leave anything), adds both sums to fp32 bins, and goes on
// in the same way until nothing is left of any term.  The integer sums are
// exact, so a row of the table is off by the fp32 additions of its own sums
// alone, whatever the gradients of other rows are.  The blocks' bins are
// summed in block order.
#include "common.cuh"

#include <type_traits>

namespace affb {

constexpr int BB_THREADS = 256;
constexpr int BB_STEPS = 4;          // steps of BB_THREADS * PAIRS pairs in a tile
constexpr int BB_HEADS = 4;          // heads side by side in shared memory; heads of one backward block
constexpr int BB_MAX_EDGES = 64;
constexpr int BB_LUT = 8192;         // distances answered by a byte table, else the edges are searched
constexpr int BB_BITS = 19;          // of a rounded term: 2^19 * 2048 terms stay below 2^31
// Blocks of the backward on an SM.  With 16-bit gradients the fifth costs a
// few spilled registers and hides more of the lists' latency; fp32 ones take
// twice the registers (stage 1: bf16 186 us with four, 178 with five; fp32
// 246 and 270; with three 201 and 259).
constexpr int BB_BLOCKS_PER_SM = 5, BB_BLOCKS_PER_SM_F32 = 4;
constexpr int BB_TABLE_SMEM = 64 * 1024;   // of one block's heads

struct BucketArgs {
  int edges[BB_MAX_EDGES];
  int k;                // number of edges
  int lut;              // distances up to the last edge, last + 1 (0: more than BB_LUT)
  int use_lut;          // a byte table of them is filled, else the edges are searched
  int one_sided;
  int axes;
  int per_axis;         // index values of one axis
  int rows;             // rows of the table
  int span;             // offsets of one axis up to the last edge: 2 last + 1 (one sided: last + 1)
  const void* q_pos;    // [B,Nq,axes]
  const void* k_pos;    // [B,Nk,axes]
  const int* member;    // [B,Nq,M] or null (M = Nk)
  int B, H;
  int Nk, M;
  int NM;               // pairs of one batch element in this launch (a multiple of M, below 2^31)
  int64_t batch_pairs;  // pairs of a whole batch element: stride of lists, biases and gradients
  int64_t q_batch;      // queries of a whole batch element
  uint32_t div_mul, div_shift;  // n / M for n < 2^31
};

// n / M by a multiplication.
__device__ __forceinline__ int query_of(const BucketArgs& a, int nm) {
  return (int)((__umulhi(a.div_mul, (uint32_t)nm) + (uint32_t)nm) >> a.div_shift);
}

// A NaN counts as the farthest key before the query.
__device__ __forceinline__ int offset_of(float k, float q) {
  return __float2int_rn(fminf(fmaxf(k - q, -1073741824.f), 1073741824.f));
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

// Where a kernel finds buckets: a byte table of distances, or (null) the edges.
struct Buckets {
  const uint8_t* lut;
  const int* edges;
};
// c(n) by binary search of the edges (in shared memory).
__device__ __forceinline__ int search_edges(const int* edges, int k, int n) {
  int c = 0;
#pragma unroll
  for (int s = BB_MAX_EDGES; s > 0; s >>= 1)
    if (c + s <= k && edges[c + s - 1] <= n) c += s;
  return c;
}
// Fills the edges (BB_MAX_EDGES ints at `sm`) and, after them, the byte table
// where one is wanted; ends with a barrier.
__device__ __forceinline__ Buckets fill_buckets(const BucketArgs& a, int* sm) {
  for (int i = threadIdx.x; i < a.k; i += BB_THREADS) sm[i] = a.edges[i];
  __syncthreads();
  uint8_t* lut = reinterpret_cast<uint8_t*>(sm + BB_MAX_EDGES);
  if (a.use_lut) {
    for (int i = threadIdx.x; i < a.lut; i += BB_THREADS) lut[i] = (uint8_t)search_edges(sm, a.k, i);
    __syncthreads();
  }
  return {a.use_lut ? lut : nullptr, sm};
}
__device__ __forceinline__ int axis_index(const BucketArgs& a, const Buckets& f, int d) {
  const int n = a.one_sided ? max(-d, 0) : abs(d);
  const int c = f.lut ? f.lut[min(n, a.lut - 1)] : search_edges(f.edges, a.k, n);
  return a.one_sided ? c : d < 0 ? a.k - c : a.k + c;
}
// The offset that index i of [0, span) stands for where offsets are cut off at
// the last edge.
__device__ __forceinline__ int unclipped(const BucketArgs& a, int i) { return a.one_sided ? -i : i - (a.lut - 1); }

// Index of a pair's offset along each axis, combined.  BY_OFFSET: of the
// offset cut off at the last edge, else of its bucket.
template <typename P, int AXES, bool BY_OFFSET>
struct EntryOf {
  const BucketArgs& a;
  const Buckets find;
  int last, high;       // offsets are cut off to [-last, high]
  int mx, my, add;      // entry = mx x + my y + add

  __device__ __forceinline__ EntryOf(const BucketArgs& args, const Buckets& f) : a(args), find(f) {
    last = a.lut - 1;
    high = a.one_sided ? 0 : last;
    mx = a.one_sided ? -1 : 1;
    my = AXES == 2 ? mx * a.span : 0;
    add = a.one_sided ? 0 : last * (AXES == 2 ? a.span + 1 : 1);
    if (std::is_same<P, float>::value) add = (int)((uint32_t)add - 0x4B400000u * (uint32_t)(mx + my));
  }
  // The cut-off offset; of fp32 positions plus 0x4B400000, which `add` takes
  // out again: adding 1.5 * 2^23 rounds to an integer (ties to even) in the
  // low mantissa bits.
  __device__ __forceinline__ uint32_t cut(P k, P q) const {
    if constexpr (std::is_same<P, float>::value)
      return __float_as_uint(fminf(fmaxf(k - q, (float)-last), (float)high) + 12582912.f);
    else
      return (uint32_t)max(-last, min(high, offset_of(k, q)));
  }
  __device__ __forceinline__ int one(P k, P q) const {
    if constexpr (BY_OFFSET) return (int)((uint32_t)mx * cut(k, q) + (uint32_t)add);
    return axis_index(a, find, offset_of(k, q));
  }
  __device__ __forceinline__ int two(P kx, P ky, P qx, P qy) const {
    if constexpr (BY_OFFSET)
      return (int)((uint32_t)my * cut(ky, qy) + ((uint32_t)mx * cut(kx, qx) + (uint32_t)add));
    return axis_index(a, find, offset_of(ky, qy)) * a.per_axis + axis_index(a, find, offset_of(kx, qx));
  }
};

template <typename P> struct alignas(2 * sizeof(P)) Pos2 { P x, y; };

// Entries of the pairs nm + u * STEP + j of batch element b (`none` where there
// is no such pair or the list names no key; Nk >= 1).  PAIRS == 2: nm and M
// even.  Free of branches, so that the loads of all steps are in flight
// together.
template <typename P, int AXES, int PAIRS, bool BY_OFFSET>
__device__ __forceinline__ void tile_entries(const BucketArgs& a, const EntryOf<P, AXES, BY_OFFSET>& entry, int b, int nm,
                                             int none, int (*e)[PAIRS]) {
  constexpr int STEP = BB_THREADS * PAIRS;
  using K = typename std::conditional<AXES == 2, Pos2<P>, P>::type;
  const K* qb = (const K*)a.q_pos + (int64_t)b * a.q_batch;
  const K* kb = (const K*)a.k_pos + (int64_t)b * a.Nk;
  uint32_t id[BB_STEPS][PAIRS];
  K q[BB_STEPS], k[BB_STEPS][PAIRS];
#pragma unroll
  for (int u = 0; u < BB_STEPS; ++u) {
    const bool in = nm + u * STEP < a.NM;
    const int n = in ? nm + u * STEP : 0;
    const int query = query_of(a, n);
    if (a.member) {
      const int* mp = a.member + (int64_t)b * a.batch_pairs + n;
      if constexpr (PAIRS == 2) {
        const uint2 w = __ldg(reinterpret_cast<const uint2*>(mp));
        id[u][0] = w.x;
        id[u][1] = w.y;
      } else {
        id[u][0] = (uint32_t)__ldg(mp);
      }
      if (!in) {
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) id[u][j] = ~0u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < PAIRS; ++j) id[u][j] = in ? (uint32_t)(n - query * a.M + j) : ~0u;
    }
    q[u] = qb[query];
  }
  const uint32_t top = (uint32_t)a.Nk - 1;
#pragma unroll
  for (int u = 0; u < BB_STEPS; ++u)
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) k[u][j] = kb[min(id[u][j], top)];
#pragma unroll
  for (int u = 0; u < BB_STEPS; ++u)
#pragma unroll
    for (int j = 0; j < PAIRS; ++j) {
      int v;
      if constexpr (AXES == 2) v = entry.two(k[u][j].x, k[u][j].y, q[u].x, q[u].y);
      else v = entry.one(k[u][j], q[u]);
      e[u][j] = id[u][j] <= top ? v : none;
    }
}

// Four heads of one table entry, in the output's type.
template <typename T> struct Heads4 { using type = uint2; };
template <> struct Heads4<float> { using type = float4; };
__device__ __forceinline__ uint32_t head_bits(const uint2& v, int h) {
  const uint32_t w = h < 2 ? v.x : v.y;
  return h & 1 ? w >> 16 : w & 0xffffu;
}
__device__ __forceinline__ float head_value(const float4& v, int h) {
  return h == 0 ? v.x : h == 1 ? v.y : h == 2 ? v.z : v.w;
}

// Block (x: tiles taken in turn, y: chunk of `groups` groups of four heads).
template <typename T, typename TB, typename P, int AXES, int PAIRS, bool BY_OFFSET>
__global__ void __launch_bounds__(BB_THREADS, 4)
    bucket_fwd_kernel(const __grid_constant__ BucketArgs a, const TB* __restrict__ table, int groups,
                      T* __restrict__ out) {
  using V = typename Heads4<T>::type;
  extern __shared__ unsigned char sm[];
  const int entries = BY_OFFSET ? (AXES == 2 ? a.span * a.span : a.span) : a.rows;
  V* tab = reinterpret_cast<V*>(sm);                                        // [groups][entries + 1]
  const int h0 = blockIdx.y * groups * BB_HEADS, nh = min(groups * BB_HEADS, a.H - h0);
  const Buckets find = fill_buckets(a, reinterpret_cast<int*>(sm + (size_t)groups * (entries + 1) * sizeof(V)));
  const auto fill = [&](int i, int row) {  // entry i: the heads of a table row (row < 0: zero)
    for (int g = 0; g < groups; ++g) {
      T* t = reinterpret_cast<T*>(tab + g * (entries + 1) + i);
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h)
        stf(t + h, row >= 0 && g * BB_HEADS + h < nh ? ldf(table + row * a.H + h0 + g * BB_HEADS + h) : 0.f);
    }
  };
  if (threadIdx.x == 0) fill(entries, -1);
  if (BY_OFFSET && AXES == 2) {
    // a warp takes whole rows of offsets along y
    for (int y = threadIdx.x >> 5; y < a.span; y += BB_THREADS / 32) {
      const int ry = axis_index(a, find, unclipped(a, y)) * a.per_axis;
      for (int x = threadIdx.x & 31; x < a.span; x += 32) fill(y * a.span + x, ry + axis_index(a, find, unclipped(a, x)));
    }
  } else {
    for (int i = threadIdx.x; i < entries; i += BB_THREADS) fill(i, BY_OFFSET ? axis_index(a, find, unclipped(a, i)) : i);
  }
  __syncthreads();
  constexpr int STEP = BB_THREADS * PAIRS, TILE = STEP * BB_STEPS;
  const EntryOf<P, AXES, BY_OFFSET> entry(a, find);
  const uint32_t per = ((uint32_t)a.NM + TILE - 1) / TILE;
  const int64_t total = (int64_t)per * a.B;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int b = total < (1ll << 31) ? (int)((uint32_t)t / per) : (int)(t / per);
    const int nm = (int)(t - (int64_t)b * per) * TILE + threadIdx.x * PAIRS;
    int e[BB_STEPS][PAIRS];
    tile_entries<P, AXES, PAIRS, BY_OFFSET>(a, entry, b, nm, entries, e);
    for (int g = 0; g < groups; ++g) {
      const V* tg = tab + g * (entries + 1);
      T* o = out + ((int64_t)b * a.H + h0 + g * BB_HEADS) * a.batch_pairs + nm;
      V v[BB_STEPS][PAIRS];
#pragma unroll
      for (int u = 0; u < BB_STEPS; ++u)
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) v[u][j] = tg[e[u][j]];
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h) {
        if (g * BB_HEADS + h >= nh) break;
#pragma unroll
        for (int u = 0; u < BB_STEPS; ++u) {
          if (nm + u * STEP >= a.NM) break;
          T* p = o + h * a.batch_pairs + u * STEP;
          if constexpr (sizeof(T) == 2) {
            if constexpr (PAIRS == 2)
              *reinterpret_cast<uint32_t*>(p) = head_bits(v[u][0], h) | (head_bits(v[u][1], h) << 16);
            else
              *reinterpret_cast<uint16_t*>(p) = (uint16_t)head_bits(v[u][0], h);
          } else {
            if constexpr (PAIRS == 2)
              *reinterpret_cast<float2*>(p) = make_float2(head_value(v[u][0], h), head_value(v[u][1], h));
            else
              *p = head_value(v[u][0], h);
          }
        }
      }
    }
  }
}

__device__ __forceinline__ float bb_max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

__device__ __forceinline__ float power_of_two(int t) { return __int_as_float((127 + t) << 23); }
constexpr float ROUND = 12582912.f;      // 1.5 * 2^23: a sum with it is rounded to an integer, in the low mantissa bits
constexpr int ROUND_BITS = 0x4B400000;
constexpr int NO_POWER = -1000;
// 2^t and 2^-t as products of two powers, since 2^t itself may pass fp32's range.
struct Power {
  float up, up2, down, down2;
  __device__ __forceinline__ explicit Power(int t, bool whole = false) {  // whole: |t| < 127, in one power
    const int a = whole ? t : t / 2, b = t - a;
    up = power_of_two(a);
    up2 = power_of_two(b);
    down = power_of_two(-a);
    down2 = power_of_two(-b);
  }
  // v 2^t rounded to an integer; v keeps the rest, which is exact and at most half a unit 2^-t.
  __device__ __forceinline__ int round_off(float& v) const {
    const float whole = fmaf(v * up, up2, ROUND);
    v = fmaf((whole - ROUND) * -down, down2, v);
    return __float_as_int(whole) - ROUND_BITS;
  }
  __device__ __forceinline__ float value(int n) const { return (float)n * down * down2; }
};

// A lane's gradients of one head as they were loaded.
template <typename T, int PAIRS>
struct Terms {
  static constexpr int PER = sizeof(T) == 4 ? PAIRS : 1;  // words of a step
  static constexpr int WORDS = BB_STEPS * PER;
  static __device__ __forceinline__ void load(const T* p, bool in, int u, uint32_t* w) {
    if constexpr (PER == 2) {
      const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(p)) : make_uint2(0u, 0u);
      w[2 * u] = v.x;
      w[2 * u + 1] = v.y;
    } else if constexpr (sizeof(T) * PAIRS == 4) {
      w[u] = in ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
    } else {
      w[u] = in ? __ldg(reinterpret_cast<const uint16_t*>(p)) : 0u;
    }
  }
  static __device__ __forceinline__ float get(const uint32_t* w, int j) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    const uint32_t half = PAIRS == 1 ? w[j] : j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(half << 16);
    return __half2float(__ushort_as_half((unsigned short)half));
  }
};

// Block (x: tiles taken in turn, y: group of BB_HEADS heads).
template <typename T, typename P, int AXES, int PAIRS, bool BY_OFFSET>
__global__ void __launch_bounds__(BB_THREADS, sizeof(T) == 4 ? BB_BLOCKS_PER_SM_F32 : BB_BLOCKS_PER_SM)
    bucket_bwd_kernel(const __grid_constant__ BucketArgs a, const T* __restrict__ dout, float* __restrict__ part,
                      int resume) {
  constexpr int STEP = BB_THREADS * PAIRS, TILE = STEP * BB_STEPS, PER = BB_STEPS * PAIRS;
  extern __shared__ unsigned char sm[];
  __shared__ float wmax[BB_HEADS][BB_THREADS / 32];
  const int none = a.rows;
  const int stride = a.rows + 1;  // a bin more for pairs that have no row
  float* acc = reinterpret_cast<float*>(sm);                            // [BB_HEADS][stride]
  int* bins = reinterpret_cast<int*>(acc + BB_HEADS * stride);          // [coarse, fine][BB_HEADS][stride]
  float* raw = reinterpret_cast<float*>(bins + 2 * BB_HEADS * stride);  // [TILE] values, only of an odd tile
  uint16_t* raw_row = reinterpret_cast<uint16_t*>(raw + TILE);          // [TILE]
  // BY_OFFSET: the row of every combined clipped offset, and `none` last
  const int offsets = AXES == 2 ? a.span * a.span : a.span;
  uint16_t* rows = raw_row + TILE;
  const int h0 = blockIdx.y * BB_HEADS, nh = min(BB_HEADS, a.H - h0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Buckets find = fill_buckets(a, reinterpret_cast<int*>(rows + (BY_OFFSET ? (offsets + 2) & ~1 : 0)));
  if (BY_OFFSET) {
    if (threadIdx.x == 0) rows[offsets] = (uint16_t)none;
    if (AXES == 2) {
      for (int y = threadIdx.x >> 5; y < a.span; y += BB_THREADS / 32) {
        const int ry = axis_index(a, find, unclipped(a, y)) * a.per_axis;
        for (int x = threadIdx.x & 31; x < a.span; x += 32)
          rows[y * a.span + x] = (uint16_t)(ry + axis_index(a, find, unclipped(a, x)));
      }
    } else {
      for (int i = threadIdx.x; i < offsets; i += BB_THREADS) rows[i] = (uint16_t)axis_index(a, find, unclipped(a, i));
    }
  }
  float* mine = part + ((int64_t)blockIdx.x * a.H + h0) * a.rows;
  for (int h = 0; h < BB_HEADS; ++h)
    for (int i = threadIdx.x; i < stride; i += BB_THREADS) {
      // what the launch before (of more than 2^31 pairs) has summed
      acc[h * stride + i] = resume && h < nh && i < a.rows ? mine[h * a.rows + i] : 0.f;
      bins[h * stride + i] = bins[(BB_HEADS + h) * stride + i] = 0;
    }
  __syncthreads();
  const EntryOf<P, AXES, BY_OFFSET> entry(a, find);
  const uint32_t per = ((uint32_t)a.NM + TILE - 1) / TILE;
  const int64_t total = (int64_t)per * a.B;
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int b = total < (1ll << 31) ? (int)((uint32_t)t / per) : (int)(t / per);
    const int nm = (int)(t - (int64_t)b * per) * TILE + threadIdx.x * PAIRS;
    uint32_t g[BB_HEADS][Terms<T, PAIRS>::WORDS];
    const T* p0 = dout + ((int64_t)b * a.H + h0) * a.batch_pairs + nm;
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
      if (h >= nh) break;
      const T* p = p0 + h * a.batch_pairs;
      float top = 0.f;
#pragma unroll
      for (int u = 0; u < BB_STEPS; ++u) Terms<T, PAIRS>::load(p + u * STEP, nm + u * STEP < a.NM, u, g[h]);
#pragma unroll
      for (int j = 0; j < PER; ++j) top = bb_max_nan(top, fabsf(Terms<T, PAIRS>::get(g[h], j)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = bb_max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (lane == 0) wmax[h][warp] = top;
    }
    int row[PER];
    tile_entries<P, AXES, PAIRS, BY_OFFSET>(a, entry, b, nm, BY_OFFSET ? offsets : none,
                                            reinterpret_cast<int(*)[PAIRS]>(row));
    if (BY_OFFSET) {
#pragma unroll
      for (int j = 0; j < PER; ++j) row[j] = rows[row[j]];
    }
    __syncthreads();
    int power[BB_HEADS];  // of a head's scale 2^power, NO_POWER: nothing to add
    bool odd = false;     // an infinity or NaN among the tile's gradients
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
      power[h] = NO_POWER;
      if (h >= nh) continue;
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < BB_THREADS / 32; ++w) top = bb_max_nan(top, wmax[h][w]);
      if (!isfinite(top)) odd = true;
      else if (top > 0.f) power[h] = BB_BITS - (((__float_as_int(top) >> 23) & 255) - 126);  // top < 2^e: 2^(BITS - e)
    }
    bool left = false;  // of any term after two roundings
#pragma unroll
    for (int h = 0; h < BB_HEADS; ++h) {
      if (power[h] == NO_POWER) continue;
      int* bin = bins + h * stride;
      int* fine = bin + BB_HEADS * stride;
      const bool small = power[h] > -100 && power[h] < 100;  // the scales and their inverses stay in fp32's range
      const Power one(power[h], small), two(power[h] + BB_BITS + 1, small);
      // a term of at least 2^(mantissa) units is a whole number of them
      const float whole_from = sizeof(T) == 4 ? INFINITY : (std::is_same<T, __half>::value ? 1024.f : 128.f) * one.down * one.down2;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        float v = Terms<T, PAIRS>::get(g[h], j);
        const bool rest = sizeof(T) == 4 || fabsf(v) < whole_from;
        atomicAdd(bin + row[j], one.round_off(v));
        if (rest) {
          const int n = two.round_off(v);
          if (n != 0) atomicAdd(fine + row[j], n);
          left |= v != 0.f;
        }
      }
    }
    const bool more = __syncthreads_or(left);
    for (int i = threadIdx.x; i <= a.rows; i += BB_THREADS) {
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h) {
        if (power[h] != NO_POWER) {
          int* bin = bins + h * stride + i;
          int* fine = bin + BB_HEADS * stride;
          acc[h * stride + i] += Power(power[h]).value(*bin) + Power(power[h] + BB_BITS + 1).value(*fine);
          *bin = *fine = 0;
        }
      }
    }
    if (more) {  // head by head, a lane's rests and rows in its own places of raw
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h) {
        int t = power[h];
        if (t == NO_POWER) continue;
        left = false;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          float v = Terms<T, PAIRS>::get(g[h], j);
          Power(t).round_off(v);
          Power(t + BB_BITS + 1).round_off(v);
          raw[threadIdx.x * PER + j] = v;
          raw_row[threadIdx.x * PER + j] = (uint16_t)row[j];
          left |= v != 0.f;
        }
        int* bin = bins + h * stride;
        for (t += 2 * (BB_BITS + 1); __syncthreads_or(left); t += BB_BITS + 1) {
          left = false;
          const Power unit(t);
#pragma unroll 1
          for (int j = threadIdx.x * PER; j < (int)(threadIdx.x + 1) * PER; ++j) {
            float v = raw[j];
            const int n = unit.round_off(v);
            if (n != 0) atomicAdd(bin + raw_row[j], n);
            raw[j] = v;
            left |= v != 0.f;
          }
          __syncthreads();
          for (int i = threadIdx.x; i <= a.rows; i += BB_THREADS) {
            acc[h * stride + i] += unit.value(bin[i]);
            bin[i] = 0;
          }
        }
      }
    }
    if (odd) {  // those heads: a thread per bin adds the tile's values in order
#pragma unroll
      for (int h = 0; h < BB_HEADS; ++h) {
        float top = 0.f;
        for (int w = 0; w < BB_THREADS / 32 && h < nh; ++w) top = bb_max_nan(top, wmax[h][w]);
        if (!isfinite(top)) {
          __syncthreads();
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            raw[threadIdx.x * PER + j] = Terms<T, PAIRS>::get(g[h], j);
            raw_row[threadIdx.x * PER + j] = (uint16_t)row[j];
          }
          __syncthreads();
          for (int i = threadIdx.x; i < a.rows; i += BB_THREADS)
            for (int j = 0; j < TILE; ++j)
              if (raw_row[j] == i) acc[h * stride + i] += raw[j];
        }
      }
    }
    __syncthreads();
  }
  for (int h = 0; h < nh; ++h)
    for (int i = threadIdx.x; i < a.rows; i += BB_THREADS) mine[h * a.rows + i] = acc[h * stride + i];
}

// dtable[row, h] = sum over blocks of part[block][h][row], in a fixed order:
// 32 elements x 32 lanes of blocks.
template <typename TB>
__global__ void __launch_bounds__(1024) bucket_table_kernel(const float* __restrict__ part, int64_t blocks, int rows,
                                                            int H, TB* __restrict__ dtable) {
  __shared__ float red[32][33];
  const int x = threadIdx.x & 31, l = threadIdx.x >> 5;
  const int64_t n = (int64_t)rows * H, i = (int64_t)blockIdx.x * 32 + x;
  float v = 0.f;
  if (i < n) {
#pragma unroll 8
    for (int64_t b = l; b < blocks; b += 32) v += __ldg(part + b * n + i);
  }
  red[l][x] = v;
  __syncthreads();
  v = warp_sum(red[x][l]);  // lane x holds lane-sum x of element l
  const int64_t j = (int64_t)blockIdx.x * 32 + l;
  if (x == 0 && j < n) {
    const int64_t h = j / rows, r = j - h * rows;
    stf(dtable + r * H + h, v);
  }
}

// Blocks of the backward along x, `per_sm` of them on an SM: sized for the
// narrower tile, so that it does not depend on alignment.
static int64_t bucket_bwd_blocks(int64_t B, int64_t H, int64_t NM, int per_sm) {
  const int64_t tile = BB_THREADS * BB_STEPS;
  const int64_t tiles = (NM + tile - 1) / tile * B, groups = (H + BB_HEADS - 1) / BB_HEADS;
  const int64_t want = ((int64_t)sm_count() * per_sm + groups - 1) / groups;
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
  AFFB_REQUIRE(B < (1ll << 31) && H < (1 << 18) && Nq < (1ll << 40) && Nk < (1ll << 30) && M < (1ll << 30),
               "bucket_bias: size too large");
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
  a->Nk = (int)Nk;
  a->M = (int)M;
  a->batch_pairs = Nq * M;
  a->q_batch = Nq;
  const int64_t last = edges[n_edges - 1];
  a->span = a->lut ? (int)(one_sided ? last + 1 : 2 * last + 1) : 0;
  uint32_t l = 0;
  while ((1ll << l) < M) ++l;
  a->div_shift = l;
  if (M >= 1) a->div_mul = (uint32_t)(((1ull << 32) * ((1ull << l) - (uint64_t)M)) / (uint64_t)M + 1);
  if (B * a->batch_pairs > 0 && Nk > 0) AFFB_REQUIRE(q_pos && k_pos, "bucket_bias: null positions");
  const uintptr_t pair = pos_type == AFFB_POS_I64 ? 16 : 8;
  AFFB_REQUIRE(axes == 1 || (((uintptr_t)q_pos | (uintptr_t)k_pos) & (pair - 1)) == 0,
               "bucket_bias: positions of two axes must be aligned to a pair of coordinates");
  return AFFB_OK;
}

// The launches that cover all queries, each with fewer than 2^31 pairs a batch
// element: f(arguments, first pair).
template <typename F>
static cudaError_t bb_chunks(const BucketArgs& all, int64_t pos_size, F f) {
  const int64_t most = ((1ll << 31) - 65536) / all.M;  // queries of a launch
  for (int64_t q = 0; q < all.q_batch; q += most) {
    BucketArgs a = all;
    a.NM = (int)(imin64(most, all.q_batch - q) * all.M);
    a.q_pos = (const char*)all.q_pos + q * all.axes * pos_size;
    if (a.member) a.member += q * all.M;
    const cudaError_t e = f(a, q * all.M);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// Two pairs a lane: both of one query, and 4- or 8-byte accesses aligned.
static bool bb_two(const BucketArgs& a, const void* t, int64_t size) {
  return a.M % 2 == 0 && ((uintptr_t)t & (2 * size - 1)) == 0 && ((uintptr_t)a.member & 7) == 0;
}
// Entries of a table by offset, or 0 where it is not worth expanding: it has
// to fit, and a block has to read it oftener than it writes it.
static int64_t bb_offsets(const BucketArgs& a, int64_t entry_bytes, int64_t most_bytes, int64_t blocks) {
  if (!a.span) return 0;
  const int64_t n = a.axes == 2 ? (int64_t)a.span * a.span : a.span;
  return n * entry_bytes <= most_bytes && n * blocks <= (int64_t)a.NM * a.B ? n : 0;
}

// A byte table of distances is filled where a block looks up more of them than
// that (an expanded table asks for `span` of them, or one axis's worth).
static int bb_use_lut(const BucketArgs& a, int64_t offsets, int64_t blocks) {
  if (!a.lut) return 0;
  return offsets > 0 || (int64_t)a.lut * blocks <= (int64_t)a.NM * a.B * a.axes;
}

#define BB_POS(pos_type, P, ...)                                   \
  switch (pos_type) {                                              \
    case AFFB_POS_F32: { using P = float; __VA_ARGS__; break; }    \
    case AFFB_POS_I32: { using P = int; __VA_ARGS__; break; }      \
    default: { using P = int64_t; __VA_ARGS__; break; }            \
  }

template <typename T, typename TB, typename P, int AXES, int PAIRS>
static cudaError_t bucket_fwd_launch(const BucketArgs& a, const void* table, void* out, cudaStream_t st) {
  const int64_t v = sizeof(typename Heads4<T>::type);
  const int64_t tiles = ((int64_t)a.NM + BB_THREADS * PAIRS * BB_STEPS - 1) / (BB_THREADS * PAIRS * BB_STEPS) * a.B;
  const int64_t blocks = imin64(tiles, (int64_t)sm_count() * 4);
  const int64_t all = (a.H + BB_HEADS - 1) / BB_HEADS;
  const int64_t offsets = bb_offsets(a, v, BB_TABLE_SMEM, blocks);
  const int64_t entries = (offsets ? offsets : a.rows) + 1;
  const int64_t fit = BB_TABLE_SMEM / (entries * v);
  const int groups = (int)(fit < 1 ? 1 : fit < all ? fit : all);
  BucketArgs c = a;
  c.use_lut = bb_use_lut(a, offsets, blocks);
  const int smem = (int)(groups * entries * v) + BB_MAX_EDGES * 4 + (c.use_lut ? a.lut : 0);
  auto* k = offsets ? bucket_fwd_kernel<T, TB, P, AXES, PAIRS, true> : bucket_fwd_kernel<T, TB, P, AXES, PAIRS, false>;
  const cudaError_t e = allow_dynamic_smem(k, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)blocks, (unsigned)((all + groups - 1) / groups));
  k<<<grid, BB_THREADS, smem, st>>>(c, (const TB*)table, groups, (T*)out);
  return cudaGetLastError();
}

template <typename T, typename P, int AXES, int PAIRS>
static cudaError_t bucket_bwd_launch(const BucketArgs& a, const void* dout, float* part, int64_t blocks, bool resume,
                                     cudaStream_t st) {
  const int64_t offsets = bb_offsets(a, 2, 16 * 1024, blocks);
  const int tile = BB_THREADS * PAIRS * BB_STEPS;
  BucketArgs c = a;
  c.use_lut = bb_use_lut(a, offsets, blocks);
  const int smem = 3 * BB_HEADS * (a.rows + 1) * 4 + tile * 6 + (offsets ? (int)((offsets + 2) & ~1) * 2 : 0) +
                   BB_MAX_EDGES * 4 + (c.use_lut ? a.lut : 0);
  auto* k = offsets ? bucket_bwd_kernel<T, P, AXES, PAIRS, true> : bucket_bwd_kernel<T, P, AXES, PAIRS, false>;
  const cudaError_t e = allow_dynamic_smem(k, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)blocks, (unsigned)((a.H + BB_HEADS - 1) / BB_HEADS));
  k<<<grid, BB_THREADS, smem, st>>>(c, (const T*)dout, part, resume);
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
  if (B * a.batch_pairs == 0) return AFFB_OK;
  AFFB_REQUIRE(table && out, "bucket_bias: null pointer");
  const bool two = bb_two(a, out, out_dtype == AFFB_F32 ? 4 : 2);
  cudaStream_t st = as_stream(stream);
  if (Nk == 0)  // lists that can only name keys that are not there
    return bb_status(cudaMemsetAsync(out, 0, (size_t)(B * H * a.batch_pairs * (out_dtype == AFFB_F32 ? 4 : 2)), st));
  cudaError_t e = cudaSuccess;
  AFFB_DISPATCH(table_dtype, TB, {
    AFFB_DISPATCH(out_dtype, T, {
      BB_POS(pos_type, P, {
        e = bb_chunks(a, sizeof(P), [&](const BucketArgs& c, int64_t first) {
          T* o = (T*)out + first;
          if (axes == 1) return two ? bucket_fwd_launch<T, TB, P, 1, 2>(c, table, o, st)
                                    : bucket_fwd_launch<T, TB, P, 1, 1>(c, table, o, st);
          return two ? bucket_fwd_launch<T, TB, P, 2, 2>(c, table, o, st)
                     : bucket_fwd_launch<T, TB, P, 2, 1>(c, table, o, st);
        });
      })
    })
  });
  return bb_status(e);
}

extern "C" int64_t affb_bucket_bias_bwd_workspace_bytes(int n_edges, int one_sided, int axes, int64_t B, int64_t H,
                                                        int64_t Nq, int64_t M) {
  if (B * Nq * M <= 0 || H < 1) return 0;
  const int64_t n = one_sided ? n_edges + 1 : 2 * n_edges + 1;
  return bucket_bwd_blocks(B, H, Nq * M, BB_BLOCKS_PER_SM) * H * (axes == 1 ? n : n * n) * 4;
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
  if (B * a.batch_pairs > 0 && Nk > 0) {
    AFFB_REQUIRE(dout, "bucket_bias: null pointer");
    blocks = bucket_bwd_blocks(B, H, a.batch_pairs, dout_dtype == AFFB_F32 ? BB_BLOCKS_PER_SM_F32 : BB_BLOCKS_PER_SM);
    AFFB_REQUIRE(workspace && workspace_bytes >= blocks * n * 4, "bucket_bias: workspace too small");
    const bool two = bb_two(a, dout, dout_dtype == AFFB_F32 ? 4 : 2);
    cudaError_t e = cudaSuccess;
    AFFB_DISPATCH(dout_dtype, T, {
      BB_POS(pos_type, P, {
        float* part = (float*)workspace;
        e = bb_chunks(a, sizeof(P), [&](const BucketArgs& c, int64_t first) {
          const T* g = (const T*)dout + first;
          const bool more = first > 0;
          if (axes == 1) return two ? bucket_bwd_launch<T, P, 1, 2>(c, g, part, blocks, more, st)
                                    : bucket_bwd_launch<T, P, 1, 1>(c, g, part, blocks, more, st);
          return two ? bucket_bwd_launch<T, P, 2, 2>(c, g, part, blocks, more, st)
                     : bucket_bwd_launch<T, P, 2, 1>(c, g, part, blocks, more, st);
        });
      })
    });
    if ((rc = bb_status(e))) return rc;
  }
  AFFB_DISPATCH(table_dtype, TB,
                bucket_table_kernel<TB><<<(unsigned)((n + 31) / 32), 1024, 0, st>>>((const float*)workspace, blocks,
                                                                                   a.rows, (int)H, (TB*)dtable));
  AFFB_LAUNCH_CHECK("affb_bucket_bias_bwd");
  return AFFB_OK;
}
