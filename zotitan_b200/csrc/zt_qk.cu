// RMS norm of every query and key head with the rotary embedding in the same pass, forward
// and backward. For a head x of hd elements (h = hd / 2), weight w and the position's cos, sin:
//
//   n = 1 / sqrt(mean(x^2) + eps),  y = w * x * n
//   out[i]     = y[i] cos[i] - y[i + h] sin[i]
//   out[i + h] = y[i + h] cos[i + h] + y[i] sin[i + h]
//
// and with g the gradient of out:
//
//   dy[i] = g[i] cos[i] + g[i + h] sin[i + h],  dy[i + h] = g[i + h] cos[i + h] - g[i] sin[i]
//   dw[i] = sum over positions and heads of dy[i] x[i] n
//   dx    = n w dy - x n^3 mean(w dy x)
//
// All of it in fp32 with one rounding at the store. Bandwidth is the bound: the forward
// reads and writes each head once, the backward reads x and g and writes dx. A lane owns
// the same 16 bytes of both halves of a head, so the rotation's partner is in its own
// registers; the lanes of a head (8 of a warp for bf16 heads of 128) share the sum of
// squares by shuffles. A warp walks the heads of one position, whose cos and sin it loads
// once and keeps packed in registers.
#include <math.h>

#include <mutex>

#include "zt_common.cuh"

namespace {

constexpr int kWarps = 4;          // warps of a forward block; they share nothing
constexpr int kBwdWarps = 8;       // warps of a backward block; they share the weight gradient's sum
constexpr int kBwdBlocks = 2;      // of them on an SM
// Ring kernels: blocks on an SM and the steps a warp has in flight. 32768 positions of 40 x 128 bf16
// forward take 140 us with two blocks, 110 with three, 123 with four, 126 with five (more rows under
// way at a time cost DRAM more than they hide); the backward of 8192 takes 54 us with two steps,
// 57 with four.
constexpr int kFwdBlocks = 3;
constexpr int kFwdRing = 8;
constexpr int kBwdRing = 2;
constexpr int kMaxHeadDim = 512;   // 32 lanes x 8 elements of each half
constexpr int kE = 8;              // elements of each half that a lane holds at most

struct QkParams {
  const void* x[2];    // q, k heads
  const void* g[2];    // gradients of the outputs (backward)
  void* out[2];        // rotated heads, or the gradients of q and k
  const void* w[2];
  const void* cos;
  const void* sin;
  float* partial;      // [blocks][2][hd] weight gradients of a block (backward)
  int64_t xs[2][3];    // element strides over batch, position, head
  int64_t gs[2][3];
  int64_t os[2][3];
  int32_t heads[2];
  int32_t groups[2];   // steps of a warp over the heads: ceil(heads / heads per warp)
  int32_t rows, seq, hd, half;
  int32_t lanes;       // lanes of one head, a power of two
  int32_t split;       // warps that share one position's heads
  int32_t per_batch;   // cos / sin rows: batch * seq instead of seq
  int32_t w_dtype, t_dtype;
  float eps, inv_hd;
};

template <int DT> struct El;
template <> struct El<ZT_F32> {
  using T = float;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct El<ZT_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from(float v) { return __float2bfloat16_rn(v); }
};
template <> struct El<ZT_F16> {
  using T = __half;
  static __device__ __forceinline__ float to(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from(float v) { return __float2half_rn(v); }
};

// A lane's share of one half of a head: NC chunks of V consecutive elements, chunk c at
// (c * lanes + lane) * V, kept as loaded.
template <int DT, int V, int NC> struct Piece {
  using T = typename El<DT>::T;
  static constexpr int kWords = V * (int)sizeof(T) >= 4 ? V * (int)sizeof(T) / 4 : 1;
  uint32_t w[NC][kWords];

  __device__ __forceinline__ void load(const T* p, int sub, int lanes, int half) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = (c * lanes + sub) * V;
#pragma unroll
      for (int j = 0; j < kWords; ++j) w[c][j] = 0;
      if (i < half) {
        if constexpr (V * sizeof(T) == 16) {
          const uint4 u = *reinterpret_cast<const uint4*>(p + i);
          w[c][0] = u.x; w[c][1] = u.y; w[c][2] = u.z; w[c][3] = u.w;
        } else if constexpr (sizeof(T) == 2) {
          w[c][0] = *reinterpret_cast<const uint16_t*>(p + i);
        } else {
          w[c][0] = *reinterpret_cast<const uint32_t*>(p + i);
        }
      }
    }
  }
  __device__ __forceinline__ void take(const uint4& u) {
    w[0][0] = u.x; w[0][1] = u.y; w[0][2] = u.z; w[0][3] = u.w;
  }
  __device__ __forceinline__ float at(int c, int j) const {
    if constexpr (DT == ZT_F32) {
      return __uint_as_float(w[c][j]);
    } else if constexpr (DT == ZT_BF16) {
      return (j & 1) ? __uint_as_float(w[c][j >> 1] & 0xffff0000u) : __uint_as_float(w[c][j >> 1] << 16);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[c][j >> 1]);
      return (j & 1) ? __high2float(h) : __low2float(h);
    }
  }
};

template <int DT, int V, int NC>
__device__ __forceinline__ void store_piece(typename El<DT>::T* p, const float (&v)[NC][V], int sub, int lanes, int half) {
  using T = typename El<DT>::T;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * lanes + sub) * V;
    if (i >= half) continue;
    if constexpr (V == 4 && DT == ZT_F32) {
      *reinterpret_cast<float4*>(p + i) = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
    } else if constexpr (V == 8) {
      uint32_t r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DT == ZT_BF16) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[c][2 * j], v[c][2 * j + 1]);
          r[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __half2 h = __floats2half2_rn(v[c][2 * j], v[c][2 * j + 1]);
          r[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<uint4*>(p + i) = make_uint4(r[0], r[1], r[2], r[3]);
    } else {
      p[i] = El<DT>::from(v[c][0]);
    }
  }
}

// A lane's V elements of a weight or table row, of the heads' type or fp32, as fp32.
template <int DT, int V, int NC>
__device__ __forceinline__ void load_side(float (&v)[NC][V], const void* base, int64_t off, int32_t dtype, int sub, int lanes,
                                          int half) {
  using T = typename El<DT>::T;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int i = (c * lanes + sub) * V;
#pragma unroll
    for (int j = 0; j < V; ++j) v[c][j] = 0.f;
    if (i >= half) continue;
    if (DT != ZT_F32 && dtype == ZT_F32) {
      const float* p = static_cast<const float*>(base) + off + i;
      if constexpr (V % 4 == 0) {
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          const float4 u = *reinterpret_cast<const float4*>(p + q);
          v[c][q] = u.x; v[c][q + 1] = u.y; v[c][q + 2] = u.z; v[c][q + 3] = u.w;
        }
      } else {
        v[c][0] = *p;
      }
    } else {
      Piece<DT, V, 1> u;
      u.load(static_cast<const T*>(base) + off + i, 0, 1, V);
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = u.at(0, j);
    }
  }
}

// Sum over the lanes of a head; LANES = 0: known at run time only.
template <int LANES> __device__ __forceinline__ float lanes_sum(float v, int lanes) {
  if constexpr (LANES > 0) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  } else {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  return v;
}

// A warp's part of the groups [0, groups) of q or k, whose first lies `before` groups into
// the position's: those congruent to `part` modulo `split`.
__device__ __forceinline__ int first_of(int before, int part, int split) {
  return part >= before ? part - before : (split - (before - part) % split) % split;
}

// ---- the plain kernels: single elements -------------------------------------------------------
//
// One warp a position and part of its heads, NC elements of each half a lane (two up to heads of
// 128, where eight would leave a quarter of the warps). Weight, cos and sin enter as their products
// (w cos and w' sin, once per position), and n at the end:
//   out[i] = n (x[i] (w[i] cos[i]) - x[i + h] (w[i + h] sin[i])), out[i + h] alike.
template <int DT, int NC>
__global__ void __launch_bounds__(32 * kWarps) qk_forward_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  constexpr int V = 1;
  const int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (item >= (int64_t)P.rows * P.split) return;
  const int row = (int)(item / P.split), part = (int)(item - (int64_t)row * P.split);
  const int lanes = P.lanes, per_warp = 32 / lanes;
  const int lane = threadIdx.x & 31, sub = lane & (lanes - 1), mine = lane / lanes;
  const int b = row / P.seq, t = row - b * P.seq;
  const int64_t trow = (int64_t)(P.per_batch ? row : t) * P.hd;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    int grp = first_of(which ? P.groups[0] : 0, part, P.split);
    if (grp >= P.groups[which]) continue;
    float ac[NC][V], as[NC][V], bc[NC][V], bs[NC][V];   // w cos, w' sin of the first half; w' cos', w sin' of the second
    {
      float wl[NC][V], wh[NC][V];
      load_side<DT, V, NC>(wl, P.w[which], 0, P.w_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(wh, P.w[which], P.half, P.w_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(ac, P.cos, trow, P.t_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(bc, P.cos, trow + P.half, P.t_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(as, P.sin, trow, P.t_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(bs, P.sin, trow + P.half, P.t_dtype, sub, lanes, P.half);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        ac[c][0] *= wl[c][0];
        as[c][0] *= wh[c][0];
        bc[c][0] *= wh[c][0];
        bs[c][0] *= wl[c][0];
      }
    }
    for (; grp < P.groups[which]; grp += P.split) {
      const int head = grp * per_warp + mine;
      const bool on = head < P.heads[which];
      const T* x = static_cast<const T*>(P.x[which]) + b * P.xs[which][0] + t * P.xs[which][1] + head * P.xs[which][2];
      Piece<DT, V, NC> lo, hi;
      lo.load(x, sub, lanes, on ? P.half : 0);
      hi.load(x + P.half, sub, lanes, on ? P.half : 0);
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        ss = fmaf(lo.at(c, 0), lo.at(c, 0), ss);
        ss = fmaf(hi.at(c, 0), hi.at(c, 0), ss);
      }
      const float n = rsqrtf(fmaf(lanes_sum<0>(ss, lanes), P.inv_hd, P.eps));
      float ol[NC][V], oh[NC][V];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float xl = lo.at(c, 0), xh = hi.at(c, 0);
        ol[c][0] = n * fmaf(xl, ac[c][0], -xh * as[c][0]);
        oh[c][0] = n * fmaf(xh, bc[c][0], xl * bs[c][0]);
      }
      if (on) {
        T* o = static_cast<T*>(P.out[which]) + b * P.os[which][0] + t * P.os[which][1] + head * P.os[which][2];
        store_piece<DT, V, NC>(o, ol, sub, lanes, P.half);
        store_piece<DT, V, NC>(o + P.half, oh, sub, lanes, P.half);
      }
    }
  }
}

// A block's weight gradients: lanes of the same elements in a warp, then the warps in order.
template <int V, int NC>
__device__ __forceinline__ void block_weights(const QkParams& P, float (&dl)[2][NC][V], float (&dh)[2][NC][V], float* sums, int warp,
                                              int lanes, int sub, int mine) {
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j)
        for (int o = lanes; o < 32; o <<= 1) {
          dl[a][c][j] += __shfl_xor_sync(0xffffffffu, dl[a][c][j], o);
          dh[a][c][j] += __shfl_xor_sync(0xffffffffu, dh[a][c][j], o);
        }
  if (mine == 0) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const int i = (c * lanes + sub) * V + j;
          if (i < P.half) {
            sums[(warp * 2 + a) * P.hd + i] = dl[a][c][j];
            sums[(warp * 2 + a) * P.hd + P.half + i] = dh[a][c][j];
          }
        }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * P.hd; i += 32 * kBwdWarps) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kBwdWarps; ++q) v += sums[q * 2 * P.hd + i];
    P.partial[(int64_t)blockIdx.x * 2 * P.hd + i] = v;
  }
}

// Persistent warps over (position, part of its heads); each lane sums its elements of the
// weight gradients in registers, a block adds its warps' sums in warp order.
template <int DT, int NC>
__global__ void __launch_bounds__(32 * kBwdWarps) qk_backward_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  constexpr int V = 1;
  extern __shared__ float sums[];   // [kBwdWarps][2][hd]
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int lanes = P.lanes, per_warp = 32 / lanes, sub = lane & (lanes - 1), mine = lane / lanes;
  float dl[2][NC][V], dh[2][NC][V];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c) dl[a][c][0] = dh[a][c][0] = 0.f;

  const int64_t items = (int64_t)P.rows * P.split;
  for (int64_t item = (int64_t)blockIdx.x * kBwdWarps + warp; item < items; item += (int64_t)gridDim.x * kBwdWarps) {
    const int row = (int)(item / P.split), part = (int)(item - (int64_t)row * P.split);
    const int b = row / P.seq, t = row - b * P.seq;
    const int64_t trow = (int64_t)(P.per_batch ? row : t) * P.hd;
    float cl[NC][V], ch[NC][V], sl[NC][V], sh[NC][V];
    load_side<DT, V, NC>(cl, P.cos, trow, P.t_dtype, sub, lanes, P.half);
    load_side<DT, V, NC>(ch, P.cos, trow + P.half, P.t_dtype, sub, lanes, P.half);
    load_side<DT, V, NC>(sl, P.sin, trow, P.t_dtype, sub, lanes, P.half);
    load_side<DT, V, NC>(sh, P.sin, trow + P.half, P.t_dtype, sub, lanes, P.half);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      int grp = first_of(which ? P.groups[0] : 0, part, P.split);
      if (grp >= P.groups[which]) continue;
      float wl[NC][V], wh[NC][V];
      load_side<DT, V, NC>(wl, P.w[which], 0, P.w_dtype, sub, lanes, P.half);
      load_side<DT, V, NC>(wh, P.w[which], P.half, P.w_dtype, sub, lanes, P.half);
      for (; grp < P.groups[which]; grp += P.split) {
        const int head = grp * per_warp + mine;
        const bool on = head < P.heads[which];
        const T* x = static_cast<const T*>(P.x[which]) + b * P.xs[which][0] + t * P.xs[which][1] + head * P.xs[which][2];
        const T* g = static_cast<const T*>(P.g[which]) + b * P.gs[which][0] + t * P.gs[which][1] + head * P.gs[which][2];
        Piece<DT, V, NC> xl, xh, gl, gh;
        xl.load(x, sub, lanes, on ? P.half : 0);
        xh.load(x + P.half, sub, lanes, on ? P.half : 0);
        gl.load(g, sub, lanes, on ? P.half : 0);
        gh.load(g + P.half, sub, lanes, on ? P.half : 0);
        float ss = 0.f, sd = 0.f;
        float yl[NC][V], yh[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const float a = xl.at(c, 0), z = xh.at(c, 0);
          ss = fmaf(a, a, ss);
          ss = fmaf(z, z, ss);
          yl[c][0] = fmaf(gl.at(c, 0), cl[c][0], gh.at(c, 0) * sh[c][0]);
          yh[c][0] = fmaf(gh.at(c, 0), ch[c][0], -gl.at(c, 0) * sl[c][0]);
          sd = fmaf(yl[c][0] * wl[c][0], a, sd);
          sd = fmaf(yh[c][0] * wh[c][0], z, sd);
        }
        ss = lanes_sum<0>(ss, lanes);
        sd = lanes_sum<0>(sd, lanes);
        if (on) {   // a head that is not there has no x to be finite
          const float n = rsqrtf(fmaf(ss, P.inv_hd, P.eps));
          const float m = n * n * sd * P.inv_hd;   // dx = n w dy - (x n) m
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const float a = xl.at(c, 0) * n, z = xh.at(c, 0) * n;
            dl[which][c][0] = fmaf(yl[c][0], a, dl[which][c][0]);
            dh[which][c][0] = fmaf(yh[c][0], z, dh[which][c][0]);
            yl[c][0] = fmaf(-a, m, n * (yl[c][0] * wl[c][0]));
            yh[c][0] = fmaf(-z, m, n * (yh[c][0] * wh[c][0]));
          }
          T* o = static_cast<T*>(P.out[which]) + b * P.os[which][0] + t * P.os[which][1] + head * P.os[which][2];
          store_piece<DT, V, NC>(o, yl, sub, lanes, P.half);
          store_piece<DT, V, NC>(o + P.half, yh, sub, lanes, P.half);
        }
      }
    }
  }
  block_weights<V, NC>(P, dl, dh, sums, warp, lanes, sub, mine);
}

// ---- the ring kernels: 16 bytes of a head a lane ---------------------------------------------
//
// The kernels above wait for memory several times a position (tables, then each step's heads), and
// the registers that their loads land in bound the warps of an SM. Here a warp walks many
// positions and copies the heads of the next steps to its own ring in shared memory (cp.async;
// a lane reads back only what it copied itself, so no barrier is needed).

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 smem_load16(uint32_t src) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(src) : "memory");
  return u;
}
__device__ __forceinline__ void smem_store16(uint32_t dst, const float* v) {
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
}
// A lane's V fp32 values, 512 bytes (a warp's 16) apart every four.
template <int V> __device__ __forceinline__ void smem_get(float (&v)[V], uint32_t src) {
#pragma unroll
  for (int q = 0; q < V; q += 4) {
    const uint4 u = smem_load16(src + q * 128);
    v[q] = __uint_as_float(u.x); v[q + 1] = __uint_as_float(u.y); v[q + 2] = __uint_as_float(u.z); v[q + 3] = __uint_as_float(u.w);
  }
}
template <int V> __device__ __forceinline__ void smem_put(uint32_t dst, const float (&v)[V]) {
#pragma unroll
  for (int q = 0; q < V; q += 4) smem_store16(dst + q * 128, v + q);
}

// Item i of a launch: a position and a part of its heads (rows x split stays below 2^26).
struct Item {
  int row, part, b, t;
  __device__ __forceinline__ Item(const QkParams& P, int i) {
    row = P.split == 1 ? i : (int)((uint32_t)i / (uint32_t)P.split);
    part = P.split == 1 ? 0 : i - row * P.split;
    b = (int)((uint32_t)row / (uint32_t)P.seq);
    t = row - b * P.seq;
  }
  template <class T> __device__ __forceinline__ T* at(T* base, const int64_t (&s)[3], int head) const {
    return base + b * s[0] + t * s[1] + head * s[2];
  }
};

// Walks a warp's steps: items from `item` on in strides of `stride`, in each the part's groups of
// q, then of k. The pointers are the lane's own.
template <class T, bool GRAD> struct Cursor {
  int item, items, stride;
  int which, head, left;   // the lane's head, and the groups left in this section
  const T *x, *g;

  // The part's first group of q (w = 0) or k of the current item, or of a later one.
  __device__ __forceinline__ void enter(const QkParams& P, int w, int per_warp, int mine, int at) {
    while (item < items) {
      const Item it(P, item);
#pragma unroll 1
      for (; w < 2; ++w) {
        const int grp = first_of(w ? P.groups[0] : 0, it.part, P.split);
        if (grp < P.groups[w]) {
          which = w;
          left = P.split == 1 ? P.groups[w] : (P.groups[w] - grp + P.split - 1) / P.split;
          head = grp * per_warp + mine;
          x = it.at(static_cast<const T*>(P.x[w]), P.xs[w], head) + at;
          if (GRAD) g = it.at(static_cast<const T*>(P.g[w]), P.gs[w], head) + at;
          return;
        }
      }
      item += stride;
      w = 0;
    }
  }
  __device__ __forceinline__ void advance(const QkParams& P, int per_warp, int mine, int at) {
    if (--left > 0) {
      const int hstep = per_warp * P.split;
      head += hstep;
      x += hstep * P.xs[which][2];
      if (GRAD) g += hstep * P.gs[which][2];
    } else {
      const int w = which + 1;
      if (w == 2) item += stride;
      enter(P, w & 1, per_warp, mine, at);
    }
  }
};

// cos and sin of a position, a lane's pieces: of the heads' type they are loaded a position ahead
// and kept packed until they are used; fp32 ones of 16-bit heads are loaded where they are used.
template <int DT> struct Tables {
  static constexpr int V = DT == ZT_F32 ? 4 : 8;
  Piece<DT, V, 1> piece[4];   // cos, cos', sin, sin'
  int64_t row;

  __device__ __forceinline__ void fetch(const QkParams& P, const Item& it, int sub, int lanes) {
    using T = typename El<DT>::T;
    row = (int64_t)(P.per_batch ? it.row : it.t) * P.hd;
    if (P.t_dtype == DT) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        piece[i].load(static_cast<const T*>(i < 2 ? P.cos : P.sin) + row + (i & 1) * P.half, sub, lanes, P.half);
    }
  }
  __device__ __forceinline__ void get(float (&v)[V], int i, const QkParams& P, int sub, int lanes) const {
    if (P.t_dtype == DT) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = piece[i].at(0, j);
    } else {
      load_side<DT, V, 1>(reinterpret_cast<float(&)[1][V]>(v), i < 2 ? P.cos : P.sin, row + (i & 1) * P.half, P.t_dtype, sub,
                          lanes, P.half);
    }
  }
};

// The block's copy of both norm weights, widened: lane-wise as the heads are.
template <int DT> struct Weights {
  static constexpr int kV = DT == ZT_F32 ? 4 : 8;
  float w[2][2][kV / 4][32][4];   // of q and k, both halves

  __device__ __forceinline__ void fill(const QkParams& P, int warp, int lane, int sub, int lanes) {   // the first four warps
    float v[1][kV];
    load_side<DT, kV, 1>(v, P.w[warp / 2], (warp & 1) * P.half, P.w_dtype, sub, lanes, P.half);
    smem_put(smem_at(&w[warp / 2][warp & 1][0][lane]), v[0]);
  }
};

template <int DT, int LANES>
__global__ void __launch_bounds__(32 * kWarps, kFwdBlocks) qk_forward_ring_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  constexpr int V = 16 / (int)sizeof(T), D = kFwdRing;
  __shared__ uint4 rings[kWarps][D][2][32];
  __shared__ Weights<DT> weights;
  const int lanes = LANES > 0 ? LANES : P.lanes, per_warp = 32 / lanes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, sub = lane & (lanes - 1), mine = lane / lanes;
  const uint32_t ring = smem_at(&rings[warp][0][0][lane]);   // a step's slot is 1024 bytes
  const bool in = sub * V < P.half;
  Cursor<T, false> ahead;
  ahead.item = blockIdx.x * kWarps + warp;
  ahead.items = P.rows * P.split;
  ahead.stride = gridDim.x * kWarps;
  ahead.enter(P, 0, per_warp, mine, sub * V);
  auto fetch = [&](uint32_t slot) {
    if (ahead.item < ahead.items) {
      if (in && ahead.head < P.heads[ahead.which]) {
        copy16(slot, ahead.x);
        copy16(slot + 512, ahead.x + P.half);
      }
      ahead.advance(P, per_warp, mine, sub * V);
    }
    copy_commit();
  };
#pragma unroll 1
  for (int d = 0; d < D; ++d) fetch(ring + d * 1024);
  const int items = ahead.items, stride = ahead.stride;
  int item = blockIdx.x * kWarps + warp;
  Tables<DT> tables;
  if (item < items) tables.fetch(P, Item(P, item), sub, lanes);
  weights.fill(P, warp, lane, sub, lanes);
  __syncthreads();
  int slot = 0;
  for (; item < items; item += stride) {
    const Item it(P, item);
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      int grp = first_of(which ? P.groups[0] : 0, it.part, P.split);
      const bool some = grp < P.groups[which];
      float ac[V], as[V], bc[V], bs[V];   // w cos, w' sin of the first half; w' cos', w sin' of the second
      if (some) {
        float wl[V], wh[V];
        smem_get(wl, smem_at(&weights.w[which][0][0][lane]));
        smem_get(wh, smem_at(&weights.w[which][1][0][lane]));
        tables.get(ac, 0, P, sub, lanes);
        tables.get(bc, 1, P, sub, lanes);
        tables.get(as, 2, P, sub, lanes);
        tables.get(bs, 3, P, sub, lanes);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          ac[j] *= wl[j];
          as[j] *= wh[j];
          bc[j] *= wh[j];
          bs[j] *= wl[j];
        }
      }
      if (which && item + stride < items) tables.fetch(P, Item(P, item + stride), sub, lanes);
      if (!some) continue;
      const int hstep = per_warp * P.split, heads = P.heads[which];
      int head = grp * per_warp + mine;
      T* o = it.at(static_cast<T*>(P.out[which]), P.os[which], head) + sub * V;
      const int64_t ostep = hstep * P.os[which][2];
      for (; grp < P.groups[which]; grp += P.split) {
        const bool on = in && head < heads;
        const uint32_t here = ring + slot * 1024;
        copy_wait<D - 1>();
        Piece<DT, V, 1> lo, hi;
        lo.take(smem_load16(here));
        hi.take(smem_load16(here + 512));
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          ss = fmaf(lo.at(0, j), lo.at(0, j), ss);
          ss = fmaf(hi.at(0, j), hi.at(0, j), ss);
        }
        ss = lanes_sum<LANES>(on ? ss : 0.f, lanes);   // a slot that nothing was copied to holds anything
        fetch(here);                                   // the sum has read this slot
        slot = (slot + 1) & (D - 1);
        const float n = rsqrtf(fmaf(ss, P.inv_hd, P.eps));
        float ol[1][V], oh[1][V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xl = lo.at(0, j), xh = hi.at(0, j);
          ol[0][j] = n * fmaf(xl, ac[j], -xh * as[j]);
          oh[0][j] = n * fmaf(xh, bc[j], xl * bs[j]);
        }
        if (on) {
          store_piece<DT, V, 1>(o, ol, 0, 1, V);
          store_piece<DT, V, 1>(o + P.half, oh, 0, 1, V);
        }
        head += hstep;
        o += ostep;
      }
    }
  }
}

// The tables and weights of a step are read from shared memory, widened: in registers they would
// take half of what a thread may have, and packed there their widening at every step measured a
// fifth of the instructions.
template <int DT> struct BwdShared {
  static constexpr int kV = DT == ZT_F32 ? 4 : 8;
  uint4 ring[kBwdWarps][kBwdRing][4][32];
  float table[kBwdWarps][4][kV / 4][32][4];   // cos, cos', sin, sin' of the warp's position
  Weights<DT> weights;
};

template <int DT, int LANES>
__global__ void __launch_bounds__(32 * kBwdWarps, kBwdBlocks) qk_backward_ring_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  constexpr int V = 16 / (int)sizeof(T), D = kBwdRing;
  constexpr uint32_t kSide = V * 128;   // bytes of a warp's V fp32 values a lane
  extern __shared__ uint4 dynamic[];    // BwdShared; at the end the warps' sums
  BwdShared<DT>& S = *reinterpret_cast<BwdShared<DT>*>(dynamic);
  const int lanes = LANES > 0 ? LANES : P.lanes, per_warp = 32 / lanes;
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, sub = lane & (lanes - 1), mine = lane / lanes;
  const uint32_t ring = smem_at(&S.ring[warp][0][0][lane]);   // a step's slot is 2048 bytes
  const uint32_t table = smem_at(&S.table[warp][0][0][lane]), weight = smem_at(&S.weights.w[0][0][0][lane]);
  const bool in = sub * V < P.half;
  float dl[2][1][V], dh[2][1][V];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int j = 0; j < V; ++j) dl[a][0][j] = dh[a][0][j] = 0.f;

  Cursor<T, true> ahead;
  ahead.item = blockIdx.x * kBwdWarps + warp;
  ahead.items = P.rows * P.split;
  ahead.stride = gridDim.x * kBwdWarps;
  ahead.enter(P, 0, per_warp, mine, sub * V);
  auto fetch = [&](uint32_t slot) {
    if (ahead.item < ahead.items) {
      if (in && ahead.head < P.heads[ahead.which]) {
        copy16(slot, ahead.x);
        copy16(slot + 512, ahead.x + P.half);
        copy16(slot + 1024, ahead.g);
        copy16(slot + 1536, ahead.g + P.half);
      }
      ahead.advance(P, per_warp, mine, sub * V);
    }
    copy_commit();
  };
#pragma unroll 1
  for (int d = 0; d < D; ++d) fetch(ring + d * 2048);
  const int items = ahead.items, stride = ahead.stride;
  int item = blockIdx.x * kBwdWarps + warp;
  Tables<DT> tables;
  if (item < items) tables.fetch(P, Item(P, item), sub, lanes);
  if (warp < 4) S.weights.fill(P, warp, lane, sub, lanes);
  __syncthreads();
  int slot = 0;
  for (; item < items; item += stride) {
    const Item it(P, item);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v[V];
      tables.get(v, i, P, sub, lanes);
      smem_put(table + i * kSide, v);
    }
    if (item + stride < items) tables.fetch(P, Item(P, item + stride), sub, lanes);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      int grp = first_of(which ? P.groups[0] : 0, it.part, P.split);
      if (grp >= P.groups[which]) continue;
      const int hstep = per_warp * P.split, heads = P.heads[which];
      int head = grp * per_warp + mine;
      T* o = it.at(static_cast<T*>(P.out[which]), P.os[which], head) + sub * V;
      const int64_t ostep = hstep * P.os[which][2];
      for (; grp < P.groups[which]; grp += P.split) {
        const bool on = in && head < heads;
        const uint32_t here = ring + slot * 2048;
        copy_wait<D - 1>();
        Piece<DT, V, 1> xl, xh, gl, gh;
        gl.take(smem_load16(here + 1024));
        gh.take(smem_load16(here + 1536));
        xl.take(smem_load16(here));
        xh.take(smem_load16(here + 512));
        float yl[V], yh[V], wl[V], wh[V];   // dy, then w dy
        {
          float c[V], s[V];
          smem_get(c, table);
          smem_get(s, table + 3 * kSide);
#pragma unroll
          for (int j = 0; j < V; ++j) yl[j] = fmaf(gl.at(0, j), c[j], gh.at(0, j) * s[j]);
          smem_get(c, table + kSide);
          smem_get(s, table + 2 * kSide);
#pragma unroll
          for (int j = 0; j < V; ++j) yh[j] = fmaf(gh.at(0, j), c[j], -gl.at(0, j) * s[j]);
        }
        smem_get(wl, weight + which * 2 * kSide);
        smem_get(wh, weight + which * 2 * kSide + kSide);
        float ss = 0.f, sd = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float a = xl.at(0, j), z = xh.at(0, j);
          ss = fmaf(a, a, ss);
          ss = fmaf(z, z, ss);
          wl[j] *= yl[j];
          wh[j] *= yh[j];
          sd = fmaf(wl[j], a, sd);
          sd = fmaf(wh[j], z, sd);
        }
        ss = lanes_sum<LANES>(on ? ss : 0.f, lanes);   // a slot that nothing was copied to holds anything
        sd = lanes_sum<LANES>(on ? sd : 0.f, lanes);
        fetch(here);                                   // the sums have read this slot
        slot = (slot + 1) & (D - 1);
        if (on) {
          const float n = rsqrtf(fmaf(ss, P.inv_hd, P.eps));
          const float m = n * n * sd * P.inv_hd;   // dx = n w dy - (x n) m
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = xl.at(0, j) * n, z = xh.at(0, j) * n;
            dl[which][0][j] = fmaf(yl[j], a, dl[which][0][j]);
            dh[which][0][j] = fmaf(yh[j], z, dh[which][0][j]);
            wl[j] = fmaf(-a, m, n * wl[j]);
            wh[j] = fmaf(-z, m, n * wh[j]);
          }
          store_piece<DT, V, 1>(o, reinterpret_cast<const float(&)[1][V]>(wl), 0, 1, V);
          store_piece<DT, V, 1>(o + P.half, reinterpret_cast<const float(&)[1][V]>(wh), 0, 1, V);
        }
        head += hstep;
        o += ostep;
      }
    }
  }
  copy_wait<0>();
  __syncthreads();   // the rings become the warps' sums
  block_weights<V, 1>(P, dl, dh, reinterpret_cast<float*>(dynamic), warp, lanes, sub, mine);
}

// The blocks' weight gradients, summed in a fixed order by 32 x 32 threads per 32 columns and
// rounded to the weights' type.
template <int DT>
__global__ void __launch_bounds__(1024) qk_weight_kernel(const float* __restrict__ partial, int32_t blocks, int32_t hd,
                                                         typename El<DT>::T* __restrict__ dwq,
                                                         typename El<DT>::T* __restrict__ dwk) {
  __shared__ float part[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x / 32, col = blockIdx.x * 32 + x;
  float v = 0.f;
  if (col < 2 * hd) {
#pragma unroll 8
    for (int b = y; b < blocks; b += 32) v += partial[(int64_t)b * 2 * hd + col];
  }
  part[y][x] = v;
  __syncthreads();
  float s = part[x][y];   // warp y now sums column y of these 32
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int c = blockIdx.x * 32 + y;
  if (x == 0 && c < 2 * hd) {
    if (c < hd) dwq[c] = El<DT>::from(s);
    else dwk[c - hd] = El<DT>::from(s);
  }
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int bwd_blocks(int64_t items) {
  const int64_t need = (items + kBwdWarps - 1) / kBwdWarps, most = (int64_t)zt::sm_count() * kBwdBlocks;
  return (int)(need < most ? need : most);
}

// Whether a call's heads can go through the ring, 16 bytes a lane: whole 16-byte vectors
// everywhere, at most 32 of them in a half. Else a lane takes single elements (head
// sizes that are no multiple of 16 elements, 8 in fp32; views off their alignment).
bool ring_fits(const zt_qk_args* a, bool backward) {
  const int v = a->dtype == ZT_F32 ? 4 : 8;
  if ((a->head_dim / 2) % v || a->head_dim / 2 > 32 * v) return false;
  auto strides = [&](const int64_t* s) {   // those of a dimension of one are never used
    return (a->batch == 1 || s[0] % v == 0) && (a->seq == 1 || s[1] % v == 0) &&
           ((a->q_heads == 1 && a->k_heads == 1) || s[2] % v == 0);
  };
  for (const void* p : {a->q, a->k, (const void*)a->q_out, (const void*)a->k_out, a->q_weight, a->k_weight, a->cos, a->sin})
    if (!aligned(p, 16)) return false;
  if (!strides(a->q_strides) || !strides(a->k_strides) || !strides(a->q_out_strides) || !strides(a->k_out_strides))
    return false;
  return !backward || (aligned(a->q_grad, 16) && aligned(a->k_grad, 16) && strides(a->q_grad_strides) &&
                       strides(a->k_grad_strides));
}

int check_args(const zt_qk_args* a, bool backward, const char* who) {
  const std::string w(who);
  if (!a) return zt::set_error(ZT_ERR_INVALID, w + ": null arguments");
  if (a->batch < 0 || a->seq < 0 || a->q_heads <= 0 || a->k_heads <= 0)
    return zt::set_error(ZT_ERR_INVALID, w + ": negative size or no heads");
  if (a->head_dim < 2 || a->head_dim % 2 || a->head_dim > kMaxHeadDim)
    return zt::set_error(ZT_ERR_INVALID, w + ": head_dim must be even and at most 512");
  if (a->dtype != ZT_F32 && a->dtype != ZT_BF16 && a->dtype != ZT_F16)
    return zt::set_error(ZT_ERR_INVALID, w + ": unknown dtype");
  if ((a->weight_dtype != a->dtype && a->weight_dtype != ZT_F32) || (a->table_dtype != a->dtype && a->table_dtype != ZT_F32))
    return zt::set_error(ZT_ERR_INVALID, w + ": weights and tables must have the heads' dtype or fp32");
  if (a->table_batch != 0 && a->table_batch != 1) return zt::set_error(ZT_ERR_INVALID, w + ": table_batch must be 0 or 1");
  if (!(a->eps >= 0.f) || isinf(a->eps)) return zt::set_error(ZT_ERR_INVALID, w + ": eps must be finite and not negative");
  if (a->seq > 0 && a->batch > ((int64_t)1 << 25) / a->seq)
    return zt::set_error(ZT_ERR_LIMIT, w + ": more than 2^25 positions");
  if (a->q_heads > 65535 || a->k_heads > 65535) return zt::set_error(ZT_ERR_LIMIT, w + ": more than 65535 heads");
  if (a->batch * a->seq == 0 && !backward) return ZT_OK;
  if (!a->q_weight || !a->k_weight || (a->batch * a->seq > 0 && (!a->q || !a->k || !a->q_out || !a->k_out || !a->cos || !a->sin)))
    return zt::set_error(ZT_ERR_INVALID, w + ": null pointer");
  if (backward && (!a->dq_weight || !a->dk_weight || (a->batch * a->seq > 0 && (!a->q_grad || !a->k_grad || !a->workspace))))
    return zt::set_error(ZT_ERR_INVALID, w + ": null pointer");
  return ZT_OK;
}

int pow2_at_least(int v) {
  int p = 1;
  while (p < v) p <<= 1;
  return p;
}

// Lanes of a head, and the warps that share a position's heads: 1 where the positions
// alone give every SM `per_sm` warps, else as many as bring the launch up to that.
void shape(const zt_qk_args* a, bool ring, int per_sm, QkParams* P) {
  const int v = !ring ? 1 : a->dtype == ZT_F32 ? 4 : 8;
  P->hd = a->head_dim;
  P->half = a->head_dim / 2;
  const int lanes = pow2_at_least((P->half + v - 1) / v);
  P->lanes = lanes > 32 ? 32 : lanes;
  const int per_warp = 32 / P->lanes;
  P->heads[0] = a->q_heads;
  P->heads[1] = a->k_heads;
  P->groups[0] = (a->q_heads + per_warp - 1) / per_warp;
  P->groups[1] = (a->k_heads + per_warp - 1) / per_warp;
  P->rows = (int32_t)(a->batch * a->seq);
  P->seq = (int32_t)a->seq;
  P->per_batch = a->table_batch;
  P->w_dtype = a->weight_dtype;
  P->t_dtype = a->table_dtype;
  P->eps = a->eps;
  P->inv_hd = 1.0f / (float)a->head_dim;
  const int64_t want = (int64_t)zt::sm_count() * per_sm;
  const int64_t split = P->rows > 0 ? (want + P->rows - 1) / P->rows : 1;
  const int total = P->groups[0] + P->groups[1];
  P->split = (int32_t)(split < total ? split : total);
}

void fill(const zt_qk_args* a, QkParams* P) {
  P->x[0] = a->q; P->x[1] = a->k;
  P->g[0] = a->q_grad; P->g[1] = a->k_grad;
  P->out[0] = a->q_out; P->out[1] = a->k_out;
  P->w[0] = a->q_weight; P->w[1] = a->k_weight;
  P->cos = a->cos; P->sin = a->sin;
  P->partial = static_cast<float*>(a->workspace);
  for (int i = 0; i < 3; ++i) {
    P->xs[0][i] = a->q_strides[i]; P->xs[1][i] = a->k_strides[i];
    P->gs[0][i] = a->q_grad_strides[i]; P->gs[1][i] = a->k_grad_strides[i];
    P->os[0][i] = a->q_out_strides[i]; P->os[1][i] = a->k_out_strides[i];
  }
}

template <int DT, int LANES> int launch_ring(const QkParams& P, bool backward, int blocks, cudaStream_t s) {
  if (!backward) {
    qk_forward_ring_kernel<DT, LANES><<<blocks, 32 * kWarps, 0, s>>>(P);
    return ZT_OK;
  }
  static std::mutex mu;
  static bool ready[64] = {false};
  int dev = 0;
  if (int rc = zt::check_cuda(cudaGetDevice(&dev), "zt_qk_norm_rope_backward: cudaGetDevice")) return rc;
  if (dev < 0 || dev >= 64) return zt::set_error(ZT_ERR_LIMIT, "zt_qk_norm_rope_backward: device ordinal >= 64");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!ready[dev]) {
      if (int rc = zt::check_cuda(cudaFuncSetAttribute(qk_backward_ring_kernel<DT, LANES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)sizeof(BwdShared<DT>)), "zt_qk_norm_rope_backward: shared memory attribute"))
        return rc;
      ready[dev] = true;
    }
  }
  qk_backward_ring_kernel<DT, LANES><<<blocks, 32 * kBwdWarps, sizeof(BwdShared<DT>), s>>>(P);
  return ZT_OK;
}

template <int DT, int NC> void launch_plain(const QkParams& P, bool backward, int blocks, cudaStream_t s) {
  if (backward)
    qk_backward_kernel<DT, NC><<<blocks, 32 * kBwdWarps, sizeof(float) * kBwdWarps * 2 * P.hd, s>>>(P);
  else
    qk_forward_kernel<DT, NC><<<blocks, 32 * kWarps, 0, s>>>(P);
}

template <int DT> int launch_typed(const QkParams& P, bool backward, bool ring, int blocks, cudaStream_t s) {
  if (ring) {
    if (P.lanes == 4) return launch_ring<DT, 4>(P, backward, blocks, s);
    if (P.lanes == 8) return launch_ring<DT, 8>(P, backward, blocks, s);
    if (P.lanes == 16) return launch_ring<DT, 16>(P, backward, blocks, s);
    return launch_ring<DT, 0>(P, backward, blocks, s);
  }
  P.half <= 64 ? launch_plain<DT, 2>(P, backward, blocks, s) : launch_plain<DT, kE>(P, backward, blocks, s);
  return ZT_OK;
}

int launch(const zt_qk_args* a, const QkParams& P, bool backward, bool ring, int blocks, cudaStream_t s) {
  if (a->dtype == ZT_F32) return launch_typed<ZT_F32>(P, backward, ring, blocks, s);
  if (a->dtype == ZT_BF16) return launch_typed<ZT_BF16>(P, backward, ring, blocks, s);
  return launch_typed<ZT_F16>(P, backward, ring, blocks, s);
}

}  // namespace

extern "C" {

int zt_qk_norm_rope(const zt_qk_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_args(a, false, "zt_qk_norm_rope")) return rc;
  if (a->batch * a->seq == 0) return ZT_OK;
  QkParams P = {};
  const bool ring = ring_fits(a, false);
  shape(a, ring, kFwdBlocks * kWarps, &P);
  fill(a, &P);
  int64_t blocks = ((int64_t)P.rows * P.split + kWarps - 1) / kWarps;
  if (ring && blocks > (int64_t)zt::sm_count() * kFwdBlocks) blocks = (int64_t)zt::sm_count() * kFwdBlocks;
  if (int rc = launch(a, P, false, ring, (int)blocks, zt::as_stream(stream))) return rc;
  return zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope launch");
}

size_t zt_qk_norm_rope_workspace_bytes(int32_t head_dim) {
  zt::clear_error();
  if (head_dim < 2 || head_dim % 2 || head_dim > kMaxHeadDim) {
    zt::set_error(ZT_ERR_INVALID, "zt_qk_norm_rope_workspace_bytes: head_dim must be even and at most 512");
    return 0;
  }
  return sizeof(float) * 2 * (size_t)head_dim * (size_t)(zt::sm_count() * kBwdBlocks);
}

int zt_qk_norm_rope_backward(const zt_qk_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_args(a, true, "zt_qk_norm_rope_backward")) return rc;
  QkParams P = {};
  int blocks = 0;
  cudaStream_t s = zt::as_stream(stream);
  if (a->batch * a->seq > 0) {
    if (a->workspace_bytes < zt_qk_norm_rope_workspace_bytes(a->head_dim))
      return zt::set_error(ZT_ERR_INVALID, "zt_qk_norm_rope_backward: workspace too small");
    const bool ring = ring_fits(a, true);
    shape(a, ring, kBwdBlocks * kBwdWarps, &P);
    fill(a, &P);
    blocks = bwd_blocks((int64_t)P.rows * P.split);
    if (int rc = launch(a, P, true, ring, blocks, s)) return rc;
    if (int rc = zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope_backward launch")) return rc;
  }
  const unsigned grid = (unsigned)((2 * a->head_dim + 31) / 32);
  const float* part = static_cast<const float*>(a->workspace);
  if (a->weight_dtype == ZT_F32)
    qk_weight_kernel<ZT_F32><<<grid, 1024, 0, s>>>(part, blocks, a->head_dim, static_cast<float*>(a->dq_weight),
                                                  static_cast<float*>(a->dk_weight));
  else if (a->weight_dtype == ZT_BF16)
    qk_weight_kernel<ZT_BF16><<<grid, 1024, 0, s>>>(part, blocks, a->head_dim, static_cast<__nv_bfloat16*>(a->dq_weight),
                                                   static_cast<__nv_bfloat16*>(a->dk_weight));
  else
    qk_weight_kernel<ZT_F16><<<grid, 1024, 0, s>>>(part, blocks, a->head_dim, static_cast<__half*>(a->dq_weight),
                                                  static_cast<__half*>(a->dk_weight));
  return zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope_backward: weight launch");
}

}  // extern "C"
