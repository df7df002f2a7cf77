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

#include "zt_common.cuh"

namespace {

constexpr int kWarps = 4;          // warps of a forward block; they share nothing
constexpr int kBwdWarps = 8;       // warps of a backward block; they share the weight gradient's sum
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
    if constexpr (V * sizeof(T) == 16) {
      uint4 u;
      if constexpr (DT == ZT_F32) {
        u = make_uint4(__float_as_uint(v[c][0]), __float_as_uint(v[c][1]), __float_as_uint(v[c][2]), __float_as_uint(v[c][3]));
      } else if constexpr (DT == ZT_BF16) {
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[c][2 * j], v[c][2 * j + 1]);
          r[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        u = make_uint4(r[0], r[1], r[2], r[3]);
      } else {
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2 h = __floats2half2_rn(v[c][2 * j], v[c][2 * j + 1]);
          r[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
        u = make_uint4(r[0], r[1], r[2], r[3]);
      }
      *reinterpret_cast<uint4*>(p + i) = u;
    } else {
      p[i] = El<DT>::from(v[c][0]);
    }
  }
}

// Weights and tables: packed in the heads' own type (SAME), or of either type, widened to
// fp32 as they are loaded.
template <int DT, int V, int NC, bool SAME> struct Side;
template <int DT, int V, int NC> struct Side<DT, V, NC, true> {
  Piece<DT, V, NC> lo, hi;
  __device__ __forceinline__ void load(const void* base, int64_t off, int32_t, int sub, int lanes, int half) {
    const typename El<DT>::T* p = static_cast<const typename El<DT>::T*>(base) + off;
    lo.load(p, sub, lanes, half);
    hi.load(p + half, sub, lanes, half);
  }
  __device__ __forceinline__ float l(int c, int j) const { return lo.at(c, j); }
  __device__ __forceinline__ float h(int c, int j) const { return hi.at(c, j); }
};
template <int DT, int V, int NC> struct Side<DT, V, NC, false> {
  float lo[NC][V], hi[NC][V];
  __device__ __forceinline__ static float one(const void* base, int64_t i, int32_t dtype) {
    if (dtype == ZT_F32) return static_cast<const float*>(base)[i];
    return El<DT>::to(static_cast<const typename El<DT>::T*>(base)[i]);
  }
  __device__ __forceinline__ void load(const void* base, int64_t off, int32_t dtype, int sub, int lanes, int half) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = (c * lanes + sub) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        lo[c][j] = i + j < half ? one(base, off + i + j, dtype) : 0.f;
        hi[c][j] = i + j < half ? one(base, off + half + i + j, dtype) : 0.f;
      }
    }
  }
  __device__ __forceinline__ float l(int c, int j) const { return lo[c][j]; }
  __device__ __forceinline__ float h(int c, int j) const { return hi[c][j]; }
};

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp: position `row`, its head groups part, part + split, ...
template <int DT, int V, int NC, bool SAME>
__global__ void __launch_bounds__(32 * kWarps) qk_forward_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  const int64_t item = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  if (item >= (int64_t)P.rows * P.split) return;
  const int row = (int)(item / P.split), part = (int)(item - (int64_t)row * P.split);
  const int lane = threadIdx.x & 31;
  const int sub = lane & (P.lanes - 1), mine = lane / P.lanes, per_warp = 32 / P.lanes;
  const int b = row / P.seq, t = row - b * P.seq;
  const int64_t trow = (int64_t)(P.per_batch ? row : t) * P.hd;

  Side<DT, V, NC, SAME> cs, sn, w;
  cs.load(P.cos, trow, P.t_dtype, sub, P.lanes, P.half);
  sn.load(P.sin, trow, P.t_dtype, sub, P.lanes, P.half);
  const int total = P.groups[0] + P.groups[1];
  int loaded = -1;
  for (int grp = part; grp < total; grp += P.split) {
    const int which = grp >= P.groups[0];
    const int head = (grp - (which ? P.groups[0] : 0)) * per_warp + mine;
    const bool on = head < P.heads[which];
    if (which != loaded) {
      w.load(P.w[which], 0, P.w_dtype, sub, P.lanes, P.half);
      loaded = which;
    }
    Piece<DT, V, NC> lo, hi;
    const T* x = static_cast<const T*>(P.x[which]) + b * P.xs[which][0] + t * P.xs[which][1] + head * P.xs[which][2];
    lo.load(x, sub, P.lanes, on ? P.half : 0);
    hi.load(x + P.half, sub, P.lanes, on ? P.half : 0);
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        ss = fmaf(lo.at(c, j), lo.at(c, j), ss);
        ss = fmaf(hi.at(c, j), hi.at(c, j), ss);
      }
    const float n = rsqrtf(fmaf(lanes_sum(ss, P.lanes), P.inv_hd, P.eps));
    float ol[NC][V], oh[NC][V];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float yl = lo.at(c, j) * n * w.l(c, j), yh = hi.at(c, j) * n * w.h(c, j);
        ol[c][j] = fmaf(yl, cs.l(c, j), -yh * sn.l(c, j));
        oh[c][j] = fmaf(yh, cs.h(c, j), yl * sn.h(c, j));
      }
    if (on) {
      T* o = static_cast<T*>(P.out[which]) + b * P.os[which][0] + t * P.os[which][1] + head * P.os[which][2];
      store_piece<DT, V, NC>(o, ol, sub, P.lanes, P.half);
      store_piece<DT, V, NC>(o + P.half, oh, sub, P.lanes, P.half);
    }
  }
}

// Persistent warps over (position, part of its heads); each lane sums its elements of the
// weight gradients in registers, a block adds its warps' sums in warp order.
template <int DT, int V, int NC, bool SAME>
__global__ void __launch_bounds__(32 * kBwdWarps) qk_backward_kernel(const __grid_constant__ QkParams P) {
  using T = typename El<DT>::T;
  extern __shared__ float sums[];   // [kBwdWarps][2][hd]
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int sub = lane & (P.lanes - 1), mine = lane / P.lanes, per_warp = 32 / P.lanes;
  const int total = P.groups[0] + P.groups[1];
  float dl[2][NC][V], dh[2][NC][V];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) dl[a][c][j] = dh[a][c][j] = 0.f;

  const int64_t items = (int64_t)P.rows * P.split;
  for (int64_t item = (int64_t)blockIdx.x * kBwdWarps + warp; item < items; item += (int64_t)gridDim.x * kBwdWarps) {
    const int row = (int)(item / P.split), part = (int)(item - (int64_t)row * P.split);
    const int b = row / P.seq, t = row - b * P.seq;
    const int64_t trow = (int64_t)(P.per_batch ? row : t) * P.hd;
    Side<DT, V, NC, SAME> cs, sn, w;
    cs.load(P.cos, trow, P.t_dtype, sub, P.lanes, P.half);
    sn.load(P.sin, trow, P.t_dtype, sub, P.lanes, P.half);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int first = which ? P.groups[0] : 0, last = which ? total : P.groups[0];
      // the first group of this part at or after `first`
      int grp = part >= first ? part : part + (first - part + P.split - 1) / P.split * P.split;
      if (grp >= last) continue;
      w.load(P.w[which], 0, P.w_dtype, sub, P.lanes, P.half);
      for (; grp < last; grp += P.split) {
        const int head = (grp - first) * per_warp + mine;
        const bool on = head < P.heads[which];
        const T* x = static_cast<const T*>(P.x[which]) + b * P.xs[which][0] + t * P.xs[which][1] + head * P.xs[which][2];
        const T* g = static_cast<const T*>(P.g[which]) + b * P.gs[which][0] + t * P.gs[which][1] + head * P.gs[which][2];
        Piece<DT, V, NC> xl, xh, gl, gh;
        xl.load(x, sub, P.lanes, on ? P.half : 0);
        xh.load(x + P.half, sub, P.lanes, on ? P.half : 0);
        gl.load(g, sub, P.lanes, on ? P.half : 0);
        gh.load(g + P.half, sub, P.lanes, on ? P.half : 0);
        float ss = 0.f, sd = 0.f;
        float yl[NC][V], yh[NC][V];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = xl.at(c, j), z = xh.at(c, j);
            ss = fmaf(a, a, ss);
            ss = fmaf(z, z, ss);
            yl[c][j] = fmaf(gl.at(c, j), cs.l(c, j), gh.at(c, j) * sn.h(c, j));
            yh[c][j] = fmaf(gh.at(c, j), cs.h(c, j), -gl.at(c, j) * sn.l(c, j));
            sd = fmaf(yl[c][j] * w.l(c, j), a, sd);
            sd = fmaf(yh[c][j] * w.h(c, j), z, sd);
          }
        ss = lanes_sum(ss, P.lanes);
        sd = lanes_sum(sd, P.lanes);
        const float n = rsqrtf(fmaf(ss, P.inv_hd, P.eps));
        const float m = n * n * sd * P.inv_hd;   // dx = n (w dy - x m)
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = xl.at(c, j), z = xh.at(c, j);
            if (on) {   // a head that is not there has no x to be finite
              dl[which][c][j] = fmaf(yl[c][j], a * n, dl[which][c][j]);
              dh[which][c][j] = fmaf(yh[c][j], z * n, dh[which][c][j]);
            }
            yl[c][j] = n * fmaf(-a, m, yl[c][j] * w.l(c, j));
            yh[c][j] = n * fmaf(-z, m, yh[c][j] * w.h(c, j));
          }
        if (on) {
          T* o = static_cast<T*>(P.out[which]) + b * P.os[which][0] + t * P.os[which][1] + head * P.os[which][2];
          store_piece<DT, V, NC>(o, yl, sub, P.lanes, P.half);
          store_piece<DT, V, NC>(o + P.half, yh, sub, P.lanes, P.half);
        }
      }
    }
  }
  // lanes of the same elements in a warp, then the block's warps
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j)
        for (int o = P.lanes; o < 32; o <<= 1) {
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
          const int i = (c * P.lanes + sub) * V + j;
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

// The blocks' weight gradients, summed in block order by 8 x 32 threads per 32 columns and
// rounded to the weights' type.
template <int DT>
__global__ void __launch_bounds__(256) qk_weight_kernel(const float* __restrict__ partial, int32_t blocks, int32_t hd,
                                                        typename El<DT>::T* __restrict__ dwq,
                                                        typename El<DT>::T* __restrict__ dwk) {
  __shared__ float part[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x / 32;
  float v = 0.f;
  if (col < 2 * hd)
    for (int b = y; b < blocks; b += 8) v += partial[(int64_t)b * 2 * hd + col];
  part[y][threadIdx.x & 31] = v;
  __syncthreads();
  if (y == 0 && col < 2 * hd) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
    if (col < hd) dwq[col] = El<DT>::from(s);
    else dwk[col - hd] = El<DT>::from(s);
  }
}

bool aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

int bwd_blocks(int64_t items) {
  const int64_t need = (items + kBwdWarps - 1) / kBwdWarps, most = (int64_t)zt::sm_count() * 2;
  return (int)(need < most ? need : most);
}

// Whether a lane can take 16 bytes at a time: the halves and every stride are whole
// vectors and every pointer is aligned to them.
bool wide(const zt_qk_args* a, bool backward) {
  const int v = a->dtype == ZT_F32 ? 4 : 8;
  if ((a->head_dim / 2) % v) return false;
  auto strides = [&](const int64_t* s) { return s[0] % v == 0 && s[1] % v == 0 && s[2] % v == 0; };
  const void* ptrs[] = {a->q, a->k, a->q_out, a->k_out, a->q_weight, a->k_weight, a->cos, a->sin};
  for (const void* p : ptrs)
    if (!aligned(p, 16)) return false;
  if (!strides(a->q_strides) || !strides(a->k_strides) || !strides(a->q_out_strides) || !strides(a->k_out_strides))
    return false;
  if (backward && (!aligned(a->q_grad, 16) || !aligned(a->k_grad, 16) || !strides(a->q_grad_strides) ||
                   !strides(a->k_grad_strides)))
    return false;
  return true;
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
  if (a->seq > 0 && a->batch > (int64_t)(INT32_MAX / 64) / a->seq)
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
void shape(const zt_qk_args* a, bool is_wide, int per_sm, QkParams* P) {
  const int v = is_wide ? (a->dtype == ZT_F32 ? 4 : 8) : 1;
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

template <int DT, int V, int NC, bool SAME>
void launch_one(const QkParams& P, bool backward, int blocks, cudaStream_t s) {
  if (backward)
    qk_backward_kernel<DT, V, NC, SAME><<<blocks, 32 * kBwdWarps, sizeof(float) * kBwdWarps * 2 * P.hd, s>>>(P);
  else
    qk_forward_kernel<DT, V, NC, SAME><<<blocks, 32 * kWarps, 0, s>>>(P);
}

template <int DT>
void launch_half(const QkParams& P, bool backward, bool is_wide, bool same, int blocks, cudaStream_t s) {
  if (is_wide) same ? launch_one<DT, 8, 1, true>(P, backward, blocks, s) : launch_one<DT, 8, 1, false>(P, backward, blocks, s);
  else same ? launch_one<DT, 1, kE, true>(P, backward, blocks, s) : launch_one<DT, 1, kE, false>(P, backward, blocks, s);
}

void launch(const zt_qk_args* a, const QkParams& P, bool backward, bool is_wide, int blocks, cudaStream_t s) {
  const bool same = a->weight_dtype == a->dtype && a->table_dtype == a->dtype;
  if (a->dtype == ZT_BF16) return launch_half<ZT_BF16>(P, backward, is_wide, same, blocks, s);
  if (a->dtype == ZT_F16) return launch_half<ZT_F16>(P, backward, is_wide, same, blocks, s);
  if (!is_wide) return launch_one<ZT_F32, 1, kE, true>(P, backward, blocks, s);
  if (P.half <= 128) return launch_one<ZT_F32, 4, 1, true>(P, backward, blocks, s);
  launch_one<ZT_F32, 4, 2, true>(P, backward, blocks, s);
}

}  // namespace

extern "C" {

int zt_qk_norm_rope(const zt_qk_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_args(a, false, "zt_qk_norm_rope")) return rc;
  if (a->batch * a->seq == 0) return ZT_OK;
  QkParams P = {};
  const bool is_wide = wide(a, false);
  shape(a, is_wide, 32, &P);
  fill(a, &P);
  const int64_t items = (int64_t)P.rows * P.split;
  launch(a, P, false, is_wide, (int)((items + kWarps - 1) / kWarps), zt::as_stream(stream));
  return zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope launch");
}

size_t zt_qk_norm_rope_workspace_bytes(int32_t head_dim) {
  zt::clear_error();
  if (head_dim < 2 || head_dim % 2 || head_dim > kMaxHeadDim) {
    zt::set_error(ZT_ERR_INVALID, "zt_qk_norm_rope_workspace_bytes: head_dim must be even and at most 512");
    return 0;
  }
  return sizeof(float) * 2 * (size_t)head_dim * (size_t)(zt::sm_count() * 2);
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
    const bool is_wide = wide(a, true);
    shape(a, is_wide, 2 * kBwdWarps, &P);
    fill(a, &P);
    blocks = bwd_blocks((int64_t)P.rows * P.split);
    launch(a, P, true, is_wide, blocks, s);
    if (int rc = zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope_backward launch")) return rc;
  }
  const unsigned grid = (unsigned)((2 * a->head_dim + 31) / 32);
  const float* part = static_cast<const float*>(a->workspace);
  if (a->weight_dtype == ZT_F32)
    qk_weight_kernel<ZT_F32><<<grid, 256, 0, s>>>(part, blocks, a->head_dim, static_cast<float*>(a->dq_weight),
                                                  static_cast<float*>(a->dk_weight));
  else if (a->weight_dtype == ZT_BF16)
    qk_weight_kernel<ZT_BF16><<<grid, 256, 0, s>>>(part, blocks, a->head_dim, static_cast<__nv_bfloat16*>(a->dq_weight),
                                                   static_cast<__nv_bfloat16*>(a->dk_weight));
  else
    qk_weight_kernel<ZT_F16><<<grid, 256, 0, s>>>(part, blocks, a->head_dim, static_cast<__half*>(a->dq_weight),
                                                  static_cast<__half*>(a->dk_weight));
  return zt::check_cuda(cudaGetLastError(), "zt_qk_norm_rope_backward: weight launch");
}

}  // extern "C"
