// Distillation from a teacher's top logits, on rows of logits: loss, and its gradient.
// For a row z of vocab logits, temperature T and the teacher's list (i_k, t_k):
//
//   q = softmax(z / T),  p = softmax over the list of t_k / T,  lse = log sum_v exp(z_v / T)
//   loss = T^2 sum_k p_k (log p_k - log q[i_k])
//   d loss / dz_v = T (q_v - sum over k with i_k = v of p_k),  d lse / dz_v = q_v / T
//
// Bandwidth is the bound: the forward reads each logit once, the backward reads it and
// writes its gradient, and zt_distill_rows_grad, whose row weights are known beforehand,
// holds the row in the shared memory of a CTA cluster and so reads and writes once in all.
// One more warp than those that stream the row reads the teacher's list, gathers the listed
// logits and does the list's arithmetic while the row passes by.
#include <math.h>

#include <mutex>

#include "zt_distill.cuh"
#include "zt_tc.cuh"

namespace {

using namespace zt::distill;
using zt::tc::cluster_rank;
using zt::tc::cluster_sync_all;
using zt::tc::peer_addr;

constexpr int kStream = 256;             // threads that stream the row
constexpr int kThreads = kStream + 32;   // and the list's warp
constexpr int kWarps = kStream / 32;
constexpr int kMaxCluster = 8;

struct RowsParams {
  const void* z;
  void* grad;
  TopList list;
  const float* g;      // [rows] gradient of the loss, or the row weights
  const float* g_lse;  // [rows] gradient of lse, or NULL
  float* loss;
  float* lse;
  float2* stats;       // [rows] (m, s); s = 0: no teacher
  int64_t ld, ld_grad;
  int32_t vocab, parts, part_len;   // CTAs of a row and the elements of each, a multiple of 16 bytes
  float c, temperature;
};

template <int DT> struct El;
template <> struct El<ZT_F32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <> struct El<ZT_BF16> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct El<ZT_F16> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float to(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// A CTA's elements [lo, hi) of a row: up to the first 16-byte boundary, whole 16-byte
// vectors, and the rest.
template <int DT> struct Span {
  using T = typename El<DT>::T;
  const T* row;
  int32_t lo, hi, body, n_vec;   // body: the first element of the vectors

  __device__ __forceinline__ Span(const T* r, int32_t lo_, int32_t hi_) : row(r), lo(lo_), hi(hi_) {
    constexpr int V = El<DT>::kVec;
    const int over = (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
    body = min(hi, lo + (over ? V - over : 0));
    n_vec = (hi - body) / V;
  }
  __device__ __forceinline__ const uint4* vec() const { return reinterpret_cast<const uint4*>(row + body); }
  __device__ __forceinline__ int32_t tail() const { return body + n_vec * El<DT>::kVec; }
};

template <int DT> __device__ __forceinline__ Span<DT> span_of(const RowsParams& P, const void* base, int64_t ld, int64_t row, int part) {
  const int lo = min(P.vocab, part * P.part_len), hi = min(P.vocab, lo + P.part_len);
  return Span<DT>(static_cast<const typename El<DT>::T*>(base) + row * ld, lo, hi);
}

// The block's (m, s): the stream warps' in warp order. All stream threads call it.
__device__ __forceinline__ void block_stat(Stat st, float c, Stat* red) {
  st = warp_merge(st, c);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = st;
}

__device__ __forceinline__ Stat total_of(const Stat* red, int n, float c) {
  Stat r = red[0];
  for (int i = 1; i < n; ++i) r = merge(r, red[i], c);
  return r;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// The parts' (m, s) of a row, merged in part order by every CTA of its cluster alike. `mine`
// is this CTA's, in shared memory; ends with all of them read.
__device__ __forceinline__ Stat cluster_stat(const Stat* mine, int parts, float c) {
  cluster_sync_all();
  Stat r{-INFINITY, 0.f};
  for (int i = 0; i < parts; ++i) {
    const uint32_t a = peer_addr(mine, (uint32_t)i);
    const Stat o{ld_cluster_f32(a), ld_cluster_f32(a + 4)};
    r = merge(r, o, c);
  }
  return r;
}

// (m, s) of a row's finished sum as it is kept: no finite logit, or an index that does not
// exist, makes the row NaN.
__device__ __forceinline__ Stat final_stat(Stat st, bool bad) {
  if (bad || st.m == -INFINITY) st.s = NAN;
  return st;
}

// The row's logits at the list's indices inside [lo, hi).
template <int DT>
__device__ __forceinline__ void gather(List& s, const typename El<DT>::T* row, int top, int32_t lo, int32_t hi) {
#pragma unroll 4
  for (int k = threadIdx.x & 31; k < top; k += 32) {
    const int32_t i = s.idx[k];
    s.z[k] = i >= lo && i < hi ? El<DT>::to(row[i]) : 0.f;
  }
}

template <int DT>
__global__ void __launch_bounds__(kThreads) distill_forward_kernel(const __grid_constant__ RowsParams P) {
  using T = typename El<DT>::T;
  constexpr int V = El<DT>::kVec, U = 4;
  __shared__ Stat red[kWarps];
  __shared__ Stat mine;
  __shared__ List list;
  __shared__ int none;   // this row has no teacher: its logits need not be read
  const int parts = P.parts;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts);
  const int tid = threadIdx.x;
  if (tid == 0) none = 0;
  __syncthreads();

  Teacher t;
  if (tid >= kStream) {
    t = read_list(list, P.list, row);
    if (!t.any && (tid & 31) == 0) *(volatile int*)&none = 1;
    if (part == 0) {
      gather<DT>(list, static_cast<const T*>(P.z) + row * P.ld, P.list.top, 0, P.vocab);
      list_softmax(list, P.list.top, P.c);
    }
  } else {
    const Span<DT> sp = span_of<DT>(P, P.z, P.ld, row, part);
    Stat st{-INFINITY, 0.f};
    const uint4* v = sp.vec();
    int i = tid;
    for (; i + (U - 1) * kStream < sp.n_vec; i += U * kStream) {
      uint4 u[U];
#pragma unroll
      for (int j = 0; j < U; ++j) u[j] = __ldcs(v + i + j * kStream);
      if (*(volatile int*)&none) break;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float f[V];
        El<DT>::unpack(u[j], f);
        absorb(st, f, P.c);
      }
    }
    for (; i < sp.n_vec; i += kStream) {
      if (*(volatile int*)&none) break;
      float f[V];
      El<DT>::unpack(__ldcs(v + i), f);
      absorb(st, f, P.c);
    }
    if (tid < sp.body - sp.lo) {
      const float f[1] = {El<DT>::to(sp.row[sp.lo + tid])};
      absorb(st, f, P.c);
    }
    if (tid < sp.hi - sp.tail()) {
      const float f[1] = {El<DT>::to(sp.row[sp.tail() + tid])};
      absorb(st, f, P.c);
    }
    block_stat(st, P.c, red);
  }
  __syncthreads();
  Stat st;
  if (parts > 1) {
    if (tid == 0) mine = total_of(red, kWarps, P.c);
    __syncwarp();
    st = cluster_stat(&mine, parts, P.c);
  } else if (tid >= kStream) {
    st = total_of(red, kWarps, P.c);
  }
  if (tid >= kStream && part == 0) {
    st = final_stat(st, t.bad);
    const float loss = list_loss(list, P.list.top, st, P.c, P.temperature);
    if ((tid & 31) == 0) {
      if (!t.any) st.s = 0.f;
      P.loss[row] = t.any ? (t.bad ? NAN : loss) : 0.f;
      P.lse[row] = t.any ? st.m / P.temperature + logf(st.s) : 0.f;
      if (P.stats) P.stats[row] = make_float2(st.m, st.s);
    }
  }
  if (parts > 1) cluster_sync_all();   // no CTA leaves while its sum may still be read
}

// The gradient at the listed indices is A q - B (the sum of p over the entries with that
// index): list_sums leaves that sum, in list order, in lp, and patch writes the gradient over
// the dense part's value there. Entries that share an index write the same value.
__device__ __forceinline__ void list_sums(List& s, int top) {
  __syncwarp();
  for (int k = threadIdx.x & 31; k < top; k += 32) {
    const int32_t own = s.idx[k];
    float a = 0.f;
#pragma unroll 8
    for (int j = 0; j < top; ++j) a += s.idx[j] == own ? s.p[j] : 0.f;
    s.lp[k] = a;
  }
}

template <int DT>
__device__ __forceinline__ void patch(const List& s, int top, const Stat& st, float A, float B, float c,
                                      typename El<DT>::T* grad, int32_t lo, int32_t hi) {
  for (int k = threadIdx.x & 31; k < top; k += 32) {
    const int32_t i = s.idx[k];
    if (i >= lo && i < hi) grad[i] = El<DT>::from(A * (ex2((s.z[k] - st.m) * c) / st.s) - B * s.lp[k]);
  }
}

// dz = a 2^((z - m) c) over a span; the gradient's row has its own 16-byte phase.
template <int DT> __device__ __forceinline__ float dense(float z, float m, float a, float c) { return a * ex2((z - m) * c); }

template <int DT>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const __grid_constant__ RowsParams P) {
  using T = typename El<DT>::T;
  constexpr int V = El<DT>::kVec, U = 4;
  // last rows first: those the forward read last may still be in L2
  const unsigned place = gridDim.x - 1 - blockIdx.x;
  const int64_t row = place / P.parts;
  const int part = (int)(place - row * P.parts);
  const int tid = threadIdx.x;
  const float2 s2 = P.stats[row];
  const Stat st{s2.x, s2.y};
  const Span<DT> sp = span_of<DT>(P, P.z, P.ld, row, part);
  T* out = static_cast<T*>(P.grad) + row * P.ld_grad;
  const bool none = st.s == 0.f;
  const float g = P.g ? P.g[row] : 0.f, gl = P.g_lse ? P.g_lse[row] : 0.f;
  const float B = g * P.temperature, A = B + gl / P.temperature;
  const bool in_place = P.grad == P.z;

  __shared__ List list;
  if (tid >= kStream && !none) {
    read_list(list, P.list, row);
    gather<DT>(list, sp.row, P.list.top, sp.lo, sp.hi);
    list_softmax(list, P.list.top, P.c);
    list_sums(list, P.list.top);
  }
  if (in_place) __syncthreads();   // the listed logits are read before they are overwritten
  if (tid < kStream) {
    const float a = A / st.s;
    const uint4* v = sp.vec();
    const bool same = ((uintptr_t)(out + sp.body) & 15) == 0;
    if (none) {
      for (int i = sp.lo + tid; i < sp.hi; i += kStream) out[i] = El<DT>::from(0.f);
    } else if (same) {
      uint4* o = reinterpret_cast<uint4*>(out + sp.body);
      int i = tid;
      for (; i + (U - 1) * kStream < sp.n_vec; i += U * kStream) {
        uint4 u[U];
#pragma unroll
        for (int j = 0; j < U; ++j) u[j] = __ldcs(v + i + j * kStream);
#pragma unroll
        for (int j = 0; j < U; ++j) {
          float f[V];
          El<DT>::unpack(u[j], f);
#pragma unroll
          for (int k = 0; k < V; ++k) f[k] = dense<DT>(f[k], st.m, a, P.c);
          __stcs(o + i + j * kStream, El<DT>::pack(f));
        }
      }
      for (; i < sp.n_vec; i += kStream) {
        float f[V];
        El<DT>::unpack(__ldcs(v + i), f);
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = dense<DT>(f[k], st.m, a, P.c);
        __stcs(o + i, El<DT>::pack(f));
      }
      if (tid < sp.body - sp.lo) out[sp.lo + tid] = El<DT>::from(dense<DT>(El<DT>::to(sp.row[sp.lo + tid]), st.m, a, P.c));
      if (tid < sp.hi - sp.tail())
        out[sp.tail() + tid] = El<DT>::from(dense<DT>(El<DT>::to(sp.row[sp.tail() + tid]), st.m, a, P.c));
    } else {
      for (int i = sp.lo + tid; i < sp.hi; i += kStream) out[i] = El<DT>::from(dense<DT>(El<DT>::to(sp.row[i]), st.m, a, P.c));
    }
  }
  __syncthreads();
  if (tid >= kStream && !none) patch<DT>(list, P.list.top, st, A, B, P.c, out, sp.lo, sp.hi);
}

// Loss and gradient at once: a cluster's CTAs hold the row, so it is read once. A thread
// copies its own vectors to shared memory (cp.async: no registers, no barrier), adds them up
// as they land, and after the cluster has merged its sums turns the same vectors into the
// gradient.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(zt::tc::smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int DT>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(const __grid_constant__ RowsParams P) {
  using T = typename El<DT>::T;
  constexpr int V = El<DT>::kVec, U = 2, D = 8;   // D groups of U vectors a thread in flight
  extern __shared__ uint4 held[];
  __shared__ Stat red[kWarps];
  __shared__ Stat mine;
  __shared__ List list;
  __shared__ int none, bad;   // no teacher; an index that does not exist
  const int parts = P.parts;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts);
  const int tid = threadIdx.x;
  const Span<DT> sp = span_of<DT>(P, P.z, P.ld, row, part);
  const uint4* v = sp.vec();
  if (tid < kStream) {   // the first groups are on their way before anything else
#pragma unroll
    for (int d = 0; d < D; ++d) {
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = tid + (d * U + j) * kStream;
        if (i < sp.n_vec) copy16(held + i, v + i);
      }
      copy_commit();
    }
  }
  if (tid == 0) none = 0;
  __syncthreads();

  float head = 0.f, tail = 0.f;   // the elements before and behind the vectors
  if (tid >= kStream) {
    const Teacher t = read_list(list, P.list, row);
    if ((tid & 31) == 0) {
      bad = t.bad;
      if (!t.any) *(volatile int*)&none = 1;
    }
    gather<DT>(list, static_cast<const T*>(P.z) + row * P.ld, P.list.top, 0, P.vocab);
    list_softmax(list, P.list.top, P.c);
  } else {
    Stat st{-INFINITY, 0.f};
    if (tid < sp.body - sp.lo) {
      head = El<DT>::to(sp.row[sp.lo + tid]);
      const float f[1] = {head};
      absorb(st, f, P.c);
    }
    if (tid < sp.hi - sp.tail()) {
      tail = El<DT>::to(sp.row[sp.tail() + tid]);
      const float f[1] = {tail};
      absorb(st, f, P.c);
    }
    for (int g = 0; g * U * kStream < sp.n_vec; ++g) {
      copy_wait<D - 1>();
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = tid + (g * U + j) * kStream;
        if (i < sp.n_vec) {
          float f[V];
          El<DT>::unpack(held[i], f);
          absorb(st, f, P.c);
        }
      }
      if (!*(volatile int*)&none) {
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const int i = tid + ((g + D) * U + j) * kStream;
          if (i < sp.n_vec) copy16(held + i, v + i);
        }
      }
      copy_commit();
    }
    copy_wait<0>();
    block_stat(st, P.c, red);
  }
  __syncthreads();
  Stat st;
  if (parts > 1) {
    if (tid == 0) mine = total_of(red, kWarps, P.c);
    __syncwarp();
    st = cluster_stat(&mine, parts, P.c);
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this thread has read the peers' sums
  } else {
    st = total_of(red, kWarps, P.c);
  }
  const float B = P.g[row] * P.temperature, A = B + (P.g_lse ? P.g_lse[row] / P.temperature : 0.f);
  T* out = static_cast<T*>(P.grad) + row * P.ld_grad;
  const bool any = !none;
  st = final_stat(st, bad);
  if (tid >= kStream) {
    if (part == 0) {
      const float loss = list_loss(list, P.list.top, st, P.c, P.temperature);
      if ((tid & 31) == 0) {
        P.loss[row] = any ? (bad ? NAN : loss) : 0.f;
        P.lse[row] = any ? st.m / P.temperature + logf(st.s) : 0.f;
      }
    }
    list_sums(list, P.list.top);   // after the loss: it takes the place of log2 p
  } else {
    const float a = A / st.s;
    const bool same = ((uintptr_t)(out + sp.body) & 15) == 0;
    if (!any) {
      for (int i = sp.lo + tid; i < sp.hi; i += kStream) out[i] = El<DT>::from(0.f);
    } else {
      uint4* o = reinterpret_cast<uint4*>(out + sp.body);
      for (int i = tid; i < sp.n_vec; i += kStream) {
        float f[V];
        El<DT>::unpack(held[i], f);
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = dense<DT>(f[k], st.m, a, P.c);
        if (same) {
          __stcs(o + i, El<DT>::pack(f));
        } else {
          T* e = out + sp.body + i * V;
#pragma unroll
          for (int k = 0; k < V; ++k) e[k] = El<DT>::from(f[k]);
        }
      }
      if (tid < sp.body - sp.lo) out[sp.lo + tid] = El<DT>::from(dense<DT>(head, st.m, a, P.c));
      if (tid < sp.hi - sp.tail()) out[sp.tail() + tid] = El<DT>::from(dense<DT>(tail, st.m, a, P.c));
    }
  }
  __syncthreads();
  if (tid >= kStream && any) patch<DT>(list, P.list.top, st, A, B, P.c, out, sp.lo, sp.hi);
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // no CTA leaves while its sum may be read
}

int check_rows(const zt_distill_args* a, bool grad, const std::string& who) {
  if (!a) return zt::set_error(ZT_ERR_INVALID, who + ": null arguments");
  if (a->rows < 0 || a->vocab <= 0 || a->ld < a->vocab || (grad && a->ld_grad < a->vocab))
    return zt::set_error(ZT_ERR_INVALID, who + ": bad shape");
  if (a->vocab > (int64_t)1 << 30) return zt::set_error(ZT_ERR_LIMIT, who + ": vocab above 2^30");
  if (a->rows > (int64_t)INT32_MAX / kMaxCluster) return zt::set_error(ZT_ERR_LIMIT, who + ": more than 2^28 - 1 rows");
  if (a->dtype != ZT_F32 && a->dtype != ZT_BF16 && a->dtype != ZT_F16)
    return zt::set_error(ZT_ERR_INVALID, who + ": unknown dtype");
  const bool empty = a->rows == 0;
  if (int rc = check_list(a->top_idx, a->top_logits, a->top, a->idx_bits, a->top_dtype, a->temperature, empty, who)) return rc;
  if (!empty && (!a->logits || (grad && !a->grad))) return zt::set_error(ZT_ERR_INVALID, who + ": null pointer");
  const uintptr_t esz = a->dtype == ZT_F32 ? 4 : 2;
  if (((uintptr_t)a->logits | (uintptr_t)(grad ? a->grad : nullptr)) & (esz - 1))
    return zt::set_error(ZT_ERR_INVALID, who + ": logits and their gradient must be aligned to their elements");
  if (grad && a->grad == a->logits && a->ld_grad != a->ld)
    return zt::set_error(ZT_ERR_INVALID, who + ": in place, the row strides must be equal");
  return ZT_OK;
}

// CTAs of a row: 1 where the rows alone fill the SMs twice, else the power of two up to 8
// that does, while a part still has kMinPart elements (below that a part is all latency).
constexpr int kMinPart = 2048;

int parts_for(int64_t rows, int64_t vocab) {
  const int64_t want = 2 * (int64_t)zt::sm_count();
  int parts = 1;
  while (parts < kMaxCluster && rows * parts < want && vocab / (2 * parts) >= kMinPart) parts *= 2;
  return parts;
}

RowsParams rows_params(const zt_distill_args* a, int parts) {
  RowsParams P = {};
  P.z = a->logits;
  P.grad = a->grad;
  P.list = TopList{a->top_idx, a->top_logits, a->top, a->idx_bits == 64, a->top_dtype, a->vocab};
  P.g = a->weight;
  P.g_lse = a->weight_lse;
  P.loss = a->loss;
  P.lse = a->lse;
  P.stats = reinterpret_cast<float2*>(a->stats);
  P.ld = a->ld;
  P.ld_grad = a->ld_grad;
  P.vocab = (int32_t)a->vocab;
  P.parts = parts;
  P.part_len = (int32_t)(((a->vocab + parts - 1) / parts + 7) / 8 * 8);
  P.c = kLog2e / a->temperature;
  P.temperature = a->temperature;
  return P;
}

template <class K> int launch(K kernel, const RowsParams& P, int64_t rows, bool cluster, size_t smem, cudaStream_t s, const char* who) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * P.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr = {};
  if (cluster && P.parts > 1) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)P.parts;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  return zt::check_cuda(cudaLaunchKernelEx(&cfg, kernel, P), who);
}

int forward(const zt_distill_args* a, cudaStream_t s, const char* who) {
  const RowsParams P = rows_params(a, parts_for(a->rows, a->vocab));
  if (a->dtype == ZT_BF16) return launch(distill_forward_kernel<ZT_BF16>, P, a->rows, true, 0, s, who);
  if (a->dtype == ZT_F16) return launch(distill_forward_kernel<ZT_F16>, P, a->rows, true, 0, s, who);
  return launch(distill_forward_kernel<ZT_F32>, P, a->rows, true, 0, s, who);
}

int backward(const zt_distill_args* a, cudaStream_t s, const char* who) {
  const RowsParams P = rows_params(a, parts_for(a->rows, a->vocab));
  if (a->dtype == ZT_BF16) return launch(distill_backward_kernel<ZT_BF16>, P, a->rows, false, 0, s, who);
  if (a->dtype == ZT_F16) return launch(distill_backward_kernel<ZT_F16>, P, a->rows, false, 0, s, who);
  return launch(distill_backward_kernel<ZT_F32>, P, a->rows, false, 0, s, who);
}

// A part of distill_grad_kernel's row in shared memory: 64 KB leave room for three CTAs on an
// SM, whose loads, sums and stores overlap; longer rows take up to kMaxPart in each of
// eight parts, and rows beyond that the forward and the backward kernel.
constexpr size_t kGoodPart = 64 * 1024;
constexpr size_t kMaxPart = 200 * 1024;

size_t part_bytes(const zt_distill_args* a, int parts) {
  const size_t len = (size_t)(((a->vocab + parts - 1) / parts + 7) / 8 * 8);
  return len * (a->dtype == ZT_F32 ? 4 : 2);
}

template <int DT> int grad_once(const RowsParams& P, int64_t rows, size_t smem, cudaStream_t s) {
  static std::mutex mu;
  static bool ready[64] = {false};
  int dev = 0;
  if (int rc = zt::check_cuda(cudaGetDevice(&dev), "zt_distill_rows_grad: cudaGetDevice")) return rc;
  if (dev < 0 || dev >= 64) return zt::set_error(ZT_ERR_LIMIT, "zt_distill_rows_grad: device ordinal >= 64");
  {
    std::lock_guard<std::mutex> lock(mu);
    if (!ready[dev]) {
      if (int rc = zt::check_cuda(cudaFuncSetAttribute(distill_grad_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)kMaxPart), "zt_distill_rows_grad: shared memory attribute"))
        return rc;
      ready[dev] = true;
    }
  }
  return launch(distill_grad_kernel<DT>, P, rows, true, smem, s, "zt_distill_rows_grad launch");
}

}  // namespace

extern "C" {

int zt_distill_rows(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, false, "zt_distill_rows")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->loss || !a->lse) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows: null pointer");
  return forward(a, zt::as_stream(stream), "zt_distill_rows launch");
}

int zt_distill_rows_backward(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, true, "zt_distill_rows_backward")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->stats) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows_backward: null pointer");
  return backward(a, zt::as_stream(stream), "zt_distill_rows_backward launch");
}

int zt_distill_rows_grad(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, true, "zt_distill_rows_grad")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->loss || !a->lse || !a->stats || !a->weight) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows_grad: null pointer");
  int parts = parts_for(a->rows, a->vocab);
  while (parts < kMaxCluster && part_bytes(a, parts) > kGoodPart) parts *= 2;
  const size_t smem = part_bytes(a, parts);
  cudaStream_t s = zt::as_stream(stream);
  if (smem > kMaxPart) {   // the row does not fit a cluster's shared memory
    if (int rc = forward(a, s, "zt_distill_rows_grad launch")) return rc;
    return backward(a, s, "zt_distill_rows_grad launch");
  }
  const RowsParams P = rows_params(a, parts);
  if (a->dtype == ZT_BF16) return grad_once<ZT_BF16>(P, a->rows, smem, s);
  if (a->dtype == ZT_F16) return grad_once<ZT_F16>(P, a->rows, smem, s);
  return grad_once<ZT_F32>(P, a->rows, smem, s);
}

}  // extern "C"
