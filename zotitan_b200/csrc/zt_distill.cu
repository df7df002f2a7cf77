// Distillation from a teacher's top logits, on rows of logits: loss, and its gradient.
// For a row z of vocab logits, temperature T and the teacher's list (i_k, t_k):
//
//   q = softmax(z / T),  p = softmax over the list of t_k / T,  lse = log sum_v exp(z_v / T)
//   loss = T^2 sum_k p_k (log p_k - log q[i_k])
//   d loss / dz_v = T (q_v - sum over k with i_k = v of p_k),  d lse / dz_v = q_v / T
//
// Bandwidth is the bound: the forward reads each logit once, the backward reads it and
// writes its gradient, and zt_distill_rows_grad, whose row weights are known beforehand, does
// both while the row is still in L2, so that memory is read and written once in all.
// A CTA takes a row, or with few rows a cluster of CTAs does, merging their sums over
// distributed shared memory. One more warp than those that stream the row reads the teacher's
// list, gathers the listed logits and does the list's arithmetic while the row passes by.
#include <math.h>

#include "zt_distill.cuh"
#include "zt_tc.cuh"

namespace {

using namespace zt::distill;
using zt::tc::cluster_rank;
using zt::tc::cluster_sync_all;
using zt::tc::peer_addr;

// Threads that stream a row, beside the list's warp, and the CTAs of an SM that the compiler is asked
// for. A thread's step is two vectors in the forward and four elsewhere. The forward lives on warps: of
// 4096 x 128256 bf16 it takes 180 us with six CTAs of two vectors, 184 with four of four, 199 to
// 226 where a thread also loads its next step ahead (its registers cost warps). Asked for six it
// takes 32 registers (the 16-bit ones spill six of them), with which seven are resident; the rules below
// count six.
constexpr int kSumThreads = 256, kSumCtas = 6, kSumStep = 2;
// The backward, and loss and gradient at once: rows of up to kMidRow bytes go to CTAs half as wide,
// twice as many (4000 x 32000 bf16, 64 KB: 117 us so, 152 with the wide ones; 2048 x 100000, 200 KB:
// 189 and 179).
constexpr int kWriteStep = 4;
constexpr int kWideThreads = 512, kWideCtas = 2, kMidThreads = 256, kMidCtas = 4;
constexpr int64_t kMidRow = 112 * 1024;
constexpr int kRowWarps = 8;         // rows of a block where a warp takes a row
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
  template <int U> static __device__ __forceinline__ float max_of(const uint4 (&u)[U]) {   // NaN aside
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float f[4];
      unpack(u[i], f);
      m = fmaxf(m, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])));
    }
    return m;
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
  template <int U> static __device__ __forceinline__ float max_of(const uint4 (&u)[U]) {   // NaN aside, two at a time
    using P2 = __nv_bfloat162;
    auto two = [](const uint32_t& w) { return *reinterpret_cast<const P2*>(&w); };
    P2 m = __hmax2(__hmax2(two(u[0].x), two(u[0].y)), __hmax2(two(u[0].z), two(u[0].w)));
#pragma unroll
    for (int i = 1; i < U; ++i)
      m = __hmax2(m, __hmax2(__hmax2(two(u[i].x), two(u[i].y)), __hmax2(two(u[i].z), two(u[i].w))));
    return fmaxf(__bfloat162float(__low2bfloat16(m)), __bfloat162float(__high2bfloat16(m)));
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
  template <int U> static __device__ __forceinline__ float max_of(const uint4 (&u)[U]) {   // NaN aside, two at a time
    using P2 = __half2;
    auto two = [](const uint32_t& w) { return *reinterpret_cast<const P2*>(&w); };
    P2 m = __hmax2(__hmax2(two(u[0].x), two(u[0].y)), __hmax2(two(u[0].z), two(u[0].w)));
#pragma unroll
    for (int i = 1; i < U; ++i)
      m = __hmax2(m, __hmax2(__hmax2(two(u[i].x), two(u[i].y)), __hmax2(two(u[i].z), two(u[i].w))));
    return fmaxf(__half2float(__low2half(m)), __half2float(__high2half(m)));
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

// Step g of S threads, U vectors each, over a span; 2^((-inf - m) c) = 0 stands in for what is beyond.
template <int DT, int S, int U>
__device__ __forceinline__ void load_step(uint4 (&u)[U], const Span<DT>& sp, int tid, int g, bool again) {
  const int i = tid + g * (U * S);
  const uint4* v = sp.vec() + i;
  if ((g + 1) * (U * S) <= sp.n_vec) {
#pragma unroll
    for (int j = 0; j < U; ++j) u[j] = again ? __ldcg(v + j * S) : __ldcs(v + j * S);
  } else {
    const uint32_t w = DT == ZT_F32 ? 0xff800000u : DT == ZT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      u[j] = make_uint4(w, w, w, w);
      if (i + j * S < sp.n_vec) u[j] = again ? __ldcg(v + j * S) : __ldcs(v + j * S);
    }
  }
}

template <int DT, int S, int U> __device__ __forceinline__ int steps_of(const Span<DT>& sp) { return (sp.n_vec + U * S - 1) / (U * S); }

template <int DT, int U> __device__ __forceinline__ void absorb_step(Stat& st, const uint4 (&u)[U], float c) {
  constexpr int V = El<DT>::kVec;
  float f[U * V];
#pragma unroll
  for (int j = 0; j < U; ++j) {
    float g[V];
    El<DT>::unpack(u[j], g);
#pragma unroll
    for (int k = 0; k < V; ++k) f[j * V + k] = g[k];
  }
  absorb(st, f, El<DT>::max_of(u), c);
}

// Thread tid's share of a span's sum; gives up once the row is known to have no teacher (where
// `none` is watched). `again`: the span will be read once more and should stay in L2.
template <int DT, int S, int U>
__device__ __forceinline__ Stat sum_span(const Span<DT>& sp, int tid, float c, const volatile int* none, bool again) {
  Stat st{-INFINITY, 0.f};
  const int n = steps_of<DT, S, U>(sp);
  uint4 u[U];
  for (int g = 0; g < n; ++g) {
    load_step<DT, S, U>(u, sp, tid, g, again);
    if (none && *none) break;
    absorb_step<DT, U>(st, u, c);
  }
  if (tid < sp.body - sp.lo) {
    const float f[1] = {El<DT>::to(sp.row[sp.lo + tid])};
    absorb(st, f, c);
  }
  if (tid < sp.hi - sp.tail()) {
    const float f[1] = {El<DT>::to(sp.row[sp.tail() + tid])};
    absorb(st, f, c);
  }
  return st;
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// What the CTAs of a row share, and a CTA's threads.
template <int S> struct Shared {
  unsigned long long list[kMaxTop * List::kBytes / 8];
  Stat red[S / 32];   // the warps' sums
  Stat mine, total;   // this CTA's, the row's
  int none, bad;      // no teacher: the row's logits need not be read; a list that makes the row NaN
};

// The list's warp: the row's finished sum from the stream warps' and, over the cluster, the
// parts'. Every CTA of a cluster merges alike. The block is in step before and after.
template <int S> __device__ __forceinline__ void finish_sum(Shared<S>& sh, int parts, float c) {
  const int lane = threadIdx.x & 31;
  const bool list_warp = threadIdx.x >= S;
  __syncthreads();
  if (list_warp) {
    Stat st = lane < S / 32 ? sh.red[lane] : Stat{-INFINITY, 0.f};
    st = warp_merge(st, c);
    if (lane == 0) sh.mine = st;
    __syncwarp();
  }
  if (parts > 1) {
    cluster_sync_all();
    if (list_warp) {
      Stat st{-INFINITY, 0.f};
      if (lane < parts) {
        const uint32_t a = peer_addr(&sh.mine, (uint32_t)lane);
        st = Stat{ld_cluster_f32(a), ld_cluster_f32(a + 4)};
      }
      st = warp_merge(st, c);
      if (lane == 0) sh.total = st;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // the peers' sums are read
  } else if (list_warp && lane == 0) {
    sh.total = sh.mine;
  }
  __syncthreads();
}

// No CTA leaves while a peer may still read its sum.
__device__ __forceinline__ void leave(int parts) {
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// (m, s) of a row's finished sum as it is kept: no finite logit, or a list with an index that does not
// exist or a value that is no number, makes the row NaN.
__device__ __forceinline__ Stat final_stat(Stat st, bool bad) {
  if (bad || st.m == -INFINITY) st.s = NAN;
  return st;
}

// The row's logits at the list's indices inside [lo, hi).
template <int DT>
__device__ __forceinline__ void gather(const List& s, const typename El<DT>::T* row, int top, int32_t lo, int32_t hi) {
#pragma unroll 4
  for (int k = threadIdx.x & 31; k < top; k += 32) {
    const int32_t i = s.idx[k];
    s.z[k] = i >= lo && i < hi ? El<DT>::to(row[i]) : 0.f;
  }
}

// The list's warp before the sum is there: reads the list, gathers its logits in [lo, hi), and
// the teacher's probabilities.
template <int DT, int S>
__device__ __forceinline__ void prepare_list(Shared<S>& sh, const RowsParams& P, int64_t row, int32_t lo, int32_t hi) {
  const List list(sh.list, kMaxTop);
  const Teacher t = read_list(list, P.list, row);
  if ((threadIdx.x & 31) == 0) {
    sh.bad = t.bad;
    if (!t.any) *(volatile int*)&sh.none = 1;
  }
  gather<DT>(list, static_cast<const typename El<DT>::T*>(P.z) + row * P.ld, P.list.top, lo, hi);
  list_softmax(list, P.list.top, P.c);
}

// and after: loss, lse and what the backward needs.
__device__ __forceinline__ void write_loss(const List& list, const RowsParams& P, int64_t row, Stat st, bool none, bool bad) {
  const float loss = list_loss(list, P.list.top, st, P.c, P.temperature);
  if ((threadIdx.x & 31) == 0) {
    P.loss[row] = none ? 0.f : bad ? NAN : loss;
    P.lse[row] = none ? 0.f : sum_lse(st, P.c, P.temperature);
    if (P.stats) P.stats[row] = make_float2(st.m, none ? 0.f : st.s);
  }
}

template <int DT>
__global__ void __launch_bounds__(kSumThreads + 32, kSumCtas) distill_forward_kernel(const __grid_constant__ RowsParams P) {
  constexpr int S = kSumThreads;
  __shared__ Shared<S> sh;
  const int parts = P.parts;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts);
  const int tid = threadIdx.x;
  if (tid == 0) sh.none = 0;
  __syncthreads();
  if (tid >= S) {
    prepare_list<DT>(sh, P, row, 0, P.vocab);
  } else {
    const Stat st = warp_merge(sum_span<DT, S, kSumStep>(span_of<DT>(P, P.z, P.ld, row, part), tid, P.c, &sh.none, false), P.c);
    if ((tid & 31) == 0) sh.red[tid / 32] = st;
  }
  finish_sum<S>(sh, parts, P.c);
  if (tid >= S && part == 0)
    write_loss(List(sh.list, kMaxTop), P, row, final_stat(sh.total, sh.bad), sh.none, sh.bad);
  leave(parts);
}

// Whether all indices of a list differ, by a hash table in the place of `order`, half full at most.
__device__ __forceinline__ bool list_distinct(const List& s, int top) {
  const int lane = threadIdx.x & 31, size = 2 * list_capacity(top);
  int32_t* table = reinterpret_cast<int32_t*>(s.order);
  for (int q = lane; q < size; q += 32) table[q] = -1;
  __syncwarp();
  bool twice = false;
  for (int k = lane; k < top; k += 32) {
    const int32_t own = s.idx[k];
    if (own < 0) continue;
    uint32_t at = (uint32_t)own * 2654435761u >> 16;   // Knuth's multiplicative hashing
    for (;; ++at) {
      const int32_t was = atomicCAS(table + (at & (size - 1)), -1, own);
      if (was == -1) break;
      if (was == own) {
        twice = true;
        break;
      }
    }
  }
  twice = __any_sync(0xffffffffu, twice);
  __syncwarp();
  return !twice;
}

// The gradient at the listed indices is A q - B (the sum of p over the entries with that
// index): list_sums leaves that sum, in list order, in lp, and patch writes the gradient over
// the dense part's value there. Entries that share an index write the same value. Teachers' lists
// seldom hold an index twice: only then are they sorted.
__device__ __forceinline__ void list_sums(const List& s, int top) {
  const int lane = threadIdx.x & 31;
  if (list_distinct(s, top)) {
    for (int k = lane; k < top; k += 32) s.lp[k] = s.p[k];
    return;
  }
  list_sort(s, top, [](int32_t idx) { return (uint32_t)idx; });
  for (int q = lane; q < top; q += 32) {
    const uint32_t own = (uint32_t)(s.order[q] >> 32);
    if (own == 0xffffffffu) break;   // no mass from here on
    int first = q;   // equal indices stand together, in list order
    while (first > 0 && (uint32_t)(s.order[first - 1] >> 32) == own) --first;
    float a = 0.f;
    for (int r = first; r < top && (uint32_t)(s.order[r] >> 32) == own; ++r) a += s.p[(uint32_t)s.order[r]];
    s.lp[(uint32_t)s.order[q]] = a;
  }
  __syncwarp();
}

template <int DT>
__device__ __forceinline__ void patch(const List& s, int top, const Stat& st, float A, float B, float c,
                                      typename El<DT>::T* grad, int32_t lo, int32_t hi) {
  const Base base(st.m, c);
  for (int k = threadIdx.x & 31; k < top; k += 32) {
    const int32_t i = s.idx[k];
    if (i >= lo && i < hi) grad[i] = El<DT>::from(A * (ex2(base.rel(s.z[k], c)) / st.s) - B * s.lp[k]);
  }
}

// The dense part of a row's gradient, dz = a 2^((z - m) c) with a = A / s. For 16-bit gradients
// |a| goes into the exponent, 2^(z c + k) with k = log2 |a| - mc, and the sign onto the rounded
// pair: a multiplication less. Rounding k costs 2^-24 |k| of the result, so only where |mc| is at most
// 64 (4e-6, a hundredth of fp16's half step).
template <int DT> struct Dense {
  static constexpr int V = El<DT>::kVec;
  Base base;
  float a, k;
  uint32_t sign;
  bool fold;

  __device__ __forceinline__ Dense(const Stat& st, float A, float c) : base(st.m, c), a(A / st.s), k(0.f), sign(0), fold(false) {
    if (DT != ZT_F32) {
      if (a < 0.f) sign = 0x80008000u;   // the paired sign bits
      a = fabsf(a);
      k = log2f(a) - base.mc;
      fold = fabsf(base.mc) <= 64.f;
    }
  }
  __device__ __forceinline__ typename El<DT>::T one(typename El<DT>::T z, float c) const {
    const float v = fold ? ex2(__fmaf_rn(El<DT>::to(z), c, k)) : a * ex2(base.rel(El<DT>::to(z), c));
    return El<DT>::from(sign ? -v : v);
  }
  template <bool FOLD> __device__ __forceinline__ uint4 vec(const uint4& u, float c) const {
    float f[V];
    El<DT>::unpack(u, f);
    if (FOLD) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = ex2(__fmaf_rn(f[i], c, k));
    } else if (!base.far()) {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = a * ex2(__fmaf_rn(f[i], c, -base.mc));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = a * ex2((f[i] - base.m) * c);
    }
    uint4 r = El<DT>::pack(f);
    if (DT != ZT_F32) {
      r.x ^= sign; r.y ^= sign; r.z ^= sign; r.w ^= sign;
    }
    return r;
  }
};

// The vectors of a row's gradient over a span; `u` holds step 0, loaded before the caller waited
// for anything, and each step is loaded before the one before it is written. SAME: the gradient's
// vectors are as aligned as the logits'.
template <int DT, int S, int U, bool FOLD, bool SAME>
__device__ __forceinline__ void write_vecs(uint4 (&u)[U], const Span<DT>& sp, int tid, typename El<DT>::T* out, const Dense<DT>& D,
                                           float c) {
  using T = typename El<DT>::T;
  constexpr int V = El<DT>::kVec;
  const int n = steps_of<DT, S, U>(sp);
  int i = tid;
  T* o = out + sp.body + i * V;
  uint4 next[U];
  for (int g = 0; g < n; ++g) {
    if (g + 1 < n) load_step<DT, S, U>(next, sp, tid, g + 1, false);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const uint4 r = D.template vec<FOLD>(u[j], c);
      if (i + j * S < sp.n_vec) {
        if (SAME) {
          __stcs(reinterpret_cast<uint4*>(o) + j * S, r);
        } else {   // an element at a time; in place this cannot be
          const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
          for (int k = 0; k < V; ++k) o[j * S * V + k] = e[k];
        }
      }
      u[j] = next[j];
    }
    i += U * S;
    o += U * S * V;
  }
}

// The stream threads' part of a row's gradient over a span. out has its own 16-byte phase.
template <int DT, int S, int U>
__device__ __forceinline__ void write_span(uint4 (&u)[U], const Span<DT>& sp, int tid, typename El<DT>::T* out, const Dense<DT>& D,
                                           float c) {
  if (((uintptr_t)(out + sp.body) & 15) != 0) write_vecs<DT, S, U, false, false>(u, sp, tid, out, D, c);
  else if (DT != ZT_F32 && D.fold) write_vecs<DT, S, U, true, true>(u, sp, tid, out, D, c);
  else write_vecs<DT, S, U, false, true>(u, sp, tid, out, D, c);
  if (tid < sp.body - sp.lo) out[sp.lo + tid] = D.one(sp.row[sp.lo + tid], c);
  if (tid < sp.hi - sp.tail()) out[sp.tail() + tid] = D.one(sp.row[sp.tail() + tid], c);
}

// The gradient of a row without a teacher.
template <int DT, int S>
__device__ __forceinline__ void zero_span(typename El<DT>::T* out, int tid, int32_t lo, int32_t hi) {
  const Span<DT> o(out, lo, hi);
  const typename El<DT>::T zero = El<DT>::from(0.f);
  uint4* v = reinterpret_cast<uint4*>(out + o.body);
  for (int i = tid; i < o.n_vec; i += S) v[i] = make_uint4(0, 0, 0, 0);
  if (tid < o.body - o.lo) out[o.lo + tid] = zero;
  if (tid < o.hi - o.tail()) out[o.tail() + tid] = zero;
}

template <int DT, int S, int CTAS>
__global__ void __launch_bounds__(S + 32, CTAS) distill_backward_kernel(const __grid_constant__ RowsParams P) {
  using T = typename El<DT>::T;
  constexpr int U = kWriteStep;
  __shared__ unsigned long long list_room[kMaxTop * List::kBytes / 8];
  const List list(list_room, kMaxTop);
  // last rows first: those the forward read last may still be in L2
  const unsigned place = gridDim.x - 1 - blockIdx.x;
  const int64_t row = place / P.parts;
  const int part = (int)(place - row * P.parts);
  const int tid = threadIdx.x;
  const Span<DT> sp = span_of<DT>(P, P.z, P.ld, row, part);
  uint4 u[U];
  if (tid < S) load_step<DT, S, U>(u, sp, tid, 0, false);
  const float2 s2 = P.stats[row];
  const Stat st{s2.x, s2.y};
  T* out = static_cast<T*>(P.grad) + row * P.ld_grad;
  const bool none = st.s == 0.f;
  const float B = (P.g ? P.g[row] : 0.f) * P.temperature, A = B + (P.g_lse ? P.g_lse[row] / P.temperature : 0.f);
  if (tid >= S && !none) {
    read_list(list, P.list, row);
    gather<DT>(list, sp.row, P.list.top, sp.lo, sp.hi);
    list_softmax(list, P.list.top, P.c);
    list_sums(list, P.list.top);
  }
  if (P.grad == P.z) __syncthreads();   // in place: the listed logits are read before they are overwritten
  if (tid < S) {
    if (none) zero_span<DT, S>(out, tid, sp.lo, sp.hi);
    else write_span<DT, S, U>(u, sp, tid, out, Dense<DT>(st, A, P.c), P.c);
  }
  __syncthreads();
  if (tid >= S && !none) patch<DT>(list, P.list.top, st, A, B, P.c, out, sp.lo, sp.hi);
}

// Loss and gradient at once: the sum reads the row from memory, the gradient reads it again from
// L2. (Held in the shared memory of a cluster of four instead, the row's loads, sums and
// stores took turns: 2048 x 128256 bf16 257 us, so 223 with the same inner loop; 213 with the
// unpredicated steps that came later, with which the other form was not measured.)
template <int DT, int S, int CTAS>
__global__ void __launch_bounds__(S + 32, CTAS) distill_grad_kernel(const __grid_constant__ RowsParams P) {
  using T = typename El<DT>::T;
  constexpr int U = kWriteStep;
  __shared__ Shared<S> sh;
  const int parts = P.parts;
  const int64_t row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x - row * parts);
  const int tid = threadIdx.x;
  const Span<DT> sp = span_of<DT>(P, P.z, P.ld, row, part);
  if (tid == 0) sh.none = 0;
  __syncthreads();
  const List list(sh.list, kMaxTop);
  uint4 u[U];
  if (tid >= S) {
    prepare_list<DT>(sh, P, row, 0, P.vocab);   // in place: all of it before any part writes
  } else {
    const Stat st = warp_merge(sum_span<DT, S, U>(sp, tid, P.c, &sh.none, true), P.c);
    if ((tid & 31) == 0) sh.red[tid / 32] = st;
    load_step<DT, S, U>(u, sp, tid, 0, false);
  }
  finish_sum<S>(sh, parts, P.c);
  const bool none = sh.none;
  const Stat st = final_stat(sh.total, sh.bad);
  const float B = P.g[row] * P.temperature, A = B + (P.g_lse ? P.g_lse[row] / P.temperature : 0.f);
  T* out = static_cast<T*>(P.grad) + row * P.ld_grad;
  if (tid >= S) {
    if (part == 0) write_loss(list, P, row, st, none, sh.bad);
    list_sums(list, P.list.top);   // after the loss: it takes the place of log2 p
  } else if (none) {
    zero_span<DT, S>(out, tid, sp.lo, sp.hi);
  } else {
    write_span<DT, S, U>(u, sp, tid, out, Dense<DT>(st, A, P.c), P.c);
  }
  __syncthreads();
  if (tid >= S && !none) patch<DT>(list, P.list.top, st, A, B, P.c, out, sp.lo, sp.hi);
  leave(parts);
}

// Many short rows: a warp takes a row by itself, list and all. SUM: forward; WRITE: backward;
// both: loss and gradient at once. (A CTA's start, its list and its end take about 5 us whatever
// the row's length, and an SM has two to six CTAs under way, but 16 to 32 of these warps.)
template <int DT, bool SUM, bool WRITE>
__global__ void __launch_bounds__(32 * kRowWarps) distill_warp_kernel(const __grid_constant__ RowsParams P, int64_t rows, int cap) {
  using T = typename El<DT>::T;
  constexpr int U = 4;
  extern __shared__ unsigned long long room[];
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + warp;
  if (row >= rows) return;
  const List list(room + (size_t)warp * cap * (List::kBytes / 8), cap);
  const Span<DT> sp(static_cast<const T*>(P.z) + row * P.ld, 0, P.vocab);
  T* out = WRITE ? static_cast<T*>(P.grad) + row * P.ld_grad : nullptr;
  Stat st{0.f, 0.f};
  bool none;
  if (SUM) {
    const Teacher t = read_list(list, P.list, row);
    none = !t.any;
    if (none) {
      if (lane == 0) {
        P.loss[row] = P.lse[row] = 0.f;
        if (P.stats) P.stats[row] = make_float2(0.f, 0.f);
      }
    } else {
      gather<DT>(list, sp.row, P.list.top, 0, P.vocab);
      st = warp_merge(sum_span<DT, 32, U>(sp, lane, P.c, nullptr, WRITE), P.c);
      st.m = __shfl_sync(0xffffffffu, st.m, 0);
      st.s = __shfl_sync(0xffffffffu, st.s, 0);
      st = final_stat(st, t.bad);
      list_softmax(list, P.list.top, P.c);
      write_loss(list, P, row, st, false, t.bad);
    }
  } else {
    const float2 s2 = P.stats[row];
    st = Stat{s2.x, s2.y};
    none = st.s == 0.f;
    if (!none) {
      read_list(list, P.list, row);
      gather<DT>(list, sp.row, P.list.top, 0, P.vocab);
      list_softmax(list, P.list.top, P.c);
    }
  }
  if (!WRITE) return;
  if (none) {
    zero_span<DT, 32>(out, lane, 0, P.vocab);
    return;
  }
  uint4 u[U];
  load_step<DT, 32, U>(u, sp, lane, 0, false);
  const float B = (P.g ? P.g[row] : 0.f) * P.temperature, A = B + (P.g_lse ? P.g_lse[row] / P.temperature : 0.f);
  list_sums(list, P.list.top);   // in place: its logits have been gathered
  write_span<DT, 32, U>(u, sp, lane, out, Dense<DT>(st, A, P.c), P.c);
  __syncwarp();
  patch<DT>(list, P.list.top, st, A, B, P.c, out, 0, P.vocab);
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

// CTAs of a row: doubled up to 8 while all of them still run at once, and a part keeps at least
// kMinPart elements. (Splitting rows that fill the GPU's slots already, to even out their last
// wave, costs more than it gives: 1001 x 50257 fp16 forward 34 us in two parts, 27 in one.)
constexpr int64_t kMinPart = 2048;

int parts_for(const zt_distill_args* a, int ctas) {
  const int64_t slots = (int64_t)zt::sm_count() * ctas;
  int parts = 1;
  while (parts < kMaxCluster && 2 * parts * a->rows <= slots && a->vocab / (2 * parts) >= kMinPart) parts *= 2;
  return parts;
}

int64_t row_bytes(const zt_distill_args* a) { return a->vocab * (a->dtype == ZT_F32 ? 4 : 2); }

// The same for loss and gradient at once, whose rows under way have to stay in L2 between their
// two readings: at most kInFlight bytes of them (2048 x 128256 fp32, 152 MB under way 450 us, in
// two parts 424; 1500 x 200000 bf16, 118 MB: 263, in two parts 278).
constexpr int64_t kInFlight = 128ll << 20;

int parts_for_grad(const zt_distill_args* a, int ctas) {
  const int64_t slots = (int64_t)zt::sm_count() * ctas;
  int parts = parts_for(a, ctas);
  while (parts < kMaxCluster && slots / parts * row_bytes(a) > kInFlight && a->rows * parts >= slots) parts *= 2;
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

template <class K>
int launch(K kernel, int threads, const RowsParams& P, int64_t rows, bool cluster, cudaStream_t s, const char* who) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * P.parts));
  cfg.blockDim = dim3((unsigned)threads);
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

// Whether a warp takes a row by itself: rows of at most `most` bytes, where the CTAs would need more
// waves than there are 8 KB in a row (a wave of short rows takes about 5 us, a warp's row 4 us
// and 6 for each 8 KB). Measured on 64 entries of bf16, a warp against a CTA a row: forward
// 8000 x 20000 74 and 84 us; backward 2000 x 8000 21.2 and 21.6, 2000 x 12000 28 and 25; loss and
// gradient 8000 x 12000 122 and 147, 4000 x 16000 82 and 77.
constexpr int64_t kShortSum = 48 * 1024, kShortWrite = 16 * 1024, kShortGrad = 24 * 1024, kShortStep = 8 * 1024;

bool short_rows(const zt_distill_args* a, int64_t most, int ctas) {
  const int64_t bytes = row_bytes(a), slots = (int64_t)zt::sm_count() * ctas;
  return bytes <= most && a->rows * kShortStep > slots * (bytes > kShortStep ? bytes : kShortStep);
}

template <int DT, bool SUM, bool WRITE>
int launch_warps(const zt_distill_args* a, cudaStream_t s, const char* who) {
  const int cap = list_capacity(a->top);
  distill_warp_kernel<DT, SUM, WRITE><<<(unsigned)((a->rows + kRowWarps - 1) / kRowWarps), 32 * kRowWarps,
                                       (size_t)kRowWarps * cap * List::kBytes, s>>>(rows_params(a, 1), a->rows, cap);
  return zt::check_cuda(cudaGetLastError(), who);
}

template <bool SUM, bool WRITE> int launch_warps(const zt_distill_args* a, cudaStream_t s, const char* who) {
  if (a->dtype == ZT_BF16) return launch_warps<ZT_BF16, SUM, WRITE>(a, s, who);
  if (a->dtype == ZT_F16) return launch_warps<ZT_F16, SUM, WRITE>(a, s, who);
  return launch_warps<ZT_F32, SUM, WRITE>(a, s, who);
}

template <int DT> int launch_backward(const zt_distill_args* a, cudaStream_t s) {
  const char* who = "zt_distill_rows_backward launch";
  if (row_bytes(a) <= kMidRow)
    return launch(distill_backward_kernel<DT, kMidThreads, kMidCtas>, kMidThreads + 32,
                  rows_params(a, parts_for(a, kMidCtas)), a->rows, false, s, who);
  return launch(distill_backward_kernel<DT, kWideThreads, kWideCtas>, kWideThreads + 32,
                rows_params(a, parts_for(a, kWideCtas)), a->rows, false, s, who);
}

template <int DT> int launch_grad(const zt_distill_args* a, cudaStream_t s) {
  const char* who = "zt_distill_rows_grad launch";
  if (row_bytes(a) <= kMidRow)
    return launch(distill_grad_kernel<DT, kMidThreads, kMidCtas>, kMidThreads + 32,
                  rows_params(a, parts_for_grad(a, kMidCtas)), a->rows, true, s, who);
  return launch(distill_grad_kernel<DT, kWideThreads, kWideCtas>, kWideThreads + 32,
                rows_params(a, parts_for_grad(a, kWideCtas)), a->rows, true, s, who);
}

}  // namespace

extern "C" {

int zt_distill_rows(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, false, "zt_distill_rows")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->loss || !a->lse) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows: null pointer");
  if (short_rows(a, kShortSum, kSumCtas)) return launch_warps<true, false>(a, zt::as_stream(stream), "zt_distill_rows launch");
  const RowsParams P = rows_params(a, parts_for(a, kSumCtas));
  auto* kernel = a->dtype == ZT_BF16 ? distill_forward_kernel<ZT_BF16>
                 : a->dtype == ZT_F16 ? distill_forward_kernel<ZT_F16> : distill_forward_kernel<ZT_F32>;
  return launch(kernel, kSumThreads + 32, P, a->rows, true, zt::as_stream(stream), "zt_distill_rows launch");
}

int zt_distill_rows_backward(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, true, "zt_distill_rows_backward")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->stats) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows_backward: null pointer");
  cudaStream_t s = zt::as_stream(stream);
  if (short_rows(a, kShortWrite, kMidCtas)) return launch_warps<false, true>(a, s, "zt_distill_rows_backward launch");
  if (a->dtype == ZT_BF16) return launch_backward<ZT_BF16>(a, s);
  if (a->dtype == ZT_F16) return launch_backward<ZT_F16>(a, s);
  return launch_backward<ZT_F32>(a, s);
}

int zt_distill_rows_grad(const zt_distill_args* a, void* stream) {
  zt::clear_error();
  if (int rc = check_rows(a, true, "zt_distill_rows_grad")) return rc;
  if (a->rows == 0) return ZT_OK;
  if (!a->loss || !a->lse || !a->weight) return zt::set_error(ZT_ERR_INVALID, "zt_distill_rows_grad: null pointer");
  cudaStream_t s = zt::as_stream(stream);
  if (short_rows(a, kShortGrad, kMidCtas)) return launch_warps<true, true>(a, s, "zt_distill_rows_grad launch");
  if (a->dtype == ZT_BF16) return launch_grad<ZT_BF16>(a, s);
  if (a->dtype == ZT_F16) return launch_grad<ZT_F16>(a, s);
  return launch_grad<ZT_F32>(a, s);
}

}  // extern "C"
