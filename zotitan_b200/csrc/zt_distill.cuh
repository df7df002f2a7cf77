// What the distillation kernels share: the scorer's exponent arithmetic and a row's teacher
// list, held by one warp.
#pragma once
#include <math.h>

#include "zt_common.cuh"

namespace zt {
namespace distill {

constexpr int kMaxTop = ZT_DISTILL_MAX_TOP;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A sum over v of 2^((z_v - m) c) as (m, s). m is a z near the largest one: it follows the
// running maximum only when that is more than kSlack powers of two ahead, because with a running
// maximum of their own some lane of a warp has a new one at almost every step, and the rescaling
// measured a third of the instructions. A sum of 2^30 such terms stays below 2^47.
//
// (z - m) c is fma(z, c, -mc) with mc = round(m c): one instruction, and what mc's rounding takes
// off the exponent is the same for every term, so that it cancels as long as all uses of a sum
// take the same mc. That holds while it is small: beyond |mc| = kFar (where it may be 2^-4) the
// difference is taken first, which is exact for z near m. So rows with a common part of
// any size keep their softmax, a logit at its type's lowest value gives 2^-inf = 0, and a row of
// nothing else stays finite.
struct Stat {
  float m, s;
};

constexpr float kFar = 1048576.f;
constexpr float kSlack = 16.f;

struct Base {
  float m, mc;   // 0 where there is no finite maximum yet
  __device__ __forceinline__ Base(float max, float c) {
    m = max == -INFINITY ? 0.f : max;
    mc = __fmul_rn(m, c);
  }
  __device__ __forceinline__ bool far() const { return fabsf(mc) > kFar; }
  __device__ __forceinline__ float rel(float z, float c) const { return far() ? (z - m) * c : __fmaf_rn(z, c, -mc); }
};

// The factor that takes a sum from base a to the larger b: 2 to the difference of what the two
// sums are relative to, mc or, far out, m c itself.
__device__ __forceinline__ float rescale(float a, float b, float c) {
  if (a == -INFINITY) return 0.f;
  const float ac = __fmul_rn(a, c), bc = __fmul_rn(b, c);
  const bool fa = fabsf(ac) > kFar, fb = fabsf(bc) > kFar;
  if (!fa && !fb) return ex2(__fsub_rn(ac, bc));
  float d = (a - b) * c;
  if (!fa) d -= __fmaf_rn(a, c, -ac);
  if (!fb) d += __fmaf_rn(b, c, -bc);
  return ex2(d);
}

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -INFINITY) {
    r.s = a.s + b.s;   // nothing on either side, or NaN
  } else {
    r.s = a.s * rescale(a.m, r.m, c) + b.s * rescale(b.m, r.m, c);
  }
  return r;
}

__device__ __forceinline__ Stat warp_merge(Stat v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat u;
    u.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    v = merge(v, u, c);
  }
  return v;
}

// N values, cm the largest of them, into a running (m, s).
template <int N> __device__ __forceinline__ void absorb(Stat& st, const float (&f)[N], float cm, float c) {
  if (cm > st.m + kSlack / c) {   // and wherever m is still -inf
    st.s *= rescale(st.m, cm, c);
    st.m = cm;
  }
  const Base base(st.m, c);
  float a[2] = {0.f, 0.f};
  if (base.far()) {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i & 1] += ex2((f[i] - base.m) * c);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) a[i & 1] += ex2(__fmaf_rn(f[i], c, -base.mc));
  }
  st.s += a[0] + a[1];
}

template <int N> __device__ __forceinline__ void absorb(Stat& st, const float (&f)[N], float c) {
  float cm = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) cm = fmaxf(cm, f[i]);
  absorb(st, f, cm, c);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// A teacher's list of a row, as the caller stores it.
struct TopList {
  const void* idx;   // int32 or int64
  const void* val;   // fp32, bf16 or fp16
  int32_t top, idx64, val_dtype;
  int64_t vocab;
};

// A row's list in shared memory, worked on by one warp: lane l owns entries l, l + 32, ...
// An entry with a negative index or the value -inf carries no mass and its other half is not
// looked at.
struct List {
  unsigned long long* order;   // key and place of the entries, sorted (list_sort)
  int32_t* idx;                // -1: no mass
  float* p;                    // teacher probability, 0 without mass
  float* lp;                   // its log2, 0 where p is 0
  float* z;                    // the row's logit at idx

  static constexpr int kBytes = 24;   // an entry's, all together
  // room for `cap` entries, a power of two, at 8-byte aligned shared memory
  __device__ __forceinline__ List(void* base, int cap) {
    order = static_cast<unsigned long long*>(base);
    idx = reinterpret_cast<int32_t*>(order + cap);
    p = reinterpret_cast<float*>(idx + cap);
    lp = p + cap;
    z = lp + cap;
  }
};

// The capacity that a list of `top` entries takes.
__host__ __device__ inline int list_capacity(int top) {
  int n = 1;
  while (n < top) n <<= 1;
  return n;
}

struct Teacher {
  bool any;   // the row has a teacher
  bool bad;   // an index >= vocab, or a value that is NaN or +inf, on an entry with mass: the row is NaN
};

// The loads of four entries a lane are on their way before the first is looked at.
template <class I, class F>
__device__ __forceinline__ Teacher read_list(const List& s, const I* __restrict__ idx, const F* __restrict__ val, int top, int64_t vocab) {
  bool some = false, out = false;
  for (int k0 = threadIdx.x & 31; k0 < top; k0 += 128) {
    I i[4];
    F v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      i[e] = -1;
      if (k0 + 32 * e < top) {
        i[e] = __ldg(idx + k0 + 32 * e);
        v[e] = __ldg(val + k0 + 32 * e);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (k0 + 32 * e < top) {
        const float f = (float)v[e];
        const bool on = i[e] >= 0 && !(f == -INFINITY);
        some = some || on;
        out = out || (on && ((int64_t)i[e] >= vocab || !(f < INFINITY)));
        s.idx[k0 + 32 * e] = on && (int64_t)i[e] < vocab ? (int32_t)i[e] : -1;
        s.p[k0 + 32 * e] = on ? f : -INFINITY;
      }
  }
  Teacher t;
  t.any = __any_sync(0xffffffffu, some);
  t.bad = __any_sync(0xffffffffu, out);
  return t;
}

template <class I> __device__ __forceinline__ Teacher read_list_as(const List& s, const TopList& L, int64_t at) {
  const I* i = static_cast<const I*>(L.idx) + at;
  if (L.val_dtype == ZT_F32) return read_list(s, i, static_cast<const float*>(L.val) + at, L.top, L.vocab);
  if (L.val_dtype == ZT_BF16) return read_list(s, i, static_cast<const __nv_bfloat16*>(L.val) + at, L.top, L.vocab);
  return read_list(s, i, static_cast<const __half*>(L.val) + at, L.top, L.vocab);
}

__device__ __forceinline__ Teacher read_list(const List& s, const TopList& L, int64_t row) {
  if (L.idx64) return read_list_as<long long>(s, L, row * L.top);
  return read_list_as<int32_t>(s, L, row * L.top);
}

// p <- softmax of the values times c / log2(e) over the entries with mass.
__device__ __forceinline__ void list_softmax(const List& s, int top, float c) {
  const int lane = threadIdx.x & 31;
  float m = -INFINITY;
  for (int k = lane; k < top; k += 32) m = fmaxf(m, s.p[k]);
  m = warp_max(m);
  float t = 0.f;
  for (int k = lane; k < top; k += 32) {
    const float l = (s.p[k] - m) * c, p = s.idx[k] >= 0 ? exp2f(l) : 0.f;
    s.lp[k] = l;
    s.p[k] = p;
    t += p;
  }
  t = warp_sum(t);
  const float lt = log2f(t);
  for (int k = lane; k < top; k += 32) {
    const float p = s.p[k];   // a row without a teacher has t = 0
    s.p[k] = p == 0.f ? 0.f : p / t;
    s.lp[k] = p == 0.f ? 0.f : s.lp[k] - lt;
  }
}

// order <- the entries by rising key(idx), and by place in the list where keys are equal; an entry
// without mass has the key 2^32 - 1. A bitonic sort: 36 steps of four pairs a lane for 256
// entries, where counting every entry's rank against all others took 64 x 8 comparisons of four.
template <class Key> __device__ __forceinline__ void list_sort(const List& s, int top, Key key) {
  const int lane = threadIdx.x & 31, n = list_capacity(top);
  for (int k = lane; k < n; k += 32)
    s.order[k] = k < top ? (unsigned long long)key(s.idx[k]) << 32 | (unsigned)k : ~0ull;
  for (int size = 2; size <= n; size <<= 1)
    for (int j = size >> 1; j > 0; j >>= 1) {
      __syncwarp();
      for (int q = lane; q < n / 2; q += 32) {
        const int lo = 2 * q - (q & (j - 1)), hi = lo + j;
        const unsigned long long a = s.order[lo], b = s.order[hi];
        if ((a > b) == ((lo & size) == 0)) {
          s.order[lo] = b;
          s.order[hi] = a;
        }
      }
    }
  __syncwarp();
}

// log sum_v exp(z_v / T) of a finished sum.
__device__ __forceinline__ float sum_lse(const Stat& st, float c, float temperature) {
  const Base base(st.m, c);
  return base.far() ? st.m / temperature + logf(st.s) : fmaf(base.mc, kLn2, logf(st.s));
}

// T^2 sum_k p_k (log p_k - log q_k) from the list and the logits at its indices.
__device__ __forceinline__ float list_loss(const List& s, int top, const Stat& st, float c, float temperature) {
  const float ls = log2f(st.s);
  const Base base(st.m, c);
  float a = 0.f;
  for (int k = threadIdx.x & 31; k < top; k += 32)
    if (s.p[k] != 0.f) a = fmaf(s.p[k], s.lp[k] - (base.rel(s.z[k], c) - ls), a);
  return warp_sum(a) * (kLn2 * temperature * temperature);
}

inline int check_list(const void* idx, const void* val, int32_t top, int32_t idx_bits, int32_t val_dtype,
                      float temperature, bool empty, const std::string& who) {
  if (top < 1 || top > kMaxTop)
    return set_error(ZT_ERR_LIMIT, who + ": the teacher's list must have 1 to " + std::to_string(kMaxTop) + " entries");
  if (idx_bits != 32 && idx_bits != 64) return set_error(ZT_ERR_INVALID, who + ": indices must be int32 or int64");
  if (val_dtype != ZT_F32 && val_dtype != ZT_BF16 && val_dtype != ZT_F16)
    return set_error(ZT_ERR_INVALID, who + ": unknown dtype of the teacher's logits");
  if (!(temperature >= 1e-3f && temperature <= 1e3f))
    return set_error(ZT_ERR_INVALID, who + ": temperature must lie in [0.001, 1000]");
  if (!empty && (!idx || !val)) return set_error(ZT_ERR_INVALID, who + ": null pointer");
  return ZT_OK;
}

}  // namespace distill
}  // namespace zt
