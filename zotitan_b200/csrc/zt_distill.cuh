// What the distillation kernels share: the scorer's exponent arithmetic and a row's teacher
// list, held by one warp.
#pragma once
#include <math.h>

#include "zt_common.cuh"

namespace zt {
namespace distill {

constexpr int kMaxTop = ZT_DISTILL_MAX_TOP;
constexpr int kPer = kMaxTop / 32;   // list entries of a lane
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// sum over v of 2^((z_v - m) c) as (m, s). The maximum is subtracted before the scaling, so
// that a logit at its type's lowest value gives 2^-inf = 0 and a row of nothing but such
// values stays finite.
struct Stat {
  float m, s;
};

__device__ __forceinline__ Stat merge(const Stat& a, const Stat& b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -INFINITY) {
    r.s = a.s + b.s;   // nothing on either side, or NaN
  } else {
    r.s = a.s * ex2((a.m - r.m) * c) + b.s * ex2((b.m - r.m) * c);
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

// N values into a running (m, s).
template <int N> __device__ __forceinline__ void absorb(Stat& st, const float (&f)[N], float c) {
  float cm = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) cm = fmaxf(cm, f[i]);
  if (cm > st.m) {
    st.s *= ex2((st.m - cm) * c);
    st.m = cm;
  }
  const float base = st.m == -INFINITY ? 0.f : st.m;
  float a0 = 0.f, a1 = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    a0 += ex2((f[i] - base) * c);
    if (i + 1 < N) a1 += ex2((f[i + 1] - base) * c);
  }
  st.s += a0 + a1;
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

  __device__ __forceinline__ int64_t index(int64_t i) const {
    return idx64 ? static_cast<const int64_t*>(idx)[i] : (int64_t)static_cast<const int32_t*>(idx)[i];
  }
  __device__ __forceinline__ float value(int64_t i) const {
    if (val_dtype == ZT_F32) return static_cast<const float*>(val)[i];
    if (val_dtype == ZT_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(val)[i]);
    return __half2float(static_cast<const __half*>(val)[i]);
  }
};

// One warp's view of a row's list: lane l holds entries l, l + 32, ... An entry with a
// negative index or the value -inf carries no mass and its value is not looked at.
struct Teacher {
  int32_t idx[kPer];   // -1: no mass
  float p[kPer];       // teacher probability
  float lp[kPer];      // its log2 (0 where p is 0)
  bool any;            // the row has a teacher
  bool bad;            // an index >= vocab

  __device__ __forceinline__ void read(const TopList& L, int64_t row) {
    const int lane = threadIdx.x & 31;
    bool some = false, out = false;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const int k = lane + 32 * e;
      idx[e] = -1;
      p[e] = -INFINITY;
      if (32 * e < L.top && k < L.top) {
        const int64_t i = L.index(row * L.top + k);
        if (i >= 0) {
          const float v = L.value(row * L.top + k);
          if (!(v == -INFINITY)) {
            some = true;
            out = out || i >= L.vocab;
            idx[e] = i < L.vocab ? (int32_t)i : -1;
            p[e] = v;
          }
        }
      }
    }
    any = __any_sync(0xffffffffu, some);
    bad = __any_sync(0xffffffffu, out);
  }

  // p <- softmax of the values times c / log2(e) over the entries with mass
  __device__ __forceinline__ void softmax(float c) {
    float m = -INFINITY;
#pragma unroll
    for (int e = 0; e < kPer; ++e) m = fmaxf(m, p[e]);
    m = warp_max(m);
    float t = 0.f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      lp[e] = (p[e] - m) * c;
      p[e] = idx[e] >= 0 ? exp2f(lp[e]) : 0.f;
      t += p[e];
    }
    t = warp_sum(t);
    const float lt = log2f(t);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      p[e] = p[e] == 0.f ? 0.f : p[e] / t;   // a row without a teacher has t = 0
      lp[e] = p[e] == 0.f ? 0.f : lp[e] - lt;
    }
  }
};

// T^2 sum_k p_k (log p_k - log q_k) from the list and the logits at its indices.
__device__ __forceinline__ float list_loss(const Teacher& t, const float (&z)[kPer], const Stat& st, float c,
                                           float temperature) {
  const float ls = log2f(st.s);
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    if (t.p[e] != 0.f) a = fmaf(t.p[e], t.lp[e] - ((z[e] - st.m) * c - ls), a);
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
