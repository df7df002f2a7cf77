// Fused linear distillation: the lm_head GEMM and the loss against a teacher's top logits
// in one tcgen05 kernel, so no logit reaches HBM.
//
//   z[r, v] = X[r, :] . W[v, :]   (fp32, not rounded)
//   lse[r] = log sum_v exp(z[r, v] / T),
//   loss[r] = T^2 sum_k p_k (log p_k - z[r, i_k] / T + lse[r]),  p = softmax(t_k / T)
//
// Bound by the tensor cores where rows are many (2 rows vocab k flops), by reading W where
// they are few. Three kernels:
// 1. list_kernel, a warp per row: p from the teacher's list, its entries sorted by token.
// 2. linear_distill_kernel on CTA pairs (tcgen05.mma.cta_group::2, 256 x 256 tiles, K-block
//    64, 6 TMA stages, accumulators double-buffered in tensor memory), scheduled like the
//    cross-entropy GEMM: the vocabulary cut into splits of a few tiles, row blocks fastest,
//    so that the pairs in flight share W tiles in L2. The tensor cores truncate as they
//    accumulate: over a K of 2048 that alone puts the loss 1.8e-6 off, over 4096 3.6e-6. So an
//    accumulator takes 1024 of K, and the epilogue threads add these up in registers, rounding
//    to nearest: 0.9e-6 at any K, for 1.5% of the time. Smaller pieces cost more than they give here:
//    512 of K halves the error again for 6 to 9% (8192 x 128256 x 2048 3.2 -> 3.4 ms, 2048 x 32000 x 2048
//    225 -> 249 us), 256 quarters it for 38%. The bf16 operands are up to 2^-8 = 4e-3 of themselves off.
//    An epilogue thread owns half an accumulator row, 128 columns. It also follows the part of
//    its row's list that lies in its columns through the tiles: where one of a warp's rows has
//    a listed token among 16 columns, its threads put theirs into shared memory, each for itself,
//    and pick theirs out by index.
// 3. combine_kernel: a row's sums over the splits, then its list.
// Every mbarrier wait is bounded; on expiry the kernel records an error
// (zt_linear_distill_take_error), drains its own copies and MMAs, frees its tensor memory and leaves
// NaN for every sum that it did not finish.
#include <math.h>

#include "zt_distill.cuh"
#include "zt_tc.cuh"

namespace {

using namespace zt::tc;
using namespace zt::distill;

constexpr int kThreads = 320;  // warp 0 TMA, warp 1 MMA (leader), warps 2-9 epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kChunk = 16;     // K-blocks of one accumulator: 1024 of K
constexpr int kStages = 6;
constexpr uint32_t kHalfRows = 128;
constexpr uint32_t kStageA = kHalfRows * kBK * 2;  // 16 KB of X
constexpr uint32_t kStageBytes = 2 * kStageA;       // + 16 KB of W (this CTA's half of the N tile)
constexpr int kTile = 256;
constexpr uint32_t kTmemCols = 2 * kTile;
constexpr int kWindow = 16;    // entries of a row's list that an epilogue thread has at hand
constexpr int kSlab = 16;      // columns that it puts into shared memory to pick from
constexpr int kLanes = 32 * kEpilogueWarps;
constexpr int kHalfShift = 24; // takes the bit of a column's half tile (128) to bit 31
static_assert((kTile / 2) << kHalfShift == (int)0x80000000, "the half's bit leads the sorting key");
constexpr size_t kSmem = 1024 + kStages * kStageBytes + 256 + (kWindow + kSlab) * 32 * kEpilogueWarps * 4;
constexpr uint32_t kIdesc = idesc_bf16(256, 256);
constexpr int kListWarps = 8;
enum { kHasTeacher = 0, kNoTeacher = 1, kBadList = 2 };

__device__ int g_distill_error = 0;

struct Params {
  CUtensorMap tmap_x;  // X [rows, k], box {64, 128}
  CUtensorMap tmap_w;  // W [vocab, k], box {64, 128}
  TopList list;
  int32_t* status;     // [rows]: 4 x (entries of the first half columns) + one of the above
  int32_t* idx;        // [rows][top] tokens, those of the first half columns of their tiles, then those
                       // of the second, each in rising order; INT32_MAX behind the last with mass
  float* lp;           // [rows][top] log2 p in that order
  float* z;            // [rows][top] logits in that order
  float2* partials;    // [2 n_splits][rows_pad] (m, s), of both halves of a split's tiles
  float* loss;
  float* lse;
  int32_t rows, vocab, top, k_blocks, n_chunks;
  int32_t m_tiles, n_tiles, split_tiles, n_splits, rows_pad;
  float c, temperature;
  int32_t stall_loads;    // test hook: the loader issues no copies
  long long wait_cycles;  // bound of every wait
};

__global__ void __launch_bounds__(32 * kListWarps) list_kernel(const __grid_constant__ Params P) {
  const int64_t row = (int64_t)blockIdx.x * kListWarps + threadIdx.x / 32;
  if (row >= P.rows) return;
  const int lane = threadIdx.x & 31;
  __shared__ unsigned long long room[kListWarps][kMaxTop * List::kBytes / 8];
  const List s(room[threadIdx.x / 32], kMaxTop);
  const Teacher t = read_list(s, P.list, row);
  list_softmax(s, P.top, P.c);
  for (int k = lane; k < P.top; k += 32)
    if (s.p[k] == 0.f) s.idx[k] = -1;   // no mass: behind the others
  // tokens of the first half of a tile's columns stand before those of the second, both rising
  list_sort(s, P.top, [](int32_t idx) { return idx < 0 ? 0xffffffffu : (uint32_t)idx | ((uint32_t)idx & (kTile / 2)) << kHalfShift; });
  int first = 0;
  for (int k0 = 0; k0 < P.top; k0 += 32) {
    const int k = k0 + lane;
    uint32_t key = 0xffffffffu;
    if (k < P.top) {
      const unsigned long long e = s.order[k];
      key = (uint32_t)(e >> 32);
      P.idx[row * P.top + k] = key == 0xffffffffu ? INT32_MAX : (int32_t)(key & 0x7fffffffu);
      P.lp[row * P.top + k] = s.lp[(uint32_t)e];
    }
    first += __popc(__ballot_sync(0xffffffffu, key < 0x80000000u));
  }
  if (lane == 0) P.status[row] = first << 2 | (!t.any ? kNoTeacher : t.bad ? kBadList : kHasTeacher);
}

__device__ __forceinline__ void item_range(const Params& P, int item, int& mt, int& split, int& nt0, int& nt1) {
  split = item / P.m_tiles;
  mt = item - split * P.m_tiles;
  nt0 = split * P.split_tiles;
  nt1 = min(nt0 + P.split_tiles, P.n_tiles);
}

// 32 lanes x 16 consecutive fp32 columns of tensor memory (lane = thread of the warp).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    linear_distill_kernel(const __grid_constant__ Params P) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* stage_base = smem;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  uint64_t* full = bars;                    // [kStages], used in the leader
  uint64_t* empty = bars + kStages;         // [kStages]
  uint64_t* accf = bars + 2 * kStages;      // [2]
  uint64_t* acce = bars + 2 * kStages + 2;  // [2], used in the leader
  uint64_t* drain = bars + 2 * kStages + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int32_t* windows = reinterpret_cast<int32_t*>(smem + kStages * kStageBytes + 256);   // [kWindow][epilogue threads]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&accf[b], 1); mbar_init(&acce[b], 2 * kEpilogueWarps); }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {  // warp 0 of both CTAs allocates the pair's tensor memory
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  cluster_sync_all();  // barriers of both CTAs initialised before any cross-CTA signal
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t peer_abort = peer_addr((const void*)abort, rank ^ 1u);

  const int n_items = P.m_tiles * P.n_splits;
  const int cid = (int)cluster_id_x(), ncl = (int)n_clusters_x();
  if (warp == 0) {
    if (lane == 0) {  // ---- TMA producer (both CTAs)
      int last_phase[kStages];
      for (int s = 0; s < kStages; ++s) last_phase[s] = -1;
      uint32_t it = 0;
      bool ok = !P.stall_loads;
      for (int item = cid; ok && item < n_items; item += ncl) {
        int mt, split, nt0, nt1;
        item_range(P, item, mt, split, nt0, nt1);
        for (int nt = nt0; ok && nt < nt1; ++nt) {
          for (int kb = 0; kb < P.k_blocks; ++kb, ++it) {
            const int s = it % kStages;
            const uint32_t round = it / kStages;
            if (!mbar_wait_pair(&empty[s], (round & 1) ^ 1, abort, peer_abort, &g_distill_error, 1, P.wait_cycles)) {
              ok = false;
              break;
            }
            uint8_t* sa = stage_base + s * kStageBytes;
            const uint32_t leader_full = peer_addr(&full[s], 0);
            if (leader) mbar_expect_tx(&full[s], 2 * kStageBytes);
            tma_load_2d_pair(sa, &P.tmap_x, leader_full, kb * kBK, mt * kTile + (int)rank * (int)kHalfRows);
            tma_load_2d_pair(sa + kStageA, &P.tmap_w, leader_full, kb * kBK, nt * kTile + (int)rank * (int)kHalfRows);
            last_phase[s] = (int)(round & 1);
          }
        }
      }
      // Drain (leader): each armed phase of a full barrier completes only when both CTAs'
      // copies for it have landed, so no copy is in flight when the pair leaves.
      if (leader)
        for (int s = 0; s < kStages; ++s)
          if (last_phase[s] >= 0) mbar_drain(&full[s], (uint32_t)last_phase[s]);
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {  // ---- MMA issuer (leader CTA only)
      uint32_t it = 0, tcount = 0;
      bool ok = true, issued = false;
      for (int item = cid; ok && item < n_items; item += ncl) {
        int mt, split, nt0, nt1;
        item_range(P, item, mt, split, nt0, nt1);
        for (int nt = nt0; ok && nt < nt1; ++nt) {
          for (int k0 = 0; ok && k0 < P.k_blocks; k0 += kChunk, ++tcount) {
            const uint32_t b = tcount & 1;
            if (!mbar_wait_pair(&acce[b], ((tcount >> 1) & 1) ^ 1, abort, peer_abort, &g_distill_error, 2, P.wait_cycles)) {
              ok = false;
              break;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + b * kTile;
            const int k1 = min(k0 + kChunk, P.k_blocks);
            for (int kb = k0; kb < k1; ++kb, ++it) {
              const int s = it % kStages;
              if (!mbar_wait_pair(&full[s], (it / kStages) & 1, abort, peer_abort, &g_distill_error, 3, P.wait_cycles)) {
                ok = false;
                break;
              }
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
              const uint32_t sa = smem_u32(stage_base + s * kStageBytes);
              const uint32_t sb = sa + kStageA;
#pragma unroll
              for (int k = 0; k < kBK / kUmmaK; ++k)
                umma_bf16_pair<kIdesc>(tmem_d, umma_desc(sa + k * kUmmaK * 2), umma_desc(sb + k * kUmmaK * 2),
                                       kb != k0 || k != 0);
              issued = true;
              umma_commit_pair(&empty[s]);  // stage s is free in both CTAs once these MMAs have read it
            }
            if (!ok) break;
            umma_commit_pair(&accf[b]);  // accumulator b is complete in both CTAs
          }
        }
      }
      if (issued) {  // wait (bounded) for every MMA issued by this thread before exit
        umma_commit_pair_local(drain);
        mbar_drain(drain, 0);
      }
    }
  } else {  // ---- epilogue: warps 2..9 of both CTAs; each thread owns half an accumulator row
    const int q = warp & 3, half = (warp - 2) >> 2;
    const int row_local = q * 32 + lane;
    const uint32_t leader_acce0 = peer_addr(&acce[0], 0), leader_acce1 = peer_addr(&acce[1], 0);
    uint32_t tcount = 0;
    bool ok = true;
    for (int item = cid; item < n_items; item += ncl) {
      int mt, split, nt0, nt1;
      item_range(P, item, mt, split, nt0, nt1);
      const int row = mt * kTile + (int)rank * (int)kHalfRows + row_local;
      if (!ok) {   // a wait has expired: what is left of the queue is not a number
        if (row < P.rows) P.partials[(size_t)(2 * split + half) * P.rows_pad + row] = make_float2(-INFINITY, NAN);
        continue;
      }
      // the row's entries of this half's columns, from this split's first column on
      const int32_t* list = P.idx + (int64_t)row * P.top;
      float* z = P.z + (int64_t)row * P.top;
      int pos = 0, end = 0, next = INT32_MAX;
      int have = 0, ready = 0;   // places before `have` have been fetched, before `ready` are at hand
      int32_t* window = windows + (warp - 2) * 32 + lane;   // place p in slot p mod kWindow
      float* slab = reinterpret_cast<float*>(window + kWindow * kLanes);
      auto fetch = [&]() {   // the next half window
#pragma unroll
        for (int j = 0; j < kWindow / 2; ++j)
          if (have + j < end)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                         ::"r"(smem_u32(window + ((have + j) & (kWindow - 1)) * kLanes)), "l"(list + have + j)
                         : "memory");
        have += kWindow / 2;
      };
      auto arrived = [&]() {
        asm volatile("cp.async.wait_all;" ::: "memory");
        ready = have;
      };
      auto look = [&]() {   // next <- the token at pos
        if (pos >= end) {
          next = INT32_MAX;
          return;
        }
        while (pos >= ready) {   // only after more than half a window in one tile
          if (pos >= have) fetch();
          arrived();
        }
        next = *(volatile int32_t*)(window + (pos & (kWindow - 1)) * kLanes);
      };
      if (row < P.rows) {
        const int firsts = P.status[row] >> 2;
        pos = half ? firsts : 0;
        end = half ? P.top : firsts;
        int hi = nt0 > 0 ? end : pos;
        while (pos < hi) {
          const int mid = (pos + hi) >> 1;
          if (list[mid] < nt0 * kTile) pos = mid + 1;
          else hi = mid;
        }
        arrived();   // what the last item's row had asked for
        have = ready = pos;
        fetch();
        fetch();
        look();
      }
      __syncwarp();
      Stat st{-INFINITY, 0.f};
      for (int nt = nt0; ok && nt < nt1; ++nt) {
        const int tile0 = nt * kTile;
        float sum[kTile / 2];
        arrived();   // asked for at the last tile
        if (have - pos <= kWindow / 2 && have < end) fetch();
        for (int ch = 0; ch < P.n_chunks; ++ch, ++tcount) {
          const uint32_t b = tcount & 1;
          int okw = 1;
          if (lane == 0) okw = mbar_wait_pair(&accf[b], (tcount >> 1) & 1, abort, peer_abort, &g_distill_error, 4, P.wait_cycles) ? 1 : 0;
          okw = __shfl_sync(0xffffffffu, okw, 0);
          if (!okw) { ok = false; break; }
          __syncwarp();
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t acc = tmem_base + ((uint32_t)(q * 32) << 16) + b * kTile;
#pragma unroll
          for (int c0 = 0; c0 < kTile / 2; c0 += 16) {
            uint32_t r[16];
            tmem_ld16(acc + (uint32_t)(half * (kTile / 2) + c0), r);
            if (ch == 0) {
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[c0 + j] = __uint_as_float(r[j]);
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[c0 + j] += __uint_as_float(r[j]);
            }
          }
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(b ? leader_acce1 : leader_acce0);  // accumulator b may be overwritten
        }
        if (!ok) break;
        const int col0 = tile0 + half * (kTile / 2);
        if (col0 + kTile / 2 > P.vocab) {  // the padded columns of the last tile
#pragma unroll
          for (int j = 0; j < kTile / 2; ++j)
            if (col0 + j >= P.vocab) sum[j] = -INFINITY;
        }
        absorb(st, sum, P.c);
#pragma unroll
        for (int c0 = 0; c0 < kTile / 2; c0 += kSlab) {
          if (!__any_sync(0xffffffffu, next < col0 + c0 + kSlab)) continue;
#pragma unroll
          for (int j = 0; j < kSlab; ++j) slab[j * kLanes] = sum[c0 + j];
          while (next < col0 + c0 + kSlab) {   // once more where the token stands in the list several times
            z[pos] = slab[(next - (col0 + c0)) * kLanes];
            ++pos;
            look();
          }
          __syncwarp();
        }
      }
      if (row < P.rows) P.partials[(size_t)(2 * split + half) * P.rows_pad + row] = make_float2(st.m, ok ? st.s : NAN);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");   // no copy is in flight when the thread leaves
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while its peer may still signal it or read its shared memory
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 0) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
  }
}

// Eight rows a block. Its threads merge the rows' splits (eight adjacent rows, 64 bytes, a group
// of eight threads), then a warp takes a row's list, which it loaded before.
constexpr int kCombineRows = kListWarps;

__global__ void __launch_bounds__(32 * kListWarps) combine_kernel(const __grid_constant__ Params P) {
  __shared__ Stat part[kListWarps][kCombineRows];
  const int64_t row0 = (int64_t)blockIdx.x * kCombineRows;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
  const int64_t row = row0 + warp;
  constexpr int kHeld = 4;   // list entries of a lane loaded ahead
  int32_t idx[kHeld], status = kNoTeacher;
  float lp[kHeld], z[kHeld];
#pragma unroll
  for (int e = 0; e < kHeld; ++e) {
    idx[e] = INT32_MAX;
    if (row < P.rows && lane + 32 * e < P.top) {
      const int64_t at = row * P.top + lane + 32 * e;
      idx[e] = __ldg(P.idx + at);
      lp[e] = __ldg(P.lp + at);
      z[e] = __ldg(P.z + at);   // not written where idx is INT32_MAX, and then not looked at
    }
  }
  if (row < P.rows) status = __ldg(P.status + row) & 3;
  Stat st{-INFINITY, 0.f};
#pragma unroll 4
  for (int sp = tid / kCombineRows; sp < 2 * P.n_splits; sp += 32 * kListWarps / kCombineRows) {   // rows_pad covers the block
    const float2 o = __ldg(P.partials + (size_t)sp * P.rows_pad + row0 + tid % kCombineRows);
    st = merge(st, Stat{o.x, o.y}, P.c);
  }
#pragma unroll
  for (int o = kCombineRows; o < 32; o <<= 1) {
    Stat u;
    u.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    st = merge(st, u, P.c);
  }
  if (lane < kCombineRows) part[warp][lane] = st;
  __syncthreads();
  if (row >= P.rows) return;
  st = part[0][warp];
#pragma unroll
  for (int w = 1; w < kListWarps; ++w) st = merge(st, part[w][warp], P.c);
  if (st.m == -INFINITY) st.s = NAN;
  const float ls = log2f(st.s);
  const Base base(st.m, P.c);
  float a = 0.f;
  auto add = [&](float l, float v) { a = fmaf(exp2f(l), l - (base.rel(v, P.c) - ls), a); };
#pragma unroll
  for (int e = 0; e < kHeld; ++e)
    if (idx[e] != INT32_MAX) add(lp[e], z[e]);
  for (int k = lane + 32 * kHeld; k < P.top; k += 32) {
    const int64_t at = row * P.top + k;
    if (P.idx[at] != INT32_MAX) add(P.lp[at], P.z[at]);
  }
  a = warp_sum(a) * (kLn2 * P.temperature * P.temperature);
  if (lane == 0) {
    P.loss[row] = status == kNoTeacher ? 0.f : status == kBadList ? NAN : a;
    P.lse[row] = status == kNoTeacher ? 0.f : status == kBadList ? NAN : sum_lse(st, P.c, P.temperature);
  }
}

// Per-device kernel attributes and the number of CTA pairs resident at once.
int g_max_pairs[64] = {0};

int prepare(int dev) {
  static std::mutex mu;
  std::lock_guard<std::mutex> lock(mu);
  if (g_max_pairs[dev] > 0) return ZT_OK;
  if (int rc = zt::check_cuda(cudaFuncSetAttribute(linear_distill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)kSmem), "zt_linear_distill: shared memory attribute"))
    return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(zt::sm_count() / 2));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  int n = 0;
  if (int rc = zt::check_cuda(cudaOccupancyMaxActiveClusters(&n, linear_distill_kernel, &cfg),
                              "zt_linear_distill: cudaOccupancyMaxActiveClusters"))
    return rc;
  if (n <= 0) return zt::set_error(ZT_ERR_CUDA, "zt_linear_distill: no CTA pair fits on this GPU");
  g_max_pairs[dev] = n;
  return ZT_OK;
}

// Vocabulary split: the split length (in 256-column tiles) whose round-robin schedule over
// `pairs` CTA pairs has the shortest longest queue, an item counting an eighth of a tile more than
// its tiles: at its start every row looks up its place in its list, and at its end leaves
// a partial sum to be merged (8192 x 128256 rows in splits of one tile: 33 MB of them).
struct Split {
  int32_t m_tiles, n_tiles, split_tiles, n_splits, rows_pad;
};

Split choose_split(int64_t rows, int64_t vocab, int pairs) {
  Split sp;
  sp.m_tiles = (int32_t)((rows + kTile - 1) / kTile);
  sp.n_tiles = (int32_t)((vocab + kTile - 1) / kTile);
  sp.rows_pad = sp.m_tiles * kTile;
  long long best = -1;
  sp.split_tiles = sp.n_tiles;
  for (int st = 1; st <= sp.n_tiles && st <= 64; ++st) {
    const long long splits = (sp.n_tiles + st - 1) / st;
    const long long items = splits * sp.m_tiles;
    const long long queue = (items + pairs - 1) / pairs * (8 * st + 1);
    if (best < 0 || queue <= best) {
      best = queue;
      sp.split_tiles = st;
    }
  }
  sp.n_splits = (sp.n_tiles + sp.split_tiles - 1) / sp.split_tiles;
  return sp;
}

int device_pairs(int* dev, int* pairs) {
  if (int rc = zt::check_cuda(cudaGetDevice(dev), "zt_linear_distill: cudaGetDevice")) return rc;
  if (*dev < 0 || *dev >= 64) return zt::set_error(ZT_ERR_LIMIT, "zt_linear_distill: device ordinal >= 64");
  if (int rc = prepare(*dev)) return rc;
  *pairs = g_max_pairs[*dev];
  return ZT_OK;
}

// The items (row blocks x splits, at most one split per tile) are counted in 32 bits.
int check_shape(int64_t rows, int64_t vocab, int64_t k, int32_t top) {
  if (rows <= 0 || rows > (int64_t)1 << 28) return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: rows outside [1, 2^28]");
  if (vocab <= 0 || vocab > (int64_t)1 << 28) return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: vocab outside [1, 2^28]");
  if (k <= 0 || k % kBK != 0 || k > (int64_t)1 << 30)
    return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: k must be a positive multiple of 64");
  if (top < 1 || top > kMaxTop)
    return zt::set_error(ZT_ERR_LIMIT, "zt_linear_distill: the teacher's list must have 1 to 256 entries");
  if (((rows + kTile - 1) / kTile) * ((vocab + kTile - 1) / kTile) > (int64_t)INT32_MAX / 2)
    return zt::set_error(ZT_ERR_LIMIT, "zt_linear_distill: rows x vocab above 2^46");
  return ZT_OK;
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// The workspace: partials, sorted tokens, log2 p, logits, status.
struct Layout {
  size_t idx, lp, z, status, total;
};

Layout layout(const Split& sp, int64_t rows, int32_t top) {
  const size_t entries = (size_t)rows * (size_t)top * 4;
  Layout L;
  L.idx = up256(2 * sizeof(float2) * (size_t)sp.n_splits * (size_t)sp.rows_pad);
  L.lp = L.idx + up256(entries);
  L.z = L.lp + up256(entries);
  L.status = L.z + up256(entries);
  L.total = L.status + up256((size_t)rows * 4);
  return L;
}

}  // namespace

extern "C" {

size_t zt_linear_distill_workspace_bytes(int64_t rows, int64_t vocab, int64_t k, int32_t top) {
  zt::clear_error();
  if (check_shape(rows, vocab, k, top)) return 0;
  int dev = 0, pairs = 0;
  if (device_pairs(&dev, &pairs)) return 0;
  return layout(choose_split(rows, vocab, pairs), rows, top).total;
}

int zt_linear_distill(const zt_linear_distill_args* a, void* stream) {
  zt::clear_error();
  if (!a || !a->x || !a->w || !a->loss || !a->lse || !a->workspace)
    return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: null pointer");
  if (int rc = check_shape(a->rows, a->vocab, a->k, a->top)) return rc;
  if (int rc = check_list(a->top_idx, a->top_logits, a->top, a->idx_bits, a->top_dtype, a->temperature, false,
                          "zt_linear_distill"))
    return rc;
  auto mis16 = [](const void* p) { return ((uintptr_t)p & 15u) != 0; };
  if (mis16(a->x) || mis16(a->w) || mis16(a->workspace))
    return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: x, w and workspace must be 16-byte aligned");
  int dev = 0, pairs = 0;
  if (int rc = device_pairs(&dev, &pairs)) return rc;
  const Split sp = choose_split(a->rows, a->vocab, pairs);
  const Layout L = layout(sp, a->rows, a->top);
  if (a->workspace_bytes < L.total) return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill: workspace too small");
  EncodeFn enc = nullptr;
  if (int rc = get_encode(&enc, "zt_linear_distill")) return rc;
  Params P;
  if (int rc = make_map_bf16(enc, &P.tmap_x, a->x, (uint64_t)a->rows, (uint64_t)a->k, kHalfRows, "zt_linear_distill"))
    return rc;
  if (int rc = make_map_bf16(enc, &P.tmap_w, a->w, (uint64_t)a->vocab, (uint64_t)a->k, kHalfRows, "zt_linear_distill"))
    return rc;
  char* ws = static_cast<char*>(a->workspace);
  P.list = TopList{a->top_idx, a->top_logits, a->top, a->idx_bits == 64, a->top_dtype, a->vocab};
  P.partials = reinterpret_cast<float2*>(ws);
  P.idx = reinterpret_cast<int32_t*>(ws + L.idx);
  P.lp = reinterpret_cast<float*>(ws + L.lp);
  P.z = reinterpret_cast<float*>(ws + L.z);
  P.status = reinterpret_cast<int32_t*>(ws + L.status);
  P.loss = a->loss;
  P.lse = a->lse;
  P.rows = (int32_t)a->rows;
  P.vocab = (int32_t)a->vocab;
  P.top = a->top;
  P.k_blocks = (int32_t)(a->k / kBK);
  P.n_chunks = (P.k_blocks + kChunk - 1) / kChunk;
  P.m_tiles = sp.m_tiles;
  P.n_tiles = sp.n_tiles;
  P.split_tiles = sp.split_tiles;
  P.n_splits = sp.n_splits;
  P.rows_pad = sp.rows_pad;
  P.c = kLog2e / a->temperature;
  P.temperature = a->temperature;
  P.stall_loads = a->test_stall_loads ? 1 : 0;
  P.wait_cycles = a->test_wait_cycles > 0 ? (long long)a->test_wait_cycles : kWaitCycles;
  const int items = sp.m_tiles * sp.n_splits;
  const int clusters = items < pairs ? items : pairs;
  cudaStream_t s = zt::as_stream(stream);
  const unsigned row_blocks = (unsigned)((a->rows + kListWarps - 1) / kListWarps);
  list_kernel<<<row_blocks, 32 * kListWarps, 0, s>>>(P);
  if (int rc = zt::check_cuda(cudaGetLastError(), "zt_linear_distill: list launch")) return rc;
  linear_distill_kernel<<<2 * clusters, kThreads, kSmem, s>>>(P);
  if (int rc = zt::check_cuda(cudaGetLastError(), "zt_linear_distill: gemm launch")) return rc;
  combine_kernel<<<(unsigned)((a->rows + kCombineRows - 1) / kCombineRows), 32 * kListWarps, 0, s>>>(P);
  return zt::check_cuda(cudaGetLastError(), "zt_linear_distill: combine launch");
}

int zt_linear_distill_take_error(int32_t* code) {
  zt::clear_error();
  if (!code) return zt::set_error(ZT_ERR_INVALID, "zt_linear_distill_take_error: null pointer");
  int v = 0;
  if (int rc = zt::check_cuda(cudaMemcpyFromSymbol(&v, g_distill_error, sizeof(int)), "zt_linear_distill_take_error: read"))
    return rc;
  const int zero = 0;
  if (int rc = zt::check_cuda(cudaMemcpyToSymbol(g_distill_error, &zero, sizeof(int)), "zt_linear_distill_take_error: clear"))
    return rc;
  *code = v;
  return ZT_OK;
}

}  // extern "C"
