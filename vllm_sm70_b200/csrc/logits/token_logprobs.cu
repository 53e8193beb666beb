// Log-probability, rank, entropy and top alternatives of given tokens, and
// the gradient of the log-probability and the entropy.
//
//   z = x / T,  p = softmax(z),  lp_j = log p_j
//   logprob = lp_y          rank = 1 + #{j before y}
//   entropy = -sum p lp     top_n = the first n of the row
// "before" is the order (larger x, then lower id). A row without any finite
// or infinite logit above -inf has no distribution: lse -inf, log-probs -inf,
// entropy 0, gradient 0. A NaN or a +inf makes the row's sums NaN, as the
// formula has it; a NaN is never counted or listed.
//
// One pass. A CTA (or a cluster of 2 to 8 when there are few rows) streams a
// row once and keeps per thread: the maximum, the two base-2 sums of rows.cuh
// and the count of elements before y. The alternatives need no second pass
// over the row: a value tau that the maxima of n THREADS reach is a lower
// bound of the row's n-th largest value, so every alternative is an element
// >= tau of a thread whose maximum is >= tau. With j = ceil(n / warps), tau is
// the ceil(n / j)-th largest of the warps' j-th largest maxima: each warp
// finds its own with j warp reductions, no bisection over the whole CTA. A
// thread also leaves the maximum of each of its groups of vectors in shared
// memory: the some n to 2 n groups that reach tau are all that is read again
// (from L2), and the few elements above tau are ranked by counting. Elements
// equal to tau enter by lowest id. Rows where too many elements pass (values
// that cluster in few threads) raise tau to the exact n-th largest value by
// bisection first.
//
// Bound: bytes, the row read once. 4096 x 128256 bf16, normal logits: 191 us
// without alternatives (5500 GB/s of the 6454 that a copy reaches), 223 with one,
// 242 with 20 (233 where a model's peaks stand out), 282 with 64: a row's last
// steps are some thousands of clocks of barriers and dependent reads, which the
// SM's other three CTAs hide in part. fp32 512 x 151936: 55 us without
// alternatives (5640 GB/s), 71 with 64. Four CTAs of 256 threads an SM, not two
// of 512 (207 us): more rows end at different times. CTAs that keep to an SM
// and fetch the next row's start ahead were slower (224 us). The inner loop
// leaves checks to the two vectors that need them (233 us with them inside).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "common/launch.h"
#include "common/tmap.h"
#include "logits/logits_api.h"
#include "logits/rows.cuh"

namespace b200 {
namespace {

using namespace rows;

constexpr int NT = 256;
constexpr int kWarps = NT / 32;
constexpr int U = 4;          // vectors of a thread worked on at a time
constexpr int kCand = 512;    // elements above tau kept before tau is raised
constexpr int kEq = 256;      // elements equal to tau kept before they are found in id order
constexpr int kHits = 512;    // groups read again by themselves; more: the whole slice
constexpr int kSlots = 64;    // groups of a thread where CTAs can be added
constexpr int kBwdThreads = 128;  // (256: 357 us instead of 317 at 4096 x 128256)
constexpr int kMaxCluster = 8;

struct FwdParams {
  const void* x;
  const void* ids;
  int64_t ld;
  int V, top_n;
  bool ids64;
  float c, inv_t;  // log2(e) / T, 1 / T
  float least;     // floor_of(c)
  float* logprob;
  int* rank;
  float* entropy;
  float* lse;
  int* top_ids;
  float* top_lp;
  float4* stats;
};

struct Smem {
  Acc acc[kWarps];
  int cnt[kWarps];
  uint32_t jth[kWarps];        // each warp's j-th largest maximum
  int hit[kHits];              // group * NT + thread of those that reach tau
  unsigned long long cand[kCand + kEq];
  int eq[kEq];
  int scan[kWarps];
  int n_hit, n_gt, n_eq, n_at;
  float m, log2_s;
  // filled by the CTAs of the cluster in rank 0's copy
  Acc part[kMaxCluster];
  int part_cnt[kMaxCluster];
  unsigned long long merged[kMaxCluster * kMaxTopN];
};

// (key, lowest id first) as one number, larger = earlier.
__device__ __forceinline__ unsigned long long entry(uint32_t key, int id) {
  return ((unsigned long long)key << 32) | (uint32_t)~(uint32_t)id;
}

// The key that n of the CTA's thread maxima reach (see the head of this file),
// from the warps' j-th largest in sm.jth.
__device__ __forceinline__ uint32_t find_tau(const Smem& sm, int n) {
  const int j = (n + kWarps - 1) / kWarps, need = (n + j - 1) / j;
  const uint32_t k = sm.jth[threadIdx.x % kWarps];
  int reach = 0;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) reach += sm.jth[i] >= k ? 1 : 0;
  return __reduce_max_sync(0xffffffffu, reach >= need ? k : 0u);
}

// Calls f(key, id) for every element of the groups in sm.hit.
template <typename T, typename F>
__device__ __forceinline__ void visit(const Smem& sm, const Row<T>& row, const Slice& sl,
                                      F f) {
  const int n_groups = (sl.b - sl.a + U * NT - 1) / (U * NT);
  const bool all = sm.n_hit > kHits;
  const int n = all ? sl.hi - sl.lo : sm.n_hit * U;
  for (int w = threadIdx.x; w < n; w += NT) {
    int u = sl.lo + w;
    if (!all) {
      const int h = sm.hit[w / U], it = h / NT, t = h % NT, k = w % U;
      u = sl.a + (it * U + k) * NT + t;
      if (it == n_groups) u = k > 0 ? -1 : t == 0 ? sl.head : t == 1 ? sl.tail : -1;
      else if (u >= sl.b) u = -1;
      if (u < 0) continue;
    }
    const uint4 v = row.load(u);
#pragma unroll
    for (int i = 0; i < Traits<T>::E / 2; ++i) {
      float a, b;
      Traits<T>::pair(v, i, a, b);
      const int id = row.index(u, 2 * i);
      if (id >= 0 && id < row.V) f(key_of(a), id);
      if (id + 1 >= 0 && id + 1 < row.V) f(key_of(b), id + 1);
    }
  }
}

// Elements above tau into sm.cand (up to kCand; sm.n_gt counts them, or is
// larger than that), the ids of those equal to it into sm.eq (up to kEq;
// sm.n_eq likewise).
// The order in which they arrive does not matter: the lists are ranked.
template <typename T>
__device__ __forceinline__ void collect(Smem& sm, const Row<T>& row, const Slice& sl,
                                        uint32_t tau) {
  visit(sm, row, sl, [&](uint32_t k, int id) {
    // (Counts above what the lists hold only say so.)
    if (k > tau) {
      if (*(volatile int*)&sm.n_gt > kCand) return;
      const int at = atomicAdd(&sm.n_gt, 1);
      if (at < kCand) sm.cand[at] = entry(k, id);
    } else if (k == tau) {
      if (*(volatile int*)&sm.n_eq > kEq) return;
      const int at = atomicAdd(&sm.n_eq, 1);
      if (at < kEq) sm.eq[at] = id;
    }
  });
  __syncthreads();
}

// Exact n-th largest key among the elements of the groups in sm.hit (more
// than n of them lie above the present tau).
template <typename T>
__device__ __noinline__ uint32_t raise_tau(Smem& sm, Row<T> row, Slice sl, int n) {
  uint32_t tau = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t cand = tau | (1u << b);
    __syncthreads();
    if (threadIdx.x == 0) sm.n_at = 0;
    __syncthreads();
    int c = 0;
    visit(sm, row, sl, [&](uint32_t k, int) { c += k >= cand ? 1 : 0; });
    c = __reduce_add_sync(0xffffffffu, c);
    if (threadIdx.x % 32 == 0 && c) atomicAdd(&sm.n_at, c);
    __syncthreads();
    if (sm.n_at >= n) tau = cand;
  }
  if (threadIdx.x == 0) sm.n_gt = sm.n_eq = 0;
  __syncthreads();
  return tau;
}

// The lowest ids whose key is tau, up to `need` (<= kEq), into sm.eq[0 ..
// sm.n_eq): vectors in index order, NT at a time, until enough are found. For
// rows where very many elements tie (a mask leaves fewer than n): there the
// first vectors hold enough.
template <typename T>
__device__ __noinline__ void collect_equal(Smem& sm, Row<T> row, Slice sl, uint32_t tau, int need) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int found = 0;  // uniform
  for (int u0 = sl.lo; u0 < sl.hi && found < need; u0 += NT) {
    const int u = u0 + threadIdx.x;
    uint32_t mask = 0;  // bit e: element e of my vector equals tau
    if (u < sl.hi) {
      const uint4 v = row.load(u);
#pragma unroll
      for (int i = 0; i < Traits<T>::E / 2; ++i) {
        float a, b;
        Traits<T>::pair(v, i, a, b);
        const int id = row.index(u, 2 * i);
        if (id >= 0 && id < row.V && key_of(a) == tau) mask |= 1u << (2 * i);
        if (id + 1 >= 0 && id + 1 < row.V && key_of(b) == tau) mask |= 2u << (2 * i);
      }
    }
    const int mine = __popc(mask);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 31) sm.scan[warp] = incl;
    __syncthreads();
    int before = found, total = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    int at = before + incl - mine;
    for (int e = 0; e < Traits<T>::E; ++e)
      if ((mask >> e) & 1u) {
        if (at < need) sm.eq[at] = row.index(u, e);
        ++at;
      }
    found += total;
  }
  __syncthreads();
  if (threadIdx.x == 0) sm.n_eq = min(found, need);
  __syncthreads();
}

// This thread's sums where its warp's maximum lies far out: element by element
// against its own maximum.
template <typename T>
__device__ __noinline__ Acc slow_sums(Row<T> row, Slice sl, float c) {
  Acc a{-INFINITY, 0.f, 0.f};
  for_vectors<NT>(sl, [&](int u) {
    const uint4 v = row.load(u);
    const float mx = Traits<T>::max_of(v);
    if (mx > a.m) rebase(a, mx, c);
    const float m = shift_of(a.m);
#pragma unroll
    for (int i = 0; i < Traits<T>::E / 2; ++i) {
      float x[2];
      Traits<T>::pair(v, i, x[0], x[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float d = (x[k] - m) * c, e = ex2(d);
        a.s += e;
        a.t += e == 0.f ? 0.f : e * d;
      }
    }
  });
  return a;
}

// How many of list[0 .. n) are larger than e, for groups of 4 threads that
// share an e; all of them get it.
__device__ __forceinline__ int rank_of(const unsigned long long* list, int n,
                                       unsigned long long e) {
  int before = 0;
  for (int j = threadIdx.x % 4; j < n; j += 4) before += list[j] > e ? 1 : 0;
  before += __shfl_xor_sync(0xffffffffu, before, 1);
  before += __shfl_xor_sync(0xffffffffu, before, 2);
  return before;
}

// CL CTAs a row. TOP: alternatives wanted.
template <typename T, int CL, bool TOP>
__global__ void __launch_bounds__(NT, 4) token_logprobs_kernel(const FwdParams p) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  __shared__ Smem sm;
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / CL;
  const int part = blockIdx.x % CL;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int n = p.top_n;
  if (TOP && tid == 0) sm.n_hit = sm.n_gt = sm.n_eq = 0;
  // Every CTA of the cluster has started before its memory is written to.
  if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  const Row<T> row(p.x, r, p.ld, p.V);
  const Slice sl(row, part, CL);
  const int64_t y = load_id(p.ids, p.ids64, r);
  const bool has_y = y >= 0 && y < p.V;
  const float xy = has_y ? Tr::to_f(row.x[y]) : NAN;
  const int uy = has_y ? ((int)y + row.pad) / E : 0x7fffffff;
  const float c = p.c;

  // Sums against r = the rounded m c of the thread's maximum m so far: one
  // fused product an element. (rows.cuh's form follows at the end: r's own
  // rounding is taken out of s and t.)
  float m = -INFINITY, r0 = 0.f, s = 0.f, t = 0.f;
  uint32_t cnt = 0;
  const uint64_t c2 = f32x2_pack(c, c);
  // A given token at -inf ties with everything that is masked: those before
  // it are counted on their own.
  const bool y_masked = xy == -INFINITY;
  extern __shared__ uint16_t slots[];
  int n_slots = 0;
  for_groups<NT, U>(row, sl, [&](const uint4(&v)[U], int u, int it) {
    typename Tr::Max vm[U];
#pragma unroll
    for (int k = 0; k < U; ++k) vm[k] = Tr::vmax(v[k]);
    static_assert(U == 4, "tree of maxima");
    const float mx = Tr::value(Tr::vmax(Tr::vmax(vm[0], vm[1]), Tr::vmax(vm[2], vm[3])));
    if constexpr (TOP) {
      // The upper half of the float keeps the order.
      slots[it * NT + tid] = (uint16_t)(__float_as_uint(mx) >> 16);
      n_slots = it + 1;
    }
    if (mx > m) {
      const float rn = __fmul_rn(fmaxf(mx, p.least), c), d = r0 - rn;
      const float f = m == -INFINITY ? 0.f : ex2(d);
      t = f == 0.f ? 0.f : f * (t + d * s);
      s = f == 0.f ? 0.f * s : f * s;
      m = mx;
      r0 = rn;
    }
    const uint64_t nr2 = f32x2_pack(-r0, -r0);
    uint64_t s2 = f32x2_pack(0.f, 0.f), t2 = s2;
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float xa, xb, da, db;
        Tr::pair_floor(v[k], i, p.least, xa, xb);
        const uint64_t d2 = f32x2_fma(f32x2_pack(xa, xb), c2, nr2);
        f32x2_unpack(d2, da, db);
        const uint64_t e2 = f32x2_pack(ex2(da), ex2(db));
        s2 = f32x2_add(s2, e2);
        t2 = f32x2_fma(e2, d2, t2);
      }
      // Elements before y: most vectors hold none above it.
      const int uk = u + k * NT;
      if (!Tr::all_below(vm[k], xy)) {
        if (uk < uy && !y_masked)
          Tr::template count<true>(v[k], xy, cnt);
        else if (uk != uy)
          Tr::template count<false>(v[k], xy, cnt);
      }
    }
    float s0, s1, t0, t1;
    f32x2_unpack(s2, s0, s1);
    f32x2_unpack(t2, t0, t1);
    s += s0 + s1;
    t += t0 + t1;
  });
  int n_before = Tr::counted(cnt);
  if (y_masked)
    for (int u = sl.lo + tid; u < min(sl.hi, uy); u += NT) {
      const uint4 v = row.load(u);
      for (int i = 0; i < E / 2; ++i) {
        float xa, xb;
        Tr::pair(v, i, xa, xb);
        const int id = row.index(u, 2 * i);
        n_before += id >= 0 && id < p.V && xa == -INFINITY;
        n_before += id + 1 >= 0 && id + 1 < p.V && xb == -INFINITY;
      }
    }
  if (has_y && uy >= sl.lo && uy < sl.hi && (uy - sl.lo) % NT == tid) {
    // The vector that holds y, element by element.
    const uint4 v = row.load(uy);
    for (int i = 0; i < E / 2; ++i) {
      float xa, xb;
      Tr::pair(v, i, xa, xb);
      const int id = row.index(uy, 2 * i);
      if (id >= 0 && id < p.V) n_before += xa > xy || (xa == xy && id < y);
      if (id + 1 >= 0 && id + 1 < p.V) n_before += xb > xy || (xb == xy && id + 1 < y);
    }
  }

  // A warp's sums against its own maximum, in a fixed order.
  const uint32_t key = key_of(m);
  const uint32_t key_w = __reduce_max_sync(0xffffffffu, key);
  const float m_w = value_of(key_w);
  Acc a{m, s, t};
  if (!slow_range(m_w, c, kFarEntropy)) {
    const float e = fmaf(m, c, -r0);  // what r lacks of m c
    if (m > p.least) {
      a.t = (t - e * s) * ex2(-e);
      a.s = s * ex2(-e);
    } else {
      a = Acc{-INFINITY, s != s ? s : 0.f, 0.f};  // nothing against the warp's maximum
    }
  } else if (m_w == -INFINITY) {
    a = Acc{-INFINITY, s != s ? s : 0.f, 0.f};
  } else {
    a = slow_sums(row, sl, c);
  }
  rebase(a, m_w, c);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  n_before = __reduce_add_sync(0xffffffffu, n_before);
  if (lane == 0) {
    sm.acc[warp] = a;
    sm.cnt[warp] = n_before;
  }
  if constexpr (TOP) {
    uint32_t left = key, jth = key_w;
    for (int j = (n + kWarps - 1) / kWarps; j > 1; --j) {
      if (lane == __ffs(__ballot_sync(0xffffffffu, left == jth)) - 1) left = 0u;
      jth = __reduce_max_sync(0xffffffffu, left);
    }
    if (lane == 0) sm.jth[warp] = jth;
  }
  __syncthreads();

  // Warp 0 adds the warps up, and where the row is one CTA's, finishes it.
  auto finish = [&](const Acc& q, int k) {
    const bool empty = q.m == -INFINITY && q.s == 0.f;  // nothing above -inf, no NaN
    const float m0 = shift_of(q.m);
    const float l2 = log2f(q.s);  // -inf for an empty row
    const float ent = empty ? 0.f : (l2 - q.t / q.s) * kLn2;
    p.entropy[r] = ent;
    p.lse[r] = fmaf(m0, p.inv_t, l2 * kLn2);
    const float lp = empty ? -INFINITY : fmaf(xy - m0, p.inv_t, -l2 * kLn2);
    p.logprob[r] = has_y ? lp : 0.f;
    p.rank[r] = has_y && xy == xy ? k + 1 : 0;
    const float inv = empty ? 0.f : 1.f / q.s;
    p.stats[r] = make_float4(m0, inv, empty ? 0.f : l2, ent);
    sm.m = m0;
    sm.log2_s = empty ? INFINITY : l2;
  };
  if (warp == 0) {
    Acc q = lane < kWarps ? sm.acc[lane] : Acc{-INFINITY, 0.f, 0.f};
    rebase(q, value_of(__reduce_max_sync(0xffffffffu, key_of(q.m))), c);
    q.s = warp_sum(q.s);
    q.t = warp_sum(q.t);
    const int k = __reduce_add_sync(0xffffffffu, lane < kWarps ? sm.cnt[lane] : 0);
    if constexpr (CL == 1) {
      if (lane == 0) finish(q, k);
    } else {
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      if (lane == 0) {
        const uint32_t dst = mapa_shared(smem_u32(&sm.part[part]), 0);
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(q.m) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(q.s) : "memory");
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(q.t) : "memory");
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(
                         mapa_shared(smem_u32(&sm.part_cnt[part]), 0)),
                     "r"(k)
                     : "memory");
      }
    }
  } else if constexpr (CL > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }

  // The CTA's first n elements: `n_list` entries of sm.cand, those among them.
  int n_list = 0;
  if constexpr (TOP) {
    uint32_t tau = find_tau(sm, n);
    if (key >= tau) {
      uint32_t tau_up = key_of(__uint_as_float(__float_as_uint(value_of(tau)) & 0xffff0000u));
      // Nothing but -inf reaches tau: groups of those are not read again, the
      // first of them are found in id order.
      const bool masked = tau == key_of(-INFINITY);
      tau_up += masked ? 1u : 0u;
      if (masked) sm.n_eq = kEq + 1;
#pragma unroll 4
      for (int i = 0; i < n_slots; ++i)
        if (key_of(__uint_as_float((uint32_t)slots[i * NT + tid] << 16)) >= tau_up) {
          const int at = atomicAdd(&sm.n_hit, 1);
          if (at < kHits) sm.hit[at] = i * NT + tid;
        }
    }
    __syncthreads();
    collect(sm, row, sl, tau);
    if (sm.n_gt > kCand) {
      tau = raise_tau(sm, row, sl, n);
      collect(sm, row, sl, tau);
    }
    const int n_gt = min(sm.n_gt, kCand);
    n_list = n_gt;
    if (n_gt < n) {
      if (sm.n_eq > kEq) collect_equal(sm, row, sl, tau, n - n_gt);
      const int n_eq = sm.n_eq;
      if (tid < n_eq) sm.cand[n_gt + tid] = entry(tau, sm.eq[tid]);
      n_list += n_eq;
      __syncthreads();
    }
  }

  if constexpr (CL > 1) {
    if constexpr (TOP) {
      // Its first n, by rank, into rank 0's list; empty places hold 0.
      const uint32_t dst = mapa_shared(smem_u32(&sm.merged[part * kMaxTopN]), 0);
      if (tid < n && tid >= n_list)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + tid * 8), "l"(0ull) : "memory");
      for (int i0 = 0; i0 < n_list; i0 += NT / 4) {
        const int i = i0 + tid / 4;
        const unsigned long long e = i < n_list ? sm.cand[i] : 0ull;
        const int before = rank_of(sm.cand, n_list, e);
        if (i < n_list && before < n && tid % 4 == 0)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + before * 8), "l"(e)
                       : "memory");
      }
    }
    cluster_sync_all();
    if (part != 0) return;
    if (warp == 0) {
      Acc q = lane < CL ? sm.part[lane] : Acc{-INFINITY, 0.f, 0.f};
      rebase(q, value_of(__reduce_max_sync(0xffffffffu, key_of(q.m))), c);
      q.s = warp_sum(q.s);
      q.t = warp_sum(q.t);
      const int k = __reduce_add_sync(0xffffffffu, lane < CL ? sm.part_cnt[lane] : 0);
      if (lane == 0) finish(q, k);
    }
    if constexpr (TOP) {
      // The CTAs' lists, closed up.
      const int i = tid;
      for (int j = i; j < CL * n; j += NT) sm.cand[j] = sm.merged[j / n * kMaxTopN + j % n];
      n_list = CL * n;
      __syncthreads();
    }
  }
  if constexpr (TOP) {
    // sm.m and sm.log2_s: written before the last barrier.
    const float m0 = sm.m, l2 = sm.log2_s;
    for (int i0 = 0; i0 < n_list; i0 += NT / 4) {
      const int i = i0 + tid / 4;
      const unsigned long long e = i < n_list ? sm.cand[i] : 0ull;
      const int before = rank_of(sm.cand, n_list, e);
      if (e != 0 && before < n && tid % 4 == 0) {
        p.top_ids[r * n + before] = (int)~(uint32_t)e;
        p.top_lp[r * n + before] = fmaf(value_of((uint32_t)(e >> 32)) - m0, p.inv_t, -l2 * kLn2);
      }
    }
    // Places that no element fills (fewer than n numbers in the row).
    const int have = rank_of(sm.cand, n_list, 0ull);
    if (tid < n && tid >= have) {
      p.top_ids[r * n + tid] = -1;
      p.top_lp[r * n + tid] = -INFINITY;
    }
  }
}

// dx_j = (g_lp ([j = y] - p_j) - g_H p_j (log p_j + H)) / T. Elementwise on
// the saved (m, 1 / s, log2 s, H): reads the logits once, writes the gradient
// once. One CTA a (row, chunk of kBwdThreads * U vectors). Bound: bytes; 4096 x
// 128256 bf16 321 us (6550 GB/s; a copy of the same tensor 323), fp32 512 x 151936
// 102 (6130).
struct BwdParams {
  const void* x;
  const void* ids;
  int64_t ld;
  int V;
  bool ids64;
  float c, inv_t;
  const float4* stats;
  const float* g_lp;
  const float* g_ent;
  void* grad;
};

template <typename T, bool ENT>
__global__ void __launch_bounds__(kBwdThreads) token_logprobs_bwd_kernel(const BwdParams p) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.y;
  const Row<T> row(p.x, r, p.ld, p.V);
  T* out = reinterpret_cast<T*>(p.grad) + r * p.V;
  const int64_t y = load_id(p.ids, p.ids64, r);
  const bool has_y = y >= 0 && y < p.V;
  const float4 st = p.stats[r];
  const float c = p.c;
  const float gl = p.g_lp && has_y ? p.g_lp[r] * p.inv_t : 0.f;
  const float ge = ENT ? p.g_ent[r] * p.inv_t : 0.f;
  // Nothing comes back to this row: its gradient is zero whatever it holds.
  // (A row without a distribution, 1 / s = 0, has none to pass on either.)
  const bool none = (gl == 0.f && ge == 0.f) || st.y == 0.f;
  // Coefficients of p_j and of p_j log2 p_j.
  const float k0 = -gl - ge * st.w, k1 = -ge * kLn2;
  const uint64_t c2 = f32x2_pack(c, c), nm2 = f32x2_pack(-st.x, -st.x);
  // The gradient rows are contiguous: their alignment is their own.
  const int u0 = blockIdx.x * (kBwdThreads * U) + threadIdx.x;
  uint4 v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * kBwdThreads;
    v[k] = u < row.n_vec && !none ? row.load(u) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * kBwdThreads;
    if (u >= row.n_vec) break;
    float g[E];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      float xa, xb, da, db;
      Tr::pair(v[k], i, xa, xb);
      f32x2_unpack(f32x2_mul(f32x2_add(f32x2_pack(xa, xb), nm2), c2), da, db);
      const float pa = ex2(da) * st.y, pb = ex2(db) * st.y;
      if constexpr (ENT) {
        // p log2 p; a zero p (its logarithm may be -inf) adds nothing
        g[2 * i] = pa * fmaf(k1, fmaxf(da, -1e4f) - st.z, k0);
        g[2 * i + 1] = pb * fmaf(k1, fmaxf(db, -1e4f) - st.z, k0);
      } else {
        g[2 * i] = pa * k0;
        g[2 * i + 1] = pb * k0;
      }
    }
    if (none) {
#pragma unroll
      for (int e = 0; e < E; ++e) g[e] = 0.f;
    }
    const int id0 = row.index(u, 0);
    if (has_y && !none && y >= id0 && y < id0 + E) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (id0 + e == y) g[e] += gl;
    }
    T* dst = out + id0;
    if (row.full(u) && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
      *reinterpret_cast<uint4*>(dst) = Tr::pack(g);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (id0 + e >= 0 && id0 + e < p.V) dst[e] = Tr::from_f(g[e]);
    }
  }
}

// Groups of a thread where CL CTAs share a row, a last one for the partial
// vectors among them.
template <typename T>
int groups_of(int V, int cl) {
  const int n_vec = (V + 2 * Traits<T>::E - 2) / Traits<T>::E;
  return ((n_vec + cl - 1) / cl + U * NT - 1) / (U * NT) + 1;
}
// Their maxima's bytes at the largest vocabulary, 8 CTAs a row.
constexpr int kSlotBytes = ((kMaxVocab / 4 + 2) / kMaxCluster / (U * NT) + 2) * NT * 2;

template <typename T, int CL>
void launch_fwd(const FwdParams& p, int64_t rows, cudaStream_t stream) {
  cudaLaunchAttribute cl;
  cl.id = cudaLaunchAttributeClusterDimension;
  cl.val.clusterDim.x = CL;
  cl.val.clusterDim.y = cl.val.clusterDim.z = 1;
  const dim3 grid((unsigned)(rows * CL));
  const cudaLaunchAttribute* extra = CL > 1 ? &cl : nullptr;
  auto kernel = p.top_n > 0 ? token_logprobs_kernel<T, CL, true> : token_logprobs_kernel<T, CL, false>;
  static bool attr[kMaxDevices] = {};
  if (p.top_n > 0) set_smem_attr_once(kernel, kSlotBytes, attr, "token_logprobs");
  const int smem = p.top_n > 0 ? groups_of<T>(p.V, CL) * NT * 2 : 0;
  launch_pdl(kernel, grid, dim3(NT), smem, stream, extra, p);
}

template <typename T>
void launch_fwd_t(const FwdParams& p, int64_t rows, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  int cl = row_split(rows, p.V / Traits<T>::E, 4 * num_sms(dev), NT);
  // (32 KB of maxima a CTA: four an SM)
  while (p.top_n > 0 && cl < kMaxCluster && groups_of<T>(p.V, cl) > kSlots) cl *= 2;
  switch (cl) {
    case 1: return launch_fwd<T, 1>(p, rows, stream);
    case 2: return launch_fwd<T, 2>(p, rows, stream);
    case 4: return launch_fwd<T, 4>(p, rows, stream);
    default: return launch_fwd<T, 8>(p, rows, stream);
  }
}

void check_rows(const LogitRows& in, const char* what) {
  if (in.V < 1 || in.V > kMaxVocab)
    throw std::runtime_error(std::string(what) + ": vocabulary outside [1, 2^22]");
  if (in.rows > (1 << 24)) throw std::runtime_error(std::string(what) + ": more than 2^24 rows");
}

}  // namespace

void token_logprobs_launch(const TokenLogprobsArgs& a, cudaStream_t stream) {
  check_rows(a.in, "token_logprobs");
  if (a.top_n < 0 || a.top_n > kMaxTopN || a.top_n > a.in.V)
    throw std::runtime_error("token_logprobs: top_n must be in [0, min(64, vocabulary)]");
  if (a.in.rows <= 0) return;
  FwdParams p{a.in.x,  a.ids,       a.in.ld,    a.in.V,
              a.top_n, a.ids64,     (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
              floor_of((float)(1.4426950408889634 / a.temperature)),
              a.logprob, a.rank,    a.entropy,  a.lse,
              a.top_ids, a.top_lp,  reinterpret_cast<float4*>(a.stats)};
  if (a.in.bf16)
    launch_fwd_t<__nv_bfloat16>(p, a.in.rows, stream);
  else
    launch_fwd_t<float>(p, a.in.rows, stream);
}

void token_logprobs_bwd_launch(const TokenLogprobsBwdArgs& a, cudaStream_t stream) {
  check_rows(a.in, "token_logprobs_bwd");
  if (a.in.rows <= 0) return;
  BwdParams p{a.in.x, a.ids, a.in.ld, a.in.V, a.ids64,
              (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
              reinterpret_cast<const float4*>(a.stats), a.g_logprob, a.g_entropy, a.grad};
  const int E = a.in.bf16 ? 8 : 4;
  const unsigned chunks = (unsigned)((a.in.V + 2 * E - 2) / E + kBwdThreads * U - 1) / (kBwdThreads * U);
  // grid.y holds at most 65535 rows a launch
  for (int64_t r0 = 0; r0 < a.in.rows; r0 += 65535) {
    const unsigned n = (unsigned)(a.in.rows - r0 < 65535 ? a.in.rows - r0 : 65535);
    BwdParams q = p;
    const int64_t eb = a.in.bf16 ? 2 : 4;
    q.x = reinterpret_cast<const char*>(p.x) + r0 * p.ld * eb;
    q.ids = reinterpret_cast<const char*>(p.ids) + r0 * (p.ids64 ? 8 : 4);
    q.stats = p.stats + r0;
    q.g_lp = p.g_lp ? p.g_lp + r0 : nullptr;
    q.g_ent = p.g_ent ? p.g_ent + r0 : nullptr;
    q.grad = reinterpret_cast<char*>(p.grad) + r0 * p.V * eb;
    const dim3 grid(chunks, n);
    if (a.in.bf16) {
      if (a.g_entropy)
        launch_pdl(token_logprobs_bwd_kernel<__nv_bfloat16, true>, grid, dim3(kBwdThreads), 0, stream,
                   nullptr, q);
      else
        launch_pdl(token_logprobs_bwd_kernel<__nv_bfloat16, false>, grid, dim3(kBwdThreads), 0, stream,
                   nullptr, q);
    } else {
      if (a.g_entropy)
        launch_pdl(token_logprobs_bwd_kernel<float, true>, grid, dim3(kBwdThreads), 0, stream, nullptr, q);
      else
        launch_pdl(token_logprobs_bwd_kernel<float, false>, grid, dim3(kBwdThreads), 0, stream, nullptr, q);
    }
  }
}

}  // namespace b200
