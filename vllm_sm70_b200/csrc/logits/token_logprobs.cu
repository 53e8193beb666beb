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
// over the row: the n-th largest of the THREADS' maxima, tau, is a lower bound
// of the row's n-th largest value (n threads hold an element that large), so
// every alternative is an element >= tau of a thread whose maximum is >= tau.
// About n threads qualify; only their elements are read again (from L2), and
// the few above tau are ranked by counting. Elements equal to tau enter by
// lowest id. Rows where too many elements pass (values that cluster in few
// threads) raise tau to the exact n-th largest value by bisection first.
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

constexpr int NT = 512;
constexpr int kWarps = NT / 32;
constexpr int U = 4;          // vectors of a thread in flight
constexpr int kCand = 512;    // elements above tau kept before tau is raised
constexpr int kEq = 256;      // elements equal to tau kept before they are found in id order
constexpr int kMaxCluster = 8;

struct FwdParams {
  const void* x;
  const void* ids;
  int64_t ld;
  int V, top_n;
  bool ids64;
  float c, inv_t;  // log2(e) / T, 1 / T
  float* logprob;
  int* rank;
  float* entropy;
  float* lse;
  int* top_ids;
  float* top_lp;
  float4* stats;
};

struct Smem {
  float red[kWarps];
  Acc acc[kWarps];
  int cnt[kWarps];
  uint32_t tmax[NT];           // key of each thread's maximum
  int qual[NT];                // threads with elements >= tau
  unsigned long long cand[kCand + kEq];
  int eq[kEq];
  int scan[kWarps];
  int n_qual, n_gt, n_eq, n_hit;
  uint32_t tau;
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

// Largest key k with at least n of the CTA's thread maxima >= k (n <= NT).
// Warp 0 bisects over the key's bits with 16 maxima a lane in registers.
template <typename T>
__device__ void find_tau(Smem& sm, int n) {
  if (threadIdx.x < 32) {
    uint32_t k[kWarps];
#pragma unroll
    for (int i = 0; i < kWarps; ++i) k[i] = sm.tmax[i * 32 + threadIdx.x];
    uint32_t tau = 0;
    for (int b = 31; b >= Traits<T>::kKeyLowBit; --b) {
      const uint32_t cand = tau | (1u << b);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) c += k[i] >= cand ? 1 : 0;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c >= n) tau = cand;
      if (c == n) break;  // any bound that n maxima reach will do
    }
    // The bound as a key that an element can have: the smallest maximum
    // above it, so that "equal to tau" means something.
    uint32_t low = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kWarps; ++i)
      if (k[i] >= tau) low = min(low, k[i]);
    low = __reduce_min_sync(0xffffffffu, low);
    if (threadIdx.x == 0) sm.tau = low;
  }
  __syncthreads();
}

// Calls f(key, id) for every element of the qualified threads' vectors.
template <typename T, typename F>
__device__ __forceinline__ void visit_qualified(const Smem& sm, const Row<T>& row, int u_lo,
                                                int u_hi, F f) {
  const int per = (u_hi - u_lo + NT - 1) / NT;  // vectors of a thread, at most
  for (int w = threadIdx.x; w < sm.n_qual * per; w += NT) {
    const int u = u_lo + sm.qual[w / per] + (w % per) * NT;
    if (u >= u_hi) continue;
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

// Elements above tau into sm.cand (up to kCand; sm.n_gt counts all of them),
// the ids of those equal to it into sm.eq (up to kEq; sm.n_eq counts them).
// The order in which they arrive does not matter: the lists are ranked.
template <typename T>
__device__ void collect(Smem& sm, const Row<T>& row, int u_lo, int u_hi) {
  const uint32_t tau = sm.tau;
  __syncthreads();
  if (threadIdx.x == 0) sm.n_qual = sm.n_gt = sm.n_eq = 0;
  __syncthreads();
  if (sm.tmax[threadIdx.x] >= tau) sm.qual[atomicAdd(&sm.n_qual, 1)] = threadIdx.x;
  __syncthreads();
  visit_qualified(sm, row, u_lo, u_hi, [&](uint32_t k, int id) {
    if (k > tau) {
      const int at = atomicAdd(&sm.n_gt, 1);
      if (at < kCand) sm.cand[at] = entry(k, id);
    } else if (k == tau) {
      const int at = atomicAdd(&sm.n_eq, 1);
      if (at < kEq) sm.eq[at] = id;
    }
  });
  __syncthreads();
}

// Exact n-th largest key among the qualified threads' elements (more than n
// of them lie above the present tau).
template <typename T>
__device__ void raise_tau(Smem& sm, const Row<T>& row, int u_lo, int u_hi, int n) {
  uint32_t tau = 0;
  for (int b = 31; b >= 0; --b) {
    const uint32_t cand = tau | (1u << b);
    __syncthreads();
    if (threadIdx.x == 0) sm.n_hit = 0;
    __syncthreads();
    int c = 0;
    visit_qualified(sm, row, u_lo, u_hi, [&](uint32_t k, int) { c += k >= cand ? 1 : 0; });
    c = __reduce_add_sync(0xffffffffu, c);
    if (threadIdx.x % 32 == 0 && c) atomicAdd(&sm.n_hit, c);
    __syncthreads();
    if (sm.n_hit >= n) tau = cand;
  }
  __syncthreads();
  if (threadIdx.x == 0) sm.tau = tau;
  __syncthreads();
}

// The lowest ids whose key is tau, up to `need` (<= kEq), into sm.eq[0 ..
// sm.n_eq): vectors in index order, NT at a time, until enough are found. For
// rows where very many elements tie (a mask leaves fewer than n): there the
// first vectors hold enough.
template <typename T>
__device__ void collect_equal(Smem& sm, const Row<T>& row, int u_lo, int u_hi, int need) {
  const uint32_t tau = sm.tau;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int found = 0;  // uniform
  for (int u0 = u_lo; u0 < u_hi && found < need; u0 += NT) {
    const int u = u0 + threadIdx.x;
    uint32_t mask = 0;  // bit e: element e of my vector equals tau
    if (u < u_hi) {
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

// CL CTAs a row. TOP: alternatives wanted.
template <typename T, int CL, bool TOP>
__global__ void __launch_bounds__(NT, 2) token_logprobs_kernel(const FwdParams p) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  __shared__ Smem sm;
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / CL;
  const int part = blockIdx.x % CL;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  // Every CTA of the cluster has started before its memory is written to.
  if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  const Row<T> row(p.x, r, p.ld, p.V);
  const int per = (row.n_vec + CL - 1) / CL;
  const int u_lo = min(part * per, row.n_vec), u_hi = min(u_lo + per, row.n_vec);
  const int64_t y = load_id(p.ids, p.ids64, r);
  const bool has_y = y >= 0 && y < p.V;
  const float xy = has_y ? Tr::to_f(row.x[y]) : NAN;
  const int uy = has_y ? ((int)y + row.pad) / E : 0x7fffffff;
  const float c = p.c;

  Acc a{-INFINITY, 0.f, 0.f};
  uint32_t cnt = 0;
  for (int u = u_lo + tid; u < u_hi; u += U * NT) {
    uint4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int uk = u + k * NT;
      v[k] = uk < u_hi ? row.load(uk)
                       : make_uint4(Tr::kNegInf, Tr::kNegInf, Tr::kNegInf, Tr::kNegInf);
    }
    float mx = Tr::max_of(v[0]);
#pragma unroll
    for (int k = 1; k < U; ++k) mx = fmaxf(mx, Tr::max_of(v[k]));
    if (mx > a.m) rebase(a, mx, c);
    const float m = shift_of(a.m);
    const uint64_t c2 = f32x2_pack(c, c), nm2 = f32x2_pack(-m, -m);
    uint64_t s2 = f32x2_pack(0.f, 0.f), t2 = s2;
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float xa, xb, da, db, ea, eb;
        Tr::pair(v[k], i, xa, xb);
        const uint64_t d2 = f32x2_add(f32x2_pack(xa, xb), nm2);
        f32x2_unpack(f32x2_mul(d2, c2), ea, eb);
        const uint64_t e2 = f32x2_pack(ex2(ea), ex2(eb));
        s2 = f32x2_add(s2, e2);
        // -inf times a zero exponential is zero here
        f32x2_unpack(d2, da, db);
        t2 = f32x2_fma(e2, f32x2_pack(fmaxf(da, -1e30f), fmaxf(db, -1e30f)), t2);
      }
      const int uk = u + k * NT;
      if (uk < uy) {
        Tr::template count<true>(v[k], xy, cnt);
      } else if (uk > uy) {
        Tr::template count<false>(v[k], xy, cnt);
      }
    }
    float s0, s1, t0, t1;
    f32x2_unpack(s2, s0, s1);
    f32x2_unpack(t2, t0, t1);
    a.s += s0 + s1;
    a.t += t0 + t1;
  }
  int n_before = Tr::counted(cnt);
  if (has_y && uy >= u_lo && uy < u_hi && (uy - u_lo) % NT == tid) {
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

  // The CTA's sums, in a fixed order.
  const float own_max = a.m;
  if constexpr (TOP) sm.tmax[tid] = key_of(own_max);
  const float m = block_max<NT>(own_max, sm.red);
  rebase(a, m, c);
  a.s = warp_sum(a.s);
  a.t = warp_sum(a.t);
  n_before = __reduce_add_sync(0xffffffffu, n_before);
  if (lane == 0) {
    sm.acc[warp] = a;
    sm.cnt[warp] = n_before;
  }
  __syncthreads();

  // The CTA's first n elements: `n_local` entries of sm.cand.
  int n_local = 0;
  const int n = p.top_n;
  if constexpr (TOP) {
    find_tau<T>(sm, n);
    collect(sm, row, u_lo, u_hi);
    if (sm.n_gt > kCand) {
      raise_tau(sm, row, u_lo, u_hi, n);
      collect(sm, row, u_lo, u_hi);
    }
    const int n_gt = min(sm.n_gt, kCand);
    const int need = max(0, n - n_gt);
    if (need > 0) {
      if (sm.n_eq > kEq) collect_equal(sm, row, u_lo, u_hi, need);
      if (tid < sm.n_eq) sm.cand[n_gt + tid] = entry(sm.tau, sm.eq[tid]);
      __syncthreads();
    }
    n_local = n_gt + (need > 0 ? sm.n_eq : 0);
  }

  unsigned long long* list = sm.cand;
  int n_list = n_local;
  if constexpr (CL > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (tid == 0) {
      Acc q = sm.acc[0];
      int k = sm.cnt[0];
      for (int w = 1; w < kWarps; ++w) {
        q.s += sm.acc[w].s;
        q.t += sm.acc[w].t;
        k += sm.cnt[w];
      }
      const uint32_t dst = mapa_shared(smem_u32(&sm.part[part]), 0);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(q.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 4), "f"(q.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + 8), "f"(q.t) : "memory");
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(
                       mapa_shared(smem_u32(&sm.part_cnt[part]), 0)),
                   "r"(k)
                   : "memory");
    }
    if constexpr (TOP) {
      // Its first n, by rank, into rank 0's list; empty places hold 0.
      const uint32_t dst = mapa_shared(smem_u32(&sm.merged[part * kMaxTopN]), 0);
      if (tid < n && tid >= n_local)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + tid * 8), "l"(0ull) : "memory");
      for (int i = tid; i < n_local; i += NT) {
        const unsigned long long e = sm.cand[i];
        int before = 0;
        for (int j = 0; j < n_local; ++j) before += sm.cand[j] > e ? 1 : 0;
        if (before < n)
          asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dst + before * 8), "l"(e)
                       : "memory");
      }
    }
    cluster_sync_all();
    if (part != 0) return;
  }

  if (tid == 0) {
    Acc q;
    int k;
    if constexpr (CL > 1) {
      float mm = sm.part[0].m;
      for (int i = 1; i < CL; ++i) mm = fmaxf(mm, sm.part[i].m);
      q = Acc{mm, 0.f, 0.f};
      k = 0;
      for (int i = 0; i < CL; ++i) {
        Acc b = sm.part[i];
        rebase(b, mm, c);
        q.s += b.s;
        q.t += b.t;
        k += sm.part_cnt[i];
      }
    } else {
      q = sm.acc[0];
      k = sm.cnt[0];
      for (int w = 1; w < kWarps; ++w) {
        q.s += sm.acc[w].s;
        q.t += sm.acc[w].t;
        k += sm.cnt[w];
      }
    }
    const bool empty = q.m == -INFINITY && q.s == 0.f;  // nothing above -inf, no NaN
    const float m0 = shift_of(q.m);
    const float l2 = log2f(q.s);  // -inf for an empty row
    const float ent = empty ? 0.f : (l2 - q.t / q.s * c) * kLn2;
    p.entropy[r] = ent;
    p.lse[r] = fmaf(m0, p.inv_t, l2 * kLn2);
    const float lp = empty ? -INFINITY : fmaf(xy - m0, p.inv_t, -l2 * kLn2);
    p.logprob[r] = has_y ? lp : 0.f;
    p.rank[r] = has_y && xy == xy ? k + 1 : 0;
    const float inv = empty ? 0.f : 1.f / q.s;
    p.stats[r] = make_float4(m0, inv, empty ? 0.f : l2, ent);
    sm.m = m0;
    sm.log2_s = empty ? INFINITY : l2;
  }
  if constexpr (TOP) {
    if constexpr (CL > 1) {
      // Rank 0's list: CL runs of kMaxTopN places, n used in each.
      list = sm.merged;
      n_list = CL * kMaxTopN;
    }
    __syncthreads();
    const float m0 = sm.m, l2 = sm.log2_s;
    // Places that no element fills (fewer than n numbers in the row).
    if (tid < n) {
      int have = n_list;
      if constexpr (CL > 1) {
        have = 0;
        for (int q = 0; q < CL; ++q)
          for (int j = 0; j < n; ++j) have += list[q * kMaxTopN + j] != 0 ? 1 : 0;
      }
      if (tid >= have) {
        p.top_ids[r * n + tid] = -1;
        p.top_lp[r * n + tid] = -INFINITY;
      }
    }
    for (int i = tid; i < n_list; i += NT) {
      if (CL > 1 && i % kMaxTopN >= n) continue;
      const unsigned long long e = list[i];
      if (CL > 1 && e == 0) continue;
      int before = 0;
      if constexpr (CL > 1) {
        for (int q = 0; q < CL; ++q)
          for (int j = 0; j < n; ++j) before += list[q * kMaxTopN + j] > e ? 1 : 0;
      } else {
        for (int j = 0; j < n_list; ++j) before += list[j] > e ? 1 : 0;
      }
      if (before < n) {
        p.top_ids[r * n + before] = (int)~(uint32_t)e;
        p.top_lp[r * n + before] = fmaf(value_of((uint32_t)(e >> 32)) - m0, p.inv_t, -l2 * kLn2);
      }
    }
  }
}

// dx_j = (g_lp ([j = y] - p_j) - g_H p_j (log p_j + H)) / T. Elementwise on
// the saved (m, 1 / s, log2 s, H): reads the logits once, writes the gradient
// once. One CTA a (row, chunk of NT * U vectors).
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
__global__ void __launch_bounds__(NT) token_logprobs_bwd_kernel(const BwdParams p) {
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
  const int u0 = blockIdx.x * (NT * U) + threadIdx.x;
  uint4 v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * NT;
    v[k] = u < row.n_vec && !none ? row.load(u) : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u0 + k * NT;
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

template <typename T, int CL>
void launch_fwd(const FwdParams& p, int64_t rows, cudaStream_t stream) {
  cudaLaunchAttribute cl;
  cl.id = cudaLaunchAttributeClusterDimension;
  cl.val.clusterDim.x = CL;
  cl.val.clusterDim.y = cl.val.clusterDim.z = 1;
  const dim3 grid((unsigned)(rows * CL));
  const cudaLaunchAttribute* extra = CL > 1 ? &cl : nullptr;
  if (p.top_n > 0)
    launch_pdl(token_logprobs_kernel<T, CL, true>, grid, dim3(NT), 0, stream, extra, p);
  else
    launch_pdl(token_logprobs_kernel<T, CL, false>, grid, dim3(NT), 0, stream, extra, p);
}

template <typename T>
void launch_fwd_t(const FwdParams& p, int64_t rows, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  switch (row_split(rows, p.V / Traits<T>::E, num_sms(dev), NT)) {
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
  const unsigned chunks = (unsigned)((a.in.V + 2 * E - 2) / E + NT * U - 1) / (NT * U);
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
        launch_pdl(token_logprobs_bwd_kernel<__nv_bfloat16, true>, grid, dim3(NT), 0, stream,
                   nullptr, q);
      else
        launch_pdl(token_logprobs_bwd_kernel<__nv_bfloat16, false>, grid, dim3(NT), 0, stream,
                   nullptr, q);
    } else {
      if (a.g_entropy)
        launch_pdl(token_logprobs_bwd_kernel<float, true>, grid, dim3(NT), 0, stream, nullptr, q);
      else
        launch_pdl(token_logprobs_bwd_kernel<float, false>, grid, dim3(NT), 0, stream, nullptr, q);
    }
  }
}

}  // namespace b200
