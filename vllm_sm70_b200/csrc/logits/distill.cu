// Distillation from a teacher's top log-probabilities, forward and backward.
//
// A row has K teacher tokens with log-probs (p_k = exp(lp_k); `tail` false:
// renormalised over the K) and the student's logits x, z = x / T, q =
// softmax(z). With `tail`, the teacher's remaining mass p_t = max(0, 1 - sum
// p_k) is held against the student's mass outside the K, q_t:
//   L = sum_k p_k (log p_k - log q_k)  [+ p_t (log p_t - log q_t)]
//   dL/dz_j = M q_j - P_j               j among the K (P_j: its p, summed
//                                       over repeated ids), M = sum p_k + p_t
//           = (M - p_t / q_t) q_j       other j
// q_t is the sum over the other j themselves (never 1 - sum q_k, which would
// cancel for a student that agrees with its teacher): the row's teacher ids
// are left out of the sum, and their K exponentials are added on their own.
// Each of the two sums stands against its own maximum, m_o and m_i, so that
// neither is lost where the other lies far above it (a student that is sure of
// a teacher's token by 90 nats, which at a low temperature are a few logits):
// log q_t comes from the two logarithms, and the other j's gradient is taken
// against m_o, e_j (M 2^((m_o - m) c) / s - p_t / s_o), e_j = 2^((x_j - m_o) c).
//
// A row with weight 0 has loss 0 and gradient 0 whatever it holds, and is not
// read. Ids outside [0, V) are absent: their mass joins the tail.
//
// Bound: bytes. The training form computes loss and gradient in one kernel:
// the logits are read once, the gradient written once.
//   * A cluster of 1 to 8 CTAs holds a row in shared memory (at 8 CTAs a row
//     as much as an SM has), two or three of them an SM. A warp copies its own
//     part of the row with asynchronous copies, takes out the teacher's
//     elements (they read as -inf from then on), and sums the rest; the warps
//     of the whole cluster exchange (maxima, sums) through each other's shared
//     memory, the row's only meeting. Then each warp writes its part of the
//     gradient, and as it is done with a vector starts the copy of the next
//     row's into its place: the clusters are persistent and memory is read
//     while they work. 4096 x 128256 bf16, K = 64: 446 us, 4710 GB/s of the
//     6454 that a copy reaches. What is left is latency: of a row's ~16000
//     clocks a third is the gradient, a quarter the sums, the rest the
//     teacher's elements and the exchange, on six warps a scheduler. (Rows
//     read twice, the second time from L2: 512 us; a barrier of the cluster
//     instead of words that carry their row's number: 540, it waits for the
//     gradient's stores.)
//   * Rows too long for that (more than 8 CTAs' shared memory) and calls
//     without gradient stream the row; a bitmap of the teacher's ids leaves
//     them out of the sum. 4096 x 128256 bf16 without gradient: 176 us,
//     5970 GB/s; the gradient from saved numbers (distill_bwd): 345 us, 6090.
//   * fp32, 2048 x 128256, K = 64: 162 us without gradient, 425 with it (4940
//     GB/s), 329 from saved numbers.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "common/launch.h"
#include "common/tmap.h"
#include "logits/logits_api.h"
#include "logits/rows.cuh"
#include "ops_api.h"

namespace b200 {
namespace {

using namespace rows;

constexpr int NT = 256;
constexpr int kWarps = NT / 32;
constexpr int U = 4;
constexpr int kBwdThreads = 128;
constexpr int kBwdCtas = 10;  // an SM
static_assert(kMaxTeacherK <= kBwdThreads, "a thread a teacher entry");
constexpr int kMaxCluster = 8;

struct Params {
  const void* x;
  const int* t_ids;
  const float* t_lp;
  const float* weights;
  int64_t ld;
  int V, K;
  int64_t rows;
  bool tail;
  float c, inv_t, gscale;  // log2(e) / T; 1 / T; upstream gradient / T of a row of weight 1
  float least;             // floor_of(c)
  float* row_loss;
  float4* stats;
  void* grad;
  unsigned int* err;
  int* taken;  // rows taken beyond the clusters' first
};

constexpr int kIds = kMaxTeacherK / 32;  // teacher entries a lane holds

// A row's teacher: entry lane + 32 i in every warp's registers.
struct Teacher {
  int id[kIds];      // -1: absent
  float lp[kIds], p[kIds];
  float norm, sum_p;  // subtracted from the given log-probs; sum of p

  __device__ __forceinline__ void load(const int* ids, const float* lps, int K) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      const int k = threadIdx.x % 32 + 32 * i;
      id[i] = k < K ? ids[k] : -1;
      lp[i] = k < K ? lps[k] : -INFINITY;
    }
  }
  // Ids outside the vocabulary are absent; without a tail the rest is
  // renormalised.
  __device__ __forceinline__ void prepare(const Params& q) {
    norm = sum_p = 0.f;
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      if (id[i] >= q.V) id[i] = -1;
    if (!q.tail) {
      float mx = -INFINITY, z = 0.f;
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (id[i] >= 0) mx = fmaxf(mx, lp[i]);
      mx = warp_max(mx);
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (32 * i < q.K && id[i] >= 0) z += expf(lp[i] - mx);
      // A teacher that gives none of its ids any probability has no mass.
      norm = mx == -INFINITY ? 0.f : mx + logf(warp_sum(z));
    }
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      p[i] = 0.f;
      if (32 * i < q.K) {
        if (id[i] >= 0) p[i] = expf(lp[i] -= norm);
        sum_p += p[i];
      }
    }
    sum_p = warp_sum(sum_p);
  }
  // The p of all entries with entry (lane, i)'s id; -1 at those that are not
  // the first of theirs. For all lanes of a warp.
  __device__ __forceinline__ void masses(int K, float (&mass)[kIds]) const {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int i = 0; i < kIds; ++i) mass[i] = 0.f;
    for (int k = 0; k < K; ++k) {
      int idk = -1;
      float pk = 0.f;
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (k / 32 == i) {
          idk = __shfl_sync(0xffffffffu, id[i], k % 32);
          pk = __shfl_sync(0xffffffffu, p[i], k % 32);
        }
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (id[i] == idk && mass[i] != -1.f) {
          if (k < lane + 32 * i)
            mass[i] = -1.f;
          else
            mass[i] += pk;
        }
    }
  }
};

// Which of a lane's entries (bit i: entry lane + 32 i) are the first of their
// id, with kDup set.
constexpr uint32_t kDup = 1u << 31;
__device__ __noinline__ uint32_t first_of_ids(uint32_t own, const int* ids, int K) {
  for (int i = 0; i < kIds; ++i)
    if ((own >> i) & 1u)
      for (int k = 0; k < (int)threadIdx.x % 32 + 32 * i; ++k)
        if (ids[k] == ids[threadIdx.x % 32 + 32 * i]) own &= ~(1u << i);
  return own | kDup;
}
// The p of all entries with this id.
__device__ __noinline__ float mass_of_id(int id, const int* ids, const float* p, int K) {
  float m = 0.f;
  for (int k = 0; k < K; ++k)
    if (ids[k] == id) m += p[k];
  return m;
}

// Maximum and sum of the elements outside the teacher's ids, and of those at
// the ids (the first of each), of a warp, a slice or a row.
struct __align__(16) Sums {  // (exchanged as one vector)
  float m_out, s_out, m_in, s_in;
};

// a's factor to stand against m. (A part without any element above -inf has
// no sum to rebase.)
__device__ __forceinline__ float against(float a, float m, float c) {
  return a == -INFINITY || a == m ? 1.f : ex2((a - m) * c);
}

// Two parts a lane, added up over the warp.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
  Sums q;
  q.m_out = warp_max(fmaxf(a.m_out, b.m_out));
  q.m_in = warp_max(fmaxf(a.m_in, b.m_in));
  q.s_out = warp_sum(a.s_out * against(a.m_out, q.m_out, c) +
                     b.s_out * against(b.m_out, q.m_out, c));
  q.s_in = warp_sum(a.s_in * against(a.m_in, q.m_in, c) + b.s_in * against(b.m_in, q.m_in, c));
  return q;
}

// What the gradient takes of a row. With x against m_out or m:
//   outside: 2^((x - m_out) c) k_out       at an id: 2^((x - m) c) k_in - its p
// k_in (M / s) is 0 for a row without a distribution.
struct Numbers {
  float m_out, k_out, m, k_in, norm;  // norm: the teacher's log-normaliser
};
__device__ __forceinline__ void save(float4* stats, int64_t r, const Numbers& n) {
  stats[2 * r] = make_float4(n.m_out, n.k_out, n.m, n.k_in);
  stats[2 * r + 1] = make_float4(n.norm, 0.f, 0.f, 0.f);
}
__device__ __forceinline__ Numbers saved(const float4* stats, int64_t r) {
  const float4 n = stats[2 * r];
  return Numbers{n.x, n.y, n.z, n.w, stats[2 * r + 1].x};
}
// The sum of all exponentials, against m.
__device__ __forceinline__ float total(const Sums& q, float m, float c) {
  return q.s_out * against(q.m_out, m, c) + q.s_in * against(q.m_in, m, c);
}

__device__ __forceinline__ Numbers row_numbers(float norm, float sum_p, bool tail, const Sums& q,
                                               float c) {
  const float m = fmaxf(q.m_out, q.m_in), s = total(q, m, c);
  const float p_t = tail ? fmaxf(0.f, 1.f - sum_p) : 0.f, mass = sum_p + p_t;
  const float k_in = s == 0.f ? 0.f : mass / s;
  // (Without any mass outside every q_j there is 0.)
  const float k_out = q.s_out == 0.f ? 0.f
                                     : k_in * against(q.m_out, m, c) -
                                           (p_t > 0.f ? p_t / q.s_out : 0.f);
  return Numbers{shift_of(q.m_out), k_out, shift_of(m), k_in, norm};
}

// The row's loss, on a whole warp; xk: the student's logits at the ids.
__device__ __forceinline__ float row_loss(const Teacher& t, const Params& p, const Sums& q,
                                          const float (&xk)[kIds]) {
  const float m = fmaxf(q.m_out, q.m_in), m0 = shift_of(m), s = total(q, m, p.c);
  // An empty row: every log q is -inf, the loss inf where the teacher has mass.
  const float l2 = s == 0.f ? 0.f : log2f(s);
  float loss = 0.f;
  bool any = false;
#pragma unroll
  for (int i = 0; i < kIds; ++i) {
    const float pk = t.p[i];
    any |= t.id[i] >= 0 && t.id[i] < p.V;
    if (pk > 0.f)
      loss += pk * (t.lp[i] - fmaf(xk[i] - m0, p.inv_t, -l2 * kLn2));
    else if (pk != pk)
      loss = pk;
  }
  loss = warp_sum(loss);
  const float p_t = p.tail ? fmaxf(0.f, 1.f - t.sum_p) : 0.f;
  // (Without any token p_t = q_t = 1, in a row without a distribution too.)
  if (p_t > 0.f && __any_sync(0xffffffffu, any))
    loss += p_t * (logf(p_t) - fmaf(q.m_out - m0, p.inv_t, (log2f(q.s_out) - l2) * kLn2));
  return loss;
}

// 2^((x - m) c) of a vector, times coef, for the gradient. kSlow: (x - m)
// rounded by itself; otherwise one fused product against r = the rounded m c,
// whose rounding the caller has put into coef (see rows.cuh).
template <typename T, bool kSlow>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, float c, float m_or_r, float coef) {
  using Tr = Traits<T>;
  float g[Tr::E];
  const uint64_t c2 = f32x2_pack(c, c), n2 = f32x2_pack(-m_or_r, -m_or_r),
                 k2 = f32x2_pack(coef, coef);
#pragma unroll
  for (int i = 0; i < Tr::E / 2; ++i) {
    float a, b, da, db;
    Tr::pair(v, i, a, b);
    const uint64_t x2 = f32x2_pack(a, b);
    f32x2_unpack(kSlow ? f32x2_mul(f32x2_add(x2, n2), c2) : f32x2_fma(x2, c2, n2), da, db);
    f32x2_unpack(f32x2_mul(f32x2_pack(ex2(da), ex2(db)), k2), g[2 * i], g[2 * i + 1]);
  }
  return Tr::pack(g);
}

// The elements of vector u that the row has, one by one.
template <typename T>
__device__ __forceinline__ void store_part(T* out, const Row<T>& row, int u, const uint4& v) {
  constexpr int E = Traits<T>::E;
  const int id0 = row.index(u, 0);
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (id0 + i >= 0 && id0 + i < row.V) out[id0 + i] = e[i];
}
template <typename T>
__device__ __forceinline__ void store_vec(T* out, const Row<T>& row, int u, const uint4& v) {
  T* dst = out + row.index(u, 0);
  if (row.full(u) && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0)
    *reinterpret_cast<uint4*>(dst) = v;
  else
    store_part(out, row, u, v);
}

// This thread's part of a streamed slice's sum, against m, element by element.
template <typename T>
__device__ __noinline__ float slow_sum(Row<T> row, Slice sl, const uint8_t* bitmap, float m,
                                       float c) {
  float s = 0.f;
  for_vectors<NT>(sl, [&](int u) {
    uint4 v = row.load(u);
    Traits<T>::blank(v, bitmap[u - sl.lo]);
    for (int i = 0; i < Traits<T>::E / 2; ++i) {
      float a, b;
      Traits<T>::pair(v, i, a, b);
      s += ex2((a - m) * c) + ex2((b - m) * c);
    }
  });
  return s;
}

// A value and the number of the exchange that it belongs to, as one 8-byte
// word: who sees the number sees the value, so no fence is needed (one would
// wait for the gradient's stores).
__device__ __forceinline__ unsigned long long word_of(float v, uint32_t seq) {
  return ((unsigned long long)seq << 32) | __float_as_uint(v);
}
template <int CL>
__device__ __forceinline__ void send(unsigned long long* to, int rank, float v, uint32_t seq) {
  if constexpr (CL == 1)
    *reinterpret_cast<volatile unsigned long long*>(to) = word_of(v, seq);
  else
    asm volatile("st.relaxed.cluster.shared::cluster.b64 [%0], %1;" ::"r"(
                     mapa_shared(smem_u32(to), rank)),
                 "l"(word_of(v, seq))
                 : "memory");
}
__device__ __forceinline__ unsigned long long peek(unsigned long long* from) {
  unsigned long long q;
  asm volatile("ld.relaxed.cluster.shared::cta.b64 %0, [%1];"
               : "=l"(q)
               : "r"(smem_u32(from))
               : "memory");
  return q;
}
__device__ __forceinline__ float value_in(unsigned long long word) {
  return __uint_as_float((uint32_t)word);
}
// Waits for the word of exchange `seq` (2 s at most, see mbar_wait); false
// where it does not come.
__device__ __forceinline__ bool receive(unsigned long long* from, uint32_t seq,
                                        unsigned long long& word, unsigned int* err) {
  unsigned long long t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    word = peek(from);
    if ((uint32_t)(word >> 32) == seq) return true;
    if ((spins & 63u) == 63u) {
      if (t0 == 0) t0 = globaltimer();
      if (globaltimer() - t0 > kWaitTimeoutNs) {
        atomicCAS(err, kErrNone, kErrMbarTimeout);
        return false;
      }
      if (*(volatile unsigned int*)err != kErrNone) return false;
    }
  }
}

// Vectors of a warp, of `per` a CTA: whole steps of 32 lanes.
__host__ __device__ __forceinline__ int warp_vectors(int per) {
  return (per + 32 * kWarps - 1) / (32 * kWarps) * 32;
}

// Loss and gradient of rows held in shared memory: CL CTAs a row. A cluster
// begins with the row of its number and takes the others from a counter: some
// SMs hold fewer CTAs than others, whose clusters are faster.
template <typename T, int CL>
__global__ void __launch_bounds__(NT, 3) distill_fused_kernel(const Params p) {
  using Tr = Traits<T>;
  using Tag = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
  constexpr int E = Tr::E;
  // What the warps send one another, and a row's teacher: every warp writes
  // the same there, so none waits for another to read it. Two rows' worth: a
  // warp that has the sums of a row knows that all others are done with the
  // row before, and only then writes over that.
  __shared__ unsigned long long parts[2][4][CL * kWarps];
  __shared__ unsigned long long xks[2][kMaxTeacherK];  // in the cluster's first CTA
  __shared__ unsigned long long ahead[2][2];  // the next row, and its weight
  __shared__ uint64_t bar[2];
  __shared__ int t_id[2][kMaxTeacherK];  // as given
  __shared__ float t_lp[2][kMaxTeacherK];
  __shared__ float t_p[2][kMaxTeacherK], t_x[2][kMaxTeacherK];
  extern __shared__ __align__(16) uint8_t dyn[];
  uint4* kept = reinterpret_cast<uint4*>(dyn);
  const int part = blockIdx.x % CL, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (threadIdx.x == 0) {
    mbar_init(&bar[0], CL * kWarps);
    mbar_init(&bar[1], CL * kWarps);
    fence_barrier_init();
  }
  for (int i = threadIdx.x; i < 8 * CL * kWarps; i += NT) (&parts[0][0][0])[i] = 0ull;
  for (int i = threadIdx.x; i < 2 * kMaxTeacherK; i += NT) (&xks[0][0])[i] = 0ull;
  if (threadIdx.x < 4) (&ahead[0][0])[threadIdx.x] = 0ull;
  if constexpr (CL > 1)
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
  else
    __syncthreads();
  pdl_wait();
  pdl_trigger();
  // My warp's vectors of any row: [first, first + cap), those that exist.
  const int per = ((p.V + 2 * E - 2) / E + CL - 1) / CL, cap = warp_vectors(per);
  const int first = part * per + warp * cap, last = min(first + cap, (part + 1) * per);
  uint4* mine = kept + warp * cap - first;  // indexed by the vector
  T* elem = reinterpret_cast<T*>(mine);
  const float c = p.c;

  auto weight = [&](int64_t r) { return r >= p.rows ? 0.f : p.weights ? p.weights[r] : 1.f; };
  auto fetch = [&](const Row<T>& row, int u) {
    if (row.full(u)) {
      cp_async_16(smem_u32(mine + u), row.x + ((int64_t)u * E - row.pad));
    } else {
      mine[u] = make_uint4(Tr::kNegInf, Tr::kNegInf, Tr::kNegInf, Tr::kNegInf);
#pragma unroll 1
      for (int e = max(0, row.pad - u * E); e < min(E, row.pad + p.V - u * E); ++e)
        elem[u * E + e] = row.x[row.index(u, e)];
    }
  };
  auto fetch_teacher = [&](int64_t r, int buf) {
#pragma unroll 1
    for (int k = lane; k < p.K; k += 32) {
      cp_async_4(smem_u32(&t_id[buf][k]), p.t_ids + r * p.K + k);
      cp_async_4(smem_u32(&t_lp[buf][k]), p.t_lp + r * p.K + k);
    }
  };

  int64_t r = blockIdx.x / CL;
  float w = weight(r);
  Row<T> row(p.x, min(r, p.rows - 1), p.ld, p.V);
  if (w != 0.f) {
    const int end = min(last, row.n_vec);
    for (int u = first + lane; u < end; u += 32) fetch(row, u);
    fetch_teacher(r, 0);
  }
  if constexpr (CL > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");

  for (uint32_t n = 0; r < p.rows; ++n) {
    const int end = w != 0.f ? min(last, row.n_vec) : first;
    T* out = reinterpret_cast<T*>(p.grad) + r * p.V;
    // The next row, by the time of the exchange.
    int64_t r_next = 0;
    float w_next = 0.f;
    if (part == 0 && threadIdx.x == 0) {
      r_next = p.rows;
      if (p.taken) r_next = gridDim.x / CL + atomicAdd(p.taken, 1);
      w_next = weight(r_next);
    }
    const int buf = n & 1;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();

    // The teacher's elements of my part out of the row: value, then a tag of
    // the entry (repeated ids overwrite one another's), then -inf.
    uint32_t own = 0;  // entries lane + 32 i here, the first of their id
    float m_k = -INFINITY;
    int at[kIds], here = 0;
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      at[i] = -1;
      if (32 * i < p.K && w != 0.f) {
        const int k = lane + 32 * i, id = k < p.K ? t_id[buf][k] : -1;
        const bool in = id >= 0 && id < p.V &&
                        (uint32_t)(id + row.pad - first * E) < (uint32_t)(max(end - first, 0) * E);
        if (in) at[i] = id + row.pad;
        here += __popc(__ballot_sync(0xffffffffu, in));
      }
    }
    if (here > 0) {
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (at[i] >= 0) {
          const float x = Tr::to_f(elem[at[i]]);
          t_x[buf][lane + 32 * i] = x;
          m_k = fmaxf(m_k, x);
          own |= 1u << i;
          send<CL>(&xks[buf][lane + 32 * i], 0, x, n + 1);
        }
      __syncwarp();
      bool dup = false;
      if (here > 1) {
#pragma unroll
        for (int i = 0; i < kIds; ++i)
          if (at[i] >= 0) reinterpret_cast<Tag*>(elem)[at[i]] = (Tag)(lane + 32 * i);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kIds; ++i)
          if (at[i] >= 0)
            dup |= reinterpret_cast<const Tag*>(elem)[at[i]] != (Tag)(lane + 32 * i);
        dup = __any_sync(0xffffffffu, dup);
      }
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (at[i] >= 0) reinterpret_cast<Tag*>(elem)[at[i]] = (Tag)Tr::kNegInf;
      if (dup) own = first_of_ids(own, t_id[buf], p.K);
      __syncwarp();
    }

    // The rest: maximum, then sum.
    const int n4 = end > first ? (end - first) / 128 * 128 : 0, tail = first + n4;
    typename Tr::Max vm = Tr::vmax(make_uint4(Tr::kNegInf, Tr::kNegInf, Tr::kNegInf, Tr::kNegInf));
#pragma unroll 1
    for (int u = first + lane; u < tail; u += 128) {
      typename Tr::Max q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) q[k] = Tr::vmax(mine[u + 32 * k]);
      vm = Tr::vmax(vm, Tr::vmax(Tr::vmax(q[0], q[1]), Tr::vmax(q[2], q[3])));
    }
#pragma unroll 1
    for (int u = tail + lane; u < end; u += 32) vm = Tr::vmax(vm, Tr::vmax(mine[u]));
    const float m_w = warp_max(Tr::value(vm)), m_in = here > 0 ? warp_max(m_k) : -INFINITY;
    float s = 0.f;
    if (!slow_range(m_w, c, kFar)) {
      const float rw = __fmul_rn(m_w, c);
      const uint64_t c2 = f32x2_pack(c, c), nr2 = f32x2_pack(-rw, -rw);
      uint64_t s2[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) s2[k] = f32x2_pack(0.f, 0.f);
      auto add = [&](const uint4& v, uint64_t& sum) {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          float a, b;
          Tr::pair(v, i, a, b);
          f32x2_unpack(f32x2_fma(f32x2_pack(a, b), c2, nr2), a, b);
          sum = f32x2_add(sum, f32x2_pack(ex2(a), ex2(b)));
        }
      };
#pragma unroll 1
      for (int u = first + lane; u < tail; u += 128) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = mine[u + 32 * k];
#pragma unroll
        for (int k = 0; k < 4; ++k) add(v[k], s2[k]);
      }
#pragma unroll 1
      for (int u = tail + lane; u < end; u += 32) add(mine[u], s2[0]);
      float a, b;
      f32x2_unpack(f32x2_add(f32x2_add(s2[0], s2[1]), f32x2_add(s2[2], s2[3])), a, b);
      s = (a + b) * ex2(-fmaf(m_w, c, -rw));  // what rw lacks of m c
    } else {
      const float m = shift_of(m_w);
#pragma unroll 1
      for (int u = first + lane; u < end; u += 32)
#pragma unroll 1
        for (int e = 0; e < E; ++e) s += ex2((Tr::to_f(elem[u * E + e]) - m) * c);
    }
    float s_in = 0.f;
#pragma unroll 1
    for (int i = 0; 32 * i < p.K; ++i)
      if ((own >> i) & 1u) s_in += ex2((t_x[buf][lane + 32 * i] - shift_of(m_in)) * c);
    s = warp_sum(s);
    if (here > 0) s_in = warp_sum(s_in);
    // To every CTA of the cluster; each warp hears from every other.
    if (part == 0 && warp == 0) {
      const int rn = __shfl_sync(0xffffffffu, (int)min(r_next, p.rows), 0);
      const float wn = __shfl_sync(0xffffffffu, w_next, 0);
      if (lane < CL) {
        send<CL>(&ahead[buf][0], lane, __int_as_float(rn), n + 1);
        send<CL>(&ahead[buf][1], lane, wn, n + 1);
      }
    }
    if (lane < CL) {
      send<CL>(&parts[buf][0][part * kWarps + warp], lane, m_w, n + 1);
      send<CL>(&parts[buf][1][part * kWarps + warp], lane, s, n + 1);
      send<CL>(&parts[buf][2][part * kWarps + warp], lane, m_in, n + 1);
      send<CL>(&parts[buf][3][part * kWarps + warp], lane, s_in, n + 1);
      // (The barrier is where a warp sleeps until all have sent; what it then
      // reads carries its own proof.)
      if constexpr (CL == 1)
        mbar_arrive(&bar[buf]);
      else
        mbar_arrive_cluster_relaxed(mapa_shared(smem_u32(&bar[buf]), lane));
    }
    // Meanwhile the teacher's probabilities.
    float norm, sum_p;
    {
      Teacher t;
      t.load(t_id[buf], t_lp[buf], w != 0.f ? p.K : 0);
      t.prepare(p);
      norm = t.norm, sum_p = t.sum_p;
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (lane + 32 * i < p.K) t_p[buf][lane + 32 * i] = t.p[i];
    }
    bool met = mbar_wait(&bar[buf], (n >> 1) & 1u, p.err);
    // (All words first: they are there as a rule.)
    constexpr int kParts = CL * kWarps, kMine = (kParts + 31) / 32;
    unsigned long long word[4 * kMine + 2];
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        word[4 * i + e] = peek(&parts[buf][e][min(lane + 32 * i, kParts - 1)]);
    word[4 * kMine] = peek(&ahead[buf][0]);
    word[4 * kMine + 1] = peek(&ahead[buf][1]);
    bool there = true;
#pragma unroll
    for (int i = 0; i < 4 * kMine + 2; ++i) there &= (uint32_t)(word[i] >> 32) == n + 1;
    if (!there) {
#pragma unroll
      for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          met &= receive(&parts[buf][e][min(lane + 32 * i, kParts - 1)], n + 1, word[4 * i + e], p.err);
      met &= receive(&ahead[buf][0], n + 1, word[4 * kMine], p.err);
      met &= receive(&ahead[buf][1], n + 1, word[4 * kMine + 1], p.err);
    }
    Sums got[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      got[i] = Sums{-INFINITY, 0.f, -INFINITY, 0.f};
      if (i < kMine && lane + 32 * i < kParts)
        got[i] = Sums{value_in(word[4 * i]), value_in(word[4 * i + 1]), value_in(word[4 * i + 2]),
                      value_in(word[4 * i + 3])};
    }
    w_next = value_in(word[4 * kMine + 1]);
    if (!__all_sync(0xffffffffu, met)) break;  // (the status word is set)
    r_next = __float_as_int(value_in(word[4 * kMine]));
    const Row<T> next(p.x, min(r_next, p.rows - 1), p.ld, p.V);
    const int end_next = w_next != 0.f ? min(last, next.n_vec) : first;
    if (w_next != 0.f) fetch_teacher(r_next, buf ^ 1);
    if (w == 0.f) {
      if (part == 0 && threadIdx.x == 0) {
        p.row_loss[r] = 0.f;
        save(p.stats, r, Numbers{});
      }
      for (int u = first + lane; u < min(last, row.n_vec); u += 32)
        store_vec(out, row, u, make_uint4(0u, 0u, 0u, 0u));
      for (int u = first + lane; u < end_next; u += 32) fetch(next, u);
      r = r_next, w = w_next, row = next;
      continue;
    }

    // Every warp finishes the row's numbers (the same in all of them).
    const Sums q = join(got[0], got[1], c);
    const Numbers st = row_numbers(norm, sum_p, p.tail, q, c);
    if (part == 0 && warp == 0) {
      Teacher t;
      t.load(t_id[buf], t_lp[buf], p.K);
      float xk[kIds];
#pragma unroll
      for (int i = 0; i < kIds; ++i) {
        t.p[i] = xk[i] = 0.f;
        t.lp[i] -= norm;
        if (lane + 32 * i < p.K) {
          t.p[i] = t_p[buf][lane + 32 * i];
          if (t.id[i] >= 0 && t.id[i] < p.V) {
            unsigned long long x;
            met &= receive(&xks[buf][lane + 32 * i], n + 1, x, p.err);
            xk[i] = value_in(x);
          }
        }
      }
      t.sum_p = sum_p;
      const float loss = row_loss(t, p, q, xk);
      if (!__all_sync(0xffffffffu, met)) break;
      if (lane == 0) {
        p.row_loss[r] = loss * w;
        save(p.stats, r, st);
      }
    }
    // The gradient: every element as an outside one (the teacher's are -inf by
    // now), then the teacher's over it. The next row's vectors follow.
    const float up = w * p.gscale;
    const bool slow = slow_range(st.m_out, c, kFar);
    const float rm = __fmul_rn(st.m_out, c),
                coef = st.k_out * up * (slow ? 1.f : ex2(-fmaf(st.m_out, c, -rm)));
    // Whole steps of 128 full vectors without checks.
    uint4* dst = reinterpret_cast<uint4*>(out - row.pad);
    const uint4* src = reinterpret_cast<const uint4*>(next.x - next.pad);
    const bool aligned = (reinterpret_cast<uintptr_t>(dst) & 15u) == 0;
    const int fa = aligned && !slow ? row.full_lo : p.V, fb = row.full_lo + (int)row.n_full;
    const int next_fa = next.full_lo, next_fb = next.full_lo + (int)next.n_full;
#pragma unroll 1
    for (int u0 = first; u0 < end || u0 < end_next; u0 += 128) {
      const int u = u0 + lane;
      if (u0 >= fa && u0 + 128 <= min(fb, end)) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = mine[u + 32 * k];
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[u + 32 * k] = grad_vec<T, false>(v[k], c, rm, coef);
        if (u0 >= next_fa && u0 + 128 <= min(next_fb, end_next)) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            cp_async_16(smem_u32(mine + u + 32 * k), src + u + 32 * k);
          continue;
        }
      } else {
#pragma unroll 1
        for (int v = u; v < min(u0 + 128, end); v += 32)
          store_vec(out, row, v,
                    slow ? grad_vec<T, true>(mine[v], c, st.m_out, coef)
                         : grad_vec<T, false>(mine[v], c, rm, coef));
      }
#pragma unroll 1
      for (int v = u; v < min(u0 + 128, end_next); v += 32) fetch(next, v);
    }
    __syncwarp();
#pragma unroll 1
    for (int i = 0; 32 * i < p.K; ++i)
      if ((own >> i) & 1u) {
        const int k = lane + 32 * i, id = t_id[buf][k];
        float mass = t_p[buf][k];
        if (own & kDup) mass = mass_of_id(id, t_id[buf], t_p[buf], p.K);
        const float qk = ex2((t_x[buf][k] - st.m) * c) * st.k_in;
        out[id] = Tr::from_f((qk - (st.k_in == 0.f ? 0.f : mass)) * up);
      }
    r = r_next, w = w_next, row = next;
  }
  // (No CTA leaves while another's exchange may still reach it.)
  asm volatile("cp.async.wait_all;" ::: "memory");
  if constexpr (CL > 1) cluster_sync_all();
}

struct Smem {
  Acc acc[kWarps];
  int dup;                   // some id of this slice is there twice
  Sums part[kMaxCluster];
};

// Loss, and with GRAD the gradient, of rows that are streamed: CL CTAs a row.
template <typename T, int CL, bool GRAD>
__global__ void __launch_bounds__(NT, 4) distill_stream_kernel(const Params p) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  __shared__ Smem sm;
  extern __shared__ __align__(16) uint8_t dyn[];  // the bitmap: a byte a vector
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / CL;
  const int part = blockIdx.x % CL;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  const Row<T> row(p.x, r, p.ld, p.V);
  const Slice sl(row, part, CL);
  T* out = GRAD ? reinterpret_cast<T*>(p.grad) + r * p.V : nullptr;
  const float w = p.weights ? p.weights[r] : 1.f;
  if (w == 0.f) {  // uniform over the cluster
    if constexpr (GRAD)
      for (int u = sl.lo + tid; u < sl.hi; u += NT)
        store_vec(out, row, u, make_uint4(0u, 0u, 0u, 0u));
    if (part == 0 && tid == 0) {
      p.row_loss[r] = 0.f;
      save(p.stats, r, Numbers{});
    }
    if constexpr (CL > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    return;
  }

  uint8_t* bitmap = dyn;
  for (int i = tid; i < (sl.hi - sl.lo + 15) / 16; i += NT)
    reinterpret_cast<uint4*>(bitmap)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) sm.dup = 0;
  Teacher t;
  t.load(p.t_ids + r * p.K, p.t_lp + r * p.K, p.K);
  __syncthreads();
  // Warp 0 marks the ids of this slice.
  float xk[kIds];
  uint32_t own = 0;
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) {
      xk[i] = -INFINITY;
      if (t.id[i] >= 0 && t.id[i] < p.V) {
        const int u = (t.id[i] + row.pad) / E, e = (t.id[i] + row.pad) % E, at = u - sl.lo;
        xk[i] = Tr::to_f(row.x[t.id[i]]);
        if (u >= sl.lo && u < sl.hi) {
          const uint32_t bit = 1u << (8 * (at % 4) + e);
          own |= 1u << i;
          if (atomicOr(reinterpret_cast<uint32_t*>(bitmap) + at / 4, bit) & bit) sm.dup = 1;
        }
      }
    }
  }
  __syncthreads();

  // The slice's sum over the elements that are not the teacher's.
  const float c = p.c;
  const uint64_t c2 = f32x2_pack(c, c);
  float m = -INFINITY, r0 = 0.f, s = 0.f;
  for_groups<NT, U>(row, sl, [&](const uint4(&x)[U], int u, int) {
    uint4 v[U];
    typename Tr::Max vm[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int uk = u + k * NT;
      v[k] = x[k];
      const uint32_t in = uk < sl.hi ? bitmap[uk - sl.lo] : 0u;
      if (in) Tr::blank(v[k], in);
      vm[k] = Tr::vmax(v[k]);
    }
    static_assert(U == 4, "tree of maxima");
    const float mx = Tr::value(Tr::vmax(Tr::vmax(vm[0], vm[1]), Tr::vmax(vm[2], vm[3])));
    if (mx > m) {
      const float rn = __fmul_rn(fmaxf(mx, p.least), c);
      s *= m == -INFINITY ? (s != s ? s : 0.f) : ex2(r0 - rn);
      m = mx;
      r0 = rn;
    }
    const uint64_t nr2 = f32x2_pack(-r0, -r0);
    uint64_t s2 = f32x2_pack(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float a, b;
        Tr::pair(v[k], i, a, b);
        f32x2_unpack(f32x2_fma(f32x2_pack(a, b), c2, nr2), a, b);
        s2 = f32x2_add(s2, f32x2_pack(ex2(a), ex2(b)));
      }
    }
    float a, b;
    f32x2_unpack(s2, a, b);
    s += a + b;
  });
  // A warp's sums against its own maximum, in a fixed order.
  const float m_w = warp_max(m);
  if (slow_range(m_w, c, kFar) && m_w != -INFINITY) {
    s = slow_sum(row, sl, bitmap, m_w, c);
  } else {
    const float e = fmaf(m, c, -r0);  // what r0 lacks of m c
    if (m > p.least)
      s *= ex2(-e) * (m == m_w ? 1.f : ex2((m - m_w) * c));
    else
      s = s != s ? s : 0.f;  // nothing against the warp's maximum
  }
  s = warp_sum(s);
  if (lane == 0) sm.acc[warp] = Acc{m_w, s, 0.f};
  __syncthreads();

  // Warp 0 adds the warps up, with the ids' own exponentials.
  Sums q;
  float mass[kIds];
  if (warp == 0) {
    t.prepare(p);
#pragma unroll
    for (int i = 0; i < kIds; ++i) mass[i] = t.p[i];
    if (sm.dup) {
      t.masses(p.K, mass);
#pragma unroll
      for (int i = 0; i < kIds; ++i)
        if (mass[i] == -1.f) own &= ~(1u << i);
    }
    Acc a = lane < kWarps ? sm.acc[lane] : Acc{-INFINITY, 0.f, 0.f};
    const float m_out = warp_max(a.m);
    rebase(a, m_out, c);
    float m_in = -INFINITY, s_in = 0.f;
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      if ((own >> i) & 1u) m_in = fmaxf(m_in, xk[i]);
    m_in = warp_max(m_in);
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      if ((own >> i) & 1u) s_in += ex2((xk[i] - shift_of(m_in)) * c);
    q = Sums{m_out, warp_sum(a.s), m_in, warp_sum(s_in)};
    if constexpr (CL > 1) {
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      // Every CTA of the cluster gets every slice's sums.
      if (lane < CL)
        st_dsmem_f4(mapa_shared(smem_u32(&sm.part[part]), lane),
                    make_float4(q.m_out, q.s_out, q.m_in, q.s_in));
    }
  } else if constexpr (CL > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  if constexpr (CL > 1) cluster_sync_all();
  __shared__ Numbers numbers;
  if (warp == 0) {
    if constexpr (CL > 1) {
      const Sums none{-INFINITY, 0.f, -INFINITY, 0.f};
      q = join(lane < CL ? sm.part[lane] : none, none, c);
    }
    const Numbers st = row_numbers(t.norm, t.sum_p, p.tail, q, c);
    if (part == 0) {
      const float loss = row_loss(t, p, q, xk);
      if (lane == 0) {
        p.row_loss[r] = loss * w;
        save(p.stats, r, st);
      }
    }
    if (lane == 0) numbers = st;
  }
  if constexpr (!GRAD) return;
  __syncthreads();

  // The gradient: every element as an outside one, then the teacher's ids of
  // this slice over it (same CTA, after the barrier).
  const Numbers st = numbers;
  const float up = w * p.gscale;
  if (!slow_range(st.m_out, c, kFar)) {
    const float rm = __fmul_rn(st.m_out, c), coef = st.k_out * up * ex2(-fmaf(st.m_out, c, -rm));
    const int groups = (sl.b - sl.a + U * NT - 1) / (U * NT);
    for_groups<NT, U>(row, sl, [&](const uint4(&v)[U], int u, int it) {
      if (it == groups) return;  // the partial vectors, below
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (u + k * NT < sl.b)
          store_vec(out, row, u + k * NT, grad_vec<T, false>(v[k], c, rm, coef));
    });
    const int e = tid == 0 ? sl.head : tid == 1 ? sl.tail : -1;
    if (e >= 0) store_part(out, row, e, grad_vec<T, false>(row.load(e), c, rm, coef));
  } else {
    for (int u = sl.lo + tid; u < sl.hi; u += NT)
      store_vec(out, row, u, grad_vec<T, true>(row.load(u), c, st.m_out, st.k_out * up));
  }
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int i = 0; i < kIds; ++i)
      if ((own >> i) & 1u) {
        const float qk = ex2((xk[i] - st.m) * c) * st.k_in;
        out[t.id[i]] = Tr::from_f((qk - (st.k_in == 0.f ? 0.f : mass[i])) * up);
      }
  }
}

// The same gradient for an upstream value a row: elementwise on the saved
// numbers, a CTA a (row, chunk of kBwdThreads * U vectors).
struct BwdParams {
  Params f;
  const float* g;
  int g_stride;
  int chunks;
};

template <typename T>
__device__ __forceinline__ void bwd_chunk(const BwdParams& b, unsigned r0, unsigned chunk) {
  const int64_t r = r0;
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  constexpr int kBits = kBwdThreads * U * E;  // elements of the chunk
  __shared__ uint32_t seen[kBits / 32];
  __shared__ int dup;
  const Params& p = b.f;
  const int tid = threadIdx.x;
  const Row<T> row(p.x, r, p.ld, p.V);
  const int u_lo = chunk * (kBwdThreads * U), u_hi = min(u_lo + kBwdThreads * U, row.n_vec);
  if (u_lo >= u_hi) return;
  T* out = reinterpret_cast<T*>(p.grad) + r * p.V;
  const float w = p.weights ? p.weights[r] : 1.f;
  const float up = w == 0.f ? 0.f : w * p.gscale * b.g[r * b.g_stride];
  if (up == 0.f) {
    for (int u = u_lo + tid; u < u_hi; u += kBwdThreads) store_vec(out, row, u, make_uint4(0u, 0u, 0u, 0u));
    return;
  }
  uint4 v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u_lo + tid + k * kBwdThreads;
    v[k] = u < u_hi ? row.load(u) : make_uint4(0u, 0u, 0u, 0u);
  }
  // Thread k's teacher entry, if it is of this chunk, and whether an id of
  // the chunk is there twice.
  const int id = tid < p.K ? p.t_ids[r * p.K + tid] : -1;
  const int at = id + row.pad - u_lo * E;
  const bool mine = id >= 0 && id < p.V && at >= 0 && at / E < u_hi - u_lo;
  const Numbers st = saved(p.stats, r);
  const float xk = mine ? Tr::to_f(row.x[id]) : 0.f;
  float mass = mine ? expf(p.t_lp[r * p.K + tid] - st.norm) : 0.f;
  for (int i = tid; i < kBits / 32; i += kBwdThreads) seen[i] = 0u;
  if (tid == 0) dup = 0;
  __syncthreads();
  if (mine && (atomicOr(&seen[at / 32], 1u << (at % 32)) >> (at % 32)) & 1u) dup = 1;
  if (!slow_range(st.m_out, p.c, kFar)) {
    const float rm = __fmul_rn(st.m_out, p.c), coef = st.k_out * up * ex2(-fmaf(st.m_out, p.c, -rm));
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = u_lo + tid + k * kBwdThreads;
      if (u < u_hi) store_vec(out, row, u, grad_vec<T, false>(v[k], p.c, rm, coef));
    }
  } else {
    for (int u = u_lo + tid; u < u_hi; u += kBwdThreads)
      store_vec(out, row, u, grad_vec<T, true>(row.load(u), p.c, st.m_out, st.k_out * up));
  }
  __syncthreads();
  if (!mine) return;
  if (dup) {  // the p of all entries with this id, at the first of them
    mass = 0.f;
    for (int j = 0; j < p.K; ++j)
      if (p.t_ids[r * p.K + j] == id) {
        if (j < tid) return;
        mass += expf(p.t_lp[r * p.K + j] - st.norm);
      }
  }
  const float q = ex2((xk - st.m) * p.c) * st.k_in;
  out[id] = Tr::from_f((q - (st.k_in == 0.f ? 0.f : mass)) * up);
}

template <typename T>
__global__ void __launch_bounds__(kBwdThreads) distill_bwd_kernel(const __grid_constant__ BwdParams b) {
  pdl_wait();
  pdl_trigger();
  bwd_chunk<T>(b, blockIdx.y, blockIdx.x);
}

// Where the upstream scalar is 1 the forward pass has left the gradient as it
// has to be. Any other value's is computed anew from the logits (as many bytes
// as scaling would move), so that it is rounded once too. As many CTAs as run
// at the same time: as a rule they have nothing to do.
template <typename T>
__global__ void __launch_bounds__(kBwdThreads, kBwdCtas) distill_redo_kernel(const __grid_constant__ BwdParams b) {
  pdl_wait();
  pdl_trigger();
  if (*b.g == 1.f) return;
  const int64_t n = b.f.rows * b.chunks;
  for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
    const int64_t r = i / b.chunks;
    bwd_chunk<T>(b, (unsigned)r, (unsigned)(i - r * b.chunks));
    __syncthreads();
  }
}

// loss = scale * sum of the rows' losses, one CTA, fixed order.
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* x, int64_t n, float scale,
                                                        float* out) {
  pdl_wait();
  pdl_trigger();
  __shared__ float part[32];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += x[i];
  s = warp_sum(s);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(part[threadIdx.x]);
    if (threadIdx.x == 0) *out = s * scale;
  }
}

void check(const LogitRows& in, int K, const char* what) {
  if (in.V < 1 || in.V > kMaxVocab)
    throw std::runtime_error(std::string(what) + ": vocabulary outside [1, 2^22]");
  if (in.rows > (1 << 24)) throw std::runtime_error(std::string(what) + ": more than 2^24 rows");
  if (K < 1 || K > kMaxTeacherK)
    throw std::runtime_error(std::string(what) + ": between 1 and 128 teacher values a row");
}

// A CTA's part of a row: as few CTAs a row as leave two an SM (three up to
// 64 KB). More of them hold less of an SM's memory and meet more others: 2048
// x 151936 bf16 takes 310 us at 4 CTAs a row of 76 KB, 362 at 8 of 40 KB; 2048
// x 100000 187 us at 2 of 100 KB, 204 at 4.
constexpr int kSmemSlice = 104 * 1024;
constexpr int kSmemMost = 208 * 1024;
constexpr int kBitmapMost = 160 * 1024;

cudaLaunchAttribute cluster_of(int n) {
  cudaLaunchAttribute cl;
  cl.id = cudaLaunchAttributeClusterDimension;
  cl.val.clusterDim.x = n;
  cl.val.clusterDim.y = cl.val.clusterDim.z = 1;
  return cl;
}
// Vectors of a CTA where CL of them share a row.
template <typename T>
int slice_vectors(int V, int cl) {
  return ((V + 2 * Traits<T>::E - 2) / Traits<T>::E + cl - 1) / cl;
}
// Shared memory that holds them, in equal parts a warp.
template <typename T>
int slice_bytes(int V, int cl) {
  return warp_vectors(slice_vectors<T>(V, cl)) * kWarps * 16;
}

template <typename T, int CL>
void launch_fused(Params p, int* counter, cudaStream_t stream) {
  auto kernel = distill_fused_kernel<T, CL>;
  static bool attr[kMaxDevices] = {};
  set_smem_attr_once(kernel, kSmemMost, attr, "distill_loss");
  const int smem = slice_bytes<T>(p.V, CL);
  // Clusters that run at the same time, asked for once a size.
  struct Known {
    int dev = -1, smem = 0, clusters = 0;
  };
  static thread_local Known known;
  int dev = 0;
  cudaGetDevice(&dev);
  p.err = device_status_ptr(dev);
  const cudaLaunchAttribute cl = cluster_of(CL);
  if (known.dev != dev || known.smem != smem) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(CL);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = const_cast<cudaLaunchAttribute*>(&cl);
    cfg.numAttrs = 1;
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (e != cudaSuccess || n < 1)
      throw std::runtime_error(std::string("distill_loss: no cluster fits: ") +
                               cudaGetErrorString(e));
    known = Known{dev, smem, n};
  }
  const int64_t clusters = p.rows < known.clusters ? p.rows : known.clusters;
  if (clusters < p.rows) {
    p.taken = counter;
    const cudaError_t e = cudaMemsetAsync(counter, 0, sizeof(int), stream);
    if (e != cudaSuccess)
      throw std::runtime_error(std::string("distill_loss: ") + cudaGetErrorString(e));
  }
  launch_pdl(kernel, dim3((unsigned)(clusters * CL)), dim3(NT), smem, stream,
             CL > 1 ? &cl : nullptr, p);
}

template <typename T, int CL, bool GRAD>
void launch_stream(const Params& p, cudaStream_t stream) {
  auto kernel = distill_stream_kernel<T, CL, GRAD>;
  static bool attr[kMaxDevices] = {};
  set_smem_attr_once(kernel, kBitmapMost, attr, "distill_loss");
  const cudaLaunchAttribute cl = cluster_of(CL);
  const int bitmap = (slice_vectors<T>(p.V, CL) + 15) / 16 * 16;
  launch_pdl(kernel, dim3((unsigned)(p.rows * CL)), dim3(NT), bitmap, stream,
             CL > 1 ? &cl : nullptr, p);
}

template <typename T>
void launch_t(const Params& p, int* counter, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = num_sms(dev);
  if (p.grad && slice_bytes<T>(p.V, kMaxCluster) <= kSmemMost) {
    int cl = row_split(p.rows, p.V / Traits<T>::E, 5 * sms / 2, NT);
    while (cl < kMaxCluster && slice_bytes<T>(p.V, cl) > kSmemSlice) cl *= 2;
    switch (cl) {
      case 1: return launch_fused<T, 1>(p, counter, stream);
      case 2: return launch_fused<T, 2>(p, counter, stream);
      case 4: return launch_fused<T, 4>(p, counter, stream);
      default: return launch_fused<T, 8>(p, counter, stream);
    }
  }
  if (p.grad) return launch_stream<T, 8, true>(p, stream);
  int cl = row_split(p.rows, p.V / Traits<T>::E, 4 * sms, NT);
  // bitmaps of a very large vocabulary: 32 KB, for four CTAs an SM
  while (cl < kMaxCluster && slice_vectors<T>(p.V, cl) > 32 * 1024) cl *= 2;
  switch (cl) {
    case 1: return launch_stream<T, 1, false>(p, stream);
    case 2: return launch_stream<T, 2, false>(p, stream);
    case 4: return launch_stream<T, 4, false>(p, stream);
    default: return launch_stream<T, 8, false>(p, stream);
  }
}

}  // namespace

void distill_launch(const DistillArgs& a, cudaStream_t stream) {
  check(a.in, a.K, "distill_loss");
  if (a.in.rows > 0) {
    Params p{a.in.x, a.t_ids, a.t_lp, a.weights, a.in.ld, a.in.V, a.K, a.in.rows, a.tail,
             (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
             (float)((double)a.grad_scale / a.temperature),
             floor_of((float)(1.4426950408889634 / a.temperature)), a.row_loss,
             reinterpret_cast<float4*>(a.stats), a.grad, nullptr, nullptr};
    if (a.in.bf16)
      launch_t<__nv_bfloat16>(p, a.counter, stream);
    else
      launch_t<float>(p, a.counter, stream);
  }
  if (a.loss)
    launch_pdl(sum_rows_kernel, dim3(1), dim3(1024), 0, stream, nullptr, (const float*)a.row_loss,
               a.in.rows, a.grad_scale, a.loss);
}

void distill_bwd_launch(const DistillBwdArgs& a, cudaStream_t stream) {
  check(a.in, a.K, "distill_loss_bwd");
  if (a.in.rows <= 0) return;
  const int E = a.in.bf16 ? 8 : 4;
  const int64_t eb = a.in.bf16 ? 2 : 4;
  const unsigned chunks = (unsigned)((a.in.V + 2 * E - 2) / E + kBwdThreads * U - 1) / (kBwdThreads * U);
  // grid.y holds at most 65535 rows a launch
  const int64_t most = a.unless_one ? a.in.rows : 65535;
  for (int64_t r0 = 0; r0 < a.in.rows; r0 += most) {
    const int64_t n = a.in.rows - r0 < most ? a.in.rows - r0 : most;
    BwdParams b{};
    b.f = Params{reinterpret_cast<const char*>(a.in.x) + r0 * a.in.ld * eb, a.t_ids + r0 * a.K,
                 a.t_lp + r0 * a.K, a.weights ? a.weights + r0 : nullptr, a.in.ld, a.in.V, a.K, n,
                 a.tail, (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
                 (float)((double)a.g_scale / a.temperature), 0.f, nullptr,
                 reinterpret_cast<float4*>(const_cast<float*>(a.stats)) + 2 * r0,
                 reinterpret_cast<char*>(a.grad) + r0 * a.in.V * eb, nullptr, nullptr};
    b.g = a.g_rows + r0 * a.g_stride;
    b.g_stride = a.g_stride;
    b.chunks = (int)chunks;
    dim3 grid(chunks, (unsigned)n);
    if (a.unless_one) {
      int dev = 0;
      cudaGetDevice(&dev);
      const int64_t items = n * chunks, ctas = (int64_t)kBwdCtas * num_sms(dev);
      grid = dim3((unsigned)(items < ctas ? items : ctas));
    }
    auto kernel = a.in.bf16 ? (a.unless_one ? distill_redo_kernel<__nv_bfloat16>
                                            : distill_bwd_kernel<__nv_bfloat16>)
                            : (a.unless_one ? distill_redo_kernel<float> : distill_bwd_kernel<float>);
    launch_pdl(kernel, grid, dim3(kBwdThreads), 0, stream, nullptr, b);
  }
}

}  // namespace b200
