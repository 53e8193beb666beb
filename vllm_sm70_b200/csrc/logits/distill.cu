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
// cancel for a student that agrees with its teacher): a bitmap of the row's
// teacher ids in shared memory leaves them out of the streamed sum, and their
// K exponentials are added on their own.
//
// A row with weight 0 has loss 0 and gradient 0 whatever it holds, and is not
// read. Ids outside [0, V) are absent: their mass joins the tail.
//
// Bound: bytes. The training form computes loss and gradient in one kernel: a
// cluster of CTAs shares a row, each streams its slice once for the sums and
// keeps as much of it as fits in shared memory; after one exchange of the
// sums within the cluster the gradient is written from there.
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
constexpr int U = 4;
constexpr int kMaxCluster = 8;
constexpr int K_ = kMaxTeacherK;

struct Params {
  const void* x;
  const int* t_ids;
  const float* t_lp;
  const float* weights;
  int64_t ld;
  int V, K, keep;  // keep: vectors of a thread held in shared memory
  bool tail;
  float c, inv_t, gscale;  // log2(e) / T; 1 / T; upstream gradient / T of a row of weight 1
  float* row_loss;
  float4* stats;
  void* grad;
};

struct Smem {
  float red[kWarps];
  float2 sum[kWarps];
  int id[K_];        // teacher ids, -1 absent
  float p[K_];       // teacher probabilities
  float lp[K_];
  float xk[K_];      // student logits at the ids
  int dup;           // some id of this slice is there twice
  float4 row;        // m, M / s, outside coefficient, 1 (0: empty row)
  float4 part[kMaxCluster];  // a slice's max, sum outside, sum at the ids
};

// The teacher's side of a row into shared memory: threads 0 .. K - 1.
// Returns nothing; ends with a __syncthreads.
__device__ void load_teacher(Smem& sm, const Params& p, int64_t r) {
  const int k = threadIdx.x;
  if (k < p.K) {
    const int id = p.t_ids[r * p.K + k];
    sm.id[k] = id >= 0 && id < p.V ? id : -1;
    sm.lp[k] = p.t_lp[r * p.K + k];
  }
  __syncthreads();
  if (!p.tail) {
    // renormalise over the ids that are present
    float mx = -INFINITY, z = 0.f;
    for (int j = 0; j < p.K; ++j)
      if (sm.id[j] >= 0) mx = fmaxf(mx, sm.lp[j]);
    for (int j = 0; j < p.K; ++j)
      if (sm.id[j] >= 0) z += expf(sm.lp[j] - mx);
    __syncthreads();
    if (k < p.K) sm.lp[k] = sm.lp[k] - mx - logf(z);
  }
  if (k < p.K) sm.p[k] = sm.id[k] >= 0 ? expf(sm.lp[k]) : 0.f;
  __syncthreads();
}

// Whether teacher entry k is the first with its id, and P there: the p of
// every entry with that id.
__device__ __forceinline__ bool first_of_id(const Smem& sm, int K, int k, float& mass) {
  mass = sm.p[k];
  if (!sm.dup) return true;
  const int id = sm.id[k];
  float m = 0.f;
  for (int j = 0; j < K; ++j)
    if (sm.id[j] == id) {
      if (j < k) return false;
      m += sm.p[j];
    }
  mass = m;
  return true;
}

// Gradient of the elements of one vector, all taken as outside ones: g =
// coef * 2^((x - m) c). coef 0 leaves exact zeros (-inf logits included).
template <typename T>
__device__ __forceinline__ uint4 grad_vec(const uint4& v, float c, float m, float coef) {
  using Tr = Traits<T>;
  float g[Tr::E];
  const uint64_t c2 = f32x2_pack(c, c), nm2 = f32x2_pack(-m, -m);
#pragma unroll
  for (int i = 0; i < Tr::E / 2; ++i) {
    float a, b, da, db;
    Tr::pair(v, i, a, b);
    f32x2_unpack(f32x2_mul(f32x2_add(f32x2_pack(a, b), nm2), c2), da, db);
    g[2 * i] = ex2(da) * coef;
    g[2 * i + 1] = ex2(db) * coef;
  }
  return Tr::pack(g);
}

template <typename T>
__device__ __forceinline__ void store_vec(T* out, const Row<T>& row, int u, const uint4& v) {
  constexpr int E = Traits<T>::E;
  const int id0 = row.index(u, 0);
  T* dst = out + id0;
  if (row.full(u) && (reinterpret_cast<uintptr_t>(dst) & 15u) == 0) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (id0 + i >= 0 && id0 + i < row.V) dst[i] = e[i];
  }
}

template <typename T, int CL, bool GRAD>
__global__ void __launch_bounds__(NT, 2) distill_kernel(const Params p) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  __shared__ Smem sm;
  extern __shared__ __align__(16) uint8_t dyn[];  // kept vectors, then the bitmap
  pdl_wait();
  pdl_trigger();
  const int64_t r = blockIdx.x / CL;
  const int part = blockIdx.x % CL;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if constexpr (CL > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");

  const Row<T> row(p.x, r, p.ld, p.V);
  const int per = (row.n_vec + CL - 1) / CL;
  const int u_lo = min(part * per, row.n_vec), u_hi = min(u_lo + per, row.n_vec);
  T* out = GRAD ? reinterpret_cast<T*>(p.grad) + r * p.V : nullptr;
  const float w = p.weights ? p.weights[r] : 1.f;
  if (w == 0.f) {  // uniform over the cluster
    if constexpr (GRAD)
      for (int u = u_lo + tid; u < u_hi; u += NT)
        store_vec(out, row, u, make_uint4(0u, 0u, 0u, 0u));
    if (part == 0 && tid == 0) {
      p.row_loss[r] = 0.f;
      p.stats[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    if constexpr (CL > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    return;
  }

  uint4* kept = reinterpret_cast<uint4*>(dyn);
  uint8_t* bitmap = dyn + (size_t)p.keep * NT * 16;  // E bits (a byte or half) a vector
  for (int i = tid; i < (per + 15) / 16; i += NT)
    reinterpret_cast<uint4*>(bitmap)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) sm.dup = 0;
  load_teacher(sm, p, r);
  // The ids of this slice: owned by thread k.
  bool mine = false;
  float xk = -INFINITY;
  if (tid < p.K && sm.id[tid] >= 0) {
    const int id = sm.id[tid], u = (id + row.pad) / E, e = (id + row.pad) % E;
    xk = Tr::to_f(row.x[id]);
    sm.xk[tid] = xk;
    mine = u >= u_lo && u < u_hi;
    if (mine) {
      const int at = u - u_lo;
      const uint32_t bit = 1u << (8 * (at % 4) + e);
      if (atomicOr(reinterpret_cast<uint32_t*>(bitmap) + at / 4, bit) & bit) sm.dup = 1;
    }
  }
  __syncthreads();
  float mass_k = 0.f;
  const bool own = mine && first_of_id(sm, p.K, tid, mass_k);

  // The slice's sum over the elements that are not the teacher's.
  const float c = p.c;
  const uint64_t c2 = f32x2_pack(c, c);
  Acc a{-INFINITY, 0.f, 0.f};
  for (int u = u_lo + tid, it = 0; u < u_hi; u += U * NT, it += U) {
    uint4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int uk = u + k * NT;
      v[k] = uk < u_hi ? row.load(uk) : make_uint4(Tr::kNegInf, Tr::kNegInf, Tr::kNegInf, Tr::kNegInf);
    }
    float mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int uk = u + k * NT;
      if (GRAD && it + k < p.keep) kept[(it + k) * NT + tid] = v[k];
      const uint32_t in = uk < u_hi ? bitmap[uk - u_lo] : 0u;
      if (in) Tr::blank(v[k], in);
      mx = fmaxf(mx, Tr::max_of(v[k]));
    }
    if (mx > a.m) rebase(a, mx, c);
    const float m = shift_of(a.m);
    const uint64_t nm2 = f32x2_pack(-m, -m);
    uint64_t s2 = f32x2_pack(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < U; ++k) {
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float xa, xb, da, db;
        Tr::pair(v[k], i, xa, xb);
        f32x2_unpack(f32x2_mul(f32x2_add(f32x2_pack(xa, xb), nm2), c2), da, db);
        s2 = f32x2_add(s2, f32x2_pack(ex2(da), ex2(db)));
      }
    }
    float s0, s1;
    f32x2_unpack(s2, s0, s1);
    a.s += s0 + s1;
  }
  const float m = block_max<NT>(own ? fmaxf(a.m, xk) : a.m, sm.red);
  rebase(a, m, c);
  const float s_out_w = warp_sum(a.s);
  const float s_in_w = warp_sum(own ? ex2((xk - shift_of(m)) * c) : 0.f);
  if (lane == 0) sm.sum[warp] = make_float2(s_out_w, s_in_w);
  __syncthreads();
  if (warp == 0) {
    // Every CTA of the cluster gets every slice's sums.
    float s_out = 0.f, s_in = 0.f;
    for (int i = 0; i < kWarps; ++i) {
      s_out += sm.sum[i].x;
      s_in += sm.sum[i].y;
    }
    if constexpr (CL > 1) {
      asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
      if (lane < CL)
        st_dsmem_f4(mapa_shared(smem_u32(&sm.part[part]), lane), make_float4(m, s_out, s_in, 0.f));
    } else if (lane == 0) {
      sm.part[0] = make_float4(m, s_out, s_in, 0.f);
    }
  } else if constexpr (CL > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  if constexpr (CL > 1)
    cluster_sync_all();
  else
    __syncthreads();

  // Warp 0 finishes the row's numbers (the same in every CTA of the cluster).
  if (warp == 0) {
    float mm = -INFINITY;
    for (int i = 0; i < CL; ++i) mm = fmaxf(mm, sm.part[i].x);
    const float m0 = shift_of(mm);
    float s_out = 0.f, s_in = 0.f;
    for (int i = 0; i < CL; ++i) {
      const float4 q = sm.part[i];
      // a slice without any element above -inf has no sums to rebase
      const float f = q.x == -INFINITY || q.x == mm ? 1.f : ex2((q.x - mm) * c);
      s_out += q.y * f;
      s_in += q.z * f;
    }
    float sum_p = 0.f;
    for (int k = lane; k < p.K; k += 32) sum_p += sm.p[k];
    sum_p = warp_sum(sum_p);
    const float s = s_out + s_in;
    // An empty row: every log q is -inf, the loss inf where the teacher has mass.
    const float l2 = s == 0.f ? 0.f : log2f(s);
    float loss = 0.f;
    for (int k = lane; k < p.K; k += 32) {
      const float pk = sm.p[k];
      if (pk > 0.f)
        loss += pk * (sm.lp[k] - fmaf(sm.xk[k] - m0, p.inv_t, -l2 * kLn2));
      else if (pk != pk)
        loss = pk;
    }
    loss = warp_sum(loss);
    const float p_t = p.tail ? fmaxf(0.f, 1.f - sum_p) : 0.f;
    if (p_t > 0.f) loss += p_t * (logf(p_t) - (log2f(s_out) - l2) * kLn2);
    if (lane == 0) {
      const float mass = sum_p + p_t;
      const float inv = s == 0.f ? 0.f : 1.f / s;
      // A student with no mass outside has q_j = 0 there.
      const float ratio = p_t > 0.f && s_out != 0.f ? p_t * s / s_out : 0.f;
      sm.row = make_float4(m0, mass * inv, s_out == 0.f ? 0.f : (mass - ratio) * inv,
                           s == 0.f ? 0.f : 1.f);
      if (part == 0) {
        p.row_loss[r] = loss * w;
        p.stats[r] = sm.row;
      }
    }
  }
  if constexpr (!GRAD) return;
  __syncthreads();

  // The gradient: every element as an outside one, then the teacher's ids of
  // this slice over it (same CTA, after the barrier).
  const float4 st = sm.row;
  const float up = w * p.gscale;
  for (int u = u_lo + tid, it = 0; u < u_hi; u += NT, ++it) {
    const uint4 v = it < p.keep ? kept[it * NT + tid] : row.load(u);
    store_vec(out, row, u, grad_vec<T>(v, c, st.x, st.z * up));
  }
  __syncthreads();
  if (own) {
    const float q = ex2((xk - st.x) * c) * st.y;
    out[sm.id[tid]] = Tr::from_f((q - mass_k * st.w) * up);
  }
}

// The same gradient for an upstream value a row: elementwise on the saved
// numbers. One CTA a (row, chunk of NT * U vectors).
struct BwdParams {
  Params f;
  const float* g;
  int g_stride;
};

template <typename T>
__global__ void __launch_bounds__(NT) distill_bwd_kernel(const BwdParams b) {
  using Tr = Traits<T>;
  constexpr int E = Tr::E;
  __shared__ Smem sm;
  pdl_wait();
  pdl_trigger();
  const Params& p = b.f;
  const int64_t r = blockIdx.y;
  const int tid = threadIdx.x;
  const Row<T> row(p.x, r, p.ld, p.V);
  const int u_lo = blockIdx.x * (NT * U), u_hi = min(u_lo + NT * U, row.n_vec);
  if (u_lo >= u_hi) return;
  T* out = reinterpret_cast<T*>(p.grad) + r * p.V;
  const float w = p.weights ? p.weights[r] : 1.f;
  const float up = w == 0.f ? 0.f : w * p.gscale * b.g[r * b.g_stride];
  const float4 st = p.stats[r];
  const bool none = up == 0.f;
  uint4 v[U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u_lo + tid + k * NT;
    v[k] = u < u_hi && !none ? row.load(u) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (tid == 0) sm.dup = 1;  // no bitmap here: repeats are looked for
  if (!none) load_teacher(sm, p, r);
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int u = u_lo + tid + k * NT;
    if (u < u_hi)
      store_vec(out, row, u,
                none ? make_uint4(0u, 0u, 0u, 0u) : grad_vec<T>(v[k], p.c, st.x, st.z * up));
  }
  if (none) return;
  __syncthreads();
  if (tid < p.K && sm.id[tid] >= 0) {
    const int id = sm.id[tid], u = (id + row.pad) / E;
    float mass;
    if (u >= u_lo && u < u_hi && first_of_id(sm, p.K, tid, mass)) {
      const float q = ex2((Tr::to_f(row.x[id]) - st.x) * p.c) * st.y;
      out[id] = Tr::from_f((q - mass * st.w) * up);
    }
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

template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(T* x, int64_t n, const float* scale) {
  pdl_wait();
  pdl_trigger();
  const float f = *scale;
  if (f == 1.f) return;
  constexpr int E = Traits<T>::E;
  const int64_t stride = (int64_t)gridDim.x * 256;
  const int64_t nv = n / E;  // x is 16-byte aligned
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nv; i += stride) {
    uint4 v = reinterpret_cast<uint4*>(x)[i];
    float g[E];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      Traits<T>::pair(v, k, g[2 * k], g[2 * k + 1]);
      g[2 * k] *= f;
      g[2 * k + 1] *= f;
    }
    reinterpret_cast<uint4*>(x)[i] = Traits<T>::pack(g);
  }
  for (int64_t i = nv * E + (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += stride)
    x[i] = Traits<T>::from_f(Traits<T>::to_f(x[i]) * f);
}

void check(const LogitRows& in, int K, const char* what) {
  if (in.V < 1 || in.V > kMaxVocab)
    throw std::runtime_error(std::string(what) + ": vocabulary outside [1, 2^22]");
  if (in.rows > (1 << 24)) throw std::runtime_error(std::string(what) + ": more than 2^24 rows");
  if (K < 1 || K > kMaxTeacherK)
    throw std::runtime_error(std::string(what) + ": between 1 and 128 teacher values a row");
}

constexpr int kSmemLimit = 96 * 1024;  // two CTAs an SM

template <typename T, int CL, bool GRAD>
void launch_cl(Params p, int64_t rows, cudaStream_t stream) {
  const int n_vec = (p.V + 2 * Traits<T>::E - 2) / Traits<T>::E;
  const int per = (n_vec + CL - 1) / CL;
  const int bitmap = (per + 15) / 16 * 16;
  p.keep = 0;
  if (GRAD) {
    p.keep = (per + NT - 1) / NT;
    const int fit = (kSmemLimit - bitmap) / (NT * 16);
    p.keep = p.keep < fit ? p.keep : (fit > 0 ? fit : 0);
  }
  const int smem = p.keep * NT * 16 + bitmap;
  auto kernel = distill_kernel<T, CL, GRAD>;
  static bool attr[kMaxDevices] = {};
  set_smem_attr_once(kernel, 208 * 1024, attr, "distill_loss");
  if (smem > 208 * 1024) throw std::runtime_error("distill_loss: vocabulary too large");
  cudaLaunchAttribute cl;
  cl.id = cudaLaunchAttributeClusterDimension;
  cl.val.clusterDim.x = CL;
  cl.val.clusterDim.y = cl.val.clusterDim.z = 1;
  launch_pdl(kernel, dim3((unsigned)(rows * CL)), dim3(NT), smem, stream, CL > 1 ? &cl : nullptr,
             p);
}

template <typename T, bool GRAD>
void launch_t(const Params& p, int64_t rows, cudaStream_t stream) {
  int dev = 0;
  cudaGetDevice(&dev);
  int cl = row_split(rows, p.V / Traits<T>::E, num_sms(dev), NT);
  // The gradient pass wants the whole slice in shared memory.
  if (GRAD)
    while (cl < 8 && (int64_t)p.V * (int)sizeof(T) / cl > kSmemLimit - 16 * 1024) cl *= 2;
  // bitmaps of a very large vocabulary
  while (cl < 8 && p.V / Traits<T>::E / cl > 64 * 1024) cl *= 2;
  switch (cl) {
    case 1: return launch_cl<T, 1, GRAD>(p, rows, stream);
    case 2: return launch_cl<T, 2, GRAD>(p, rows, stream);
    case 4: return launch_cl<T, 4, GRAD>(p, rows, stream);
    default: return launch_cl<T, 8, GRAD>(p, rows, stream);
  }
}

}  // namespace

void distill_launch(const DistillArgs& a, cudaStream_t stream) {
  check(a.in, a.K, "distill_loss");
  if (a.in.rows > 0) {
    Params p{a.in.x, a.t_ids, a.t_lp, a.weights, a.in.ld, a.in.V, a.K, 0, a.tail,
             (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
             (float)((double)a.grad_scale / a.temperature), a.row_loss,
             reinterpret_cast<float4*>(a.stats), a.grad};
    if (a.in.bf16)
      a.grad ? launch_t<__nv_bfloat16, true>(p, a.in.rows, stream)
             : launch_t<__nv_bfloat16, false>(p, a.in.rows, stream);
    else
      a.grad ? launch_t<float, true>(p, a.in.rows, stream)
             : launch_t<float, false>(p, a.in.rows, stream);
  }
  if (a.loss)
    launch_pdl(sum_rows_kernel, dim3(1), dim3(1024), 0, stream, nullptr, (const float*)a.row_loss,
               a.in.rows, a.grad_scale, a.loss);
}

void distill_bwd_launch(const DistillBwdArgs& a, cudaStream_t stream) {
  check(a.in, a.K, "distill_loss_bwd");
  const int E = a.in.bf16 ? 8 : 4;
  const int64_t eb = a.in.bf16 ? 2 : 4;
  const unsigned chunks = (unsigned)((a.in.V + 2 * E - 2) / E + NT * U - 1) / (NT * U);
  for (int64_t r0 = 0; r0 < a.in.rows; r0 += 65535) {  // grid.y limit
    const unsigned n = (unsigned)(a.in.rows - r0 < 65535 ? a.in.rows - r0 : 65535);
    BwdParams b{};
    b.f = Params{reinterpret_cast<const char*>(a.in.x) + r0 * a.in.ld * eb, a.t_ids + r0 * a.K,
                 a.t_lp + r0 * a.K, a.weights ? a.weights + r0 : nullptr, a.in.ld, a.in.V, a.K, 0,
                 a.tail, (float)(1.4426950408889634 / a.temperature), (float)(1.0 / a.temperature),
                 (float)((double)a.g_scale / a.temperature), nullptr,
                 reinterpret_cast<float4*>(const_cast<float*>(a.stats)) + r0,
                 reinterpret_cast<char*>(a.grad) + r0 * a.in.V * eb};
    b.g = a.g_rows + r0 * a.g_stride;
    b.g_stride = a.g_stride;
    if (a.in.bf16)
      launch_pdl(distill_bwd_kernel<__nv_bfloat16>, dim3(chunks, n), dim3(NT), 0, stream, nullptr,
                 b);
    else
      launch_pdl(distill_bwd_kernel<float>, dim3(chunks, n), dim3(NT), 0, stream, nullptr, b);
  }
}

void scale_by_launch(void* x, bool bf16, int64_t n, const float* scale, cudaStream_t stream) {
  if (n <= 0) return;
  int dev = 0;
  cudaGetDevice(&dev);
  const int64_t want = (n + 256 * 8 - 1) / (256 * 8);
  const unsigned grid = (unsigned)(want < 8 * num_sms(dev) ? want : 8 * num_sms(dev));
  if (bf16)
    launch_pdl(scale_by_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, stream, nullptr,
               (__nv_bfloat16*)x, n, scale);
  else
    launch_pdl(scale_by_kernel<float>, dim3(grid), dim3(256), 0, stream, nullptr, (float*)x, n,
               scale);
}

}  // namespace b200
