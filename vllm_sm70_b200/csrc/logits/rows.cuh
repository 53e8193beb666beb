// Building blocks of the kernels that stream rows of logits.
//
// A row is walked as 16-byte vectors from the last 16-byte boundary at or
// before its first element: `pad` elements of the first vector lie before the
// row, so only the first and the last vector can be partial, whatever V, the
// row stride or the base address are. Elements outside the row read as -inf,
// which adds nothing to any sum, maximum or count below.
//
// Sums of exponentials are kept in base 2 against the largest element m of
// what was seen: e_j = 2^((x_j - m) c), c = log2(e) / T. x_j - m is rounded
// once, relative to itself, so elements near the top are exact to 2^-24 however
// large m is, and m may be the type's lowest value (m c would overflow).
// p_j = e_j / s, log p_j = ((x_j - m) c - log2 s) ln 2. The long sums take one
// fused product x_j c - r instead, r the rounded m c: what r lacks of m c is
// known exactly (one more fused product) and taken out of the sum at the end.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstring>

#include "common/launch.h"
#include "common/ptx.cuh"

namespace b200 {
namespace rows {

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// How far out a maximum m may lie for m c to be taken out of x c. r is off by up
// to 2^-24 |m c|, and against r every exponential of the row is off by as many
// powers of 2, which have to fit fp32: 64 of them at kFar. A sum of e_j d_j
// (the entropy's) loses 2^-24 of r's error times its number of steps besides:
// half a power of 2 at kFarEntropy. Parts of rows whose maximum lies further
// out are summed element by element (slow_sum, slow_sums).
constexpr float kFar = 1610612736.f;  // 1.5 * 2^30
constexpr float kFarEntropy = 16777216.f;  // 2^24
__device__ __forceinline__ bool slow_range(float m, float c, float far) {
  return !(fabsf(m * c) <= far);
}

// In sums that go on before the maximum is known, elements below this count as
// this: -2^31 / c, cut to a bf16 value. Against a maximum within kFar their
// exponentials are zero all the same, and what a thread sums while it has seen
// nothing else stays finite.
inline float floor_of(float c) {
  const float f = -2147483648.f / c;
  uint32_t b;
  memcpy(&b, &f, 4);
  b &= 0xffff0000u;
  float r;
  memcpy(&r, &b, 4);
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// 16 bytes to shared memory behind the thread's back; both 16-byte aligned.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// Order-preserving 32-bit key: a larger value has a larger key, -0 and +0
// the same; NaN has key 0, below every number's.
__device__ __forceinline__ uint32_t key_of(float f) {
  if (f != f) return 0u;
  const uint32_t b = __float_as_uint(f + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

template <typename T>
struct Traits;

template <>
struct Traits<__nv_bfloat16> {
  static constexpr int E = 8;                        // elements of a 16-byte vector
  static constexpr uint32_t kNegInf = 0xff80ff80u;   // one word of -inf elements
  __device__ static __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
  // Elements 2i and 2i + 1 of a vector.
  __device__ static __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    a = bf16_bits_lo(w);
    b = bf16_bits_hi(w);
  }
  // A vector's maximum, kept packed; NaN elements do not count.
  using Max = __nv_bfloat162;
  __device__ static __forceinline__ Max vmax(const uint4& v) {
    const __nv_bfloat162 a = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&v.x),
                                     *reinterpret_cast<const __nv_bfloat162*>(&v.y));
    const __nv_bfloat162 b = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&v.z),
                                     *reinterpret_cast<const __nv_bfloat162*>(&v.w));
    return __hmax2(a, b);
  }
  __device__ static __forceinline__ Max vmax(Max a, Max b) { return __hmax2(a, b); }
  __device__ static __forceinline__ float value(Max m) {
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ static __forceinline__ float max_of(const uint4& v) { return value(vmax(v)); }
  // Is every element below y (an element's value)?
  __device__ static __forceinline__ bool all_below(Max m, float y) {
    return __hblt2(m, __float2bfloat162_rn(y));
  }
  // Elements 2i and 2i + 1, not below `least` (a bf16 value).
  __device__ static __forceinline__ void pair_floor(const uint4& v, int i, float least, float& a,
                                                    float& b) {
    const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
    const __nv_bfloat162 f = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w),
                                         __float2bfloat162_rn(least));
    const uint32_t u = *reinterpret_cast<const uint32_t*>(&f);
    a = bf16_bits_lo(u);
    b = bf16_bits_hi(u);
  }
  // Packed counter of elements above (or, GE, at or above) a value: adds one
  // 16-bit all-ones mask a hit. n = lo + hi with sum = 65536 (lo - hi) - lo.
  template <bool GE>
  __device__ static __forceinline__ void count(const uint4& v, float y, uint32_t& acc) {
    const __nv_bfloat162 y2 = __float2bfloat162_rn(y);  // exact: y is one of the elements
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 x2 = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      acc += GE ? __hge2_mask(x2, y2) : __hgt2_mask(x2, y2);
    }
  }
  __device__ static __forceinline__ int counted(uint32_t acc) {
    const uint32_t lo = (0u - acc) & 0xffffu;
    const uint32_t diff = (acc + lo) >> 16;  // lo - hi mod 2^16
    return (int)lo + (int)((lo - diff) & 0xffffu);
  }
  // The elements whose bit is set, as -inf.
  __device__ static __forceinline__ void blank(uint4& v, uint32_t bits) {
    uint32_t* w[4] = {&v.x, &v.y, &v.z, &v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = ((bits >> (2 * i)) & 1u ? 0x0000ffffu : 0u) |
                         ((bits >> (2 * i)) & 2u ? 0xffff0000u : 0u);
      *w[i] = (*w[i] & ~m) | (kNegInf & m);
    }
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
  __device__ static __forceinline__ __nv_bfloat16 from_f(float f) { return __float2bfloat16_rn(f); }
};

template <>
struct Traits<float> {
  static constexpr int E = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  __device__ static __forceinline__ float to_f(float v) { return v; }
  __device__ static __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    a = __uint_as_float(i == 0 ? v.x : v.z);
    b = __uint_as_float(i == 0 ? v.y : v.w);
  }
  using Max = float;
  __device__ static __forceinline__ Max vmax(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ static __forceinline__ Max vmax(Max a, Max b) { return fmaxf(a, b); }
  __device__ static __forceinline__ float value(Max m) { return m; }
  __device__ static __forceinline__ float max_of(const uint4& v) { return vmax(v); }
  __device__ static __forceinline__ bool all_below(Max m, float y) { return m < y; }
  __device__ static __forceinline__ void pair_floor(const uint4& v, int i, float least, float& a,
                                                    float& b) {
    pair(v, i, a, b);
    a = max_nan(a, least);
    b = max_nan(b, least);
  }
  template <bool GE>
  __device__ static __forceinline__ void count(const uint4& v, float y, uint32_t& acc) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = __uint_as_float(w[i]);
      acc += (GE ? x >= y : x > y) ? 1u : 0u;
    }
  }
  __device__ static __forceinline__ int counted(uint32_t acc) { return (int)acc; }
  __device__ static __forceinline__ void blank(uint4& v, uint32_t bits) {
    if (bits & 1u) v.x = kNegInf;
    if (bits & 2u) v.y = kNegInf;
    if (bits & 4u) v.z = kNegInf;
    if (bits & 8u) v.w = kNegInf;
  }
  __device__ static __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  __device__ static __forceinline__ float from_f(float f) { return f; }
};

// One row as aligned vectors (see the head of this file).
template <typename T>
struct Row {
  static constexpr int E = Traits<T>::E;
  const T* x;    // the row's first element
  int pad, V;
  int n_vec;     // vectors that hold some element of the row
  int full_lo;   // first full vector
  uint32_t n_full;

  __device__ __forceinline__ Row(const void* base, int64_t row, int64_t ld, int V_) : V(V_) {
    x = reinterpret_cast<const T*>(base) + row * ld;
    pad = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    n_vec = (pad + V + E - 1) / E;
    full_lo = pad > 0 ? 1 : 0;
    const int full_hi = (pad + V) / E;
    n_full = full_hi > full_lo ? (uint32_t)(full_hi - full_lo) : 0u;
  }
  __device__ __forceinline__ bool full(int u) const { return (uint32_t)(u - full_lo) < n_full; }
  __device__ __forceinline__ int index(int u, int e) const { return u * E + e - pad; }
  __device__ __forceinline__ uint4 load(int u) const {
    if (full(u)) return ldg_stream(x + ((int64_t)u * E - pad));
    return load_partial(x, u * E - pad, V);
  }
  // Elements i0 .. i0 + E - 1, those outside [0, V) as -inf. (By value and out
  // of line: at most two vectors of a row come here.)
  __device__ static __noinline__ uint4 load_partial(const T* x, int i0, int V) {
    union {
      uint4 v;
      T e[E];
      uint32_t w[4];
    } r;
    r.w[0] = r.w[1] = r.w[2] = r.w[3] = Traits<T>::kNegInf;
    for (int e = 0; e < E; ++e)
      if (i0 + e >= 0 && i0 + e < V) r.e[e] = x[i0 + e];
    return r.v;
  }
};

// Part `part` of `parts` of a row's vectors: [lo, hi), of which [a, b) are
// full; the row's first and last vector, where they are partial and here (-1
// otherwise), belong to threads 0 and 1.
struct Slice {
  int lo, hi, a, b, head, tail;
  template <typename T>
  __device__ __forceinline__ Slice(const Row<T>& row, int part, int parts) {
    const int per = (row.n_vec + parts - 1) / parts;
    lo = min(part * per, row.n_vec);
    hi = min(lo + per, row.n_vec);
    const int full_hi = row.full_lo + (int)row.n_full;
    a = max(lo, row.full_lo);
    b = max(a, min(hi, full_hi));
    head = lo == 0 && hi > 0 && row.full_lo > 0 ? 0 : -1;
    tail = hi == row.n_vec && hi > lo && hi > full_hi && hi - 1 != head ? hi - 1 : -1;
  }
};

// Calls f(v, u0, it) for groups it = 0 .. of U vectors of this thread, those of
// vectors u0 + k NT; vectors past the end are -inf. The partial vectors make a
// last group, of warp 0 alone. The next group's loads are out while one is
// worked on. Full groups run without checks: at the rate HBM
// delivers, an SM has some ten issue slots an element.
template <int NT, int U, typename T, typename F>
__device__ __forceinline__ void for_groups(const Row<T>& row, const Slice& s, F&& f) {
  const uint4 none = make_uint4(Traits<T>::kNegInf, Traits<T>::kNegInf, Traits<T>::kNegInf,
                                Traits<T>::kNegInf);
  const int tid = threadIdx.x, n = s.b - s.a;
  const uint4* p = reinterpret_cast<const uint4*>(row.x - row.pad) + s.a + tid;
  uint4 v[U];
  int left = n, u = s.a + tid, it = 0;
  if (left >= U * NT) {
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = ldg_stream(p + k * NT);
#pragma unroll 2
    while (left >= 2 * U * NT) {
      uint4 w[U];
      p += U * NT;
#pragma unroll
      for (int k = 0; k < U; ++k) w[k] = ldg_stream(p + k * NT);
      f(v, u, it++);
      u += U * NT;
      left -= U * NT;
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = w[k];
    }
    p += U * NT;
    left -= U * NT;
    if (left > 0) {
      uint4 w[U];
#pragma unroll
      for (int k = 0; k < U; ++k) w[k] = tid + k * NT < left ? ldg_stream(p + k * NT) : none;
      f(v, u, it++);
#pragma unroll
      for (int k = 0; k < U; ++k) v[k] = w[k];
      u += U * NT;
    }
    f(v, u, it++);
  } else if (left > 0) {
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = tid + k * NT < left ? ldg_stream(p + k * NT) : none;
    f(v, u, it++);
  }
  if ((s.head >= 0 || s.tail >= 0) && tid < 32) {
    const int e = tid == 0 ? s.head : tid == 1 ? s.tail : -1;
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = none;
    if (e >= 0) v[0] = row.load(e);
    f(v, e >= 0 ? e : row.n_vec, it);
  }
}

// Calls f(u) for the vectors that for_groups gives this thread: a warp that
// goes over its part again meets what it summed, and nothing of another's.
template <int NT, typename F>
__device__ __forceinline__ void for_vectors(const Slice& s, F&& f) {
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int u = s.a + tid; u < s.b; u += NT) f(u);
  const int e = tid == 0 ? s.head : tid == 1 ? s.tail : -1;
  if (e >= 0) f(e);
}

__device__ __forceinline__ int64_t load_id(const void* ids, bool ids64, int64_t row) {
  return ids64 ? reinterpret_cast<const int64_t*>(ids)[row]
               : (int64_t) reinterpret_cast<const int*>(ids)[row];
}

__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Running sums of a thread, a CTA or a cluster: m = max x, s = sum 2^((x - m) c),
// t = sum 2^((x - m) c) (x - m) c. Empty: m = -inf, s = t = 0.
struct Acc {
  float m, s, t;
};
// What is subtracted from x: the maximum, or 0 while there is none.
__device__ __forceinline__ float shift_of(float m) { return m == -INFINITY ? 0.f : m; }
// The sums of `a` against max `m` >= a.m.
__device__ __forceinline__ void rebase(Acc& a, float m, float c) {
  if (a.m == m) return;
  if (a.m != -INFINITY) {
    const float d = (a.m - m) * c;
    const float f = ex2(d);
    a.t = f == 0.f ? 0.f : f * (a.t + d * a.s);
    a.s *= f;
  }
  a.m = m;
}

// max over the warp of a float that is no NaN
__device__ __forceinline__ float warp_max(float v) {
  return value_of(__reduce_max_sync(0xffffffffu, key_of(v)));
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// CTAs that share a row, by the number of rows: as many as run at the same
// time (`resident`), while a CTA keeps at least `min_vec` vectors. (A second
// wave costs more than larger parts: 128 rows of 128256 took 13 us at 8 CTAs a
// row, in two waves.)
inline int row_split(int64_t rows, int64_t n_vec, int resident, int min_vec) {
  int cl = 1;
  while (cl < 8 && rows * 2 * cl <= resident && n_vec / (2 * cl) >= min_vec) cl *= 2;
  return cl;
}

}  // namespace rows
}  // namespace b200
