// Attention of a tree of drafted tokens over the paged cache.
//
// The cache holds a sequence's context and, in its last q_len slots, the keys
// and values of the tree's nodes. Node j attends to every key of the prefix
// (within the sliding window, if there is one) and to the nodes whose bit is
// set in its mask row:
//   o_j = sum_k p_jk v_k / (sum_k p_jk [+ exp(sink)]),  p_jk = exp(scale q_j . k_k)
//
// Rows. The q_len x G (nodes x query heads of a key head) rows of a (sequence,
// key head) are packed into tiles of 128 (row r -> node r / G, head r % G), so
// a key tile is read once for up to 128 rows. tcgen05 works on 128 rows
// whatever their number; with fewer valid rows the spare ones cost tensor
// time that the bytes hide (a 128-key tile is 64 KB: ~2900 SM cycles of HBM
// time against ~1000 of tensor time), and warps without a valid row skip the
// softmax.
//
// Work split. One persistent CTA an SM. The key tiles of all (sequence, key
// head, row tile) units form one list, and CTA c takes the c-th equal share
// of it, whatever the contexts' lengths: ragged batches stay balanced and one
// long context spreads over the whole device. A unit cut at a share's edge
// leaves (max, sum, unnormalised o) pieces in the workspace, which a second
// kernel joins in share order; whole units are written directly. The split
// depends on the lengths only, so results repeat bit for bit.
//
// Eleven warps a CTA:
//   warp 0     K / V producer: one (cache block, 64-column) box a lane, one
//              warp-wide bulk-tensor instruction a tile, into one ring in the
//              order of use K0 K1 V0 K2 V1 ...
//   warp 1     TMEM owner and MMA issuer: S = Q K^T into one of two S buffers,
//              then O += P V of the tile before it
//   warps 2-9  softmax: two threads a row, one for each half of the tile's
//              keys (warps w and w + 4 of the same 32 TMEM lanes), which
//              exchange their maxima through shared memory. Exponentials in
//              base 2 with a lazily raised reference (O is rescaled when a
//              row's max grows by more than 2^8 over it), P as bf16 to TMEM;
//              the unit's epilogue, half of O's columns each
//   warp 10    Q loader: the next unit's rows while the present one runs
// The pipeline runs across units: the next unit's first S is issued before
// the last P V of the present one.
//
// Rounding: P is rounded to bf16 for the tensor core (relative 2^-8 a term at
// most, as the output's own rounding); scores, maxima, sums and O are fp32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "attention/tree_attn.h"
#include "common/launch.h"
#include "common/ptx.cuh"
#include "common/tmap.h"
#include "ops_api.h"

namespace b200 {
namespace {

constexpr int FM = 128;
constexpr int kThreads = 352;
constexpr int kSoftmaxWarps = 8;
constexpr int kBarBytes = 512;
constexpr int kMaxBytes = 2 * 2 * FM * 4;  // [tile parity][half][row] floats
constexpr int kMinShare = 2;  // key tiles of a CTA, at least

template <int D_>
struct Cfg {
  static constexpr int D = D_;
  static constexpr int FN = D <= 128 ? 128 : 64;  // keys of a tile
  static constexpr int kDC = D / 64;              // 64-column chunks of a row
  static constexpr int kQChunk = FM * 128;
  static constexpr int kQBytes = kDC * kQChunk;
  static constexpr int kChunk = FN * 128;
  static constexpr int kTile = kDC * kChunk;      // K or V of a tile
  static constexpr int NQ = D <= 128 ? 2 : 1;     // Q buffers
  static constexpr int NS = D == 64 ? 10 : 5;     // ring slots
  static constexpr int kSmem = NQ * kQBytes + NS * kTile + kBarBytes + kMaxBytes;
  static_assert(2 * FN + D + FN <= 512, "TMEM columns");
  static_assert(kSmem <= 232448, "shared memory");
};

struct Params {
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  const int* block_table;
  const int* seq_lens;
  const int* cu_q;
  const uint32_t* mask;
  const float* sinks;
  float* part_o;        // [grid][2][FM][D]
  float2* part_ml;      // [grid][2][FM]
  long long* seq_tile;  // [num_seqs + 1]: first tile of each sequence, then the share
  int num_seqs, Hq, Hkv, G, block_size, block_shift, max_blocks, num_blocks;
  int mask_words, window;
  long long T, q_stride, o_stride;
  float scale_log2;
  unsigned int* err;
};

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t sw_off(int row, int chunk) {
  return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz)
               : "memory");
}

// One sequence's part of the work.
struct Seq {
  int q0, q_len, seq_len, nodes, prefix, k_first, k_lo, n_tiles, n_rt;
  long long total;  // tiles of all its units
};
template <int FN>
__device__ __forceinline__ Seq load_seq(const Params& p, int s) {
  Seq r;
  r.q0 = p.cu_q[s];
  r.q_len = (int)max(0ll, min((long long)p.cu_q[s + 1], p.T) - r.q0);
  r.seq_len = max(0, p.seq_lens[s]);
  r.nodes = min(r.q_len, r.seq_len);
  r.prefix = r.seq_len - r.nodes;
  // The first key that some node sees: a root sits at position `prefix`.
  r.k_first = p.window > 0 ? max(0, r.prefix - p.window + 1) : 0;
  r.k_lo = r.k_first / FN * FN;
  r.n_tiles = max(1, (r.seq_len - r.k_lo + FN - 1) / FN);
  r.n_rt = (r.q_len * p.G + FM - 1) / FM;
  r.total = (long long)r.n_tiles * r.n_rt * p.Hkv;
  return r;
}

// The units of a CTA's share, in order: unit = key head * n_rt + row tile,
// key tiles [j0, j1) of it.
template <int FN>
struct Walk {
  int s, unit, j0, j1;
  long long off, left;
  Seq q;
  __device__ __forceinline__ Walk(const Params& p, int s0, long long off0, long long n)
      : s(s0), off(off0), left(n) {
    if (left > 0) q = load_seq<FN>(p, s);
  }
  __device__ __forceinline__ bool next(const Params& p) {
    if (left <= 0) return false;
    while (off >= q.total) {
      if (++s >= p.num_seqs) return false;
      q = load_seq<FN>(p, s);
      off = 0;
    }
    unit = (int)(off / q.n_tiles);
    j0 = (int)(off - (long long)unit * q.n_tiles);
    j1 = j0 + (int)min((long long)(q.n_tiles - j0), left);
    off += j1 - j0;
    left -= j1 - j0;
    return true;
  }
  __device__ __forceinline__ int kvh() const { return unit / q.n_rt; }
  __device__ __forceinline__ int row0() const { return unit % q.n_rt * FM; }
};

// 32 bits of a node's mask row from node `o` on (o may be negative); bits of
// nodes outside [0, nodes) are 0.
__device__ __forceinline__ uint32_t mask_word(const uint32_t* row, int words, int nodes, int i) {
  if (i < 0 || i >= words || 32 * i >= nodes) return 0u;
  const int n = nodes - 32 * i;
  const uint32_t w = __ldg(row + i);
  return n >= 32 ? w : w & ((1u << n) - 1u);
}
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* row, int words, int nodes, int o) {
  if (o <= -32 || o >= nodes) return 0u;
  const int i = o >> 5;
  return __funnelshift_r(mask_word(row, words, nodes, i), mask_word(row, words, nodes, i + 1),
                         o & 31);
}
// Bits [lo, hi) of a 32-bit word, clamped to it.
__device__ __forceinline__ uint32_t range_bits(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  if (hi <= lo) return 0u;
  const uint32_t top = hi >= 32 ? 0xffffffffu : (1u << hi) - 1u;
  return top & ~((1u << lo) - 1u);
}

template <int D_>
__global__ void __launch_bounds__(kThreads, 1)
tree_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                 const Params p) {
  using C = Cfg<D_>;
  constexpr int D = C::D, FN = C::FN, kDC = C::kDC, NS = C::NS, NQ = C::NQ;
  // The 128-byte swizzle wants 1024-byte aligned tiles: all shared memory is
  // dynamic, and there is no room for a margin.
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sKV = sQ + NQ * C::kQBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sKV + NS * C::kTile);  // [NS]
  uint64_t* empty = full + NS;                                        // [NS]
  uint64_t* q_full = empty + NS;                                      // [NQ]
  uint64_t* q_empty = q_full + NQ;                                    // [NQ]
  uint64_t* s_full = q_empty + NQ;                                    // [2]
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* p_free = p_full + 2;
  uint64_t* o_full = p_free + 2;
  uint64_t* o_free = o_full + 1;
  uint64_t* pair = o_free + 1;                                        // [4]
  uint64_t* done = pair + 4;
  long long* share_of = reinterpret_cast<long long*>(done + 1);  // sequence, offset, tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(share_of + 3);
  static_assert((2 * NS + 2 * NQ + 8 + 2 + 4 + 1 + 3) * 8 + 4 <= kBarBytes, "barriers");
  float(*sh_max)[2][FM] = reinterpret_cast<float(*)[2][FM]>(sKV + NS * C::kTile + kBarBytes);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_wait();
  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < NQ; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], kSoftmaxWarps);
      mbar_init(&p_full[i], kSoftmaxWarps);
      mbar_init(&p_free[i], 1);
    }
    mbar_init(o_full, 1);
    mbar_init(o_free, kSoftmaxWarps);
    for (int i = 0; i < 4; ++i) mbar_init(&pair[i], 2);
    mbar_init(done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 10) {
    // The share: a scan over the sequences, 32 at a time, for the total and
    // then for the sequence in which this CTA's first tile lies.
    long long total = 0;
    for (int b = 0; b < p.num_seqs; b += 32) {
      const int s = b + lane;
      long long n = s < p.num_seqs ? load_seq<FN>(p, s).total : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += up;
      }
      if (blockIdx.x == 0 && s < p.num_seqs) p.seq_tile[s + 1] = total + n;
      total += __shfl_sync(0xffffffffu, n, 31);
    }
    const long long share =
        max((long long)kMinShare, (total + gridDim.x - 1) / (long long)gridDim.x);
    if (blockIdx.x == 0 && lane == 0) {
      p.seq_tile[0] = 0;
      p.seq_tile[p.num_seqs + 1] = share;
    }
    const long long t0 = share * blockIdx.x;
    const long long n = min(share, total - t0);
    int seq = 0;
    long long off = 0, seen = 0;
    bool found = n <= 0;
    for (int b = 0; b < p.num_seqs && !found; b += 32) {
      const int s = b + lane;
      const long long own = s < p.num_seqs ? load_seq<FN>(p, s).total : 0;
      long long c = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += up;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, seen + c > t0);
      if (hit) {
        const int l = __ffs(hit) - 1;
        seq = b + l;
        off = t0 - (seen + __shfl_sync(0xffffffffu, c - own, l));
        found = true;
      }
      seen += __shfl_sync(0xffffffffu, c, 31);
    }
    if (lane == 0) {
      share_of[0] = seq;
      share_of[1] = off;
      share_of[2] = n > 0 ? n : 0;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base, tO = tmem_base + 2 * FN, tP = tO + D;
  const int N = (int)share_of[2];  // key tiles of this CTA
  Walk<FN> walk(p, (int)share_of[0], share_of[1], share_of[2]);
  // Ring position of V_n; K_n sits at 2n - 1 (K_0 at 0).
  auto pos_v = [&](int n) { return n == N - 1 ? 2 * N - 1 : 2 * n + 2; };

  if (warp == 0) {
    // -------------------------------------------------------------- producer
    const int BS = p.block_size;
    const int nb = BS >= FN ? 1 : FN / BS;
    const int rows_box = BS >= FN ? FN : BS;
    const int bi = lane % nb, h = lane / nb;
    struct Box {
      int blk, y;
    };
    // Tile j of the present unit: this lane's cache block and row.
    auto box_of = [&](int j) {
      const int kbase = walk.q.k_lo + j * FN;
      const int last = min(max(0, (walk.q.seq_len - 1) >> p.block_shift), p.max_blocks - 1);
      const int b = min((kbase >> p.block_shift) + bi, last);
      const int id = __ldg(p.block_table + (long long)walk.s * p.max_blocks + b);
      Box x;
      x.blk = in_bounds(id >= 0 && id < p.num_blocks, p.err) ? id : 0;
      x.y = walk.kvh() * BS + (BS > FN ? (kbase & (BS - 1)) : 0);
      return x;
    };
    int pos = 0;
    auto put = [&](const CUtensorMap* tm, const Box& x) -> bool {
      const int st = pos % NS;
      int ok = 1;
      if (lane == 0) {
        ok = mbar_wait(&empty[st], (uint32_t)(((pos / NS) & 1) ^ 1), p.err) ? 1 : 0;
        if (ok) mbar_arrive_expect_tx(&full[st], (uint32_t)C::kTile);
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
      if (h < kDC)
        tma_load_3d(sKV + st * C::kTile + h * C::kChunk + bi * rows_box * 128, tm, &full[st],
                    h * 64, x.y, x.blk);
      ++pos;
      return true;
    };
    bool ok = true, more = walk.next(p);
    int j = more ? walk.j0 : 0;
    Box cur{0, 0}, before{0, 0};
    if (more) cur = box_of(j);
    for (int n = 0; n < N && ok; ++n) {
      // Ids one tile ahead of their use.
      Box nxt = cur;
      if (more && ++j == walk.j1) {
        more = walk.next(p);
        j = more ? walk.j0 : 0;
      }
      if (more) nxt = box_of(j);
      ok = put(&tmk, cur) && (n == 0 || put(&tmv, before));
      before = cur;
      cur = nxt;
    }
    if (ok && N > 0) put(&tmv, before);
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0 && N > 0) {
      constexpr uint32_t idesc_s = umma_idesc_f16(FM, FN, true);
      constexpr uint32_t idesc_pv = umma_idesc_f16(FM, D, true) | (1u << 16);  // B MN-major
      int units_s = 0, units_o = 0;  // units whose S / whose P V has begun
      auto pv = [&](int n, bool first, bool last) -> bool {
        const int pos = pos_v(n), st = pos % NS, pb = n & 1;
        if (first) {
          // O is free once the epilogue of the unit before has read it.
          if (!mbar_wait(o_free, (uint32_t)((units_o & 1) ^ 1), p.err)) return false;
          ++units_o;
        }
        if (!mbar_wait(&p_full[pb], (uint32_t)((n >> 1) & 1), p.err) ||
            !mbar_wait(&full[st], (uint32_t)((pos / NS) & 1), p.err))
          return false;
        tc_fence_after();
        const uint32_t sv = smem_u32(sKV + st * C::kTile);
#pragma unroll
        for (int s = 0; s < FN / 16; ++s) {
          const uint64_t bv = umma_desc_sw128_mn(sv + s * 16 * 128, C::kChunk, 1024u);
          umma_f16_ts(tO, tP + pb * (FN / 2) + s * 8, bv, idesc_pv, (!first || s > 0) ? 1u : 0u);
        }
        umma_commit(&p_free[pb]);
        umma_commit(&empty[st]);
        if (last) umma_commit(o_full);
        return true;
      };
      bool ok = true, first_b = false, last_b = false;
      int n = 0;
      while (ok && walk.next(p)) {
        const int qb = units_s % NQ;
        ok = mbar_wait(&q_full[qb], (uint32_t)((units_s / NQ) & 1), p.err);
        ++units_s;
        for (int j = walk.j0; j < walk.j1 && ok; ++j, ++n) {
          const int pos = n == 0 ? 0 : 2 * n - 1, st = pos % NS, sb = n & 1;
          if (!mbar_wait(&s_free[sb], (uint32_t)(((n >> 1) & 1) ^ 1), p.err) ||
              !mbar_wait(&full[st], (uint32_t)((pos / NS) & 1), p.err)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sq = smem_u32(sQ + qb * C::kQBytes);
          const uint32_t sk = smem_u32(sKV + st * C::kTile);
#pragma unroll
          for (int kb = 0; kb < kDC; ++kb) {
            const uint64_t aq = umma_desc_sw128(sq + kb * C::kQChunk);
            const uint64_t bk = umma_desc_sw128(sk + kb * C::kChunk);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16(tS + sb * FN, aq + (uint64_t)(2 * k), bk + (uint64_t)(2 * k), idesc_s,
                       (kb > 0 || k > 0) ? 1u : 0u);
          }
          umma_commit(&s_full[sb]);
          umma_commit(&empty[st]);
          if (j == walk.j1 - 1) umma_commit(&q_empty[qb]);
          if (n > 0) ok = pv(n - 1, first_b, last_b);
          first_b = j == walk.j0;
          last_b = j == walk.j1 - 1;
        }
      }
      if (ok) pv(N - 1, first_b, last_b);
      // Every MMA done before the TMEM goes.
      umma_commit(done);
      mbar_wait(done, 0, p.err);
    }
    __syncwarp();
  } else if (warp == 10) {
    // -------------------------------------------------------------- Q loader
    int units = 0;
    while (walk.next(p)) {
      const int qb = units % NQ;
      int ok = 1;
      if (lane == 0) ok = mbar_wait(&q_empty[qb], (uint32_t)(((units / NQ) & 1) ^ 1), p.err) ? 1 : 0;
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      const int row0 = walk.row0(), kvh = walk.kvh();
      const int rows = min(FM, walk.q.q_len * p.G - row0);
      const uint32_t dst = smem_u32(sQ + qb * C::kQBytes);
      // Spare rows of a softmax warp that has valid ones are zero; the others
      // are never looked at.
      const int fill = (rows + 31) / 32 * 32;
      for (int i = lane; i < fill * (D / 8); i += 32) {
        const int r = i / (D / 8), ch = i % (D / 8);
        const bool valid = r < rows;
        const int g = row0 + (valid ? r : 0);
        const __nv_bfloat16* src = p.q + (long long)(walk.q.q0 + g / p.G) * p.q_stride +
                                   (long long)(kvh * p.G + g % p.G) * D + ch * 8;
        cp_async_16(dst + (ch >> 3) * C::kQChunk + sw_off(r, ch & 7), src, valid);
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[qb]);
      ++units;
    }
  } else {
    // --------------------------------------------------------------- softmax
    const int q4 = warp & 3;         // the 32 TMEM lanes this warp may touch
    const int half = (warp - 2) / 4; // which half of the tile's keys
    const int row = q4 * 32 + lane;
    const int stid = (int)threadIdx.x - 64;  // 0 .. 255
    constexpr int HN = FN / 2;               // keys of a half
    constexpr int HD = D / 2;                // O columns of a half
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const float sc = p.scale_log2;
    const uint64_t sc2 = f32x2_pack(sc, sc);
    bool ok = true;
    int n = 0, units = 0, meets = 0;
    // Both warps of these 32 rows meet (a wait with a limit, like the others:
    // either may have given up).
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair[q4]);
      const bool r = mbar_wait(&pair[q4], (uint32_t)(meets & 1), p.err);
      ++meets;
      return __all_sync(0xffffffffu, r);
    };
    while (ok && walk.next(p)) {
      const int row0 = walk.row0(), kvh = walk.kvh();
      const int n_rows = walk.q.q_len * p.G - row0;
      const bool valid = row < n_rows;
      const bool warp_on = q4 * 32 < n_rows;
      const int node = (row0 + (valid ? row : 0)) / p.G;
      const int head = kvh * p.G + (row0 + (valid ? row : 0)) % p.G;
      const uint32_t* mrow = p.mask + (long long)(walk.q.q0 + node) * p.mask_words;
      const int nodes = walk.q.nodes, prefix = walk.q.prefix, seq_len = walk.q.seq_len;
      // First key of the prefix this row sees. A node's position is the
      // prefix plus its depth, the number of its ancestors.
      int key_lo = 0;
      if (p.window > 0 && warp_on) {
        int depth = 0;
        for (int i = 0; 32 * i < nodes; ++i)
          depth += __popc(mask_word(mrow, p.mask_words, nodes, i));
        key_lo = prefix + max(depth - 1, 0) - p.window + 1;
      }
      // Exponent reference (log2 units; the same in both halves), this half's sum.
      float m_used = -INFINITY, l = 0.f;
      for (int j = walk.j0; j < walk.j1; ++j, ++n) {
        const int sb = n & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[sb], (uint32_t)((n >> 1) & 1), p.err));
        if (!ok) break;
        tc_fence_after();
        const int kbase = walk.q.k_lo + j * FN;
        const int kb = kbase + half * HN;
        if (warp_on) {
          // The half row of scores, masked, and its maximum.
          uint32_t r[HN / 32][32];
#pragma unroll
          for (int w = 0; w < HN / 32; ++w)
            tmem_ld_32x32b_x32(tS + lane_base + sb * FN + half * HN + w * 32, r[w]);
          tmem_wait_ld();
          if (__any_sync(0xffffffffu, key_lo > kb) || kb + HN > prefix) {
#pragma unroll
            for (int w = 0; w < HN / 32; ++w) {
              const int k0 = kb + 32 * w;
              const uint32_t vis = valid ? range_bits(key_lo - k0, prefix - k0) |
                                               mask_bits(mrow, p.mask_words, nodes, k0 - prefix)
                                         : 0u;
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((vis >> i) & 1u)) r[w][i] = 0xff800000u;
            }
          }
          float mxs[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int w = 0; w < HN / 32; ++w)
#pragma unroll
            for (int i = 0; i < 32; ++i) mxs[i & 3] = fmaxf(mxs[i & 3], __uint_as_float(r[w][i]));
          const float own = fmaxf(fmaxf(mxs[0], mxs[1]), fmaxf(mxs[2], mxs[3]));
          sh_max[sb][half][row] = own;
          ok = meet();
          if (!ok) break;
          float mx = fmaxf(own, sh_max[sb][half ^ 1][row]);
          mx = mx == -INFINITY ? mx : mx * sc;
          const bool resc = mx > m_used + 8.f || (m_used == -INFINITY && mx != -INFINITY);
          if (__any_sync(0xffffffffu, resc)) {
            const float alpha = !resc ? 1.f : m_used == -INFINITY ? 0.f : exp2f(m_used - mx);
            if (resc) {
              l *= alpha;
              m_used = mx;
            }
            if (j > walk.j0) {
              // O is final for the tiles before once P V of tile n - 1 is done.
              ok = __all_sync(0xffffffffu, mbar_wait(&p_free[sb ^ 1],
                                                     (uint32_t)(((n - 1) >> 1) & 1), p.err));
              if (!ok) break;
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < HD / 32; ++c) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tO + lane_base + half * HD + c * 32, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st_32x32b_x32(tO + lane_base + half * HD + c * 32, o);
              }
            }
          }
          const float mu = m_used == -INFINITY ? 0.f : m_used;
          const uint64_t nmu2 = f32x2_pack(-mu, -mu);
          uint64_t acc[2] = {f32x2_pack(0.f, 0.f), f32x2_pack(0.f, 0.f)};
          uint32_t w[HN / 2];
#pragma unroll
          for (int i = 0; i < HN / 2; ++i) {
            float ea, eb;
            f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(r[i >> 4][(2 * i) & 31]),
                                              __uint_as_float(r[i >> 4][(2 * i + 1) & 31])),
                                   sc2, nmu2),
                         ea, eb);
            ea = fast_exp2(ea);
            eb = fast_exp2(eb);
            acc[i & 1] = f32x2_add(acc[i & 1], f32x2_pack(ea, eb));
            w[i] = pack_bf16x2(ea, eb);
          }
          float a0, a1;
          f32x2_unpack(f32x2_add(acc[0], acc[1]), a0, a1);
          l += a0 + a1;
          // This P buffer is free once P V of tile n - 2 has completed.
          if (n >= 2) ok = mbar_wait(&p_free[sb], (uint32_t)(((n - 2) >> 1) & 1), p.err);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const uint32_t p_row = tP + lane_base + sb * (FN / 2) + half * (HN / 2);
          if constexpr (HN == 64)
            tmem_st_32x32b_x32(p_row, *reinterpret_cast<uint32_t(*)[32]>(w));
          else
            tmem_st_32x32b_x16(p_row, *reinterpret_cast<uint32_t(*)[16]>(w));
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[sb]);
        if (kbase + FN > seq_len || kbase < walk.q.k_first) {
          // V rows that no node sees (past the end, before the window) may
          // hold anything, and 0 x NaN is not 0: they become zero.
          const int pos = pos_v(n);
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&full[pos % NS], (uint32_t)((pos / NS) & 1), p.err));
          if (!ok) break;
          uint8_t* sv = sKV + (pos % NS) * C::kTile;
          constexpr int kU = D / 8;
          for (int i = stid; i < FN * kU; i += kSoftmaxWarps * 32) {
            const int k = i / kU, c16 = i % kU;
            if (kbase + k >= seq_len || kbase + k < walk.q.k_first)
              *reinterpret_cast<uint4*>(sv + (c16 >> 3) * C::kChunk + sw_off(k, c16 & 7)) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_shared();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&p_full[sb]);
      }
      if (!ok) break;
      // ---------------------------------------------------- the unit's epilogue
      if (warp_on) {
        // (The buffer is the next unit's first tile's, hence the second meeting.)
        sh_max[n & 1][half][row] = l;
        ok = meet();
        if (!ok) break;
        l = sh_max[n & 1][0][row] + sh_max[n & 1][1][row];
        ok = meet();
        if (!ok) break;
      }
      ok = __all_sync(0xffffffffu, mbar_wait(o_full, (uint32_t)(units & 1), p.err));
      if (!ok) break;
      ++units;
      tc_fence_after();
      if (warp_on) {
        const bool whole = walk.j0 == 0 && walk.j1 == walk.q.n_tiles;
        float f = 1.f;
        if (whole) {
          float den = l;
          if (p.sinks != nullptr)
            den = m_used == -INFINITY ? 1.f
                                      : l + exp2f(p.sinks[head] * 1.4426950408889634f - m_used);
          f = den > 0.f ? 1.f / den : 0.f;
        }
        __nv_bfloat16* dst = p.out + (long long)(walk.q.q0 + node) * p.o_stride +
                             (long long)head * D + half * HD;
        const long long piece = ((long long)blockIdx.x * 2 + (walk.j0 > 0 ? 0 : 1)) * FM + row;
        float* part = p.part_o + piece * D + half * HD;
        if (!whole && valid && half == 0) p.part_ml[piece] = make_float2(m_used, l);
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + lane_base + half * HD + c * 32, o);  // warp-collective
          tmem_wait_ld();
          if (!valid) continue;
          if (whole) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(__uint_as_float(o[8 * v + 2 * e]) * f,
                                   __uint_as_float(o[8 * v + 2 * e + 1]) * f);
              *reinterpret_cast<uint4*>(dst + c * 32 + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4*>(part + c * 32 + v * 4) =
                  make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the pieces of units that were cut, in share order: one warp a
// (token, head) row. Rows of whole units return at once.
template <int D_>
__global__ void __launch_bounds__(128) tree_join_kernel(const Params p) {
  constexpr int D = D_, FN = Cfg<D_>::FN;
  constexpr int V = D >= 128 ? D / 128 : 1;  // float4 of a lane
  pdl_wait();
  pdl_trigger();
  const long long id = (long long)blockIdx.x * 4 + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  if (id >= p.T * p.Hq) return;
  const int tok = (int)(id / p.Hq), head = (int)(id % p.Hq);
  // The token's sequence: the last s with cu_q[s] <= tok.
  int lo = 0, hi = p.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (p.cu_q[mid] <= tok) lo = mid;
    else hi = mid - 1;
  }
  const Seq q = load_seq<FN>(p, lo);
  if (tok < q.q0 || tok >= q.q0 + q.q_len) return;
  const int g = (tok - q.q0) * p.G + head % p.G;
  const int unit = head / p.G * q.n_rt + g / FM, row = g % FM;
  const long long share = p.seq_tile[p.num_seqs + 1];
  const long long a = p.seq_tile[lo] + (long long)unit * q.n_tiles, b = a + q.n_tiles;
  const int c0 = (int)(a / share), c1 = (int)((b - 1) / share);
  if (c0 == c1) return;
  auto piece = [&](int c) {
    return ((long long)c * 2 + (a < c * share ? 0 : 1)) * FM + row;
  };
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, p.part_ml[piece(c)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float den = 0.f;
  float4 acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool on = D >= 128 || lane < D / 4;
  for (int c = c0; c <= c1; ++c) {
    const long long pc = piece(c);
    const float2 ml = p.part_ml[pc];
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
    den += ml.y * f;
    if (on) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float4 o = *reinterpret_cast<const float4*>(p.part_o + pc * D + (v * 32 + lane) * 4);
        acc[v].x += o.x * f;
        acc[v].y += o.y * f;
        acc[v].z += o.z * f;
        acc[v].w += o.w * f;
      }
    }
  }
  if (p.sinks != nullptr)
    den = m == -INFINITY ? 1.f : den + exp2f(p.sinks[head] * 1.4426950408889634f - m);
  const float inv = den > 0.f ? 1.f / den : 0.f;
  if (on) {
    __nv_bfloat16* dst = p.out + (long long)tok * p.o_stride + (long long)head * D;
#pragma unroll
    for (int v = 0; v < V; ++v)
      *reinterpret_cast<uint2*>(dst + (v * 32 + lane) * 4) =
          make_uint2(pack_bf16x2(acc[v].x * inv, acc[v].y * inv),
                     pack_bf16x2(acc[v].z * inv, acc[v].w * inv));
  }
}

template <int D_>
void launch_d(const TreeAttnArgs& a, cudaStream_t stream) {
  using C = Cfg<D_>;
  constexpr int D = C::D, FN = C::FN;
  auto kernel = tree_attn_kernel<D>;
  static bool attr[kMaxDevices] = {};
  set_smem_attr_once(kernel, C::kSmem, attr, "tree_attention");
  const int BS = a.block_size;
  const uint64_t rows = (uint64_t)a.Hkv * BS;
  const uint32_t box = (uint32_t)(BS >= FN ? FN : BS);
  CUtensorMap tk = make_tmap_3d(a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                (uint64_t)a.num_blocks, rows, D, (uint64_t)D * 2,
                                (uint64_t)a.kv_block_stride * 2, 1, box, 64);
  CUtensorMap tv = make_tmap_3d(a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2,
                                (uint64_t)a.num_blocks, rows, D, (uint64_t)D * 2,
                                (uint64_t)a.kv_block_stride * 2, 1, box, 64);
  int dev = 0;
  cudaGetDevice(&dev);
  const int grid = num_sms(dev);
  Params p{};
  p.q = reinterpret_cast<const __nv_bfloat16*>(a.q);
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.block_table = a.block_table;
  p.seq_lens = a.seq_lens;
  p.cu_q = a.cu_q;
  p.mask = a.tree_mask;
  p.sinks = a.sinks;
  p.part_o = a.workspace;
  p.part_ml = reinterpret_cast<float2*>(a.workspace + (size_t)grid * 2 * FM * D);
  p.seq_tile = reinterpret_cast<long long*>(p.part_ml + (size_t)grid * 2 * FM);
  p.num_seqs = a.num_seqs;
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.G = a.Hq / a.Hkv;
  p.block_size = BS;
  p.block_shift = __builtin_ctz(BS);
  p.max_blocks = a.max_blocks;
  p.num_blocks = a.num_blocks;
  p.mask_words = a.mask_words;
  p.window = a.window;
  p.T = a.num_tokens;
  p.q_stride = a.q_stride_t;
  p.o_stride = a.o_stride_t;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.err = device_status_ptr(dev);
  launch_pdl(kernel, dim3(grid), dim3(kThreads), C::kSmem, stream, nullptr, tk, tv, p);
  launch_pdl(tree_join_kernel<D>, dim3((unsigned)((a.num_tokens * a.Hq + 3) / 4)), dim3(128), 0,
             stream, nullptr, p);
}

}  // namespace

size_t tree_attention_workspace_bytes(int num_seqs, int head_dim, int num_sm) {
  return (size_t)num_sm * 2 * FM * (head_dim + 2) * 4 + (size_t)(num_seqs + 2) * 8;
}

void tree_attention_launch(const TreeAttnArgs& a, cudaStream_t stream) {
  if (a.Hkv < 1 || a.Hq % a.Hkv != 0)
    throw std::runtime_error("tree_attention: Hq must be a multiple of Hkv");
  if (a.block_size < 8 || (a.block_size & (a.block_size - 1)) != 0)
    throw std::runtime_error("tree_attention: block_size must be a power of two >= 8");
  if (a.num_tokens <= 0 || a.num_seqs <= 0) return;
  switch (a.head_dim) {
    case 64: return launch_d<64>(a, stream);
    case 128: return launch_d<128>(a, stream);
    case 256: return launch_d<256>(a, stream);
    default: throw std::runtime_error("tree_attention: head_dim must be 64, 128 or 256");
  }
}

}  // namespace b200
