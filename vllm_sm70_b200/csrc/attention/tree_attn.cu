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
// time that the bytes hide (a 128-key tile is 64 KB: ~2800 SM cycles of HBM
// time against ~1000 of tensor time), and warps without a valid row skip the
// softmax.
//
// Work split. One persistent CTA an SM. The key tiles of all (sequence, key
// head, row tile) units form one list, and CTA c takes the c-th equal share
// of it (a unit's edge counts as some tiles), whatever the contexts' lengths:
// ragged batches stay balanced and one long context spreads over the whole
// device. A unit cut at a share's edge
// leaves (max, sum, unnormalised o) pieces in the workspace, which a second
// kernel joins in share order; whole units are written directly. The split
// depends on the lengths only, so results repeat bit for bit.
//
// Where every sequence has a multiple of `team` row tiles, the shares are those
// of teams of that many CTAs: each takes another row tile over the same keys at
// about the same time, which HBM then delivers once, and L2 to the others.
//
// Thirteen warps a CTA:
//   warp 0     K producer, warp 1 V producer: one (cache block, 64-column)
//              box a lane, one warp-wide bulk-tensor instruction a tile (that
//              costs its warp ~80 cycles a box, hence two warps), each into a
//              ring of its own: one producer and one consumer, so that a
//              barrier's parity always tells its rounds apart. Warp 0 also walks
//              the share and publishes each unit's numbers, one unit ahead, so
//              that nobody else waits for lengths or divides.
//   warps 2-9  softmax: two groups of four warps, a row a thread, on every
//              other tile, so that one's waits are the other's work. O has one
//              exponent reference a row (base 2, raised lazily: O is rescaled
//              when a row's max grows by more than 2^8 over it), which the
//              groups hand to each other in tile order through shared memory
//              as soon as a tile's maximum is known. P (bf16) goes over the
//              first half of its scores. A unit's epilogue (half of O's
//              columns each) comes after the next unit's first tile, when the
//              last P V has long finished.
//   warp 10    issues S = Q K^T into one of three buffers, as soon as P V of
//              the tile before in it is done
//   warp 11    issues O += P V (its own warp: an issuing thread spends longer
//              on waits and descriptors than the tensor core on a product)
//   warp 12    loads Q rows (the next unit's while the present one runs) and
//              zeroes V rows that no node of the tile sees (past the end,
//              before the window, slots of nodes whose bit is nowhere set):
//              they may hold anything, and 0 x NaN is not 0.
// TMEM columns: S0 | S1 | S2 | O.
//
// Measured (32 query, 8 key heads of 128, blocks of 16), on inputs that change
// from call to call: 64 trees of 8 to 16 nodes over contexts of 1024 to 4096
// tokens (2605 on average, 695 MB) 136 to 143 us, up to 5100 GB/s of the 6454
// that a copy reaches; the steady state is HBM's, the rest is the start, a few
// us at each unit's edge, and the join. Trees of 64 and 45 nodes over 60001 and
// 42812 tokens (94.6 TFLOP) 148 to 152 us, 640 TFLOP/s; on the same inputs again
// and again, when a part of them stays in L2, 129. Bound by a group's way from
// scores to P, ~3300 cycles of which 1900 are the exponentials, a tile every
// ~1900. A third group with a buffer each was no faster (S of tile n + 3 then
// waits for P V of tile n), nor were exponentials on the FMA pipe or scores
// fetched ahead.
//
// Rounding: P is rounded to bf16, since one product has operands of one type
// and V is bf16 (relative 2^-8 a term at most, as the output's own rounding; the
// output's error against 64 bits, relative to its norm, is 0.0023 with it and
// 0.0017 without). Scores, maxima, sums and O are fp32; a row's sum adds the
// exponentials before that rounding.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "attention/exp2.cuh"
#include "attention/tree_attn.h"
#include "common/launch.h"
#include "common/ptx.cuh"
#include "common/tmap.h"
#include "ops_api.h"

namespace b200 {
namespace {

constexpr int FM = 128;
constexpr int kThreads = 416;
constexpr int kSoftmaxWarps = 8;
constexpr int kBarBytes = 1024;  // barriers and published units
constexpr int kUnits = 4;       // published units
constexpr int kRowBytes = 3 * FM * 4;  // a reference and two sums a row
constexpr int kMaxTeam = 8;  // CTAs that read the same keys
constexpr int kMinShare = 2;  // key tiles of a CTA, at least

template <int D_>
struct Cfg {
  static constexpr int D = D_;
  static constexpr int FN = D <= 128 ? 128 : 64;  // keys of a tile
  static constexpr int kDC = D / 64;              // 64-column chunks of a row
  static constexpr int kQChunk = FM * 128;
  static constexpr int kQBytes = kDC * kQChunk;
  static constexpr int NQ = D <= 128 ? 2 : 1;     // Q buffers
  static constexpr int kChunk = FN * 128;
  static constexpr int kTile = kDC * kChunk;      // K or V of a tile
  static constexpr int NK = D == 64 ? 6 : 2;      // K ring slots
  static constexpr int NV = D == 64 ? 6 : 3;      // V: held until P is there, two tiles on
  // What a unit's edge costs, in tiles: a masked tile, the output, at D = 256
  // also the wait for Q's one buffer. Shares of several short units get fewer
  // tiles (16 trees of up to 24 nodes over 2000 to 8000 tokens, 16/2 heads of
  // 256, window 4096: 72 -> 64 us; 64 of up to 8 nodes over 1024 to 4096 tokens,
  // 16/16 heads of 64: 217 -> 194); long units do not notice. It moves shares'
  // borders only.
  static constexpr int kEdge = D <= 128 ? 2 : 10;
  static constexpr int kSmem = NQ * kQBytes + (NK + NV) * kTile + kBarBytes + kRowBytes;
  static_assert(3 * FN + D <= 512, "TMEM columns");
  static_assert(kSmem <= 232448, "shared memory");
};

// The cut at the start of a CTA's share, for tree_join_kernel: the unit that
// began in the share before and goes on in this one (rows 0: none), with its
// pieces up to the one of CTA `last`.
struct __align__(16) Cut {
  int q0, kvh, row0, rows;
  int last, step, pad[2];  // step: from one of its CTAs to the next
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
  Cut* cut;             // [grid]
  int num_seqs, Hq, Hkv, G, block_size, block_shift, max_blocks, num_blocks;
  int mask_words, window;
  long long T, q_stride, o_stride;
  float scale_log2;
  unsigned int* err;
};

__device__ __forceinline__ uint32_t sw_off(int row, int chunk) {
  return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4));
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(sz)
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// (volatile: issued where it stands, ahead of the tile's work)
__device__ __forceinline__ uint32_t ld_word(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
// One sequence's part of the work.
struct Seq {
  int q0, q_len, seq_len, nodes, prefix, k_first, k_lo, n_tiles, n_rt;
  int total;  // tiles of all its units with their edges (the host bounds it)
};
template <int FN, int kEdge>
__device__ __forceinline__ Seq load_seq(const Params& p, int s) {
  // Both come from the device unseen by the host: nodes beyond q's rows and keys
  // beyond the block table do not exist, whatever the numbers say. (The host's
  // bound of `total` rests on that too.)
  Seq r;
  r.q0 = max(0, p.cu_q[s]);
  r.q_len = (int)max(0ll, min((long long)p.cu_q[s + 1], p.T) - r.q0);
  r.seq_len = (int)max(0ll, min((long long)p.seq_lens[s], (long long)p.max_blocks * p.block_size));
  r.nodes = min(r.q_len, r.seq_len);
  r.prefix = r.seq_len - r.nodes;
  // The first key that some node sees: a root sits at position `prefix`.
  r.k_first = p.window > 0 ? max(0, r.prefix - p.window + 1) : 0;
  r.k_lo = r.k_first / FN * FN;
  r.n_tiles = max(1, (r.seq_len - r.k_lo + FN - 1) / FN);
  r.n_rt = (r.q_len * p.G + FM - 1) / FM;
  r.total = (r.n_tiles + kEdge) * r.n_rt * p.Hkv;
  return r;
}

// Lane l's sequence, to the whole warp.
__device__ __forceinline__ Seq share_seq(const Seq& q, int l) {
  Seq r;
  r.q0 = __shfl_sync(0xffffffffu, q.q0, l);
  r.q_len = __shfl_sync(0xffffffffu, q.q_len, l);
  r.seq_len = __shfl_sync(0xffffffffu, q.seq_len, l);
  r.nodes = __shfl_sync(0xffffffffu, q.nodes, l);
  r.prefix = __shfl_sync(0xffffffffu, q.prefix, l);
  r.k_first = __shfl_sync(0xffffffffu, q.k_first, l);
  r.k_lo = __shfl_sync(0xffffffffu, q.k_lo, l);
  r.n_tiles = __shfl_sync(0xffffffffu, q.n_tiles, l);
  r.n_rt = __shfl_sync(0xffffffffu, q.n_rt, l);
  r.total = __shfl_sync(0xffffffffu, q.total, l);
  return r;
}

// The units of a CTA's share, in order: unit = key head * n_rt + row tile,
// key tiles [j0, j1) of it. Of `team` row tiles that are taken together, this
// is the sub-th.
template <int FN, int kEdge>
struct Walk {
  int s, unit, j0, j1, kvh, row0;
  int off, left;
  int team, sub;
  Seq q;
  __device__ __forceinline__ void set(const Seq& x) {
    q = x;
    q.n_rt /= team;
    q.total /= team;
  }
  __device__ __forceinline__ bool next(const Params& p) {
    while (left > 0) {
      while (off >= q.total) {
        if (++s >= p.num_seqs) return false;
        set(load_seq<FN, kEdge>(p, s));
        off = 0;
      }
      const int len = q.n_tiles + kEdge;
      unit = off / len;
      j0 = off - unit * len;
      const int n = min(len - j0, left);
      j1 = min(j0 + n, q.n_tiles);
      off += n;
      left -= n;
      if (j0 >= q.n_tiles) continue;  // the share began at a unit's edge
      kvh = unit / q.n_rt;
      row0 = ((unit - kvh * q.n_rt) * team + sub) * FM;
      return true;
    }
    return false;
  }
};

// A unit as warp 0 publishes it. j0 == j1: no more units.
struct __align__(16) Unit {
  int seq, kvh, j0, j1;
  int q0, row0, rows, whole;  // first token; first row; rows from it on; not cut
  int nodes, prefix, seq_len, k_lo;
  int k_first, pad[3];
  template <int FN>
  __device__ __forceinline__ bool dirty(int j) const {
    // May tile j have rows of V that no node sees? (A node's own slot is one
    // where no mask row has its bit.)
    const int kbase = k_lo + j * FN;
    return kbase + FN > prefix || kbase < k_first;
  }
};

// 32 bits of a node's mask row from node `o` on (o may be negative); bits of
// nodes outside [0, nodes) are 0.
struct MaskRow {
  const uint32_t* row;
  int words, nodes;
  uint32_t w0, w1;  // the first two words (64 nodes), fetched ahead
  __device__ __forceinline__ uint32_t word(int i) const {
    if (i < 0 || i >= words || 32 * i >= nodes) return 0u;
    const int n = nodes - 32 * i;
    const uint32_t w = i == 0 ? w0 : i == 1 ? w1 : __ldg(row + i);
    return n >= 32 ? w : w & ((1u << n) - 1u);
  }
  __device__ __forceinline__ uint32_t bits(int o) const {
    if (o <= -32 || o >= nodes) return 0u;
    const int i = o >> 5;
    return __funnelshift_r(word(i), word(i + 1), o & 31);
  }
};
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
  constexpr int D = C::D, FN = C::FN, kDC = C::kDC, NK = C::NK, NV = C::NV, NQ = C::NQ;
  // The 128-byte swizzle wants 1024-byte aligned tiles: all shared memory is
  // dynamic, and there is no room for a margin.
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + NQ * C::kQBytes;
  uint8_t* sV = sK + NK * C::kTile;
  uint8_t* sEnd = sV + NV * C::kTile;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(sEnd);               // [NK]
  uint64_t* k_empty = k_full + NK;                                    // [NK]
  uint64_t* v_full = k_empty + NK;                                    // [NV]
  uint64_t* v_empty = v_full + NV;                                    // [NV]
  uint64_t* q_full = v_empty + NV;                                    // [2]
  uint64_t* q_empty = q_full + 2;                                     // [2]
  // A tile's S and P are announced by barrier n % 4: a group's tiles n and
  // n + 2 may both be on their way, n + 4 only when all have seen n.
  uint64_t* s_full = q_empty + 2;                                     // [4]
  uint64_t* p_full = s_full + 4;                                      // [4]
  uint64_t* s_free = p_full + 4;                                      // [3], by buffer
  uint64_t* post = s_free + 3;                                        // [2][4]
  uint64_t* pair = post + 8;                                          // [4]
  uint64_t* o_full = pair + 4;
  uint64_t* o_free = o_full + 1;
  uint64_t* done = o_free + 1;
  uint64_t* u_full = done + 1;                                        // [kUnits]
  uint64_t* u_empty = u_full + kUnits;                                // [kUnits]
  uint64_t* v_dirty = u_empty + kUnits;
  uint64_t* v_clean = v_dirty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_clean + 1);
  static_assert((2 * (NK + NV) + 4 + 11 + 12 + 3 + 2 * kUnits + 2) * 8 + 8 +
                    kUnits * (int)sizeof(Unit) <= kBarBytes, "barriers and units");
  Unit* units_sh = reinterpret_cast<Unit*>(sEnd + kBarBytes) - kUnits;
  float* sh_ref = reinterpret_cast<float*>(sEnd + kBarBytes);  // [FM]
  float* sh_sum = sh_ref + FM;                                                // [2][FM]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 3; ++i) mbar_init(&s_free[i], 1);
    for (int i = 0; i < 8; ++i) mbar_init(&post[i], 1);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pair[i], 2);
    }
    mbar_init(v_dirty, 1);
    mbar_init(v_clean, 1);
    mbar_init(o_full, 1);
    mbar_init(o_free, kSoftmaxWarps);
    mbar_init(done, 2);
    for (int i = 0; i < kUnits; ++i) {
      mbar_init(&u_full[i], 1);
      mbar_init(&u_empty[i], kSoftmaxWarps + 4);  // and warps 1, 10, 11, 12
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmk);
    tma_prefetch_desc(&tmv);
  }
  if (warp == 11) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tS = tmem_base, tO = tS + 3 * FN;
  // Unit u for a reader (a warp, or one thread with `alone`).
  auto take = [&](int u, Unit& x, bool alone) -> bool {
    const int e = u % kUnits;
    const bool ok = mbar_wait(&u_full[e], (uint32_t)((u / kUnits) & 1), p.err);
    x = units_sh[e];
    if (!alone) __syncwarp();
    if (alone || lane == 0) mbar_arrive(&u_empty[e]);
    return alone ? ok : __all_sync(0xffffffffu, ok);
  };

  if (warp == 0 || warp == 1) {
    // ------------------------------------------------- producers (K: 0, V: 1)
    const bool is_v = warp == 1;
    const CUtensorMap* tm = is_v ? &tmv : &tmk;
    uint64_t* full = is_v ? v_full : k_full;
    uint64_t* empty = is_v ? v_empty : k_empty;
    uint8_t* ring = is_v ? sV : sK;
    const int slots = is_v ? NV : NK;
    const int BS = p.block_size;
    const int nb = BS >= FN ? 1 : FN / BS;
    const int rows_box = BS >= FN ? FN : BS;
    const int bi = lane % nb, h = lane / nb;
    // The share (warp 0): a scan over the sequences, 32 at a time, for the
    // total and then for the sequence in which this CTA's first tile lies.
    Walk<FN, C::kEdge> walk;
    int share = 0;
    if (!is_v) {
      long long total = 0, sums = 0;
      uint32_t by = (2u << kMaxTeam) - 1u;  // bit d: d divides every number of row tiles
      Seq mine;
      for (int b = 0; b < p.num_seqs; b += 32) {
        long long c = 0;
        if (b + lane < p.num_seqs) {
          const Seq q = load_seq<FN, C::kEdge>(p, b + lane);
          c = q.total;
#pragma unroll
          for (int d = 2; d <= kMaxTeam; ++d)
            if (q.n_rt % d) by &= ~(1u << d);
          if (b == 0) mine = q;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long up = __shfl_up_sync(0xffffffffu, c, o);
          if (lane >= o) c += up;
        }
        if (b == 0) sums = c;
        total += __shfl_sync(0xffffffffu, c, 31);
      }
      const int team = 31 - __clz(__reduce_and_sync(0xffffffffu, by));
      walk.team = team;
      walk.sub = (int)blockIdx.x % team;
      // (64-bit divisions take microseconds off a short call.)
      if (team > 1) total /= team;
      const int teams = (int)gridDim.x / team, me = (int)blockIdx.x / team;
      const long long per =
          max((long long)kMinShare, total < (1ll << 30)
                                        ? (long long)(((uint32_t)total + teams - 1) / (uint32_t)teams)
                                        : (total + teams - 1) / teams);
      const long long t0 = per * me, n = me < teams ? min(per, total - t0) : 0;
      share = (int)per;
      walk.left = (int)max(0ll, n);
      walk.s = walk.off = 0;
      long long seen = 0;
      bool found = n <= 0;
      for (int b = 0; b < p.num_seqs && !found; b += 32) {
        long long c = sums;  // sums up to and with this lane's sequence
        if (b > 0) {
          c = 0;
          if (b + lane < p.num_seqs) {
            mine = load_seq<FN, C::kEdge>(p, b + lane);
            c = mine.total;
          }
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, c, o);
            if (lane >= o) c += up;
          }
        }
        const long long before = __shfl_up_sync(0xffffffffu, c, 1);
        const uint32_t hit = __ballot_sync(0xffffffffu, seen + c > t0 * team);
        if (hit) {
          const int l = __ffs(hit) - 1;
          walk.s = b + l;
          const long long base = seen + __shfl_sync(0xffffffffu, lane > 0 ? before : 0, l);
          walk.off = (int)(t0 - (team > 1 ? base / team : base));
          walk.set(share_seq(mine, l));
          found = true;
        }
        seen += __shfl_sync(0xffffffffu, c, 31);
      }
    } else {
      walk.left = 0;
    }
    int published = 0;
    auto publish = [&](Unit& x) -> bool {  // the next unit, to the others and to x
      const int e = published % kUnits;
      int ok = 1;
      if (lane == 0)
        ok = mbar_wait(&u_empty[e], (uint32_t)(((published / kUnits) & 1) ^ 1), p.err) ? 1 : 0;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      const bool more = walk.next(p);
      x.seq = walk.s;
      x.kvh = walk.kvh;
      x.j0 = more ? walk.j0 : 0;
      x.j1 = more ? walk.j1 : 0;
      x.q0 = walk.q.q0;
      x.row0 = walk.row0;
      x.rows = walk.q.q_len * p.G - walk.row0;
      x.whole = walk.j0 == 0 && walk.j1 == walk.q.n_tiles;
      x.nodes = walk.q.nodes;
      x.prefix = walk.q.prefix;
      x.seq_len = walk.q.seq_len;
      x.k_lo = walk.q.k_lo;
      x.k_first = walk.q.k_first;
      if (ok && lane == 0) {
        units_sh[e] = x;
        mbar_arrive(&u_full[e]);
        if (published == 0) {
          // Tiles of the unit from its first on; an earlier edge than this
          // one joins a unit that began more than a share before.
          const bool mine = more && x.j0 > 0 && x.j0 <= share;
          const int last =
              (int)blockIdx.x + (walk.q.n_tiles - x.j0 - 1) / max(share, 1) * walk.team;
          p.cut[blockIdx.x] = Cut{x.q0, x.kvh,     x.row0, mine ? min(FM, x.rows) : 0,
                                  last, walk.team, {0, 0}};
        }
      }
      ++published;
      return ok != 0;
    };
    int taken = 0;
    auto fetch = [&](Unit& x) -> bool { return is_v ? take(taken++, x, false) : publish(x); };
    struct Box {
      int blk, y;
    };
    // Tile j of a unit: this lane's cache block and row.
    auto box_of = [&](const Unit& x, int j) {
      const int kbase = x.k_lo + j * FN;
      const int last = min(max(0, (x.seq_len - 1) >> p.block_shift), p.max_blocks - 1);
      const int b = min((kbase >> p.block_shift) + bi, last);
      const int id = __ldg(p.block_table + (long long)x.seq * p.max_blocks + b);
      Box r;
      r.blk = in_bounds(id >= 0 && id < p.num_blocks, p.err) ? id : 0;
      r.y = x.kvh * BS + (BS > FN ? (kbase & (BS - 1)) : 0);
      return r;
    };
    Unit unit, next;
    bool ok = fetch(unit);
    Box cur{0, 0};
    if (ok && unit.j0 < unit.j1) cur = box_of(unit, unit.j0);
    int st = 0;
    uint32_t round = 0;  // parity of the ring's round
    while (ok && unit.j0 < unit.j1) {
      ok = fetch(next);
      for (int j = unit.j0; j < unit.j1 && ok; ++j) {
        // Ids one tile ahead of their use.
        Box nxt = cur;
        if (j + 1 < unit.j1) nxt = box_of(unit, j + 1);
        else if (next.j0 < next.j1) nxt = box_of(next, next.j0);
        int go = 1;
        if (lane == 0) {
          go = mbar_wait(&empty[st], round ^ 1u, p.err) ? 1 : 0;
          if (go) mbar_arrive_expect_tx(&full[st], (uint32_t)C::kTile);
        }
        ok = __shfl_sync(0xffffffffu, go, 0);
        if (ok && h < kDC)
          tma_load_3d(ring + st * C::kTile + h * C::kChunk + bi * rows_box * 128, tm, &full[st],
                      h * 64, cur.y, cur.blk);
        if (++st == slots) {
          st = 0;
          round ^= 1u;
        }
        cur = nxt;
      }
      unit = next;
    }
  } else if (warp == 10) {
    // -------------------------------------------------------------- S issuer
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_f16(FM, FN, true);
      const uint64_t dq0 = umma_desc_sw128(smem_u32(sQ)), dk0 = umma_desc_sw128(smem_u32(sK));
      Unit x;
      bool ok = true;
      int n = 0, st = 0;
      uint32_t round = 0;
      for (int u = 0; ok && take(u, x, true) && x.j0 < x.j1; ++u) {
        const int qb = u % NQ;
        ok = mbar_wait(&q_full[qb], (uint32_t)((u / NQ) & 1), p.err);
        for (int j = x.j0; j < x.j1 && ok; ++j, ++n) {
          const int sb = n % 3;
          // K is there, and P V of tile n - 3 done with the buffer.
          ok = mbar_wait(&k_full[st], round, p.err) &&
               mbar_wait(&s_free[sb], (uint32_t)(((n / 3) & 1) ^ 1), p.err);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dq = dq0 + (uint64_t)(qb * (C::kQBytes >> 4));
          const uint64_t dk = dk0 + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
          for (int kb = 0; kb < kDC; ++kb)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16(tS + sb * FN, dq + (uint64_t)(kb * (C::kQChunk >> 4) + 2 * k),
                       dk + (uint64_t)(kb * (C::kChunk >> 4) + 2 * k), idesc,
                       (kb > 0 || k > 0) ? 1u : 0u);
          umma_commit(&s_full[n & 3]);
          umma_commit(&k_empty[st]);
          if (++st == NK) {
            st = 0;
            round ^= 1u;
          }
        }
        umma_commit(&q_empty[qb]);
      }
      // Every MMA done before the TMEM goes.
      umma_commit(done);
      mbar_wait(done, 0, p.err);
    }
    __syncwarp();
  } else if (warp == 11) {
    // ------------------------------------------------------------ P V issuer
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc_f16(FM, D, true) | (1u << 16);  // B MN-major
      const uint64_t dv0 = umma_desc_sw128_mn(smem_u32(sV), C::kChunk, 1024u);
      Unit x;
      bool ok = true;
      int n = 0, st = 0, cleaned = 0;  // V tiles given to warp 12 and taken back
      uint32_t round = 0;
      for (int u = 0; ok && take(u, x, true) && x.j0 < x.j1; ++u) {
        for (int j = x.j0; j < x.j1 && ok; ++j, ++n) {
          const int pb = n % 3;
          const bool dirty = x.template dirty<FN>(j);
          // V is there, without rows that no node sees; P is; O has been read
          // by the epilogue of the unit before.
          ok = mbar_wait(&v_full[st], round, p.err);
          if (ok && dirty) mbar_arrive(v_dirty);
          ok = ok && mbar_wait(&p_full[n & 3], (uint32_t)((n >> 2) & 1), p.err) &&
               (!dirty || mbar_wait(v_clean, (uint32_t)(cleaned & 1), p.err)) &&
               (j > x.j0 || mbar_wait(o_free, (uint32_t)((u & 1) ^ 1), p.err));
          if (!ok) break;
          if (dirty) ++cleaned;
          tc_fence_after();
          const uint64_t dv = dv0 + (uint64_t)(st * (C::kTile >> 4));
#pragma unroll
          for (int s = 0; s < FN / 16; ++s)
            umma_f16_ts(tO, tS + pb * FN + s * 8, dv + (uint64_t)(s * (16 * 128 >> 4)), idesc,
                        (j > x.j0 || s > 0) ? 1u : 0u);
          umma_commit(&s_free[pb]);
          umma_commit(&v_empty[st]);
          if (++st == NV) {
            st = 0;
            round ^= 1u;
          }
        }
        umma_commit(o_full);
      }
      umma_commit(done);
      mbar_wait(done, 0, p.err);
    }
    __syncwarp();
  } else if (warp == 12) {
    // ------------------------------------------------- Q loader, V cleaner
    int n = 0, got = 0;
    // Q rows of unit u into its buffer: eight lanes a 128-byte piece of a row,
    // four rows at a time. Spare rows of a softmax warp that has valid ones
    // are zero, so that their scores are numbers.
    auto load_q = [&](int u, const Unit& x) -> bool {
      const int qb = u % NQ;
      const bool free = mbar_wait(&q_empty[qb], (uint32_t)(((u / NQ) & 1) ^ 1), p.err);
      if (!__all_sync(0xffffffffu, free)) return false;
      const int rows = min(FM, x.rows), fill = (rows + 31) / 32 * 32, sub = lane & 7;
      const uint32_t dst = smem_u32(sQ + qb * C::kQBytes);
      int r = lane >> 3;
      int t = (x.row0 + r) / p.G, hd = x.row0 + r - t * p.G;
      for (; r < fill; r += 4) {
        const bool valid = r < rows;
        const __nv_bfloat16* src =
            valid ? p.q + (long long)(x.q0 + t) * p.q_stride + (long long)(x.kvh * p.G + hd) * D + sub * 8
                  : p.q;
#pragma unroll
        for (int c = 0; c < kDC; ++c)
          cp_async_16(dst + c * C::kQChunk + sw_off(r, sub), src + (valid ? c * 64 : 0), valid);
        for (hd += 4; hd >= p.G; hd -= p.G) ++t;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[qb]);
      return true;
    };
    Unit x, next;
    bool ok = take(0, x, false);
    if (ok && x.j0 < x.j1) ok = load_q(0, x);
    for (int u = 0; ok && x.j0 < x.j1; ++u) {
      ok = take(u + 1, next, false);
      const bool more = next.j0 < next.j1;
      if (ok && more && NQ > 1) ok = load_q(u + 1, next);
      for (int j = x.j0; j < x.j1 && ok; ++j, ++n) {
        if (!x.template dirty<FN>(j)) continue;
        const int kbase = x.k_lo + j * FN;
        // The tile's tree slots that some row of this unit sees; none from
        // the end on. (Read before the wait for V.)
        uint32_t seen[FN / 32];
#pragma unroll
        for (int w = 0; w < FN / 32; ++w) seen[w] = 0u;
        if (kbase + FN > x.prefix) {
          const int last = (x.row0 + min(FM, x.rows) - 1) / p.G;
          for (int t = x.row0 / p.G + lane; t <= last; t += 32) {
            MaskRow m{p.mask + (long long)(x.q0 + t) * p.mask_words, p.mask_words, x.nodes, 0u, 0u};
            m.w0 = __ldg(m.row);
            if (p.mask_words > 1) m.w1 = __ldg(m.row + 1);
#pragma unroll
            for (int w = 0; w < FN / 32; ++w) seen[w] |= m.bits(kbase + 32 * w - x.prefix);
          }
#pragma unroll
          for (int w = 0; w < FN / 32; ++w) seen[w] = __reduce_or_sync(0xffffffffu, seen[w]);
        }
        // (Its V has landed: warp 11 has waited for it.)
        ok = __all_sync(0xffffffffu, mbar_wait(v_dirty, (uint32_t)(got & 1), p.err));
        if (!ok) break;
        uint8_t* sv = sV + (n % NV) * C::kTile;
        constexpr int kU = D / 8;
        auto zero = [&](int from, int to) {  // rows [from, to)
          for (int i = from * kU + lane; i < to * kU; i += 32) {
            const int k = i / kU, c16 = i % kU;
            *reinterpret_cast<uint4*>(sv + (c16 >> 3) * C::kChunk + sw_off(k, c16 & 7)) =
                make_uint4(0, 0, 0, 0);
          }
        };
        zero(0, min(FN, x.k_first - kbase));
        zero(max(0, x.seq_len - kbase), FN);
#pragma unroll
        for (int w = 0; w < FN / 32; ++w) {
          const int k0 = kbase + 32 * w;
          for (uint32_t b = range_bits(x.prefix - k0, x.seq_len - k0) & ~seen[w]; b; b &= b - 1)
            zero(32 * w + __ffs(b) - 1, 32 * w + __ffs(b));
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_clean);
        ++got;
      }
      if (ok && more && NQ == 1) ok = load_q(u + 1, next);
      x = next;
    }
  } else {
    // --------------------------------------------------------------- softmax
    const int q4 = warp & 3;         // the 32 TMEM lanes this warp may touch
    const int grp = (warp - 2) / 4;  // tiles n with n % 2 == grp
    const int row = q4 * 32 + lane;
    constexpr int HD = D / 2;        // O columns of a group in the epilogue
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const float sc = p.scale_log2;
    const uint64_t sc2 = f32x2_pack(sc, sc);
    bool ok = true;
    int n = 0, meets = 0;
    // The two warps of these 32 rows meet (a wait with a limit, like the
    // others: either may have given up).
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(&pair[q4]);
      const bool r = mbar_wait(&pair[q4], (uint32_t)(meets & 1), p.err);
      ++meets;
      return __all_sync(0xffffffffu, r);
    };
    // The reference after tile i, as the warp of these rows in tile i's group
    // left it.
    auto ref_after = [&](int i, float& m) -> bool {
      const bool r = mbar_wait(&post[(i & 1) * 4 + q4], (uint32_t)((i >> 1) & 1), p.err);
      m = sh_ref[row];
      return __all_sync(0xffffffffu, r);
    };
    // Exponent reference of O (log2 units), this group's sum against m_own.
    float m_own = -INFINITY, l = 0.f;
    // A finished unit's row, until its O is read.
    struct Done {
      long long dst;  // element of out, or of part_o for a cut unit
      float m, l;
      int piece;      // row of part_ml, or -1 for a whole unit
      int head;
      bool valid, on;
    } fin{0, 0.f, 0.f, -1, 0, false, false};
    int finished = 0;
    auto epilogue = [&]() -> bool {
      if (fin.on) {
        // The row's sum: the groups'. (Met twice: the places are used again.)
        sh_sum[grp * FM + row] = fin.l;
        if (!meet()) return false;
        fin.l = sh_sum[row] + sh_sum[FM + row];
        if (!meet()) return false;
      }
      if (!__all_sync(0xffffffffu, mbar_wait(o_full, (uint32_t)(finished & 1), p.err)))
        return false;
      ++finished;
      tc_fence_after();
      if (fin.on) {
        const bool whole = fin.piece < 0;
        float f = 1.f;
        if (whole) {
          float den = fin.l;
          if (p.sinks != nullptr)
            den = fin.m == -INFINITY
                      ? 1.f
                      : den + exp2f(p.sinks[fin.head] * 1.4426950408889634f - fin.m);
          f = den > 0.f ? 1.f / den : 0.f;
        } else if (fin.valid && grp == 0) {
          p.part_ml[fin.piece] = make_float2(fin.m, fin.l);
        }
#pragma unroll 1
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t o[16];
          tmem_ld_32x32b_x16(tO + lane_base + grp * HD + c * 16, o);  // warp-collective
          tmem_wait_ld();
          if (!fin.valid) continue;
          if (whole) {
            __nv_bfloat16* dst = p.out + fin.dst + c * 16;
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(__uint_as_float(o[8 * v + 2 * e]) * f,
                                   __uint_as_float(o[8 * v + 2 * e + 1]) * f);
              *reinterpret_cast<uint4*>(dst + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            float* dst = p.part_o + fin.dst + c * 16;
#pragma unroll
            for (int v = 0; v < 4; ++v)
              *reinterpret_cast<uint4*>(dst + v * 4) =
                  make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      return true;
    };
    // This group's sum against the unit's last reference.
    auto close = [&](float m) {
      fin.m = m;
      fin.l = m_own == -INFINITY ? 0.f : l * exp2f(m_own - m);
    };

    Unit x;
    for (int u = 0; ok; ++u) {
      ok = take(u, x, false);
      if (!ok || x.j0 >= x.j1) break;
      const bool valid = row < x.rows;
      const bool warp_on = q4 * 32 < x.rows;
      const int g = x.row0 + (valid ? row : 0), node = g / p.G;
      const int head = x.kvh * p.G + g - node * p.G;
      MaskRow mask{p.mask + (long long)(x.q0 + node) * p.mask_words, p.mask_words, x.nodes, 0u, 0u};
      mask.w0 = ld_word(mask.row);
      if (p.mask_words > 1) mask.w1 = ld_word(mask.row + 1);
      // First key of the prefix this row sees. A node's position is the
      // prefix plus its depth, the number of its ancestors.
      int key_lo = 0;
      if (p.window > 0 && warp_on) {
        int depth = 0;
        for (int i = 0; 32 * i < x.nodes; ++i) depth += __popc(mask.word(i));
        key_lo = x.prefix + max(depth - 1, 0) - p.window + 1;
      }
      for (int j = x.j0; j < x.j1; ++j, ++n) {
        if ((n & 1) == grp) {
          ok = __all_sync(0xffffffffu, mbar_wait(&s_full[n & 3], (uint32_t)((n >> 2) & 1), p.err));
          if (!ok) break;
          tc_fence_after();
          const uint32_t s_row = tS + lane_base + n % 3 * FN;
          const int kb = x.k_lo + j * FN;
          if (warp_on && (__any_sync(0xffffffffu, key_lo > kb) || kb + FN > x.prefix)) {
            // Hidden scores become -inf in TMEM, by a loop of its own: the code
            // that every tile runs stays short.
#pragma unroll 1
            for (int w = 0; w < FN / 32; ++w) {
              const int k0 = kb + 32 * w;
              const uint32_t vis =
                  valid ? range_bits(key_lo - k0, x.prefix - k0) | mask.bits(k0 - x.prefix) : 0u;
              if (__all_sync(0xffffffffu, vis == 0xffffffffu)) continue;
              uint32_t t[32];
              tmem_ld_32x32b_x32(s_row + w * 32, t);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const uint32_t keep = (uint32_t)((int)(vis << (31 - i)) >> 31);
                t[i] = (t[i] & keep) | (0xff800000u & ~keep);
              }
              tmem_st_32x32b_x32(s_row + w * 32, t);
            }
            tmem_wait_st();
          }
          // The row's maximum (log2 units), 32 scores at a time. (Short loops:
          // an SM's instruction cache misses cost more than unrolling gains.)
          float own = -INFINITY;
          if (warp_on) {
            float mxa = -INFINITY, mxb = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < FN / 32; ++c) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(s_row + c * 32, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; i += 2) {
                mxa = max3(mxa, __uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                mxb = max3(mxb, __uint_as_float(r[2 * i + 2]), __uint_as_float(r[2 * i + 3]));
              }
            }
            own = fmaxf(mxa, mxb);
            own = own == -INFINITY ? own : own * sc;
          }
          // The reference from the tile before, to the tile after.
          float m_prev = -INFINITY;
          if (n > 0) {
            ok = ref_after(n - 1, m_prev);
            if (!ok) break;
          }
          if (j == x.j0) {
            if (u > 0) close(m_prev);  // of the unit before
            m_prev = m_own = -INFINITY;
            l = 0.f;
          }
          const bool resc = own > m_prev + 8.f || (m_prev == -INFINITY && own != -INFINITY);
          const float m = resc ? own : m_prev;
          sh_ref[row] = m;
          __syncwarp();
          if (lane == 0) mbar_arrive(&post[grp * 4 + q4]);
          if (warp_on) {
            if (j > x.j0 && __any_sync(0xffffffffu, resc)) {
              // O is final for the tiles before once P V of tile n - 1 is done.
              // (Its buffer's barrier is in that round: S of tile n - 1 went
              // there after the round before, and P V of tile n + 2 comes
              // after this tile's.)
              ok = __all_sync(0xffffffffu, mbar_wait(&s_free[(n - 1) % 3],
                                                     (uint32_t)(((n - 1) / 3) & 1), p.err));
              if (!ok) break;
              tc_fence_after();
              const float alpha = !resc ? 1.f : m_prev == -INFINITY ? 0.f : exp2f(m_prev - m);
#pragma unroll 1
              for (int c = 0; c < D / 16; ++c) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(tO + lane_base + c * 16, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st_32x32b_x16(tO + lane_base + c * 16, o);
              }
            }
            if (m != m_own) {
              l = m_own == -INFINITY ? 0.f : l * exp2f(m_own - m);
              m_own = m;
            }
            // P = 2^(S scale - m) as bf16 pairs, over scores already read.
            const float mu = m == -INFINITY ? 0.f : m;
            const uint64_t nmu2 = f32x2_pack(-mu, -mu);
            uint64_t acc[2] = {f32x2_pack(0.f, 0.f), f32x2_pack(0.f, 0.f)};
#pragma unroll 1
            for (int c = 0; c < FN / 32; ++c) {
              uint32_t r[32], w[16];
              tmem_ld_32x32b_x32(s_row + c * 32, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float ea, eb;
                f32x2_unpack(f32x2_fma(f32x2_pack(__uint_as_float(r[2 * i]),
                                                  __uint_as_float(r[2 * i + 1])), sc2, nmu2),
                             ea, eb);
                ea = fast_exp2(ea);
                eb = fast_exp2(eb);
                acc[i & 1] = f32x2_add(acc[i & 1], f32x2_pack(ea, eb));
                w[i] = pack_bf16x2(ea, eb);
              }
              tmem_st_32x32b_x16(s_row + c * 16, w);
            }
            float a0, a1;
            f32x2_unpack(f32x2_add(acc[0], acc[1]), a0, a1);
            l += a0 + a1;
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[n & 3]);
        } else if (j == x.j0) {
          // The other group's tile: this one did the last of the unit before.
          if (u > 0) close(m_own);
          m_own = -INFINITY;
          l = 0.f;
        }
        if (j == x.j0 && u > 0) {
          ok = epilogue();  // of the unit before
          if (!ok) break;
        }
        if (j == x.j0) {
          fin.head = head;
          fin.valid = valid;
          fin.on = warp_on;
          // A cut unit leaves pieces: 0 for one that began before this share.
          const int piece = ((int)blockIdx.x * 2 + (x.j0 > 0 ? 0 : 1)) * FM + row;
          fin.piece = x.whole ? -1 : piece;
          fin.dst = (x.whole ? (long long)(x.q0 + node) * p.o_stride + (long long)head * D
                             : (long long)piece * D) + grp * HD;
        }
      }
    }
    if (ok && n > 0) {
      float m = m_own;
      if (((n - 1) & 1) != grp) ok = ref_after(n - 1, m);
      if (ok) {
        close(m);
        epilogue();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 11) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Joins the pieces of units that were cut, in share order: a warp a row, one
// block for eight rows of the unit that is cut where share blockIdx.x + 1
// begins.
constexpr int kJoinRows = 8;
template <int D_>
__global__ void __launch_bounds__(kJoinRows * 32) tree_join_kernel(const Params p) {
  constexpr int D = D_;
  constexpr int V = D >= 128 ? D / 128 : 1;  // float4 of a lane
  constexpr int kAhead = 8;                  // pieces in flight
  pdl_wait();
  pdl_trigger();
  const int c1 = blockIdx.x + 1;
  const Cut cut = p.cut[c1];
  const int row = blockIdx.y * kJoinRows + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (row >= cut.rows) return;
  const int g = cut.row0 + row, t = g / p.G, head = cut.kvh * p.G + g - t * p.G;
  const bool on = D >= 128 || lane < D / 4;
  const int n = (cut.last - c1) / cut.step + 2;
  // Piece i: the first is the last of the share before, the others open theirs.
  auto piece = [&](int i) { return ((long long)(c1 + (i - 1) * cut.step) * 2 + (i == 0 ? 1 : 0)) * FM + row; };
  float m = -INFINITY;
  for (int i = lane; i < n; i += 32) m = fmaxf(m, p.part_ml[piece(i)].x);
  float den = 0.f;
  float4 acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float4 o[kAhead][V];
    float2 ml[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (i0 + k < n) {
        const long long pc = piece(i0 + k);
        ml[k] = p.part_ml[pc];
        if (on) {
#pragma unroll
          for (int v = 0; v < V; ++v)
            o[k][v] = *reinterpret_cast<const float4*>(p.part_o + pc * D + (v * 32 + lane) * 4);
        }
      }
    }
    if (i0 == 0) {
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 + k >= n) break;
      const float f = ml[k].x == -INFINITY ? 0.f : exp2f(ml[k].x - m);
      den += ml[k].y * f;
      if (on) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          acc[v].x += o[k][v].x * f;
          acc[v].y += o[k][v].y * f;
          acc[v].z += o[k][v].z * f;
          acc[v].w += o[k][v].w * f;
        }
      }
    }
  }
  if (p.sinks != nullptr)
    den = m == -INFINITY ? 1.f : den + exp2f(p.sinks[head] * 1.4426950408889634f - m);
  const float inv = den > 0.f ? 1.f / den : 0.f;
  if (on) {
    __nv_bfloat16* dst = p.out + (long long)(cut.q0 + t) * p.o_stride + (long long)head * D;
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
  p.cut = reinterpret_cast<Cut*>(p.part_ml + (size_t)grid * 2 * FM);
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
  const long long most = p.T * p.G < FM ? p.T * p.G : FM;
  if (grid > 1)
    // (A row tile has no more rows than the call.)
    launch_pdl(tree_join_kernel<D>, dim3(grid - 1, (int)((most + kJoinRows - 1) / kJoinRows)),
               dim3(kJoinRows * 32), 0, stream, nullptr, p);
}

}  // namespace

size_t tree_attention_workspace_bytes(int head_dim, int num_sm) {
  return (size_t)num_sm * (2 * FM * (head_dim + 2) * 4 + sizeof(Cut));
}

void tree_attention_launch(const TreeAttnArgs& a, cudaStream_t stream) {
  if (a.Hkv < 1 || a.Hq % a.Hkv != 0)
    throw std::runtime_error("tree_attention: Hq must be a multiple of Hkv");
  if (a.block_size < 8 || (a.block_size & (a.block_size - 1)) != 0)
    throw std::runtime_error("tree_attention: block_size must be a power of two >= 8");
  // Tiles of one sequence are counted in 32 bits.
  const double tiles = ((double)a.max_blocks * a.block_size / 64 + 12) * a.Hkv *
                       ((double)a.num_tokens * (a.Hq / a.Hkv) / FM + 1);
  if (tiles > 2e9) throw std::runtime_error("tree_attention: block table too wide for the batch");
  if (a.num_tokens <= 0 || a.num_seqs <= 0) return;
  switch (a.head_dim) {
    case 64: return launch_d<64>(a, stream);
    case 128: return launch_d<128>(a, stream);
    case 256: return launch_d<256>(a, stream);
    default: throw std::runtime_error("tree_attention: head_dim must be 64, 128 or 256");
  }
}

}  // namespace b200
