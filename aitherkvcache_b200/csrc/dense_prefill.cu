// Attention of chunks of new tokens over the dense (fp16 / bf16) paged cache, on the 5th-generation tensor cores.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = 2^(c q_i.k_j - m_i),  j in (p_i - window, p_i],  p_i = len - new + i
//
// Bound by the tensor pipe: 4 D flops per visible (row, key) pair, with one exponential per pair beside it - 128 x 128
// scores take 1024 cycles of the exponential unit and, at D = 128, 1024 cycles of the tensor pipe for both products.
//
// Row tiles.  A CTA works on a row tile - up to 256 rows (token, query head) of one sequence and KV head, two halves of
// 128 rows = TT = 128 / G tokens each - against key tiles of 128 keys.  Per half and key tile:
//   S[128][128] = Q K^T      A = Q in shared memory, B = the keys as they lie in the pages (K-major);
//   O[128][D]  += P V        A = P in tensor memory (over the columns of S), B = the values as they lie in the pages:
//                            [key][dim] rows are the MN-major form of the operand, nothing is transposed.
// K, V and Q come by TMA with the 128-byte swizzle straight out of the paged tensors (a box per run of keys inside a
// block); rows of values that no row may see (behind the sequence's end, before all windows) are zeroed
// in shared memory, since 0 * NaN is NaN.
//
// Twelve warps: 0-3 softmax of half 0 and 4-7 of half 1 (thread = row), 8 and 10 issue the MMAs of one half each, 9 copies the
// keys and Q, 11 the values.  A half's tile goes through in two sub-tiles of 64 keys with a score buffer each, and its MMAs
// are issued in the order  P V of sub-tile u, S of u + 2,  so while a softmax warp works on sub-tile u the scores of u + 1
// are there already: it never waits for the tensor pipe's round trip (P written -> P V and the next S: 1300 cycles and more),
// and the two halves' warps, two per scheduler, fill each other's gaps in the exponential unit.  64-key scores cost the tensor
// pipe 385 cycles instead of 256 (the operands' shared-memory traffic), 2485 per tile pair in all where 2048 would be the least;
// with whole 128-key tiles in one buffer a tile pair took 4850 cycles, 2900 of each half's period waiting for that round trip.
// MMAs complete in order, so "S of u is there" also says that P V of u - 2 is done and the buffer of P u - 2 was free.
// The row's reference moves only when a weight would pass 2^8 times the last reference's (DENSE_TOP in dense_attn.cuh), so O
// is rescaled a few times per row; that waits for P V of u - 1.
//
// Few rows.  Where a row tile has rows for one half only (at most TT new tokens left), the halves take alternate key tiles of
// the same rows, half 0 the piece's first, third ..., half 1 the others, and at the piece's end half 0 adds half 1's O, which
// lies in the same lanes of tensor memory, to its own.  1 to 8 new tokens behind 32 sequences of 4000 (28 / 4 heads of
// 64): 56.7 us against 65.7 with one half idle when this came, 48 now.
//
// Work split.  The (row tile, key tile) pairs of the whole call are laid end to end and cut into equal ranges, one per SM:
// every SM has the same share whatever the lengths.  Row tiles that are cut (at most two per CTA) leave float32 partials in
// the workspace, joined by dense_prefill_merge_kernel in a fixed order; a cut within DP_SNAP tiles of a
// row tile's edge is moved to the edge (a partial costs about as much as two key tiles).
//
// Rounds.  The CTAs' ranges begin anywhere in the keys, so a KV head's keys and values are wanted at all times of its round,
// and what does not fit into L2 comes from HBM again for every row tile: at a power limit that costs clock (131 MB of
// keys and values ran at 1.34 GHz, 24 MB at 1.47).  So the (sequence, KV head) pairs are taken in rounds of about
// DP_ROUND_BYTES of keys and values, each cut into ranges for all SMs.  A round more costs some 10 us (its cuts, and the SMs' wait
// for the first keys), so only the keys of sequences with DP_ROUND_TILES row tiles or more count.  Inside a graph, keys from HBM
// (32 / 8 heads of 128): 2048 tokens behind 60000 take 1.89 ms in rounds and 2.13 without, 1000 behind 60000 0.99 and 1.13, 800
// behind 40000 536 us and 578.  With the keys of all sequences counted, 440 behind 20000 would take 166 us instead of 148, 100
// behind 20000 76 instead of 61, and 32 sequences of 4096 with 4 new tokens (4 KV heads of 64) 52 instead of 45.
//
// Measured: 2048 tokens behind 30000 (32 / 8 heads of 128) 0.98 ms in a sustained run at the power limit (1.45 GHz), 1.06 PFLOP/s,
// 77 % of the measured sustained matrix rate; 0.87 ms, 1.2 PFLOP/s in short bursts, 0.77 ms with zero data; 2900 cycles per tile
// pair.  Some SMs take 14 % longer than the others for the same share and set the end.  Twelve prompts of 1 to 2000 tokens 174 us
// with keys from HBM, 0.67 PFLOP/s, and 153 us with keys in L2 (10 pieces per CTA, each with 1700 cycles of its own for the last
// P V and the first scores, and 2600 for the epilogue); the 1 to 8 new tokens above 48 us, 3 TB/s.
//
// Every wait is bounded (umma.cuh): a wait that gives up sets g_dense_prefill_status and a flag that ends all loops.
#include "dense_attn.cuh"
#include "umma.cuh"
#include <cuda.h>
#include <math.h>
#include <math_constants.h>

namespace akv {
namespace {

__device__ int g_dense_prefill_status;           // 1: a bounded wait gave up, 2: tensor-memory columns were kept
__device__ int g_dense_prefill_withhold = -1;    // test hook: CTA 0 issues neither the score MMAs nor the commit of this tile

constexpr int DP_KT = 128;                       // keys per tile
constexpr int DP_MAX_SEQS = 384;                 // sequences of one launch
constexpr int DP_MAX_ROUNDS = 4;
constexpr int64_t DP_ROUND_BYTES = 68 << 20;     // keys and values of a round
constexpr int DP_ROUND_TILES = 8;                // row tiles that make keys worth keeping in L2
// a cut this near to a row tile's edge is moved there, in key tiles (0 and 6: 158 us for the prompts above with keys in L2, 4: 156, 2: 153)
constexpr int DP_SNAP = 2;
constexpr int DP_PIECE = 2;                      // what a row tile costs besides its key tiles, in key tiles

struct DpMaps { CUtensorMap q, k, v; };

template <int D> struct DpL {
  static constexpr int WARPS = 12, THREADS = 384, MMA_WARP = 8, K_WARP = 9, MMA_WARP2 = 10, V_WARP = 11;
  static constexpr int HALVES = D / 64;                    // 64-element columns of an operand
  static constexpr int TILE = 128 * D * 2;                 // bytes of 128 rows
  static constexpr int NP = D == 128 ? 2 : 4;              // ring slots of K tiles, and of V tiles
  static constexpr int Q = 0, KV = 2 * TILE, BAR = KV + 2 * NP * TILE;      // K slot, V slot, K slot ...
  static constexpr int PRE = BAR + 512;                    // int64 [DP_MAX_SEQS + 1]: units before a sequence ...
  static constexpr int PREK = PRE + (DP_MAX_SEQS + 1) * 8; // ... and keys before it that count towards the rounds
  static constexpr int SROW = 80;                          // staging of results: 64 bytes of a row, padded to other banks
  static constexpr int SEQ = PRE + (DP_MAX_SEQS + 1) * 16;       // int [DP_MAX_SEQS][3]: DpSeq of every sequence
  static constexpr int STAGE = (SEQ + DP_MAX_SEQS * 12 + 15) / 16 * 16;     // [8 warps][32 rows][SROW]
  static constexpr int SMEM = STAGE + 8 * 32 * SROW + 1024;
  static_assert(STAGE % 16 == 0, "staging");
  static constexpr int T_O = 256;                          // tensor memory: S 0, S 1 (128 columns each), O 0, O 1
  static_assert(SMEM + 512 <= 232448, "shared memory");
};
// barriers (bytes behind BAR)
constexpr uint32_t P_PAIR = 0 /* V of tile g and K of tile g + 1 are there */, P_KFIRST = 32, P_KFREE = 64, P_VFREE = 96, P_QFULL = 128, P_QFREE = 144, P_SFULL = 160, P_PFULL = 192, P_PVDONE = 224,
                   P_TAIL = 240, P_DRAIN = 248, P_TMEM = 264, P_FAILED = 268, P_JOIN = 272, P_OFULL = 288;

// What dense_prefill_merge_kernel needs to know about the row tile whose first part CTA c wrote (parts < 2: nothing)
struct DpDesc { int parts, slot0, row0, ntok, kvh, pad[3]; };

__device__ __forceinline__ void dp_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void dp_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void dp_tma4(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z, int w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               :: "r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void dp_tma3(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
               :: "r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// MN-major operand, 128-byte swizzle: a key's 64 dims are one 128-byte row; groups of 8 keys 1024 B apart (stride offset),
// the next 64 dims 16 KB on (leading offset).
__device__ __forceinline__ uint64_t dp_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ bool dp_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
// two floats per register pair: the FMA pipe's packed instructions
__device__ __forceinline__ uint64_t dp_pk(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void dp_upk(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t dp_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t dp_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// max(a, b, c) that keeps a NaN
__device__ __forceinline__ float dp_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// MMAs of kind::f16 with descriptors given as halves: operands that differ in the address field only share the upper
// half, and an unrolled sequence costs one addition per operand (short code matters: the issuing warps share the
// instruction caches with eight softmax warps in long loops).
template <bool ACC>
__device__ __forceinline__ void dp_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}\n"
      :: "r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "n"(ACC ? 1 : 0) : "memory");
}
__device__ __forceinline__ void dp_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}\n"
      :: "r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(acc) : "memory");
}

struct DpSeq { int q0, qlen, total; };           // first query row, new tokens, tokens
struct DpTile { int tok0, ntok, t0, n; };        // first token and tokens of a row tile, its first key tile, key tiles

__device__ __forceinline__ DpSeq dp_seq(const DenseArgs& a, int s) {
  DpSeq r;
  int64_t q0 = load_index(a.starts, a.qs_dtype, s), q1 = load_index(a.starts, a.qs_dtype, s + 1);
  if (q0 < 0) q0 = 0;
  if (q1 > a.n_tokens) q1 = a.n_tokens;
  r.q0 = (int)q0;
  r.qlen = q1 > q0 ? (int)(q1 - q0) : 0;
  r.total = (int)load_ctx(a.seq_lens, a.sl_dtype, s, (int64_t)a.max_blocks_per_seq * a.block_size);
  return r;
}
__device__ __forceinline__ int dp_tiles(const DpSeq& q, int tt2) { return (q.qlen + tt2 - 1) / tt2; }
__device__ __forceinline__ DpTile dp_tile(const DenseArgs& a, const DpSeq& q, int tt2, int i) {
  DpTile t;
  t.tok0 = i * tt2;
  t.ntok = q.qlen - t.tok0 < tt2 ? q.qlen - t.tok0 : tt2;
  const int pos0 = q.total - q.qlen + t.tok0, kend = pos0 + t.ntok;      // kend <= total
  const int klo = a.window > 0 && pos0 + 1 > a.window ? pos0 + 1 - a.window : 0;
  t.t0 = klo / DP_KT;
  t.n = kend > 0 ? (kend + DP_KT - 1) / DP_KT - t.t0 : 0;
  if (t.n < 1) t.n = 1;                          // rows that see nothing: one masked tile, they come out as zeros
  return t;
}

// The call's work, laid end to end: sequences, their KV heads, their row tiles; a row tile counts DP_PIECE + key tiles units.
// A place in that list: row tile (s, kvh, i) of tile t, and the unit inside it.
struct DpPlace { int s, kvh, i, off; DpTile t; };

struct DpWork {                                  // what every role of the CTA knows about the call
  const int64_t* pre;                            // units before a sequence
  const DpSeq* seq;
  int seqs, tt2, n_rounds;
};

__device__ __forceinline__ uint32_t dp_div(int64_t a, int64_t b) {      // quotients below 2^32
  return ((a | b) >> 32) == 0 ? (uint32_t)a / (uint32_t)b : (uint32_t)(a / b);
}

// All lanes of a warp: the place of unit u, 0 <= u < pre[seqs].
__device__ __forceinline__ DpPlace dp_locate(const DenseArgs& a, const DpWork& w, int64_t u, int lane) {
  DpPlace p;
  int lo = 0, hi = w.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (w.pre[mid] <= u) lo = mid; else hi = mid;
  }
  p.s = lo;
  const int64_t in = u - w.pre[lo], per = dp_div(w.pre[lo + 1] - w.pre[lo], a.num_kv_heads);
  p.kvh = (int)dp_div(in, per);
  int64_t rem = in - (int64_t)p.kvh * per;
  const DpSeq q = w.seq[lo];
  const int tiles = dp_tiles(q, w.tt2);
  for (int base = 0;; base += 32) {
    const int i = base + lane, n = i < tiles ? DP_PIECE + dp_tile(a, q, w.tt2, i).n : 0;
    int inc = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, inc > rem);
    if (hit != 0u || base + 32 >= tiles) {
      const int l = hit != 0u ? __ffs(hit) - 1 : 31;
      p.i = base + l;
      p.off = (int)(rem - (__shfl_sync(0xffffffffu, inc, l) - __shfl_sync(0xffffffffu, n, l)));
      p.t = dp_tile(a, q, w.tt2, p.i);
      return p;
    }
    rem -= __shfl_sync(0xffffffffu, inc, 31);
  }
}

// The row tile behind p's (there is one)
__device__ __forceinline__ void dp_advance(const DenseArgs& a, const DpWork& w, DpPlace* p) {
  p->off = 0;
  if (++p->i >= dp_tiles(w.seq[p->s], w.tt2)) {
    p->i = 0;
    if (++p->kvh == a.num_kv_heads) {
      p->kvh = 0;
      do { ++p->s; } while (w.seq[p->s].qlen == 0);
    }
  }
  p->t = dp_tile(a, w.seq[p->s], w.tt2, p->i);
}

// Where the units [lo, hi) are cut before CTA c of the n that share them ...
__device__ __forceinline__ int64_t dp_cut(int64_t lo, int64_t hi, int n, int c) {
  const int64_t units = hi - lo;
  if ((units >> 32) == 0) return lo + (int64_t)((uint32_t)units / (uint32_t)n) * c + (uint32_t)units % (uint32_t)n * (uint32_t)c / (uint32_t)n;
  return lo + units / n * c + units % n * c / n;
}

// ... and, all lanes of a warp: first unit of CTA c (the cut, moved to a row tile's edge where one is
// near, so that an offset inside a row tile is above DP_PIECE), and its place.
__device__ __forceinline__ int64_t dp_begin(const DenseArgs& a, const DpWork& w, int64_t lo, int64_t hi, int n, int c, int lane, DpPlace* place) {
  if (c >= n) return hi;
  int64_t u = dp_cut(lo, hi, n, c);
  DpPlace p = dp_locate(a, w, u, lane);
  const int m = DP_PIECE + p.t.n;
  if (p.off > 0 && p.off <= DP_PIECE + DP_SNAP) {
    u -= p.off;
    p.off = 0;
  } else if (p.off > 0 && m - p.off <= DP_SNAP) {
    u += m - p.off;
    if (u >= hi) return hi;
    dp_advance(a, w, &p);
  }
  *place = p;
  return u;
}

// A round: the units [lo, hi) of consecutive (sequence, KV head) pairs, shared by n CTAs; this CTA's part [u0, u1) of it
// (the end: end_off units inside a row tile, 0 at an edge)
struct DpRound { int64_t lo, hi, u0, u1; int n, end_off; DpPlace place; };

// A role's way through the CTA's part, piece by piece (a piece: consecutive key tiles of one row tile)
struct DpCursor {
  DpPlace at;
  DpSeq q;
  int off, cnt;                 // key tiles at.t.t0 + off .. + cnt - 1
  int64_t left;                 // units behind this piece
  int nq;                       // halves that work
  bool twin;                    // tokens for one half only, and key tiles for two: half h takes tiles off + h, off + h + 2 ... for the same rows
  int round;
  bool first;                   // the first piece of this CTA's part of the round

  __device__ __forceinline__ void settle(const DpWork& w, int64_t avail) {      // avail > DP_PIECE where at.off == 0
    q = w.seq[at.s];
    const int m = DP_PIECE + at.t.n, end = avail < m - at.off ? at.off + (int)avail : m;
    off = at.off > DP_PIECE ? at.off - DP_PIECE : 0;
    cnt = end - DP_PIECE - off;
    left = avail - (end - at.off);
    const bool one = 2 * at.t.ntok <= w.tt2;
    twin = one && cnt > 1;
    nq = one && !twin ? 1 : 2;
  }
  // key tiles of half h (h < nq), and whether its first one is the piece's first
  __device__ __forceinline__ int tiles(int h) const { return twin ? (cnt + 1 - h) >> 1 : cnt; }
  __device__ __forceinline__ bool leads(int h) const { return h < nq && !(twin && h == 1); }
  // the part of the next round that has one; false: there is none
  __device__ __forceinline__ bool next_round(const DpWork& w, const DpRound* rounds) {
    do {
      if (++round >= w.n_rounds) return false;
    } while (rounds[round].u1 <= rounds[round].u0);
    at = rounds[round].place;
    first = true;
    settle(w, rounds[round].u1 - rounds[round].u0);
    return true;
  }
  __device__ __forceinline__ bool next(const DenseArgs& a, const DpWork& w, const DpRound* rounds) {
    if (left <= 0) return next_round(w, rounds);
    first = false;
    dp_advance(a, w, &at);
    settle(w, left);
    return true;
  }
};

template <bool BF, int D>
__global__ void __launch_bounds__(384, 1)
dense_prefill_kernel(const __grid_constant__ DenseArgs a, const __grid_constant__ DpMaps maps, int seqs, int G, int TT, int box,
                     int max_rounds, DpDesc* desc, float* part_ml, float* part_acc) {
  using L = DpL<D>;
  constexpr int NP = L::NP;
  extern __shared__ uint8_t dp_smem[];
  const uint32_t raw_s = smem_u32(dp_smem);
  const uint32_t base_s = (raw_s + 1023u) & ~1023u;
  uint8_t* base = dp_smem + (base_s - raw_s);
  const uint32_t bar_s = base_s + L::BAR, failed_s = bar_s + P_FAILED;
  int64_t* pre = reinterpret_cast<int64_t*>(base + L::PRE);
  int64_t* prek = reinterpret_cast<int64_t*>(base + L::PREK);
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int tt2 = 2 * TT;
  __shared__ DpRound s_round[DP_MAX_ROUNDS];
  __shared__ int s_tiles[L::WARPS], s_copied[2];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (tid == 0) {
    for (int i = 0; i < NP; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" :: "r"(bar_s + P_PAIR + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" :: "r"(bar_s + P_KFREE + 8 * i));      // both halves
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" :: "r"(bar_s + P_VFREE + 8 * i));
    }
    for (int i = 0; i < 2; ++i) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_QFULL + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_QFREE + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_PVDONE + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_OFULL + 8 * i));
    }
    for (int i = 0; i < 4; ++i) {           // half, sub-tile
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_SFULL + 8 * i));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" :: "r"(bar_s + P_PFULL + 8 * i));
    }
    for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 4;" :: "r"(bar_s + P_JOIN + 8 * i));
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_TAIL));
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_KFIRST));
    for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" :: "r"(bar_s + P_DRAIN + 8 * i));
    asm volatile("st.shared.u32 [%0], %1;" :: "r"(failed_s), "r"(0u) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  if (warp == L::MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" :: "r"(bar_s + P_TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");      // what the kernel before this one wrote is read from here on
  // ---- the sequences, units per sequence (a warp per sequence, lanes over its row tiles), then prefix sums ----
  DpSeq* seq = reinterpret_cast<DpSeq*>(base + L::SEQ);
  for (int s = tid; s < seqs; s += L::THREADS) seq[s] = dp_seq(a, s);
  __syncthreads();
  int my_tiles = 0;
  for (int s = warp; s < seqs; s += L::WARPS) {
    const DpSeq q = seq[s];
    const int tiles = dp_tiles(q, tt2);
    int64_t n = 0;
    for (int i = lane; i < tiles; i += 32) n += DP_PIECE + dp_tile(a, q, tt2, i).n;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) n += __shfl_xor_sync(0xffffffffu, n, d);
    if (lane == 0) {
      pre[s + 1] = n * a.num_kv_heads;
      prek[s + 1] = tiles < DP_ROUND_TILES ? 0 : (a.window > 0 && a.window < q.total - q.qlen ? a.window + q.qlen : q.total);
    }
    my_tiles += tiles;
  }
  if (lane == 0) s_tiles[warp] = my_tiles;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp < 2) {
    int64_t* p = warp == 0 ? pre : prek;
    int64_t run = 0;
    for (int b = 0; b < seqs; b += 32) {
      int64_t x = b + lane < seqs ? p[b + lane + 1] : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      x += run;
      if (b + lane < seqs) p[b + lane + 1] = x;
      run = __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) p[0] = 0;
  }
  __syncthreads();
  const int64_t units = pre[seqs];
  // rounds: as many as it takes for a round's keys and values to stay in L2 while the CTAs walk over them again and again
  const int64_t kv_bytes = prek[seqs] * a.num_kv_heads * (4 * D);
  int n_rounds = (int)((kv_bytes + DP_ROUND_BYTES - 1) / DP_ROUND_BYTES < max_rounds ? (kv_bytes + DP_ROUND_BYTES - 1) / DP_ROUND_BYTES : max_rounds);
  if (n_rounds < 1) n_rounds = 1;
  if (units == 0) n_rounds = 0;
  const DpWork w{pre, seq, seqs, tt2, n_rounds};
  if (warp < 2 * n_rounds) {              // two warps per round: where this CTA's part begins and where it ends
    // first unit of round r: that of the first (sequence, KV head) pair with r / n_rounds of all keys before it
    auto edge = [&](int r) -> int64_t {
      if (r <= 0) return 0;
      if (r >= n_rounds) return units;
      const int64_t want = prek[seqs] * a.num_kv_heads * r / n_rounds;
      int lo = 0, hi = seqs;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prek[mid] * a.num_kv_heads <= want) lo = mid; else hi = mid;
      }
      const int64_t keys = prek[lo + 1] - prek[lo], in = want - prek[lo] * a.num_kv_heads;
      int64_t h = keys > 0 ? (in + keys - 1) / keys : a.num_kv_heads;
      if (h > a.num_kv_heads) h = a.num_kv_heads;
      return pre[lo] + h * ((pre[lo + 1] - pre[lo]) / a.num_kv_heads);
    };
    const int round = warp >> 1;
    const int64_t lo = edge(round), hi = edge(round + 1);
    // CTAs that share it: all, but not more than there are row tiles or groups of six units: a part costs about two (5 tokens
    // behind 20000, 8 / 1 heads of 128: 25 us; with eight units 28), and four or fewer could be moved away whole
    int64_t want = (hi - lo) / 6;
    if (n_rounds == 1) {
      int64_t rts = 0;
      for (int x = 0; x < L::WARPS; ++x) rts += s_tiles[x];
      rts *= a.num_kv_heads;
      if (want < rts) want = rts;
    } else if (want < 1) {
      want = 1;
    }
    const int n = want < (int64_t)gridDim.x ? (int)want : (int)gridDim.x;
    DpPlace place{0, 0, 0, 0, {0, 0, 0, 0}};
    const int64_t u = hi > lo ? dp_begin(a, w, lo, hi, n, (int)blockIdx.x + (warp & 1), lane, &place) : hi;
    if (lane == 0) {
      DpRound& r = s_round[round];
      if (warp & 1) {
        r.u1 = u;
        r.end_off = place.off;
      } else {
        r.lo = lo; r.hi = hi; r.n = n;
        r.u0 = u;
        r.place = place;
      }
    }
  }
  __syncthreads();
  const uint32_t tmem = lds_u32(bar_s + P_TMEM);
  DpCursor cur;
  cur.round = -1;
  cur.left = 0;
  const bool work = cur.next_round(w, s_round);

  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if (lds_u32(failed_s) != 0u) return false;
    if (mbar_wait(bar, parity)) return true;
    g_dense_prefill_status = 1;
    asm volatile("st.shared.u32 [%0], %1;" :: "r"(failed_s), "r"(1u) : "memory");
    return false;
  };
  auto wait_warp = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, wait(bar, parity)); };

  if (work && (warp == L::MMA_WARP || warp == L::MMA_WARP2)) {
    // ================= MMA warps, one per half: all lanes follow the loop, one elected lane issues =================
    // (uniform control flow, so that an MMA's operands are computed in uniform registers: with one lane in a divergent
    // loop the issue of a sub-tile's 12 MMAs took 1200 cycles of the 621 they need; and two warps, so that one's waits
    // are covered by the other's MMAs)
    constexpr uint32_t TYPES = BF ? (1u << 7) | (1u << 10) : 0u;
    constexpr uint32_t IDESC_S = (1u << 4) | TYPES | ((64u >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | TYPES | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
    const int h = warp == L::MMA_WARP ? 0 : 1;
    const int withhold = blockIdx.x == 0 ? g_dense_prefill_withhold : -1;
    // descriptors: upper halves, and lower halves of the half's Q and of the first K and V slots
    const uint32_t k_hi = (uint32_t)(umma_desc(0u) >> 32), v_hi = (uint32_t)(dp_desc_mn(0u) >> 32);
    const uint32_t q_d = (uint32_t)umma_desc(base_s + L::Q + (uint32_t)(h * L::TILE)), k_d = (uint32_t)umma_desc(base_s + L::KV);
    const uint32_t v_d = (uint32_t)dp_desc_mn(base_s + L::KV + L::TILE);
    const uint32_t t_s = tmem + (uint32_t)(h * 128), t_o = tmem + (uint32_t)(L::T_O + h * 128);
    uint32_t q_phase = 0, p_phase = 0;      // parities of the next waits
    // scores of sub-tile u of tile number g of the CTA; last: the piece's last tile
    auto issue_s = [&](int g, int u, bool last) {
      const uint32_t kd = k_d + (uint32_t)(2 * (g % NP)) * (L::TILE >> 4) + (uint32_t)(u * (8192 >> 4));
      dp_mma_ss<false>(t_s + (uint32_t)(u * 64), q_d, kd, k_hi, IDESC_S);
#pragma unroll
      for (int kk = 1; kk < D / 16; ++kk) {
        const uint32_t off = (uint32_t)((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
        dp_mma_ss<true>(t_s + (uint32_t)(u * 64), q_d + off, kd + off, k_hi, IDESC_S);
      }
      umma_commit(bar_s + P_SFULL + 8 * (uint32_t)(2 * h + u));
      if (u == 1 && last) umma_commit(bar_s + P_QFREE + 8 * h);
      if (u == 1) umma_commit(bar_s + P_KFREE + 8 * (uint32_t)(g % NP));
    };
    // O += P V of sub-tile u; first, last: the half's first and last tile of the piece
    auto issue_pv = [&](int g, int u, bool first, bool last) {
      const uint32_t vd = v_d + (uint32_t)(2 * (g % NP)) * (L::TILE >> 4) + (uint32_t)(u * (8192 >> 4));
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        dp_mma_ts(t_o, t_s + (uint32_t)(u * 64 + kk * 8), vd + (uint32_t)(kk * (2048 >> 4)), v_hi, IDESC_O, (u | kk) != 0 || !first ? 1u : 0u);
      umma_commit(bar_s + P_PVDONE + 8 * h);
      if (u == 1 && last) umma_commit(bar_s + P_OFULL + 8 * h);
      if (u == 1) umma_commit(bar_s + P_VFREE + 8 * (uint32_t)(g % NP));
    };
    auto q_there = [&]() -> bool {
      const uint32_t parity = q_phase;
      q_phase ^= 1u;
      return wait_warp(bar_s + P_QFULL + 8 * h, parity);
    };
    auto test_warp = [&](uint32_t bar, uint32_t parity) -> bool {
      uint32_t done;
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}\n"
          : "=r"(done) : "r"(bar), "r"(parity) : "memory");
      return __all_sync(0xffffffffu, done != 0u);
    };
    bool go = wait_warp(bar_s + P_KFIRST, 0u), there = false;
    if (go && cur.leads(h)) {
      go = q_there();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (go && withhold != 0 && dp_elect()) {
        issue_s(0, 0, cur.tiles(h) == 1);
        issue_s(0, 1, cur.tiles(h) == 1);
      }
      __syncwarp();
    } else if (go && lane == 0) {
      dp_arrive(bar_s + P_KFREE);           // not this half's: the tile is free as far as it goes
    }
    __syncwarp();
    // One tile: P V of its sub-tiles, each followed by the scores of the next tile's.  V of this tile and K of the next are
    // tested for before the previous tile's last MMAs are issued, so that nothing is waited for in the regular flow (the
    // tensor pipe's queue lasts some 350 cycles).
    auto pair_there = [&](int g) -> bool {
      return there || wait_warp(bar_s + P_PAIR + 8 * (uint32_t)(g % NP), (uint32_t)((g / NP) & 1));
    };
    auto test_pair = [&](int g) { there = test_warp(bar_s + P_PAIR + 8 * (uint32_t)(g % NP), (uint32_t)((g / NP) & 1)); };
    auto p_there = [&](int u) -> bool {
      if (!wait_warp(bar_s + P_PFULL + 8 * (uint32_t)(2 * h + u), p_phase)) return false;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      return true;
    };
    int g = 0;
    while (go) {
      if (cur.twin) {
        // ---- every other tile is this half's; those between are free as far as it goes ----
        there = false;
        const int end = g + cur.cnt;
        if (h == 1) {                       // its first scores
          if (!pair_there(g) || !q_there()) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (g + 1 != withhold && dp_elect()) {
            issue_s(g + 1, 0, cur.cnt <= 3);
            issue_s(g + 1, 1, cur.cnt <= 3);
          }
          __syncwarp();
          if (lane == 0) dp_arrive(bar_s + P_VFREE + 8 * (uint32_t)(g % NP));
          __syncwarp();
          ++g;
        }
        for (bool first = true; g < end; g += 2, first = false) {
          const bool other = g + 1 < end, next = g + 2 < end;
          if (!pair_there(g)) { go = false; break; }
          if (other && lane == 0) dp_arrive(bar_s + P_KFREE + 8 * (uint32_t)((g + 1) % NP));
          __syncwarp();
          if (!p_there(0)) { go = false; break; }
          if (dp_elect()) issue_pv(g, 0, first, false);
          __syncwarp();
          if (other && !pair_there(g + 1)) { go = false; break; }
          if (next && g + 2 != withhold && dp_elect()) issue_s(g + 2, 0, false);
          __syncwarp();
          if (!p_there(1)) { go = false; break; }
          if (dp_elect()) {
            issue_pv(g, 1, false, !next);
            if (next && g + 2 != withhold) issue_s(g + 2, 1, g + 4 >= end);
          }
          __syncwarp();
          if (other && lane == 0) dp_arrive(bar_s + P_VFREE + 8 * (uint32_t)((g + 1) % NP));
          __syncwarp();
          p_phase ^= 1u;
        }
        if (!go) break;
        g = end;                            // the first tile of the next piece, whose keys are there
        if (!cur.next(a, w, s_round)) break;
        if (cur.leads(h)) {
          if (!q_there()) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          if (g != withhold && dp_elect()) {
            issue_s(g, 0, cur.tiles(h) == 1);
            issue_s(g, 1, cur.tiles(h) == 1);
          }
        } else if (lane == 0) {
          dp_arrive(bar_s + P_KFREE + 8 * (uint32_t)(g % NP));
        }
        __syncwarp();
        continue;
      }
      // ---- tiles of the piece that are followed by another of the same piece: the loop that counts ----
      if (h < cur.nq) {
        for (int j = 0; j + 1 < cur.cnt; ++j, ++g) {
          if (!pair_there(g) || !p_there(0)) { go = false; break; }
          if (dp_elect()) {
            issue_pv(g, 0, j == 0, false);
            if (g + 1 != withhold) issue_s(g + 1, 0, false);
          }
          __syncwarp();
          if (!p_there(1)) { go = false; break; }
          test_pair(g + 1);
          if (dp_elect()) {
            issue_pv(g, 1, false, false);
            if (g + 1 != withhold) issue_s(g + 1, 1, j + 2 == cur.cnt);
          }
          __syncwarp();
          p_phase ^= 1u;
        }
      } else {                              // no rows in this half: the tiles are free as far as it goes
        for (int j = 0; j + 1 < cur.cnt; ++j, ++g) {
          there = false;
          if (!pair_there(g)) { go = false; break; }
          if (lane == 0) {
            dp_arrive(bar_s + P_VFREE + 8 * (uint32_t)(g % NP));
            dp_arrive(bar_s + P_KFREE + 8 * (uint32_t)((g + 1) % NP));
          }
          __syncwarp();
        }
      }
      if (!go) break;
      // ---- the piece's last tile, with the scores of the next piece's first ----
      DpCursor ahead = cur;
      const bool more = ahead.next(a, w, s_round), pv = h < cur.nq, sc = more && ahead.leads(h);
      if (!pair_there(g)) break;
#pragma unroll 1
      for (int u = 0; u < 2 && go; ++u) {
        if (pv) {
          go = p_there(u);
          if (go && dp_elect()) issue_pv(g, u, cur.cnt == 1, true);
          __syncwarp();
        }
        if (go && sc) {
          if (u == 0) {
            go = q_there();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          if (go && g + 1 != withhold && dp_elect()) issue_s(g + 1, u, ahead.tiles(h) == 1);
          __syncwarp();
        }
      }
      if (!go || !more) break;
      there = false;
      if (pv) p_phase ^= 1u;
      if (lane == 0) {
        if (!pv) dp_arrive(bar_s + P_VFREE + 8 * (uint32_t)(g % NP));
        if (!sc) dp_arrive(bar_s + P_KFREE + 8 * (uint32_t)((g + 1) % NP));
      }
      __syncwarp();
      ++g;
      cur = ahead;
    }
  } else if (work && (warp == L::K_WARP || warp == L::V_WARP)) {
    // ================= copies: one warp brings the keys (and Q), one the values =================
    // (two warps and uniform issue: a tile of 16-key blocks is 32 copies of 2 KB, and with a lane per block, which the
    // hardware runs through one by one, their issue alone took 3000 cycles per tile)
    const bool of_k = warp == L::K_WARP;
    const int boxes = DP_KT / box;          // runs of keys inside a block
    const uint32_t box_bytes = (uint32_t)box * 128u;
    uint32_t q_used = 0, q_phase = 0;       // a bit per half: Q was loaded before; parity of its last load's barriers
    int tails = 0, g = 0;                   // tiles copied
    bool go = true;
    // lane p's block and position hold run p of the tile
    auto copy = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int blk, int pos, int kvh) {
      if (dp_elect()) dp_expect(bar, L::TILE);
      __syncwarp();
      for (int p = 0; p < boxes; ++p) {
        const int b = __shfl_sync(0xffffffffu, blk, p), z = __shfl_sync(0xffffffffu, pos, p);
        if (dp_elect()) {
#pragma unroll
          for (int x = 0; x < L::HALVES; ++x) dp_tma4(dst + (uint32_t)(x * 16384) + (uint32_t)p * box_bytes, map, bar, 64 * x, kvh, z, b);
        }
        __syncwarp();
      }
    };
    // Q of the halves of piece c, each as soon as the last scores of its previous one are done
    auto load_q = [&](const DpCursor& c) -> bool {
      for (int h = 0; h < c.nq; ++h) {
        if ((q_used >> h) & 1u) {
          const uint32_t parity = (q_phase >> h) & 1u;
          if (!wait_warp(bar_s + P_QFREE + 8 * h, parity)) return false;
          q_phase ^= 1u << h;
        }
        q_used |= 1u << h;
        if (dp_elect()) {
          dp_expect(bar_s + P_QFULL + 8 * h, (uint32_t)(TT * G * D * 2));
#pragma unroll
          for (int x = 0; x < L::HALVES; ++x)
            dp_tma3(base_s + L::Q + (uint32_t)(h * L::TILE + x * 16384), &maps.q, bar_s + P_QFULL + 8 * h, 64 * x, c.at.kvh * G,
                    c.q.q0 + c.at.t.tok0 + (c.twin ? 0 : h * TT));
        }
        __syncwarp();
      }
      return true;
    };
    do {
      int blk = 0, pos = 0;
      auto find = [&](int j) {              // block and position of this lane's run of keys in tile j of the piece
        if (lane < boxes && j < cur.cnt) {
          const int key = (cur.at.t.t0 + cur.off + j) * DP_KT + lane * box;
          const int b = key / a.block_size;
          pos = key - b * a.block_size;
          blk = (int)dense_block(a, cur.at.s, b);
        }
      };
      find(0);
      for (int j = 0; j < cur.cnt && go; ++j, ++g) {
        const int blk_j = blk, pos_j = pos;
        find(j + 1);                        // in flight while the ring is waited for
        const uint32_t slot = (uint32_t)(g % NP);
        if (of_k) {
          if (g >= NP) go = wait_warp(bar_s + P_KFREE + 8 * slot, (uint32_t)((g / NP - 1) & 1));
          if (!go) break;
          copy(&maps.k, base_s + L::KV + 2 * slot * L::TILE, g == 0 ? bar_s + P_KFIRST : bar_s + P_PAIR + 8 * (uint32_t)((g - 1) % NP), blk_j, pos_j, cur.at.kvh);
          if (j == 0) go = load_q(cur);
        } else {
          if (g >= NP) go = wait_warp(bar_s + P_VFREE + 8 * slot, (uint32_t)((g / NP - 1) & 1));
          if (!go) break;
          const uint32_t full = bar_s + P_PAIR + 8 * slot, dst = base_s + L::KV + (2 * slot + 1) * L::TILE;
          // keys of the tile that a row of the row tile may see: inside the sequence, and not before all rows' windows
          const int key0 = (cur.at.t.t0 + cur.off + j) * DP_KT, z = cur.q.total - key0;
          const int before = a.window > 0 ? cur.q.total - cur.q.qlen + cur.at.t.tok0 + 1 - a.window - key0 : 0;
          const bool part = z < DP_KT || before > 0;
          copy(&maps.v, dst, part ? bar_s + P_TAIL : full, blk_j, pos_j, cur.at.kvh);
          if (part) {                       // the other values are zeroed before the tile is handed over
            const bool there = __all_sync(0xffffffffu, mbar_wait(bar_s + P_TAIL, (uint32_t)(tails++ & 1)));      // also when others gave up: the copy is in flight
            if (!there) {
              g_dense_prefill_status = 1;
              asm volatile("st.shared.u32 [%0], %1;" :: "r"(failed_s), "r"(1u) : "memory");
              go = false;
              break;
            }
            auto zero = [&](int from, int to) {      // keys of the tile
              for (int e = from * 8 + lane; e < to * 8; e += 32)
#pragma unroll
                for (int x = 0; x < L::HALVES; ++x)
                  asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" :: "r"(dst + (uint32_t)(x * 16384 + e * 16)), "r"(0u) : "memory");
            };
            zero(0, before < DP_KT ? before : DP_KT);
            zero(z < 0 ? 0 : z, DP_KT);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) dp_arrive(full);
          }
        }
      }
    } while (go && cur.next(a, w, s_round));
    // A CTA must not leave while copies into its shared memory are in flight, also when it gives up: the last barriers once
    // more.  The values are announced for tiles < gv, the keys on the barriers of tiles < gk - 1 (there are no keys behind
    // the last tile, and a side that gave up announces nothing more): the side that is behind stands in.
    if (lane == 0) s_copied[of_k ? 1 : 0] = g;
    asm volatile("bar.sync 2, 64;" ::: "memory");
    const int gv = s_copied[0], gk = s_copied[1], all = gv > gk - 1 ? gv : gk - 1;
    if (lane == 0)
      for (int p = of_k ? (gk > 0 ? gk - 1 : 0) : gv; p < all; ++p) dp_arrive(bar_s + P_PAIR + 8 * (uint32_t)(p % NP));
    __syncwarp();
    if (gk > 0) mbar_wait(bar_s + P_KFIRST, 0u);
    for (int p = all - NP < 0 ? 0 : all - NP; p < all; ++p) mbar_wait(bar_s + P_PAIR + 8 * (uint32_t)(p % NP), (uint32_t)((p / NP) & 1));
    for (int h = 0; h < 2; ++h)
      if ((q_used >> h) & 1u) mbar_wait(bar_s + P_QFULL + 8 * h, (q_phase >> h) & 1u);
  } else if (work) {
    // ================= softmax warps: half = warp / 4, thread = row =================
    const int half = warp >> 2, quad = warp & 3;
    const int r = quad * 32 + lane;
    const uint32_t t_lane = ((uint32_t)(quad * 32)) << 16;
    const uint32_t t_s = tmem + t_lane + (uint32_t)(half * 128), t_o = tmem + t_lane + (uint32_t)(L::T_O + half * 128);
    const int r_tok = r / G;
    const float c = a.scale_log2;
    uint8_t* stage = base + L::STAGE + warp * 32 * L::SROW;
    uint32_t rows4 = 0, heads4 = 0;      // token and head of rows 8 e + lane / 4 of the warp, a byte each
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rr = quad * 32 + 8 * e + (lane >> 2), t = rr / G;
      rows4 |= (uint32_t)t << (8 * e);
      heads4 |= (uint32_t)(rr - t * G) << (8 * e);
    }
    int step = 0;               // sub-tiles of this half
    uint32_t joined = 0, pieces = 0;      // parities of the next join and of this half's next piece
    bool ok = true;
    do {
      if (half < cur.nq) {
        const int of = cur.twin ? 0 : half;         // the half of the row tile that its rows are
        const int tok = cur.at.t.tok0 + of * TT + r_tok;
        const bool live = r_tok < TT && tok < cur.q.qlen;
        const int lim = live ? cur.q.total - cur.q.qlen + tok + 1 : 0x7fffffff;      // keys below it; a row without a token masks nothing
        const int low = live && a.window > 0 && lim > a.window ? lim - a.window : 0;
        const int lim_w = __reduce_min_sync(0xffffffffu, lim), low_w = __reduce_max_sync(0xffffffffu, low);
        float m = -CUDART_INF_F, l = 0.f;      // reference in log2 units, sum of the weights
        for (int x = 0; x < 2 * cur.tiles(half); ++x) {
          const int u = x & 1;
          if (!wait_warp(bar_s + P_SFULL + 8 * (uint32_t)(2 * half + u), (uint32_t)((step >> 1) & 1))) { ok = false; break; }
          ++step;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          uint32_t v[64];
          tmem_ld32(t_s + 64 * u, *reinterpret_cast<uint32_t (*)[32]>(&v[0]));
          tmem_ld32(t_s + 64 * u + 32, *reinterpret_cast<uint32_t (*)[32]>(&v[32]));
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          const int key0 = (cur.at.t.t0 + cur.off) * DP_KT + 64 * x + (cur.twin ? (x >> 1) * DP_KT + half * DP_KT : 0);
          if (key0 + 64 > lim_w || key0 < low_w) {
            // a bit per key: those below the limit and not below the window's edge (bits by constant position become predicates
            // several at a time)
            const int hi = lim - key0, lo = low - key0;
            const uint64_t upto = hi >= 64 ? ~0ull : (hi <= 0 ? 0ull : (1ull << hi) - 1), from = lo >= 64 ? 0ull : (lo <= 0 ? ~0ull : ~0ull << lo);
            const uint32_t see0 = (uint32_t)(upto & from), see1 = (uint32_t)((upto & from) >> 32);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              v[i] = (see0 & (1u << i)) != 0u ? v[i] : 0xff800000u;
              v[32 + i] = (see1 & (1u << i)) != 0u ? v[32 + i] : 0xff800000u;
            }
          }
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = dp_max3(__uint_as_float(v[i]), __uint_as_float(v[4 + i]), __uint_as_float(v[8 + i]));
#pragma unroll
          for (int i = 12; i < 60; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = dp_max3(mx[e], __uint_as_float(v[i + e]), __uint_as_float(v[i + 4 + e]));
          mx[0] = dp_max3(mx[0], __uint_as_float(v[60]), __uint_as_float(v[61]));
          mx[1] = dp_max3(mx[1], __uint_as_float(v[62]), __uint_as_float(v[63]));
          const float top = dp_max3(mx[0], mx[1], dp_max3(mx[2], mx[3], mx[3])) * c;
          const bool grow = live && !(top <= m + DENSE_TOP<BF>);      // also for a NaN, which then stays
          if (__any_sync(0xffffffffu, grow)) {
            const float to = top - DENSE_SHIFT<BF>, f = grow ? dense_ex2(m - to) : 1.0f;      // m = -inf: 0
            if (grow) { m = to; l *= f; }
            if (x > 0) {                    // O holds the products of the sub-tiles before: P V of the last one may still run
              if (!wait_warp(bar_s + P_PVDONE + 8 * half, (uint32_t)((step - 2) & 1))) { ok = false; break; }
              asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
              for (int y = 0; y < D / 32; ++y) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * y, o);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                tmem_st32(t_o + 32 * y, o);
              }
            }
          }
          const float ref = m == -CUDART_INF_F ? 0.f : -m;
          // weights, rounded once to the cache's type for the product; the sum takes them before
          const uint64_t c2 = dp_pk(c, c), ref2 = dp_pk(ref, ref);
          uint64_t sum = 0;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t ph[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              dp_upk(dp_fma2(dp_pk(__uint_as_float(v[32 * y + 2 * i]), __uint_as_float(v[32 * y + 2 * i + 1])), c2, ref2), x0, x1);
              const float p0 = dense_ex2(x0), p1 = dense_ex2(x1);
              sum = dp_add2(sum, dp_pk(p0, p1));
              ph[i] = dense_pack<BF>(p0, p1);
            }
            tmem_st16(t_s + 64 * u + 16 * y, ph);
          }
          {
            float l0, l1;
            dp_upk(sum, l0, l1);
            l += l0 + l1;
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) dp_arrive(bar_s + P_PFULL + 8 * (uint32_t)(2 * half + u));
        }
        // all products of the piece have a barrier of their own: the one that counts sub-tiles may be two ahead of a warp that
        // waits here, which a parity does not tell
        if (!ok || !wait_warp(bar_s + P_OFULL + 8 * half, pieces)) { ok = false; break; }
        pieces ^= 1u;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (cur.twin) {
          // The same rows' other tiles: half 1 hands over its maximum and sum; its O lies in the same lanes of tensor memory, and
          // half 0 adds it to its own:  O = 2^(m0 - M) O0 + 2^(m1 - M) O1.
          float2* ml = reinterpret_cast<float2*>(base + L::STAGE + (4 + quad) * 32 * L::SROW) + lane;
          if (half == 1) {
            *ml = make_float2(m, l);
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) dp_arrive(bar_s + P_JOIN);
            if (!wait_warp(bar_s + P_JOIN + 8, joined)) { ok = false; break; }      // O and the staging are free again
            joined ^= 1u;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            continue;
          }
          if (!wait_warp(bar_s + P_JOIN, joined)) { ok = false; break; }
          joined ^= 1u;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const float2 o1 = *ml;
          const float top = fmaxf(m, o1.x);
          const bool has0 = m != -CUDART_INF_F, has1 = o1.x != -CUDART_INF_F;      // a side that saw no key adds nothing
          const float f0 = has0 ? dense_ex2(m - top) : 0.f, f1 = has1 ? dense_ex2(o1.x - top) : 0.f;
          m = top;
          l = f0 * l + f1 * o1.y;
#pragma unroll 1
          for (int y = 0; y < D / 32; ++y) {
            uint32_t o[32], p[32];
            tmem_ld32(t_o + 32 * y, o);
            tmem_ld32(t_o + 128 + 32 * y, p);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint((has0 ? __uint_as_float(o[i]) * f0 : 0.f) + (has1 ? __uint_as_float(p[i]) * f1 : 0.f));
            tmem_st32(t_o + 32 * y, o);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) dp_arrive(bar_s + P_JOIN + 8);
        }
        const bool whole = cur.cnt == cur.at.t.n;
        const int64_t slot = ((int64_t)cur.round * gridDim.x + blockIdx.x) * 2 + (cur.first ? 0 : 1);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        // A thread holds a row, but a store instruction should write whole pieces of few rows: 64 bytes of each of the warp's
        // 32 rows at a time go through shared memory, four lanes then write a row's piece (thread by thread, the stores
        // of a row tile took 10000 cycles: 32 lines per instruction).
        const int c4 = lane & 3;
        uint32_t alive = 0;                 // of rows 8 e + lane / 4
        char* dst4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = (rows4 >> (8 * e)) & 255, hd = (heads4 >> (8 * e)) & 255, tok_e = cur.at.t.tok0 + of * TT + t;
          if (t < TT && tok_e < cur.q.qlen) alive |= 1u << e;
          dst4[e] = static_cast<char*>(a.out) + 2 * ((int64_t)(cur.q.q0 + tok_e) * a.out_st + (int64_t)(cur.at.kvh * G + hd) * a.out_sh + 8 * c4);
        }
        if (whole) {
          uint32_t w[D / 2];
#pragma unroll
          for (int x = 0; x < D / 64; ++x) {
            uint32_t o[64];
            tmem_ld32(t_o + 64 * x, *reinterpret_cast<uint32_t (*)[32]>(&o[0]));
            tmem_ld32(t_o + 64 * x + 32, *reinterpret_cast<uint32_t (*)[32]>(&o[32]));
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 32; ++e)      // l == 0: no key was seen (0 times whatever is there would keep a NaN)
              w[32 * x + e] = l == 0.f ? 0u : dense_pack<BF>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
          }
#pragma unroll
          for (int x = 0; x < D / 32; ++x) {
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(stage + lane * L::SROW + 16 * e) = make_uint4(w[16 * x + 4 * e], w[16 * x + 4 * e + 1], w[16 * x + 4 * e + 2], w[16 * x + 4 * e + 3]);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if ((alive >> e) & 1u)
                *reinterpret_cast<uint4*>(dst4[e] + 64 * x) = *reinterpret_cast<const uint4*>(stage + (8 * e + (lane >> 2)) * L::SROW + 16 * c4);
          }
        } else {
          // float4 of 4 columns, rows fastest: a store instruction writes 512 bytes in a row
          float4* part = reinterpret_cast<float4*>(part_acc) + slot * 64 * D + of * 128 + r;
#pragma unroll 1
          for (int x = 0; x < D / 32; ++x) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * x, o);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
            for (int e = 0; e < 8; ++e)
              part[(8 * x + e) * 256] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          }
        }
        if (live && !whole) {
          part_ml[(slot * 256 + of * 128 + r) * 2] = m;
          part_ml[(slot * 256 + of * 128 + r) * 2 + 1] = l;
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      }
    } while (cur.next(a, w, s_round));
  }

  // ---- per round, the row tile that this CTA begins and does not finish (the last of its part): how many parts it has ----
  if (warp < max_rounds) {
    DpDesc d{0, 0, 0, 0, 0, {0, 0, 0}};
    if (warp < n_rounds && s_round[warp].u1 > s_round[warp].u0 && s_round[warp].end_off > 0 && lds_u32(failed_s) == 0u) {
      const DpRound& r = s_round[warp];
      const int64_t begin = r.u1 - r.end_off;
      if (begin >= r.u0) {
        const DpPlace p = dp_locate(a, w, begin, lane);
        // the last CTA that begins before the row tile's end.  A cut behind that end stays behind it when it is moved, one before
        // it may be moved to it (asking for the CTAs' beginnings one by one took 0.6 us each, 16 us for 5 tokens behind 30000)
        const int64_t end = begin + DP_PIECE + p.t.n;
        int c1 = (int)blockIdx.x + 1, above = r.n;
        while (above - c1 > 1) {
          const int mid = (c1 + above) >> 1;
          if (dp_cut(r.lo, r.hi, r.n, mid) < end) c1 = mid; else above = mid;
        }
        DpPlace e;
        while (c1 > (int)blockIdx.x + 1 && dp_begin(a, w, r.lo, r.hi, r.n, c1, lane, &e) >= end) --c1;
        d.parts = c1 - (int)blockIdx.x + 1;
        d.slot0 = begin == r.u0 ? 0 : 1;
        d.row0 = w.seq[p.s].q0 + p.t.tok0;
        d.ntok = p.t.ntok;
        d.kvh = p.kvh;
      }
    }
    if (lane == 0) desc[warp * gridDim.x + blockIdx.x] = d;
  }

  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  // a CTA in which a wait gave up may still have MMAs in flight: commit once more and wait (bounded) before the columns go back
  int leak = 0;
  if ((warp == L::MMA_WARP || warp == L::MMA_WARP2) && lds_u32(failed_s) != 0u && dp_elect()) {
    const uint32_t bar = bar_s + P_DRAIN + (warp == L::MMA_WARP ? 0u : 8u);
    umma_commit(bar);
    leak = mbar_wait(bar, 0u) ? 0 : 1;
    if (leak) g_dense_prefill_status = 2;
  }
  __syncwarp();
  leak = __syncthreads_or(leak);
  if (warp == L::MMA_WARP && !leak) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem) : "memory");
  }
}

// Row tiles that were cut: out = sum_p 2^(m_p - M) acc_p / sum_p 2^(m_p - M) l_p.  A slice is 16 columns (a 32-byte sector) of
// 128 rows, half of a row tile; a thread takes a row of it, neighbouring threads neighbouring rows (the partials' layout).  Two
// blocks per SM: starting a block costs some 10 ns.
// !SPREAD: a block per half of the row tile that a CTA began, round by round.  Most have two or three parts.
// SPREAD, for calls of few row tiles, which have many parts each: every block lists the halves that have parts, the slices are
// spread over all blocks, and where that leaves threads idle, `groups` of 128 threads share a slice: group g takes parts g,
// g + groups, ..., and the groups are joined in order through shared memory (their number depends on the call's lengths alone,
// so results repeat).  Inside a graph, keys from HBM: 100 tokens behind 20000 (32 / 8 heads of 128, 18 parts per row tile) take 61 us
// with it and 68 without, 60 tokens (8 / 1 heads, two row tiles of 20 parts) 34 and 56, 5 tokens 25 and 34; 5 tokens behind 5000 (5
// parts) 20.7 either way.
constexpr int PM_THREADS = 1024, PM_LIST = DP_MAX_ROUNDS * 256 * 2;      // at most 256 SMs
constexpr int PM_SMEM = PM_THREADS * 18 * (int)sizeof(float);
template <bool BF, int D, bool SPREAD>
__global__ void __launch_bounds__(PM_THREADS)
dense_prefill_merge_kernel(DenseArgs a, int G, int TT, int rounds, int ctas, int head, int tail, const DpDesc* desc, const float* part_ml, const float* part_acc) {
  extern __shared__ float s_part[];                    // [18][PM_THREADS]: maximum, sum, 16 columns
  __shared__ uint16_t s_list[SPREAD ? PM_LIST : 1];    // 2 * place in desc + half
  __shared__ int s_count[32], s_most[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  auto zeros = [&](int64_t from, int64_t to) {
    for (int64_t row = (from > 0 ? from : 0) + blockIdx.x; row < to && row < a.n_tokens; row += gridDim.x)
      for (int e = tid; e < a.num_q_heads * (D / 8); e += PM_THREADS)
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.out_st + (int64_t)(e / (D / 8)) * a.out_sh + e % (D / 8) * 8) =
            make_uint4(0u, 0u, 0u, 0u);
  };
  // rows before the first sequence and behind the last (`tail` of them in this launch) come out as zeros
  if (head) zeros(0, load_index(a.starts, a.qs_dtype, 0));
  if (tail >= 0) zeros(load_index(a.starts, a.qs_dtype, tail), a.n_tokens);
  const int in_half = tid & 127, tok_in = in_half / G;
  // columns 16 c16 .. + 15 of half `half` of the row tile whose first part is described at `first`
  auto slice = [&](bool there, int first, int half, int c16, int group, int groups) {
    DpDesc d{0, 0, 0, 0, 0, {0, 0, 0}};
    if (there) d = desc[first];
    const int r = half * 128 + in_half, tok = half * TT + tok_in;
    const bool live = d.parts > 1 && tok_in < TT && tok < d.ntok;
    float top = -CUDART_INF_F, sum = 0.f;
    float4 acc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    // one more set of values: maximum, sum and columns
    auto add = [&](const float2& ml, const float4 (&v)[4], float t) {
      if (ml.x == -CUDART_INF_F) return;      // no key of this row was seen
      const float f = dense_ex2(ml.x - t);
      sum += f * ml.y;
#pragma unroll
      for (int k = 0; k < 4; ++k) { acc[k].x += f * v[k].x; acc[k].y += f * v[k].y; acc[k].z += f * v[k].z; acc[k].w += f * v[k].w; }
    };
    auto rise = [&](float t) {
      const float f = top == -CUDART_INF_F ? 0.f : dense_ex2(top - t);
      top = t;
      sum *= f;
#pragma unroll
      for (int k = 0; k < 4; ++k) { acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f; }
    };
    if (live) {
      auto slot = [&](int p) -> int64_t { return ((int64_t)first + p) * 2 + (p == 0 ? d.slot0 : 0); };
      constexpr int B = 2;
      for (int base = group; base < d.parts; base += B * groups) {
        float2 ml[B];
        float4 v[B][4];
#pragma unroll
        for (int b = 0; b < B; ++b) {
          const int p = base + b * groups;
          const bool in = p < d.parts;
          ml[b] = in ? *reinterpret_cast<const float2*>(part_ml + (slot(p) * 256 + r) * 2) : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[b][k] = in ? reinterpret_cast<const float4*>(part_acc)[slot(p) * 64 * D + (4 * c16 + k) * 256 + r] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        rise(fmaxf(fmaxf(top, ml[0].x), ml[1].x));
#pragma unroll
        for (int b = 0; b < B; ++b) add(ml[b], v[b], top);
      }
    }
    if (SPREAD && groups > 1) {
      s_part[tid] = top;
      s_part[PM_THREADS + tid] = sum;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s_part[(2 + 4 * k) * PM_THREADS + tid] = acc[k].x;
        s_part[(3 + 4 * k) * PM_THREADS + tid] = acc[k].y;
        s_part[(4 + 4 * k) * PM_THREADS + tid] = acc[k].z;
        s_part[(5 + 4 * k) * PM_THREADS + tid] = acc[k].w;
      }
      __syncthreads();
      if (group == 0 && live) {
        float t = top;
        for (int g = 1; g < groups; ++g) t = fmaxf(t, s_part[tid + 128 * g]);
        rise(t);
#pragma unroll 1
        for (int g = 1; g < groups; ++g) {
          const float* from = s_part + tid + 128 * g;
          float4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[k] = make_float4(from[(2 + 4 * k) * PM_THREADS], from[(3 + 4 * k) * PM_THREADS], from[(4 + 4 * k) * PM_THREADS], from[(5 + 4 * k) * PM_THREADS]);
          add(make_float2(from[0], from[PM_THREADS]), v, top);
        }
      }
      __syncthreads();
    }
    if (group == 0 && live) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      uint32_t o[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[2 * k] = dense_pack<BF>(acc[k].x * inv, acc[k].y * inv);
        o[2 * k + 1] = dense_pack<BF>(acc[k].z * inv, acc[k].w * inv);
      }
      uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + (int64_t)(d.row0 + tok) * a.out_st + (int64_t)(d.kvh * G + in_half - tok_in * G) * a.out_sh + 16 * c16);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  };
  if constexpr (!SPREAD) {
    const int half = (int)blockIdx.x >= ctas ? 1 : 0, c = (int)blockIdx.x - half * ctas;
    for (int z = 0; z < rounds; ++z) slice(tid < 128 * (D / 16), z * ctas + c, half, tid >> 7, 0, 1);
  } else {
    // ---- the halves with parts, in the order of desc (the same list in every block) ----
    int entries = 0, most = 0;
    for (int base = 0; base < rounds * ctas; base += PM_THREADS) {
      const int at = base + tid;
      int parts = 0, n = 0;
      if (at < rounds * ctas) {
        parts = desc[at].parts;
        n = parts < 2 ? 0 : (desc[at].ntok > TT ? 2 : 1);
      }
      int inc = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += x;
      }
      const int top = __reduce_max_sync(0xffffffffu, n > 0 ? parts : 0);
      if (lane == 31) s_count[warp] = inc;
      if (lane == 0) s_most[warp] = top;
      __syncthreads();
      const int c = s_count[lane], before = __reduce_add_sync(0xffffffffu, lane < warp ? c : 0);
      most = max(most, __reduce_max_sync(0xffffffffu, s_most[lane]));
      for (int h = 0; h < n; ++h) s_list[entries + before + inc - n + h] = (uint16_t)(2 * at + h);
      entries += __reduce_add_sync(0xffffffffu, c);
      __syncthreads();
    }
    const int slices = entries * (D / 16);
    int groups = 1;      // four parts each at least
    while (groups < 8 && groups * 4 < most && slices * groups * 2 <= (int)gridDim.x * (PM_THREADS / 128)) groups *= 2;
    const int at_once = PM_THREADS / 128 / groups, sub = (tid >> 7) / groups, group = (tid >> 7) - sub * groups;
    for (int s0 = blockIdx.x * at_once; s0 < slices; s0 += gridDim.x * at_once) {      // the same rounds for all threads of the block
      const int s = s0 + sub, entry = s < slices ? s_list[s / (D / 16)] : 0;
      slice(s < slices, entry >> 1, entry & 1, s % (D / 16), group, groups);
    }
  }
}

typedef CUresult (*dp_encode_fn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
dp_encode_fn dp_encoder() {
  static const dp_encode_fn fn = []() -> dp_encode_fn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<dp_encode_fn>(p);
    cudaGetLastError();
    return nullptr;
  }();
  return fn;
}

int gcd(int a, int b) { return b == 0 ? a : gcd(b, a % b); }

// Maps over the call's query and caches (this GPU's memory).  A stride of a dimension of one element is never used by a
// copy but still checked by the driver: the row pitch stands in for it.
bool dp_make_maps(const DenseArgs& a, bool bf, int G, int TT, int box, DpMaps* m) {
  const dp_encode_fn enc = dp_encoder();
  if (enc == nullptr) return false;
  const CUtensorMapDataType type = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const cuuint64_t row = (cuuint64_t)a.head_dim * 2;
  auto pitch = [&](int64_t stride, int64_t n) -> cuuint64_t { return n > 1 ? (cuuint64_t)(stride * 2) : row; };
  {
    const cuuint64_t dims[3] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.num_q_heads, (cuuint64_t)a.n_tokens};
    const cuuint64_t strides[2] = {pitch(a.q_sh, a.num_q_heads), pitch(a.q_st, a.n_tokens)};
    const cuuint32_t b[3] = {64, (cuuint32_t)G, (cuuint32_t)TT};
    if (enc(&m->q, type, 3, const_cast<void*>(a.q), dims, strides, b, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return false;
  }
  for (int side = 0; side < 2; ++side) {
    const cuuint64_t dims[4] = {(cuuint64_t)a.head_dim, (cuuint64_t)a.num_kv_heads, (cuuint64_t)a.block_size, (cuuint64_t)a.num_blocks};
    const cuuint64_t strides[3] = {pitch(side ? a.v_sh : a.k_sh, a.num_kv_heads), pitch(side ? a.v_sp : a.k_sp, a.block_size),
                                   pitch(side ? a.v_sb : a.k_sb, a.num_blocks)};
    const cuuint32_t b[4] = {64, 1, (cuuint32_t)box, 1};
    if (enc(side ? &m->v : &m->k, type, 4, const_cast<void*>(side ? a.v : a.k), dims, strides, b, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return false;
  }
  return true;
}

struct DpWorkspace { DpDesc* desc; float* ml; float* acc; };
size_t dp_workspace(int head_dim, int rounds, char* base, DpWorkspace* w) {
  const size_t n = (size_t)sm_count() * rounds;
  const size_t d = (n * sizeof(DpDesc) + 255) / 256 * 256, ml = n * 2 * 256 * 2 * sizeof(float), acc = n * 2 * 256 * (size_t)head_dim * sizeof(float);
  if (w != nullptr) *w = DpWorkspace{reinterpret_cast<DpDesc*>(base), reinterpret_cast<float*>(base + d), reinterpret_cast<float*>(base + d + ml)};
  return d + ml + acc;
}

// Rounds that a call may need: its keys and values are at most those of the pool, or of full block-table rows, and only
// sequences of DP_ROUND_TILES row tiles count, which fewer new tokens than that cannot have (for one drafted token over a large pool
// at head_dim 128 the workspace is 40 MB instead of the 158 of four rounds).
int dp_rounds(int num_tokens, int group, int num_kv_heads, int head_dim, int64_t num_blocks, int block_size, int num_seqs, int max_blocks_per_seq) {
  if (group > 0 && num_tokens <= (DP_ROUND_TILES - 1) * 2 * (128 / group)) return 1;
  const double rows = (double)num_seqs * max_blocks_per_seq, blocks = rows < (double)num_blocks ? rows : (double)num_blocks;
  const double n = blocks * block_size * num_kv_heads * 4.0 * head_dim / (double)DP_ROUND_BYTES;
  return n <= 1.0 ? 1 : (n >= DP_MAX_ROUNDS ? DP_MAX_ROUNDS : (int)ceil(n));
}

// A call without sequences: no row belongs to one.  The merge without parts writes their zeros.
template <int D>
int dp_launch_zeros(const DenseArgs& a, int G, int TT, cudaStream_t st) {
  dense_prefill_merge_kernel<false, D, false><<<2 * sm_count(), PM_THREADS, 0, st>>>(a, G, TT, 0, sm_count(), 1, 0, nullptr, nullptr, nullptr);
  return check_launch("dense_prefill_merge_kernel");
}

template <bool BF, int D>
int dp_launch(const DenseArgs& all, const DpMaps& maps, int G, int TT, int box, int rounds, bool zero_tail, const DpWorkspace& w, cudaStream_t st) {
  using L = DpL<D>;
  cudaError_t e = cudaFuncSetAttribute(dense_prefill_kernel<BF, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e != cudaSuccess) return fail((int)e, "dense prefill attention: smem attribute: %s", cudaGetErrorString(e));
  const int grid = sm_count(), tt2 = 2 * TT;
  // few row tiles (at most a quarter of the SMs' number, so four parts or more each) that may be long (64 key tiles, eight parts)
  const bool spread = (int64_t)all.max_blocks_per_seq * all.block_size >= 64 * DP_KT &&
                      ((int64_t)all.n_tokens / tt2 + (all.num_seqs < all.n_tokens ? all.num_seqs : all.n_tokens)) * all.num_kv_heads <= grid / 4 &&
                      grid <= PM_LIST / 2 / DP_MAX_ROUNDS;
  auto merge = spread ? dense_prefill_merge_kernel<BF, D, true> : dense_prefill_merge_kernel<BF, D, false>;
  if (spread) {
    e = cudaFuncSetAttribute(merge, cudaFuncAttributeMaxDynamicSharedMemorySize, PM_SMEM);
    if (e != cudaSuccess) return fail((int)e, "dense prefill merge: smem attribute: %s", cudaGetErrorString(e));
  }
  for (int s0 = 0; s0 < all.num_seqs; s0 += DP_MAX_SEQS) {
    const int seqs = all.num_seqs - s0 < DP_MAX_SEQS ? all.num_seqs - s0 : DP_MAX_SEQS;
    DenseArgs a = all;
    a.starts = static_cast<const char*>(all.starts) + (size_t)s0 * (all.qs_dtype == AKV_I64 ? 8 : 4);
    a.seq_lens = static_cast<const char*>(all.seq_lens) + (size_t)s0 * (all.sl_dtype == AKV_I64 ? 8 : 4);
    a.block_tables = static_cast<const char*>(all.block_tables) + (int64_t)s0 * all.bt_stride * (all.bt_dtype == AKV_I64 ? 8 : 4);
    // programmatic launches: the kernels set up (barriers, tensor memory) while the one before them ends, and wait for its
    // end before they read anything
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(L::THREADS);
    cfg.dynamicSmemBytes = L::SMEM;
    e = cudaLaunchKernelEx(&cfg, dense_prefill_kernel<BF, D>, a, maps, seqs, G, TT, box, rounds, w.desc, w.ml, w.acc);
    if (e != cudaSuccess) return fail((int)e, "dense prefill attention: %s", cudaGetErrorString(e));
    if (int rc = check_launch("dense_prefill_attn_kernel")) return rc;
    cfg.dynamicSmemBytes = spread ? PM_SMEM : 0;
    cfg.gridDim = dim3((unsigned)(2 * grid));
    cfg.blockDim = dim3(PM_THREADS);
    e = cudaLaunchKernelEx(&cfg, merge, a, G, TT, rounds, grid, zero_tail && s0 == 0 ? 1 : 0, zero_tail && s0 + seqs == all.num_seqs ? seqs : -1, (const DpDesc*)w.desc, (const float*)w.ml, (const float*)w.acc);
    if (e != cudaSuccess) return fail((int)e, "dense prefill merge: %s", cudaGetErrorString(e));
    if (int rc = check_launch("dense_prefill_merge_kernel")) return rc;
  }
  return AKV_OK;
}

}  // namespace

int dense_prefill_status(int* host_out, int reset) {
  cudaError_t e = cudaMemcpyFromSymbol(host_out, g_dense_prefill_status, sizeof(int));
  if (e == cudaSuccess && reset) { const int z = 0; e = cudaMemcpyToSymbol(g_dense_prefill_status, &z, sizeof(int)); }
  return e == cudaSuccess ? AKV_OK : fail((int)e, "dense prefill status: %s", cudaGetErrorString(e));
}

int dense_prefill_withhold(int tile) {
  cudaError_t e = cudaMemcpyToSymbol(g_dense_prefill_withhold, &tile, sizeof(int));
  return e == cudaSuccess ? AKV_OK : fail((int)e, "dense prefill test hook: %s", cudaGetErrorString(e));
}

}  // namespace akv

AKV_EXPORT size_t akv_dense_prefill_attn_workspace_bytes(int num_kv_heads, int head_dim, int64_t num_blocks, int block_size, int num_seqs,
                                                          int max_blocks_per_seq) {
  if (num_kv_heads <= 0 || head_dim <= 0 || num_blocks < 0 || block_size <= 0 || num_seqs < 0 || max_blocks_per_seq < 0) return 0;
  return akv::dp_workspace(head_dim, akv::dp_rounds(0x7fffffff, 1, num_kv_heads, head_dim, num_blocks, block_size, num_seqs, max_blocks_per_seq), nullptr, nullptr);
}

AKV_EXPORT size_t akv_dense_prefill_attn_call_bytes(int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int64_t num_blocks,
                                                    int block_size, int num_seqs, int max_blocks_per_seq) {
  if (num_tokens < 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0 || num_blocks < 0 || block_size <= 0 || num_seqs < 0 ||
      max_blocks_per_seq < 0) return 0;
  return akv::dp_workspace(head_dim, akv::dp_rounds(num_tokens, num_q_heads / num_kv_heads, num_kv_heads, head_dim, num_blocks, block_size, num_seqs, max_blocks_per_seq),
                           nullptr, nullptr);
}

AKV_EXPORT int akv_dense_prefill_attn(const akv_dense_attn_params* p) {
  akv::DenseArgs a;
  if (int rc = akv::dense_common(p, "akv_dense_prefill_attn", &a)) return rc;
  if (a.n_tokens == 0 || (a.num_seqs == 0 && !p->zero_tail)) return AKV_OK;
  if (!a.out) return akv::fail(AKV_ERR_ARG, "akv_dense_prefill_attn: null out");
  if (!a.starts) return akv::fail(AKV_ERR_ARG, "akv_dense_prefill_attn: null query_start_loc");
  const int G = a.num_q_heads / a.num_kv_heads;
  const int box = a.block_size % 128 == 0 ? 128 : akv::gcd(a.block_size, 128);
  if (a.head_dim == 256 || G > 128 || box < 8 || a.max_blocks_per_seq == 0 || a.num_blocks > 0x7fffffffll)
    return akv::fail(AKV_ERR_UNSUPPORTED, "akv_dense_prefill_attn: head_dim %d, %d query heads per KV head, block_size %d, %d blocks per "
                     "sequence (64 or 128, at most 128, a multiple of 8, at least 1)", a.head_dim, G, a.block_size, a.max_blocks_per_seq);
  const int TT = 128 / G;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(p->stream);
  if (a.num_seqs == 0) return a.head_dim == 128 ? akv::dp_launch_zeros<128>(a, G, TT, st) : akv::dp_launch_zeros<64>(a, G, TT, st);
  akv::DpWorkspace w;
  const int rounds = akv::dp_rounds(a.n_tokens, G, a.num_kv_heads, a.head_dim, a.num_blocks, a.block_size, a.num_seqs, a.max_blocks_per_seq);
  const size_t need = akv::dp_workspace(a.head_dim, rounds, static_cast<char*>(p->workspace), &w);
  if (!p->workspace || p->workspace_bytes < need || ((uintptr_t)p->workspace & 255))
    return akv::fail(AKV_ERR_WORKSPACE, "akv_dense_prefill_attn: workspace of %zu bytes (256-byte aligned) needed, got %zu", need, p->workspace_bytes);
  akv::DpMaps maps;
  const bool bf = p->dtype == AKV_BF16;
  if (!akv::dp_make_maps(a, bf, G, TT, box, &maps))
    return akv::fail(AKV_ERR_UNSUPPORTED, "akv_dense_prefill_attn: these strides cannot be described to the copy unit");
  if (a.head_dim == 128) return bf ? akv::dp_launch<true, 128>(a, maps, G, TT, box, rounds, p->zero_tail != 0, w, st) : akv::dp_launch<false, 128>(a, maps, G, TT, box, rounds, p->zero_tail != 0, w, st);
  return bf ? akv::dp_launch<true, 64>(a, maps, G, TT, box, rounds, p->zero_tail != 0, w, st) : akv::dp_launch<false, 64>(a, maps, G, TT, box, rounds, p->zero_tail != 0, w, st);
}
