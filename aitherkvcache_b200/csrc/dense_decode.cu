// Attention of single tokens over the dense (fp16 / bf16) paged cache.
//
//   o = sum_j w_j v_j / sum_j w_j,   w_j = 2^(c q.k_j - m),   c = scale log2(e),  j in [max(0, len - window), len)
//
// Bound by HBM: 4 D bytes per key and KV head are read once, whatever the number G of query heads that share them; the
// products are 8 D G flops for them, which mma.sync covers at a tenth of its rate.
//
// Work split.  The keys of a row - one sequence and one group of up to 8 NT query heads of a KV head - are cut into steps of
// 16 (32 at D = 64).  The steps of all rows are laid end to end and cut into one equal range per CTA (one or two per SM), so that any mixture
// of lengths keeps every SM busy to the end; every CTA finds its range itself from the lengths (block-wide prefix sum in shared memory).
// A CTA walks over the pieces of rows in its range; its warps take a piece's steps in turn, each with a ring of its own
// in shared memory filled by 16-byte cp.async copies (NS - 1 steps ahead, across the ends of pieces): no barrier in the
// loop.  At the end of a piece the warps' results are joined in a fixed order; a piece that is a whole row is written as
// output, others (two per CTA at most) go to the workspace and dense_decode_merge_kernel joins them, again in a fixed order.
//
// 16 keys in a warp: S^T[16 keys][8 heads] = K Q^T (keys as the rows of the product, so that up to 8 heads waste nothing),
// probabilities in float32, rounded once to the cache's type, transposed in registers (movmatrix) into the second
// operand of O^T[D][8 heads] += V^T P^T.  Scores, maxima, sums and O are float32.  The reference m moves only when a weight
// would pass 2^8 times the last reference's (DENSE_TOP in dense_attn.cuh), so the shuffles and the rescaling of O run a few times per row.
// Keys outside the range are filled with zeros by the copy and masked: whatever stale pages hold does not matter.
#include "dense_attn.cuh"
#include "umma.cuh"
#include <math_constants.h>

namespace akv {
namespace {

constexpr int DD_MAX_SEQS = 1024;        // sequences of one launch (their prefix sums live in shared memory)

template <int D, int NT> struct DdL {
  // two CTAs per SM where their rings fit: one streams while the other joins its warps' results at the end of a piece
  static constexpr int CTAS = D * NT <= 128 ? 2 : 1, W = 4, THREADS = 32 * W;
  static constexpr int KS = D == 64 ? 32 : 16;                // keys of a step: 8 KB of keys and values at D = 64 and 128
  static constexpr int STEP = KS * D * 2;                     // bytes of one operand of a step
  // about 192 KB of rings per SM (what 6.5 TB/s at over a microsecond of latency keep in flight, three times over), less
  // where the join buffer of 16 heads x 256 needs the room
  static constexpr int NS = D * NT == 512 ? 2 : 196608 / CTAS / (2 * STEP * W);
  static constexpr int RING = 2 * STEP * NS;                  // per warp
  static constexpr int H = 8 * NT;                            // heads of a row
  static constexpr int O = W * RING;                          // join buffer: [W / 2][H][OROW] float
  static constexpr int OROW = D + 4;                          // four rows apart: other banks
  static constexpr int ML = O + (W / 2) * H * OROW * 4;       // [2][W][H][2] float
  static constexpr int PRE = ML + 2 * W * H * 2 * 4;          // prefix sums of the steps
  static constexpr int SMEM = PRE + (DD_MAX_SEQS + 1) * 4 + 64;
  static_assert(CTAS * (SMEM + 256 + 1024) <= 233472, "shared memory");
};

__device__ __forceinline__ void dd_cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void dd_ldm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dd_ldm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t dd_movm(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool BF>
__device__ __forceinline__ void dd_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Keys [lo, len) that a sequence's token sees, in steps of KS from step lo / KS.
struct DdSpan { int lo, len, first, steps; };
template <int KS>
__device__ __forceinline__ DdSpan dd_span(const DenseArgs& a, int s) {
  DdSpan p;
  p.len = (int)load_ctx(a.seq_lens, a.sl_dtype, s, (int64_t)a.max_blocks_per_seq * a.block_size);
  p.lo = a.window > 0 && p.len > a.window ? p.len - a.window : 0;
  p.first = p.lo / KS;
  p.steps = (p.len + KS - 1) / KS - p.first;
  return p;
}

// What dense_decode_merge_kernel needs to know about the row whose first part CTA c wrote (parts < 2: nothing)
struct DdDesc { int parts, slot0, s, vh; };

// The CTAs that share T units: as many as are left with `least` units each (four steps per warp, about a round of its ring; a
// row shorter than that is not worth a second CTA and the join), at most the grid.
__device__ __forceinline__ int dd_ctas(int64_t units, int grid, int least) {
  const int64_t n = units / least;
  return n < 1 ? 1 : (n < grid ? (int)n : grid);
}
__device__ __forceinline__ int64_t dd_begin(int64_t units, int n, int c) { return units * c / n; }

// A warp's way through its CTA's range: piece (s, vh) with steps [t, t_end) of the row, this warp's next step `t`.
struct DdCursor {
  int s, vh, t, t_end;          // t counts from the row's first step
  int64_t left;                 // units behind this piece
  DdSpan span;
};

// PAGE16: 16 aligned keys lie inside one block.  HEADS: the CTA's warps take a row each of four neighbouring rows.
template <bool BF, int D, int NT, bool PAGE16, bool HEADS>
__global__ void __launch_bounds__(DdL<D, NT>::THREADS, DdL<D, NT>::CTAS)
dense_decode_kernel(DenseArgs a, int seqs0, int seqs, int rows, float* part_acc, float* part_ml, DdDesc* desc) {
  // rows: of a sequence; vheads: of the sequence in the list of units (four rows at a time with HEADS)
  using L = DdL<D, NT>;
  constexpr int W = L::W, NS = L::NS, H = L::H, KS = L::KS;
  constexpr int CPR = D / 8, RPP = 32 / CPR, PASSES = KS / RPP;     // 16-byte pieces per row, rows per pass of a warp
  const int vheads = HEADS ? rows / 4 : rows;
  extern __shared__ __align__(128) uint8_t dd_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* pre = reinterpret_cast<int*>(dd_smem + L::PRE);
  __shared__ int s_warp[W];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- prefix sums of the steps per sequence ----
  constexpr int PER = DD_MAX_SEQS / L::THREADS;
  {
    int n[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = tid * PER + i;
      n[i] = s < seqs ? dd_span<KS>(a, seqs0 + s).steps : 0;
      sum += n[i];
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += x;
    }
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    int base = inc - sum;
    for (int w = 0; w < warp; ++w) base += s_warp[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = tid * PER + i;
      if (s < seqs) pre[s] = base;
      base += n[i];
      if (s == seqs - 1) pre[seqs] = base;
    }
    __syncthreads();
  }
  // rows of sequences without keys: zeros
  for (int s = blockIdx.x; s < seqs; s += gridDim.x)
    if (pre[s + 1] == pre[s])
      for (int e = tid; e < a.num_q_heads * D; e += L::THREADS)
        dense_store<BF>(a.out, (int64_t)(seqs0 + s) * a.out_st + (int64_t)(e / D) * a.out_sh + e % D, 0.f);
  const int64_t units = (int64_t)pre[seqs] * vheads;
  const int n_ctas = dd_ctas(units, gridDim.x, HEADS ? 4 : 4 * W);
  if ((int)blockIdx.x >= n_ctas || units == 0) {
    if (tid == 0) desc[blockIdx.x] = DdDesc{0, 0, 0, 0};
    return;
  }
  const int64_t u0 = dd_begin(units, n_ctas, blockIdx.x), u1 = dd_begin(units, n_ctas, blockIdx.x + 1);

  // ---- the first piece ----
  auto row_units = [&](const DdCursor& c) -> int { return c.span.steps; };
  DdCursor cur;
  {
    int lo = 0, hi = seqs;       // the last sequence with pre[s] * vheads <= u0 (sequences without steps are passed over)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if ((int64_t)pre[mid] * vheads <= u0) lo = mid; else hi = mid;
    }
    cur.s = lo;
    cur.span = dd_span<KS>(a, seqs0 + lo);
    const int64_t in_seq = u0 - (int64_t)pre[lo] * vheads;
    cur.vh = (int)(in_seq / cur.span.steps);
    cur.t = (int)(in_seq - (int64_t)cur.vh * cur.span.steps);
    const int64_t rest = u1 - u0;
    cur.t_end = cur.t + (int)(rest < row_units(cur) - cur.t ? rest : row_units(cur) - cur.t);
    cur.left = rest - (cur.t_end - cur.t);
  }
  // next piece of the range; false at its end
  auto next_piece = [&](DdCursor& c) -> bool {
    if (c.left <= 0) return false;
    if (++c.vh == vheads) {
      c.vh = 0;
      do { ++c.s; } while (pre[c.s + 1] == pre[c.s]);      // left > 0: there is one with steps
      c.span = dd_span<KS>(a, seqs0 + c.s);
    }
    c.t = 0;
    c.t_end = (int)(c.left < row_units(c) ? c.left : row_units(c));
    c.left -= c.t_end;
    return true;
  };

  const uint32_t ring = smem_u32(dd_smem) + (uint32_t)(warp * L::RING);
  const char* kbase = reinterpret_cast<const char*>(a.k);
  const char* vbase = reinterpret_cast<const char*>(a.v);
  const int group = a.num_q_heads / a.num_kv_heads, per_kv = rows / a.num_kv_heads;
  auto row_of = [&](int vh) -> int { return HEADS ? 4 * vh + warp : vh; };

  // ---- producer side: this warp's next step to copy ----
  DdCursor ld = cur;
  bool more = true;
  ld.t += HEADS ? 0 : warp;
  auto settle = [&]() {         // move on to the piece that holds a step for this warp
    while (more && ld.t >= ld.t_end) {
      more = next_piece(ld);
      ld.t += HEADS ? 0 : warp;
    }
  };
  settle();
  constexpr int KB = KS / 16;
  int64_t entry[KB];            // blocks of the step to copy, read one step ahead
  auto fetch_entry = [&]() {
    if (PAGE16 && more)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) entry[kb] = dense_block(a, seqs0 + ld.s, ((ld.span.first + ld.t) * KS + 16 * kb) / a.block_size);
  };
  fetch_entry();
  int stage_ld = 0;
  const int my_c = lane % CPR, my_r = lane / CPR;
  auto issue = [&]() {
    if (more) {
      const int key0 = (ld.span.first + ld.t) * KS;
      const int kvh = row_of(ld.vh) / per_kv;
      const uint32_t dk = ring + (uint32_t)(stage_ld * 2 * L::STEP), dv = dk + L::STEP;
      const char *kp = nullptr, *vp = nullptr;
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        const int r = my_r + i * RPP, key = key0 + r;
        const uint32_t bytes = key >= ld.span.lo && key < ld.span.len ? 16u : 0u;
        const uint32_t off = (uint32_t)(r * (D * 2) + ((my_c ^ (r & 7)) << 4));
        if (!PAGE16 || i * RPP % 16 == 0) {      // a new block may begin
          const int64_t blk = PAGE16 ? entry[i * RPP / 16] : dense_block(a, seqs0 + ld.s, key / a.block_size);
          const int pos = PAGE16 ? (key0 + i * RPP) % a.block_size + my_r : key % a.block_size;
          kp = kbase + 2 * (blk * a.k_sb + (int64_t)pos * a.k_sp + (int64_t)kvh * a.k_sh + my_c * 8);
          vp = vbase + 2 * (blk * a.v_sb + (int64_t)pos * a.v_sp + (int64_t)kvh * a.v_sh + my_c * 8);
        }
        dd_cp16(dk + off, kp, bytes);
        dd_cp16(dv + off, vp, bytes);
        if (PAGE16) { kp += 2 * RPP * a.k_sp; vp += 2 * RPP * a.v_sp; }
      }
      ld.t += HEADS ? 1 : W;
      settle();
      fetch_entry();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    stage_ld = stage_ld == NS - 1 ? 0 : stage_ld + 1;
  };
#pragma unroll 1
  for (int i = 0; i < NS - 1; ++i) issue();

  // ---- consumer side ----
  const int g = lane >> 2, tq = lane & 3;
  float* s_o = reinterpret_cast<float*>(dd_smem + L::O);
  float* s_ml = reinterpret_cast<float*>(dd_smem + L::ML);
  int stage = 0, parity = 0;
  bool first_piece = true;
  bool have = true;
  while (have) {
    const int row = row_of(cur.vh), kvh = row / per_kv, h0 = (row - kvh * per_kv) * H;      // first head of the row inside its group
    const int n_heads = group - h0 < H ? group - h0 : H;
    uint32_t qb[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + g;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + (int64_t)(seqs0 + cur.s) * a.q_st +
                           (int64_t)(kvh * group + h0 + (h < n_heads ? h : 0)) * a.q_sh + 2 * tq;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qb[nt][kk][0] = h < n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * kk) : 0u;
        qb[nt][kk][1] = h < n_heads ? *reinterpret_cast<const uint32_t*>(qp + 16 * kk + 8) : 0u;
      }
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }
    const int piece_t0 = cur.t;
#pragma unroll 1
    for (int t = cur.t + (HEADS ? 0 : warp); t < cur.t_end; t += HEADS ? 1 : W) {
      asm volatile("cp.async.wait_group %0;" :: "n"(NS - 2) : "memory");
      __syncwarp();
      issue();                  // into the stage that the previous step has left
      const uint32_t sk = ring + (uint32_t)(stage * 2 * L::STEP), sv = sk + L::STEP;
      stage = stage == NS - 1 ? 0 : stage + 1;
      float c[KB][NT][4];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[kb][nt][0] = c[kb][nt][1] = c[kb][nt][2] = c[kb][nt][3] = 0.f;
      {
        const int r = (lane & 7) + ((lane >> 3) & 1) * 8, ch = lane >> 4;
        const uint32_t row = sk + (uint32_t)(r * (D * 2));
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            uint32_t ka[4];
            dd_ldm4(row + (uint32_t)(kb * 16 * D * 2 + (((2 * kk + ch) ^ (r & 7)) << 4)), ka);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) dd_mma<BF>(c[kb][nt], ka, qb[nt][kk][0], qb[nt][kk][1]);
          }
      }
      const int key0 = (cur.span.first + t) * KS;
      const bool edge = key0 < cur.span.lo || key0 + KS > cur.span.len;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = -CUDART_INF_F;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            c[kb][nt][i] *= a.scale_log2;
            const int key = key0 + kb * 16 + g + (i >> 1) * 8;
            if (edge && (key < cur.span.lo || key >= cur.span.len)) c[kb][nt][i] = -CUDART_INF_F;
            top[nt][i & 1] = fmaxf(top[nt][i & 1], c[kb][nt][i]);
          }
      }
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) grow = grow || top[nt][0] > m[nt][0] + DENSE_TOP<BF> || top[nt][1] > m[nt][1] + DENSE_TOP<BF>;
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float mx = top[nt][x];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            mx -= DENSE_SHIFT<BF>;
            if (mx > m[nt][x]) {
              const float f = dense_ex2(m[nt][x] - mx);      // -inf before the first key: 0
              m[nt][x] = mx;
              l[nt][x] *= f;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) { o[nt][i][x] *= f; o[nt][i][x + 2] *= f; }
            }
          }
      }
      uint32_t pb[KB][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m[nt][0] == -CUDART_INF_F ? 0.f : m[nt][0], m1 = m[nt][1] == -CUDART_INF_F ? 0.f : m[nt][1];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const float p0 = dense_ex2(c[kb][nt][0] - m0), p1 = dense_ex2(c[kb][nt][1] - m1);
          const float p2 = dense_ex2(c[kb][nt][2] - m0), p3 = dense_ex2(c[kb][nt][3] - m1);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pb[kb][nt][0] = dd_movm(dense_pack<BF>(p0, p1));
          pb[kb][nt][1] = dd_movm(dense_pack<BF>(p2, p3));
        }
      }
      {
        const int r = (lane & 7) + (lane >> 4) * 8, ch = (lane >> 3) & 1;
        const uint32_t row = sv + (uint32_t)(r * (D * 2));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t va[4];
            dd_ldm4t(row + (uint32_t)(kb * 16 * D * 2 + (((2 * i + ch) ^ (r & 7)) << 4)), va);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) dd_mma<BF>(o[nt][i], va, pb[kb][nt][0], pb[kb][nt][1]);
          }
      }
    }

    const bool whole = piece_t0 == 0 && cur.t_end == cur.span.steps;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], d);
    if constexpr (HEADS) {
      // the row is this warp's alone
      const int64_t part = (((int64_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * 4 + warp) * H;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int h = nt * 8 + 2 * tq + x;
          if (h < n_heads) {
            const float inv = l[nt][x] == 0.f ? 0.f : 1.f / l[nt][x];
            const int64_t dst = (int64_t)(seqs0 + cur.s) * a.out_st + (int64_t)(kvh * group + h0 + h) * a.out_sh + g;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              if (whole) {
                dense_store<BF>(a.out, dst + 16 * i, l[nt][x] == 0.f ? 0.f : o[nt][i][x] * inv);
                dense_store<BF>(a.out, dst + 16 * i + 8, l[nt][x] == 0.f ? 0.f : o[nt][i][x + 2] * inv);
              } else {
                part_acc[(part + h) * D + g + 16 * i] = o[nt][i][x];
                part_acc[(part + h) * D + g + 16 * i + 8] = o[nt][i][x + 2];
              }
            }
            if (!whole && g == 0) reinterpret_cast<float2*>(part_ml)[part + h] = make_float2(m[nt][x], l[nt][x]);
          }
        }
    } else {
      // ---- join the warps' results in a fixed order ----
      float* ml = s_ml + parity * W * H * 2;
      parity ^= 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (g == 0) {
            const int h = nt * 8 + 2 * tq + x;
            ml[(warp * H + h) * 2] = m[nt][x];
            ml[(warp * H + h) * 2 + 1] = l[nt][x];
          }
        }
      __syncthreads();            // also: everybody has read the join buffer of the previous piece
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int h = nt * 8 + 2 * tq + x;
          float top = -CUDART_INF_F;
#pragma unroll
          for (int w = 0; w < W; ++w) top = fmaxf(top, ml[(w * H + h) * 2]);
          const float f = m[nt][x] == -CUDART_INF_F ? 0.f : dense_ex2(m[nt][x] - top);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) { o[nt][i][x] *= f; o[nt][i][x + 2] *= f; }
        }
      auto put = [&](int slot, bool add) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float* dst = s_o + (slot * H + nt * 8 + 2 * tq + x) * L::OROW + g;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              float v0 = o[nt][i][x], v1 = o[nt][i][x + 2];
              if (add) { v0 += dst[16 * i]; v1 += dst[16 * i + 8]; }
              dst[16 * i] = v0;
              dst[16 * i + 8] = v1;
            }
          }
      };
      if (warp >= W / 2) put(warp - W / 2, false);
      __syncthreads();
      if (warp < W / 2) put(warp, true);
      __syncthreads();
      const int64_t part = ((int64_t)blockIdx.x * 2 + (first_piece ? 0 : 1)) * H;
      for (int e = tid; e < n_heads * D; e += L::THREADS) {
        const int h = e / D, d = e - h * D;
        float top = -CUDART_INF_F, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, ml[(w * H + h) * 2]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float mw = ml[(w * H + h) * 2];
          sum += ml[(w * H + h) * 2 + 1] * (mw == -CUDART_INF_F ? 1.f : dense_ex2(mw - top));      // no keys: 0, or a NaN to pass on
        }
#pragma unroll
        for (int w = 0; w < W / 2; ++w) acc += s_o[(w * H + h) * L::OROW + d];
        if (whole) {
          dense_store<BF>(a.out, (int64_t)(seqs0 + cur.s) * a.out_st + (int64_t)(kvh * group + h0 + h) * a.out_sh + d,
                          sum == 0.f ? 0.f : acc / sum);
        } else {
          part_acc[(part + h) * D + d] = acc;
          if (d == 0) reinterpret_cast<float2*>(part_ml)[part + h] = make_float2(top, sum);
        }
      }
    }
    if (cur.left <= 0 && tid == 0) {          // the last piece: a row that begins here and ends in another CTA's range?
      DdDesc d{0, 0, 0, 0};
      if (piece_t0 == 0 && cur.t_end < cur.span.steps) {
        const int64_t end = u1 - cur.t_end + cur.span.steps;      // the row's last unit is end - 1
        d.parts = (int)((end * n_ctas - 1) / units) - (int)blockIdx.x + 1;
        d.slot0 = first_piece ? 0 : 1;
        d.s = seqs0 + cur.s;
        d.vh = cur.vh;
      }
      desc[blockIdx.x] = d;
    }
    first_piece = false;
    have = next_piece(cur);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Rows whose steps fell into several CTAs' ranges: out = sum_p 2^(m_p - M) acc_p / sum_p 2^(m_p - M) l_p, parts in the
// order of the keys.  A warp takes one query head of one such row.  What it costs is latency: one block per SM (starting a
// block takes some 10 ns), every warp with a CTA of its own to look after, and the reads of eight parts, their maxima and
// sums among them, on their way together (the maximum runs along; parts in groups of eight are enough for most rows).
constexpr int DM_THREADS = 1024;
template <bool BF, int D, int NT>
__global__ void __launch_bounds__(DM_THREADS)
dense_decode_merge_kernel(DenseArgs a, int rows, int per, int ctas, const float* part_acc, const float* part_ml, const DdDesc* desc) {
  constexpr int H = 8 * NT, V = D / 64;      // V pairs of columns per lane
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.num_q_heads / a.num_kv_heads, per_kv = rows / a.num_kv_heads;
  const int heads = group < H ? group : H, mine = (ctas - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
  for (int job = warp; job < mine * per * heads; job += DM_THREADS / 32) {
    const int c = blockIdx.x + job / (per * heads) * gridDim.x, y = job / heads % per, h = job % heads;
    const DdDesc d = desc[c];
    if (d.parts < 2) continue;
    const int row = d.vh * per + y, kvh = row / per_kv, h0 = (row - kvh * per_kv) * H;
    if (h >= group - h0) continue;
    // later parts begin where their CTA's range begins
    auto at = [&](int i) -> int64_t { return (((int64_t)(c + i) * 2 + (i == 0 ? d.slot0 : 0)) * per + y) * H + h; };
    float top = -CUDART_INF_F, sum = 0.f;
    float2 acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = make_float2(0.f, 0.f);
    constexpr int B = D == 256 ? 4 : 8;
    for (int base = 0; base < d.parts; base += B) {
      float2 ml[B], v[B][V];
#pragma unroll
      for (int p = 0; p < B; ++p) {
        const bool there = base + p < d.parts;
        ml[p] = there ? reinterpret_cast<const float2*>(part_ml)[at(base + p)] : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[p][i] = there ? reinterpret_cast<const float2*>(part_acc + at(base + p) * D)[lane + 32 * i] : make_float2(0.f, 0.f);
      }
      float t = top;
#pragma unroll
      for (int p = 0; p < B; ++p) t = fmaxf(t, ml[p].x);
      const float f0 = top == -CUDART_INF_F ? 0.f : dense_ex2(top - t);
      sum *= f0;
#pragma unroll
      for (int i = 0; i < V; ++i) { acc[i].x *= f0; acc[i].y *= f0; }
      top = t;
#pragma unroll
      for (int p = 0; p < B; ++p) {
        const float f = ml[p].x == -CUDART_INF_F ? 0.f : dense_ex2(ml[p].x - t);
        sum += f * ml[p].y;
#pragma unroll
        for (int i = 0; i < V; ++i) { acc[i].x += f * v[p][i].x; acc[i].y += f * v[p][i].y; }
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + (int64_t)d.s * a.out_st + (int64_t)(kvh * group + h0 + h) * a.out_sh) + lane;
#pragma unroll
    for (int i = 0; i < V; ++i) dst[32 * i] = dense_pack<BF>(acc[i].x * inv, acc[i].y * inv);
  }
}

template <bool BF, int D, int NT>
int dd_launch(const DenseArgs& a, float* part_acc, float* part_ml, DdDesc* desc, cudaStream_t st) {
  using L = DdL<D, NT>;
  const int group = a.num_q_heads / a.num_kv_heads;
  const int vheads = a.num_kv_heads * ((group + L::H - 1) / L::H), grid = L::CTAS * sm_count();
  const bool page16 = a.block_size % 16 == 0;
  // head_dim 64: four rows side by side, a warp each, where a sequence's rows come in fours.  Neighbouring heads of a key are
  // then read at the same time; its 128-byte pieces alone reach half of the HBM rate (200 windowed sequences x 8 heads: 93 us
  // with the keys shared out among the warps, 70 us this way).  At head_dim 128 it gains nothing: 16 sequences of 6 K to 32 K tokens
  // (32 / 8 heads) take 203 to 206 us both ways.
  const bool heads = D == 64 && vheads % 4 == 0;
  auto kernel = page16 ? dense_decode_kernel<BF, D, NT, true, false> : dense_decode_kernel<BF, D, NT, false, false>;
  if constexpr (D == 64)
    if (heads) kernel = page16 ? dense_decode_kernel<BF, D, NT, true, true> : dense_decode_kernel<BF, D, NT, false, true>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
  if (e != cudaSuccess) return fail((int)e, "dense attention: smem attribute: %s", cudaGetErrorString(e));
  // sequences of one launch: prefix sums in shared memory, and of fewer than 2^31 steps even if every sequence were full
  const int64_t full = ((int64_t)a.max_blocks_per_seq * a.block_size + L::KS - 1) / L::KS;
  int most = DD_MAX_SEQS;
  if (full * most > 0x7fffffffll) most = (int)(0x7fffffffll / full);
  for (int s0 = 0; s0 < a.num_seqs; s0 += most) {
    const int seqs = a.num_seqs - s0 < most ? a.num_seqs - s0 : most;
    kernel<<<grid, L::THREADS, L::SMEM, st>>>(a, s0, seqs, vheads, part_acc, part_ml, desc);
    if (int rc = check_launch("dense_decode_attn_kernel")) return rc;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)sm_count());
    cfg.blockDim = dim3(DM_THREADS);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, dense_decode_merge_kernel<BF, D, NT>, a, vheads, heads ? 4 : 1, grid, (const float*)part_acc, (const float*)part_ml, (const DdDesc*)desc);
    if (e != cudaSuccess) return fail((int)e, "dense attention merge: %s", cudaGetErrorString(e));
    if (int rc = check_launch("dense_decode_merge_kernel")) return rc;
  }
  return AKV_OK;
}

template <bool BF>
int dd_dispatch(const DenseArgs& a, float* part_acc, float* part_ml, DdDesc* desc, cudaStream_t st) {
  const bool one = a.num_q_heads / a.num_kv_heads <= 8;
  if (a.head_dim == 64) return one ? dd_launch<BF, 64, 1>(a, part_acc, part_ml, desc, st) : dd_launch<BF, 64, 2>(a, part_acc, part_ml, desc, st);
  if (a.head_dim == 128) return one ? dd_launch<BF, 128, 1>(a, part_acc, part_ml, desc, st) : dd_launch<BF, 128, 2>(a, part_acc, part_ml, desc, st);
  return one ? dd_launch<BF, 256, 1>(a, part_acc, part_ml, desc, st) : dd_launch<BF, 256, 2>(a, part_acc, part_ml, desc, st);
}

size_t dd_desc_bytes() { return ((size_t)sm_count() * 2 * sizeof(DdDesc) + 255) / 256 * 256; }

}  // namespace

int dense_common(const akv_dense_attn_params* p, const char* who, DenseArgs* a) {
  if (!p) return fail(AKV_ERR_ARG, "%s: null params", who);
  if (p->num_seqs < 0 || p->num_tokens < 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->block_size <= 0 ||
      p->max_blocks_per_seq < 0 || p->num_blocks < 0 || p->num_q_heads % p->num_kv_heads)
    return fail(AKV_ERR_ARG, "%s: %d sequences, %d tokens, %d / %d heads, %d blocks of %d per sequence, %lld blocks", who,
                p->num_seqs, p->num_tokens, p->num_q_heads, p->num_kv_heads, p->max_blocks_per_seq, p->block_size, (long long)p->num_blocks);
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return fail(AKV_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", who, p->head_dim);
  if (p->dtype != AKV_F16 && p->dtype != AKV_BF16) return fail(AKV_ERR_UNSUPPORTED, "%s: element type %d (fp16 or bf16)", who, p->dtype);
  if (p->window < 0) return fail(AKV_ERR_ARG, "%s: window %d", who, p->window);
  if ((int64_t)p->max_blocks_per_seq * p->block_size > 0x7fffff00ll)
    return fail(AKV_ERR_UNSUPPORTED, "%s: %d blocks of %d per sequence pass 2^31 keys", who, p->max_blocks_per_seq, p->block_size);
  if ((p->bt_dtype | p->sl_dtype | p->qs_dtype) & ~1) return fail(AKV_ERR_ARG, "%s: unknown index type", who);
  if (!(p->scale > 0.f && p->scale <= 1.0e38f)) return fail(AKV_ERR_ARG, "%s: scale %g (positive and finite)", who, (double)p->scale);
  if (p->num_tokens > 0 && p->num_seqs > 0) {
    if (!p->query || !p->out || !p->seq_lens) return fail(AKV_ERR_ARG, "%s: null query, out or lengths", who);
    if (p->max_blocks_per_seq > 0 && (!p->block_tables || !p->k_cache || !p->v_cache || p->num_blocks == 0))
      return fail(AKV_ERR_ARG, "%s: null block tables or caches, or a cache without blocks", who);
  }
  // the stride of a dimension of one element is never used
  auto used = [](int64_t stride, int64_t n) -> int64_t { return n > 1 ? stride : 0; };
  const int64_t caches = used(p->k_stride_blk | p->v_stride_blk, p->num_blocks) | used(p->k_stride_pos | p->v_stride_pos, p->block_size) |
                         used(p->k_stride_head | p->v_stride_head, p->num_kv_heads);
  if ((((uintptr_t)p->k_cache | (uintptr_t)p->v_cache) & 15) || (caches & 7))
    return fail(AKV_ERR_ARG, "%s: cache rows must start on 16-byte boundaries", who);
  const int64_t rows = used(p->q_stride_tok | p->out_stride_tok, p->num_tokens) | used(p->q_stride_head | p->out_stride_head, p->num_q_heads);
  if ((((uintptr_t)p->query | (uintptr_t)p->out) & 15) || (rows & 7))
    return fail(AKV_ERR_ARG, "%s: query and output rows must start on 16-byte boundaries", who);
  *a = DenseArgs{};
  a->q = p->query; a->q_st = p->q_stride_tok; a->q_sh = p->q_stride_head;
  a->k = p->k_cache; a->k_sb = p->k_stride_blk; a->k_sp = p->k_stride_pos; a->k_sh = p->k_stride_head;
  a->v = p->v_cache; a->v_sb = p->v_stride_blk; a->v_sp = p->v_stride_pos; a->v_sh = p->v_stride_head;
  a->block_tables = p->block_tables; a->bt_dtype = p->bt_dtype; a->bt_stride = p->bt_stride_seq;
  a->seq_lens = p->seq_lens; a->sl_dtype = p->sl_dtype;
  a->starts = p->query_start_loc; a->qs_dtype = p->qs_dtype;
  a->num_seqs = p->num_seqs; a->n_tokens = p->num_tokens;
  a->num_q_heads = p->num_q_heads; a->num_kv_heads = p->num_kv_heads; a->head_dim = p->head_dim;
  a->block_size = p->block_size; a->max_blocks_per_seq = p->max_blocks_per_seq; a->num_blocks = p->num_blocks;
  a->scale_log2 = p->scale * 1.4426950408889634f;
  // one that no sequence fills is none (and positions minus the window stay above -2^31)
  a->window = p->window >= (int64_t)p->max_blocks_per_seq * p->block_size ? 0 : p->window;
  a->out = p->out; a->out_st = p->out_stride_tok; a->out_sh = p->out_stride_head;
  return AKV_OK;
}

}  // namespace akv

// Two times up to four partial rows for each of up to two CTAs per SM, and what the merge has to know.
AKV_EXPORT size_t akv_dense_paged_attn_workspace_bytes(int num_q_heads, int num_kv_heads, int head_dim) {
  if (num_kv_heads <= 0 || num_q_heads < num_kv_heads || head_dim <= 0) return 0;
  const int heads = num_q_heads / num_kv_heads <= 8 ? 8 : 16;
  return akv::dd_desc_bytes() + (size_t)akv::sm_count() * 16 * heads * (head_dim + 2) * sizeof(float);
}

AKV_EXPORT int akv_dense_paged_attn(const akv_dense_attn_params* p) {
  akv::DenseArgs a;
  if (int rc = akv::dense_common(p, "akv_dense_paged_attn", &a)) return rc;
  if (a.num_seqs == 0) return AKV_OK;
  if (a.n_tokens < a.num_seqs)
    return akv::fail(AKV_ERR_ARG, "akv_dense_paged_attn: %d query rows for %d sequences", a.n_tokens, a.num_seqs);
  const size_t need = akv_dense_paged_attn_workspace_bytes(a.num_q_heads, a.num_kv_heads, a.head_dim);
  if (!p->workspace || p->workspace_bytes < need || ((uintptr_t)p->workspace & 15))
    return akv::fail(AKV_ERR_WORKSPACE, "akv_dense_paged_attn: workspace of %zu bytes (16-byte aligned) needed, got %zu", need, p->workspace_bytes);
  akv::DdDesc* desc = reinterpret_cast<akv::DdDesc*>(p->workspace);
  float* part_acc = reinterpret_cast<float*>(static_cast<char*>(p->workspace) + akv::dd_desc_bytes());
  float* part_ml = part_acc + (size_t)akv::sm_count() * 16 * (a.num_q_heads / a.num_kv_heads <= 8 ? 8 : 16) * a.head_dim;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(p->stream);
  return p->dtype == AKV_BF16 ? akv::dd_dispatch<true>(a, part_acc, part_ml, desc, st) : akv::dd_dispatch<false>(a, part_acc, part_ml, desc, st);
}
