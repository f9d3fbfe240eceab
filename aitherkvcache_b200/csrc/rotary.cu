// Rotary positions with one or several axes, and the append of keys and values to a dense paged cache with that
// rotation on the way.
//
// Pair p of a vector - elements (p, p + R/2), or (2p, 2p + 1) with adjacent pairs, R = rotary_dim - turns by the angle
// a = pos[axis(p)] * f(p):  y0 = s (x0 cos a - x1 sin a),  y1 = s (x1 cos a + x0 sin a);  inverse: a -> -a.  Elements
// R .. head_dim - 1 pass through.
//
// Angles.  A float32 product pos * f(p) is wrong by 2^-24 of its value: 0.06 rad at position 10^6.  Here the frequency
// is a 64-bit fraction of a turn, step(p) = f(p) / 2 pi * 2^64 modulo 2^64, and pos * step(p) modulo 2^64 is the angle
// modulo a full turn with nothing rounded (the integer product wraps exactly where the angle does; positions may be
// negative).  Its upper 32 bits, as a signed fraction of a turn, go to float32 (2^-25 of half a turn) and sincospif.
// No table of cosines is read: 4 bytes per pair and axis step instead of 8 per pair and position.
//
// Bound by HBM: every vector is read once and written once.  A block takes a few tokens: first every thread works out the
// cosine and sine of about one (token, pair) - a sincospif is some 40 instructions, so each is done once and not once per
// head - into shared memory, while its first loads are under way; then the block streams through the heads, a thread 16
// elements of a row at a time (8 pairs, two 16-byte loads for 16-bit types), the 8 threads of a 128-element row next to
// each other.  That phase needs few registers, so enough loads are in flight.
// Measured (inside a graph): 32768 tokens of 32 + 8 + 8 heads of 128, fp16, into the cache, 806 MB in 134 us, 6.0 TB/s, 92 % of
// the measured copy bandwidth; 8192 tokens of 32 + 8 heads with three axes, 168 MB in 32.4 us, 5.2 TB/s; 4099 tokens of 9 + 3
// heads of 96 float32, adjacent pairs, 38 MB in 10.5 us; 16 tokens 2.3 us, with the append 3.1.  With the angles worked out
// again for every head the first two took 225 and 67 us; with blocks of 256 threads 144 and 33.6, of 64 threads 138 and 32.4,
// with one couple per thread 141 and 32.6; with loads that pass L1 by 136 and 32.5, the third 11.3 (its sectors are read in halves).
#include "common.cuh"

// Mirrors of akv_rotary_tables, akv_rotary_params and akv_rotary_append_params in include/akv_b200.h.
struct akv_rotary_tables {
  int head_dim, rotary_dim, num_axes, adjacent;
  const uint64_t* steps; const int* axes;
  float scaling;
};
struct akv_rotary_params {
  const akv_rotary_tables* tables;
  const void* positions; int pos_dtype; int64_t pos_stride_axis, pos_stride_tok;
  int64_t num_tokens;
  int in_dtype, out_dtype;
  const void* query; int64_t q_stride_tok, q_stride_head; int num_q_heads;
  void* q_out; int64_t qo_stride_tok, qo_stride_head;
  const void* key; int64_t k_stride_tok, k_stride_head; int num_kv_heads;
  void* k_out; int64_t ko_stride_tok, ko_stride_head;
  int inverse;
  void* stream;
};
struct akv_rotary_append_params {
  akv_rotary_params rotary;
  const void* value; int64_t v_stride_tok, v_stride_head;
  const void* slot_mapping; int slot_dtype;
  void* k_cache; int64_t kc_stride_blk, kc_stride_pos, kc_stride_head;
  void* v_cache; int64_t vc_stride_blk, vc_stride_pos, vc_stride_head;
  int block_size; int64_t num_blocks;
};

namespace akv {
namespace {

constexpr int ROT_THREADS = 128;
constexpr int ROT_MAX_AXES = 4;

struct RotArgs {
  const unsigned long long* steps;
  const int* axes;
  int D, R, num_axes, adjacent, inverse;
  float scaling;
  const void* positions; int pos_dtype; int64_t pos_sa, pos_st;
  int64_t tokens;
  int in_dtype, out_dtype;
  const void* q; int64_t q_st, q_sh; int qh; void* qo; int64_t qo_st, qo_sh;
  const void* k; int64_t k_st, k_sh; int kh; void* ko; int64_t ko_st, ko_sh;      // ko null: into the cache
  // append
  const void* v; int64_t v_st, v_sh; int vh;
  const void* slots; int slot_dtype;
  void* kc; int64_t kc_sb, kc_sp, kc_sh;
  void* vc; int64_t vc_sb, vc_sp, vc_sh;
  int block_size; int64_t num_blocks;
  int heads, tb, slice;                                                          // qh + kh + vh; tokens and heads of a block
};

// cos and sin of pos * step turns (2^64 steps to a turn), times the scaling
__device__ __forceinline__ void rot_cs(int64_t pos, unsigned long long step, const RotArgs& a, float& c, float& s) {
  const unsigned long long turn = (unsigned long long)pos * step;
  sincospif((float)(int)(turn >> 32) * 4.656612873077393e-10f /* 2^-31: half turns */, &s, &c);
  if (a.inverse) s = -s;
  c *= a.scaling;
  s *= a.scaling;
}

// eight elements as they lie in memory, and as floats
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw8<T> rot_load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.w[i].x), "=r"(r.w[i].y), "=r"(r.w[i].z), "=r"(r.w[i].w) : "l"(reinterpret_cast<const uint4*>(p) + i));
  return r;
}
template <typename T> __device__ __forceinline__ void rot_floats(const Raw8<T>& r, float (&f)[8]);
template <> __device__ __forceinline__ void rot_floats<__half>(const Raw8<__half>& r, float (&f)[8]) {
  const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
    f[2 * i] = t.x; f[2 * i + 1] = t.y;
  }
}
template <> __device__ __forceinline__ void rot_floats<__nv_bfloat16>(const Raw8<__nv_bfloat16>& r, float (&f)[8]) {
  const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
template <> __device__ __forceinline__ void rot_floats<float>(const Raw8<float>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f[4 * i] = __uint_as_float(r.w[i].x); f[4 * i + 1] = __uint_as_float(r.w[i].y);
    f[4 * i + 2] = __uint_as_float(r.w[i].z); f[4 * i + 3] = __uint_as_float(r.w[i].w);
  }
}
template <typename T> __device__ __forceinline__ void rot_store8(T* p, const float (&f)[8]);
template <> __device__ __forceinline__ void rot_store8<__half>(__half* p, const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); u[i] = *reinterpret_cast<const uint32_t*>(&h); }
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
template <> __device__ __forceinline__ void rot_store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&f)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); u[i] = *reinterpret_cast<const uint32_t*>(&h); }
  *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
template <> __device__ __forceinline__ void rot_store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// Where head h of token t is read and written; false: the token has no slot.  h counts queries, then keys, then values.
template <typename TI, typename TO>
__device__ __forceinline__ bool rot_row(const RotArgs& a, int64_t t, int h, int64_t blk, int64_t in_blk, const TI*& src, TO*& dst) {
  if (h < a.qh) {
    src = reinterpret_cast<const TI*>(a.q) + t * a.q_st + h * a.q_sh;
    dst = reinterpret_cast<TO*>(a.qo) + t * a.qo_st + h * a.qo_sh;
    return true;
  }
  h -= a.qh;
  if (h < a.kh) {
    src = reinterpret_cast<const TI*>(a.k) + t * a.k_st + h * a.k_sh;
    if (a.ko != nullptr) { dst = reinterpret_cast<TO*>(a.ko) + t * a.ko_st + h * a.ko_sh; return true; }
    dst = reinterpret_cast<TO*>(a.kc) + blk * a.kc_sb + in_blk * a.kc_sp + h * a.kc_sh;
    return blk >= 0;
  }
  h -= a.kh;
  src = reinterpret_cast<const TI*>(a.v) + t * a.v_st + h * a.v_sh;
  dst = reinterpret_cast<TO*>(a.vc) + blk * a.vc_sb + in_blk * a.vc_sp + h * a.vc_sh;
  return blk >= 0;
}

// Block and position of token t's slot; block -1: none (negative, or behind the cache)
__device__ __forceinline__ void rot_slot(const RotArgs& a, int64_t t, int64_t& blk, int64_t& in_blk) {
  blk = -1;
  in_blk = 0;
  if (a.slots == nullptr) return;
  const int64_t slot = load_index(a.slots, a.slot_dtype, t);
  if (slot < 0) return;
  blk = slot / a.block_size;
  in_blk = slot - blk * a.block_size;
  if (blk >= a.num_blocks) blk = -1;
}

constexpr int ROT_MAX_PAIRS = 1024;      // (token, pair) couples of a block

template <typename TI, typename TO>
__global__ void __launch_bounds__(ROT_THREADS, sizeof(TI) == 4 ? 6 : 8)
rotary_rows_kernel(RotArgs a) {
  __shared__ __align__(16) float s_cos[ROT_MAX_PAIRS], s_sin[ROT_MAX_PAIRS];
  __shared__ int64_t s_blk[16];
  __shared__ int s_pos[16];
  const int units = a.D >> 4, runits = a.R >> 4, half = a.R >> 1;
  const int64_t t0 = (int64_t)blockIdx.x * a.tb;
  const int tb = a.tokens - t0 < a.tb ? (int)(a.tokens - t0) : a.tb;
  const int h_lo = blockIdx.y * a.slice, hs = a.heads - h_lo < a.slice ? a.heads - h_lo : a.slice;
  const int items = tb * hs * units;
  // item: (token, head, unit), units next to each other; a thread's next item is ROT_THREADS further on
  const int row_step = ROT_THREADS / units, u_step = ROT_THREADS - row_step * units, t_step = row_step / hs, h_step = row_step - t_step * hs;
  int tt, h, u, e0, e1;
  const TI* src;
  TO* dst;
  bool turned, there;
  auto spans = [&]() {
    turned = u < runits && h < a.qh + a.kh;
    e0 = u < runits ? (a.adjacent ? 16 * u : 8 * u) : 16 * u;
    e1 = u < runits && !a.adjacent ? half + 8 * u : e0 + 8;
  };
  Raw8<TI> r0, r1;
  int64_t blk, in_blk;
  int item = threadIdx.x;
  there = false;
  if (item < items) {
    const int row = item / units;
    u = item - row * units;
    tt = row / hs;
    h = h_lo + row - tt * hs;
    spans();
    rot_slot(a, t0 + tt, blk, in_blk);
    there = rot_row<TI, TO>(a, t0 + tt, h, blk, in_blk, src, dst);
    if (there) {
      r0 = rot_load8<TI>(src + e0);
      r1 = rot_load8<TI>(src + e1);
    }
  }
  if (threadIdx.x < tb) {
    int64_t b, p;
    rot_slot(a, t0 + threadIdx.x, b, p);
    s_blk[threadIdx.x] = b;
    s_pos[threadIdx.x] = (int)p;
  }
  if (h_lo < a.qh + a.kh)
    for (int x = threadIdx.x; x < tb * half; x += ROT_THREADS) {
      const int t = x / half, p = x - t * half;
      const int ax = a.num_axes > 1 ? a.axes[p] : 0;
      rot_cs(load_index(a.positions, a.pos_dtype, ax * a.pos_sa + (t0 + t) * a.pos_st), a.steps[p], a, s_cos[x], s_sin[x]);
    }
  __syncthreads();
#pragma unroll 1
  while (item < items) {
    float x0[8], x1[8];
    TO* d = dst;
    const int f0 = e0, f1 = e1, cs = tt * half + 8 * u;
    const bool turn = turned, store = there;
    if (there) {
      rot_floats<TI>(r0, x0);
      rot_floats<TI>(r1, x1);
    }
    item += ROT_THREADS;
    if (item < items) {                     // the next item's loads before this one's arithmetic
      u += u_step;
      tt += t_step;
      h += h_step;
      if (u >= units) { u -= units; ++h; }
      if (h >= h_lo + hs) { h -= hs; ++tt; }
      spans();
      there = rot_row<TI, TO>(a, t0 + tt, h, s_blk[tt], s_pos[tt], src, dst);
      if (there) {
        r0 = rot_load8<TI>(src + e0);
        r1 = rot_load8<TI>(src + e1);
      }
    }
    if (!store) continue;
    if (turn) {
      float c[8], s[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        reinterpret_cast<float4*>(c)[i] = reinterpret_cast<const float4*>(s_cos + cs)[i];
        reinterpret_cast<float4*>(s)[i] = reinterpret_cast<const float4*>(s_sin + cs)[i];
      }
      if (a.adjacent) {          // x0: pairs 0..3 of the unit, x1: pairs 4..7
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = x0[2 * i], q = x0[2 * i + 1], r = x1[2 * i], w = x1[2 * i + 1];
          x0[2 * i] = p * c[i] - q * s[i];
          x0[2 * i + 1] = q * c[i] + p * s[i];
          x1[2 * i] = r * c[4 + i] - w * s[4 + i];
          x1[2 * i + 1] = w * c[4 + i] + r * s[4 + i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float p = x0[i], q = x1[i];
          x0[i] = p * c[i] - q * s[i];
          x1[i] = q * c[i] + p * s[i];
        }
      }
    }
    rot_store8<TO>(d + f0, x0);
    rot_store8<TO>(d + f1, x1);
  }
}

// Any head_dim, any even rotary_dim, any alignment: a thread takes one pair, or one element behind the rotated part, of
// one head.
template <typename TI, typename TO>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_elements_kernel(RotArgs a) {
  const int half = a.R >> 1, per_row = half + (a.D - a.R);
  const uint32_t idx = blockIdx.x * ROT_THREADS + threadIdx.x;
  const uint32_t row = idx / (uint32_t)per_row;
  const int e = (int)(idx - row * per_row);
  const int64_t t = row / (uint32_t)a.heads;
  const int h = (int)(row - (uint32_t)t * a.heads);
  if (t >= a.tokens) return;
  int64_t blk, in_blk;
  rot_slot(a, t, blk, in_blk);
  const TI* src;
  TO* dst;
  if (!rot_row<TI, TO>(a, t, h, blk, in_blk, src, dst)) return;
  auto get = [&](int i) -> float { return load_as_float(src, a.in_dtype, i); };
  auto put = [&](int i, float v) { store_from_float(dst, a.out_dtype, i, v); };
  if (e >= half) {
    const int i = a.R + (e - half);
    put(i, get(i));
    return;
  }
  const int i0 = a.adjacent ? 2 * e : e, i1 = a.adjacent ? 2 * e + 1 : half + e;
  const float x0 = get(i0), x1 = get(i1);
  if (h >= a.qh + a.kh) { put(i0, x0); put(i1, x1); return; }
  float c, s;
  const int ax = a.num_axes > 1 ? a.axes[e] : 0;
  rot_cs(load_index(a.positions, a.pos_dtype, ax * a.pos_sa + t * a.pos_st), a.steps[e], a, c, s);
  put(i0, x0 * c - x1 * s);
  put(i1, x1 * c + x0 * s);
}

template <typename TI, typename TO>
int rot_launch(const RotArgs& a, bool rows16, dim3 grid, cudaStream_t st) {
  if (rows16) rotary_rows_kernel<TI, TO><<<grid, ROT_THREADS, 0, st>>>(a);
  else rotary_elements_kernel<TI, TO><<<grid, ROT_THREADS, 0, st>>>(a);
  return check_launch(rows16 ? "rotary_rows_kernel" : "rotary_elements_kernel");
}

template <typename TI>
int rot_launch_in(const RotArgs& a, bool rows16, dim3 grid, cudaStream_t st) {
  if (a.out_dtype == AKV_F16) return rot_launch<TI, __half>(a, rows16, grid, st);
  if (a.out_dtype == AKV_BF16) return rot_launch<TI, __nv_bfloat16>(a, rows16, grid, st);
  return rot_launch<TI, float>(a, rows16, grid, st);
}

int rot_run(RotArgs a, const char* who, cudaStream_t st) {
  // 16-byte accesses: every row of every operand starts on a 16-byte boundary, and the rotated part and the row are whole
  // units of 16 elements; and a token's pairs fit into a block's shared memory
  const int64_t in_mask = a.in_dtype == AKV_F32 ? 3 : 7, out_mask = a.out_dtype == AKV_F32 ? 3 : 7;
  const uintptr_t ptrs = (uintptr_t)a.q | (uintptr_t)a.qo | (uintptr_t)a.k | (uintptr_t)a.ko | (uintptr_t)a.v | (uintptr_t)a.kc | (uintptr_t)a.vc;
  const int64_t ins = a.q_st | a.q_sh | a.k_st | a.k_sh | a.v_st | a.v_sh;
  const int64_t outs = a.qo_st | a.qo_sh | a.ko_st | a.ko_sh | a.kc_sb | a.kc_sp | a.kc_sh | a.vc_sb | a.vc_sp | a.vc_sh;
  a.heads = a.qh + a.kh + a.vh;
  const bool rows16 = a.D % 16 == 0 && a.R % 16 == 0 && a.R / 2 <= ROT_MAX_PAIRS && (ptrs & 15) == 0 && (ins & in_mask) == 0 &&
                      (outs & out_mask) == 0 && (int64_t)a.heads * a.D < ((int64_t)1 << 26);
  const int per_token = a.R / 2 + (a.D - a.R);
  int64_t most;                 // tokens of one launch: grid and thread indices stay below 2^31
  if (rows16) {
    // two (token, pair) couples per thread; all heads of a token in one block where that gives every SM eight blocks, else
    // as many slices of heads as it takes, down to one item per thread (a decode step: latency)
    a.tb = a.R > 0 ? 2 * ROT_THREADS / (a.R / 2) : 4;
    if (a.tb < 1) a.tb = 1;
    if (a.tb > 16) a.tb = 16;
    const int64_t want = 8 * (int64_t)sm_count();
    if (a.tokens / want < a.tb) a.tb = a.tokens / want > 1 ? (int)(a.tokens / want) : 1;
    // between half and all of that, the number whose items fill the threads best: with blocks of 256 threads, 4099 tokens of
    // 12 x 96 float32 took 11.8 us six at a time (432 items, two rounds) and 14.0 four at a time (288, also two)
    double best = 0.0;
    for (int tb = a.tb, lo = (a.tb + 1) / 2; tb >= lo; --tb) {
      const int64_t items = (int64_t)tb * a.heads * (a.D / 16);
      const double fill = (double)items / (double)((items + ROT_THREADS - 1) / ROT_THREADS * ROT_THREADS);
      if (fill > best) { best = fill; a.tb = tb; }
    }
    const int64_t blocks = (a.tokens + a.tb - 1) / a.tb;
    int64_t slices = blocks >= want ? 1 : (want + blocks - 1) / blocks;
    const int64_t finest = ((int64_t)a.tb * a.heads * (a.D / 16) + ROT_THREADS - 1) / ROT_THREADS;      // one item per thread
    if (slices > finest) slices = finest;
    a.slice = (int)((a.heads + slices - 1) / slices);
    most = (int64_t)a.tb << 30;
  } else {
    most = ((int64_t)1 << 31) / ((int64_t)a.heads * per_token);
  }
  if (most < 1) return fail(AKV_ERR_ARG, "%s: %d heads of %d elements per token are too many", who, a.heads, a.D);
  const int isz = a.in_dtype == AKV_F32 ? 4 : 2, osz = a.out_dtype == AKV_F32 ? 4 : 2, ssz = a.slot_dtype == AKV_I64 ? 8 : 4, psz = a.pos_dtype == AKV_I64 ? 8 : 4;
  int64_t left = a.tokens;
  while (left > 0) {
    a.tokens = left < most ? left : most;
    const dim3 grid = rows16 ? dim3((unsigned)((a.tokens + a.tb - 1) / a.tb), (unsigned)((a.heads + a.slice - 1) / a.slice))
                             : dim3((unsigned)((a.tokens * a.heads * per_token + ROT_THREADS - 1) / ROT_THREADS));
    int rc;
    if (a.in_dtype == AKV_F16) rc = rot_launch_in<__half>(a, rows16, grid, st);
    else if (a.in_dtype == AKV_BF16) rc = rot_launch_in<__nv_bfloat16>(a, rows16, grid, st);
    else rc = rot_launch_in<float>(a, rows16, grid, st);
    if (rc) return rc;
    left -= a.tokens;
    if (left > 0) {
      auto step = [](const void* p, int64_t bytes) -> const void* { return p == nullptr ? p : static_cast<const char*>(p) + bytes; };
      a.q = step(a.q, a.tokens * a.q_st * isz);
      a.k = step(a.k, a.tokens * a.k_st * isz);
      a.v = step(a.v, a.tokens * a.v_st * isz);
      a.qo = const_cast<void*>(step(a.qo, a.tokens * a.qo_st * osz));
      a.ko = const_cast<void*>(step(a.ko, a.tokens * a.ko_st * osz));
      a.slots = step(a.slots, a.tokens * ssz);
      a.positions = step(a.positions, a.tokens * a.pos_st * psz);
    }
  }
  return AKV_OK;
}

bool float_type(int t) { return t == AKV_F16 || t == AKV_BF16 || t == AKV_F32; }
bool index_type(int t) { return t == AKV_I32 || t == AKV_I64; }

// Checks what both entry points share and fills the common part of the kernel arguments.
int rot_common(const akv_rotary_params* p, const char* who, RotArgs* a) {
  if (!p || !p->tables) return fail(AKV_ERR_ARG, "%s: null params or tables", who);
  const akv_rotary_tables* t = p->tables;
  if (t->head_dim <= 0 || t->rotary_dim < 0 || t->rotary_dim > t->head_dim || t->rotary_dim % 2)
    return fail(AKV_ERR_ARG, "%s: rotary_dim %d of head_dim %d (even, at most head_dim)", who, t->rotary_dim, t->head_dim);
  if (t->num_axes < 1 || t->num_axes > ROT_MAX_AXES) return fail(AKV_ERR_ARG, "%s: %d axes (1 to %d)", who, t->num_axes, ROT_MAX_AXES);
  if (t->rotary_dim > 0 && (!t->steps || (t->num_axes > 1 && !t->axes))) return fail(AKV_ERR_ARG, "%s: null table", who);
  if (p->num_tokens < 0 || p->num_q_heads < 0 || p->num_kv_heads < 0) return fail(AKV_ERR_ARG, "%s: negative size", who);
  if (!float_type(p->in_dtype) || !float_type(p->out_dtype)) return fail(AKV_ERR_ARG, "%s: unknown element type", who);
  if (!index_type(p->pos_dtype)) return fail(AKV_ERR_ARG, "%s: unknown index type", who);
  if (p->num_tokens > 0 && !p->positions && t->rotary_dim > 0) return fail(AKV_ERR_ARG, "%s: null positions", who);
  if (p->num_tokens > 0 && ((p->num_q_heads > 0 && (!p->query || !p->q_out)) || (p->num_kv_heads > 0 && !p->key)))
    return fail(AKV_ERR_ARG, "%s: null query, query output or key", who);
  *a = RotArgs{};
  a->steps = reinterpret_cast<const unsigned long long*>(t->steps);
  a->axes = t->axes;
  a->D = t->head_dim; a->R = t->rotary_dim; a->num_axes = t->num_axes; a->adjacent = t->adjacent != 0; a->inverse = p->inverse != 0;
  a->scaling = t->scaling;
  a->positions = p->positions; a->pos_dtype = p->pos_dtype; a->pos_sa = p->pos_stride_axis; a->pos_st = p->pos_stride_tok;
  a->tokens = p->num_tokens;
  a->in_dtype = p->in_dtype; a->out_dtype = p->out_dtype;
  a->q = p->query; a->q_st = p->q_stride_tok; a->q_sh = p->q_stride_head; a->qh = p->num_q_heads;
  a->qo = p->q_out; a->qo_st = p->qo_stride_tok; a->qo_sh = p->qo_stride_head;
  a->k = p->key; a->k_st = p->k_stride_tok; a->k_sh = p->k_stride_head; a->kh = p->num_kv_heads;
  return AKV_OK;
}

}  // namespace
}  // namespace akv

AKV_EXPORT int akv_rotary(const akv_rotary_params* p) {
  akv::RotArgs a;
  if (int rc = akv::rot_common(p, "akv_rotary", &a)) return rc;
  if (a.kh > 0 && a.tokens > 0 && !p->k_out) return akv::fail(AKV_ERR_ARG, "akv_rotary: null key output");
  a.ko = p->k_out; a.ko_st = p->ko_stride_tok; a.ko_sh = p->ko_stride_head;
  if (a.tokens == 0 || a.qh + a.kh == 0) return AKV_OK;
  return akv::rot_run(a, "akv_rotary", reinterpret_cast<cudaStream_t>(p->stream));
}

AKV_EXPORT int akv_rotary_kv_append(const akv_rotary_append_params* p) {
  if (!p) return akv::fail(AKV_ERR_ARG, "akv_rotary_kv_append: null params");
  akv::RotArgs a;
  if (int rc = akv::rot_common(&p->rotary, "akv_rotary_kv_append", &a)) return rc;
  if (!akv::index_type(p->slot_dtype)) return akv::fail(AKV_ERR_ARG, "akv_rotary_kv_append: unknown index type");
  if (p->block_size <= 0 || p->num_blocks < 0) return akv::fail(AKV_ERR_ARG, "akv_rotary_kv_append: %lld blocks of %d", (long long)p->num_blocks, p->block_size);
  if (a.tokens == 0 || a.qh + a.kh == 0) return AKV_OK;
  if (!p->slot_mapping || (a.kh > 0 && (!p->value || !p->k_cache || !p->v_cache)))
    return akv::fail(AKV_ERR_ARG, "akv_rotary_kv_append: null slots, value or cache");
  a.v = p->value; a.v_st = p->v_stride_tok; a.v_sh = p->v_stride_head; a.vh = a.kh;
  a.slots = p->slot_mapping; a.slot_dtype = p->slot_dtype;
  a.kc = p->k_cache; a.kc_sb = p->kc_stride_blk; a.kc_sp = p->kc_stride_pos; a.kc_sh = p->kc_stride_head;
  a.vc = p->v_cache; a.vc_sb = p->vc_stride_blk; a.vc_sp = p->vc_stride_pos; a.vc_sh = p->vc_stride_head;
  a.block_size = p->block_size; a.num_blocks = p->num_blocks;
  return akv::rot_run(a, "akv_rotary_kv_append", reinterpret_cast<cudaStream_t>(p->rotary.stream));
}
