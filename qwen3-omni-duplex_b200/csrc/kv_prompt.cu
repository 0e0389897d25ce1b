// Attention over the 8-bit paged KV cache for many query rows a sequence (prompts, chunks of them),
// on the tensor cores: the formulas of kv_attend.cu over 256 query rows and 128 tokens at a time.
//
// Bound by products: 4 dim flops per row and token.  A CTA holds 256 rows (the heads of a KV group
// are rows like any other) as two tiles of 128 in shared memory, and their scores and outputs in
// tensor memory: S0, S1 [128 x 128] fp32 and O0, O1 [128 x dim] fp32, all 512 columns at dim 128.
// The tiles take turns, so that one tile's softmax runs under the other's products:
//
//   warps 0-3, 4-7   softmax of tile 0, 1: a thread owns a row.  S from tensor memory, exp2, P back as
//                    fp16 into S's own columns (the next product's A operand)
//   warps 8-15       keys and values from the cache's codes to fp16 operands in shared memory, two buffers
//                    each: code times its block's scale over the sequence's largest.  That is exact for
//                    powers of two up to 2^14 apart.  Where a sequence has others, the operands are the
//                    codes themselves and the scales are factors in the softmax, in fp32: of the scores for
//                    keys, of the probabilities for values (over the largest scale that the row has seen,
//                    with which its O is rescaled like with the maximum).  So a row's result hangs on what
//                    the row sees, whatever the blocks that it does not.  Such a prompt of 8192: 1.7 times
//                    the time
//   warp 16          issues the products: S = Q K^T (both shared memory), O += P V
//
// The running maximum is a reference that may lag by 2^kSlack, so O is rescaled rarely.  The products of a
// tile's first 64 tokens start while the softmax is at the second 64.
//
// One B200, 32 query heads on 4, dim 128: a prompt of 8192 tokens takes 649 us (captured calls one
// after another), 847 TFLOP/s, 51 % of a plain bf16 product's rate; 4200 cycles a step of 256 rows and 128
// tokens, of which products are 2048.  A step is a chain: softmax of a tile (2500), its products (1500); the
// other tile's chain fills in, but two tiles are what 512 columns hold.  Skipping the exponentials, or the search for the maximum, or the
// conversion each gains 3 to 8 %.  An item costs 4 steps more: query rows in, results out, masks.
//
// Work is one list of (row tile, head) items, 128 tokens a unit, cut into equal contiguous pieces, one
// per SM; kv_prompt_plan_kernel writes it (causal row tiles differ in length), kv_prompt_join_kernel
// joins the items that a cut went through.  The roles meet only at the barriers of the buffers they
// share, so the next item's keys are under way while the last one's rows are written.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_attend.cuh"
#include "umma.cuh"

namespace duplex {

constexpr int kPTok = 128, kPRows = 256, kPThreads = 640, kPMaxCtas = 160;

// An item costs as much as its tiles and kPOver more (query rows in, results out, the pipeline's ends).
constexpr int kPOver = 4;

// A (sequence, row tile): every head has one such item.
struct PromptItem {
  int64_t off;  // units before it (of all heads)
  int b, rt;
  KvSeq s;
  Span sp;
  int per;      // units: its tiles and kPOver
  int first_pos, last_pos;
};

// Of a sequence and head: the power of two in the largest key scale that a row sees, the largest value scale,
// and whether scores and probabilities need a factor by their block: a scale is no power of two, or far below
// the largest (e4m3's least code is 2^-9, fp16's least step 2^-24), or an id is out of range (a mask).
struct PromptRef {
  float k, v;
  int by_block, pad;
};

DEVI float pow2_of(float x) { return __uint_as_float(__float_as_uint(x) & 0x7F800000u); }
DEVI bool far_below(float least, float most) { return least < most * 6.103515625e-5f; }  // 2^-14

struct PromptParams {
  AttendParams a;
  PromptItem* list;  // pairs (sequence, row tile), and an end
  PromptRef* ref;    // [batch][heads]
  int* n_pairs;
  int64_t* total;
};

// A piece's units: an equal share, but no fewer than make the pieces worth joining.
DEVI int64_t share_of(int64_t total, int ctas) { return max((total + ctas - 1) / ctas, (int64_t)(2 * kPOver)); }

DEVI int units_in(const Span& sp) {
  return sp.sink_units + (sp.end > sp.lo ? (sp.end - sp.lo + kPTok - 1) / kPTok : 0);
}

// CTA 0: the list.  CTA 1 + i: the scales of (sequence, head) i.
constexpr int kPlanThreads = 256;

__global__ void __launch_bounds__(kPlanThreads) kv_prompt_plan_kernel(PromptParams pp) {
  extern __shared__ int tiles[];  // [batch + 1] row tiles before each sequence
  __shared__ int64_t warp_sum[kPlanThreads / 32];
  __shared__ float2 s_k[kPlanThreads / 32], s_v[kPlanThreads / 32];
  const AttendParams& p = pp.a;
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = c.batch;
  pdl_launch_dependents();
  if (blockIdx.x > 0) {
    const int b = (blockIdx.x - 1) / c.heads, h = (blockIdx.x - 1) - b * c.heads;
    const KvSeq s = kv_seq(c, b);
    const int lo_x = p.window ? s.first - p.window + 1 : 0, cols = s.rows ? (s.n + c.block - 1) / c.block : 0;
    float mk = 0.f, mv = 0.f, lk = INFINITY, lv = INFINITY;  // largest and least (a scale of 0 is exact anywhere)
    int by_block = 0;
    for (int col = tid; col < cols; col += kPlanThreads) {
      const int tok = col * c.block;
      if (tok + c.block <= lo_x && tok >= p.sinks) continue;
      const int id = kv_block_at(c, b, col, p.err);
      if (id < 0) by_block = 1;
      else {
        const float k = __ldg(c.k_scale + (int64_t)id * c.heads + h), v = __ldg(c.v_scale + (int64_t)id * c.heads + h);
        by_block |= k != pow2_of(k) || v != pow2_of(v);
        mk = fmaxf(mk, pow2_of(k));
        mv = fmaxf(mv, v);
        if (k != 0.f) lk = fminf(lk, k);
        if (v != 0.f) lv = fminf(lv, v);
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      mk = fmaxf(mk, __shfl_xor_sync(~0u, mk, o));
      mv = fmaxf(mv, __shfl_xor_sync(~0u, mv, o));
      lk = fminf(lk, __shfl_xor_sync(~0u, lk, o));
      lv = fminf(lv, __shfl_xor_sync(~0u, lv, o));
    }
    if (lane == 0) {
      s_k[warp] = make_float2(mk, lk);
      s_v[warp] = make_float2(mv, lv);
    }
    by_block = __syncthreads_or(by_block);
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kPlanThreads / 32; ++w) {
        mk = fmaxf(mk, s_k[w].x);
        mv = fmaxf(mv, s_v[w].x);
        lk = fminf(lk, s_k[w].y);
        lv = fminf(lv, s_v[w].y);
      }
      by_block |= far_below(lk, mk) || far_below(lv, mv);
      pp.ref[blockIdx.x - 1] = PromptRef{fmaxf(mk, pow2f(-126)), fmaxf(mv, pow2f(-126)), by_block, 0};
    }
    return;
  }
  auto scan = [&](int64_t x, int64_t& all) {  // exclusive, over the block
    int64_t incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int64_t before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    return before + incl - x;
  };
  int64_t base = 0, all = 0;
  const bool fall = offsets_fall(c);
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int t = 0;
    if (b < B) {
      const KvSeq s = kv_seq(c, b);
      t = (int)(((int64_t)s.rows * p.group + kPRows - 1) / kPRows);
      if (too_long(c, s)) set_error(p.err, DUPLEX_DEVERR_LENGTH);
    }
    const int64_t at = scan(t, all);
    if (b < B) tiles[b] = (int)(base + at);
    base += all;
  }
  if (tid == 0) tiles[B] = (int)base;
  // the list has room for the pairs of offsets that rise (max_pairs)
  const bool none = __syncthreads_or(fall);
  if (none && tid == 0) set_error(p.err, DUPLEX_DEVERR_OFFSETS);
  const int pairs = none ? 0 : tiles[B];
  base = 0;
  for (int i0 = 0; i0 < pairs; i0 += kPlanThreads) {
    const int i = i0 + tid;
    PromptItem it{};
    if (i < pairs) {
      int lo = 0, hi = B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tiles[mid] <= i) lo = mid; else hi = mid - 1;
      }
      it.b = lo;
      it.rt = i - tiles[lo];
      it.s = kv_seq(c, lo);
      it.first_pos = it.s.first + it.rt * kPRows / p.group;
      it.last_pos = it.s.first + (min(it.rt * kPRows + kPRows, it.s.rows * p.group) - 1) / p.group;
      it.sp = span_of<kPTok>(p, it.first_pos, it.last_pos, it.s.n);
      it.per = units_in(it.sp) + kPOver;
    }
    it.off = base + scan((int64_t)it.per * c.heads, all);
    if (i < pairs) pp.list[i] = it;
    base += all;
  }
  if (tid == 0) {
    pp.list[pairs].off = base;
    *pp.n_pairs = pairs;
    *pp.total = base;
  }
}

// the last pair whose first unit is <= u, 32 of them a look (by whole warps)
DEVI int pair_of(const PromptItem* list, int pairs, int64_t u) {
  const int lane = threadIdx.x & 31;
  int lo = 0, left = pairs;
  while (left > 1) {
    const int step = (left + 31) / 32, at = lo + lane * step;
    const bool before = at < lo + left && list[at].off <= u;
    const int i = 31 - __clz(__ballot_sync(~0u, before) | 1u);
    left = min(step, left - i * step);
    lo += i * step;
  }
  return lo;
}

// shared memory, from a 1024-byte boundary: operands in the 128-byte swizzle (umma.cuh).  Q and K
// [dim / 64][row][64 dims] are K-major; V [dim / 64][token][64 dims], the same layout, is MN-major.
template <int D> struct PromptSmem {
  static constexpr uint32_t kHalf = 128 * 128, kTile = D / 64 * kHalf;
  static constexpr uint32_t q = 0, k = 2 * kTile, v = k + 2 * kTile, undo = v + 2 * kTile,
                            bars = undo + kPRows * 4;
  static constexpr uint32_t bytes = bars + 256 + 1024;
};

// 16-byte chunk c of a row
DEVI uint32_t sw128(int row, int c) { return (uint32_t)(row * 128 + ((c ^ (row & 7)) << 4)); }

DEVI float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// two fp32 operations in one instruction
DEVI float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

DEVI float2 add2f(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <int D> constexpr int prompt_part() { return kPRows * (D + 2); }

// The piece of an item that a CTA works on next.
struct Piece {
  PromptItem it;
  int h, i0, n, len;  // head; its first tile, its tiles (0: rows that see nothing), its units
  bool whole, two;    // the item's only piece; rows in the second tile

  DEVI int row_base() const { return it.rt * kPRows; }
  DEVI int row_all(int group) const { return it.s.rows * group; }
  DEVI int base_of(int i) const {
    return i < it.sp.sink_units ? i * kPTok : it.sp.lo + (i - it.sp.sink_units) * kPTok;
  }
};

DEVI void find_piece(const PromptParams& pp, int64_t u, int64_t u_end, int& pi, Piece& x) {
  while (pp.list[pi + 1].off <= u) ++pi;
  x.it = pp.list[pi];
  const int64_t r = u - x.it.off;
  x.h = r < 0x7FFFFFFF ? (int)r / x.it.per : (int)(r / x.it.per);
  const int u0 = (int)(r - (int64_t)x.h * x.it.per), u1 = (int)min((int64_t)x.it.per, u0 + (u_end - u));
  x.len = u1 - u0;
  x.whole = u0 == 0 && u1 == x.it.per;
  x.i0 = max(u0 - kPOver, 0);
  x.n = max(u1 - kPOver, 0) - x.i0;
  x.two = x.row_base() + 128 < x.row_all(pp.a.group);
}

// Registers: 640 threads start with 96 each, 61,440; the softmax warps take what the others leave.
constexpr int kRegSoftmax = 152, kRegConvert = 56, kRegMma = 64;
static_assert(256 * kRegSoftmax + 256 * kRegConvert + 128 * kRegMma <= kPThreads * 96, "register split");

template <int D, int FMT>
__global__ void __launch_bounds__(kPThreads, 1) kv_prompt_kernel(const __grid_constant__ PromptParams pp) {
  using L = PromptSmem<D>;
  extern __shared__ uint8_t dyn[];
  uint8_t* const sm = dyn + (1024 - smem_u32(dyn) % 1024) % 1024;
  float* const s_undo = reinterpret_cast<float*>(sm + L::undo);
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;
  __shared__ int2 s_piece;  // for the products: the piece's tiles and whether its second row tile has rows; -1: no more
  const AttendParams& p = pp.a;
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6, *s_full = bar + 8, *p_ready = bar + 10,
           *o_full = bar + 12, *drain = bar + 13, *q_full = bar + 14, *p_half = bar + 16;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 8);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 8);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 4);
      mbar_init(p_half + i, 4);
    }
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    mbar_init(q_full, 8);
    fence_mbar_init();
    s_abort = 0;
  }
  if (warp == 16) tmem_alloc<512>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tm = 0;  // all 512 columns: they start at column 0
  auto t_s = [&](int mt) { return tm + mt * 128; };
  auto t_o = [&](int mt) { return tm + 256 + mt * D; };
  pdl_wait();
  pdl_launch_dependents();

  auto wait = [&](uint64_t* b, uint32_t n) -> bool {  // the n-th completion (from 0) of a barrier, by a whole warp
    bool ok = mbar_try_wait(b, n & 1);
    if (__all_sync(~0u, ok)) return true;
    ok = mbar_wait_bounded(b, n & 1, &s_abort);
    if (!ok) set_error(p.err, DUPLEX_DEVERR_TIMEOUT);
    return __all_sync(~0u, ok) != 0;
  };

  const int pairs = *pp.n_pairs;
  const int64_t total = *pp.total, share = share_of(total, gridDim.x);
  const int64_t u_begin = (int64_t)blockIdx.x * share, u_end = min(u_begin + share, total);
  int64_t u = u_begin;
  int pi = u < u_end ? pair_of(pp.list, pairs, u) : 0;
  Piece x;

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax: a thread's row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoftmax));
    const int mt = warp >> 2;
    const uint32_t lane_at = (uint32_t)(warp & 3) * 32u << 16;
    const uint32_t ts = t_s(mt) + lane_at, to = t_o(mt) + lane_at;
    uint8_t* const q_tile = sm + L::q + mt * L::kTile;
    uint32_t n_s = 0, n_o = 0;  // completions of s_full[mt], o_full so far
    bool ok = true;
    // query rows on their way: 8 rows at a time, 4 lanes a row; rows 16 i .. + 15 of the warp's 32
    uint4 raw[2][D / 32];
    auto load_rows = [&](int i) {
      const int row_all = x.row_all(p.group);
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        const int r2 = x.row_base() + 32 * warp + 16 * i + 8 * e2 + (lane & 7), t2 = p.by_group(r2);
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + 16 * (lane >> 3);
        const bool in = r2 < row_all;
        if (in) src += 2 * ((int64_t)(x.it.s.row0 + t2) * p.q_row + (int64_t)(x.h * p.group + r2 - t2 * p.group) * p.q_head);
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
          raw[e2][e] = in ? __ldg(reinterpret_cast<const uint4*>(src + 64 * e)) : make_uint4(0, 0, 0, 0);
      }
    };
    // ... and to shared memory, as fp16 scaled by a power of two (kv_attend.cu: load_q)
    auto put_rows = [&](int i) {
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        const int row = (32 * warp + 16 * i + 8 * e2 + (lane & 7)) & 127;
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < D / 32; ++e)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t y = (&raw[e2][e].x)[w];
            const float2 f = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(y) : act2<DUPLEX_DTYPE_BF16>(y);
            amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 8));
        amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 16));
        const int ex = (int)(__float_as_uint(amax) >> 23) - 127;
        const int up = (amax == 0.f || ex == 128) ? 0 : min(14 - ex, 126);
        const float f = p.scale_log2 < 0.f ? -pow2f(up) : pow2f(up);  // its sign goes with the row
        if (lane < 8) s_undo[32 * warp + 16 * i + 8 * e2 + lane] = pow2f(-up);
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
          uint4 y;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t z = (&raw[e2][e].x)[w];
            const float2 a = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(z) : act2<DUPLEX_DTYPE_BF16>(z);
            (&y.x)[w] = f2h(a.x * f, a.y * f);
          }
          const int ch = 4 * e + (lane >> 3);  // of the row's D / 8
          *reinterpret_cast<uint4*>(q_tile + (ch >> 3) * L::kHalf + sw128(row, ch & 7)) = y;
        }
      }
    };
    PromptRef ref{};
    auto next = [&]() {
      find_piece(pp, u, u_end, pi, x);
      ref = pp.ref[x.it.b * c.heads + x.h];
      if (x.n > 0) load_rows(0);
    };
    auto give_rows = [&]() {
      if (x.n <= 0) return;
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        if (i) load_rows(i);
        put_rows(i);
      }
      if (tid == 0) s_piece = make_int2(x.n, x.two);
      fence_proxy_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    };
    if (u < u_end) {
      next();
      give_rows();
    }
    while (ok && u < u_end) {
      const int n = x.n, row_base = x.row_base(), row_all = x.row_all(p.group);
      const KvSeq s = x.it.s;
      const int rr = row_base + tid, t_row = p.by_group(rr);
      const bool live = rr < row_all;
      const int pos = live ? s.first + t_row : -1;
      const int wlo = p.window ? pos - p.window : -1;  // tokens k > wlo, or k < sinks
      const int row_lo = row_base + mt * 128, row_hi = min(row_lo + 128, row_all);
      const int t_first = s.first + p.by_group(min(row_lo, row_all - 1));  // positions of the tile's rows
      const int t_last = s.first + p.by_group(row_hi - 1);
      const bool mine = mt == 0 || x.two;
      const float cs = fmaxf(s_undo[tid] * fabsf(p.scale_log2) * ref.k, 1.2e-38f);  // not 0: hidden scores are -inf
      float m = -INFINITY, l = 0.f, vref = ref.by_block ? pow2f(-126) : ref.v;  // O is in units of vref
      // Tiles from j on; BY block, with factors of scores and probabilities, and s - m of the rounded s.  The others end
      // at the first tile with scores beyond kHuge, and return it.
      auto tiles = [&](auto by, int j) {
        constexpr bool BY = decltype(by)::value;
        for (; mine && j < n; ++j) {
          const int base = x.base_of(x.i0 + j);
          // (rows past the last have zeros for a query and are not written: they need no mask)
          const bool masked = BY || base + kPTok - 1 > t_first ||
                              (p.window && base <= t_last - p.window && base + kPTok > p.sinks);
          // lane i (of 8): the scales of the block that holds tokens base + 16 i .. + 15; -1: an id out of range
          float kf = 1.f, vs = vref;
          if (BY && ref.by_block) {
            const int k = base + 16 * (lane & 7), id = k < x.it.sp.end ? c.table[(int64_t)x.it.b * c.width + k / c.block] : -1;
            kf = -1.f;
            vs = 0.f;
            if ((unsigned)id < (unsigned)c.n_blocks) {
              kf = __ldg(c.k_scale + (int64_t)id * c.heads + x.h) / ref.k;
              vs = __ldg(c.v_scale + (int64_t)id * c.heads + x.h);
            }
          }
          if (!(ok = wait(s_full + mt, n_s + j))) return n;
          tc_fence_after();
          // The loops are short on purpose: unrolled over the row they outgrow the instruction caches, and
          // the tile takes 1.8 times as long.
          float mx = -INFINITY;
          if (masked) {
            const int k_max = pos - base, k_min = wlo - base, k_sink = p.sinks - base;  // columns k <= k_max, k > k_min or k < k_sink
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
              uint32_t w[32];
              tmem_ld32(ts + 32 * q, w);
              tc_wait_ld();
              auto below = [](int k) { return k <= 0 ? 0u : k >= 32 ? ~0u : (1u << k) - 1; };  // bits of columns < k
              const uint32_t see = below(k_max + 1 - 32 * q) & (~below(k_min + 1 - 32 * q) | below(k_sink - 32 * q));
              if (BY) {
                const float f[2] = {__shfl_sync(~0u, kf, 2 * q), __shfl_sync(~0u, kf, 2 * q + 1)};
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  w[e] = f[e >> 4] < 0.f ? __float_as_uint(-INFINITY) : __float_as_uint(__uint_as_float(w[e]) * f[e >> 4]);
              }
#pragma unroll
              for (int e = 0; e < 32; ++e) w[e] = (see >> e) & 1u ? w[e] : __float_as_uint(-INFINITY);
              __syncwarp();
              tmem_st16(ts + 32 * q, reinterpret_cast<const uint32_t(&)[16]>(w[0]));
              tmem_st16(ts + 32 * q + 16, reinterpret_cast<const uint32_t(&)[16]>(w[16]));
#pragma unroll
              for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(w[e]));
            }
            tc_wait_st();
          } else {
#pragma unroll 1
            for (int q = 0; q < 2; ++q) {
              uint32_t w[2][32];
              tmem_ld32(ts + 64 * q, w[0]);
              tmem_ld32(ts + 64 * q + 32, w[1]);
              tc_wait_ld();
              float y[4] = {mx, mx, mx, mx};
#pragma unroll
              for (int e = 0; e < 32; ++e) y[e & 3] = max3(y[e & 3], __uint_as_float(w[0][e]), __uint_as_float(w[1][e]));
              mx = max3(y[0], y[1], fmaxf(y[2], y[3]));
            }
          }
          mx *= cs;
          float vf = 1.f;
          if (BY) {  // the largest value scale of what the row sees
            float v = vref;
#pragma unroll 1
            for (int i = 0; i < kPTok / 16; ++i) {
              const float y = __shfl_sync(~0u, vs, i);
              const int k = base + 16 * i, last = min(k + 15, pos);  // the last of the 16 that the row may see
              if (last >= k && (last > wlo || k < p.sinks)) v = fmaxf(v, y);
            }
            vf = vref / v;
            vref = v;
          }
          if (__any_sync(~0u, mx > m + kSlack || (BY && vf != 1.f))) {
            const float top = mx > m + kSlack ? mx : m;
            float f = top == m ? 1.f : ex2(m - top);
            if (!BY && __any_sync(~0u, fabsf(top) > kHuge && top != -INFINITY)) return j;
            m = top;
            l *= f;
            if (BY) f *= vf;
            if (j > 0) {
#pragma unroll 1
              for (int q = 0; q < D / 16; ++q) {
                uint32_t o[16];
                tmem_ld16(to + 16 * q, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st16(to + 16 * q, o);
              }
            }
          }
          const float add = kShift - (m == -INFINITY ? 0.f : m);
          const float2 cs2 = make_float2(cs, cs), add2 = make_float2(add, add);
          float2 ls = make_float2(0.f, 0.f);
          if constexpr (BY) {  // the probabilities' sum without, the operand with the value's scale; s - m of the rounded s
            const float rv = 1.f / vref, ref_m = m == -INFINITY ? 0.f : m;
            __syncwarp();
#pragma unroll 1
            for (int q = 0; q < kPTok / 16; ++q) {
              // (beyond [0, 1], where the row sees none of it, it must not make a NaN of 0)
              const float f = fmaxf(fminf(__shfl_sync(~0u, vs, q) * rv, 1.f), 0.f);
              uint32_t w[16], P[8];
              tmem_ld16(ts + 16 * q, w);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; e += 2) {
                auto p_of = [&](uint32_t s) { return ex2(__fsub_rn(__fmul_rn(__uint_as_float(s), cs), ref_m) + kShift); };
                const float2 z = make_float2(p_of(w[e]), p_of(w[e + 1]));
                ls = add2f(ls, z);
                P[e / 2] = f2h(z.x * f, z.y * f);
              }
              tmem_st8(ts + 8 * q, P);
              if (q == kPTok / 32 - 1) {
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half + mt);
              }
            }
          } else {
            uint32_t va[32], vb[32];
            auto part = [&](const uint32_t (&w)[32], int q) {  // P's columns 16 q .. + 15 lie over scores that are already read
              uint32_t P[16];
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float2 y = fma2(make_float2(__uint_as_float(w[e]), __uint_as_float(w[e + 1])), cs2, add2);
                const float2 z = make_float2(ex2(y.x), ex2(y.y));
                ls = add2f(ls, z);
                P[e / 2] = f2h(z.x, z.y);
              }
              tmem_st16(ts + 16 * q, P);
            };
            __syncwarp();
            tmem_ld32(ts, va);
#pragma unroll 1
            for (int q = 0; q < 4; q += 2) {
              tc_wait_ld();
              tmem_ld32(ts + 32 * q + 32, vb);
              part(va, q);
              tc_wait_ld();
              if (q == 0) tmem_ld32(ts + 64, va);
              part(vb, q + 1);
              if (q == 0) {  // the products of the first 64 tokens can start
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_half + mt);
              }
            }
          }
          l += ls.x + ls.y;
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(p_ready + mt);
        }
        return n;
      };
      const int rest = ref.by_block ? 0 : tiles(std::false_type{}, 0);
      if (rest < n) tiles(std::true_type{}, rest);
      // ---- the row's result.  Once all products are done (both tiles wait for them) the next piece's rows
      // take the query rows' place, so its first scores are computed under the writing of this one's results.
      if (!ok) break;
      const bool whole = x.whole, first = u == u_begin;
      const int h = x.h;
      const float inv = whole ? (l == 0.f ? 0.f : vref / l) : vref;
      u += x.len;
      if (u < u_end) next();
      if (n > 0 && !(ok = wait(o_full, n_o))) break;
      tc_fence_after();
      if (u < u_end) give_rows();
      if (mine) {
        if (whole) {  // a thread's row, 16 bytes a store
          const int64_t at = live ? (int64_t)(s.row0 + t_row) * p.heads + h * p.group + rr - t_row * p.group : 0;
          uint4* const row_out = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + 2 * at * D);
          auto put_out = [&](auto act) {
            constexpr int A = decltype(act)::value;
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t v[32];
              __syncwarp();
              if (n > 0) {
                tmem_ld32(to + 32 * q, v);
                tc_wait_ld();
              } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0;
              }
              if (live) {
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                  float o[8];
#pragma unroll
                  for (int k = 0; k < 8; ++k) o[k] = __uint_as_float(v[e + k]) * inv;
                  const uint2 y = pack4(A, make_float4(o[0], o[1], o[2], o[3])), z = pack4(A, make_float4(o[4], o[5], o[6], o[7]));
                  row_out[4 * q + e / 8] = make_uint4(y.x, y.y, z.x, z.y);
                }
              }
            }
          };
          if (p.act == DUPLEX_DTYPE_F16) put_out(std::integral_constant<int, DUPLEX_DTYPE_F16>{});
          else put_out(std::integral_constant<int, DUPLEX_DTYPE_BF16>{});
          if (live) put_stats(p, at, m, l);
        } else {  // a piece's as they come, [dim / 4][row]
          float* part = p.part + (2 * (int64_t)blockIdx.x + (first ? 0 : 1)) * prompt_part<D>();
          float4* to4 = reinterpret_cast<float4*>(part) + tid;
#pragma unroll 1
          for (int q = 0; q < D / 16; ++q, to4 += 4 * kPRows) {
            uint32_t v[16];
            __syncwarp();
            if (n > 0) {
              tmem_ld16(to + 16 * q, v);
              tc_wait_ld();
            } else {
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              to4[e * kPRows] = make_float4(__uint_as_float(v[4 * e]) * inv, __uint_as_float(v[4 * e + 1]) * inv,
                                            __uint_as_float(v[4 * e + 2]) * inv, __uint_as_float(v[4 * e + 3]) * inv);
          }
          part[kPRows * D + tid] = m;
          part[kPRows * D + kPRows + tid] = l;
        }
        __syncwarp();
        tc_fence_before();
        n_s += n;
      }
      if (n > 0) ++n_o;
    }
    if (tid == 0) s_piece = make_int2(-1, 0);
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
  } else if (warp < 16) {
    // ---------------------------------------------------------------- keys and values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegConvert));
    constexpr int KC = D / 64;  // 16-byte chunks a lane takes of a token
    const int t0 = 16 * (warp - 8), kt = lane & 7, kc = lane >> 3;  // the warp's 16 tokens; token of 8, chunk of 4 (of 64 dims)
    uint32_t n_tile = 0;
    bool ok = true;
    for (; ok && u < u_end; u += x.len) {
      find_piece(pp, u, u_end, pi, x);
      const int n = x.n, end = x.i0 + n;
      const int lo_x = p.window ? x.it.first_pos - p.window + 1 : 0;  // the first token past the sinks that a row sees
      const PromptRef ref = pp.ref[x.it.b * c.heads + x.h];
      const float inv_k = ref.by_block ? 0.f : 1.f / ref.k, inv_v = ref.by_block ? 0.f : 1.f / ref.v;  // 0: codes as they are
      uint4 kx[2][KC], vx[2][KC];
      float kr = 0.f, vr = 0.f;
      // the id of the block that holds the warp's tokens of tile i, as the table has it; -1: not looked at
      auto id_of = [&](int i) {
        const int tok = x.base_of(i) + t0;
        return i < end && tok < x.it.sp.end && !(tok + 15 < lo_x && tok >= p.sinks) ? c.table[(int64_t)x.it.b * c.width + tok / c.block] : -1;
      };
      auto load = [&](int i, int id, const uint8_t* codes, const float* scales, uint4 (&to)[2][KC], float& sc) {
        const bool good = (unsigned)id < (unsigned)c.n_blocks;
        const int tok = x.base_of(i) + t0;
        const int64_t bh = good ? (int64_t)id * c.heads + x.h : 0;
        const uint8_t* src = codes + ((bh * c.block + (tok & (c.block - 1)) + kt) * D + 16 * kc);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int cc = 0; cc < KC; ++cc)
            to[q][cc] = good ? __ldg(reinterpret_cast<const uint4*>(src + 8 * q * D + 64 * cc)) : make_uint4(0, 0, 0, 0);
        sc = good ? __ldg(scales + bh) : 0.f;
      };
      auto mul = [](uint32_t w, __half2 f) {
        const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&w), f);
        return *reinterpret_cast<const uint32_t*>(&y);
      };
      auto put = [&](uint8_t* dst, int base, const uint4 (&from)[2][KC], float ratio) {
        const bool clean = base + kPTok <= x.it.sp.end && (base >= lo_x || base + kPTok <= p.sinks);
        const __half2 f = __float2half2_rn(ratio);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int t = t0 + 8 * q + kt, k = base + t;
          const bool zero = !clean && !(k < x.it.sp.end && (k >= lo_x || k < p.sinks));  // it may hold anything
#pragma unroll
          for (int cc = 0; cc < KC; ++cc) {
            uint4 y = from[q][cc];
            if (zero) y = make_uint4(0, 0, 0, 0);
            uint8_t* at = dst + cc * L::kHalf;
            *reinterpret_cast<uint4*>(at + sw128(t, 2 * kc)) = make_uint4(mul(KvFmt<FMT>::lo(y.x), f), mul(KvFmt<FMT>::hi(y.x), f),
                                                                          mul(KvFmt<FMT>::lo(y.y), f), mul(KvFmt<FMT>::hi(y.y), f));
            *reinterpret_cast<uint4*>(at + sw128(t, 2 * kc + 1)) =
                make_uint4(mul(KvFmt<FMT>::lo(y.z), f), mul(KvFmt<FMT>::hi(y.z), f), mul(KvFmt<FMT>::lo(y.w), f),
                           mul(KvFmt<FMT>::hi(y.w), f));
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
      };
      int id = id_of(x.i0), id_next = id_of(x.i0 + 1);
      if (n > 0) {
        load(x.i0, id, c.k, c.k_scale, kx, kr);
        load(x.i0, id, c.v, c.v_scale, vx, vr);
      }
      for (int j = 0; j < n; ++j) {
        const uint32_t cnt = n_tile + j, slot = cnt & 1, use = cnt >> 1;
        const int i = x.i0 + j, base = x.base_of(i);
        id = id_next;
        id_next = id_of(i + 2);
        if (use > 0 && !(ok = wait(k_empty + slot, use - 1))) break;
        put(sm + L::k + slot * L::kTile, base, kx, inv_k == 0.f ? 1.f : kr * inv_k);
        if (lane == 0) mbar_arrive(k_full + slot);
        if (j + 1 < n) load(i + 1, id, c.k, c.k_scale, kx, kr);
        if (use > 0 && !(ok = wait(v_empty + slot, use - 1))) break;
        put(sm + L::v + slot * L::kTile, base, vx, inv_v == 0.f ? 1.f : vr * inv_v);
        if (lane == 0) mbar_arrive(v_full + slot);
        if (j + 1 < n) load(i + 1, id, c.v, c.v_scale, vx, vr);
      }
      n_tile += n;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegMma));
    if (warp == 16) {
      // -------------------------------------------------------------- products
      constexpr uint32_t id_qk = idesc_f16(0, 128, kPTok), id_pv = idesc_f16(0, 128, D) | kIdescBMnMajor;
      const uint32_t sq = smem_u32(sm + L::q), sk = smem_u32(sm + L::k), sv = smem_u32(sm + L::v);
      auto done = [&](uint64_t* b) {
        if (elect_one()) umma_commit(b);
      };
      auto qk = [&](int mt, uint32_t slot) {
        const uint64_t dq = smem_desc_sw128(sq + mt * L::kTile, 16), dk = smem_desc_sw128(sk + slot * L::kTile, 16);
#pragma unroll
        for (int y = 0; y < D / 16; ++y) {
          const uint32_t at = (y >> 2) * (L::kHalf >> 4) + (y & 3) * 2;
          if (elect_one()) umma_ss(t_s(mt), dq + at, dk + at, id_qk, y != 0);
        }
        done(s_full + mt);
      };
      auto pv = [&](int mt, uint32_t slot, bool more, int half) {
        const uint64_t dv = smem_desc_sw128(sv + slot * L::kTile, L::kHalf);
#pragma unroll
        for (int e = 0; e < kPTok / 32; ++e) {
          const int y = half * (kPTok / 32) + e;
          if (elect_one()) umma_ts(t_o(mt), t_s(mt) + 8 * y, dv + y * (2048 >> 4), id_pv, more || y != 0);
        }
      };
      // tile mt's output of tile j, as its probabilities come
      auto out = [&](int mt, uint32_t slot, bool more, uint32_t k) {
        if (!wait(p_half + mt, k)) return false;
        tc_fence_after();
        pv(mt, slot, more, 0);
        if (!wait(p_ready + mt, k)) return false;
        tc_fence_after();
        pv(mt, slot, more, 1);
        return true;
      };
      uint32_t n_tile = 0, n1 = 0, n_q = 0;  // tiles so far (p_ready[0], the rings); completions of p_ready[1], q_full
      bool ok = true;
      for (; ok; ++n_q) {
        if (!(ok = wait(q_full, n_q))) break;
        const int n = s_piece.x;
        const int two = s_piece.y;
        if (n < 0) break;
        if (!(ok = wait(k_full + (n_tile & 1), n_tile >> 1))) break;
        tc_fence_after();
#pragma unroll 1
        for (int mt = 0; mt <= two; ++mt) qk(mt, n_tile & 1);
        done(k_empty + (n_tile & 1));
        for (int j = 0; j < n; ++j) {
          const uint32_t cnt = n_tile + j, slot = cnt & 1, nslot = slot ^ 1;
          const bool more = j + 1 < n;
          if (!(ok = wait(v_full + slot, cnt >> 1) && (!more || wait(k_full + nslot, (cnt + 1) >> 1)))) break;
#pragma unroll 1
          for (int mt = 0; ok && mt <= two; ++mt) {
            if (!(ok = out(mt, slot, j > 0, (mt ? n1 : n_tile) + j))) break;
            if (mt == two) done(v_empty + slot);
            if (more) qk(mt, nslot);
          }
          if (!ok) break;
          if (more) done(k_empty + nslot);
        }
        if (ok) done(o_full);
        n_tile += n;
        if (two) n1 += n;
      }
      // no product may still be running when tensor memory goes
      done(drain);
      const long long t0 = clock64();
      while (!mbar_try_wait(drain, 0))
        if (clock64() - t0 > 200000000LL) {
          set_error(p.err, DUPLEX_DEVERR_TIMEOUT);
          break;
        }
      __syncwarp();
    }
  }
  __syncthreads();
  if (warp == 16) tmem_dealloc<512>(tm);
}

// CTA (j, y) joins 32 dims of the item that crosses the boundary between pieces j and j + 1, if that is
// its first one.
constexpr int kJoinThreads = 256;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_prompt_join_kernel(PromptParams pp, int ctas) {
  static_assert(kJoinThreads == kPRows, "a thread is a row");
  const AttendParams& p = pp.a;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t total = *pp.total, share = share_of(total, ctas);
  const int64_t u = (int64_t)(blockIdx.x + 1) * share;
  if (u >= total) return;
  const int pi = pair_of(pp.list, *pp.n_pairs, u);
  const PromptItem it = pp.list[pi];
  const int h = (int)((u - it.off) / it.per);
  const int64_t begin = it.off + (int64_t)h * it.per, last = begin + it.per - 1;
  if (begin == u || begin / share != blockIdx.x) return;
  const int c0 = blockIdx.x, c1 = (int)(last / share);
  const int rr = threadIdx.x, r2 = it.rt * kPRows + rr, d0 = 32 * blockIdx.y;
  if (r2 >= it.s.rows * p.group) return;
  auto slot = [&](int j) {
    const int k = (j == c0 && begin != (int64_t)c0 * share) ? 1 : 0;
    return p.part + (2 * (int64_t)j + k) * prompt_part<D>();
  };
  float M = -INFINITY;
#pragma unroll 4
  for (int j = c0; j <= c1; ++j) M = fmaxf(M, __ldcg(slot(j) + kPRows * D + rr));
  float4 o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int j = c0; j <= c1; ++j) {
    const float* ps = slot(j);
    const float mj = __ldcg(ps + kPRows * D + rr), f = mj == M ? 1.f : ex2(mj - M);
    l += __ldcg(ps + kPRows * D + kPRows + rr) * f;
    const float4* po = reinterpret_cast<const float4*>(ps) + d0 / 4 * kPRows + rr;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float4 y = __ldcg(po + e * kPRows);
      o[e].x += y.x * f;
      o[e].y += y.y * f;
      o[e].z += y.z * f;
      o[e].w += y.w * f;
    }
  }
  const int t2 = p.by_group(r2);
  const int64_t at = (int64_t)(it.s.row0 + t2) * p.heads + h * p.group + r2 - t2 * p.group;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + 2 * (at * D + d0));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint2 y = pack4(p.act, make_float4(o[e].x * inv, o[e].y * inv, o[e].z * inv, o[e].w * inv));
    const uint2 z = pack4(p.act, make_float4(o[e + 1].x * inv, o[e + 1].y * inv, o[e + 1].z * inv, o[e + 1].w * inv));
    dst[e / 2] = make_uint4(y.x, y.y, z.x, z.y);
  }
  if (blockIdx.y == 0) put_stats(p, at, M, l);
}

// Which kernel is faster, by the time each takes as measured on one B200 (128 dims, 32 query heads on 4;
// its own / kv_attend_kernel's us):
//   7 sequences of 3000 tokens, 4 rows each 36 / 27, 8 rows 36 / 37, 16 rows 37 / 55, 32 rows 45 / 95
//   64 of 4096: 4 rows 174 / 138, 8 rows 174 / 257      1 of 8192: 4 rows 39 / 20, 32 rows 47 / 44 (the
//   one of these where the rule takes the slower)
// A 128-token step of 16 rows, two CTAs an SM, takes there as long as one of 256 rows takes here, 2.3 us;
// the rest is what a call costs before and after.  Lengths are the block table's, which the host knows.
bool kv_prompt_takes(const AttendParams& p) {
  const KvView& c = p.c;
  const double rows = (double)c.n_rows * p.group / c.batch;
  if (rows <= 16) return false;
  double tokens = (double)c.width * c.block;
  if (p.window) tokens = std::min(tokens, (double)p.sinks + p.window + rows / p.group);
  const double steps = tokens / kPTok + 1, lists = (double)c.batch * c.heads;
  const double few = 18 + 2.3 * lists * std::ceil(rows / 16) * steps / 296;
  const double many = 28 + 2.3 * std::max(2.0 * kPOver, lists * std::ceil(rows / kPRows) * (steps + kPOver) / 148);
  return many < few;
}

static int64_t max_pairs(const KvView& c, int group) { return (int64_t)c.n_rows * group / kPRows + c.batch; }

static size_t list_bytes(const KvView& c, int group) {
  return (size_t)(16 + (max_pairs(c, group) + 1) * (int64_t)sizeof(PromptItem) + 127) / 128 * 128;
}

static size_t ref_bytes(const KvView& c) { return (size_t)c.batch * c.heads * sizeof(PromptRef); }

size_t kv_prompt_workspace(const KvView& c, int group) {
  return list_bytes(c, group) + (ref_bytes(c) + 127) / 128 * 128 + (size_t)2 * kPMaxCtas * (c.dim == 128 ? prompt_part<128>() : prompt_part<64>()) * 4;
}

template <int D, int FMT>
static int run(const PromptParams& pp, int ctas, cudaStream_t st) {
  constexpr size_t smem = PromptSmem<D>::bytes;
  const KvView& c = pp.a.c;
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kv_prompt_kernel<D, FMT>), (int)smem)) return rc;
  kv_prompt_plan_kernel<<<1 + c.batch * c.heads, kPlanThreads, sizeof(int) * (c.batch + 1), st>>>(pp);
  if (int rc = record_cuda(cudaGetLastError())) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kPThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (int rc = record_cuda(cudaLaunchKernelEx(&cfg, kv_prompt_kernel<D, FMT>, pp))) return rc;
  if (ctas < 2) return DUPLEX_OK;
  cfg.gridDim = dim3(ctas - 1, D / 32);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return record_cuda(cudaLaunchKernelEx(&cfg, kv_prompt_join_kernel<D>, pp, ctas));
}

int kv_prompt_ctas(const AttendParams& a, int* ctas) {
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const int64_t units = max_pairs(a.c, a.group) * a.c.heads * (((int64_t)a.c.width * a.c.block + kPTok - 1) / kPTok + kPOver);
  *ctas = (int)std::min({(int64_t)sms, (int64_t)kPMaxCtas, units});
  return DUPLEX_OK;
}

int kv_prompt_run(const AttendParams& a, void* workspace, cudaStream_t st) {
  PromptParams pp{};
  pp.a = a;
  const size_t list = list_bytes(a.c, a.group);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  pp.list = reinterpret_cast<PromptItem*>(ws + 16);
  pp.ref = reinterpret_cast<PromptRef*>(ws + list);
  pp.total = reinterpret_cast<int64_t*>(ws);
  pp.n_pairs = reinterpret_cast<int*>(ws + 8);
  pp.a.part = reinterpret_cast<float*>(ws + list + (ref_bytes(a.c) + 127) / 128 * 128);
  int ctas = 0;
  if (int rc = kv_prompt_ctas(a, &ctas)) return rc;
  if (a.c.dim == 128)
    return a.c.format == DUPLEX_KV_E4M3 ? run<128, DUPLEX_KV_E4M3>(pp, ctas, st) : run<128, DUPLEX_KV_INT8>(pp, ctas, st);
  return a.c.format == DUPLEX_KV_E4M3 ? run<64, DUPLEX_KV_E4M3>(pp, ctas, st) : run<64, DUPLEX_KV_INT8>(pp, ctas, st);
}

}  // namespace duplex
