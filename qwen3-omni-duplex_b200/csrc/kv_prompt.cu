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
//   warps 8-11       keys and values from the cache's codes to fp16 operands in shared memory (exact:
//                    code times its block's scale over the row tile's largest, a power of two), two
//                    buffers each.  Values are transposed on the way: B[dim][token]
//   warp 12          one thread issues the products: S = Q K^T (both shared memory), O += P V
//
// The running maximum is a reference that may lag by 2^kSlack, so O is rescaled rarely: the exponentials
// are taken at the old reference while the true maximum is found, and only where it has grown too far
// is the tile's O multiplied and its exponentials taken again.
//
// Work is one list of (row tile, head) items, 128 tokens a unit, cut into equal contiguous pieces, one
// per SM; kv_prompt_plan_kernel writes it (causal row tiles differ in length), kv_prompt_join_kernel
// joins the items that a cut went through.
#include <algorithm>

#include "kv_attend.cuh"
#include "umma.cuh"

namespace duplex {

constexpr int kPTok = 128, kPRows = 256, kPThreads = 512, kPMaxCtas = 160;

struct PromptItem {
  int64_t off;  // units before it (of all heads)
  int b, rt;
};

struct PromptParams {
  AttendParams a;
  PromptItem* list;  // pairs (sequence, row tile), and an end
  int* n_pairs;
  int64_t* total;
};

DEVI void prompt_rows(const AttendParams& p, const KvSeq& s, int rt, int& row_base, int& row_all, int& first_pos, int& last_pos) {
  row_base = rt * kPRows;
  row_all = s.rows * p.group;
  first_pos = s.n - s.rows + row_base / p.group;
  last_pos = s.n - s.rows + (min(row_base + kPRows, row_all) - 1) / p.group;
}

DEVI int units_in(const Span& sp) {
  return sp.sink_units + (sp.end > sp.lo ? (sp.end - sp.lo + kPTok - 1) / kPTok : 0);
}

// An item costs as much as its tiles and kPOver more (query rows in, results out, the pipeline's ends).
constexpr int kPOver = 4;

// The list of (sequence, row tile) pairs with their units, by one CTA.
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(kPlanThreads) kv_prompt_plan_kernel(PromptParams pp) {
  extern __shared__ int tiles[];  // [batch + 1] row tiles before each sequence
  __shared__ int64_t warp_sum[kPlanThreads / 32];
  const AttendParams& p = pp.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = p.c.batch;
  pdl_launch_dependents();
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
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int t = 0;
    if (b < B) t = (int)(((int64_t)kv_seq(p.c, b).rows * p.group + kPRows - 1) / kPRows);
    const int64_t at = scan(t, all);
    if (b < B) tiles[b] = (int)(base + at);
    base += all;
  }
  if (tid == 0) tiles[B] = (int)base;
  __syncthreads();
  const int pairs = tiles[B];
  base = 0;
  for (int i0 = 0; i0 < pairs; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int64_t u = 0;
    int b = 0, rt = 0;
    if (i < pairs) {
      int lo = 0, hi = B - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (tiles[mid] <= i) lo = mid; else hi = mid - 1;
      }
      b = lo;
      rt = i - tiles[b];
      const KvSeq s = kv_seq(p.c, b);
      int row_base, row_all, first_pos, last_pos;
      prompt_rows(p, s, rt, row_base, row_all, first_pos, last_pos);
      u = (int64_t)(units_in(span_of<kPTok>(p, first_pos, last_pos, s.n)) + kPOver) * p.c.heads;
    }
    const int64_t at = base + scan(u, all);
    if (i < pairs) pp.list[i] = PromptItem{at, b, rt};
    base += all;
  }
  if (tid == 0) {
    pp.list[pairs] = PromptItem{base, 0, 0};
    *pp.n_pairs = pairs;
    *pp.total = base;
  }
}

// the last pair whose first unit is <= u
DEVI int pair_of(const PromptItem* list, int pairs, int64_t u) {
  int lo = 0, hi = pairs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list[mid].off <= u) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// shared memory, from a 1024-byte boundary: operands in the 128-byte swizzle (umma.cuh).  Q and K
// [dim / 64][row][64 dims] are K-major; V [dim / 64][token][64 dims], the same layout, is MN-major.
template <int D> struct PromptSmem {
  static constexpr uint32_t kHalf = 128 * 128, kTile = D / 64 * kHalf;
  static constexpr uint32_t q = 0, k = 2 * kTile, v = k + 2 * kTile, undo = v + 2 * kTile, bars = undo + kPRows * 4;
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

// The piece of an item that a CTA works on next: its list position and what follows from it, found
// alike by every warp.
struct Piece {
  KvSeq s;
  Span sp;
  int b, h, row_base, row_all, first_pos, last_pos, lo_x;
  int i0, n, len;    // its first tile, its tiles (0: rows that see nothing), its units
  bool whole, two;   // the item's only piece; rows in the second tile

  DEVI int base_of(int i) const { return i < sp.sink_units ? i * kPTok : sp.lo + (i - sp.sink_units) * kPTok; }
  DEVI bool seen(const AttendParams& p, int k) const { return k < sp.end && (k >= lo_x || k < p.sinks); }
};

DEVI void find_piece(const PromptParams& pp, int64_t u, int64_t u_end, int& pi, Piece& x) {
  const AttendParams& p = pp.a;
  while (pp.list[pi + 1].off <= u) ++pi;
  const PromptItem item = pp.list[pi];
  x.b = item.b;
  x.s = kv_seq(p.c, item.b);
  prompt_rows(p, x.s, item.rt, x.row_base, x.row_all, x.first_pos, x.last_pos);
  x.sp = span_of<kPTok>(p, x.first_pos, x.last_pos, x.s.n);
  const int per = units_in(x.sp) + kPOver;
  const int64_t r = u - item.off;
  x.h = (int)(r / per);
  const int u0 = (int)(r - (int64_t)x.h * per), u1 = (int)min((int64_t)per, u0 + (u_end - u));
  x.len = u1 - u0;
  x.whole = u0 == 0 && u1 == per;
  x.i0 = max(u0 - kPOver, 0);
  x.n = max(u1 - kPOver, 0) - x.i0;
  x.two = x.row_base + 128 < x.row_all;
  x.lo_x = p.window ? x.first_pos - p.window + 1 : 0;  // the first token past the sinks that a row sees
}

// Registers: 512 threads start with 128 each; the softmax warps take what the others leave
// (256 * 160 + 128 * 112 + 128 * 72 < 512 * 128).
constexpr int kRegSoftmax = 160, kRegConvert = 112, kRegMma = 72;
constexpr int kWorkers = 13 * 32;  // the fourth warp group's other warps only give their registers

template <int D, int FMT>
__global__ void __launch_bounds__(kPThreads, 1) kv_prompt_kernel(const __grid_constant__ PromptParams pp) {
  using L = PromptSmem<D>;
  extern __shared__ uint8_t dyn[];
  uint8_t* const sm = dyn + (1024 - smem_u32(dyn) % 1024) % 1024;
  float* const s_undo = reinterpret_cast<float*>(sm + L::undo);
  __shared__ uint32_t s_tmem;
  __shared__ uint32_t s_ref[2];  // largest key / value scale of the piece, as bits
  __shared__ int s_bad;
  __shared__ volatile int s_abort;
  const AttendParams& p = pp.a;
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint64_t* bar = reinterpret_cast<uint64_t*>(sm + L::bars);
  uint64_t *k_full = bar, *k_empty = bar + 2, *v_full = bar + 4, *v_empty = bar + 6, *s_full = bar + 8, *p_ready = bar + 10,
           *o_full = bar + 12, *drain = bar + 13;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 4);
      mbar_init(k_empty + i, 1);
      mbar_init(v_full + i, 4);
      mbar_init(v_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_ready + i, 4);
    }
    mbar_init(o_full, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    s_abort = 0;
    s_ref[0] = s_ref[1] = 0;
    s_bad = 0;
  }
  if (warp == 12) tmem_alloc<512>(&s_tmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  constexpr uint32_t tm = 0;  // all 512 columns: they start at column 0
  auto t_s = [&](int mt) { return tm + mt * 128; };
  auto t_o = [&](int mt) { return tm + 256 + mt * D; };
  pdl_wait();
  pdl_launch_dependents();

  auto wait = [&](uint64_t* b, uint32_t n) -> bool {  // the n-th completion (from 0) of a barrier
    if (mbar_wait_bounded(b, n & 1, &s_abort)) return true;
    set_error(p.err, DUPLEX_DEVERR_TIMEOUT);
    return false;
  };

  const int pairs = *pp.n_pairs;
  const int64_t total = *pp.total, share = max((total + gridDim.x - 1) / gridDim.x, (int64_t)1);
  const int64_t u_begin = (int64_t)blockIdx.x * share, u_end = min(u_begin + share, total);
  int64_t u = u_begin;
  int pi = u < u_end ? pair_of(pp.list, pairs, u) : 0;
  Piece x;
  // each role walks the pieces, between the same two barriers a piece: query rows and scales are
  // there; the piece is done

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax: a thread's row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoftmax));
    const int mt = warp >> 2;
    const uint32_t lane_at = (uint32_t)(warp & 3) * 32u << 16;
    const uint32_t ts = t_s(mt) + lane_at, to = t_o(mt) + lane_at;
    uint32_t n_s = 0, n_o = 0;  // completions of s_full[mt], o_full so far
    while (u < u_end) {
      find_piece(pp, u, u_end, pi, x);
      const int n = x.n, h = x.h, row_base = x.row_base, row_all = x.row_all;
      const KvSeq& s = x.s;
      const Span& sp = x.sp;
      // the piece's largest scales, and whether all its block ids are good
      {
      const int per_tile = kPTok / c.block, cnt = n * per_tile;
      float mk = 0.f, mv = 0.f;
      for (int e = tid; e < cnt; e += 256) {
        const int i = e / per_tile, tok = x.base_of(x.i0 + i) + (e - i * per_tile) * c.block;
        if (tok >= sp.end || (tok + c.block <= x.lo_x && tok >= p.sinks)) continue;
        const int id = kv_block_at(c, x.b, tok / c.block, p.err);
        if (id < 0) {
          s_bad = 1;
          continue;
        }
        mk = fmaxf(mk, __ldg(c.k_scale + (int64_t)id * c.heads + h));
        mv = fmaxf(mv, __ldg(c.v_scale + (int64_t)id * c.heads + h));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        mk = fmaxf(mk, __shfl_xor_sync(~0u, mk, o));
        mv = fmaxf(mv, __shfl_xor_sync(~0u, mv, o));
      }
      if (lane == 0) {
        atomicMax(&s_ref[0], __float_as_uint(mk));
        atomicMax(&s_ref[1], __float_as_uint(mv));
      }
    }
      // query rows to shared memory, as fp16 scaled by a power of two (kv_attend.cu: load_q): a warp
      // takes 8 rows at a time, 4 lanes a row
      {
        uint4 raw[4][D / 32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r2 = row_base + 32 * warp + 8 * i + (lane & 7);
          const uint8_t* src = static_cast<const uint8_t*>(p.q) + 16 * (lane >> 3);
          const bool in = r2 < row_all;
          if (in) src += 2 * ((int64_t)(s.row0 + r2 / p.group) * p.q_row + (int64_t)(h * p.group + r2 % p.group) * p.q_head);
#pragma unroll
          for (int e = 0; e < D / 32; ++e)
            raw[i][e] = in ? __ldg(reinterpret_cast<const uint4*>(src + 64 * e)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (32 * warp + 8 * i + (lane & 7)) & 127;
          float amax = 0.f;
#pragma unroll
          for (int e = 0; e < D / 32; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t y = (&raw[i][e].x)[w];
              const float2 f = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(y) : act2<DUPLEX_DTYPE_BF16>(y);
              amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 8));
          amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 16));
          const int ex = (int)(__float_as_uint(amax) >> 23) - 127;
          const int up = (amax == 0.f || ex == 128) ? 0 : min(14 - ex, 126);
          const float f = p.scale_log2 < 0.f ? -pow2f(up) : pow2f(up);  // its sign goes with the row
          if (lane < 8) s_undo[32 * warp + 8 * i + lane] = pow2f(-up);
          uint8_t* dst = sm + L::q + (warp >> 2) * L::kTile;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) {
            uint4 y;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t z = (&raw[i][e].x)[w];
              const float2 a = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(z) : act2<DUPLEX_DTYPE_BF16>(z);
              (&y.x)[w] = f2h(a.x * f, a.y * f);
            }
            const int ch = 4 * e + (lane >> 3);  // of the row's D / 8
            *reinterpret_cast<uint4*>(dst + (ch >> 3) * L::kHalf + sw128(row, ch & 7)) = y;
          }
        }
      }
      const int rr = row_base + tid;
      const bool live = rr < row_all;
      fence_proxy_async_shared();
      named_bar_sync(1, kWorkers);
      const float kref = fmaxf(__uint_as_float(s_ref[0]), pow2f(-126)), vref = fmaxf(__uint_as_float(s_ref[1]), pow2f(-126));
      const bool bad = s_bad != 0;
      const int pos = live ? s.n - s.rows + rr / p.group : -1;
      const int wlo = p.window ? pos - p.window : -1;  // tokens k > wlo, or k < sinks
      const int t_first = s.n - s.rows + min(row_base + mt * 128, row_all - 1) / p.group;  // positions of the tile's rows
      const int t_last = s.n - s.rows + (min(row_base + mt * 128 + 128, row_all) - 1) / p.group;
      const bool ragged = row_base + mt * 128 + 128 > row_all;
      const float cs = fmaxf(s_undo[tid] * fabsf(p.scale_log2) * kref, 1.2e-38f);  // not 0: hidden scores are -inf
      float m = -INFINITY, l = 0.f;
      bool ok = mt == 0 || x.two;
      for (int j = 0; ok && j < n; ++j) {
        const int base = x.base_of(x.i0 + j);
        const bool masked = bad || ragged || base + kPTok - 1 > t_first ||
                            (p.window && base <= t_last - p.window && base + kPTok > p.sinks);
        if (!(ok = __all_sync(~0u, wait(s_full + mt, n_s + j)))) break;
        tc_fence_after();
        const int k_max = pos - base, k_min = wlo - base, k_sink = p.sinks - base;  // columns k <= k_max, k > k_min or k < k_sink
        auto hide = [&](uint32_t (&w)[16], int q) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            bool see = 16 * q + e <= k_max && (16 * q + e > k_min || 16 * q + e < k_sink);
            if (bad && see)
              see = (unsigned)c.table[(int64_t)x.b * c.width + (base + 16 * q + e) / c.block] < (unsigned)c.n_blocks;
            if (!see) w[e] = __float_as_uint(-INFINITY);
          }
        };
        // The loops are short on purpose: unrolled over the row they outgrow the instruction caches, and
        // the tile takes 1.8 times as long.
        float mx = -INFINITY;
        if (masked) {
#pragma unroll 1
          for (int q = 0; q < 8; ++q) {
            uint32_t w[16];
            __syncwarp();
            tmem_ld16(ts + 16 * q, w);
            tc_wait_ld();
            hide(w, q);
            tmem_st16(ts + 16 * q, w);
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, __uint_as_float(w[e]));
          }
          tc_wait_st();
        } else {
          __syncwarp();
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
        if (__any_sync(~0u, mx > m + kSlack)) {
          const float top = mx > m + kSlack ? mx : m;
          const float f = top == m ? 1.f : ex2(m - top);
          m = top;
          l *= f;
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
        {
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
          }
        }
        l += ls.x + ls.y;
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready + mt);
      }
      // ---- the row's result
      const bool have = ok && n > 0 && __all_sync(~0u, wait(o_full, n_o));
      if (have) tc_fence_after();
      if (ok && (have || n <= 0)) {
        const bool whole = x.whole;
        const float inv = whole ? (l == 0.f ? 0.f : vref / l) : vref;
        float* part = p.part + (2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1)) * prompt_part<D>();
        const int64_t at = live ? (int64_t)(s.row0 + rr / p.group) * p.heads + h * p.group + rr % p.group : 0;
        // a whole item's rows go through the query rows' place (all products are done), to be written
        // 16 lanes a row; a piece's [dim / 4][row] as they come
        uint8_t* stage = sm + L::q + warp * 32 * D * 2;
#pragma unroll
        for (int q = 0; q < D / 32; ++q) {
          uint32_t v[32];
          __syncwarp();
          if (have) {
            tmem_ld32(to + 32 * q, v);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float o[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = __uint_as_float(v[e + k]) * inv;
            if (whole) {
              const uint2 y = pack4(p.act, make_float4(o[0], o[1], o[2], o[3])), z = pack4(p.act, make_float4(o[4], o[5], o[6], o[7]));
              const int ch = 4 * q + e / 8;
              *reinterpret_cast<uint4*>(stage + lane * D * 2 + ((ch ^ (lane & 7)) << 4)) = make_uint4(y.x, y.y, z.x, z.y);
            } else {
              float4* to4 = reinterpret_cast<float4*>(part) + (8 * q + e / 4) * kPRows + tid;
              to4[0] = make_float4(o[0], o[1], o[2], o[3]);
              to4[kPRows] = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
        }
        __syncwarp();
        if (whole) {
          constexpr int LR = D / 8, RI = 32 / LR;  // lanes a row, rows a store
#pragma unroll 4
          for (int i = 0; i < 32; i += RI) {
            const int row = i + lane / LR, ch = lane % LR, r2 = row_base + 32 * warp + row;
            if (r2 < row_all) {
              const int64_t o = (int64_t)(s.row0 + r2 / p.group) * p.heads + h * p.group + r2 % p.group;
              *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + 2 * (o * D + 8 * ch)) =
                  *reinterpret_cast<const uint4*>(stage + row * D * 2 + ((ch ^ (row & 7)) << 4));
            }
          }
        }
        if (live) {
          if (whole) p.lse[at] = lse_of(m, l);
          else {
            part[kPRows * D + tid] = m;
            part[kPRows * D + kPRows + tid] = l;
          }
        }
        tc_fence_before();
      }
      if (tid == 0) {  // everyone has read them: the converters, before this piece's last tile
        s_ref[0] = s_ref[1] = 0;
        s_bad = 0;
      }
      named_bar_sync(1, kWorkers);
      if (s_abort) break;
      tc_fence_after();
      if (mt == 0 || x.two) n_s += n;
      if (n > 0) ++n_o;
      u += x.len;
    }
  } else if (warp < 12) {
    // ---------------------------------------------------------------- keys and values
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegConvert));
    uint32_t n_tile = 0;
    while (u < u_end) {
      find_piece(pp, u, u_end, pi, x);
      const int n = x.n, h = x.h, i0 = x.i0, lo_x = x.lo_x;
      const Span& sp = x.sp;
      constexpr int KC = D / 64;  // 16-byte chunks a lane takes of a token
      const int cw = warp - 8, kt = lane & 7, kc = lane >> 3;  // token of 8, chunk of 4 (of 64 dims)
      uint4 kx[4][KC], vx[4][KC];
      float kr[2], vr[2];  // scales of the warp's two 16-token parts
      int id[2], id_next[2];
      auto ids = [&](int i, int (&to)[2]) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = x.base_of(i) + 32 * cw + 16 * e;
          to[e] = -1;
          if (i < i0 + n && tok < sp.end && !(tok + 15 < lo_x && tok >= p.sinks))
            to[e] = kv_block_at(c, x.b, tok / c.block, nullptr);
        }
      };
      auto load = [&](int i, const uint8_t* codes, const float* scales, uint4 (&to)[4][KC], float (&sc)[2]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int e = q >> 1, tok = x.base_of(i) + 32 * cw + 8 * q + kt;
          const uint8_t* src = codes + ((((int64_t)id[e] * c.heads + h) * c.block + (tok & (c.block - 1))) * D + 16 * kc);
#pragma unroll
          for (int cc = 0; cc < KC; ++cc)
            to[q][cc] = id[e] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>(src + 64 * cc));
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) sc[e] = id[e] < 0 ? 0.f : __ldg(scales + (int64_t)id[e] * c.heads + h);
      };
      auto mul = [](uint32_t w, __half2 f) {
        const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&w), f);
        return *reinterpret_cast<const uint32_t*>(&y);
      };
      auto put = [&](uint8_t* dst, int base, bool clean, const uint4 (&from)[4][KC], const float (&sc)[2], float ref) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int t = 32 * cw + 8 * q + kt;
          const __half2 f = __float2half2_rn(sc[q >> 1] / ref);
          const bool zero = !clean && !x.seen(p, base + t);
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
      ids(i0, id);
      if (n > 0) {
        load(i0, c.k, c.k_scale, kx, kr);
        load(i0, c.v, c.v_scale, vx, vr);
      }
      named_bar_sync(1, kWorkers);
      const float kref = fmaxf(__uint_as_float(s_ref[0]), pow2f(-126)), vref = fmaxf(__uint_as_float(s_ref[1]), pow2f(-126));
      for (int j = 0; j < n; ++j) {
        const uint32_t cnt = n_tile + j, slot = cnt & 1, use = cnt >> 1;
        const int i = i0 + j, base = x.base_of(i);
        const bool clean = base + kPTok <= sp.end && (base >= lo_x || base + kPTok <= p.sinks);
        ids(i + 1, id_next);
        if (use > 0 && !wait(k_empty + slot, use - 1)) break;
        put(sm + L::k + slot * L::kTile, base, clean, kx, kr, kref);
        if (lane == 0) mbar_arrive(k_full + slot);
        id[0] = id_next[0];
        id[1] = id_next[1];
        if (j + 1 < n) load(i + 1, c.k, c.k_scale, kx, kr);
        if (use > 0 && !wait(v_empty + slot, use - 1)) break;
        put(sm + L::v + slot * L::kTile, base, clean, vx, vr, vref);
        if (lane == 0) mbar_arrive(v_full + slot);
        if (j + 1 < n) load(i + 1, c.v, c.v_scale, vx, vr);
      }
      named_bar_sync(1, kWorkers);
      if (s_abort) break;
      n_tile += n;
      u += x.len;
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegMma));
    if (warp == 12) {
      // -------------------------------------------------------------- products
      constexpr uint32_t id_qk = idesc_f16(0, 128, kPTok), id_pv = idesc_f16(0, 128, D) | kIdescBMnMajor;
      uint32_t n_tile = 0, n1 = 0;  // tiles so far (p_ready[0], the rings); completions of p_ready[1]
      while (u < u_end) {
        find_piece(pp, u, u_end, pi, x);
        const int n = x.n;
        const bool two = x.two;
        named_bar_sync(1, kWorkers);
        if (n > 0) {
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
          auto pv = [&](int mt, uint32_t slot, bool more) {
            const uint64_t dv = smem_desc_sw128(sv + slot * L::kTile, L::kHalf);
#pragma unroll
            for (int y = 0; y < kPTok / 16; ++y)
              if (elect_one()) umma_ts(t_o(mt), t_s(mt) + 8 * y, dv + y * (2048 >> 4), id_pv, more || y != 0);
          };
          auto all = [&](uint64_t* b, uint32_t k) { return __all_sync(~0u, wait(b, k)) != 0; };
          bool ok = all(k_full + (n_tile & 1), n_tile >> 1);
          if (ok) {
            tc_fence_after();
            qk(0, n_tile & 1);
            if (two) qk(1, n_tile & 1);
            done(k_empty + (n_tile & 1));
          }
          for (int j = 0; ok && j < n; ++j) {
            const uint32_t cnt = n_tile + j, slot = cnt & 1, nslot = slot ^ 1;
            if (!(ok = all(v_full + slot, cnt >> 1) && all(p_ready, cnt))) break;
            tc_fence_after();
            pv(0, slot, j > 0);
            if (j + 1 < n) {
              if (!(ok = all(k_full + nslot, (cnt + 1) >> 1))) break;
              tc_fence_after();
              qk(0, nslot);
            }
            if (two) {
              if (!(ok = all(p_ready + 1, n1 + j))) break;
              tc_fence_after();
              pv(1, slot, j > 0);
            }
            done(v_empty + slot);
            if (j + 1 < n) {
              if (two) qk(1, nslot);
              done(k_empty + nslot);
            }
          }
          if (ok) done(o_full);
        }
        __syncwarp();
        named_bar_sync(1, kWorkers);
        if (s_abort) break;
        tc_fence_after();
        n_tile += n;
        if (two) n1 += n;
        u += x.len;
      }
      // no product may still be running when tensor memory goes
      if (elect_one()) umma_commit(drain);
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
  if (warp == 12) tmem_dealloc<512>(tm);
}

// CTA j joins the item that crosses the boundary between pieces j and j + 1, if that is its first one.
constexpr int kJoinThreads = 512;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) kv_prompt_join_kernel(PromptParams pp, int ctas) {
  const AttendParams& p = pp.a;
  pdl_wait();
  const int64_t total = *pp.total, share = max((total + ctas - 1) / ctas, (int64_t)1);
  const int64_t u = (int64_t)(blockIdx.x + 1) * share;
  if (u >= total) return;
  const int pi = pair_of(pp.list, *pp.n_pairs, u);
  const PromptItem item = pp.list[pi];
  const int64_t per = (pp.list[pi + 1].off - item.off) / p.c.heads;
  const int h = (int)((u - item.off) / per);
  const int64_t begin = item.off + h * per, last = begin + per - 1;
  if (begin == u || begin / share != blockIdx.x) return;
  const int c0 = blockIdx.x, c1 = (int)(last / share);
  const KvSeq s = kv_seq(p.c, item.b);
  const int row_all = s.rows * p.group;
  for (int e = threadIdx.x; e < kPRows * D / 4; e += kJoinThreads) {
    const int rr = e % kPRows, d = e / kPRows * 4, r2 = item.rt * kPRows + rr;
    if (r2 >= row_all) continue;
    auto slot = [&](int j) {
      const int k = (j == c0 && begin != (int64_t)c0 * share) ? 1 : 0;
      return p.part + (2 * (int64_t)j + k) * prompt_part<D>();
    };
    float M = -INFINITY;
    for (int j = c0; j <= c1; ++j) M = fmaxf(M, __ldcg(slot(j) + kPRows * D + rr));
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int j = c0; j <= c1; ++j) {
      const float* ps = slot(j);
      const float mj = __ldcg(ps + kPRows * D + rr), f = mj == M ? 1.f : ex2(mj - M);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(ps) + d / 4 * kPRows + rr);
      l += __ldcg(ps + kPRows * D + kPRows + rr) * f;
      o.x += x.x * f;
      o.y += x.y * f;
      o.z += x.z * f;
      o.w += x.w * f;
    }
    const int64_t at = (int64_t)(s.row0 + r2 / p.group) * p.heads + h * p.group + r2 % p.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + 2 * (at * D + d)) =
        pack4(p.act, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (d == 0) p.lse[at] = lse_of(M, l);
  }
}

bool kv_prompt_takes(const KvView& c, int group) { return (int64_t)c.n_rows * group >= 128ll * c.batch; }

static int64_t max_pairs(const KvView& c, int group) { return (int64_t)c.n_rows * group / kPRows + c.batch; }

static size_t list_bytes(const KvView& c, int group) {
  return (size_t)((max_pairs(c, group) + 2) * (int64_t)sizeof(PromptItem) + 127) / 128 * 128;
}

size_t kv_prompt_workspace(const KvView& c, int group) {
  return list_bytes(c, group) + (size_t)2 * kPMaxCtas * (c.dim == 128 ? prompt_part<128>() : prompt_part<64>()) * 4;
}

template <int D, int FMT>
static int run(const PromptParams& pp, int ctas, cudaStream_t st) {
  constexpr size_t smem = PromptSmem<D>::bytes;
  const KvView& c = pp.a.c;
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kv_prompt_kernel<D, FMT>), (int)smem)) return rc;
  kv_prompt_plan_kernel<<<1, kPlanThreads, sizeof(int) * (c.batch + 1), st>>>(pp);
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
  cfg.gridDim = dim3(ctas - 1);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return record_cuda(cudaLaunchKernelEx(&cfg, kv_prompt_join_kernel<D>, pp, ctas));
}

int kv_prompt_run(const AttendParams& a, void* workspace, cudaStream_t st) {
  PromptParams pp{a, nullptr, nullptr, nullptr};
  const size_t list = list_bytes(a.c, a.group);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  pp.list = reinterpret_cast<PromptItem*>(ws + sizeof(PromptItem));
  pp.total = reinterpret_cast<int64_t*>(ws);
  pp.n_pairs = reinterpret_cast<int*>(ws + 8);
  pp.a.part = reinterpret_cast<float*>(ws + list);
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  const int64_t units = max_pairs(a.c, a.group) * a.c.heads * (((int64_t)a.c.width * a.c.block + kPTok - 1) / kPTok + kPOver);
  const int ctas = (int)std::min({(int64_t)sms, (int64_t)kPMaxCtas, units});
  if (a.c.dim == 128)
    return a.c.format == DUPLEX_KV_E4M3 ? run<128, DUPLEX_KV_E4M3>(pp, ctas, st) : run<128, DUPLEX_KV_INT8>(pp, ctas, st);
  return a.c.format == DUPLEX_KV_E4M3 ? run<64, DUPLEX_KV_E4M3>(pp, ctas, st) : run<64, DUPLEX_KV_INT8>(pp, ctas, st);
}

}  // namespace duplex
