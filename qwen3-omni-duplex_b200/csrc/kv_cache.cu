// The 8-bit paged KV cache's writers: append (new keys and values to codes) and eviction (the
// tokens with the largest accumulated attention weights move, in order, to other blocks).
//
// One CTA owns one (block, head) of the keys or of the values, so that block's scale, its older
// tokens' new codes and its new tokens' codes need no atomics and no second kernel.  Both are
// bound by their bytes (append reads 2 bytes and writes 1 per element, eviction reads 1 and
// writes 1): the block's values stay in registers between the search for the largest and the
// rounding, so each is read once.  Short CTAs with a chain of dependent loads (offsets, length, block id,
// rows): what counts is how many are on an SM, so the rounds are a template argument and registers bounded.
// One B200, captured calls one after another: 13,000 new tokens of 4 sequences, 4 KV heads of 128, 13.6 us
// (2.4 TB/s; with 98 registers a thread 35 us); 12 sequences of 16,384 tokens to 8192 77 us, 28 of them the
// selection.
#include <algorithm>
#include <type_traits>

#include "kv.cuh"

namespace duplex {

constexpr int kThreads = 256;  // 16 elements each: R = 1, 2 or 4 rounds for a block's values

DEVI float block_max(float x, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  float m = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
  return m;
}

DEVI float finite_or_zero(float x, bool& bad) {
  if (isfinite(x)) return x;
  bad = true;
  return 0.f;
}

struct AppendParams {
  KvView c;
  const void *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int32_t* err;
};

// Work item w of a sequence's touched blocks: sequence b owns items [cu[b]/P + 2b, cu[b+1]/P + 2(b+1)),
// which is never fewer than the blocks that its rows touch.
template <int FMT, int ACT, int kRounds>
__global__ void __launch_bounds__(kThreads, kRounds == 1 ? 6 : kRounds == 2 ? 4 : 2) kv_append_kernel(AppendParams p) {
  __shared__ float red[kThreads / 32];
  const KvView& c = p.c;
  const int P = c.block, D = c.dim, h = blockIdx.y, tid = threadIdx.x;
  const bool val = blockIdx.z != 0;
  const int64_t w = blockIdx.x;
  // Every CTA finds out whether the offsets fall before it stores: a thread has a pair of them, on their way from here,
  // and what they say goes with the values' maximum.
  int2 cu = make_int2(0, 0);
  if (c.cu && tid < c.batch) cu = make_int2(c.cu[tid], c.cu[tid + 1]);
  // the last b whose first item is <= w, 32 sequences a look
  int lo = 0, left = c.batch;
  const int lane = tid & 31;
  while (left > 1) {
    const int step = (left + 31) / 32, at = lo + lane * step;
    const bool before = at < lo + left && kv_seq(c, at).row0 / P + 2ll * at <= w;
    const int i = 31 - __clz(__ballot_sync(~0u, before) | 1u);
    left = min(step, lo + left - (lo + i * step));
    lo += i * step;
  }
  const int b = lo;
  const KvSeq s = kv_seq(c, b);
  auto idle = [&] {
    if (offsets_fall(c)) set_error(p.err, DUPLEX_DEVERR_OFFSETS);
  };
  if (s.rows == 0) return idle();
  const int first = s.first;  // slot of the sequence's first new token (< 0: no room for it)
  const int64_t item = w - (s.row0 / P + 2ll * b);
  if (item < 0) return idle();  // rows before the first sequence's
  const int64_t col = max(first, 0) / P + item;
  if (col * P >= s.n) {  // no more tokens, or no more table (which some CTA's block is past if kv_len is)
    if (tid == 0 && too_long(c, s)) set_error(p.err, DUPLEX_DEVERR_LENGTH);
    return idle();
  }
  const int id = kv_block_at(c, b, (int)col, tid == 0 ? p.err : nullptr);
  if (id < 0) return;
  const int base = (int)col * P;                  // slot of the block's first token
  const int new0 = max(first - base, 0);          // in-block slots [new0, new1) are new
  const int new1 = min(s.n - base, P);
  const uint8_t* src = static_cast<const uint8_t*>(val ? p.v : p.k) + 2 * (h * (val ? p.v_head : p.k_head));
  const int64_t row_stride = val ? p.v_row : p.k_row;
  const int64_t at = ((int64_t)id * c.heads + h) * P;
  uint8_t* codes = (val ? c.v : c.k) + at * D;
  float* scale = (val ? c.v_scale : c.k_scale) + (int64_t)id * c.heads + h;
  const int per = D / 16, n_vec = P * per;

  uint4 x[kRounds][2];
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = tid + i * kThreads, tok = e / per, d = (e - tok * per) * 16;
    x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
    if (e < n_vec && tok >= new0 && tok < new1) {
      const uint4* g = reinterpret_cast<const uint4*>(src + 2 * ((int64_t)(s.row0 + base + tok - first) * row_stride + d));
      x[i][0] = __ldg(g);
      x[i][1] = __ldg(g + 1);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = (&x[i][j >> 2].x)[j & 3];
      float2 f = act2<ACT>(u);
      f.x = finite_or_zero(f.x, bad);
      f.y = finite_or_zero(f.y, bad);
      amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
  }
  asm volatile("" : "+r"(cu.x), "+r"(cu.y));  // looked at no earlier: 13,000 tokens 13.9 us if they are, 13.6 here
  bool fall = cu.y < cu.x;
  for (int i = tid + kThreads; c.cu && i < c.batch; i += kThreads) fall |= offset_falls(c, i);
  if (fall) set_error(p.err, DUPLEX_DEVERR_OFFSETS);
  amax = block_max(fall ? INFINITY : amax, red);  // (the values are finite)
  if (amax == INFINITY) return;
  if (bad) set_error(p.err, DUPLEX_DEVERR_NONFINITE);
  int e2 = KvFmt<FMT>::exponent(amax);
  if (new0 > 0) {  // older tokens in the block: its scale never falls, and their codes follow it
    const float old = *scale;
    const uint32_t u0 = __float_as_uint(old);  // its least power of two not below, whoever wrote it
    e2 = max(e2, min((int)((u0 >> 23) & 255) - 127 + ((u0 & 0x7FFFFFu) ? 1 : 0), 127));
    const float two = pow2f(e2);
    if (two != old) {
      const float f = old / two;  // of two powers of two: exact
      for (int e = tid; e < new0 * per; e += kThreads) {
        uint4 q = *reinterpret_cast<const uint4*>(codes + e * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t& u = (&q.x)[j];
          const float2 a = h2f(KvFmt<FMT>::lo(u)), d = h2f(KvFmt<FMT>::hi(u));
          u = KvFmt<FMT>::encode4(a.x * f, a.y * f, d.x * f, d.y * f);
        }
        *reinterpret_cast<uint4*>(codes + e * 16) = q;
      }
    }
    __syncthreads();  // the old scale is read by all before it changes
  }
  const float inv = e2 == 127 ? 0.5f * pow2f(-126) : pow2f(-e2);
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = tid + i * kThreads, tok = e / per;
    if (e < n_vec && tok >= new0 && tok < new1) {
      uint4 q;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bool ignore = false;
        float2 a = act2<ACT>((&x[i][j >> 1].x)[(j & 1) * 2]), d = act2<ACT>((&x[i][j >> 1].x)[(j & 1) * 2 + 1]);
        (&q.x)[j] = KvFmt<FMT>::encode4(finite_or_zero(a.x, ignore) * inv, finite_or_zero(a.y, ignore) * inv,
                                        finite_or_zero(d.x, ignore) * inv, finite_or_zero(d.y, ignore) * inv);
      }
      *reinterpret_cast<uint4*>(codes + e * 16) = q;
    }
  }
  if (tid == 0) *scale = pow2f(e2);
  if (!val && c.weights)
    for (int i = new0 + tid; i < new1; i += kThreads) c.weights[at + i] = 0.f;
}

// ----------------------------------------------------------------- eviction
struct EvictParams {
  KvView c;
  const int32_t* dst;  // [batch][dst_width]
  int dst_width, keep, sinks, recent;
  int32_t* index;      // [batch][heads][keep] kept tokens in order, as block * P + place in it
  int32_t* new_len;    // or null
  int32_t* err;
};

// fp32 as an unsigned key of the same order; -0 is 0 and every NaN is the largest
DEVI uint32_t order_key(float x) {
  if (x == 0.f) return 0x80000000u;
  const uint32_t u = __float_as_uint(x);
  if (x != x) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;

// One CTA per (sequence, head).  The R = keep - sinks - recent largest keys of the tokens between
// sinks and recent: four passes of 8 bits find the R-th largest key (per-warp histograms), then each
// warp counts and writes its own stretch of the tokens in order: all above that key, and the first of
// those equal.  Keys stay in shared memory (SM_KEYS: up to kMaxKeys tokens), so weights and block ids
// are read once; longer sequences read them anew in each pass.
constexpr int kMaxKeys = 40 * 1024;  // and their block ids: 170 KB beside 34 KB

template <bool SM_KEYS>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(EvictParams p) {
  constexpr int W = kSelThreads / 32;
  extern __shared__ uint32_t keys[];
  __shared__ int hist[W][257];  // weights share their upper digits: one digit's counts of all warps in as many banks
  __shared__ int total[256];
  __shared__ int s_held[W], s_equal[W];
  __shared__ int s_digit, s_above;
  const KvView& c = p.c;
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  const int n = kv_seq(c, b).n;
  if (h == 0 && tid == 0 && p.new_len) p.new_len[b] = min(n, p.keep);
  if (h == 0 && tid == 0 && c.kv_len[b] > n) set_error(p.err, DUPLEX_DEVERR_LENGTH);
  int32_t* out = p.index + ((int64_t)b * c.heads + h) * p.keep;
  int32_t* ids = reinterpret_cast<int32_t*>(keys + (int64_t)c.width * c.block);  // the sequence's block ids (SM_KEYS)
  const int shift_p = __ffs(c.block) - 1;
  if (SM_KEYS) {
    for (int i = tid; i < (n + c.block - 1) / c.block; i += kSelThreads) ids[i] = kv_block_at(c, b, i, p.err);
    __syncthreads();
  }
  auto slot_of = [&](int j) -> int {  // a token's place among all blocks' tokens, or -1
    const int id = SM_KEYS ? ids[j >> shift_p] : kv_block_at(c, b, j >> shift_p, p.err);
    return id < 0 ? -1 : (id << shift_p) + (j & (c.block - 1));
  };
  if (n <= p.keep) {
    for (int j = tid; j < n; j += kSelThreads) out[j] = slot_of(j);
    return;
  }
  auto read_key = [&](int j) -> uint32_t {
    const int s = slot_of(j);
    return s < 0 ? 0u : order_key(c.weights[(((int64_t)(s >> shift_p) * c.heads + h) << shift_p) + (s & (c.block - 1))]);
  };
  const int lo = p.sinks, hi = n - p.recent;  // keep >= sinks + recent and n > keep, so lo < hi
  if (SM_KEYS) {
#pragma unroll 8
    for (int j = lo + tid; j < hi; j += kSelThreads) keys[j] = read_key(j);
  }
  auto key_of = [&](int j) -> uint32_t { return SM_KEYS ? keys[j] : read_key(j); };
  int want = p.keep - p.sinks - p.recent;
  const bool none = want == 0;
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && !none; shift -= 8) {
    for (int i = tid; i < 257 * W; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kSelThreads) {
      const uint32_t u = key_of(j);
      if ((u & mask) == prefix) atomicAdd(&hist[warp][(u >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 256) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < W; ++w) sum += hist[w][tid];
      total[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // the largest digit with `want` keys at it and above: lane i has digits 255 - 8 i down
      int mine = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += total[255 - 8 * lane - e];
      int above = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(~0u, above, o);
        if (lane >= o) above += v;
      }
      const int first = __ffs(__ballot_sync(~0u, above >= want)) - 1;  // there are at least `want` keys
      if (lane == first) {
        above -= mine;
        int d = 255 - 8 * lane;
        while (above + total[d] < want) above += total[d--];
        s_digit = d;
        s_above = above;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    want -= s_above;
    __syncthreads();
  }
  // `want` of the keys equal to prefix are kept, the first ones
  const int stretch = ((n + W - 1) / W + 31) / 32 * 32, j0 = min(warp * stretch, n), j1 = min(j0 + stretch, n);
  auto look = [&](int j, bool& held, bool& eq) {
    held = eq = false;
    if (j >= j1) return;
    if (j < lo || j >= hi) held = true;
    else if (!none) {
      const uint32_t u = key_of(j);
      held = u > prefix;
      eq = u == prefix;
    }
  };
  if (SM_KEYS) __syncthreads();
  int held_n = 0, equal_n = 0;
  for (int j = j0; j < j1; j += 32) {
    bool held, eq;
    look(j + lane, held, eq);
    held_n += __popc(__ballot_sync(~0u, held));
    equal_n += __popc(__ballot_sync(~0u, eq));
  }
  if (lane == 0) {
    s_held[warp] = held_n;
    s_equal[warp] = equal_n;
  }
  __syncthreads();
  int to = 0, equal = 0;  // kept tokens and equal keys before the warp's
  for (int w = 0; w < warp; ++w) {
    to += s_held[w] + min(s_equal[w], max(want - equal, 0));
    equal += s_equal[w];
  }
  for (int j = j0; j < j1; j += 32) {
    bool held, eq;
    look(j + lane, held, eq);
    const uint32_t be = __ballot_sync(~0u, eq), below = (1u << lane) - 1;
    if (eq && equal + __popc(be & below) < want) held = true;
    const uint32_t bh = __ballot_sync(~0u, held);
    const int i = to + __popc(bh & below);
    if (held && i < p.keep) out[i] = slot_of(j + lane);
    to += __popc(bh);
    equal += __popc(be);
  }
}

// The new lengths over the old ones, once nothing reads these any more: one CTA, which has read all before it
// writes.  (By the selection or the gather, for every call, this was 0.6 to 2 of 77 us.)
__global__ void __launch_bounds__(kSelThreads) kv_lengths_kernel(KvView c, int keep, int32_t* new_len) {
  int n[DUPLEX_KV_MAX_BATCH / kSelThreads];
#pragma unroll
  for (int i = 0; i < DUPLEX_KV_MAX_BATCH / kSelThreads; ++i) {
    const int b = threadIdx.x + i * kSelThreads;
    n[i] = b < c.batch ? min(kv_seq(c, b).n, keep) : 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < DUPLEX_KV_MAX_BATCH / kSelThreads; ++i) {
    const int b = threadIdx.x + i * kSelThreads;
    if (b < c.batch) new_len[b] = n[i];
  }
}

// One CTA per (destination block, sequence and head): its tokens' codes, keys and values, are read
// where they are, and rounded at the new block's scale.
template <int FMT, int R>
__global__ void __launch_bounds__(kThreads, R == 1 ? 5 : R == 2 ? 3 : 1) kv_gather_kernel(EvictParams p) {
  __shared__ float red[2][kThreads / 32];
  const KvView& c = p.c;
  const int P = c.block, D = c.dim, tid = threadIdx.x;
  const int b = blockIdx.y / c.heads, h = blockIdx.y - b * c.heads;
  const int base = blockIdx.x * P, per = D / 16;
  // the length and the block are loaded while the selection ends, or with the tokens' places (one sequence of
  // 4096: 20.5 -> 18.4 us); the places by plain loads, since they are written while this kernel starts
  const int id = p.dst[(int64_t)b * p.dst_width + blockIdx.x];
  const int count = min(min(kv_seq(c, b).n, p.keep) - base, P);
  pdl_wait();
  const int32_t* index = p.index + ((int64_t)b * c.heads + h) * p.keep + base;
  int src[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int tok = (tid + i * kThreads) / per;
    src[i] = tok < min(P, p.keep - base) ? index[tok] : -1;
  }
  if (count <= 0) return;
  if ((unsigned)id >= (unsigned)c.n_blocks) {
    if (tid == 0) set_error(p.err, DUPLEX_DEVERR_BLOCK);
    return;
  }
#pragma unroll
  for (int i = 0; i < R; ++i)  // places past the last token are not written
    if ((tid + i * kThreads) / per >= count) src[i] = -1;
  uint4 x[2][R];
  float sc[2][R], amax[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = tid + i * kThreads, d = (e % per) * 16;
    const int64_t bh = (int64_t)(max(src[i], 0) / P) * c.heads + h, row = bh * P + (src[i] & (P - 1));
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      x[y][i] = src[i] < 0 ? make_uint4(0, 0, 0, 0) : __ldg(reinterpret_cast<const uint4*>((y ? c.v : c.k) + row * D + d));
      sc[y][i] = src[i] < 0 ? 0.f : __ldg((y ? c.v_scale : c.k_scale) + bh);
    }
  }
  const int64_t at = ((int64_t)id * c.heads + h) * P;
  for (int i = tid; i < count; i += kThreads) {
    const int s = index[i];
    c.weights[at + i] = s < 0 ? 0.f : c.weights[((int64_t)(s / P) * c.heads + h) * P + (s & (P - 1))];
  }
#pragma unroll
  for (int y = 0; y < 2; ++y) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = h2f(KvFmt<FMT>::lo((&x[y][i].x)[j])), q = h2f(KvFmt<FMT>::hi((&x[y][i].x)[j]));
        m = fmaxf(m, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(q.x), fabsf(q.y))));
      }
      amax[y] = fmaxf(amax[y], m * sc[y][i]);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) amax[y] = fmaxf(amax[y], __shfl_xor_sync(~0u, amax[y], o));
    if ((tid & 31) == 0) red[y][tid >> 5] = amax[y];
  }
  __syncthreads();
#pragma unroll
  for (int y = 0; y < 2; ++y) {
    float m = red[y][0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) m = fmaxf(m, red[y][w]);
    const int e2 = min(KvFmt<FMT>::exponent(m), 127);
    const float inv = e2 == 127 ? 0.5f * pow2f(-126) : pow2f(-e2);
    uint8_t* to = (y ? c.v : c.k) + at * D;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int e = tid + i * kThreads;
      if (e / per >= count) continue;
      const float f = fminf(sc[y][i] * inv, 3e38f);  // (of a zero token beside much smaller ones: 0 times it must be 0)
      uint4 q;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = h2f(KvFmt<FMT>::lo((&x[y][i].x)[j])), d = h2f(KvFmt<FMT>::hi((&x[y][i].x)[j]));
        (&q.x)[j] = KvFmt<FMT>::encode4(a.x * f, a.y * f, d.x * f, d.y * f);
      }
      *reinterpret_cast<uint4*>(to + e * 16) = q;
    }
    if (tid == 0) (y ? c.v_scale : c.k_scale)[(int64_t)id * c.heads + h] = pow2f(e2);
  }
}

// ----------------------------------------------------------------- checks
int kv_check(const duplex_kv_cache* c, const duplex_kv_batch* b, KvView* out) {
  if (!c || !b || !c->k || !c->v || !c->k_scale || !c->v_scale || !b->block_table || !b->kv_len)
    return DUPLEX_ERR_ARG;
  if (c->n_blocks < 1 || c->kv_heads < 1 || b->batch < 1 || b->width < 1 || b->n_rows < 0) return DUPLEX_ERR_ARG;
  if (c->format != DUPLEX_KV_E4M3 && c->format != DUPLEX_KV_INT8) return DUPLEX_ERR_DTYPE;
  if (c->dim != 64 && c->dim != 128) return DUPLEX_ERR_UNSUPPORTED;
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128) return DUPLEX_ERR_UNSUPPORTED;
  if (c->kv_heads > 65535 || b->batch > DUPLEX_KV_MAX_BATCH || (int64_t)b->batch * c->kv_heads > 65535)
    return DUPLEX_ERR_UNSUPPORTED;
  if ((int64_t)b->width * c->block + b->n_rows > 0x7FFFFFFFll - 256) return DUPLEX_ERR_UNSUPPORTED;
  if (!b->cu_rows && b->n_rows % b->batch) return DUPLEX_ERR_ARG;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return DUPLEX_ERR_ALIGN;
  const int cap = b->width * c->block;
  *out = KvView{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, c->weights,
                c->n_blocks, c->kv_heads, c->block, c->dim, c->format, b->block_table, b->kv_len, b->cu_rows,
                b->width, b->batch, b->n_rows, cap, (int)std::min((int64_t)cap + (1 << 29), (int64_t)INT32_MAX)};
  return DUPLEX_OK;
}

}  // namespace duplex

using namespace duplex;

extern "C" int duplex_kv_append(const duplex_kv_cache* cache, const duplex_kv_batch* batch, const void* k_new,
                                const void* v_new, int act_dtype, int64_t k_row_stride, int64_t k_head_stride,
                                int64_t v_row_stride, int64_t v_head_stride, int32_t* err, void* stream) {
  AppendParams p{};
  if (int rc = kv_check(cache, batch, &p.c)) return rc;
  if (act_dtype != DUPLEX_DTYPE_F16 && act_dtype != DUPLEX_DTYPE_BF16) return DUPLEX_ERR_DTYPE;
  if (batch->n_rows == 0) return DUPLEX_OK;
  if (!k_new || !v_new) return DUPLEX_ERR_ARG;
  if ((((uintptr_t)k_new | (uintptr_t)v_new) & 15) || ((k_row_stride | k_head_stride | v_row_stride | v_head_stride) & 7))
    return DUPLEX_ERR_ALIGN;
  p.k = k_new;
  p.v = v_new;
  p.k_row = k_row_stride;
  p.k_head = k_head_stride;
  p.v_row = v_row_stride;
  p.v_head = v_head_stride;
  p.err = err;
  const int64_t items = batch->n_rows / cache->block + 2ll * batch->batch;
  const dim3 grid((unsigned)items, cache->kv_heads, 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rounds = (cache->block * cache->dim / 16 + kThreads - 1) / kThreads;
  auto go = [&](auto fmt, auto act) {
    constexpr int F = decltype(fmt)::value, A = decltype(act)::value;
    if (rounds == 1) kv_append_kernel<F, A, 1><<<grid, kThreads, 0, st>>>(p);
    else if (rounds == 2) kv_append_kernel<F, A, 2><<<grid, kThreads, 0, st>>>(p);
    else kv_append_kernel<F, A, 4><<<grid, kThreads, 0, st>>>(p);
  };
  using E4 = std::integral_constant<int, DUPLEX_KV_E4M3>;
  using I8 = std::integral_constant<int, DUPLEX_KV_INT8>;
  using F16 = std::integral_constant<int, DUPLEX_DTYPE_F16>;
  using B16 = std::integral_constant<int, DUPLEX_DTYPE_BF16>;
  const bool f16 = act_dtype == DUPLEX_DTYPE_F16;
  if (cache->format == DUPLEX_KV_E4M3) f16 ? go(E4{}, F16{}) : go(E4{}, B16{});
  else f16 ? go(I8{}, F16{}) : go(I8{}, B16{});
  return record_cuda(cudaGetLastError());
}

extern "C" int duplex_kv_evict_workspace_bytes(const duplex_kv_cache* cache, const duplex_kv_batch* batch,
                                               int32_t keep, size_t* bytes) {
  KvView v;
  if (int rc = kv_check(cache, batch, &v)) return rc;
  if (!bytes || keep < 1) return DUPLEX_ERR_ARG;
  *bytes = (size_t)batch->batch * cache->kv_heads * keep * 4;
  return DUPLEX_OK;
}

extern "C" int duplex_kv_evict(const duplex_kv_cache* cache, const duplex_kv_batch* batch, const int32_t* dst_table,
                               int32_t dst_width, int32_t keep, int32_t sinks, int32_t recent, int32_t* new_len,
                               void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  EvictParams p{};
  if (int rc = kv_check(cache, batch, &p.c)) return rc;
  if (!cache->weights || !dst_table || !new_len || keep < 1 || sinks < 0 || recent < 0) return DUPLEX_ERR_ARG;
  if ((int64_t)cache->n_blocks * cache->block > 0x7FFFFFFFll) return DUPLEX_ERR_UNSUPPORTED;  // a token's place is 32 bits
  if ((int64_t)sinks + recent > keep || (int64_t)dst_width * cache->block < keep) return DUPLEX_ERR_ARG;
  size_t need = 0;
  duplex_kv_evict_workspace_bytes(cache, batch, keep, &need);
  if (!workspace || workspace_bytes < need) return DUPLEX_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DUPLEX_ERR_ALIGN;
  p.dst = dst_table;
  p.dst_width = dst_width;
  p.keep = keep;
  p.sinks = sinks;
  p.recent = recent;
  p.index = static_cast<int32_t*>(workspace);
  // where the lengths overlap, the selections of other heads have still to read what one would write
  const bool in_place = new_len < batch->kv_len + batch->batch && batch->kv_len < new_len + batch->batch;
  p.new_len = in_place ? nullptr : new_len;
  p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 heads(cache->kv_heads, batch->batch);
  const int64_t cap = (int64_t)batch->width * cache->block;
  if (cap <= kMaxKeys) {
    if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kv_select_kernel<true>), kMaxKeys * 4 + kMaxKeys / 16 * 4))
      return rc;
    kv_select_kernel<true><<<heads, kSelThreads, (size_t)(cap + batch->width) * 4, st>>>(p);
  } else {
    kv_select_kernel<false><<<heads, kSelThreads, 0, st>>>(p);
  }
  if (int rc = record_cuda(cudaGetLastError())) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((keep + cache->block - 1) / cache->block, batch->batch * cache->kv_heads);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int rounds = (cache->block * cache->dim / 16 + kThreads - 1) / kThreads;
  auto go = [&](auto fmt) {
    constexpr int F = decltype(fmt)::value;
    return rounds == 1   ? cudaLaunchKernelEx(&cfg, kv_gather_kernel<F, 1>, p)
           : rounds == 2 ? cudaLaunchKernelEx(&cfg, kv_gather_kernel<F, 2>, p)
                         : cudaLaunchKernelEx(&cfg, kv_gather_kernel<F, 4>, p);
  };
  if (int rc = record_cuda(cache->format == DUPLEX_KV_E4M3 ? go(std::integral_constant<int, DUPLEX_KV_E4M3>{})
                                                           : go(std::integral_constant<int, DUPLEX_KV_INT8>{})))
    return rc;
  if (!in_place) return DUPLEX_OK;
  kv_lengths_kernel<<<1, kSelThreads, 0, st>>>(p.c, keep, new_len);
  return record_cuda(cudaGetLastError());
}
