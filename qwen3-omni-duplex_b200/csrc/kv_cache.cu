// The 8-bit paged KV cache's writers: append (new keys and values to codes) and eviction (the
// tokens with the largest accumulated attention weights move, in order, to other blocks).
//
// One CTA owns one (block, head) of the keys or of the values, so that block's scale, its older
// tokens' new codes and its new tokens' codes need no atomics and no second kernel.  Both are
// bound by their bytes (append reads 2 bytes and writes 1 per element, eviction reads 1 and
// writes 1): the block's values stay in registers between the search for the largest and the
// rounding, so each is read once.
#include "kv.cuh"

namespace duplex {

constexpr int kThreads = 256;  // 16 elements each, so 128 x 128 values are 4 rounds
constexpr int kRounds = 4;

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
template <int FMT, int ACT>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(AppendParams p) {
  __shared__ float red[kThreads / 32];
  const KvView& c = p.c;
  const int P = c.block, D = c.dim, h = blockIdx.y, tid = threadIdx.x;
  const bool val = blockIdx.z != 0;
  const int64_t w = blockIdx.x;
  int lo = 0, hi = c.batch - 1;
  while (lo < hi) {  // the last b whose first item is <= w
    const int mid = (lo + hi + 1) >> 1;
    if (kv_seq(c, mid).row0 / P + 2ll * mid <= w) lo = mid; else hi = mid - 1;
  }
  const int b = lo;
  const KvSeq s = kv_seq(c, b);
  if (s.rows == 0) return;
  const int first = s.n - s.rows;  // slot of the sequence's first new token (< 0: no room for it)
  const int64_t item = w - (s.row0 / P + 2ll * b);
  const int64_t col = max(first, 0) / P + item;
  if (col * P >= s.n) return;
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
  if (bad) set_error(p.err, DUPLEX_DEVERR_NONFINITE);
  amax = block_max(amax, red);
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
  int32_t* index;      // [batch][heads][keep] kept tokens in order (sequences with more than keep)
  int32_t* new_len;
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
// sinks and recent: four passes of 8 bits find the R-th largest key (per-warp histograms in shared
// memory), a last pass writes the kept tokens in order: all above it, and the first of those equal.
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(EvictParams p) {
  __shared__ int hist[kSelThreads / 32][256];
  __shared__ int warp_sum[2][kSelThreads / 32];
  __shared__ int s_digit, s_above;
  const KvView& c = p.c;
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = kv_seq(c, b).n;
  if (h == 0 && tid == 0) p.new_len[b] = min(n, p.keep);
  if (n <= p.keep) return;
  const int lo = p.sinks, hi = n - p.recent;  // keep >= sinks + recent and n > keep, so lo < hi
  int want = p.keep - p.sinks - p.recent;
  int32_t* out = p.index + ((int64_t)b * c.heads + h) * p.keep;
  auto key_of = [&](int j) -> uint32_t {
    const int id = kv_block_at(c, b, j / c.block, p.err);
    return id < 0 ? 0u : order_key(c.weights[((int64_t)id * c.heads + h) * c.block + j % c.block]);
  };
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
    for (int i = tid; i < 256 * (kSelThreads / 32); i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
    for (int j = lo + tid; j < hi; j += kSelThreads) {
      const uint32_t u = key_of(j);
      if ((u & mask) == prefix) atomicAdd(&hist[warp][(u >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 256) {
      int sum = 0;
      for (int w = 0; w < kSelThreads / 32; ++w) sum += hist[w][tid];
      hist[0][tid] = sum;
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + hist[0][d] < want) above += hist[0][d--];
      s_digit = d;
      s_above = above;
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    mask |= 255u << shift;
    want -= s_above;
    __syncthreads();
  }
  // now `want` of the keys equal to prefix are kept, the first ones
  const bool none = p.keep == p.sinks + p.recent;
  int kept = 0, equal = 0;  // kept tokens and equal keys before this round's
  for (int j0 = 0; j0 < n; j0 += kSelThreads) {
    const int j = j0 + tid;
    bool held = false, eq = false;
    if (j < n) {
      if (j < lo || j >= hi) held = true;
      else if (!none) {
        const uint32_t u = key_of(j);
        held = u > prefix;
        eq = u == prefix;
      }
    }
    const uint32_t be = __ballot_sync(~0u, eq);
    if (lane == 0) warp_sum[0][warp] = __popc(be);
    __syncthreads();
    int e_before = 0, e_all = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) e_before += warp_sum[0][w];
      e_all += warp_sum[0][w];
    }
    if (eq && equal + e_before + __popc(be & ((1u << lane) - 1)) < want) held = true;
    const uint32_t bh = __ballot_sync(~0u, held);
    if (lane == 0) warp_sum[1][warp] = __popc(bh);
    __syncthreads();
    int h_before = 0, h_all = 0;
    for (int w = 0; w < kSelThreads / 32; ++w) {
      if (w < warp) h_before += warp_sum[1][w];
      h_all += warp_sum[1][w];
    }
    const int to = kept + h_before + __popc(bh & ((1u << lane) - 1));
    if (held && to < p.keep) out[to] = j;
    kept += h_all;
    equal += e_all;
    __syncthreads();
  }
}

// One CTA per (destination block, sequence and head, keys or values): its tokens' codes are read
// where they are, brought to the largest source scale's value, and rounded at the new scale.
template <int FMT>
__global__ void __launch_bounds__(kThreads) kv_gather_kernel(EvictParams p) {
  __shared__ float red[kThreads / 32];
  const KvView& c = p.c;
  const int P = c.block, D = c.dim, tid = threadIdx.x;
  const bool val = blockIdx.z != 0;
  const int b = blockIdx.y / c.heads, h = blockIdx.y - b * c.heads;
  const int n = kv_seq(c, b).n, kept = min(n, p.keep);
  const int base = blockIdx.x * P;
  if (base >= kept) return;
  const int id = p.dst[(int64_t)b * p.dst_width + blockIdx.x];
  if ((unsigned)id >= (unsigned)c.n_blocks) {
    if (tid == 0) set_error(p.err, DUPLEX_DEVERR_BLOCK);
    return;
  }
  const int count = min(kept - base, P);
  const int32_t* index = n > p.keep ? p.index + ((int64_t)b * c.heads + h) * p.keep : nullptr;
  const uint8_t* codes = val ? c.v : c.k;
  const float* scales = val ? c.v_scale : c.k_scale;
  const int per = D / 16;
  uint4 x[kRounds];
  float sc[kRounds];
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = tid + i * kThreads, tok = e / per, d = (e - tok * per) * 16;
    x[i] = make_uint4(0, 0, 0, 0);
    sc[i] = 0.f;
    if (tok < count) {
      const int j = index ? index[base + tok] : base + tok;
      const int src = kv_block_at(c, b, j / P, p.err);
      if (src >= 0) {
        const int64_t row = ((int64_t)src * c.heads + h) * P + j % P;
        x[i] = __ldg(reinterpret_cast<const uint4*>(codes + row * D + d));
        sc[i] = scales[(int64_t)src * c.heads + h];
      }
    }
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = h2f(KvFmt<FMT>::lo((&x[i].x)[j])), q = h2f(KvFmt<FMT>::hi((&x[i].x)[j]));
      m = fmaxf(m, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(q.x), fabsf(q.y))));
    }
    amax = fmaxf(amax, m * sc[i]);
  }
  amax = block_max(amax, red);
  const int e2 = KvFmt<FMT>::exponent(amax);
  const float inv = e2 >= 127 ? 0.5f * pow2f(-126) : pow2f(-e2);
  const int64_t at = ((int64_t)id * c.heads + h) * P;
  uint8_t* to = (val ? c.v : c.k) + at * D;
#pragma unroll
  for (int i = 0; i < kRounds; ++i) {
    const int e = tid + i * kThreads, tok = e / per;
    if (tok >= count) continue;
    const float f = sc[i] * inv;
    uint4 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = h2f(KvFmt<FMT>::lo((&x[i].x)[j])), d = h2f(KvFmt<FMT>::hi((&x[i].x)[j]));
      (&q.x)[j] = KvFmt<FMT>::encode4(a.x * f, a.y * f, d.x * f, d.y * f);
    }
    *reinterpret_cast<uint4*>(to + e * 16) = q;
  }
  if (tid == 0) ((val ? c.v_scale : c.k_scale))[(int64_t)id * c.heads + h] = pow2f(min(e2, 127));
  if (!val)
    for (int i = tid; i < count; i += kThreads) {
      const int j = index ? index[base + i] : base + i;
      const int src = kv_block_at(c, b, j / P, nullptr);
      c.weights[at + i] = src < 0 ? 0.f : c.weights[((int64_t)src * c.heads + h) * P + j % P];
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
  *out = KvView{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, c->weights,
                c->n_blocks, c->kv_heads, c->block, c->dim, c->format, b->block_table, b->kv_len, b->cu_rows,
                b->width, b->batch, b->n_rows};
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
  const bool f16 = act_dtype == DUPLEX_DTYPE_F16;
  if (cache->format == DUPLEX_KV_E4M3) {
    if (f16) kv_append_kernel<DUPLEX_KV_E4M3, DUPLEX_DTYPE_F16><<<grid, kThreads, 0, st>>>(p);
    else kv_append_kernel<DUPLEX_KV_E4M3, DUPLEX_DTYPE_BF16><<<grid, kThreads, 0, st>>>(p);
  } else {
    if (f16) kv_append_kernel<DUPLEX_KV_INT8, DUPLEX_DTYPE_F16><<<grid, kThreads, 0, st>>>(p);
    else kv_append_kernel<DUPLEX_KV_INT8, DUPLEX_DTYPE_BF16><<<grid, kThreads, 0, st>>>(p);
  }
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
  p.new_len = new_len;
  p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  kv_select_kernel<<<dim3(cache->kv_heads, batch->batch), kSelThreads, 0, st>>>(p);
  if (int rc = record_cuda(cudaGetLastError())) return rc;
  const dim3 grid((keep + cache->block - 1) / cache->block, batch->batch * cache->kv_heads, 2);
  if (cache->format == DUPLEX_KV_E4M3) kv_gather_kernel<DUPLEX_KV_E4M3><<<grid, kThreads, 0, st>>>(p);
  else kv_gather_kernel<DUPLEX_KV_INT8><<<grid, kThreads, 0, st>>>(p);
  return record_cuda(cudaGetLastError());
}
