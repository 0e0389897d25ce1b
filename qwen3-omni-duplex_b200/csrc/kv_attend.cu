// Attention over the 8-bit paged KV cache for few query rows a sequence: decode, drafted tokens,
// short chunks (kv_prompt.cu takes long ones).
//
//   s_j = q . k_j * softmax_scale,  out = sum_j exp(s_j - lse) v_j,  lse = log sum_j exp(s_j)
//
// over the tokens that a row sees: j <= p, and inside the window (j > p - window) or a sink
// (j < sinks).  One pass over the cache with a running maximum.
//
// Bound by the cache's bytes: 2 dim + a little per token and KV head, read once for all query
// heads that share it.  A warp takes 32 tokens a step into the registers that mma.sync takes (keys as
// A[token][dim], values transposed as A[dim][token]; the query rows are the 8 columns, so 8 query heads
// of a group use every product), out of a ring of its own in shared memory that asynchronous copies
// fill ahead.  The codes are converted to fp16 in registers, exactly.  The products take a sixth of the
// tensor pipe; what competes with the copies is the issue of the rest (conversions, softmax, addresses),
// hence 32 tokens for one set of addresses, one vote and one rescale.
// One B200, captured calls one after another, 32 query heads on 4, dim 128, 64 sequences of 12,288 tokens
// (805 MB): 135 us, 5.9 TB/s, 91 % of a plain copy's rate.  (Before its last steps: 143 us with 32 tokens a
// step, 165 with 16, 182 with the next 16 tokens in registers instead of a ring.)  One sequence of 2000: 8.2 us,
// all of it latency (list, copies, two steps, join).
//
// The work of a launch is one list of 128-token units over (sequence, KV head, row tile); every CTA
// takes an equal, contiguous piece of it, whatever the lengths, and reads the lengths itself (a
// captured launch follows them).  Pieces that share a row tile leave partial results, which
// kv_combine_kernel joins in order: no atomics, the same bits on each run.  Few row tiles are given a
// cluster of 8 CTAs each instead, joined in the same launch.
#include <algorithm>
#include <type_traits>

#include "kv_attend.cuh"

namespace duplex {

constexpr int kWarps = 4;
constexpr int kUnit = 32 * kWarps;   // tokens
constexpr int kWUnit = 16 * kWarps;  // of kv_weights_kernel
constexpr int kMaxCtas = 148 * 4;


// The unit list of a launch: off[b] units before sequence b.  A row tile of sequence b has units(b)
// units, the most that any of its row tiles needs.
struct Plan {
  int64_t total, share;
};

// The units of a sequence where the row offsets fall: below any sum of the others, and half of
// DUPLEX_KV_MAX_BATCH of it still a number.
constexpr int64_t kFalls = -(1ll << 51);

DEVI int tiles_of(const KvSeq& s, int group, int rows) { return (int)(((int64_t)s.rows * group + rows - 1) / rows); }

DEVI int units_of(const KvSeq& s, const AttendParams& p, int rows) {
  const int all = max((s.n + kUnit - 1) / kUnit, 1);
  if (!p.window) return all;
  // a row tile's window reaches over window - 1 + (its own tokens), whose ends need not be aligned
  const int64_t span = (int64_t)p.window + (rows - 1) / p.group + 1;
  const int64_t u = (min(p.sinks, s.n) + kUnit - 1) / kUnit + (span + kUnit - 1) / kUnit + 1;
  return (int)min(u, (int64_t)all);
}

template <int ROWS, bool ITEMS = false>
DEVI Plan make_plan(const AttendParams& p, int64_t* off, int ctas) {
  __shared__ int64_t warp_sum[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = p.c.batch;
  int64_t base = 0;
  int bits = 0;
  for (int b0 = 0; b0 < B; b0 += kWarps * 32) {
    const int b = b0 + tid;
    int64_t u = 0;
    if (b < B) {
      const KvSeq s = kv_seq(p.c, b);
      u = (int64_t)p.c.heads * tiles_of(s, p.group, ROWS) * (ITEMS ? 1 : units_of(s, p, ROWS));
      if (offset_falls(p.c, b)) u = kFalls;
      if (too_long(p.c, s)) bits = DUPLEX_DEVERR_LENGTH;
    }
    int64_t incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(~0u, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    int64_t before = base, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += warp_sum[w];
      all += warp_sum[w];
    }
    if (b < B) off[b] = before + incl - u;
    base += all;
    __syncthreads();
  }
  if (tid == 0) off[B] = base;
  __syncthreads();
  if (base < 0) {
    base = 0;  // no work
    bits = DUPLEX_DEVERR_OFFSETS;
  }
  if (bits) set_error(p.err, bits);
  Plan pl;
  pl.total = base;
  pl.share = (base + ctas - 1) / ctas;
  if (pl.share < 1) pl.share = 1;
  return pl;
}

// the sequence of unit u: the last b with off[b] <= u (sequences without units are passed over)
DEVI int seq_of(const int64_t* off, int B, int64_t u) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= u) lo = mid; else hi = mid - 1;
  }
  return lo;
}

DEVI uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

// Query rows of 8: row r's 16 dims at 64 cc + 16 t, as they come.
template <int D>
DEVI void load_raw(const AttendParams& p, int64_t row, int head, int t, bool live, uint4 (&raw)[D / 64][2]) {
  const uint8_t* src = static_cast<const uint8_t*>(p.q) + 2 * (row * p.q_row + head * p.q_head);
#pragma unroll
  for (int cc = 0; cc < D / 64; ++cc)
#pragma unroll
    for (int j = 0; j < 2; ++j)
      raw[cc][j] = live ? __ldg(reinterpret_cast<const uint4*>(src + 2 * (64 * cc + 16 * t + 8 * j))) : make_uint4(0, 0, 0, 0);
}

// ... and as fp16 fragments, scaled by a power of two that brings the row's largest into [2^14, 2^15): bf16's
// 8 bits fit fp16's 11, and only values below 2^-28 of the row's largest lose bits.  Returns the factor that
// undoes it.
template <int D>
DEVI float make_q(const AttendParams& p, const uint4 (&raw)[D / 64][2], uint2 (&qf)[D / 16]) {
  float amax = 0.f;
#pragma unroll
  for (int cc = 0; cc < D / 64; ++cc)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = (&raw[cc][j].x)[i];
        const float2 f = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(w) : act2<DUPLEX_DTYPE_BF16>(w);
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
  const int ex = (int)(__float_as_uint(amax) >> 23) - 127;
  const int up = (amax == 0.f || ex == 128) ? 0 : min(14 - ex, 126);
  const float f = pow2f(up);
#pragma unroll
  for (int cc = 0; cc < D / 64; ++cc)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t w0 = (&raw[cc][s >> 1].x)[(s & 1) * 2], w1 = (&raw[cc][s >> 1].x)[(s & 1) * 2 + 1];
      const float2 a = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(w0) : act2<DUPLEX_DTYPE_BF16>(w0);
      const float2 b = p.act == DUPLEX_DTYPE_F16 ? act2<DUPLEX_DTYPE_F16>(w1) : act2<DUPLEX_DTYPE_BF16>(w1);
      qf[cc * 4 + s] = make_uint2(f2h(a.x * f, a.y * f), f2h(b.x * f, b.y * f));
    }
  return pow2f(-up);
}

template <int D>
DEVI float load_q(const AttendParams& p, int64_t row, int head, int t, bool live, uint2 (&qf)[D / 16]) {
  uint4 raw[D / 64][2];
  load_raw<D>(p, row, head, t, live, raw);
  return make_q<D>(p, raw, qf);
}

// S[nt] += K (16 tokens) . Q (8 rows), both as fragments
template <int D, int FMT, int NT>
DEVI void qk(const uint4 (&kr)[2][D / 64], const uint2 (&qf)[NT][D / 16], float (&S)[NT][4]) {
#pragma unroll
  for (int cc = 0; cc < D / 64; ++cc)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t w0 = (&kr[0][cc].x)[s], w1 = (&kr[1][cc].x)[s];
      const uint32_t a0 = KvFmt<FMT>::lo(w0), a1 = KvFmt<FMT>::lo(w1), a2 = KvFmt<FMT>::hi(w0), a3 = KvFmt<FMT>::hi(w1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) MmaOp<__half>::run(S[nt], a0, a1, a2, a3, qf[nt][cc * 4 + s].x, qf[nt][cc * 4 + s].y);
    }
}

template <int D, int NT>
constexpr int part_floats() { return 8 * NT * (D + 2); }  // O [rows][D], m [rows], l [rows]

// A warp's ring: slots of 32 tokens' keys, values and their scales.
template <int D> constexpr int stage_bytes() { return 64 * D + 128; }
template <int D, int NT> constexpr int ring_slots() { return D == 128 && NT == 1 ? 2 : 3; }

template <int D, int NT>
constexpr int front_smem() {
  const int rings = kWarps * ring_slots<D, NT>() * stage_bytes<D>(), meet = 4 * kWarps * 8 * NT * (D + 4);
  return rings > meet ? rings : meet;
}

// A slot's bytes in lines of 128 (8 chunks of 16): the chunks are turned so that the lanes that read
// together, 2 tokens x 4 chunks of the keys, 4 even tokens x 2 chunks of the values, meet no bank twice.
template <int D> DEVI int swz_k(int o) { return D == 128 ? o ^ ((o & 128) >> 1) : o; }
template <int D> DEVI int swz_v(int o) { return o ^ (((o >> (D == 128 ? 8 : 7)) & 3) << 5); }

DEVI void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
DEVI void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
DEVI void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> DEVI void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int D, int NT> constexpr int attend_ctas() { return NT == 1 ? 3 : 2; }  // an SM

// Clusters: where there are few row tiles, kCluster CTAs take one each and join it through their shared
// memories, which saves the second launch.
constexpr int kCluster = 8;

DEVI void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DEVI uint32_t cluster_addr(const void* p, int rank) {  // p of the cluster's CTA `rank`
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_u32(p)), "r"(rank));
  return d;
}
DEVI float cluster_ld(uint32_t a) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
  return x;
}
DEVI float4 cluster_ld4(uint32_t a) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(a) : "memory");
  return x;
}

template <int D, int FMT, int NT, bool CL>
__global__ void __launch_bounds__(kWarps * 32, attend_ctas<D, NT>()) kv_attend_kernel(AttendParams p) {
  constexpr int ROWS = 8 * NT, VW = D / 32, LD = D + 4, ST = ring_slots<D, NT>(), kStage = stage_bytes<D>();
  extern __shared__ __align__(128) uint8_t dyn[];
  float(*sO)[LD] = reinterpret_cast<float(*)[LD]>(dyn);  // [kWarps * ROWS], over the rings
  int64_t* off = reinterpret_cast<int64_t*>(dyn + front_smem<D, NT>());
  __shared__ float sm[kWarps][ROWS], sl[kWarps][ROWS];
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* const ring = dyn + warp * (ST * kStage);
  const int psh = __ffs(c.block) - 1;
  pdl_launch_dependents();
  __shared__ float c_m[CL ? ROWS : 1], c_l[CL ? ROWS : 1];
  const Plan plan = make_plan<ROWS, CL>(p, off, gridDim.x);
  // the CTA's piece of the units; with clusters, the cluster's row tile and the CTA's place in it
  const int rank = blockIdx.x % kCluster;
  int64_t u = CL ? blockIdx.x / kCluster : (int64_t)blockIdx.x * plan.share;
  const int64_t u_end = CL ? min(u + 1, plan.total) : min(u + plan.share, plan.total);
  if (u >= u_end) return;  // a cluster's CTAs all alike
  int b = seq_of(off, c.batch, u);
  const int64_t u_begin = u;

  while (u < u_end) {
    while (off[b + 1] <= u) ++b;
    const KvSeq s = kv_seq(c, b);
    const int rt_all = tiles_of(s, p.group, ROWS), per = CL ? 1 : units_of(s, p, ROWS);
    const int64_t r = u - off[b];
    const int it = (int)(r / per);
    int i0 = (int)(r - (int64_t)it * per), i1 = (int)min((int64_t)per, i0 + (u_end - u));
    const bool whole = !CL && i0 == 0 && i1 == per;
    const int len = i1 - i0;
    const int h = it / rt_all, rt = it - h * rt_all;
    const int row_base = rt * ROWS, row_all = s.rows * p.group;
    const int first_pos = s.first + row_base / p.group;
    const int last_row = min(row_base + ROWS, row_all) - 1;
    const int last_pos = s.first + last_row / p.group;
    const Span sp = span_of<kUnit>(p, first_pos, last_pos, s.n);
    if (CL) {
      const int n = sp.sink_units + (sp.end > sp.lo ? (sp.end - sp.lo + kUnit - 1) / kUnit : 0);
      i0 = n * rank / kCluster;
      i1 = n * (rank + 1) / kCluster;
    }

    // this warp's 32 tokens of unit i, as two parts of 16 (a block holds whole parts): the blocks' ids, or
    // -1 where no row of the tile looks
    auto base_of = [&](int i) -> int {
      return (i < sp.sink_units ? i * kUnit : sp.lo + (i - sp.sink_units) * kUnit) + 32 * warp;
    };
    auto ids_of = [&](int i) -> int2 {
      const int tok = base_of(i), lim = i < i1 ? (i < sp.sink_units ? sp.sink_end : sp.end) : 0;
      auto id = [&](int k) {
        const bool gap = p.window && k + 15 <= first_pos - p.window && k >= p.sinks;  // between sinks and window
        return (unsigned)k < (unsigned)lim && !gap ? kv_block_at(c, b, k >> psh, p.err) : -1;
      };
      return make_int2(id(tok), id(tok + 16));
    };
    // step i's copies into its ring slot, and the parts' scales beside them (a value scale of -1: nothing here)
    auto issue = [&](int i, int2 id) {
      uint8_t* st = ring + (i % ST) * kStage;
      const int tok = base_of(i);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int y = x ? id.y : id.x;
        if (y >= 0) {
          const int64_t bh = (int64_t)y * c.heads + h;
          const int64_t row = (bh * c.block + ((tok + 16 * x) & (c.block - 1))) * D + 16 * lane;
#pragma unroll
          for (int e = 0; e < D / 32; ++e) {
            const int o = 16 * D * x + 512 * e + 16 * lane;
            cp_async16(st + swz_k<D>(o), c.k + row + 512 * e);
            cp_async16(st + 32 * D + swz_v<D>(o), c.v + row + 512 * e);
          }
          if (lane < 2) cp_async4(st + 64 * D + 8 * x + 4 * lane, (lane ? c.v_scale : c.k_scale) + bh);
        } else if (lane == 0) {
          *reinterpret_cast<float*>(st + 64 * D + 8 * x + 4) = -1.f;
        }
      }
      cp_async_commit();
    };

    // ST - 1 steps' copies in flight, the block ids one step further ahead
#pragma unroll
    for (int e = 0; e < ST - 1; ++e) issue(i0 + e, ids_of(i0 + e));
    int2 id = ids_of(i0 + ST - 1);

    // query rows: as the product's columns, lane (g, t) loads row g and accumulates rows 2t, 2t + 1
    uint2 qf[NT][D / 16];
    float csc[NT][2];
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int rr = row_base + nt * 8 + g;
      const bool live = rr < row_all;
      const float undo = load_q<D>(p, s.row0 + (live ? rr / p.group : 0), h * p.group + (live ? rr % p.group : 0), t, live, qf[nt]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        csc[nt][j] = __shfl_sync(~0u, undo, (2 * t + j) * 4) * p.scale_log2;
        const int r2 = row_base + nt * 8 + 2 * t + j;
        pos[nt][j] = r2 < row_all ? s.first + r2 / p.group : -1;
      }
    }
    float O[NT][D / 16][4], m[NT][2], l[NT][2], vref = pow2f(-126), rv = pow2f(126);  // rv = 1 / vref
    float ad[NT][2], lim[NT][2];  // x = s + ad is what exp2 takes; the reference moves if an x is above lim
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = lim[nt][0] = lim[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
      ad[nt][0] = ad[nt][1] = kShift;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) O[nt][i][j] = 0.f;
    }

    // O is in units of the largest value scale so far, vref.  Where the tile's rows are of several tokens, one may not see
    // the block that has it, and would lose what lies far below it.  So O has a unit for each row, 1 / ru, the largest
    // scale that the row has seen, in the steps APART: from the first one on that not all rows see and whose scale is
    // more than 4 times those before, which all rows have seen, or, without a window, more than 4 times its other 16
    // tokens' (who sees the second 16 sees the first).  False: this is that step.  (Everywhere it would cost a twentieth
    // of the time, in registers.)
    const bool several = first_pos != last_pos;
    auto step = [&](auto apart, float (&ru)[NT][2], const uint8_t* st, int tok) -> bool {
      constexpr bool APART = decltype(apart)::value;
      const float4 sc = *reinterpret_cast<const float4*>(st + 64 * D);
      const float ks[2] = {sc.x, sc.z}, vs[2] = {sc.y, sc.w};
      if (fmaxf(vs[0], vs[1]) < 0.f) return true;
      // rows past the last have zeros for a query and are not written: they need no mask
      const bool plain = tok + 31 <= first_pos && (!p.window || tok > last_pos - p.window || tok + 31 < p.sinks) &&
                         fminf(vs[0], vs[1]) >= 0.f;
      if (!APART && several && !plain) {
        const float low = p.window ? 0.f : fminf(vs[0] < 0.f ? vs[1] : vs[0], vs[1] < 0.f ? vs[0] : vs[1]);
        if (fmaxf(vs[0], vs[1]) > 4.f * fmaxf(vref, low)) return false;
      }
      float S[2][NT][4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint4 kr[2][D / 64];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int cc = 0; cc < D / 64; ++cc)
            kr[i][cc] = *reinterpret_cast<const uint4*>(st + swz_k<D>((16 * x + g + 8 * i) * D + 64 * cc + 16 * t));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) S[x][nt][0] = S[x][nt][1] = S[x][nt][2] = S[x][nt][3] = 0.f;
        qk<D, FMT, NT>(kr, qf, S[x]);
      }
      bool grow = APART;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float& y = S[x][nt][j + 2 * i];
              y = fmaf(y, csc[nt][j] * ks[x], ad[nt][j]);
              if (!plain) {
                const int k = tok + 16 * x + g + 8 * i, q = pos[nt][j];
                if (!(k <= q && (!p.window || k > q - p.window || k < p.sinks)) || vs[x] < 0.f) y = -INFINITY;
              }
            }
          grow |= fmaxf(fmaxf(S[0][nt][j], S[0][nt][j + 2]), fmaxf(S[1][nt][j], S[1][nt][j + 2])) > lim[nt][j];
        }
      const float vmax = fmaxf(vs[0], vs[1]);
      if (__any_sync(~0u, grow || vmax > vref)) {
        float vf = 1.f;
        if (!APART && vmax > vref) {
          rv = 1.f / vmax;
          vf = vref * rv;
          vref = vmax;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float a[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float y = fmaxf(fmaxf(S[0][nt][j], S[0][nt][j + 2]), fmaxf(S[1][nt][j], S[1][nt][j + 2]));
            y = fmaxf(y, __shfl_xor_sync(~0u, y, 4));
            y = fmaxf(y, __shfl_xor_sync(~0u, y, 8));
            y = fmaxf(y, __shfl_xor_sync(~0u, y, 16));
            const float top = fmaxf(m[nt][j], y - ad[nt][j]);
            a[j] = top == m[nt][j] ? 1.f : ex2(m[nt][j] - top);
            if constexpr (APART) {
              float v = fmaxf(fmaxf(S[0][nt][j], S[0][nt][j + 2]) > -INFINITY ? vs[0] : 0.f,
                              fmaxf(S[1][nt][j], S[1][nt][j + 2]) > -INFINITY ? vs[1] : 0.f);
              v = fmaxf(v, __shfl_xor_sync(~0u, v, 4));
              v = fmaxf(v, __shfl_xor_sync(~0u, v, 8));
              v = fmaxf(v, __shfl_xor_sync(~0u, v, 16));
              const float up = v * ru[nt][j];
              vf = up > 1.f ? 1.f / up : 1.f;
              if (up > 1.f) ru[nt][j] = 1.f / v;
            }
            // by what the step's x move: the largest to kShift, whatever the rounding of a large reference
            const float by = y - ad[nt][j] > m[nt][j] ? kShift - y : 0.f;
            m[nt][j] = top;
            ad[nt][j] = kShift - (top == -INFINITY ? 0.f : top);
            const float most = top == -INFINITY ? -INFINITY : kShift + kSlack;
            lim[nt][j] = most;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float& z = S[x][nt][j + 2 * i];
                z += by;
                z = z > most ? most : z;  // (that rounding again; a NaN stays)
              }
            l[nt][j] *= a[j];
            a[j] *= vf;
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            O[nt][i][0] *= a[0];
            O[nt][i][1] *= a[1];
            O[nt][i][2] *= a[0];
            O[nt][i][3] *= a[1];
          }
        }
      }
      const float vf[2] = {APART ? vs[0] : vs[0] * rv, APART ? vs[1] : vs[1] * rv};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[j] = ex2(S[x][nt][j]);
            l[nt][j & 1] += y[j];
            y[j] *= APART ? fminf(vf[x] * ru[nt][j & 1], 1.f) : vf[x];  // (beyond 1: y is 0)
          }
          pb[nt][0] = movmatrix_trans(f2h(y[0], y[1]));
          pb[nt][1] = movmatrix_trans(f2h(y[2], y[3]));
        }
        uint32_t vr[4][VW];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* q = st + 32 * D + swz_v<D>((16 * x + 2 * t + (i & 1) + 8 * (i >> 1)) * D + (D / 8) * g);
          if constexpr (D == 128) {
            const uint4 y = *reinterpret_cast<const uint4*>(q);
            vr[i][0] = y.x;
            vr[i][1] = y.y;
            vr[i][2] = y.z;
            vr[i][3] = y.w;
          } else {
            const uint2 y = *reinterpret_cast<const uint2*>(q);
            vr[i][0] = y.x;
            vr[i][1] = y.y;
          }
        }
        if (!plain) {  // what no row sees may hold anything: not even 0 * NaN of it
          const int lo = p.window ? first_pos - p.window + 1 : 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = tok + 16 * x + 2 * t + (i & 1) + 8 * (i >> 1);
            if (k >= sp.end || (k < lo && k >= p.sinks) || vs[x] < 0.f) {
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[i][w] = 0;
            }
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7362u : 0x5140u;  // two tokens' bytes in pairs
            const uint32_t a = __byte_perm(vr[0][w], vr[1][w], sel), e = __byte_perm(vr[2][w], vr[3][w], sel);
            const uint32_t a0 = KvFmt<FMT>::lo(a), a1 = KvFmt<FMT>::hi(a), a2 = KvFmt<FMT>::lo(e), a3 = KvFmt<FMT>::hi(e);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) MmaOp<__half>::run(O[nt][2 * w + half], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        }
      }
      return true;
    };

    auto arrive = [&](int i) {
      cp_async_wait<ST - 2>();
      __syncwarp();  // everyone's copies of step i are there, and step i - 1's slot is read
      issue(i + ST - 1, id);
      id = ids_of(i + ST);
    };
    int i = i0;
    float ru[NT][2];
#pragma unroll 1
    for (; i < i1; ++i) {
      arrive(i);
      if (!step(std::false_type{}, ru, ring + (i % ST) * kStage, base_of(i))) break;
    }
    if (i < i1) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) ru[nt][j] = lim[nt][j] == -INFINITY ? pow2f(126) : rv;  // (a row that has seen nothing)
#pragma unroll 1
      while (i < i1) {
        step(std::true_type{}, ru, ring + (i % ST) * kStage, base_of(i));
        if (++i < i1) arrive(i);
      }
      vref = 1.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int x = 0; x < D / 16; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) O[nt][x][j] *= 1.f / ru[nt][j & 1];
    }
    cp_async_wait<0>();
    __syncthreads();  // the ring becomes the place where the warps meet

    // join the four warps: rows' maxima, then scaled sums through shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float x = l[nt][j];
        x += __shfl_xor_sync(~0u, x, 4);
        x += __shfl_xor_sync(~0u, x, 8);
        x += __shfl_xor_sync(~0u, x, 16);
        if (g == 0) {
          sm[warp][nt * 8 + 2 * t + j] = m[nt][j];
          sl[warp][nt * 8 + 2 * t + j] = x;
        }
      }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int rr = nt * 8 + 2 * t + j;
        float M = sm[0][rr];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm[w][rr]);
        const float f = (m[nt][j] == M ? 1.f : ex2(m[nt][j] - M)) * vref;
        float* dst = &sO[warp * ROWS + rr][(D / 8) * g];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
          *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(O[nt][i][j] * f, O[nt][i][j + 2] * f);
      }
    __syncthreads();
    float* part = p.part + (2 * (int64_t)blockIdx.x + (u == u_begin ? 0 : 1)) * part_floats<D, NT>();
    for (int e = tid; e < ROWS * D / 4; e += kWarps * 32) {
      const int rr = e / (D / 4), d = (e - rr * (D / 4)) * 4;
      float M = sm[0][rr];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) M = fmaxf(M, sm[w][rr]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&sO[w * ROWS + rr][d]);
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
        L += sl[w][rr] * (sm[w][rr] == M ? 1.f : ex2(sm[w][rr] - M));
      }
      if (CL) {  // over the first warp's sums, which this thread alone has read
        *reinterpret_cast<float4*>(&sO[rr][d]) = o;
        if (d == 0) {
          c_m[rr] = M;
          c_l[rr] = L;
        }
        continue;
      }
      if (!whole) {
        *reinterpret_cast<float4*>(part + rr * D + d) = o;
        if (d == 0) {
          part[ROWS * D + rr] = M;
          part[ROWS * D + ROWS + rr] = L;
        }
        continue;
      }
      const int r2 = row_base + rr;
      if (r2 >= row_all) continue;
      const int64_t at = (int64_t)(s.row0 + r2 / p.group) * p.heads + h * p.group + r2 % p.group;
      const float inv = L == 0.f ? 0.f : 1.f / L;
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + 2 * (at * D + d)) =
          pack4(p.act, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
      if (d == 0) put_stats(p, at, M, L);
    }
    if (CL) {
      cluster_sync();
      const int rr = rank + kCluster * (tid / (D / 4)), d = tid % (D / 4) * 4, r2 = row_base + rr;  // NT rows a CTA
      if (rr < ROWS && r2 < row_all) {
        float M = -INFINITY, L = 0.f, mj[kCluster];
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f), x[kCluster];
#pragma unroll
        for (int j = 0; j < kCluster; ++j) {
          mj[j] = cluster_ld(cluster_addr(&c_m[rr], j));
          x[j] = cluster_ld4(cluster_addr(&sO[rr][d], j));
          M = fmaxf(M, mj[j]);
        }
#pragma unroll
        for (int j = 0; j < kCluster; ++j) {
          const float f = mj[j] == M ? 1.f : ex2(mj[j] - M);
          L += f * cluster_ld(cluster_addr(&c_l[rr], j));
          o.x += x[j].x * f;
          o.y += x[j].y * f;
          o.z += x[j].z * f;
          o.w += x[j].w * f;
        }
        const int64_t at = (int64_t)(s.row0 + r2 / p.group) * p.heads + h * p.group + r2 % p.group;
        const float inv = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + 2 * (at * D + d)) =
            pack4(p.act, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
        if (d == 0) put_stats(p, at, M, L);
      }
      cluster_sync();  // no CTA leaves while its sums are read
      return;
    }
    __syncthreads();
    u += len;
  }
}

// CTA (j, y) joins the row tile that crosses the boundary between pieces j and j + 1, if that is its first
// one: 128 float4s of it (4 rows of 128 dims, 8 of 64).  The pieces' factors first, a warp a row, then
// sums with all pieces' loads independent of one another.
template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32) kv_combine_kernel(AttendParams p, int ctas) {
  constexpr int ROWS = 8 * NT, RC = 512 / D;  // rows of a CTA
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ float s_m[RC], s_l[RC];
  int64_t* off = reinterpret_cast<int64_t*>(dyn);
  const KvView& c = p.c;
  float* s_f = reinterpret_cast<float*>(off + c.batch + 1);  // [pieces][RC]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Plan plan = make_plan<ROWS>(p, off, ctas);
  const int64_t u = (int64_t)(blockIdx.x + 1) * plan.share;
  pdl_wait();
  pdl_launch_dependents();
  if (u >= plan.total) return;
  const int b = seq_of(off, c.batch, u);
  const KvSeq s = kv_seq(c, b);
  const int rt_all = tiles_of(s, p.group, ROWS), per = units_of(s, p, ROWS);
  const int it = (int)((u - off[b]) / per);
  const int64_t begin = off[b] + (int64_t)it * per, last = begin + per - 1;
  if (begin == u || begin / plan.share != blockIdx.x) return;
  const int c0 = blockIdx.x, n = (int)(last / plan.share) - c0 + 1;
  const int h = it / rt_all, rt = it - h * rt_all, row_all = s.rows * p.group;
  // piece j > 0 begins inside the row tile: its first slot.  Piece 0's is its first too if the tile begins it.
  auto slot = [&](int j) {
    const int k = (j == 0 && begin != (int64_t)c0 * plan.share) ? 1 : 0;
    return p.part + (2 * (int64_t)(c0 + j) + k) * part_floats<D, NT>();
  };
  for (int r = warp; r < RC; r += kWarps) {
    const int rr = blockIdx.y * RC + r;
    float M = -INFINITY, L = 0.f;
    for (int j = lane; j < n; j += 32) {
      const float m = __ldcg(slot(j) + ROWS * D + rr);
      s_f[j * RC + r] = m;
      M = fmaxf(M, m);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, o));
    for (int j = lane; j < n; j += 32) {
      const float m = s_f[j * RC + r], f = m == M ? 1.f : ex2(m - M);
      s_f[j * RC + r] = f;
      L += f * __ldcg(slot(j) + ROWS * D + ROWS + rr);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
    if (lane == 0) {
      s_m[r] = M;
      s_l[r] = L;
    }
  }
  __syncthreads();
  const int r = tid / (D / 4), d = (tid - r * (D / 4)) * 4, rr = blockIdx.y * RC + r, r2 = rt * ROWS + rr;
  if (r2 >= row_all) return;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int j = 0; j < n; ++j) {
    const float f = s_f[j * RC + r];
    const float4 x = __ldcg(reinterpret_cast<const float4*>(slot(j) + rr * D + d));
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  const float M = s_m[r], L = s_l[r];
  const int64_t at = (int64_t)(s.row0 + r2 / p.group) * p.heads + h * p.group + r2 % p.group;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + 2 * (at * D + d)) =
      pack4(p.act, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
  if (d == 0) put_stats(p, at, M, L);
}

// Accumulated attention weights: weights[token] += sum over the sequence's rows and the group's
// heads of exp(s - lse), after the attention itself, by the rows' maxima and sums.  A warp owns 2 x 16
// tokens: their keys stay in its registers as fp16, the query rows come by, 32 at a time, through shared
// memory.  It reads the keys again (mostly from L2), dim bytes a token; keeping the scores would be 4 bytes
// written and read for each row.  Latency of short CTAs bounds it for decode: 16 sequences of 6000 tokens
// take 18 us with 4 CTAs an SM, 21 us with 3, 24 us with four tiles a CTA.
constexpr int kRowChunk = 32, kWU = 2;  // rows in shared memory at a time, twice; 64-token units a CTA

template <int D, int FMT>
__global__ void __launch_bounds__(kWarps * 32, 4) kv_weights_kernel(AttendParams p) {
  __shared__ uint2 sq[2][kRowChunk / 8][D / 16][32];
  __shared__ float s_sc[2][kRowChunk];
  __shared__ float2 s_st[2][kRowChunk];
  __shared__ int s_pos[2][kRowChunk], s_huge[2][kWarps], s_fall[kWarps];
  const KvView& c = p.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z;
  const KvSeq s = kv_seq(c, b);
  const int tile = blockIdx.x * (kWU * kWUnit), tile_end = tile + kWU * kWUnit, start = s.first;
  // the sequence's rows that see a token of the tile
  const int t0 = max(tile - start, 0);
  int t1 = s.rows;
  if (p.window && tile >= p.sinks) t1 = (int)min((int64_t)t1, (int64_t)tile_end - 1 + p.window - start);
  if (tile >= s.n || t0 >= t1) {
    pdl_wait();
    return;
  }
  s_fall[warp] = __any_sync(~0u, offsets_fall(c));
  uint32_t kf[kWU][D / 16][4];  // the keys as fragments, fp16
  float ks[kWU], sum[kWU][2];
  int64_t at[kWU];  // the warp's 16 tokens' slot, or -1
#pragma unroll
  for (int x = 0; x < kWU; ++x) {
    const int tok = tile + x * kWUnit + 16 * warp;
    const bool hidden = tok >= s.n || (p.window && tok + 15 <= start - p.window && tok >= p.sinks);
    const int id = hidden ? -1 : kv_block_at(c, b, tok / c.block, p.err);
    const int64_t bh = (int64_t)max(id, 0) * c.heads + h;
    at[x] = id < 0 ? -1 : bh * c.block + (tok & (c.block - 1));
    sum[x][0] = sum[x][1] = ks[x] = 0.f;
    if (id >= 0) {
      const uint8_t* kp = c.k + at[x] * D + 16 * t;
#pragma unroll
      for (int cc = 0; cc < D / 64; ++cc) {
        const uint4 lo = __ldg(reinterpret_cast<const uint4*>(kp + g * D + 64 * cc));
        const uint4 hi = __ldg(reinterpret_cast<const uint4*>(kp + (g + 8) * D + 64 * cc));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          kf[x][cc * 4 + e][0] = KvFmt<FMT>::lo((&lo.x)[e]);
          kf[x][cc * 4 + e][1] = KvFmt<FMT>::lo((&hi.x)[e]);
          kf[x][cc * 4 + e][2] = KvFmt<FMT>::hi((&lo.x)[e]);
          kf[x][cc * 4 + e][3] = KvFmt<FMT>::hi((&hi.x)[e]);
        }
      }
      ks[x] = __ldg(c.k_scale + bh);
    } else {
#pragma unroll
      for (int e = 0; e < D / 16; ++e) kf[x][e][0] = kf[x][e][1] = kf[x][e][2] = kf[x][e][3] = 0;
    }
  }
  // thread 4 r + t stages row r's dims 64 cc + 16 t .. + 16 of a chunk, loaded under the chunk before it
  const int r1 = t1 * p.group, r = tid >> 2;
  uint4 raw[D / 64][2];
  float2 st;
  int pos_r;
  auto load = [&](int r0) {
    const int rr = r0 + r, tr = p.by_group(rr);
    const bool live = rr < r1;
    const int64_t row = s.row0 + (live ? tr : 0);
    const int head = h * p.group + (live ? rr - tr * p.group : 0);
    load_raw<D>(p, row, head, t, live, raw);
    st = live ? p.stats[row * p.heads + head] : make_float2(0.f, 0.f);
    st.x = kShift - st.x;
    pos_r = live ? start + tr : -1;
  };
  auto stage = [&](int buf) {
    uint2 qf[D / 16];
    const float undo = make_q<D>(p, raw, qf);
#pragma unroll
    for (int e = 0; e < D / 16; ++e) sq[buf][r >> 3][e][(r & 7) * 4 + t] = qf[e];
    s_huge[buf][warp] = __any_sync(~0u, fabsf(st.x) > kHuge);
    if (t == 0) {
      s_sc[buf][r] = undo * p.scale_log2;
      s_st[buf][r] = st;
      s_pos[buf][r] = pos_r;
    }
    __syncthreads();
  };
  int buf = 0;
  pdl_wait();  // for the statistics: the keys were there before (16 sequences of 6000 tokens 54 -> 51 us)
  load(t0 * p.group);
  stage(0);
  if (s_fall[0] | s_fall[1] | s_fall[2] | s_fall[3]) return;  // (reported by the attention)
  for (int r0 = t0 * p.group; r0 < r1; r0 += kRowChunk, buf ^= 1) {
    const bool more = r0 + kRowChunk < r1;
    if (more) load(r0 + kRowChunk);
    // all rows of the chunk see all tokens of the tile
    const int first = start + p.by_group(r0), last = start + p.by_group(min(r0 + kRowChunk, r1) - 1);
    const bool plain = tile_end - 1 <= first && (!p.window || tile > last - p.window || tile_end <= p.sinks) &&
                       !(s_huge[buf][0] | s_huge[buf][1] | s_huge[buf][2] | s_huge[buf][3]);
    float part[kWU][2];  // a chunk's sum by itself: thousands of rows added one by one would lose bits
#pragma unroll
    for (int x = 0; x < kWU; ++x) part[x][0] = part[x][1] = 0.f;
#pragma unroll 2
    for (int nt = 0; nt < kRowChunk / 8; ++nt) {
      if (r0 + nt * 8 >= r1) break;
      const float sc[2] = {s_sc[buf][nt * 8 + 2 * t], s_sc[buf][nt * 8 + 2 * t + 1]};
      const float2 st2[2] = {s_st[buf][nt * 8 + 2 * t], s_st[buf][nt * 8 + 2 * t + 1]};
      float S[kWU][4];
#pragma unroll
      for (int x = 0; x < kWU; ++x) S[x][0] = S[x][1] = S[x][2] = S[x][3] = 0.f;
#pragma unroll
      for (int e = 0; e < D / 16; ++e) {
        const uint2 q = sq[buf][nt][e][lane];
#pragma unroll
        for (int x = 0; x < kWU; ++x) MmaOp<__half>::run(S[x], kf[x][e][0], kf[x][e][1], kf[x][e][2], kf[x][e][3], q.x, q.y);
      }
#pragma unroll
      for (int x = 0; x < kWU; ++x) {
        const float f[2] = {sc[0] * ks[x], sc[1] * ks[x]};
        if (plain) {
#pragma unroll
          for (int j = 0; j < 4; ++j) part[x][j >> 1] = fmaf(ex2(fmaf(S[x][j], f[j & 1], st2[j & 1].x)), st2[j & 1].y, part[x][j >> 1]);
        } else {
          const int pos[2] = {s_pos[buf][nt * 8 + 2 * t], s_pos[buf][nt * 8 + 2 * t + 1]};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = tile + x * kWUnit + 16 * warp + g + 8 * (j >> 1), q = pos[j & 1];
            if (k <= q && (!p.window || k > q - p.window || k < p.sinks)) {
              const float w = ex2(fmaf(S[x][j], f[j & 1], st2[j & 1].x)) * st2[j & 1].y;
              part[x][j >> 1] += w > 1.f ? 1.f : w;  // (kHuge: the attention's s may be some steps away; a NaN stays)
            }
          }
        }
      }
    }
#pragma unroll
    for (int x = 0; x < kWU; ++x) {
      sum[x][0] += part[x][0];
      sum[x][1] += part[x][1];
    }
    if (more) stage(buf ^ 1);  // (the chunk before last was read by all before the last barrier)
  }
#pragma unroll
  for (int x = 0; x < kWU; ++x)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float y = sum[x][i];
      y += __shfl_xor_sync(~0u, y, 1);
      y += __shfl_xor_sync(~0u, y, 2);
      const int k = tile + x * kWUnit + 16 * warp + g + 8 * i;
      // one addition to a token's sum, so its order does not matter; sequences that share a block may add to the same one
      if (t == 0 && at[x] >= 0 && k < s.n) atomicAdd(c.weights + at[x] + g + 8 * i, y);
    }
}

// 16 rows a tile need half the passes over the cache of 8, at 2 CTAs an SM instead of 3
static int nt_of(const KvView& c, int group) {
  const int64_t rows = ((int64_t)c.n_rows * group + c.batch - 1) / c.batch;
  return rows > 8 ? 2 : 1;
}

static size_t part_bytes(const KvView& c, int nt) {
  return (size_t)2 * kMaxCtas * (c.dim == 128 ? (nt == 1 ? part_floats<128, 1>() : part_floats<128, 2>())
                                              : (nt == 1 ? part_floats<64, 1>() : part_floats<64, 2>())) * 4;
}

// Clusters up to two thirds of what is resident at once (beyond, clusters of 8 wait for one another's
// places) and up to here in tokens (8 CTAs a row tile are too few then).  With / without, 32 query heads on
// 4, dim 128, us: 1 sequence of 2000 tokens 8.2 / 12.2, of 8192 15.2 / 19.4, of 16,384 24.4 / 22.8;
// 8 sequences of 4096 13.8 / 21.3; 13 (416 CTAs) of 4096 26.1 / 22.6.  Tokens are the table's, which the host
// knows, not the lengths: a short sequence in a wide table goes without.
constexpr double kClusterTokens = 12288;

struct AttendGrid {
  bool cluster;
  int ctas;
};

template <int D, int NT>
static int grid_of(const AttendParams& p, AttendGrid* g) {
  constexpr int ROWS = 8 * NT;
  int sms = 0;
  if (int rc = device_sms(&sms)) return rc;
  // no more CTAs than units there can be
  const int64_t rows = (int64_t)p.c.n_rows * p.group;
  const int64_t tiles = p.group % ROWS == 0 ? rows / ROWS
                        : p.c.cu            ? rows / ROWS + p.c.batch
                                            : (rows / p.c.batch + ROWS - 1) / ROWS * p.c.batch;
  const int64_t units = tiles * p.c.heads * (((int64_t)p.c.width * p.c.block + kUnit - 1) / kUnit);
  double seen = (double)p.c.width * p.c.block;
  if (p.window) seen = std::min(seen, (double)p.sinks + p.window + ROWS);
  g->cluster = tiles * p.c.heads * kCluster <= (int64_t)sms * attend_ctas<D, NT>() * 2 / 3 && seen <= kClusterTokens;
  g->ctas = (int)(g->cluster ? tiles * p.c.heads * kCluster
                             : std::min(std::min((int64_t)sms * attend_ctas<D, NT>(), (int64_t)kMaxCtas), units));
  return DUPLEX_OK;
}

template <int D, int FMT, int NT>
static int run_attend(const AttendParams& p, cudaStream_t st) {
  constexpr int ROWS = 8 * NT;
  const size_t plan = sizeof(int64_t) * (p.c.batch + 1), smem = front_smem<D, NT>() + plan;
  AttendGrid g;
  if (int rc = grid_of<D, NT>(p, &g)) return rc;
  const int ctas = g.ctas;
  constexpr int most = front_smem<D, NT>() + 8 * (DUPLEX_KV_MAX_BATCH + 1);
  if (g.cluster) {
    const auto kern = kv_attend_kernel<D, FMT, NT, true>;
    if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), most)) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return record_cuda(cudaLaunchKernelEx(&cfg, kern, p));
  }
  const auto kern = kv_attend_kernel<D, FMT, NT, false>;
  if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), most)) return rc;
  kern<<<ctas, kWarps * 32, smem, st>>>(p);
  if (int rc = record_cuda(cudaGetLastError())) return rc;
  if (ctas > 1) {
    if (int rc = ensure_smem_attr(reinterpret_cast<const void*>(kv_combine_kernel<D, NT>),
                                  8 * (DUPLEX_KV_MAX_BATCH + 1) + 4 * kMaxCtas * (512 / D))) return rc;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas - 1, ROWS * D / 512);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = plan + sizeof(float) * ctas * (512 / D);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (int rc = record_cuda(cudaLaunchKernelEx(&cfg, kv_combine_kernel<D, NT>, p, ctas))) return rc;
  }
  return DUPLEX_OK;
}

template <int D, int FMT>
static int run_all(const AttendParams& p, void* workspace, cudaStream_t st) {
  const int rc = kv_prompt_takes(p) ? kv_prompt_run(p, workspace, st)
                 : nt_of(p.c, p.group) == 1    ? run_attend<D, FMT, 1>(p, st)
                                               : run_attend<D, FMT, 2>(p, st);
  if (rc || !p.c.weights) return rc;
  const int tokens = kWU * kWUnit;
  const dim3 grid((unsigned)(((int64_t)p.c.width * p.c.block + tokens - 1) / tokens), p.c.heads, p.c.batch);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return record_cuda(cudaLaunchKernelEx(&cfg, kv_weights_kernel<D, FMT>, p));
}

template <int D>
static int launches_of(const AttendParams& p, int32_t* n) {
  *n = p.c.weights ? 1 : 0;
  if (kv_prompt_takes(p)) {
    int ctas = 0;
    if (int rc = kv_prompt_ctas(p, &ctas)) return rc;
    *n += ctas > 1 ? 3 : 2;
    return DUPLEX_OK;
  }
  AttendGrid g;
  if (int rc = nt_of(p.c, p.group) == 1 ? grid_of<D, 1>(p, &g) : grid_of<D, 2>(p, &g)) return rc;
  *n += g.cluster || g.ctas < 2 ? 1 : 2;
  return DUPLEX_OK;
}

// either kernel's (the choice depends on the window too); the rows' statistics lie behind it
static size_t front_bytes(const KvView& c, int group) {
  const size_t few = part_bytes(c, nt_of(c, group));
  return nt_of(c, group) == 1 ? few : std::max(few, kv_prompt_workspace(c, group));
}

int device_sms(int* sms) {
  int dev = 0;
  if (int rc = record_cuda(cudaGetDevice(&dev))) return rc;
  return record_cuda(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
}

}  // namespace duplex

using namespace duplex;

extern "C" int duplex_kv_attend_workspace_bytes(const duplex_kv_cache* cache, const duplex_kv_batch* batch,
                                                int32_t heads, size_t* bytes) {
  KvView v;
  if (int rc = kv_check(cache, batch, &v)) return rc;
  if (!bytes || heads < 1 || heads % cache->kv_heads) return DUPLEX_ERR_ARG;
  *bytes = front_bytes(v, heads / cache->kv_heads) + (size_t)batch->n_rows * heads * (cache->weights ? 12 : 4);
  return DUPLEX_OK;
}

extern "C" int duplex_kv_attend_launches(const duplex_kv_cache* cache, const duplex_kv_batch* batch, int32_t heads,
                                         int32_t window, int32_t sinks, int32_t* launches) {
  AttendParams p{};
  if (int rc = kv_check(cache, batch, &p.c)) return rc;
  if (!launches || heads < 1 || heads % cache->kv_heads || window < 0 || sinks < 0) return DUPLEX_ERR_ARG;
  *launches = 0;
  if (batch->n_rows == 0) return DUPLEX_OK;
  p.heads = heads;
  p.set_group(heads / cache->kv_heads);
  p.set_mask(window, sinks);
  return cache->dim == 128 ? launches_of<128>(p, launches) : launches_of<64>(p, launches);
}

extern "C" int duplex_kv_attend(const duplex_kv_cache* cache, const duplex_kv_batch* batch, const void* q,
                                int act_dtype, int32_t heads, int64_t q_row_stride, int64_t q_head_stride,
                                float softmax_scale, int32_t window, int32_t sinks, void* out, float* lse,
                                void* workspace, size_t workspace_bytes, int32_t* err, void* stream) {
  AttendParams p{};
  if (int rc = kv_check(cache, batch, &p.c)) return rc;
  if (act_dtype != DUPLEX_DTYPE_F16 && act_dtype != DUPLEX_DTYPE_BF16) return DUPLEX_ERR_DTYPE;
  if (heads < 1 || heads % cache->kv_heads || window < 0 || sinks < 0) return DUPLEX_ERR_ARG;
  if (!(softmax_scale - softmax_scale == 0.f)) return DUPLEX_ERR_ARG;
  if (batch->n_rows == 0) return DUPLEX_OK;
  if (!q || !out) return DUPLEX_ERR_ARG;
  if ((((uintptr_t)q | (uintptr_t)out) & 15) || ((q_row_stride | q_head_stride) & 7)) return DUPLEX_ERR_ALIGN;
  size_t need = 0;
  if (int rc = duplex_kv_attend_workspace_bytes(cache, batch, heads, &need)) return rc;
  if (!workspace || workspace_bytes < need) return DUPLEX_ERR_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DUPLEX_ERR_ALIGN;
  p.q = q;
  p.q_row = q_row_stride;
  p.q_head = q_head_stride;
  p.act = act_dtype;
  p.heads = heads;
  p.set_group(heads / cache->kv_heads);
  // a row tile's rows are counted in 32 bits
  if ((int64_t)batch->n_rows * p.group > 0x7FFFFFFFll - 256) return DUPLEX_ERR_UNSUPPORTED;
  p.set_mask(window, sinks);
  p.scale_log2 = softmax_scale * kLog2e;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  uint8_t* rows = static_cast<uint8_t*>(workspace) + front_bytes(p.c, p.group);
  if (cache->weights) {
    p.stats = reinterpret_cast<float2*>(rows);
    rows += (size_t)batch->n_rows * heads * 8;
  }
  p.lse = lse ? lse : reinterpret_cast<float*>(rows);
  p.err = err;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->dim == 128)
    return cache->format == DUPLEX_KV_E4M3 ? run_all<128, DUPLEX_KV_E4M3>(p, workspace, st) : run_all<128, DUPLEX_KV_INT8>(p, workspace, st);
  return cache->format == DUPLEX_KV_E4M3 ? run_all<64, DUPLEX_KV_E4M3>(p, workspace, st) : run_all<64, DUPLEX_KV_INT8>(p, workspace, st);
}
