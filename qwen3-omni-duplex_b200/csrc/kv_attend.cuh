// What the two attention kernels over the 8-bit paged KV cache share (kv_attend.cu: few query rows a
// sequence; kv_prompt.cu: many).
#pragma once

#include "kv.cuh"

namespace duplex {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// p = exp2(s - m + kShift) is what fp16 holds: the reference m may be 2^kSlack behind the true
// maximum (so it rarely moves), p stays below 2^15, and a p of 2^-21 of the reference is still normal.
// That p (times its block's scale over the largest) is rounded to fp16, half a step 2^-11, because the second
// product's operands have 16 bits; l sums it unrounded, in fp32.  The tokens' errors are independent, so a row's
// is about the result's own rounding for fp16 (2.4e-4 from 64 bits where 32-bit probabilities give 2.1e-4), and
// disappears in bf16's.
constexpr float kShift = 7.f, kSlack = 8.f;
// A reference beyond this has steps that count: s - m is then taken of the rounded s, so that the largest is 0.
constexpr float kHuge = 1048576.f;

struct AttendParams {
  KvView c;
  const void* q;
  int64_t q_row, q_head;  // elements
  int act, heads, group;
  int window, sinks;
  float scale_log2;       // softmax_scale * log2(e)
  void* out;              // [n_rows][heads][dim]
  float* lse;             // [n_rows][heads]
  float2* stats;          // [n_rows][heads] for the weights, or null: see put_stats
  float* part;            // partial results, 2 slots per CTA
  int32_t* err;
  uint32_t group_mul, group_shift;  // r / group = (mulhi(r, mul) + r) >> shift for 0 <= r < 2^31

  DEVI int by_group(int r) const { return (int)((__umulhi((uint32_t)r, group_mul) + (uint32_t)r) >> group_shift); }
  void set_group(int g) {
    group = g;
    group_shift = 0;
    while ((1ull << group_shift) < (uint64_t)g) ++group_shift;
    group_mul = (uint32_t)((((1ull << group_shift) - (uint64_t)g) << 32) / (uint64_t)g + 1);
  }
  void set_mask(int w, int s) {  // a window of all that can be cached is none
    window = w >= c.cap ? 0 : w;
    sinks = s < c.cap ? s : c.cap;
  }
};

// off by at most 2^-22 of it, a thousandth of the rounding to fp16 that follows; numbers below 2^-126 are 0
DEVI float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// the tokens of one row tile: [0, sink_end) and [lo, end), in units of U tokens
struct Span {
  int sink_units, lo, end, sink_end;  // lo aligned to a unit
};

template <int U>
DEVI Span span_of(const AttendParams& p, int first_pos, int last_pos, int n) {
  Span s;
  s.end = max(min(last_pos + 1, n), 0);  // rows before token 0 see nothing
  s.lo = 0;
  s.sink_units = 0;
  s.sink_end = 0;
  if (p.window) {
    const int64_t w = (int64_t)first_pos - p.window + 1;
    s.lo = w > 0 ? (int)(w / U) * U : 0;
    s.sink_end = min(p.sinks, s.end);
    s.sink_units = (s.sink_end + U - 1) / U;
    if (s.sink_units * U >= s.lo) s.lo = s.sink_units = s.sink_end = 0;
  }
  return s;
}

// four values of one row's result, in q's type
DEVI uint2 pack4(int act, float4 o) {
  if (act == DUPLEX_DTYPE_F16) return make_uint2(f2h(o.x, o.y), f2h(o.z, o.w));
  const __nv_bfloat162 x = __floats2bfloat162_rn(o.x, o.y), y = __floats2bfloat162_rn(o.z, o.w);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// A row's sum l of exp2(s - m + kShift).  The weights take (m, 1 / l) rather than the logarithm, whose
// rounding would be as large as the rest of a weight's error (1e-6 of it instead of 3e-7).
DEVI void put_stats(const AttendParams& p, int64_t at, float m, float l) {
  p.lse[at] = l == 0.f ? -INFINITY : (m - kShift + log2f(l)) * kLn2;
  if (p.stats) p.stats[at] = l == 0.f ? make_float2(0.f, 0.f) : make_float2(m, 1.f / l);
}

int kv_check(const duplex_kv_cache* c, const duplex_kv_batch* b, KvView* out);
int device_sms(int* sms);

// kv_prompt.cu
bool kv_prompt_takes(const AttendParams& p);
size_t kv_prompt_workspace(const KvView& c, int group);
int kv_prompt_ctas(const AttendParams& p, int* ctas);
int kv_prompt_run(const AttendParams& p, void* workspace, cudaStream_t st);

}  // namespace duplex
