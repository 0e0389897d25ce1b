// Shared pieces of the 8-bit paged KV cache (kv_cache.cu, kv_attend.cu): the views of a
// cache and a batch that the kernels take, the two code formats, and the block's scale.
//
// Storage: codes [n_blocks][kv_heads][block][dim], one byte each; one fp32 scale per
// (block, head), for keys and for values; value = code * scale.  A scale that these kernels
// write is a power of two, 2^e with the least e >= -126 for which the block's largest
// |value| <= top * 2^e (top 448 for e4m3, 127 for int8).  So scaling is exact in fp32, a code
// is one rounding of its value, and when a later token raises a block's scale the e4m3 codes
// move without a second rounding unless they become subnormal.
#pragma once

#include "common.cuh"

namespace duplex {

int record_cuda(cudaError_t e);
int ensure_smem_attr(const void* fn, int bytes);

struct KvView {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  float* weights;        // [n_blocks][kv_heads][block] accumulated attention weights, or null
  int n_blocks, heads, block, dim, format;
  const int32_t* table;  // [batch][width] block ids
  const int32_t* kv_len; // [batch]
  const int32_t* cu;     // [batch + 1] row offsets, or null: rows split evenly
  int width, batch, n_rows;
  int cap;               // tokens that a row of the table holds
  int len_max;           // what is made of a kv_len beyond: 2^29 past the table, which is past any window's reach
                         // into it, so that sums of positions stay numbers
};

// rows [row0, row0 + rows) of sequence b, the first row's token, and the number of cached tokens n, held
// inside the buffers whatever the device arrays say.  (Each sequence by itself: see offsets_fall for all
// of them.)  kv_len counts more than the table holds: tokens from n on are not there (see too_long).
struct KvSeq {
  int row0, rows, n, first;
};

DEVI KvSeq kv_seq(const KvView& c, int b) {
  KvSeq s;
  int r1;
  if (c.cu) {
    s.row0 = min(max(c.cu[b], 0), c.n_rows);
    r1 = min(max(c.cu[b + 1], s.row0), c.n_rows);
  } else {
    const int t = c.n_rows / c.batch;
    s.row0 = b * t;
    r1 = s.row0 + t;
  }
  s.rows = r1 - s.row0;
  const int n = min(max(c.kv_len[b], 0), c.len_max);
  s.n = min(n, c.cap);
  s.first = n - s.rows;
  return s;
}

// whether sequence b, of this call, has more tokens than its table
DEVI bool too_long(const KvView& c, const KvSeq& s) { return s.rows > 0 && s.first + s.rows > s.n; }

// Whether this thread's share of the row offsets falls somewhere.  Where none does, no row is in two
// sequences, and what is laid out by rows (the item list, the clusters' grid) has the host's bounds; a
// call whose offsets fall stores and writes nothing but its error bit.
DEVI bool offset_falls(const KvView& c, int b) { return c.cu && c.cu[b + 1] < c.cu[b]; }

DEVI bool offsets_fall(const KvView& c) {
  bool fall = false;
  for (int b = threadIdx.x; c.cu && b < c.batch; b += blockDim.x) fall |= offset_falls(c, b);
  return fall;
}

// the block that holds token j of sequence b, or -1 (and the error bit) if its id is out of range
DEVI int kv_block_at(const KvView& c, int b, int col, int32_t* err) {
  const int id = c.table[(int64_t)b * c.width + col];
  if ((unsigned)id < (unsigned)c.n_blocks) return id;
  set_error(err, DUPLEX_DEVERR_BLOCK);
  return -1;
}

// ----------------------------------------------------------------- formats
DEVI float pow2f(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

template <int FMT> struct KvFmt;

template <> struct KvFmt<DUPLEX_KV_E4M3> {
  // the codes' low / high pair of a word as two fp16 values (exact)
  static DEVI uint32_t half2_of(uint32_t w16) {
    uint32_t d;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(d) : "r"(w16));
    return d;
  }
  static DEVI uint32_t lo(uint32_t w) { return half2_of(w); }
  static DEVI uint32_t hi(uint32_t w) { return half2_of(w >> 16); }
  // one rounding to nearest even, |x| <= 448
  static DEVI uint32_t encode4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  }
  // least e with amax <= 448 * 2^e: 448 = 1.75 * 2^8
  static DEVI int exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, -126);
  }
};

template <> struct KvFmt<DUPLEX_KV_INT8> {
  // a signed byte b as the fp16 pattern 0x6400 | (b + 128) = 1152 + b, less 1152: exact
  static DEVI uint32_t half2_of(uint32_t w, uint32_t sel) {
    const uint32_t p = __byte_perm(w ^ 0x80808080u, 0x64646464u, sel);
    const uint32_t m = 0x64806480u;
    __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&p), *reinterpret_cast<const __half2*>(&m));
    return *reinterpret_cast<uint32_t*>(&r);
  }
  static DEVI uint32_t lo(uint32_t w) { return half2_of(w, 0x4140u); }
  static DEVI uint32_t hi(uint32_t w) { return half2_of(w, 0x4342u); }
  static DEVI uint32_t byte(float x) { return (uint32_t)__float2int_rn(x) & 0xFFu; }
  static DEVI uint32_t encode4(float a, float b, float c, float d) {
    return byte(a) | (byte(b) << 8) | (byte(c) << 16) | (byte(d) << 24);
  }
  // least e with amax <= 127 * 2^e: 127 = 1.984375 * 2^6
  static DEVI int exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
    return max(e, -126);
  }
};

DEVI float2 h2f(uint32_t h) { return __half22float2(*reinterpret_cast<const __half2*>(&h)); }

DEVI uint32_t f2h(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// two 16-bit activations of a word in fp32
template <int ACT> DEVI float2 act2(uint32_t w) {
  if (ACT == DUPLEX_DTYPE_F16) return h2f(w);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

}  // namespace duplex
