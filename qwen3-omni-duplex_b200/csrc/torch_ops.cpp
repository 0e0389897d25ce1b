// PyTorch dispatcher ops over the C ABI of libduplex_b200.so (include/duplex_b200.h):
// TORCH_LIBRARY(duplex_b200, ...) with CUDA implementations that pass data pointers,
// sizes and the current CUDA stream to the extern "C" entry points and raise on a
// non-zero status.  The ops are visible to the dispatcher, the profiler (by name) and
// torch.compile (as opaque custom ops); the reference-named Python modules call the
// same entry points through ctypes.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <cmath>

#include "duplex_b200.h"

namespace {

void check(int rc, const char* what) {
  TORCH_CHECK(rc == DUPLEX_OK, "duplex_b200::", what, " failed: status ", rc, ": ",
              duplex_error_string(rc));
}

void* stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

int act_code(const at::ScalarType t) {
  if (t == at::kHalf) return DUPLEX_DTYPE_F16;
  if (t == at::kBFloat16) return DUPLEX_DTYPE_BF16;
  if (t == at::kFloat) return DUPLEX_DTYPE_F32;
  TORCH_CHECK(false, "duplex_b200: unsupported dtype ", t);
  return -1;
}

void require(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "duplex_b200: ", name, " must be a CUDA tensor (no CPU path)");
  TORCH_CHECK(t.is_contiguous(), "duplex_b200: ", name, " must be contiguous");
}

const void* opt_ptr(const std::optional<at::Tensor>& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

// unpack4 (reference fused_packed_moe.py:54-65)
at::Tensor unpack4(const at::Tensor& packed, int64_t out_cols) {
  require(packed, "packed");
  const c10::cuda::CUDAGuard guard(packed.device());
  const int64_t C = packed.size(-1), rows = packed.numel() / C;
  auto sizes = packed.sizes().vec();
  sizes.back() = out_cols;
  at::Tensor out = at::empty(sizes, packed.options().dtype(at::kInt));
  check(duplex_unpack4(packed.data_ptr<int32_t>(), rows, (int32_t)C, (int32_t)out_cols,
                       out.data_ptr<int32_t>(), stream()),
        "unpack4");
  return out;
}

// FusedPackedMoE._dequant / dequantize_weight (fused_packed_moe.py:183-189)
at::Tensor dequant(const at::Tensor& packed, const at::Tensor& scale,
                   const std::optional<at::Tensor>& zeros, int64_t cols, at::ScalarType out_dtype) {
  require(packed, "packed");
  require(scale, "scale");
  const c10::cuda::CUDAGuard guard(packed.device());
  const int64_t G = scale.size(-1), rows = packed.numel() / packed.size(-1);
  TORCH_CHECK(cols % G == 0, "duplex_b200::dequant: cols not divisible by the scale groups");
  auto sizes = packed.sizes().vec();
  sizes.back() = cols;
  at::Tensor out = at::empty(sizes, packed.options().dtype(out_dtype));
  const int32_t* z = zeros.has_value() ? zeros->data_ptr<int32_t>() : nullptr;
  check(duplex_dequant(packed.data_ptr<int32_t>(), scale.data_ptr(), act_code(scale.scalar_type()),
                       z, rows, (int32_t)cols, (int32_t)(cols / G), out.data_ptr(),
                       act_code(out_dtype), stream()),
        "dequant");
  return out;
}

// dequant_gemv (triton_dequant_gemv.py:85-113) over tile records
at::Tensor dequant_gemv(const at::Tensor& x, const at::Tensor& tiles, int64_t E, int64_t R,
                        int64_t K, int64_t group, bool has_zeros, at::ScalarType scale_dtype,
                        const at::Tensor& sel) {
  require(x, "x");
  require(tiles, "tiles");
  require(sel, "sel");
  TORCH_CHECK(sel.scalar_type() == at::kInt, "duplex_b200::dequant_gemv: sel must be int32");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t k = sel.numel();
  at::Tensor out = at::empty({k, R}, x.options().dtype(at::kFloat));
  const int64_t slot_stride = x.dim() == 1 ? 0 : K;
  check(duplex_dq_gemv(x.data_ptr(), act_code(x.scalar_type()), slot_stride, tiles.data_ptr(),
                       act_code(scale_dtype), has_zeros ? 1 : 0, (int32_t)E, (int32_t)R,
                       (int32_t)K, (int32_t)group, sel.data_ptr<int32_t>(), (int32_t)k,
                       out.data_ptr<float>(), nullptr, stream()),
        "dequant_gemv");
  return out;
}

// TritonPackedLinear.forward (triton_dequant_gemv.py:151-159), B <= 8 rows per launch
at::Tensor packed_linear(const at::Tensor& x, const at::Tensor& tiles, int64_t R, int64_t K,
                         int64_t group, bool has_zeros, at::ScalarType scale_dtype,
                         const std::optional<at::Tensor>& bias,
                         const std::optional<at::Tensor>& residual, double rms_eps) {
  require(x, "x");
  require(tiles, "tiles");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t B = x.numel() / K;
  at::Tensor out = at::empty({B, R}, x.options());
  for (int64_t r0 = 0; r0 < B; r0 += 8) {
    const int64_t b = B - r0 < 8 ? B - r0 : 8;
    const auto* xb = static_cast<const uint8_t*>(x.data_ptr()) + r0 * K * x.element_size();
    auto* ob = static_cast<uint8_t*>(out.data_ptr()) + r0 * R * out.element_size();
    const uint8_t* rb = residual.has_value()
                            ? static_cast<const uint8_t*>(residual->data_ptr()) +
                                  r0 * R * residual->element_size()
                            : nullptr;
    check(duplex_packed_linear(xb, act_code(x.scalar_type()), (int32_t)b, K, tiles.data_ptr(),
                               act_code(scale_dtype), has_zeros ? 1 : 0, (int32_t)R, (int32_t)K,
                               (int32_t)group, opt_ptr(bias), rb, R, ob, R, (float)rms_eps, 0,
                               stream()),
          "packed_linear");
  }
  auto sizes = x.sizes().vec();
  sizes.back() = R;
  return out.view(sizes);
}

// FusedPackedMoE.forward (fused_packed_moe.py:191-275) for T <= 8 tokens
at::Tensor moe_forward(const at::Tensor& x, const at::Tensor& gate_w,
                       const std::optional<at::Tensor>& gate_b, const at::Tensor& gu_tiles,
                       const at::Tensor& dn_tiles, int64_t I, int64_t top_k, bool norm_topk,
                       int64_t group, bool has_zeros, const at::Tensor& workspace,
                       const at::Tensor& err, const std::optional<at::Tensor>& residual,
                       double rms_eps) {
  require(x, "x");
  require(gate_w, "gate_w");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1), E = gate_w.size(0);
  at::Tensor out = at::empty_like(x);
  check(duplex_moe_forward(x.data_ptr(), act_code(x.scalar_type()), (int32_t)T, gate_w.data_ptr(),
                           opt_ptr(gate_b), (int32_t)E, (int32_t)H, (int32_t)I, (int32_t)top_k,
                           norm_topk ? 1 : 0, gu_tiles.data_ptr(), dn_tiles.data_ptr(),
                           act_code(x.scalar_type()), has_zeros ? 1 : 0, (int32_t)group,
                           opt_ptr(residual), out.data_ptr(), nullptr, nullptr, workspace.data_ptr(),
                           (size_t)workspace.numel(), err.data_ptr<int32_t>(), (float)rms_eps, 1,
                           stream()),
        "moe_forward");
  return out;
}

// the batched-decode layer (duplex_moe_grouped) for T <= 512 tokens
at::Tensor moe_grouped(const at::Tensor& x, const at::Tensor& gate_w,
                       const std::optional<at::Tensor>& gate_b, const at::Tensor& gu_tiles,
                       const at::Tensor& dn_tiles, int64_t I, int64_t top_k, bool norm_topk,
                       int64_t group, bool has_zeros, const at::Tensor& workspace,
                       const at::Tensor& err, const std::optional<at::Tensor>& residual) {
  require(x, "x");
  require(gate_w, "gate_w");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1), E = gate_w.size(0);
  at::Tensor out = at::empty_like(x);
  check(duplex_moe_grouped(x.data_ptr(), act_code(x.scalar_type()), (int32_t)T, gate_w.data_ptr(),
                           opt_ptr(gate_b), nullptr, (int32_t)E, (int32_t)H, (int32_t)I,
                           (int32_t)top_k, norm_topk ? 1 : 0, gu_tiles.data_ptr(),
                           dn_tiles.data_ptr(), act_code(x.scalar_type()), has_zeros ? 1 : 0,
                           (int32_t)group, opt_ptr(residual), out.data_ptr(), nullptr, nullptr,
                           workspace.data_ptr(), (size_t)workspace.numel(),
                           err.data_ptr<int32_t>(), stream()),
        "moe_grouped");
  return out;
}

// expert-parallel dispatch pack (into caller buffers) and combine
void ep_dispatch(const at::Tensor& rows, int64_t top_k, int64_t E, int64_t n_ranks,
                 int64_t ids_offset, at::Tensor& send, at::Tensor& slot_of) {
  require(rows, "rows");
  const c10::cuda::CUDAGuard guard(rows.device());
  check(duplex_ep_dispatch_pack(rows.data_ptr(), rows.stride(0), (int32_t)rows.size(0),
                                (int32_t)top_k, (int32_t)E, (int32_t)n_ranks, ids_offset,
                                send.data_ptr(), slot_of.data_ptr<int32_t>(), stream()),
        "ep_dispatch");
}

at::Tensor ep_combine(const at::Tensor& partials, const at::Tensor& slot_of,
                      const std::optional<at::Tensor>& residual, at::ScalarType out_dtype) {
  require(partials, "partials");
  const c10::cuda::CUDAGuard guard(partials.device());
  const int64_t N = partials.size(0), T = partials.size(1), H = partials.size(2);
  at::Tensor out = at::empty({T, H}, partials.options().dtype(out_dtype));
  check(duplex_ep_combine(partials.data_ptr<float>(), slot_of.data_ptr<int32_t>(), (int32_t)T,
                          (int32_t)N, (int32_t)H, opt_ptr(residual), out.data_ptr(),
                          act_code(out_dtype), stream()),
        "ep_combine");
  return out;
}

// the router of FusedPackedMoE.forward (fused_packed_moe.py:195-199), T <= 8 tokens:
// (w [T, top_k] fp32, sel [T, top_k] int32); workspace from duplex_moe_workspace_bytes,
// zero-filled once
std::tuple<at::Tensor, at::Tensor> moe_route(const at::Tensor& x, const at::Tensor& gate_w,
                                             const std::optional<at::Tensor>& gate_b, int64_t top_k,
                                             bool norm_topk, const at::Tensor& workspace) {
  require(x, "x");
  require(gate_w, "gate_w");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1), E = gate_w.size(0);
  at::Tensor w = at::empty({T, top_k}, x.options().dtype(at::kFloat));
  at::Tensor sel = at::empty({T, top_k}, x.options().dtype(at::kInt));
  check(duplex_moe_route(x.data_ptr(), act_code(x.scalar_type()), (int32_t)T, gate_w.data_ptr(),
                         opt_ptr(gate_b), (int32_t)E, (int32_t)H, (int32_t)top_k, norm_topk ? 1 : 0,
                         w.data_ptr<float>(), sel.data_ptr<int32_t>(), workspace.data_ptr(),
                         (size_t)workspace.numel(), 0.f, 0, stream()),
        "moe_route");
  return {w, sel};
}

// the Talker's MoE block (fused_moe.py:40-141), T <= 8 tokens
at::Tensor talker_moe(const at::Tensor& x, const at::Tensor& gate_w, const at::Tensor& gate_up,
                      const at::Tensor& down, const std::optional<at::Tensor>& gu_scale,
                      const std::optional<at::Tensor>& dn_scale, int64_t top_k, bool norm_topk,
                      const std::optional<at::Tensor>& sh_gate, const std::optional<at::Tensor>& sh_up,
                      const std::optional<at::Tensor>& sh_down,
                      const std::optional<at::Tensor>& sh_gate_w, const at::Tensor& workspace,
                      const at::Tensor& err) {
  require(x, "x");
  require(gate_up, "gate_up");
  require(down, "down");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1), E = gate_up.size(0), I = gate_up.size(1) / 2;
  const int64_t S = sh_gate.has_value() ? sh_gate->size(0) : 0;
  at::Tensor out = at::empty_like(x);
  check(duplex_talker_moe_forward(
            x.data_ptr(), act_code(x.scalar_type()), (int32_t)T, gate_w.data_ptr(), (int32_t)E,
            (int32_t)H, (int32_t)I, (int32_t)top_k, norm_topk ? 1 : 0, gate_up.data_ptr(),
            down.data_ptr(), gate_up.scalar_type() == at::kChar ? 1 : 0, opt_ptr(gu_scale),
            opt_ptr(dn_scale), opt_ptr(sh_gate), opt_ptr(sh_up), opt_ptr(sh_down), (int32_t)S,
            opt_ptr(sh_gate_w), out.data_ptr(), nullptr, nullptr, workspace.data_ptr(),
            (size_t)workspace.numel(), err.data_ptr<int32_t>(), stream()),
        "talker_moe");
  return out;
}

// ---- the 8-bit paged KV cache (duplex_kv_*): checks, views and workspaces

struct KvArgs {
  duplex_kv_cache cache{};
  duplex_kv_batch batch{};
};

void on_device(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), "duplex_b200: ", name, " must be on ", like.device(), ", not on ",
              t.device());
}

const int32_t* ints(const at::Tensor& t, const at::Tensor& like, const char* name, at::IntArrayRef shape) {
  require(t, name);
  on_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.sizes() == shape, "duplex_b200: ", name, " must be int32 of shape ",
              shape, ", got ", t.scalar_type(), " ", t.sizes());
  return t.data_ptr<int32_t>();
}

float* floats(const at::Tensor& t, const at::Tensor& like, const char* name, at::IntArrayRef shape) {
  require(t, name);
  on_device(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == shape, "duplex_b200: ", name, " must be float32 of shape ",
              shape, ", got ", t.scalar_type(), " ", t.sizes());
  return t.data_ptr<float>();
}

int32_t* err_ptr(const std::optional<at::Tensor>& err, const at::Tensor& like) {
  if (!err.has_value()) return nullptr;
  return const_cast<int32_t*>(ints(*err, like, "err", {1}));
}

KvArgs kv_args(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale, const at::Tensor& v_scale,
               const at::Tensor& block_table, const at::Tensor& kv_len, const std::optional<at::Tensor>& cu_q,
               const std::optional<at::Tensor>& weights, int64_t n_rows) {
  KvArgs a;
  require(k, "k cache");
  require(v, "v cache");
  on_device(v, k, "v cache");
  TORCH_CHECK(k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
              "duplex_b200: the k and v caches must be [n_blocks, kv_heads, block, dim] of one shape and type");
  TORCH_CHECK(k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kChar,
              "duplex_b200: the caches must be float8_e4m3fn or int8, got ", k.scalar_type());
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "duplex_b200: cache too large");
  TORCH_CHECK(block_table.dim() == 2, "duplex_b200: block_table must be [batch, width]");
  const int64_t B = block_table.size(0), W = block_table.size(1);
  TORCH_CHECK(B <= INT32_MAX && W <= INT32_MAX && n_rows <= INT32_MAX, "duplex_b200: batch too large");
  a.cache.k = k.data_ptr();
  a.cache.v = v.data_ptr();
  a.cache.k_scale = floats(k_scale, k, "k_scale", {k.size(0), k.size(1)});
  a.cache.v_scale = floats(v_scale, k, "v_scale", {k.size(0), k.size(1)});
  if (weights.has_value()) a.cache.weights = floats(*weights, k, "weights", {k.size(0), k.size(1), k.size(2)});
  a.cache.n_blocks = (int32_t)k.size(0);
  a.cache.kv_heads = (int32_t)k.size(1);
  a.cache.block = (int32_t)k.size(2);
  a.cache.dim = (int32_t)k.size(3);
  a.cache.format = k.scalar_type() == at::kChar ? DUPLEX_KV_INT8 : DUPLEX_KV_E4M3;
  a.batch.block_table = ints(block_table, k, "block_table", {B, W});
  a.batch.kv_len = ints(kv_len, k, "kv_len", {B});
  if (cu_q.has_value()) a.batch.cu_rows = ints(*cu_q, k, "cu_q", {B + 1});
  a.batch.width = (int32_t)W;
  a.batch.batch = (int32_t)B;
  a.batch.n_rows = (int32_t)n_rows;
  return a;
}

// rows [n, heads, dim] as the kernels take them: unit stride in dim, the others multiples of 8, 16-byte aligned
at::Tensor rows_of(const at::Tensor& x, const at::Tensor& like, const char* name, int64_t dim) {
  TORCH_CHECK(x.is_cuda(), "duplex_b200: ", name, " must be a CUDA tensor (no CPU path)");
  on_device(x, like, name);
  TORCH_CHECK(x.dim() == 3 && x.size(2) == dim, "duplex_b200: ", name, " must be [rows, heads, ", dim, "], got ",
              x.sizes());
  TORCH_CHECK(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, "duplex_b200: ", name,
              " must be fp16 or bf16, got ", x.scalar_type());
  const bool fits = x.stride(2) == 1 && x.stride(0) % 8 == 0 && x.stride(1) % 8 == 0 && x.stride(0) >= 0 &&
                    x.stride(1) >= 0 && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0;
  return fits ? x : x.clone(at::MemoryFormat::Contiguous);
}

void kv_append(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& k, const at::Tensor& v,
               const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
               const at::Tensor& kv_len, const std::optional<at::Tensor>& cu_q,
               const std::optional<at::Tensor>& weights, const std::optional<at::Tensor>& err) {
  KvArgs a = kv_args(k, v, k_scale, v_scale, block_table, kv_len, cu_q, weights, k_new.dim() ? k_new.size(0) : 0);
  const c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor kn = rows_of(k_new, k, "k_new", k.size(3)), vn = rows_of(v_new, k, "v_new", k.size(3));
  TORCH_CHECK(kn.size(1) == k.size(1) && vn.sizes() == kn.sizes() && vn.scalar_type() == kn.scalar_type(),
              "duplex_b200: k_new and v_new must be [rows, ", k.size(1), ", ", k.size(3), "] of one type");
  check(duplex_kv_append(&a.cache, &a.batch, kn.data_ptr(), vn.data_ptr(), act_code(kn.scalar_type()), kn.stride(0),
                         kn.stride(1), vn.stride(0), vn.stride(1), err_ptr(err, k), stream()),
        "kv_append");
}

void kv_attend_into(const at::Tensor& q_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale,
                    const at::Tensor& v_scale, const at::Tensor& block_table, const at::Tensor& kv_len,
                    const std::optional<at::Tensor>& cu_q, std::optional<double> softmax_scale, int64_t window,
                    int64_t sinks, const std::optional<at::Tensor>& weights, const at::Tensor& out,
                    const std::optional<at::Tensor>& lse, const std::optional<at::Tensor>& err) {
  KvArgs a = kv_args(k, v, k_scale, v_scale, block_table, kv_len, cu_q, weights, q_in.dim() ? q_in.size(0) : 0);
  const c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor q = rows_of(q_in, k, "q", k.size(3));
  const int64_t heads = q.size(1);
  TORCH_CHECK(window >= 0 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX,
              "duplex_b200: window and sinks must be in [0, 2^31)");
  require(out, "out");
  on_device(out, k, "out");
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(),
              "duplex_b200: out must have q's shape and type");
  if (q.numel()) {
    const char* o = static_cast<const char*>(out.data_ptr());
    const char* i = static_cast<const char*>(q.data_ptr());
    const int64_t extent = ((q.size(0) - 1) * q.stride(0) + (heads - 1) * q.stride(1) + q.size(2)) * 2;
    TORCH_CHECK(o + out.numel() * 2 <= i || i + extent <= o, "duplex_b200: out must not overlap q");
  }
  float* lse_p = lse.has_value() ? floats(*lse, k, "lse", {q.size(0), heads}) : nullptr;
  size_t n = 0;
  check(duplex_kv_attend_workspace_bytes(&a.cache, &a.batch, (int32_t)heads, &n), "kv_attend");
  const at::Tensor ws = at::empty({(int64_t)n}, k.options().dtype(at::kByte));
  const double scale = softmax_scale.has_value() ? *softmax_scale : 1.0 / std::sqrt((double)k.size(3));
  check(duplex_kv_attend(&a.cache, &a.batch, q.data_ptr(), act_code(q.scalar_type()), (int32_t)heads, q.stride(0),
                         q.stride(1), (float)scale, (int32_t)window, (int32_t)sinks, out.data_ptr(), lse_p,
                         ws.data_ptr(), n, err_ptr(err, k), stream()),
        "kv_attend");
}

std::tuple<at::Tensor, at::Tensor> kv_attend(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                             const at::Tensor& k_scale, const at::Tensor& v_scale,
                                             const at::Tensor& block_table, const at::Tensor& kv_len,
                                             const std::optional<at::Tensor>& cu_q,
                                             std::optional<double> softmax_scale, int64_t window, int64_t sinks,
                                             const std::optional<at::Tensor>& weights,
                                             const std::optional<at::Tensor>& err) {
  TORCH_CHECK(q.dim() == 3, "duplex_b200: q must be [rows, heads, dim], got ", q.sizes());
  const c10::cuda::CUDAGuard guard(k.device());
  at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  at::Tensor lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  kv_attend_into(q, k, v, k_scale, v_scale, block_table, kv_len, cu_q, softmax_scale, window, sinks, weights, out, lse,
                 err);
  return {out, lse};
}

at::Tensor kv_evict(const at::Tensor& k, const at::Tensor& v, const at::Tensor& k_scale, const at::Tensor& v_scale,
                    const at::Tensor& block_table, const at::Tensor& kv_len, const at::Tensor& weights,
                    const at::Tensor& dst_table, int64_t keep, int64_t sinks, int64_t recent,
                    const std::optional<at::Tensor>& err) {
  KvArgs a = kv_args(k, v, k_scale, v_scale, block_table, kv_len, std::nullopt, weights, 0);
  const c10::cuda::CUDAGuard guard(k.device());
  TORCH_CHECK(dst_table.dim() == 2 && dst_table.size(1) <= INT32_MAX, "duplex_b200: dst_table must be [batch, width]");
  const int32_t* dst = ints(dst_table, k, "dst_table", {block_table.size(0), dst_table.size(1)});
  TORCH_CHECK(keep >= 1 && keep <= INT32_MAX && sinks >= 0 && recent >= 0 && sinks + recent <= keep,
              "duplex_b200: keep must be at least 1 and sinks + recent, got ", keep, ", ", sinks, ", ", recent);
  TORCH_CHECK(dst_table.size(1) * k.size(2) >= keep, "duplex_b200: dst_table holds fewer than keep tokens");
  size_t n = 0;
  check(duplex_kv_evict_workspace_bytes(&a.cache, &a.batch, (int32_t)keep, &n), "kv_evict");
  const at::Tensor ws = at::empty({(int64_t)n}, k.options().dtype(at::kByte));
  at::Tensor new_len = at::empty_like(kv_len);
  check(duplex_kv_evict(&a.cache, &a.batch, dst, (int32_t)dst_table.size(1), (int32_t)keep, (int32_t)sinks,
                        (int32_t)recent, new_len.data_ptr<int32_t>(), ws.data_ptr(), n, err_ptr(err, k), stream()),
        "kv_evict");
  return new_len;
}

}  // namespace

TORCH_LIBRARY(duplex_b200, m) {
  m.def("unpack4(Tensor packed, int out_cols) -> Tensor");
  m.def("dequant(Tensor packed, Tensor scale, Tensor? zeros, int cols, ScalarType out_dtype) -> Tensor");
  m.def("dequant_gemv(Tensor x, Tensor tiles, int E, int R, int K, int group, bool has_zeros, "
        "ScalarType scale_dtype, Tensor sel) -> Tensor");
  m.def("packed_linear(Tensor x, Tensor tiles, int R, int K, int group, bool has_zeros, "
        "ScalarType scale_dtype, Tensor? bias, Tensor? residual, float rms_eps) -> Tensor");
  m.def("moe_forward(Tensor x, Tensor gate_w, Tensor? gate_b, Tensor gu_tiles, Tensor dn_tiles, "
        "int I, int top_k, bool norm_topk, int group, bool has_zeros, Tensor workspace, "
        "Tensor err, Tensor? residual, float rms_eps) -> Tensor");
  m.def("moe_grouped(Tensor x, Tensor gate_w, Tensor? gate_b, Tensor gu_tiles, Tensor dn_tiles, "
        "int I, int top_k, bool norm_topk, int group, bool has_zeros, Tensor workspace, "
        "Tensor err, Tensor? residual) -> Tensor");
  m.def("ep_dispatch(Tensor rows, int top_k, int E, int n_ranks, int ids_offset, "
        "Tensor(a!) send, Tensor(b!) slot_of) -> ()");
  m.def("ep_combine(Tensor partials, Tensor slot_of, Tensor? residual, ScalarType out_dtype) "
        "-> Tensor");
  m.def("moe_route(Tensor x, Tensor gate_w, Tensor? gate_b, int top_k, bool norm_topk, "
        "Tensor workspace) -> (Tensor, Tensor)");
  m.def("talker_moe(Tensor x, Tensor gate_w, Tensor gate_up, Tensor down, Tensor? gu_scale, "
        "Tensor? dn_scale, int top_k, bool norm_topk, Tensor? sh_gate, Tensor? sh_up, "
        "Tensor? sh_down, Tensor? sh_gate_w, Tensor workspace, Tensor err) -> Tensor");
  m.def("kv_append(Tensor k_new, Tensor v_new, Tensor(a!) k, Tensor(b!) v, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor block_table, Tensor kv_len, Tensor? cu_q, Tensor(e!)? weights, "
        "Tensor(f!)? err) -> ()");
  m.def("kv_attend(Tensor q, Tensor k, Tensor v, Tensor k_scale, Tensor v_scale, Tensor block_table, "
        "Tensor kv_len, Tensor? cu_q, float? softmax_scale, int window, int sinks, Tensor(a!)? weights, "
        "Tensor(b!)? err) -> (Tensor, Tensor)");
  m.def("kv_attend_into(Tensor q, Tensor k, Tensor v, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor kv_len, Tensor? cu_q, float? softmax_scale, int window, int sinks, "
        "Tensor(a!)? weights, Tensor(b!) out, Tensor(c!)? lse, Tensor(d!)? err) -> ()");
  m.def("kv_evict(Tensor(a!) k, Tensor(b!) v, Tensor(c!) k_scale, Tensor(d!) v_scale, "
        "Tensor block_table, Tensor kv_len, Tensor(e!) weights, Tensor dst_table, int keep, int sinks, "
        "int recent, Tensor(f!)? err) -> Tensor");
}

TORCH_LIBRARY_IMPL(duplex_b200, CUDA, m) {
  m.impl("unpack4", &unpack4);
  m.impl("dequant", &dequant);
  m.impl("dequant_gemv", &dequant_gemv);
  m.impl("packed_linear", &packed_linear);
  m.impl("moe_forward", &moe_forward);
  m.impl("moe_grouped", &moe_grouped);
  m.impl("ep_dispatch", &ep_dispatch);
  m.impl("ep_combine", &ep_combine);
  m.impl("moe_route", &moe_route);
  m.impl("talker_moe", &talker_moe);
  m.impl("kv_append", &kv_append);
  m.impl("kv_attend", &kv_attend);
  m.impl("kv_attend_into", &kv_attend_into);
  m.impl("kv_evict", &kv_evict);
}
