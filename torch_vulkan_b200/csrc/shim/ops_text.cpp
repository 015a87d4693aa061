// ATen operators of the 4-bit linears and of the relative-position-bias attention (b2::mx4_*, b2::bias_attn_*): the
// wrappers validate, compute strides, allocate outputs and workspaces on the current allocator and launch on the
// current stream, as those of ops.cpp do. The differentiable operators (mx4_linear, mx4_lora_linear,
// bucket_bias_attention) are C++ autograd functions: their smallest calls are bound by the host, and a Python function's
// forward and backward cost more there than the kernels.
#include <ATen/Functions.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <optional>
#include <tuple>
#include <vector>

#include "shim.h"

namespace {

at::Tensor workspace(uint64_t bytes, const at::Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

// =============================== MXFP4 ==============================================================

struct Mx4Dims {
  int64_t rows, cols;
};

// Checks codes [rows, ceil(cols/32)*16] and scales [ceil(rows/128), ceil(cols/128), 32, 4, 4].
Mx4Dims check_mx4(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* what) {
  TORCH_CHECK(codes.is_cuda() && scales.is_cuda() && codes.device() == scales.device(), what,
              ": codes and scales must be CUDA tensors on one device");
  TORCH_CHECK(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what, ": codes and scales must be uint8");
  TORCH_CHECK(codes.dim() == 2 && codes.is_contiguous() && scales.is_contiguous(), what,
              ": codes must be a contiguous matrix and scales contiguous");
  TORCH_CHECK(cols >= 0 && codes.size(1) == b2_mx4_code_bytes(cols), what, ": codes have ", codes.size(1),
              " bytes a row, but ", cols, " columns need ", b2_mx4_code_bytes(cols));
  const int64_t rows = codes.size(0);
  TORCH_CHECK(scales.numel() == b2_mx4_scale_bytes(rows, cols), what, ": scales hold ", scales.numel(), " bytes, but ",
              rows, " x ", cols, " values need ", b2_mx4_scale_bytes(rows, cols));
  TORCH_CHECK(((uintptr_t)codes.data_ptr() | (uintptr_t)scales.data_ptr()) % 16 == 0, what,
              ": codes and scales must be 16-byte aligned");
  return {rows, cols};
}

std::tuple<at::Tensor, at::Tensor> mx4_quantize(const at::Tensor& x0) {
  TORCH_CHECK(x0.is_cuda(), "mx4_quantize: a CUDA tensor is required (this package has no CPU path)");
  TORCH_CHECK(x0.dim() == 2, "mx4_quantize: a matrix is required, got ", x0.sizes());
  TORCH_CHECK(is_row_dtype(x0.scalar_type()), "mx4_quantize: float32, bfloat16 or float16 is required, got ", x0.scalar_type());
  c10::cuda::CUDAGuard guard(x0.device());
  const int64_t rows = x0.size(0), cols = x0.size(1);
  const bool in_place = (x0.stride(1) == 1 || cols <= 1) && (x0.stride(0) >= cols || rows <= 1);
  at::Tensor x = in_place ? x0 : x0.contiguous();
  const auto o = x.options().dtype(at::kByte);
  at::Tensor codes = at::empty({rows, b2_mx4_code_bytes(cols)}, o);
  at::Tensor scales = at::empty({(rows + 127) / 128, (cols + 127) / 128, 32, 4, 4}, o);
  if (x.numel() == 0) return {codes, scales};
  b2_mx4_args a{};
  a.x = x.data_ptr(), a.codes = codes.data_ptr<uint8_t>(), a.scales = scales.data_ptr<uint8_t>();
  a.rows = rows, a.cols = cols, a.ld = rows > 1 ? x.stride(0) : cols, a.dtype = dtype_code(x.scalar_type());
  b2_check(b2_mx4_quantize(&a, cur_stream()), "mx4_quantize");
  count("b2::mx4_quantize");
  return {codes, scales};
}

at::Tensor mx4_dequantize(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, at::ScalarType dtype) {
  const Mx4Dims d = check_mx4(codes, scales, cols, "mx4_dequantize");
  TORCH_CHECK(is_row_dtype(dtype), "mx4_dequantize: dtype must be float32, bfloat16 or float16");
  c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = at::empty({d.rows, d.cols}, codes.options().dtype(dtype));
  if (out.numel() == 0) return out;
  b2_mx4_args a{};
  a.codes = codes.data_ptr<uint8_t>(), a.scales = scales.data_ptr<uint8_t>(), a.out = out.data_ptr();
  a.rows = d.rows, a.cols = d.cols, a.ld = d.cols, a.dtype = dtype_code(dtype);
  b2_check(b2_mx4_dequantize(&a, cur_stream()), "mx4_dequantize");
  count("b2::mx4_dequantize");
  return out;
}

at::Tensor rows_of(const at::Tensor& t) {
  int64_t rows = 1;  // counted: -1 says nothing about a tensor without elements
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  at::Tensor m = t.reshape({rows, t.size(-1)});
  return m.is_contiguous() ? m : m.contiguous();
}

// LoRA side operands: h [rows, r] and the weight-side matrix ([N, r] forward, [r, K] in dX), both bf16.
void lora_operands(b2_mx4_gemm_args& g, const at::Tensor* h, const at::Tensor* w, at::Tensor& hc, at::Tensor& wc,
                   int64_t rows, int64_t width, c10::Device device, const char* what) {
  if (!h) return;
  TORCH_CHECK(h->device() == device && w->device() == device && h->scalar_type() == at::kBFloat16 &&
                  w->scalar_type() == at::kBFloat16, what, ": the LoRA operands must be bf16 tensors on x's device");
  hc = rows_of(*h), wc = w->contiguous();
  const int64_t r = hc.size(1);
  TORCH_CHECK(hc.size(0) == rows && r >= 8 && r <= 64 && r % 8 == 0, what,
              ": the LoRA rank must be 8..64 and a multiple of 8, one row of h per row of x; got h ", h->sizes());
  TORCH_CHECK(wc.dim() == 2 && wc.size(g.transpose_w ? 0 : 1) == r && wc.size(g.transpose_w ? 1 : 0) == width, what,
              ": LoRA matrix of shape ", w->sizes(), " does not fit");
  if (((uintptr_t)hc.data_ptr()) % 16) hc = hc.clone();
  if (((uintptr_t)wc.data_ptr()) % 16 || wc.size(1) % 8) {  // rows padded to whole 16-byte groups
    const int64_t ld = (wc.size(1) + 7) / 8 * 8;
    at::Tensor pad = at::zeros({wc.size(0), ld}, wc.options());
    pad.narrow(1, 0, wc.size(1)).copy_(wc);
    wc = pad;
  }
  g.lora_h = hc.data_ptr(), g.lora_b = wc.data_ptr();
  g.lora_h_ld = r, g.lora_b_ld = wc.size(1), g.lora_r = (int32_t)r;
}

at::Tensor mx4_fwd(const at::Tensor& x0, const at::Tensor& codes, const at::Tensor& scales,
                   const std::optional<at::Tensor>& bias0, const at::Tensor* h, const at::Tensor* b, const char* name) {
  TORCH_CHECK(x0.is_cuda() && x0.scalar_type() == at::kBFloat16, name, ": x must be a bfloat16 CUDA tensor");
  TORCH_CHECK(x0.dim() >= 1 && x0.device() == codes.device(), name, ": x and the weight must be on one device");
  const int64_t K = x0.size(-1);
  const Mx4Dims d = check_mx4(codes, scales, K, name);
  c10::cuda::CUDAGuard guard(x0.device());
  const int64_t N = d.rows;
  std::vector<int64_t> osz(x0.sizes().begin(), x0.sizes().end());
  osz.back() = N;
  at::Tensor bias;
  if (bias0.has_value() && bias0->defined()) {
    bias = bias0->contiguous();
    TORCH_CHECK(bias.device() == x0.device() && bias.scalar_type() == at::kBFloat16 && bias.numel() == N, name,
                ": bias must be a bf16 tensor of ", N, " elements on x's device, got ", bias.scalar_type(), " ", bias.sizes(), " on ",
                bias.device());
  }
  at::Tensor out = at::empty(osz, x0.options());
  if (out.numel() == 0) return out;
  TORCH_CHECK(K > 0, name, ": no input features");
  at::Tensor x = rows_of(x0);
  b2_mx4_gemm_args g{};
  at::Tensor xc, xs;
  if (b2_mx4_takes_x(x.size(0), N, K)) {
    g.x = x.data_ptr(), g.x_ld = K;
  } else {
    std::tie(xc, xs) = mx4_quantize(x);
    g.x_codes = xc.data_ptr<uint8_t>(), g.x_scales = xs.data_ptr<uint8_t>();
  }
  g.w_codes = codes.data_ptr<uint8_t>(), g.w_scales = scales.data_ptr<uint8_t>();
  g.bias = bias.defined() ? bias.data_ptr() : nullptr;
  g.out = out.data_ptr();
  g.M = x.size(0), g.N = N, g.K = K, g.out_ld = N;
  at::Tensor hc, wc;
  lora_operands(g, h, b, hc, wc, g.M, N, x.device(), name);
  at::Tensor ws = workspace(b2_mx4_gemm_workspace_bytes(&g), x);
  g.workspace = ws.defined() ? ws.data_ptr() : nullptr;
  b2_check(b2_mx4_gemm(&g, cur_stream()), name);
  count(name);
  return out;
}

at::Tensor mx4_dx(const at::Tensor& dy0, const at::Tensor& codes, const at::Tensor& scales, int64_t K, const at::Tensor* h,
                  const at::Tensor* a, const char* name) {
  TORCH_CHECK(dy0.is_cuda() && dy0.scalar_type() == at::kBFloat16, name, ": dy must be a bfloat16 CUDA tensor");
  const Mx4Dims d = check_mx4(codes, scales, K, name);
  TORCH_CHECK(dy0.dim() >= 1 && dy0.size(-1) == d.rows && dy0.device() == codes.device(), name, ": dy of shape ", dy0.sizes(),
              " does not fit a weight of ", d.rows, " output features on its device");
  c10::cuda::CUDAGuard guard(dy0.device());
  std::vector<int64_t> osz(dy0.sizes().begin(), dy0.sizes().end());
  osz.back() = K;
  at::Tensor dx = at::empty(osz, dy0.options());
  if (dx.numel() == 0) return dx;
  if (d.rows == 0) return dx.zero_();
  at::Tensor dy = rows_of(dy0);
  b2_mx4_gemm_args g{};
  g.x = dy.data_ptr();
  g.w_codes = codes.data_ptr<uint8_t>(), g.w_scales = scales.data_ptr<uint8_t>();
  g.out = dx.data_ptr();
  g.M = dy.size(0), g.N = d.rows, g.K = K, g.x_ld = d.rows, g.out_ld = K;
  g.transpose_w = 1;
  at::Tensor hc, wc;
  lora_operands(g, h, a, hc, wc, g.M, K, dy.device(), name);
  at::Tensor ws = workspace(b2_mx4_gemm_workspace_bytes(&g), dy);
  g.workspace = ws.defined() ? ws.data_ptr() : nullptr;
  b2_check(b2_mx4_gemm(&g, cur_stream()), name);
  count(name);
  return dx;
}

at::Tensor sum_rows(const at::Tensor& gy) { return rows_of(gy).sum(0); }

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Gradients of a backward that is itself recorded (create_graph): the same values, whose differentiation along `sources`, what they
// depend on, raises an error. Derivatives of these gradients are not implemented, and unrecorded they would count as constants.
struct Refuse : torch::autograd::Function<Refuse> {
  static variable_list forward(AutogradContext* ctx, const std::string& name, const at::TensorList& grads, const at::TensorList&) {
    ctx->saved_data["name"] = name;
    variable_list out;
    for (const at::Tensor& g : grads) out.push_back(g.detach());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list&) {
    TORCH_CHECK(false, ctx->saved_data["name"].toStringRef(), " cannot be differentiated twice");
  }
};
void refuse_second(variable_list& grads, const variable_list& sources, const char* name) {
  if (!at::GradMode::is_enabled()) return;
  variable_list defined;
  for (const Variable& g : grads)
    if (g.defined()) defined.push_back(g);
  if (defined.empty()) return;
  defined = Refuse::apply(std::string(name), at::TensorList(defined), at::TensorList(sources));
  size_t i = 0;
  for (Variable& g : grads)
    if (g.defined()) g = defined[i++];
}

// y = Q(x) W^T + bias; straight-through dx = dy W.
at::Tensor mx4_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                      const std::optional<at::Tensor>& bias) {
  return mx4_fwd(x, codes, scales, bias, nullptr, nullptr, "b2::mx4_linear");
}
struct Mx4Linear : torch::autograd::Function<Mx4Linear> {
  static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& codes, const Variable& scales,
                          const std::optional<Variable>& bias) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["cols"] = x.dim() ? x.size(-1) : 0;
    ctx->saved_data["bias"] = bias.has_value() && bias->defined();
    return mx4_linear(x, codes, scales, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(4);
    if (ctx->needs_input_grad(0)) {
      const variable_list saved = ctx->get_saved_variables();
      {
        at::NoGradGuard plain;
        out[0] = mx4_dx(g[0], saved[0], saved[1], ctx->saved_data["cols"].toInt(), nullptr, nullptr, "b2::mx4_linear_dx");
      }
      refuse_second(out, {g[0]}, "mx4_linear");
    }
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3)) out[3] = sum_rows(g[0]);
    return out;
  }
};
at::Tensor mx4_linear_autograd(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                               const std::optional<at::Tensor>& bias) {
  return Mx4Linear::apply(x, codes, scales, bias);
}

// y = Q(x) W^T + bias + (x a^T) b^T, with the hidden activation h = x a^T [rows, r] as the second result.
std::tuple<at::Tensor, at::Tensor> mx4_lora_fwd(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                                                const std::optional<at::Tensor>& bias, const at::Tensor& a,
                                                const at::Tensor& b) {
  const char* name = "b2::mx4_lora_linear";
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() >= 1, name, ": x must be a bfloat16 CUDA tensor");
  TORCH_CHECK(a.dim() == 2 && b.dim() == 2 && a.device() == x.device() && a.scalar_type() == at::kBFloat16 && a.size(1) == x.size(-1), name,
              ": a must be a bf16 matrix [r, ", x.size(-1), "] on x's device, got ", a.scalar_type(), " ", a.sizes(), " on ", a.device());
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor h = at::mm(rows_of(x), a.t());  // of the unquantised activation
  at::Tensor y = mx4_fwd(x, codes, scales, bias, &h, &b, name);
  return {y, h};
}
at::Tensor mx4_lora_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                           const std::optional<at::Tensor>& bias, const at::Tensor& a, const at::Tensor& b) {
  return std::get<0>(mx4_lora_fwd(x, codes, scales, bias, a, b));
}
// dx = dy W + dh a, for callers that keep h themselves (several LoRA modules on one stacked weight).
at::Tensor mx4_lora_dx(const at::Tensor& dy, const at::Tensor& codes, const at::Tensor& scales, int64_t cols,
                       const at::Tensor& dh, const at::Tensor& a) {
  return mx4_dx(dy, codes, scales, cols, &dh, &a, "b2::mx4_lora_dx");
}
struct Mx4Lora : torch::autograd::Function<Mx4Lora> {
  static Variable forward(AutogradContext* ctx, const Variable& x, const Variable& codes, const Variable& scales,
                          const std::optional<Variable>& bias, const Variable& a, const Variable& b) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [y, h] = mx4_lora_fwd(x, codes, scales, bias, a, b);
    ctx->save_for_backward({x, codes, scales, a, b, h});
    ctx->saved_data["bias"] = bias.has_value() && bias->defined();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const at::Tensor &x = s[0], &codes = s[1], &scales = s[2], &a = s[3], &b = s[4], &h = s[5];
    c10::cuda::CUDAGuard guard(x.device());
    variable_list out(6);
    // edges are counted over the tensors that were given: without a bias, a and b move up by one
    const int e = ctx->saved_data["bias"].toBool() ? 4 : 3;
    {
      at::NoGradGuard plain;
      at::Tensor gy = rows_of(g[0]);
      if (ctx->needs_input_grad(0) || ctx->needs_input_grad(e)) {
        at::Tensor dh = at::mm(gy, b);
        if (ctx->needs_input_grad(0))
          out[0] = mx4_dx(gy, codes, scales, x.size(-1), &dh, &a, "b2::mx4_lora_dx").view_as(x);
        if (ctx->needs_input_grad(e)) out[4] = at::mm(dh.t(), rows_of(x));
      }
      if (ctx->needs_input_grad(e + 1)) out[5] = at::mm(gy.t(), h);
    }
    refuse_second(out, {g[0], x, a, b}, "mx4_lora_linear");
    if (e == 4 && ctx->needs_input_grad(3)) out[3] = sum_rows(g[0]);
    return out;
  }
};
at::Tensor mx4_lora_linear_autograd(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales,
                                    const std::optional<at::Tensor>& bias, const at::Tensor& a, const at::Tensor& b) {
  return Mx4Lora::apply(x, codes, scales, bias, a, b);
}

// =============================== relative-position-bias attention ====================================

at::Tensor bshd(int64_t B, int64_t H, int64_t S, int64_t D, const at::TensorOptions& o) {
  return at::empty({B, S, H, D}, o).permute({0, 2, 1, 3});
}
// The tensor as the kernels read it in place, or a copy: unit stride along D always; 16-bit tensors of a head dim that
// the tensor-core kernels take also want 16-byte aligned rows and no broadcast (zero) strides.
at::Tensor readable(const at::Tensor& t) {
  const bool tc = t.scalar_type() != at::kFloat && t.size(3) % 8 == 0;
  bool ok = t.size(3) == 1 || t.stride(3) == 1;
  if (tc) {
    ok = ok && (uintptr_t)t.data_ptr() % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  }
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
void strides3(int64_t* dst, const at::Tensor& t) { dst[0] = t.stride(0), dst[1] = t.stride(1), dst[2] = t.stride(2); }

struct BiasAttn {
  b2_bias_attn_args a{};
  at::Tensor q, k, v, table, mask;
};

BiasAttn bias_attn_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                        const std::optional<at::Tensor>& key_mask, int64_t max_distance, bool bidirectional, bool causal,
                        double scale, int64_t q_offset, const char* name) {
  TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda() && table.is_cuda(), name, ": CUDA tensors required (this package has no CPU path)");
  TORCH_CHECK(k.device() == q.device() && v.device() == q.device() && table.device() == q.device(), name,
              ": every tensor must be on one device");
  TORCH_CHECK(is_row_dtype(q.scalar_type()) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), name,
              ": q, k and v must share float32, bfloat16 or float16");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, name, ": q, k and v must be [B, heads, S, D]");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == q.size(0) && k.size(3) == q.size(3), name, ": shapes of q ", q.sizes(),
              ", k ", k.sizes(), " and v ", v.sizes(), " do not fit together");
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) % k.size(1) == 0, name, ": ", q.size(1), " query heads are not a multiple of ",
              k.size(1), " key/value heads");
  TORCH_CHECK(q.size(3) >= 1 && q.size(3) <= 128, name, ": head dim must be 1..128, got ", q.size(3));
  TORCH_CHECK(table.dim() == 2 && table.size(1) == q.size(1) && is_row_dtype(table.scalar_type()), name,
              ": table must be a float [num_buckets, ", q.size(1), "] matrix, got ", table.scalar_type(), " ", table.sizes());
  const int64_t nb = table.size(0), side = bidirectional ? nb / 2 : nb;
  TORCH_CHECK(nb <= B2_BIAS_MAX_BUCKETS && side >= 2 && !(bidirectional && nb % 2), name, ": ", nb,
              " buckets; 2 to 128 are supported, an even number from 4 where both directions are told apart");
  TORCH_CHECK(max_distance > side / 2 && max_distance <= B2_BIAS_MAX_DISTANCE, name, ": max_distance must be above ", side / 2,
              " (half a direction's buckets) and at most ", B2_BIAS_MAX_DISTANCE, ", got ", max_distance);
  const int64_t lim = int64_t(1) << 29;
  TORCH_CHECK(q.size(2) < lim && k.size(2) < lim && q_offset < lim && q_offset > -lim, name,
              ": lengths and q_offset must be below 2^29");
  TORCH_CHECK(q.size(0) * q.size(1) <= 65535, name, ": batch * heads must be at most 65535");
  BiasAttn r;
  r.q = readable(q), r.k = readable(k), r.v = readable(v);
  r.table = table.to(at::kFloat).contiguous();
  b2_bias_attn_args& a = r.a;
  if (key_mask.has_value() && key_mask->defined()) {
    const at::Tensor& m = *key_mask;
    TORCH_CHECK(m.is_cuda() && m.device() == q.device() && m.scalar_type() == at::kBool && m.dim() == 2 &&
                    m.size(0) == q.size(0) && m.size(1) == k.size(2), name, ": key_mask must be a bool CUDA tensor [",
                q.size(0), ", ", k.size(2), "] (true = attend), got ", m.scalar_type(), " ", m.sizes());
    r.mask = m.stride(1) == 1 || m.size(1) <= 1 ? m : m.contiguous();
    a.key_mask = (const uint8_t*)r.mask.data_ptr();
    a.mask_sb = r.mask.stride(0);
  }
  a.q = r.q.data_ptr(), a.k = r.k.data_ptr(), a.v = r.v.data_ptr(), a.table = r.table.data_ptr<float>();
  a.B = q.size(0), a.H = q.size(1), a.Hk = k.size(1), a.Sq = q.size(2), a.Sk = k.size(2), a.D = q.size(3);
  strides3(a.q_s, r.q), strides3(a.k_s, r.k), strides3(a.v_s, r.v);
  a.q_offset = q_offset, a.scale = (float)scale;
  a.num_buckets = (int32_t)nb, a.max_distance = (int32_t)max_distance;
  a.bidirectional = bidirectional, a.causal = causal;
  a.dtype = dtype_code(q.scalar_type());
  return r;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> bias_attn_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                             const at::Tensor& table,
                                                             const std::optional<at::Tensor>& key_mask,
                                                             int64_t max_distance, bool bidirectional, bool causal,
                                                             double scale, int64_t q_offset, bool keep_o32) {
  const char* name = "b2::bias_attn_fwd";
  c10::cuda::OptionalCUDAGuard guard(q.is_cuda() ? std::optional<c10::Device>(q.device()) : std::nullopt);
  BiasAttn r = bias_attn_args(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset, name);
  b2_bias_attn_args& a = r.a;
  at::Tensor out = bshd(a.B, a.H, a.Sq, a.D, q.options());
  at::Tensor lse = at::empty({a.B, a.H, a.Sq}, q.options().dtype(at::kFloat));
  // the unrounded output, for a backward that wants the bias gradient (fp32 outputs are that already)
  at::Tensor o32;
  if (keep_o32 && q.scalar_type() != at::kFloat) {
    o32 = at::empty({a.B, a.H, a.Sq, a.D}, q.options().dtype(at::kFloat));
    a.o32 = o32.data_ptr<float>();
  }
  if (out.numel() == 0) return {out, lse, o32};
  a.o = out.data_ptr(), a.lse = lse.data_ptr<float>();
  strides3(a.o_s, out);
  at::Tensor ws = workspace(b2_bias_attn_workspace_bytes(&a, 0), q);
  a.workspace = ws.defined() ? ws.data_ptr() : nullptr;
  b2_check(b2_bias_attn_fwd(&a, cur_stream()), name);
  count(name);
  return {out, lse, o32};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> bias_attn_bwd(
    const at::Tensor& go0, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& o0,
    const at::Tensor& lse0, const at::Tensor& table, const std::optional<at::Tensor>& key_mask, int64_t max_distance,
    bool bidirectional, bool causal, double scale, int64_t q_offset, std::array<bool, 4> want) {
  const char* name = "b2::bias_attn_bwd";
  c10::cuda::OptionalCUDAGuard guard(q.is_cuda() ? std::optional<c10::Device>(q.device()) : std::nullopt);
  BiasAttn r = bias_attn_args(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset, name);
  b2_bias_attn_args& a = r.a;
  const bool wide = o0.scalar_type() == at::kFloat && q.scalar_type() != at::kFloat;  // the forward's unrounded output
  TORCH_CHECK(go0.sizes() == q.sizes() && o0.sizes() == q.sizes() && go0.scalar_type() == q.scalar_type() &&
                  (wide || o0.scalar_type() == q.scalar_type()) && lse0.scalar_type() == at::kFloat &&
                  lse0.numel() == a.B * a.H * a.Sq,
              name, ": grad, output and lse must match q");
  at::Tensor go = readable(go0), o = wide ? o0.contiguous() : readable(o0), lse = lse0.contiguous();
  at::Tensor dq, dk, dv, dt;
  if (want[0]) dq = bshd(a.B, a.H, a.Sq, a.D, q.options()), a.dq = dq.data_ptr(), strides3(a.dq_s, dq);
  if (want[1]) dk = bshd(a.B, a.Hk, a.Sk, a.D, q.options()), a.dk = dk.data_ptr(), strides3(a.dk_s, dk);
  if (want[2]) dv = bshd(a.B, a.Hk, a.Sk, a.D, q.options()), a.dv = dv.data_ptr(), strides3(a.dv_s, dv);
  if (want[3]) {
    dt = at::empty({a.num_buckets, a.H}, q.options().dtype(at::kFloat));
    a.dtable = dt.data_ptr<float>();
  }
  if (wide) a.o32 = o.data_ptr<float>();
  else a.o = o.data_ptr();
  a.lse = lse.data_ptr<float>(), a.d_o = go.data_ptr();
  strides3(a.o_s, o), strides3(a.do_s, go);
  at::Tensor ws = workspace(b2_bias_attn_workspace_bytes(&a, 1), q);
  a.workspace = ws.defined() ? ws.data_ptr() : nullptr;
  b2_check(b2_bias_attn_bwd(&a, cur_stream()), name);
  count(name);
  if (want[3] && table.scalar_type() != at::kFloat) dt = dt.to(table.scalar_type());
  return {dq, dk, dv, dt};
}

at::Tensor bucket_bias_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                 const std::optional<at::Tensor>& key_mask, int64_t max_distance, bool bidirectional,
                                 bool causal, double scale, int64_t q_offset) {
  return std::get<0>(bias_attn_fwd(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset, false));
}
struct BucketBiasAttention : torch::autograd::Function<BucketBiasAttention> {
  static Variable forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& v, const Variable& table,
                          const std::optional<Variable>& key_mask, int64_t max_distance, bool bidirectional, bool causal,
                          double scale, int64_t q_offset) {
    at::AutoDispatchBelowADInplaceOrView guard;
    // a backward keeps the unrounded output: its dS cancels over each row
    auto [o, lse, o32] =
        bias_attn_fwd(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset, true);
    ctx->save_for_backward({q, k, v, o32.defined() ? o32 : o, lse, table, key_mask.has_value() ? *key_mask : at::Tensor()});
    ctx->saved_data["max_distance"] = max_distance;
    ctx->saved_data["bidirectional"] = bidirectional;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["q_offset"] = q_offset;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    auto& d = ctx->saved_data;
    std::array<bool, 4> want;
    for (int i = 0; i < 4; ++i) want[i] = ctx->needs_input_grad(i);
    const std::optional<at::Tensor> mask = s[6].defined() ? std::optional<at::Tensor>(s[6]) : std::nullopt;
    variable_list out(10);
    {
      at::NoGradGuard plain;
      std::tie(out[0], out[1], out[2], out[3]) =
          bias_attn_bwd(g[0], s[0], s[1], s[2], s[3], s[4], s[5], mask, d["max_distance"].toInt(), d["bidirectional"].toBool(),
                        d["causal"].toBool(), d["scale"].toDouble(), d["q_offset"].toInt(), want);
    }
    refuse_second(out, {g[0], s[0], s[1], s[2], s[5]}, "bucket_bias_attention");
    return out;
  }
};
at::Tensor bucket_bias_attention_autograd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                          const at::Tensor& table, const std::optional<at::Tensor>& key_mask,
                                          int64_t max_distance, bool bidirectional, bool causal, double scale,
                                          int64_t q_offset) {
  // Without a backward to come (inputs that want no gradient, or no_grad around a trainable table) the forward that keeps no
  // unrounded output. Decided here: apply() has gradients switched off inside.
  bool grad = false;
  for (const at::Tensor* t : {&q, &k, &v, &table})
    grad = grad || (at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined();
  if (!grad) {
    at::AutoDispatchBelowADInplaceOrView guard;
    return bucket_bias_attention(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset);
  }
  return BucketBiasAttention::apply(q, k, v, table, key_mask, max_distance, bidirectional, causal, scale, q_offset);
}

int64_t bias_bucket(int64_t rel, int64_t num_buckets, int64_t max_distance, bool bidirectional) {
  TORCH_CHECK(num_buckets >= 0 && num_buckets <= B2_BIAS_MAX_BUCKETS && max_distance >= 0 && max_distance <= B2_BIAS_MAX_DISTANCE,
              "bias_bucket: num_buckets must be at most 128 and max_distance at most 1024");
  const int b = b2_bias_bucket(rel, (int32_t)num_buckets, (int32_t)max_distance, bidirectional ? 1 : 0);
  TORCH_CHECK(b >= 0, "bias_bucket: num_buckets ", num_buckets, " and max_distance ", max_distance, " do not fit together");
  return b;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(b2, m) {
  m.def("mx4_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("mx4_dequantize(Tensor codes, Tensor scales, int cols, ScalarType dtype) -> Tensor");
  m.def("mx4_linear(Tensor x, Tensor codes, Tensor scales, Tensor? bias) -> Tensor");
  m.def("mx4_lora_linear(Tensor x, Tensor codes, Tensor scales, Tensor? bias, Tensor a, Tensor b) -> Tensor");
  m.def("mx4_lora_fwd(Tensor x, Tensor codes, Tensor scales, Tensor? bias, Tensor a, Tensor b) -> (Tensor, Tensor)");
  m.def("mx4_lora_dx(Tensor dy, Tensor codes, Tensor scales, int cols, Tensor dh, Tensor a) -> Tensor");
  m.def("bucket_bias_attention(Tensor q, Tensor k, Tensor v, Tensor table, Tensor? key_mask, int max_distance, "
        "bool bidirectional, bool causal, float scale, int q_offset) -> Tensor");
  m.def("bias_bucket(int rel, int num_buckets, int max_distance, bool bidirectional) -> int", &bias_bucket);
}

TORCH_LIBRARY_IMPL(b2, CUDA, m) {
  m.impl("mx4_quantize", &mx4_quantize);
  m.impl("mx4_dequantize", &mx4_dequantize);
  m.impl("mx4_linear", &mx4_linear);
  m.impl("mx4_lora_linear", &mx4_lora_linear);
  m.impl("mx4_lora_fwd", &mx4_lora_fwd);
  m.impl("mx4_lora_dx", &mx4_lora_dx);
  m.impl("bucket_bias_attention", &bucket_bias_attention);
}

TORCH_LIBRARY_IMPL(b2, AutogradCUDA, m) {
  m.impl("mx4_linear", &mx4_linear_autograd);
  m.impl("mx4_lora_linear", &mx4_lora_linear_autograd);
  m.impl("bucket_bias_attention", &bucket_bias_attention_autograd);
}
