// Python bindings of the 8-bit kept activations and the norms: tensor validation, output allocation, and the
// autograd nodes.  The nodes are C++ where the other ops' are Python: these operators also run on a few rows, where
// the host's time is the pass.  Of a layer norm's forward and backward of one row, 61 us on the host, the autograd engine takes 37;
// a Python node added about 10.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "launchers.h"

namespace pan {

void gemm(torch::Tensor A, torch::Tensor B, torch::Tensor D, bool a_kmajor, bool b_kmajor,
          c10::optional<torch::Tensor> bias, c10::optional<torch::Tensor> gelu_pre, bool accumulate);  // bindings.cpp

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<torch::Tensor>;

namespace {

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream(); }

// Texts of error messages.  Built from strings alone: streaming a number from this file crashes with this image's pair
// of compiler and C++ runtime.
std::string shape_text(const torch::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string type_text(const torch::Tensor& t) { return c10::toString(t.scalar_type()); }
std::string device_text(const torch::Tensor& t) { return t.device().str(); }

void check_launch(const char* err, const char* what) {
  TORCH_CHECK(err == nullptr, what, ": ", err ? err : "");
  cudaError_t e = cudaGetLastError();
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}

// The kernels' gradients carry no graph: a backward that is itself to be differentiated would drop terms in silence.
void refuse_create_graph(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative: run its backward without create_graph");
}

// A tensor as rows of its last dimension; a copy is made only where the leading dimensions do not
// collapse to two strided levels or the last dimension is not adjacent in memory.
struct RowsOf {
  torch::Tensor t;
  RowsArg a;
  int64_t rows;
  int C;
  bool fp32;
};

RowsOf rows_of(torch::Tensor t, const char* name) {
  TORCH_CHECK_TYPE(t.is_cuda() && (t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32), name,
                   " must be bf16 or fp32 on CUDA, got ", type_text(t));
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1 && t.size(-1) < (1 << 30), name,
                    " needs a last dimension of at least 1, got shape ", shape_text(t));
  if (t.size(-1) > 1 && t.stride(-1) != 1) t = t.contiguous();
  RowsOf r;
  r.C = (int)t.size(-1);
  r.rows = t.numel() / r.C;
  r.fp32 = t.scalar_type() == torch::kFloat32;
  TORCH_CHECK(r.rows < (1ll << 31), name, " has 2^31 rows or more");
  for (int attempt = 0;; ++attempt) {
    int64_t size[2] = {1, 1}, stride[2] = {0, 0};  // inner, outer level
    int levels = 0;
    for (int64_t d = t.dim() - 2; d >= 0 && levels <= 2; --d) {
      if (t.size(d) == 1) continue;
      if (levels > 0 && t.stride(d) == size[levels - 1] * stride[levels - 1]) {
        size[levels - 1] *= t.size(d);
        continue;
      }
      if (levels < 2) {
        size[levels] = t.size(d);
        stride[levels] = t.stride(d);
      }
      ++levels;
    }
    if (levels <= 2 || attempt == 1) {
      if (levels == 0) r.a = RowsArg{t.data_ptr(), r.C, 0, 1};
      else if (levels == 1) r.a = RowsArg{t.data_ptr(), stride[0], 0, 1};
      else r.a = RowsArg{t.data_ptr(), stride[1], stride[0], size[0]};
      break;
    }
    t = t.contiguous();
  }
  if (r.a.inner < 1) r.a.inner = 1;  // no rows
  r.t = t;
  return r;
}

int64_t kept_width(int64_t C) { return (C + 31) / 32 * 32; }
int64_t kept_scales(int64_t C) { return (kept_width(C) / 32 + 3) / 4 * 4; }

Kept8Buf new_kept(const RowsOf& x, torch::Tensor& codes, torch::Tensor& scales) {
  codes = torch::empty({x.rows, kept_width(x.C)}, x.t.options().dtype(torch::kInt8));
  scales = torch::empty({x.rows, kept_scales(x.C)}, x.t.options().dtype(torch::kUInt8));
  return Kept8Buf{codes.data_ptr(), scales.data_ptr(), x.C};
}

Kept8Buf kept_of(const torch::Tensor& codes, const torch::Tensor& scales, int64_t rows, int64_t C) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == torch::kInt8 && codes.is_contiguous() && codes.dim() == 2 &&
                  codes.size(0) == rows && codes.size(1) == kept_width(C),
              "kept codes must be contiguous int8 [rows, C rounded up to 32]");
  TORCH_CHECK(scales.is_cuda() && scales.scalar_type() == torch::kUInt8 && scales.is_contiguous() &&
                  scales.dim() == 2 && scales.size(0) == rows && scales.size(1) == kept_scales(C) &&
                  scales.device() == codes.device(),
              "kept scales must be contiguous uint8 [rows, blocks rounded up to 4] beside the codes");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(scales.data_ptr()) % 16 == 0,
              "kept codes and scales must be 16-byte aligned");
  return Kept8Buf{codes.data_ptr(), scales.data_ptr(), (int)C};
}

void check_same(const RowsOf& a, const RowsOf& b, const char* what) {
  TORCH_CHECK_VALUE(a.t.sizes() == b.t.sizes() && a.fp32 == b.fp32 && a.t.device() == b.t.device(), what,
                    " differ: ", shape_text(a.t), " ", type_text(a.t), " ", device_text(a.t), " and ", shape_text(b.t), " ",
                    type_text(b.t), " ", device_text(b.t));
}

NormArgs norm_args(const RowsOf& x, const OptTensor& w, const OptTensor& b,
                   double eps, bool layer) {
  NormArgs a{};
  a.rows = x.rows;
  a.C = x.C;
  a.fp32 = x.fp32;
  a.layer = layer;
  a.eps = (float)eps;
  a.w_fp32 = x.fp32;
  TORCH_CHECK_VALUE(eps >= 0, "eps=", std::to_string(eps), " is negative");
  const OptTensor* vs[2] = {&w, &b};
  const void** ps[2] = {&a.w, &a.b};
  const char* names[2] = {"weight", "bias"};
  for (int i = 0; i < 2; ++i) {
    if (!vs[i]->has_value()) continue;
    const torch::Tensor& v = vs[i]->value();
    TORCH_CHECK_VALUE(v.dim() == 1 && v.size(0) == x.C, names[i], " ", shape_text(v),
                      " does not fit rows of width ", std::to_string(x.C));
    TORCH_CHECK_VALUE(v.device() == x.t.device(), names[i], " is on ", device_text(v), ", x on ", device_text(x.t));
    TORCH_CHECK_TYPE(v.scalar_type() == torch::kFloat32 || v.scalar_type() == torch::kBFloat16, names[i],
                     " must be bf16 or fp32, got ", type_text(v));
    TORCH_CHECK(v.is_contiguous(), names[i], " must be contiguous");
    a.w_fp32 = v.scalar_type() == torch::kFloat32;
    *ps[i] = v.data_ptr();
  }
  TORCH_CHECK_TYPE(!w.has_value() || !b.has_value() || w->scalar_type() == b->scalar_type(),
                   "weight and bias have different dtypes");
  return a;
}

}  // namespace

std::vector<torch::Tensor> keep8(torch::Tensor x_) {
  const at::cuda::CUDAGuard guard(x_.device());
  const RowsOf x = rows_of(x_, "x");
  torch::Tensor codes, scales;
  const Kept8Buf k = new_kept(x, codes, scales);
  launch_keep8(x.a, x.rows, x.fp32, k, nullptr, 0, stream());
  check_launch(nullptr, "keep8");
  return {codes, scales};
}

// Rows row0 .. row0 + out.size(0) of the kept tensor into `out` [rows, >= C], row-major.
void restore8(torch::Tensor codes, torch::Tensor scales, int64_t C, int64_t row0, torch::Tensor out) {
  const at::cuda::CUDAGuard guard(codes.device());
  const Kept8Buf k = kept_of(codes, scales, codes.size(0), C);
  TORCH_CHECK(out.is_cuda() && out.device() == codes.device() && out.dim() == 2 && out.size(1) >= C &&
                  (out.size(1) == 1 || out.stride(1) == 1) &&
                  (out.scalar_type() == torch::kBFloat16 || out.scalar_type() == torch::kFloat32),
              "restore8: out must be a row-major bf16 or fp32 [rows, >= C] CUDA matrix");
  TORCH_CHECK(row0 >= 0 && row0 + out.size(0) <= codes.size(0) && codes.size(0) < (1ll << 31),
              "restore8: rows out of range");
  launch_restore8(k, row0, out.size(0), out.scalar_type() == torch::kFloat32, out.data_ptr(), out.stride(0), (int)C,
                  stream());
  check_launch(nullptr, "restore8");
}

// The whole kept tensor in a new one of `shape`.
torch::Tensor restore8_new(torch::Tensor codes, torch::Tensor scales, std::vector<int64_t> shape, bool fp32) {
  const at::cuda::CUDAGuard guard(codes.device());
  const int64_t C = shape.back();
  const Kept8Buf k = kept_of(codes, scales, codes.size(0), C);
  auto out = torch::empty(shape, codes.options().dtype(fp32 ? torch::kFloat32 : torch::kBFloat16));
  TORCH_CHECK(out.numel() == codes.size(0) * C && codes.size(0) < (1ll << 31), "restore8: the shape has other rows");
  launch_restore8(k, 0, codes.size(0), fp32, out.data_ptr(), C, (int)C, stream());
  check_launch(nullptr, "restore8");
  return out;
}

// (h, codes and scales of gate, codes and scales of value); without `keep` those are undefined
std::vector<torch::Tensor> swiglu8_fwd(torch::Tensor gate_, torch::Tensor value_, bool keep) {
  const at::cuda::CUDAGuard guard(gate_.device());
  const RowsOf g = rows_of(gate_, "gate"), v = rows_of(value_, "value");
  check_same(g, v, "gate and value");
  auto h = torch::empty(gate_.sizes(), g.t.options());
  torch::Tensor gc, gs, vc, vs;
  Kept8Buf kg{nullptr, nullptr, g.C}, kv = kg;
  if (keep) kg = new_kept(g, gc, gs), kv = new_kept(v, vc, vs);
  launch_swiglu_fwd(g.a, v.a, g.rows, g.fp32, kg, kv, h.data_ptr(), stream());
  check_launch(nullptr, "swiglu8_fwd");
  return {h, gc, gs, vc, vs};
}

// (dgate, dvalue[, h recomputed from the codes])
std::vector<torch::Tensor> swiglu8_bwd(torch::Tensor dh_, torch::Tensor gc, torch::Tensor gs, torch::Tensor vc,
                                       torch::Tensor vs, bool want_h) {
  const at::cuda::CUDAGuard guard(dh_.device());
  const RowsOf d = rows_of(dh_, "dh");
  const Kept8Buf kg = kept_of(gc, gs, d.rows, d.C), kv = kept_of(vc, vs, d.rows, d.C);
  TORCH_CHECK(gc.device() == dh_.device() && vc.device() == dh_.device(), "swiglu8_bwd: devices differ");
  auto dg = torch::empty(dh_.sizes(), d.t.options()), dv = torch::empty(dh_.sizes(), d.t.options());
  std::vector<torch::Tensor> out = {dg, dv};
  if (want_h) out.push_back(torch::empty(dh_.sizes(), d.t.options()));
  launch_swiglu_bwd(d.a, d.rows, d.fp32, kg, kv, dg.data_ptr(), dv.data_ptr(), want_h ? out[2].data_ptr() : nullptr,
                    stream());
  check_launch(nullptr, "swiglu8_bwd");
  return out;
}

// Sum over rows in a fixed order, fp32 accumulation, in the dtype of x or fp32.
torch::Tensor row_sum(torch::Tensor x_, bool fp32_out) {
  const at::cuda::CUDAGuard guard(x_.device());
  const RowsOf x = rows_of(x_, "x");
  const int parts = column_sum_parts(x.rows, x.C);
  torch::Tensor part;
  if (parts > 1) part = torch::empty({parts, x.C}, x.t.options().dtype(torch::kFloat32));
  auto out = torch::empty({x.C}, x.t.options().dtype(fp32_out ? torch::kFloat32 : x.t.scalar_type()));
  launch_column_sum(x.a, x.rows, x.C, x.fp32, parts > 1 ? part.data_ptr<float>() : nullptr, parts, out.data_ptr(),
                    out.scalar_type() == torch::kFloat32, stream());
  check_launch(nullptr, "row_sum");
  return out;
}

// ---------------------------------------------------------------- norms
namespace {

struct NormNode : torch::autograd::Function<NormNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x_, const OptTensor& w, const OptTensor& b,
                               double eps, bool layer, bool kept, bool grad) {
    const at::cuda::CUDAGuard guard(x_.device());
    const RowsOf x = rows_of(x_, "x");
    const NormArgs a = norm_args(x, w, b, eps, layer);
    auto y = torch::empty(x_.sizes(), x.t.options());
    torch::Tensor stats, codes, scales;
    Kept8Buf k{nullptr, nullptr, x.C};
    if (grad) stats = torch::empty({x.rows, 2}, x.t.options().dtype(torch::kFloat32));
    if (grad && kept) k = new_kept(x, codes, scales);
    launch_norm_fwd(a, x.a, y.data_ptr(), grad ? stats.data_ptr<float>() : nullptr, k, stream());
    check_launch(nullptr, "norm forward");
    if (grad) {
      ctx->save_for_backward({codes.defined() ? torch::Tensor() : x_, codes, scales, stats,
                              w.has_value() ? *w : torch::Tensor()});
      ctx->saved_data["flags"] =
          (int64_t)((w.has_value() ? 1 : 0) + (b.has_value() ? 2 : 0) + (layer ? 4 : 0) + (a.w_fp32 ? 8 : 0));
    }
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const torch::Tensor& dy_ = grads[0];
    const variable_list saved = ctx->get_saved_variables();
    const int64_t flags = ctx->saved_data["flags"].toInt();
    const bool layer = flags & 4, w_fp32 = flags & 8;
    refuse_create_graph(layer ? "layer_norm" : "rms_norm");
    const bool need_dx = ctx->needs_input_grad(0), need_dw = (flags & 1) && ctx->needs_input_grad(1),
               need_db = (flags & 2) && ctx->needs_input_grad(flags & 1 ? 2 : 1);  // missing vectors have no edge
    const at::cuda::CUDAGuard guard(dy_.device());
    const RowsOf dy = rows_of(dy_, "dy");
    const torch::Tensor &codes = saved[1], &scales = saved[2], &stats = saved[3], &w = saved[4];
    NormArgs a = norm_args(dy, w.defined() ? OptTensor(w) : c10::nullopt, c10::nullopt, 0.0, layer);
    a.w_fp32 = w_fp32;
    RowsOf x = dy;
    Kept8Buf k{nullptr, nullptr, dy.C};
    if (codes.defined()) {
      k = kept_of(codes, scales, dy.rows, dy.C);
    } else {
      x = rows_of(saved[0], "x");
      check_same(dy, x, "dy and x");
    }
    torch::Tensor dx, dw, db, part;
    const auto wopt = dy.t.options().dtype(w_fp32 ? torch::kFloat32 : torch::kBFloat16);
    if (need_dx) dx = torch::empty(dy_.sizes(), dy.t.options());
    if (need_dw) dw = torch::empty({dy.C}, wopt);
    if (need_db) db = torch::empty({dy.C}, wopt);
    if (need_dw || need_db) {
      const int parts = norm_bwd_parts(a, dy.a, x.a, k);
      part = torch::empty({parts, 2, dy.C}, dy.t.options().dtype(torch::kFloat32));
    }
    launch_norm_bwd(a, dy.a, x.a, k, stats.data_ptr<float>(), need_dx ? dx.data_ptr() : nullptr,
                    part.defined() ? part.data_ptr<float>() : nullptr, need_dw ? dw.data_ptr() : nullptr,
                    need_db ? db.data_ptr() : nullptr, stream());
    check_launch(nullptr, "norm backward");
    return {dx, dw, db, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

bool wants_grad(const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }

// ---------------------------------------------------------------- linear
int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }

// Whether the GEMM's 16-byte copies can address `t` [rows, C] bf16 as it lies.
bool is_operand(const torch::Tensor& t) {
  return t.size(1) % 8 == 0 && t.stride(1) == 1 && t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// A zero-padded copy of bf16 rows.
torch::Tensor padded(const torch::Tensor& t, int64_t rows, int64_t width) {
  const RowsOf r = rows_of(t, "operand");
  auto out = torch::empty({rows, width}, t.options());
  launch_pad_rows(r.a, r.rows, r.C, out.data_ptr(), rows, width, stream());
  check_launch(nullptr, "pad_rows");
  return out;
}

// `t` as a GEMM operand: itself, or a copy with rows of C rounded up to 8 (zeros past C).
torch::Tensor operand(const torch::Tensor& t) { return is_operand(t) ? t : padded(t, t.size(0), up8(t.size(1))); }

// The weight as an operand: also its row count a multiple of 8.
torch::Tensor weight_operand(const torch::Tensor& w_) {
  const torch::Tensor w = w_.scalar_type() == torch::kBFloat16 ? w_ : w_.to(torch::kBFloat16);
  return w.size(0) % 8 == 0 && is_operand(w) ? w : padded(w, up8(w.size(0)), up8(w.size(1)));
}

// dw (+)= g[row0 : row0 + rows]^T x[: rows]; g and x as operands.
void run_wgrad(const torch::Tensor& gp, int64_t N, int64_t row0, const torch::Tensor& x, int64_t K, int64_t rows,
               torch::Tensor& dw, bool add) {
  const WgradPlan plan = wgrad_plan(rows, (int)N, (int)K);
  torch::Tensor part;
  if (plan.part_floats > 0) part = torch::empty({plan.part_floats}, gp.options().dtype(torch::kFloat32));
  check_launch(launch_wgrad(plan, static_cast<const char*>(gp.data_ptr()) + 2 * row0 * gp.stride(0), gp.stride(0),
                            x.data_ptr(), x.stride(0), rows, (int)N, (int)K, dw.data_ptr(), dw.size(1),
                            dw.scalar_type() == torch::kFloat32, add,
                            part.defined() ? part.data_ptr<float>() : nullptr, stream()),
               "weight gradient");
}

// rows of the kept input reloaded at a time for a weight gradient (bounds the bf16 temporary)
constexpr int64_t kWgradRows = 32768;

// dW [N, K] = g [rows, N]^T x, x the kept [rows, K] matrix, in fp32 or bf16.  `gp` is g as an operand.
torch::Tensor weight_grad8(const torch::Tensor& gp, int64_t N, const torch::Tensor& codes, const torch::Tensor& scales,
                           int64_t K, bool fp32) {
  const int64_t rows = codes.size(0);
  const auto dt = fp32 ? torch::kFloat32 : torch::kBFloat16;
  if (rows == 0) return torch::zeros({N, K}, gp.options().dtype(dt));
  const Kept8Buf k = kept_of(codes, scales, rows, K);
  const bool one = rows <= kWgradRows;  // later chunks add to fp32
  auto x = torch::empty({one ? rows : kWgradRows, up8(K)}, gp.options());
  auto dw = torch::empty({N, up8(K)}, gp.options().dtype(one ? dt : torch::kFloat32));
  for (int64_t r0 = 0; r0 < rows; r0 += kWgradRows) {
    const int64_t n = std::min(kWgradRows, rows - r0);
    launch_restore8(k, r0, n, false, x.data_ptr(), x.size(1), (int)x.size(1), stream());
    run_wgrad(gp, N, r0, x, K, n, dw, r0 > 0);
  }
  if (dw.scalar_type() != dt) dw = dw.to(dt);
  return K % 8 == 0 ? dw : dw.narrow(1, 0, K);
}

struct LinearNode : torch::autograd::Function<LinearNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w, const OptTensor& b,
                               bool keep, bool grad) {
    const at::cuda::CUDAGuard guard(x.device());
    const int64_t K = x.size(-1), N = w.size(0), rows = x.numel() / K;
    auto shape = x.sizes().vec();
    shape.back() = N;
    const torch::Tensor x2 = x.reshape({rows, K});
    torch::Tensor codes, scales, xp;
    if (keep) {  // an operand copy, where one is needed, comes out of the same pass
      const RowsOf r = rows_of(x2, "x");
      const Kept8Buf k = new_kept(r, codes, scales);
      const bool copy = !is_operand(x2);
      xp = copy ? torch::empty({rows, up8(K)}, x.options()) : x2;
      launch_keep8(r.a, r.rows, false, k, copy ? xp.data_ptr() : nullptr, up8(K), stream());
      check_launch(nullptr, "keep8");
    } else {
      xp = operand(x2);
    }
    auto y = torch::empty({rows, up8(N)}, x.options());
    if (rows > 0) {
      OptTensor bias;
      if (b.has_value()) {
        const torch::Tensor bf = b->scalar_type() == torch::kBFloat16 ? *b : b->to(torch::kBFloat16);
        bias = N % 8 == 0 ? bf.contiguous() : padded(bf.unsqueeze(0), 1, up8(N)).view({up8(N)});
      }
      gemm(xp, weight_operand(w), y, true, true, bias, c10::nullopt, false);
    }
    if (grad) {
      ctx->save_for_backward({codes, scales, w});
      ctx->saved_data["shape"] = x.sizes().vec();
      ctx->saved_data["b_type"] = b.has_value() ? (int64_t)b->scalar_type() : (int64_t)-1;
    }
    return N % 8 == 0 ? y.view(shape) : y.narrow(1, 0, N).view(shape);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_create_graph("kept8_linear");
    const torch::Tensor& gy = grads[0];
    const at::cuda::CUDAGuard guard(gy.device());
    const variable_list saved = ctx->get_saved_variables();
    const torch::Tensor &codes = saved[0], &scales = saved[1], &w = saved[2];
    const int64_t N = w.size(0), K = w.size(1), rows = gy.numel() / N, b_type = ctx->saved_data["b_type"].toInt();
    const bool need_dx = ctx->needs_input_grad(0), need_dw = ctx->needs_input_grad(1),
               need_db = b_type >= 0 && ctx->needs_input_grad(2);
    torch::Tensor dx, dw, db, gp;
    const torch::Tensor g2 = gy.reshape({rows, N});
    if (need_dx || need_dw) gp = operand(g2);
    if (need_dx) {
      auto out = torch::empty({rows, up8(K)}, gy.options());
      if (rows > 0) gemm(gp, weight_operand(w), out, true, false, c10::nullopt, c10::nullopt, false);
      dx = (K % 8 == 0 ? out : out.narrow(1, 0, K)).view(ctx->saved_data["shape"].toIntVector());
    }
    if (need_dw) dw = weight_grad8(gp, N, codes, scales, K, w.scalar_type() == torch::kFloat32);
    if (need_db) {
      const auto dt = (torch::ScalarType)b_type;
      db = row_sum(g2, dt == torch::kFloat32);
    }
    return {dx, dw, db, torch::Tensor(), torch::Tensor()};
  }
};

struct SwiGLUNode : torch::autograd::Function<SwiGLUNode> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& gate, const torch::Tensor& value, bool grad) {
    auto out = swiglu8_fwd(gate, value, grad);
    if (grad) ctx->save_for_backward({out[1], out[2], out[3], out[4]});
    return out[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_create_graph("kept8_swiglu");
    const variable_list k = ctx->get_saved_variables();
    auto out = swiglu8_bwd(grads[0], k[0], k[1], k[2], k[3], false);
    return {out[0], out[1], torch::Tensor()};
  }
};

}  // namespace

torch::Tensor norm(torch::Tensor x, OptTensor w, OptTensor b, double eps, bool layer, bool kept) {
  if (w.has_value() && !w->is_contiguous()) w = w->contiguous();
  if (b.has_value() && !b->is_contiguous()) b = b->contiguous();
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(w) || wants_grad(b));
  return NormNode::apply(x, w, b, eps, layer, kept, grad);
}

// x, w, b: bf16 or fp32; computed in bf16.
torch::Tensor linear8(torch::Tensor x, torch::Tensor w, OptTensor b) {
  TORCH_CHECK_TYPE(x.is_cuda() && (x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kFloat32),
                   "x must be bf16 or fp32 on CUDA, got ", type_text(x));
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x needs a last dimension of at least 1, got shape ",
                    shape_text(x));
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == x.size(-1) && w.size(0) >= 1, "weight ", shape_text(w),
                    " does not fit an input of width ", std::to_string(x.size(-1)));
  TORCH_CHECK_VALUE(w.device() == x.device(), "weight is on ", device_text(w), ", the input on ", device_text(x));
  TORCH_CHECK_TYPE(w.scalar_type() == torch::kBFloat16 || w.scalar_type() == torch::kFloat32,
                   "weight must be bf16 or fp32, got ", type_text(w));
  if (b.has_value()) {
    TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == w.size(0), "bias ", shape_text(*b), " does not fit a weight ",
                      shape_text(w));
    TORCH_CHECK_VALUE(b->device() == x.device(), "bias is on ", device_text(*b), ", the input on ", device_text(x));
    TORCH_CHECK_TYPE(b->scalar_type() == torch::kBFloat16 || b->scalar_type() == torch::kFloat32,
                     "bias must be bf16 or fp32, got ", type_text(*b));
  }
  if (x.scalar_type() != torch::kBFloat16) x = x.to(torch::kBFloat16);
  const bool on = at::GradMode::is_enabled();
  return LinearNode::apply(x, w, b, on && w.requires_grad(), on && (x.requires_grad() || w.requires_grad() || wants_grad(b)));
}

torch::Tensor swiglu8(torch::Tensor gate, torch::Tensor value) {
  return SwiGLUNode::apply(gate, value, at::GradMode::is_enabled() && (gate.requires_grad() || value.requires_grad()));
}

// A matrix or a weight as an operand of the products, for nodes that run several (Python).
torch::Tensor gemm_operand(torch::Tensor t, bool weight) {
  const at::cuda::CUDAGuard guard(t.device());
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (weight || t.scalar_type() == torch::kBFloat16),
              "gemm_operand: a bf16 CUDA matrix, or a weight");
  return weight ? weight_operand(t) : operand(t);
}

// dW [N, K] of one projection from its kept input, for nodes that hold several (Python).
torch::Tensor linear8_weight_grad(torch::Tensor g2, torch::Tensor codes, torch::Tensor scales, int64_t K, bool fp32) {
  const at::cuda::CUDAGuard guard(g2.device());
  TORCH_CHECK(g2.is_cuda() && g2.dim() == 2 && g2.scalar_type() == torch::kBFloat16 && g2.size(0) == codes.size(0),
              "linear8_weight_grad: g must be bf16 [rows, N] beside the codes");
  return weight_grad8(operand(g2), g2.size(1), codes, scales, K, fp32);
}

// dW [N, K] = g [rows, N]^T x [rows, K] of bf16 matrices, in fp32 or bf16.
torch::Tensor weight_grad(torch::Tensor g, torch::Tensor x, bool fp32) {
  const at::cuda::CUDAGuard guard(g.device());
  TORCH_CHECK(g.is_cuda() && x.is_cuda() && g.device() == x.device() && g.dim() == 2 && x.dim() == 2 &&
                  g.scalar_type() == torch::kBFloat16 && x.scalar_type() == torch::kBFloat16 && g.size(0) == x.size(0) &&
                  g.size(1) >= 1 && x.size(1) >= 1,
              "weight_grad: g [rows, N] and x [rows, K] must be bf16 CUDA matrices of as many rows");
  const int64_t rows = g.size(0), N = g.size(1), K = x.size(1);
  const auto opt = g.options().dtype(fp32 ? torch::kFloat32 : torch::kBFloat16);
  if (rows == 0) return torch::zeros({N, K}, opt);
  auto dw = torch::empty({N, up8(K)}, opt);
  run_wgrad(operand(g), N, 0, operand(x), K, rows, dw, false);
  return K % 8 == 0 ? dw : dw.narrow(1, 0, K);
}

void bind_kept8(pybind11::module_& m) {
  const auto kNoGil = py::call_guard<py::gil_scoped_release>();
  m.def("keep8", &keep8, kNoGil);
  m.def("restore8", &restore8, kNoGil);
  m.def("restore8_new", &restore8_new, kNoGil);
  m.def("weight_grad", &weight_grad, kNoGil);
  m.def("swiglu8_fwd", &swiglu8_fwd, kNoGil);
  m.def("swiglu8_bwd", &swiglu8_bwd, kNoGil);
  m.def("swiglu8", &swiglu8, kNoGil);
  m.def("row_sum", &row_sum, kNoGil);
  m.def("norm", &norm, kNoGil);
  m.def("linear8", &linear8, kNoGil);
  m.def("gemm_operand", &gemm_operand, kNoGil);
  m.def("linear8_weight_grad", &linear8_weight_grad, kNoGil);
}

}  // namespace pan
