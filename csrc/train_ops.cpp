// PyTorch bindings of the training operators: dense layers, layer norm, the
// AdamW step with the gradient norm, and packed 8-bit optimizer states.

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <vector>

#include "hip/train_ops.h"

namespace {

using torch::Tensor;
using Tensors = std::vector<Tensor>;

hipStream_t current() { return c10::hip::getCurrentHIPStream().stream(); }

void launched(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

int elem_type(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat: return 0;
    case torch::kBFloat16: return 1;
    case torch::kHalf: return 2;
    default:
      TORCH_CHECK(false, what, ": float32, bfloat16 or float16, not ",
                  t.scalar_type());
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// ------------------------------------------------------------ layer norm

// x as rows of consecutive values; a copy only where its strides need one or
// it is a negative view.
Tensor as_rows(const Tensor& given, int64_t width) {
  const Tensor x = given.resolve_neg();
  if (x.dim() == 2 && (x.stride(1) == 1 || width == 1) &&
      (x.stride(0) >= width || x.stride(0) == 0))
    return x;
  return x.contiguous().view({-1, width});
}

void check_norm(const Tensor& x, const std::optional<Tensor>& w,
                const char* name) {
  if (!w) return;
  TORCH_CHECK(w->device() == x.device(), "layer_norm: ", name,
              " is on another device than x");
  TORCH_CHECK(w->dim() == 1 && w->size(0) == x.size(-1), "layer_norm: ", name,
              " must be [", x.size(-1), "]");
  TORCH_CHECK(w->scalar_type() == x.scalar_type() ||
                  w->scalar_type() == torch::kFloat,
              "layer_norm: ", name, " must have x's type or float32");
}

void check_norm(const Tensor& x, const std::optional<Tensor>& w,
                const std::optional<Tensor>& b) {
  TORCH_CHECK(x.is_cuda(), "layer_norm: x must be on GPU");
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (1 << 24),
              "layer_norm: the last dimension must have 1 to 2^24 values");
  check_norm(x, w, "weight");
  check_norm(x, b, "bias");
  TORCH_CHECK(!w || !b || w->scalar_type() == b->scalar_type(),
              "layer_norm: weight and bias must have one type");
}

std::vector<Tensor> layer_norm_fwd(const Tensor& x, std::optional<Tensor> w,
                                   std::optional<Tensor> b, double eps,
                                   bool stats) {
  check_norm(x, w, b);
  const int type = elem_type(x, "layer_norm");
  const c10::DeviceGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor y = torch::empty(x.sizes(), x.options().memory_format(
                                         at::MemoryFormat::Contiguous));
  Tensor st;
  if (stats) st = torch::empty({2, rows}, x.options().dtype(torch::kFloat));
  if (rows > 0) {
    const Tensor xr = as_rows(x, width);
    if (w) w = w->resolve_neg().contiguous();
    if (b) b = b->resolve_neg().contiguous();
    NormArgs a{};
    a.x = xr.data_ptr();
    a.w = w ? w->data_ptr() : nullptr;
    a.b = b ? b->data_ptr() : nullptr;
    a.y = y.data_ptr();
    if (stats) {
      a.mean = st.data_ptr<float>();
      a.rstd = a.mean + rows;
    }
    a.rows = rows;
    a.width = (int)width;
    a.x_stride = rows > 1 ? xr.stride(0) : width;
    a.eps = (float)eps;
    launched(layer_norm_fwd_launch(
                 &a, type, w ? elem_type(*w, "layer_norm")
                             : b ? elem_type(*b, "layer_norm") : type,
                 current()),
             "layer_norm");
  }
  return {y, st};
}

// Returns dx, dw, db; undefined where not wanted.
std::vector<Tensor> layer_norm_bwd(const Tensor& dy, const Tensor& x,
                                   std::optional<Tensor> w,
                                   torch::ScalarType wtype, const Tensor& st,
                                   bool want_dx, bool want_dw, bool want_db) {
  TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() &&
                  dy.device() == x.device(),
              "layer_norm: the output's gradient does not match x");
  const int type = elem_type(x, "layer_norm");
  const c10::DeviceGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const auto wopts = x.options().dtype(wtype);
  Tensor dx, dw, db;
  if (want_dx)
    dx = torch::empty(x.sizes(), x.options().memory_format(
                                     at::MemoryFormat::Contiguous));
  if (want_dw)
    dw = rows ? torch::empty({width}, wopts) : torch::zeros({width}, wopts);
  if (want_db)
    db = rows ? torch::empty({width}, wopts) : torch::zeros({width}, wopts);
  if (rows > 0) {
    const Tensor xr = as_rows(x, width), dyr = as_rows(dy, width);
    if (w) w = w->resolve_neg().contiguous();
    NormArgs a{};
    a.dy = dyr.data_ptr();
    a.x = xr.data_ptr();
    a.w = w ? w->data_ptr() : nullptr;
    a.dx = want_dx ? dx.data_ptr() : nullptr;
    a.mean = st.data_ptr<float>();
    a.rstd = a.mean + rows;
    a.rows = rows;
    a.width = (int)width;
    a.x_stride = rows > 1 ? xr.stride(0) : width;
    a.dy_stride = rows > 1 ? dyr.stride(0) : width;
    a.parts = layer_norm_parts(rows, (int)width, type);
    Tensor part;
    if (want_dw || want_db) {
      part = torch::empty({a.parts, 2 * norm_part_half((int)width)},
                          x.options().dtype(torch::kFloat));
      a.part = part.data_ptr<float>();
    }
    const int wt = wtype == torch::kFloat ? 0 : type;
    launched(layer_norm_bwd_launch(&a, type, wt, current()),
             "layer_norm backward");
    if (a.part != nullptr)
      launched(sum_rows_launch(a.part, a.parts,
                               2 * norm_part_half((int)width),
                               norm_part_half((int)width), (int)width,
                               want_dw ? dw.data_ptr() : nullptr,
                               want_db ? db.data_ptr() : nullptr, wt,
                               current()),
               "layer_norm backward");
  }
  return {dx, dw, db};
}

// ---------------------------------------------------------- dense layers

// A matrix as the product kernel takes it: rows that begin at multiples of
// 16 bytes, of a whole number of 16 bytes. `t` is rows of consecutive
// values; what does not fit is copied with zeros behind each row.
struct Operand {
  Tensor held;
  int rows, width;      // width: in memory, a whole number of 16 bytes
  long ld;
  Operand(const Tensor& t, int type, hipStream_t stream) : held(t) {
    const int64_t per = 16 / t.element_size();
    rows = (int)t.size(0);
    width = (int)((t.size(1) + per - 1) / per * per);
    ld = rows > 1 ? t.stride(0) : width;
    if (t.size(1) == width && ld % per == 0 && aligned16(t.data_ptr()))
      return;
    held = torch::empty({rows, width}, t.options());
    ld = width;
    if (rows > 0 && width > 0)
      launched(linear_pad_launch(t.data_ptr(), held.data_ptr(), rows,
                                 (int)t.size(1), t.stride(0), width, type,
                                 stream),
               "linear_act");
  }
};

// Rows with a stride of their own, never overlapping.
Tensor as_matrix(const Tensor& given, int64_t rows, int64_t width) {
  const Tensor t = given.resolve_neg();
  if (t.dim() == 2 && (t.stride(1) == 1 || width <= 1) &&
      (t.stride(0) >= width || t.size(0) <= 1))
    return t;
  return t.contiguous().view({rows, width});
}

constexpr int64_t kMostRows = 1LL << 30;

// A tile's 256 rows of this many bytes are within a descriptor's range.
bool near(int64_t row) { return row * 256 + 128 < (1LL << 31); }

// `a` with x, y, the extents and the epilogue set.
void product(LinearProduct& a, int type, const Tensor& like,
             hipStream_t stream) {
  const int64_t row = std::max(a.ldx, a.ldy) * like.element_size();
  TORCH_CHECK(near(row), "linear_act: rows of ", row,
              " bytes are too far apart");
  TORCH_CHECK(linear_plan(&a, type), "linear_act: a product of ", a.m, " x ",
              a.n, " values is too large for a launch");
  Tensor part;
  if (a.splits > 1) {
    part = torch::empty({a.splits, a.m, a.ld_part},
                        like.options().dtype(torch::kFloat));
    a.part = part.data_ptr<float>();
  }
  launched(linear_product_launch(&a, type, stream), "linear_act");
}

// Returns y and what the backward keeps (undefined where not wanted).
std::vector<Tensor> linear_fwd(const Tensor& x, const Tensor& w,
                               const std::optional<Tensor>& bias, int64_t act,
                               const std::optional<Tensor>& residual,
                               bool want_kept) {
  const int type = elem_type(x, "linear_act");
  TORCH_CHECK(x.is_cuda(), "linear_act: x must be on GPU");
  TORCH_CHECK(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1) &&
                  w.size(0) >= 1,
              "linear_act: x [..., K] and weight [N, K], N at least 1; got ",
              x.sizes(), " and ", w.sizes());
  const int64_t K = x.size(-1), N = w.size(0);
  auto shape = x.sizes().vec();
  shape.back() = N;
  int64_t M = 1;
  for (size_t i = 0; i + 1 < shape.size(); ++i) M *= shape[i];
  TORCH_CHECK(M <= kMostRows && N <= kMostRows && K <= kMostRows,
              "linear_act: more than 2^30 rows or columns");
  TORCH_CHECK(!want_kept || near((N + 7) * x.element_size()),
              "linear_act: ", N, " columns are too many for the gradients");
  const auto like_x = [&](const Tensor& t, const char* name) {
    TORCH_CHECK(t.device() == x.device() &&
                    t.scalar_type() == x.scalar_type(),
                "linear_act: ", name, " must have x's type and device");
  };
  like_x(w, "weight");
  if (bias) {
    like_x(*bias, "bias");
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == N,
                "linear_act: bias must be [", N, "]");
  }
  if (residual) {
    like_x(*residual, "residual");
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(shape),
                "linear_act: residual must have the output's shape ", shape);
  }
  TORCH_CHECK(act >= kActNone && act <= kActSilu, "linear_act: activation");
  const c10::DeviceGuard guard(x.device());
  const hipStream_t stream = current();
  Tensor y = torch::empty(shape, x.options().memory_format(
                                     at::MemoryFormat::Contiguous));
  Tensor kept;
  if (want_kept && act != kActNone)
    kept = type == 0 ? torch::empty_like(y)
                     : torch::empty_like(y, torch::kShort);
  if (M == 0) return {y, kept};

  const Operand xo(as_matrix(x, M, K), type, stream);
  const Operand wo(as_matrix(w, N, K), type, stream);
  Tensor b, r;
  LinearProduct a{};
  a.x = xo.held.data_ptr();
  a.y = wo.held.data_ptr();
  a.ldx = xo.ld;
  a.ldy = wo.ld;
  a.m = a.ext_x = (int)M;
  a.n = a.ext_y = (int)N;
  a.kx = a.ky = xo.width;
  a.e.act = (int)act;
  a.e.y = y.data_ptr();
  a.e.kept = kept.defined() ? kept.data_ptr() : nullptr;
  if (bias) {
    b = bias->resolve_neg().contiguous();
    a.e.bias = b.data_ptr();
  }
  if (residual) {
    r = as_matrix(*residual, M, N);
    a.e.residual = r.data_ptr();
    a.e.ld_residual = M > 1 ? r.stride(0) : N;
  }
  product(a, type, x, stream);
  return {y, kept};
}

// Returns dx, dw, db; undefined where not wanted.
std::vector<Tensor> linear_bwd(const Tensor& dy,
                               const Tensor& kept, const Tensor& x,
                               const Tensor& w, int64_t act, bool want_dx,
                               bool want_dw, bool want_db) {
  const int type = elem_type(x, "linear_act");
  const int64_t K = x.size(-1), N = w.size(0);
  const int64_t M = K ? x.numel() / K : dy.numel() / N;
  TORCH_CHECK(dy.numel() == M * N && dy.scalar_type() == x.scalar_type() &&
                  dy.device() == x.device(),
              "linear_act: the output's gradient does not match");
  const c10::DeviceGuard guard(x.device());
  const hipStream_t stream = current();
  const auto fresh = x.options().memory_format(at::MemoryFormat::Contiguous);
  Tensor dx, dw, db;
  if (want_dx) dx = torch::empty(x.sizes(), fresh);
  if (want_dw) dw = M && K ? torch::empty({N, K}, fresh)
                           : torch::zeros({N, K}, fresh);
  if (want_db) db = M ? torch::empty({N}, fresh) : torch::zeros({N}, fresh);
  if (M == 0) return {dx, dw, db};

  // dz and the column sums in one pass; without an activation the products
  // take dy itself where it is aligned for them.
  const Tensor g = as_matrix(dy, M, N);
  const int64_t per = 16 / x.element_size();
  const int64_t Np = (N + per - 1) / per * per;
  const long ldg = M > 1 ? g.stride(0) : Np;
  const bool products = want_dx || want_dw;
  const bool as_is = act == kActNone && N == Np && ldg % per == 0 &&
                     near(ldg * x.element_size()) && aligned16(g.data_ptr());
  Tensor dz = g;
  long ld_dz = ldg;
  LinearDz z{};
  // Of a slope that is no 0 or 1, dz has more than 16 bits: the products take
  // it as the sum of two numbers.
  const bool parts = products && type != 0 && act > kActRelu;
  if (products && !as_is) {
    dz = torch::empty({parts ? 2 * M : M, Np}, fresh);
    ld_dz = Np;
    z.dz = dz.data_ptr();
    z.ld_dz = (int)Np;
    z.second = parts ? M * Np : 0;
  }
  const long second = z.second * x.element_size();
  if (z.dz != nullptr || want_db) {
    z.dy = g.data_ptr();
    z.kept = act == kActNone ? nullptr : kept.data_ptr();
    z.ld_dy = ldg;
    z.m = (int)M;
    z.n = (int)N;
    z.strips = linear_dz_strips(z.m, z.n);
    Tensor part;
    if (want_db) {
      part = torch::empty({z.strips, norm_part_half(z.n)},
                          x.options().dtype(torch::kFloat));
      z.part = part.data_ptr<float>();
    }
    launched(linear_dz_launch(&z, type, stream), "linear_act backward");
    if (want_db)
      launched(sum_rows_launch(z.part, z.strips, norm_part_half(z.n),
                               norm_part_half(z.n), z.n, db.data_ptr(),
                               nullptr, type, stream),
               "linear_act backward");
  }
  if (K == 0) return {dx, dw, db};
  if (want_dx) {
    const Operand wo(as_matrix(w, N, K), type, stream);
    LinearProduct a{};
    a.x = dz.data_ptr();
    a.second = second;
    a.ldx = ld_dz;
    a.kx = (int)Np;
    a.m = a.ext_x = (int)M;
    a.y = wo.held.data_ptr();
    a.ldy = wo.ld;
    a.y_trans = true;
    a.ky = (int)N;
    a.n = (int)K;
    a.ext_y = wo.width;
    a.e.y = dx.data_ptr();
    product(a, type, x, stream);
  }
  if (want_dw) {
    const Operand xo(as_matrix(x, M, K), type, stream);
    LinearProduct a{};
    a.x = dz.data_ptr();
    a.second = second;
    a.ldx = ld_dz;
    a.x_trans = a.y_trans = true;
    a.kx = a.ky = (int)M;
    a.m = (int)N;
    a.ext_x = (int)Np;
    a.y = xo.held.data_ptr();
    a.ldy = xo.ld;
    a.n = (int)K;
    a.ext_y = xo.width;
    a.e.y = dw.data_ptr();
    product(a, type, x, stream);
  }
  return {dx, dw, db};
}

bool is_capturing(hipStream_t stream, const char* what) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  launched(hipStreamIsCapturing(stream, &status), what);
  return status != hipStreamCaptureStatusNone;
}

// A leaf's gradient goes through the accumulator that a live graph of it
// holds, on the stream where that was made. In the capture of a backward this
// would tie that stream to the captured one, which ends the process. Whether
// it is another one than the forward's shows in the forward, also behind casts
// and views of the leaf (the head's weights are cast to its inputs' type).
bool held_elsewhere(const Tensor& x,
                    std::initializer_list<const Tensor*> inputs) {
  const auto stream = c10::hip::getCurrentHIPStream(x.device().index());
  for (const Tensor* t : inputs) {
    if (t == nullptr || !t->requires_grad()) continue;
    auto node = t->is_leaf()
                    ? torch::autograd::impl::try_get_grad_accumulator(*t)
                    : t->grad_fn();
    for (int i = 0; i < 8 && node && node->num_outputs() == 1; ++i)
      node = node->next_edge(0).function;
    if (!node || node->num_outputs() != 0) continue;
    const auto at = node->stream();
    if (at && at->id() != stream.unwrap().id()) return true;
  }
  return false;
}

void check_capture(bool held, const char* what) {
  TORCH_CHECK(!held || !is_capturing(current(), what), what,
              ": a captured backward of a leaf that an earlier graph, made on "
              "another stream, still holds; free that graph first");
}

const Tensor* given(const std::optional<Tensor>& t) {
  return t ? &*t : nullptr;
}

// The autograd nodes are in C++: small layers are bound by the host's time.
class LinearActNode
    : public torch::autograd::Function<LinearActNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx,
                        const Tensor& x, const Tensor& w,
                        const std::optional<Tensor>& bias,
                        const std::optional<Tensor>& residual, int64_t act) {
    auto out = linear_fwd(x, w, bias, act, residual, true);
    ctx->save_for_backward({x, w, out[1]});
    const bool held = held_elsewhere(x, {&x, &w, given(bias), given(residual)});
    // The edges are the given tensors' alone: which there are goes with act.
    ctx->saved_data["act"] =
        act | (bias ? 8 : 0) | (residual ? 16 : 0) | (held ? 32 : 0);
    return out[0];
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "linear_act: its gradients have no gradient (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const int64_t act = ctx->saved_data["act"].toInt();
    check_capture(act & 32, "linear_act");
    const bool bias = act & 8, residual = act & 16;
    auto g = linear_bwd(grads[0], saved[2], saved[0], saved[1], act & 7,
                        ctx->needs_input_grad(0), ctx->needs_input_grad(1),
                        bias && ctx->needs_input_grad(2));
    const bool dr = residual && ctx->needs_input_grad(bias ? 3 : 2);
    return {g[0], g[1], g[2], dr ? grads[0] : Tensor(), Tensor()};
  }
};

// The kernels know no tangents: a result without one would count as a
// derivative of zero.
void refuse_forward_mode(std::initializer_list<const Tensor*> inputs,
                         const char* what) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(t == nullptr || !t->_fw_grad(0).defined(), what,
                                ": no forward-mode derivatives");
}

bool wants_grad(const std::optional<Tensor>& t) {
  return t && t->requires_grad();
}

Tensor linear_act(const Tensor& x, const Tensor& w,
                  const std::optional<Tensor>& bias, int64_t act,
                  const std::optional<Tensor>& residual) {
  refuse_forward_mode({&x, &w, given(bias), given(residual)}, "linear_act");
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || w.requires_grad() || wants_grad(bias) ||
       wants_grad(residual)))
    return LinearActNode::apply(x, w, bias, residual, act);
  return linear_fwd(x, w, bias, act, residual, false)[0];
}

class LayerNormNode : public torch::autograd::Function<LayerNormNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx,
                        const Tensor& x, const std::optional<Tensor>& w,
                        const std::optional<Tensor>& b, double eps) {
    auto out = layer_norm_fwd(x, w, b, eps, true);
    ctx->save_for_backward({x, w ? *w : Tensor(), out[1]});
    const bool held = held_elsewhere(x, {&x, given(w), given(b)});
    // The edges are the given tensors' alone: which there are goes with the
    // parameters' type.
    ctx->saved_data["given"] =
        (int64_t)(w ? w->scalar_type()
                    : b ? b->scalar_type() : x.scalar_type()) |
        (w ? 256 : 0) | (b ? 512 : 0) | (held ? 1024 : 0);
    return out[0];
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "layer_norm: its gradients have no gradient (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const int64_t given = ctx->saved_data["given"].toInt();
    check_capture(given & 1024, "layer_norm");
    const bool weight = given & 256, bias = given & 512;
    auto g = layer_norm_bwd(
        grads[0], saved[0],
        weight ? std::optional<Tensor>(saved[1]) : std::nullopt,
        (torch::ScalarType)(given & 255), saved[2], ctx->needs_input_grad(0),
        weight && ctx->needs_input_grad(1),
        bias && ctx->needs_input_grad(weight ? 2 : 1));
    return {g[0], g[1], g[2], Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& w,
                  const std::optional<Tensor>& b, double eps) {
  refuse_forward_mode({&x, given(w), given(b)}, "layer_norm");
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wants_grad(w) || wants_grad(b)))
    return LayerNormNode::apply(x, w, b, eps);
  return layer_norm_fwd(x, w, b, eps, false)[0];
}

// ----------------------------------------------------------------- AdamW

// Ranges of memory that a call writes or reads: no written one may meet
// another.
struct Ranges {
  struct Range { uintptr_t from, to; bool written; };
  std::vector<Range> all;
  void add(const Tensor& t, bool written) {
    const auto a = (uintptr_t)t.data_ptr();
    if (t.numel())
      all.push_back({a, a + (uintptr_t)t.numel() * t.element_size(), written});
  }
  void check(const char* what) {
    std::sort(all.begin(), all.end(),
              [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t written = 0, any = 0;      // where the ranges so far end
    for (const Range& r : all) {
      TORCH_CHECK(r.from >= (r.written ? any : written), what,
                  ": a tensor to write shares memory with another");
      any = std::max(any, r.to);
      if (r.written) written = std::max(written, r.to);
    }
  }
};

// Autograd sees that a tensor's values have changed.
void changed(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

constexpr int64_t kBlock8 = 256;

void adamw_step(const Tensors& p, const Tensors& g, const Tensors& m,
                const Tensors& v, const std::optional<Tensors>& ms,
                const std::optional<Tensors>& vs,
                const std::optional<Tensor>& norm, double max_norm,
                double step, double lr, double beta1, double beta2,
                double eps, double weight_decay,
                std::optional<uint64_t> seed) {
  const size_t count = p.size();
  TORCH_CHECK(g.size() == count && m.size() == count && v.size() == count &&
                  ms.has_value() == vs.has_value() &&
                  (!ms || (ms->size() == count && vs->size() == count)),
              "adamw_step: the lists have different lengths");
  if (count == 0) return;
  const auto device = p[0].device();
  TORCH_CHECK(device.is_cuda(), "adamw_step: parameters must be on GPU");
  const auto state_type = ms ? torch::kByte : torch::kFloat;
  if (norm)
    TORCH_CHECK(norm->device() == device && norm->numel() == 1 &&
                    norm->scalar_type() == torch::kFloat,
                "adamw_step: grad_norm must be one float32 on the "
                "parameters' device");
  const c10::DeviceGuard guard(device);
  const hipStream_t stream = current();
  TORCH_CHECK(!is_capturing(stream, "adamw_step"),
              "adamw_step: the step's number and rate are the host's and "
              "would stay the same in every replay of a captured graph");

  Ranges ranges;
  ranges.all.reserve(count * (ms ? 6 : 4) + 1);
  if (norm) ranges.add(*norm, false);
  Tensors copies;               // gradients laid out like their parameter
  std::vector<const void*> grads(count);
  for (size_t i = 0; i < count; ++i) {
    TORCH_CHECK(p[i].device() == device && g[i].device() == device &&
                    m[i].device() == device && v[i].device() == device,
                "adamw_step: tensor ", i, " is on another device");
    TORCH_CHECK(!g[i].is_sparse(), "adamw_step: gradient ", i, " is sparse");
    TORCH_CHECK(g[i].scalar_type() == p[i].scalar_type() &&
                    m[i].scalar_type() == state_type &&
                    v[i].scalar_type() == state_type,
                "adamw_step: tensor ", i,
                ": the gradient must have the parameter's type and the "
                "states must be ", state_type);
    TORCH_CHECK(g[i].sizes() == p[i].sizes() && m[i].sizes() == p[i].sizes() &&
                    v[i].sizes() == p[i].sizes(),
                "adamw_step: tensor ", i, ": sizes differ");
    TORCH_CHECK(p[i].is_non_overlapping_and_dense() && !p[i].is_neg() &&
                    !m[i].is_neg() && !v[i].is_neg(),
                "adamw_step: parameter ", i, " must be dense, and it and its "
                "states no negative views");
    elem_type(p[i], "adamw_step");
    const bool plain = p[i].is_contiguous();
    const auto laid_out = [&](const Tensor& t) {
      return plain ? t.is_contiguous() : t.strides() == p[i].strides();
    };
    TORCH_CHECK(laid_out(m[i]) && laid_out(v[i]), "adamw_step: the states of "
                "tensor ", i, " must have the parameter's strides");
    if (laid_out(g[i]) && !g[i].is_neg()) {
      grads[i] = g[i].data_ptr();
      ranges.add(g[i], false);
    } else {
      copies.push_back(torch::empty_strided(p[i].sizes(), p[i].strides(),
                                            p[i].options()).copy_(g[i]));
      grads[i] = copies.back().data_ptr();
    }
    ranges.add(p[i], true);
    ranges.add(m[i], true);
    ranges.add(v[i], true);
    if (ms) {
      const int64_t blocks = (p[i].numel() + kBlock8 - 1) / kBlock8;
      for (const Tensor* s : {&(*ms)[i], &(*vs)[i]}) {
        TORCH_CHECK(s->device() == device &&
                        s->scalar_type() == torch::kByte &&
                        s->is_contiguous() && s->numel() == blocks,
                    "adamw_step: the scales of tensor ", i, " must be ",
                    blocks, " contiguous bytes");
        ranges.add(*s, true);
      }
    }
  }
  ranges.check("adamw_step");

  AdamWScalars s{};
  s.beta1 = (float)beta1;
  s.one_minus_beta1 = (float)(1.0 - beta1);
  s.beta2 = (float)beta2;
  s.one_minus_beta2 = (float)(1.0 - beta2);
  s.eps = (float)eps;
  s.decay = (float)(1.0 - lr * weight_decay);
  s.rate = (float)(lr / (1.0 - std::pow(beta1, step)));
  s.inv_bc2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, step)));
  s.max_norm = (float)max_norm;
  s.norm = norm ? norm->data_ptr<float>() : nullptr;

  // The random bits' keys go by the tensor's number in the call.
  std::vector<unsigned> keys;
  if (ms && seed) {
    const auto number = (uint64_t)(int64_t)step;
    unsigned key = 0;
    for (const uint64_t word : {*seed, number})
      key = adamw_key(adamw_key(key, (unsigned)word), (unsigned)(word >> 32));
    for (size_t i = 0; i < count; ++i)
      keys.push_back(adamw_key(key, (unsigned)i));
  }

  // One launch takes tensors of one type.
  for (int type = 0; type < 3; ++type) {
    std::vector<void*> tp, tm, tv;
    std::vector<const void*> tg;
    std::vector<unsigned char*> tms, tvs;
    std::vector<unsigned> tk;
    std::vector<long> tn;
    for (size_t i = 0; i < count; ++i) {
      if (p[i].numel() == 0 || elem_type(p[i], "adamw_step") != type) continue;
      tp.push_back(p[i].data_ptr());
      tg.push_back(grads[i]);
      tm.push_back(m[i].data_ptr());
      tv.push_back(v[i].data_ptr());
      if (ms) {
        tms.push_back((*ms)[i].data_ptr<uint8_t>());
        tvs.push_back((*vs)[i].data_ptr<uint8_t>());
      }
      if (!keys.empty()) tk.push_back(keys[i]);
      tn.push_back(p[i].numel());
    }
    if (tp.empty()) continue;
    const AdamWTensors a{(int)tp.size(), tp.data(), tg.data(), tm.data(),
                         tv.data(), ms ? tms.data() : nullptr,
                         ms ? tvs.data() : nullptr,
                         tk.empty() ? nullptr : tk.data(), tn.data()};
    launched(adamw_launch(&a, &s, type, stream), "adamw_step");
  }
  for (size_t i = 0; i < count; ++i) {
    changed(p[i]);
    changed(m[i]);
    changed(v[i]);
    if (ms) {
      changed((*ms)[i]);
      changed((*vs)[i]);
    }
  }
}

Tensor norm_of(const Tensors& g) {
  const auto device = g[0].device();
  TORCH_CHECK(device.is_cuda(), "grad_norm: tensors must be on GPU");
  const c10::DeviceGuard guard(device);
  Tensors dense;
  std::vector<const void*> at[3];
  std::vector<long> n[3];
  long parts = 0, values = 0;
  for (const Tensor& t : g) values += t.numel();
  const int chunk = square_sum_chunk(values);
  for (const Tensor& t : g) {
    TORCH_CHECK(t.device() == device,
                "grad_norm: the tensors are on several devices");
    const int type = elem_type(t, "grad_norm");
    TORCH_CHECK(!t.is_sparse(), "grad_norm: a tensor is sparse");
    if (t.numel() == 0) continue;
    if (t.is_non_overlapping_and_dense()) {   // a sign changes no square
      at[type].push_back(t.data_ptr());
    } else {
      dense.push_back(t.contiguous());
      at[type].push_back(dense.back().data_ptr());
    }
    n[type].push_back(t.numel());
    parts += (t.numel() + chunk - 1) / chunk;
  }
  const auto opts = torch::TensorOptions().device(device);
  Tensor out = torch::empty({}, opts.dtype(torch::kFloat));
  Tensor partial = torch::empty({parts}, opts.dtype(torch::kDouble));
  double* next = parts ? partial.data_ptr<double>() : nullptr;
  for (int type = 0; type < 3; ++type) {
    if (at[type].empty()) continue;
    launched(square_sum_launch(at[type].data(), n[type].data(),
                               (int)at[type].size(), chunk, type, next,
                               current()),
             "grad_norm");
    for (const long k : n[type]) next += (k + chunk - 1) / chunk;
  }
  launched(norm_launch(parts ? partial.data_ptr<double>() : nullptr,
                       (int)parts, out.data_ptr<float>(), current()),
           "grad_norm");
  return out;
}

// d |g| / d g = g / |g|, for a norm that is a part of a loss.
class GradNormNode : public torch::autograd::Function<GradNormNode> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx,
                        at::TensorList g) {
    Tensors saved = g.vec();
    saved.push_back(norm_of(saved));
    ctx->save_for_backward(saved);
    return saved.back();
  }

  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx,
      torch::autograd::variable_list grads) {
    auto saved = ctx->get_saved_variables();
    const Tensor scale = grads[0] / saved.back();
    saved.pop_back();
    for (Tensor& t : saved)
      t = (t.to(torch::kFloat) * scale).to(t.scalar_type());
    return saved;
  }
};

Tensor grad_norm(const Tensors& g) {
  TORCH_CHECK(!g.empty(), "grad_norm: no tensors");
  bool wanted = false;
  for (const Tensor& t : g) {
    refuse_forward_mode({&t}, "grad_norm");
    wanted |= t.requires_grad();
  }
  return wanted && at::GradMode::is_enabled()
             ? GradNormNode::apply(at::TensorList(g)) : norm_of(g);
}

std::tuple<Tensor, Tensor> pack_state8(const Tensor& x, bool is_signed) {
  TORCH_CHECK(x.is_cuda() && x.scalar_type() == torch::kFloat &&
                  x.is_non_overlapping_and_dense() && !x.is_neg(),
              "pack_state8: a dense float32 tensor on GPU");
  const c10::DeviceGuard guard(x.device());
  Tensor codes = torch::empty_strided(x.sizes(), x.strides(),
                                      x.options().dtype(torch::kByte));
  Tensor scales = torch::empty({(x.numel() + kBlock8 - 1) / kBlock8},
                               x.options().dtype(torch::kByte));
  if (x.numel())
    launched(pack8_launch(x.data_ptr<float>(), codes.data_ptr<uint8_t>(),
                          scales.data_ptr<uint8_t>(), x.numel(), is_signed,
                          current()),
             "pack_state8");
  return {codes, scales};
}

Tensor unpack_state8(const Tensor& codes, const Tensor& scales,
                     bool is_signed, torch::ScalarType dtype) {
  TORCH_CHECK(codes.is_cuda() && codes.scalar_type() == torch::kByte &&
                  codes.is_non_overlapping_and_dense(),
              "unpack_state8: codes must be dense bytes on GPU");
  TORCH_CHECK(scales.device() == codes.device() &&
                  scales.scalar_type() == torch::kByte &&
                  scales.is_contiguous() &&
                  scales.numel() == (codes.numel() + kBlock8 - 1) / kBlock8,
              "unpack_state8: scales must be one byte for 256 codes");
  const c10::DeviceGuard guard(codes.device());
  Tensor out = torch::empty_strided(codes.sizes(), codes.strides(),
                                    codes.options().dtype(dtype));
  const int type = elem_type(out, "unpack_state8");
  if (codes.numel())
    launched(unpack8_launch(codes.data_ptr<uint8_t>(),
                            scales.data_ptr<uint8_t>(), out.data_ptr(),
                            codes.numel(), is_signed, type, current()),
             "unpack_state8");
  return out;
}

}  // namespace

void register_train_ops(pybind11::module_& m) {
  m.def("linear_act", &linear_act,
        "matrix product + bias + activation + residual (CDNA4 MFMA)");
  m.def("layer_norm", &layer_norm, "layer norm (CDNA4)");
  m.def("adamw_step", &adamw_step, "AdamW step over many tensors (CDNA4)");
  m.def("grad_norm", &grad_norm, "2-norm over many tensors (CDNA4)");
  m.def("pack_state8", &pack_state8, "fp32 -> 8-bit optimizer state");
  m.def("unpack_state8", &unpack_state8, "8-bit optimizer state -> values");
}
