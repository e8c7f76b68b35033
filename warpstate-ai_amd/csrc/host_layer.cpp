// Host side of the residual norm, the embedding and the experts' products as PyTorch operators in
// C++: the checks, allocations, launches and autograd nodes of ops/residual_norm.py,
// ops/embedding_execution.py and ops/grouped_execution.py without Python. Shapes and types only on fake
// tensors.
//
// Autograd kernels read no data; they call operators below autograd. First derivatives by reverse
// mode only: tensors that carry a tangent are refused, and so is a second differentiation.
#include <cmath>

#include "host_common.h"

namespace {

typedef std::tuple<Tensor, Tensor> TwoTensors;
typedef std::tuple<Tensor, Tensor, Tensor> ThreeTensors;

// A tensor's rows of its last dimension, with a unit column stride and no overlap: a view or a copy.
Tensor rows_of(const Tensor& t) {
  const int64_t cols = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / cols, cols});
  const bool unit = (r.stride(1) == 1 || cols == 1) && (r.size(0) <= 1 || r.stride(0) >= cols);
  return unit ? r : r.contiguous();
}
// A size that the checks and kernels go by: a number, also of a tensor traced with symbolic sizes (the row
// counts, which may stay symbolic, are not asked for here).
int64_t fixed(const Tensor& t, int64_t dim) { return t.sym_size(dim).guard_int(__FILE__, __LINE__); }

// Gradients that are not differentiable again: where a graph of the backward is recorded, they stand
// behind a node that depends on everything they were made `from`, and refuses. `inputs`: how many of the first inputs
// of the node that is being evaluated it depends on too, by their edges, so that none has to be saved for that.
struct OnceFn : Function<OnceFn> {
  static variable_list forward(AutogradContext* ctx, at::TensorList grads, at::TensorList from, std::string message) {
    ctx->saved_data["message"] = message;
    variable_list out;
    for (const auto& g : grads) out.push_back(g.alias());
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list) {
    TORCH_CHECK(false, ctx->saved_data["message"].toStringRef());
  }
};
variable_list once(variable_list grads, const variable_list& from, const char* message, size_t inputs = 0) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list known, sources;
  for (const auto& t : from)
    if (t.defined() && t.requires_grad()) sources.push_back(t);
  if (const auto node = torch::autograd::get_current_node())
    for (size_t i = 0; i < inputs && i < node->num_outputs(); ++i)
      if (const auto& edge = node->next_edge(i); edge.is_valid()) {
        sources.push_back(at::empty({0}));
        torch::autograd::impl::set_gradient_edge(sources.back(), edge);
      }
  if (sources.empty()) return grads;
  for (const auto& g : grads)
    if (g.defined()) known.push_back(g);
  known = OnceFn::apply(at::TensorList(known), at::TensorList(sources), std::string(message));
  size_t next = 0;
  for (auto& g : grads)
    if (g.defined()) g = known[next++];
  return grads;
}

// --- residual norm --------------------------------------------------------------------------

constexpr int64_t kMaxWidth = 8192;
constexpr char kNormTwice[] = "the residual norm cannot be differentiated twice";

void check_norm(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && x.dim() >= 1, "Expected BF16 rows");
  const int64_t d = fixed(x, -1);
  TORCH_CHECK_VALUE(d >= 1 && d <= kMaxWidth, "RMSNorm takes rows of 1 to ", kMaxWidth, " columns, not ", d);
  TORCH_CHECK_VALUE(weight.scalar_type() == at::kFloat && weight.dim() == 1 && fixed(weight, 0) == d &&
                        weight.device() == x.device(),
                    "The norm's weight must be a vector of ", d, " values on ", x.device());
  if (residual.has_value())
    TORCH_CHECK_VALUE((residual->scalar_type() == at::kBFloat16 || residual->scalar_type() == at::kFloat) &&
                          residual->sym_sizes() == x.sym_sizes() && residual->device() == x.device(),
                      "The residual must be BF16 or FP32, of shape ", x.sym_sizes(), " on ", x.device());
}

TwoTensors add_rmsnorm(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  check_norm(x, residual, weight);
  c10::DeviceGuard guard(x.device());
  const Tensor a = rows_of(x), r = rows_of(residual), w = weight.contiguous();
  const int64_t rows = a.size(0), d = a.size(1);
  Tensor y = at::empty(x.sizes(), x.options()), stream = at::empty(x.sizes(), residual.options());
  check(ws_add_rmsnorm(ptr(a), row_stride(a), ptr(r), row_stride(r), r.scalar_type() == at::kFloat,
                       w.const_data_ptr<float>(), (float)eps, rows, d, ptr(y), ptr(stream), stream_of(x)),
        "ws_add_rmsnorm");
  return {y, stream};
}
// (dx, dresidual, dweight); dresidual is empty for a BF16 stream, whose gradient is dx.
ThreeTensors add_rmsnorm_backward(const Tensor& stream, const Tensor& weight, double eps, const Tensor& dy,
                                  const std::optional<Tensor>& dstream) {
  c10::DeviceGuard guard(stream.device());
  const bool f32 = stream.scalar_type() == at::kFloat;
  Tensor dx = at::empty(stream.sizes(), dy.options()), dweight = at::empty_like(weight, at::MemoryFormat::Contiguous);
  Tensor dresidual = f32 ? at::empty(stream.sizes(), stream.options()) : at::empty({0}, stream.options());
  if (stream.numel() == 0) return {dx, dresidual, dweight.zero_()};
  const Tensor s = rows_of(stream), g = rows_of(dy), w = weight.contiguous();
  const Tensor h = dstream.has_value() ? rows_of(*dstream) : Tensor();
  const int64_t rows = s.size(0), d = s.size(1);
  const int64_t need = ws_add_rmsnorm_backward_partial_floats(rows, d);
  Tensor partial = need ? floats(stream, {need}) : Tensor();
  check(ws_add_rmsnorm_backward(s.const_data_ptr(), f32, w.const_data_ptr<float>(), (float)eps,
                                g.const_data_ptr(), row_stride(g), ptr(h), h.defined() ? row_stride(h) : 0, rows, d,
                                dx.data_ptr(), f32 ? dresidual.data_ptr<float>() : nullptr, dweight.data_ptr<float>(),
                                static_cast<float*>(ptr(partial)), stream_of(stream)),
        "ws_add_rmsnorm_backward");
  return {dx, dresidual, dweight};
}

struct AddRmsnormFn : Function<AddRmsnormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& residual, const Tensor& weight,
                               double eps) {
    typedef const Tensor& T;
    static const auto op = find<TwoTensors(T, T, T, double)>("warpstate::native_add_rmsnorm");
    auto [y, stream] = below(op, x, residual, weight, eps);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({stream, weight});
    ctx->saved_data["eps"] = eps;
    return {y, stream};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    typedef const Tensor& T;
    static const auto op =
        find<ThreeTensors(T, T, double, T, const std::optional<Tensor>&)>("warpstate::native_add_rmsnorm_backward");
    const Tensor &dy = grads[0], &dstream = grads[1];
    if (!dy.defined())  // the addition alone
      return {dstream.defined() ? dstream.to(at::kBFloat16) : Tensor(), dstream, Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    auto [dx, dresidual, dweight] =
        below(op, s[0], s[1], ctx->saved_data["eps"].toDouble(), dy, dstream.defined() ? std::optional<Tensor>(dstream) : std::nullopt);
    const bool f32 = s[0].scalar_type() == at::kFloat;
    return once({dx, f32 ? dresidual : dx, dweight, Tensor()}, {s[0], s[1], dy, dstream}, kNormTwice);
  }
};
TwoTensors add_rmsnorm_autograd(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps) {
  refuse_tangents("add_rmsnorm", x, residual, weight);
  if (!records(x, residual, weight)) {
    typedef const Tensor& T;
    static const auto op = find<TwoTensors(T, T, T, double)>("warpstate::native_add_rmsnorm");
    return below(op, x, residual, weight, eps);
  }
  variable_list v = AddRmsnormFn::apply(x, residual, weight, eps);
  return {v[0], v[1]};
}
TwoTensors add_rmsnorm_meta(const Tensor& x, const Tensor& residual, const Tensor& weight, double) {
  check_norm(x, residual, weight);
  return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint(x.sym_sizes(), residual.options())};
}
ThreeTensors add_rmsnorm_backward_meta(const Tensor& stream, const Tensor& weight, double, const Tensor& dy,
                                       const std::optional<Tensor>&) {
  const bool f32 = stream.scalar_type() == at::kFloat;
  return {at::empty_symint(stream.sym_sizes(), dy.options()),
          f32 ? at::empty_symint(stream.sym_sizes(), stream.options()) : at::empty({0}, stream.options()),
          at::empty_like(weight, at::MemoryFormat::Contiguous)};
}

// (q, scale, stream) of ops/residual_norm.py's rmsnorm_quantize, the stream empty without a residual.
ThreeTensors rmsnorm_quantize(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double eps,
                              bool e8m0) {
  check_norm(x, residual, weight);
  TORCH_CHECK_VALUE(x.numel() > 0, "Quantization takes non-empty rows");
  c10::DeviceGuard guard(x.device());
  const Tensor a = rows_of(x), w = weight.contiguous();
  const Tensor r = residual.has_value() ? rows_of(*residual) : Tensor();
  const int64_t rows = a.size(0), d = a.size(1), n = blocks(d);
  Tensor q = at::empty({rows, up(d, 16)}, x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scale = e8m0 ? at::empty({rows, up(n, 4)}, x.options().dtype(at::kFloat8_e8m0fnu)) : floats(x, {n, up(rows, 4)});
  Tensor stream = r.defined() ? at::empty(x.sizes(), r.options()) : at::empty({0}, x.options());
  check(ws_rmsnorm_quantize(a.const_data_ptr(), row_stride(a), ptr(r), r.defined() ? row_stride(r) : 0,
                            r.defined() && r.scalar_type() == at::kFloat, w.const_data_ptr<float>(), (float)eps, rows,
                            d, e8m0 ? WS_SCALE_E8M0 : WS_SCALE_F32, q.data_ptr(), q.size(1), scale.data_ptr(),
                            scale.size(1), r.defined() ? stream.data_ptr() : nullptr, stream_of(x)),
        "ws_rmsnorm_quantize");
  if (q.size(1) != d) q = q.narrow(1, 0, d);
  if (!e8m0) return {q, scale.narrow(1, 0, rows).t(), stream};
  return {q, scale.size(1) == n ? scale : scale.narrow(1, 0, n), stream};
}
ThreeTensors rmsnorm_quantize_autograd(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight,
                                       double eps, bool e8m0) {
  typedef const Tensor& T;
  static const auto op =
      find<ThreeTensors(T, const std::optional<Tensor>&, T, double, bool)>("warpstate::native_rmsnorm_quantize");
  refuse_tangents("rmsnorm_quantize", x, residual.has_value() ? *residual : x, weight);
  return below(op, x, residual, weight, eps, e8m0);
}

ThreeTensors rmsnorm_quantize_meta(const Tensor& x, const std::optional<Tensor>& residual, const Tensor& weight, double,
                                   bool e8m0) {
  check_norm(x, residual, weight);
  TORCH_CHECK_VALUE(x.sym_numel() > 0, "Quantization takes non-empty rows");
  const int64_t d = fixed(x, -1), n = blocks(d);
  const c10::SymInt rows = x.sym_numel() / d;
  Tensor q = at::empty_symint({rows, up(d, 16)}, x.options().dtype(at::kFloat8_e4m3fn)).narrow(1, 0, d);
  Tensor scale = e8m0 ? at::empty_symint({rows, up(n, 4)}, x.options().dtype(at::kFloat8_e8m0fnu)).narrow(1, 0, n)
                      : at::empty_symint({n, (rows + 3) / 4 * 4}, x.options().dtype(at::kFloat)).narrow_symint(1, 0, rows).t();
  return {q, scale, residual.has_value() ? at::empty_symint(x.sym_sizes(), residual->options()) : at::empty({0}, x.options())};
}

// --- embedding ------------------------------------------------------------------------------

constexpr char kEmbeddingTwice[] = "the embedding cannot be differentiated twice";
typedef Tensor Embedding(const Tensor&, const Tensor&, double, bool);

// (The kernels multiply in FP32.)
void check_scale(double scale) {
  TORCH_CHECK_VALUE(std::isfinite((float)scale), "The scale must be finite in FP32, not ", scale);
}
void check_embedding(const Tensor& tokens, const Tensor& table, double scale) {
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong && tokens.device() == table.device(),
                    "Tokens must be int64 on the table's device");
  TORCH_CHECK_VALUE((table.scalar_type() == at::kBFloat16 || table.scalar_type() == at::kFloat) && table.dim() == 2 &&
                        table.sym_numel() > 0,
                    "Expected a non-empty BF16 or FP32 table [vocab, d]");
  check_scale(scale);
}
std::vector<int64_t> embedded(const Tensor& tokens, int64_t d) {
  std::vector<int64_t> sizes = tokens.sizes().vec();
  sizes.push_back(d);
  return sizes;
}
Tensor embedding(const Tensor& tokens_in, const Tensor& table_in, double scale, bool f32) {
  check_embedding(tokens_in, table_in, scale);
  c10::DeviceGuard guard(table_in.device());
  const Tensor tokens = tokens_in.contiguous(), table = rows_of(table_in);
  Tensor y = at::empty(embedded(tokens, table.size(1)), table.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  check(ws_embedding(table.const_data_ptr(), row_stride(table), table.scalar_type() == at::kFloat,
                     static_cast<const int64_t*>(ptr(tokens)), tokens.numel(), table.size(0), table.size(1),
                     (float)scale, ptr(y), f32, stream_of(table)),
        "ws_embedding");
  return y;
}
// The sums of dy by token into `out` [vocab, d].
void embedding_sums(const Tensor& dy, const Tensor& tokens_in, double scale, const Tensor& out, int mode) {
  c10::DeviceGuard guard(out.device());
  const Tensor tokens = tokens_in.contiguous();
  const int64_t rows = tokens.numel(), vocab = out.size(0), d = out.size(1);
  const Tensor g = rows ? rows_of(dy) : Tensor();
  const int64_t need = ws_embedding_backward_workspace_bytes(rows, vocab, d);
  Tensor work = need ? bytes(out, {need}) : Tensor();
  check(ws_embedding_backward(ptr(g), rows ? row_stride(g) : 0, rows && g.scalar_type() == at::kFloat,
                              static_cast<const int64_t*>(ptr(tokens)), rows, vocab, d, (float)scale, out.data_ptr(),
                              row_stride(out), mode, ptr(work), stream_of(out)),
        "ws_embedding_backward");
}
Tensor embedding_backward(const Tensor& dy, const Tensor& tokens, int64_t vocab, double scale, bool f32) {
  c10::DeviceGuard guard(dy.device());
  Tensor out = at::empty({vocab, dy.size(-1)}, dy.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  embedding_sums(dy, tokens, scale, out, f32 ? WS_EMBED_WRITE_F32 : WS_EMBED_WRITE_BF16);
  return out;
}
void embedding_accumulate(Tensor& gradient, const Tensor& tokens, const Tensor& dy, double scale) {
  TORCH_CHECK_VALUE(gradient.scalar_type() == at::kFloat && gradient.dim() == 2 && gradient.numel() > 0 &&
                        (gradient.stride(1) == 1 || gradient.size(1) == 1) &&
                        (gradient.size(0) == 1 || gradient.stride(0) >= gradient.size(1)),
                    "The gradient must be a non-empty FP32 matrix with a unit column stride");
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong && tokens.device() == gradient.device(),
                    "Tokens must be int64 on the gradient's device");
  TORCH_CHECK_VALUE((dy.scalar_type() == at::kBFloat16 || dy.scalar_type() == at::kFloat) &&
                        dy.sizes() == embedded(tokens, gradient.size(1)) && dy.device() == gradient.device(),
                    "Expected BF16 or FP32 rows of shape ", embedded(tokens, gradient.size(1)), " on ", gradient.device());
  check_scale(scale);
  embedding_sums(dy, tokens, scale, gradient, WS_EMBED_ADD_F32);
}

struct EmbeddingFn : Function<EmbeddingFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& tokens, const Tensor& table, double scale, bool f32) {
    static const auto op = find<Embedding>("warpstate::native_embedding");
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = table.sym_size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["f32"] = table.scalar_type() == at::kFloat;
    return below(op, tokens, table, scale, f32);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    typedef const Tensor& T;
    static const auto op = find<Tensor(T, T, c10::SymInt, double, bool)>("warpstate::native_embedding_backward");
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    Tensor d = below(op, grads[0], ctx->get_saved_variables()[0], ctx->saved_data["vocab"].toSymInt(),
                     ctx->saved_data["scale"].toDouble(), ctx->saved_data["f32"].toBool());
    return once({Tensor(), d, Tensor(), Tensor()}, {grads[0]}, kEmbeddingTwice);
  }
};
Tensor embedding_autograd(const Tensor& tokens, const Tensor& table, double scale, bool f32) {
  static const auto op = find<Embedding>("warpstate::native_embedding");
  refuse_tangents("embedding", table);
  if (!records(table)) return below(op, tokens, table, scale, f32);
  return EmbeddingFn::apply(tokens, table, scale, f32);
}
Tensor embedding_meta(const Tensor& tokens, const Tensor& table, double scale, bool f32) {
  check_embedding(tokens, table, scale);
  c10::SymDimVector sizes(tokens.sym_sizes());
  sizes.push_back(table.sym_size(1));
  return at::empty_symint(sizes, table.options().dtype(f32 ? at::kFloat : at::kBFloat16));
}
Tensor embedding_backward_meta(const Tensor& dy, const Tensor&, c10::SymInt vocab, double, bool f32) {
  return at::empty_symint({vocab, dy.sym_size(-1)}, dy.options().dtype(f32 ? at::kFloat : at::kBFloat16));
}

// --- products grouped by expert -------------------------------------------------------------

constexpr char kGroupedTwice[] = "grouped products cannot be differentiated twice";

void check_grouped(const Tensor& x, const Tensor& weight, const Tensor& offsets) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kBFloat16 && x.dim() == 2, "Grouped products take BF16 rows [rows, k]");
  TORCH_CHECK_VALUE((weight.scalar_type() == at::kBFloat16 || weight.scalar_type() == at::kFloat) &&
                        weight.dim() == 3 && fixed(weight, 0) > 0 && fixed(weight, 1) > 0 && fixed(weight, 2) > 0 &&
                        fixed(weight, 2) == fixed(x, 1) && weight.device() == x.device(),
                    "Expected non-empty BF16 or FP32 weights [groups, n, ", fixed(x, 1), "] on ", x.device());
  TORCH_CHECK_VALUE(offsets.scalar_type() == at::kLong && offsets.dim() == 1 &&
                        fixed(offsets, 0) == fixed(weight, 0) + 1 && offsets.device() == x.device(),
                    "Offsets must be an int64 vector, one more than the groups, on ", x.device());
}
// A matrix as the kernels read it: 16-byte rows of a multiple of 8, itself or a copy whose rows are
// padded with zeros.
bool whole_rows(const Tensor& t) {
  auto stride = [&](int64_t i) { return t.sym_stride(i).guard_int(__FILE__, __LINE__); };
  int64_t i = t.dim() - 1, inner = fixed(t, i);
  if (inner % 8 != 0 || (stride(i) != 1 && inner != 1) || t.sym_storage_offset().guard_int(__FILE__, __LINE__) % 8 != 0)
    return false;
  while (i-- > 0) {
    if (t.sym_size(i) > 1 && (stride(i) % 8 != 0 || stride(i) < inner)) return false;
    if (i > 0) inner = fixed(t, i) * stride(i);
  }
  return true;
}
typedef Tensor CopyRows(const Tensor&, c10::SymInt, c10::SymInt, bool);
const auto& copy_rows_op() {
  static const auto op = find<CopyRows>("warpstate::native_copy_rows");
  return op;
}
Tensor grouped_operand(const Tensor& t) {
  if (whole_rows(t)) return t.to(at::kBFloat16);
  return copy_rows_op().call(t, t.sym_size(t.dim() - 2), up(fixed(t, -1), 8), true);
}
// t [rows, cols] or [groups, rows, cols] in other sizes, padded with zeros or cut off: a new tensor, in
// BF16 or in t's type.
Tensor copy_rows(const Tensor& t_in, int64_t rows, int64_t cols, bool bf16) {
  c10::DeviceGuard guard(t_in.device());
  const bool f32 = t_in.scalar_type() == at::kFloat;
  const int64_t d = t_in.dim();
  // (Expanded and overlapping rows can be read; other column strides are copied first.)
  const Tensor t = t_in.stride(d - 1) == 1 || t_in.size(d - 1) == 1 ? t_in : t_in.contiguous();
  const int64_t groups = d == 2 ? 1 : t.size(0), rows_in = t.size(d - 2), cols_in = t.size(d - 1);
  std::vector<int64_t> sizes{rows, cols};
  if (d == 3) sizes.insert(sizes.begin(), groups);
  Tensor out = at::empty(sizes, t.options().dtype(bf16 ? at::kBFloat16 : t.scalar_type()));
  check(ws_copy_rows(ptr(t), f32, d == 2 ? 0 : t.stride(0), t.stride(d - 2), rows_in, cols_in, ptr(out), f32 && !bf16,
                     rows * cols, cols, rows, cols, groups, stream_of(t)),
        "ws_copy_rows");
  return out;
}
Tensor copy_rows_meta(const Tensor& t, c10::SymInt rows, c10::SymInt cols, bool bf16) {
  const auto options = t.options().dtype(bf16 ? at::kBFloat16 : t.scalar_type());
  if (t.dim() == 2) return at::empty_symint({rows, cols}, options);
  return at::empty_symint({t.sym_size(0), rows, cols}, options);
}

// On operands of grouped_operand: [rows, n up to the next multiple of 8] (form NT) or [rows, padded k]
// (NN, x and the reduction reach to w's rows).
Tensor grouped_rows(const Tensor& x, const Tensor& w, const Tensor& offsets_in, int64_t form) {
  c10::DeviceGuard guard(x.device());
  const Tensor offsets = offsets_in.contiguous();
  const bool nt = form == WS_GROUPED_NT;
  const int64_t rows = x.size(0), n = w.size(nt ? 1 : 2), k = w.size(nt ? 2 : 1);
  Tensor y = at::empty({rows, up(n, 8)}, x.options());
  const int64_t need = ws_grouped_workspace_floats(rows, w.size(0), n, k, (int)form);
  Tensor work = need ? floats(x, {need}) : Tensor();
  check(ws_grouped_mm(ptr(x), row_stride(x), w.const_data_ptr(), w.size(1) > 1 ? w.stride(1) : w.size(2),
                      w.size(0) > 1 ? w.stride(0) : 0, (int)form, offsets.const_data_ptr<int64_t>(), w.size(0), rows,
                      n, k, ptr(y), y.size(1), static_cast<float*>(ptr(work)), stream_of(x)),
        "ws_grouped_mm");
  return y;
}
Tensor grouped_grad(const Tensor& dy, const Tensor& x, const Tensor& offsets_in, int64_t n, bool f32) {
  c10::DeviceGuard guard(x.device());
  const Tensor offsets = offsets_in.contiguous();
  const int64_t groups = offsets.size(0) - 1, k = x.size(1);
  Tensor dw = at::empty({groups, n, k}, x.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  check(ws_grouped_weight_grad(ptr(dy), row_stride(dy), ptr(x), row_stride(x), offsets.const_data_ptr<int64_t>(),
                               groups, x.size(0), n, k, dw.data_ptr(), f32, stream_of(x)),
        "ws_grouped_weight_grad");
  return dw;
}
typedef Tensor GroupedRows(const Tensor&, const Tensor&, const Tensor&, int64_t);
typedef Tensor GroupedGrad(const Tensor&, const Tensor&, const Tensor&, int64_t, bool);
// Below autograd.
Tensor first_columns(const Tensor& t, int64_t cols) {
  return fixed(t, -1) == cols ? t : copy_rows_op().call(t, t.sym_size(0), cols, false);
}

// A BF16 operand as the kernel for few rows reads it: with unit column strides and rows apart, else a copy.
Tensor any_rows(const Tensor& t) {
  const int64_t d = t.dim(), cols = t.size(d - 1);
  const bool apart = (t.stride(d - 1) == 1 || cols == 1) && (t.size(d - 2) <= 1 || t.stride(d - 2) >= cols);
  return apart ? t : t.contiguous();
}
Tensor grouped_mm(const Tensor& x, const Tensor& weight, const Tensor& offsets) {
  check_grouped(x, weight, offsets);
  at::AutoDispatchBelowAutograd below_autograd;
  c10::DeviceGuard guard(x.device());
  if (weight.scalar_type() == at::kBFloat16 &&
      ws_grouped_tile(x.size(0), weight.size(0), weight.size(1), weight.size(2), WS_GROUPED_NT) >= 5)
    return first_columns(grouped_rows(any_rows(x), any_rows(weight), offsets, WS_GROUPED_NT), weight.size(1));
  return first_columns(grouped_rows(grouped_operand(x), grouped_operand(weight), offsets, WS_GROUPED_NT),
                       weight.size(1));
}

struct GroupedMmFn : Function<GroupedMmFn> {
  // Gradients go to the tensors x and weight, which the operands a and w were made from. Kept is what they read: dx the
  // weights, dW the rows.
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& a, const Tensor& w,
                        const Tensor& offsets) {
    static const auto op = find<GroupedRows>("warpstate::native_grouped_rows");
    at::AutoDispatchBelowAutograd guard;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({weight.requires_grad() ? a : Tensor(), x.requires_grad() ? w : Tensor(), offsets});
    ctx->saved_data["want_x"] = x.requires_grad();
    ctx->saved_data["want_w"] = weight.requires_grad();
    ctx->saved_data["n"] = fixed(weight, 1);
    ctx->saved_data["k"] = fixed(x, 1);
    ctx->saved_data["f32"] = weight.scalar_type() == at::kFloat;
    return first_columns(op.call(a, w, offsets, WS_GROUPED_NT), fixed(weight, 1));
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto rows_op = find<GroupedRows>("warpstate::native_grouped_rows");
    static const auto grad_op = find<GroupedGrad>("warpstate::native_grouped_grad");
    variable_list d(5);
    if (!grads[0].defined()) return d;
    const auto s = ctx->get_saved_variables();
    const int64_t n = ctx->saved_data["n"].toInt(), k = ctx->saved_data["k"].toInt();
    {
      at::AutoDispatchBelowAutograd guard;
      const Tensor g = grouped_operand(grads[0]);
      if (ctx->saved_data["want_x"].toBool()) d[0] = first_columns(rows_op.call(g, s[1], s[2], WS_GROUPED_NN), k);
      if (ctx->saved_data["want_w"].toBool()) {
        Tensor dw = grad_op.call(g, s[0], s[2], n, ctx->saved_data["f32"].toBool());
        if (fixed(dw, 2) != k) dw = copy_rows_op().call(dw, n, k, false);
        d[1] = dw;
      }
    }
    return once(d, {grads[0]}, kGroupedTwice, 2);
  }
};
Tensor grouped_mm_autograd(const Tensor& x, const Tensor& weight, const Tensor& offsets) {
  refuse_tangents("grouped_mm", x, weight);
  if (!records(x, weight)) {
    static const auto op = find<Tensor(const Tensor&, const Tensor&, const Tensor&)>("warpstate::native_grouped_mm");
    return below(op, x, weight, offsets);
  }
  check_grouped(x, weight, offsets);
  // (A symbolic number of rows is left to the backward.)
  if (const auto rows = x.sym_size(0).maybe_as_int())
    check(ws_grouped_backward_check(*rows, fixed(weight, 0), fixed(weight, 1), fixed(x, 1), x.requires_grad(),
                                    weight.requires_grad(), weight.scalar_type() == at::kFloat),
          "ws_grouped_backward_check");
  Tensor a = x.detach(), w = weight.detach();
  {
    at::AutoDispatchBelowAutograd below_autograd;
    a = grouped_operand(a);
    w = grouped_operand(w);
  }
  return GroupedMmFn::apply(x, weight, a, w, offsets);
}
Tensor grouped_mm_meta(const Tensor& x, const Tensor& weight, const Tensor& offsets) {
  check_grouped(x, weight, offsets);
  return at::empty_symint({x.sym_size(0), weight.sym_size(1)}, x.options());
}
Tensor grouped_rows_meta(const Tensor& x, const Tensor& w, const Tensor&, int64_t form) {
  return at::empty_symint({x.sym_size(0), up(fixed(w, form == WS_GROUPED_NT ? 1 : 2), 8)}, x.options());
}
Tensor grouped_grad_meta(const Tensor&, const Tensor& x, const Tensor& offsets, int64_t n, bool f32) {
  return at::empty_symint({offsets.sym_size(0) - 1, n, x.sym_size(1)},
                          x.options().dtype(f32 ? at::kFloat : at::kBFloat16));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(warpstate, m) {
  m.def("native_add_rmsnorm(Tensor x, Tensor residual, Tensor weight, float eps) -> (Tensor, Tensor)");
  m.def(
      "native_add_rmsnorm_backward(Tensor stream, Tensor weight, float eps, Tensor dy, Tensor? dstream) -> "
      "(Tensor, Tensor, Tensor)");
  m.def(
      "native_rmsnorm_quantize(Tensor x, Tensor? residual, Tensor weight, float eps, bool e8m0) -> (Tensor, Tensor, "
      "Tensor)");
  m.def("native_embedding(Tensor tokens, Tensor table, float scale, bool f32) -> Tensor");
  m.def("native_embedding_backward(Tensor dy, Tensor tokens, SymInt vocab, float scale, bool f32) -> Tensor");
  m.def("native_embedding_accumulate_(Tensor(a!) gradient, Tensor tokens, Tensor dy, float scale) -> ()");
  m.def("native_grouped_mm(Tensor x, Tensor weight, Tensor offsets) -> Tensor");
  m.def("native_copy_rows(Tensor t, SymInt rows, SymInt cols, bool bf16) -> Tensor");
  m.def("native_grouped_rows(Tensor x, Tensor w, Tensor offsets, int form) -> Tensor");
  m.def("native_grouped_grad(Tensor dy, Tensor x, Tensor offsets, int n, bool f32) -> Tensor");
}
TORCH_LIBRARY_IMPL(warpstate, CUDA, m) {
  m.impl("native_add_rmsnorm", &add_rmsnorm);
  m.impl("native_add_rmsnorm_backward", &add_rmsnorm_backward);
  m.impl("native_rmsnorm_quantize", &rmsnorm_quantize);
  m.impl("native_embedding", &embedding);
  m.impl("native_embedding_backward", &embedding_backward);
  m.impl("native_embedding_accumulate_", &embedding_accumulate);
  m.impl("native_grouped_mm", &grouped_mm);
  m.impl("native_copy_rows", &copy_rows);
  m.impl("native_grouped_rows", &grouped_rows);
  m.impl("native_grouped_grad", &grouped_grad);
}
TORCH_LIBRARY_IMPL(warpstate, AutogradCUDA, m) {
  m.impl("native_add_rmsnorm", &add_rmsnorm_autograd);
  m.impl("native_rmsnorm_quantize", &rmsnorm_quantize_autograd);
  m.impl("native_embedding", &embedding_autograd);
  m.impl("native_grouped_mm", &grouped_mm_autograd);
}
TORCH_LIBRARY_IMPL(warpstate, Meta, m) {
  m.impl("native_add_rmsnorm", &add_rmsnorm_meta);
  m.impl("native_add_rmsnorm_backward", &add_rmsnorm_backward_meta);
  m.impl("native_rmsnorm_quantize", &rmsnorm_quantize_meta);
  m.impl("native_embedding", &embedding_meta);
  m.impl("native_embedding_backward", &embedding_backward_meta);
  m.impl("native_grouped_mm", &grouped_mm_meta);
  m.impl("native_copy_rows", &copy_rows_meta);
  m.impl("native_grouped_rows", &grouped_rows_meta);
  m.impl("native_grouped_grad", &grouped_grad_meta);
}
