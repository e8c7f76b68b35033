// Host side of the 8-bit projections and the token scores as PyTorch operators in C++.
//
// ops/fp8_execution.py and ops/token_scores.py check their arguments in Python and launch
// through ctypes; allocating the outputs, the calls and above all the autograd nodes then take
// longer than the kernels at small sizes (one 32768-token row: 23 us of host time for 9 us of
// kernels; scores and gradient of 1000 x 10883 logits: 109 us for 35). These do the same allocations
// and make the same C calls without Python. Their arguments are the checked ones.
//
// Operators named native_* exist only with this library; warpstate::fp8_linear is defined in
// Python, with a Python kernel and autograd formula that these replace on CUDA. Autograd kernels read
// no data: they call operators below autograd, so that wrapped and fake tensors reach kernels of
// their own. None has a forward-mode derivative; tensors that carry a tangent are refused.
#include "host_common.h"

namespace {

constexpr int64_t kTransposeMinRows = 1024;  // fused_execution.TRANSPOSE_MIN_ROWS
constexpr int64_t kMaxTopK = 64, kMaxVocab = 524288;

// --- 8-bit operands -------------------------------------------------------------------------

Tensor scales(const Tensor& like, int64_t rows, int64_t n, bool e8m0) {
  return e8m0 ? bytes(like, {rows, up(n, 4)}) : floats(like, {n, up(rows, 4)});
}

FourTensors quantize(const Tensor& x, bool e8m0, int64_t form, bool transposed) {
  c10::DeviceGuard guard(x.device());
  const int64_t rows = x.size(0), cols = x.size(1);
  const bool block = form == WS_QUANT_BLOCKS;
  Tensor q, scale, qt, scale_t;
  if (form != WS_QUANT_COLUMNS) {
    q = bytes(x, {rows, up(cols, 16)});
    scale = scales(x, block ? blocks(rows) : rows, blocks(cols), e8m0);
  }
  if ((form & WS_QUANT_COLUMNS) || transposed) {
    qt = bytes(x, {cols, up(rows, 16)});
    scale_t = scales(x, block ? blocks(cols) : cols, blocks(rows), e8m0);
  }
  auto ld = [](const Tensor& t) { return t.defined() ? t.size(1) : 0; };
  check(ws_fp8_quantize(x.const_data_ptr(), row_stride(x), x.scalar_type() == at::kFloat, rows, cols, (int)form,
                        e8m0 ? WS_SCALE_E8M0 : WS_SCALE_F32, ptr(q), ld(q), ptr(scale), ld(scale), ptr(qt), ld(qt),
                        ptr(scale_t), ld(scale_t), stream_of(x)),
        "ws_fp8_quantize");
  return {q, scale, qt, scale_t};
}

void product(const Tensor& a, int64_t lda, const Tensor& sa, int64_t ld_sa, int64_t rows_a, const Tensor& b,
             int64_t ldb, const Tensor& sb, int64_t ld_sb, int64_t rows_b, bool e8m0, const Tensor& out, int64_t k) {
  c10::DeviceGuard guard(a.device());
  const int64_t m = out.size(0), n = out.size(1), wide = up(k, 16);
  const int type = e8m0 ? WS_SCALE_E8M0 : WS_SCALE_F32;
  const int64_t need = ws_fp8_mm_workspace_bytes(m, n, wide, (int)rows_b, type);
  Tensor work = need ? bytes(a, {need}) : Tensor();
  check(ws_fp8_mm(a.const_data_ptr(), lda, sa.const_data_ptr(), ld_sa, (int)rows_a, b.const_data_ptr(), ldb,
                  sb.const_data_ptr(), ld_sb, (int)rows_b, type, out.data_ptr(), row_stride(out), m, n, wide,
                  ptr(work), stream_of(a)),
        "ws_fp8_mm");
}

// --- quantize_rows and fp8_mm of ops/fp8_execution.py, with their checks -----------------------

std::tuple<Tensor, Tensor> native_quantize_rows(const Tensor& x_in, bool e8m0) {
  TORCH_CHECK_VALUE(x_in.scalar_type() == at::kBFloat16 || x_in.scalar_type() == at::kFloat,
                    "Quantization takes BF16 or FP32 matrices");
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.numel() > 0, "Quantization takes a non-empty matrix");
  const int64_t rows = x_in.size(0), cols = x_in.size(1);
  const bool unit = (x_in.stride(1) == 1 || cols == 1) && (rows == 1 || x_in.stride(0) >= cols);
  const Tensor x = unit ? x_in : x_in.contiguous();
  c10::DeviceGuard guard(x.device());
  Tensor q = at::empty({rows, up(cols, 16)}, x.options().dtype(at::kFloat8_e4m3fn));
  const int64_t n = blocks(cols);
  Tensor scale = e8m0 ? at::empty({rows, up(n, 4)}, x.options().dtype(at::kFloat8_e8m0fnu)) : floats(x, {n, up(rows, 4)});
  check(ws_fp8_quantize(x.const_data_ptr(), row_stride(x), x.scalar_type() == at::kFloat, rows, cols, WS_QUANT_ROWS,
                        e8m0 ? WS_SCALE_E8M0 : WS_SCALE_F32, q.data_ptr(), q.size(1), scale.data_ptr(),
                        scale.size(1), nullptr, 0, nullptr, 0, stream_of(x)),
        "ws_fp8_quantize");
  if (q.size(1) != cols) q = q.narrow(1, 0, cols);
  if (!e8m0) return {q, scale.narrow(1, 0, rows).t()};
  return {q, scale.size(1) == n ? scale : scale.narrow(1, 0, n)};
}

void check_operand(const Tensor& q, const char* name) {
  TORCH_CHECK_VALUE(q.is_cuda(), "8-bit kernels require CUDA tensors");
  TORCH_CHECK_VALUE(q.scalar_type() == at::kFloat8_e4m3fn && q.dim() == 2 && q.numel() > 0, name,
                    " must be a non-empty float8_e4m3fn matrix");
}

// An operand with rows of whole 16-byte pieces: itself, or a zero-padded copy.
Tensor packed(const Tensor& q_in) {
  const int64_t rows = q_in.size(0), k = q_in.size(1);
  if (q_in.stride(1) == 1 && k % 16 == 0 && reinterpret_cast<uintptr_t>(q_in.const_data_ptr()) % 16 == 0 &&
      (rows == 1 || (q_in.stride(0) % 16 == 0 && q_in.stride(0) >= k)))
    return q_in;
  Tensor q = q_in.view(at::kByte);
  if (std::min(q.stride(0), q.stride(1)) < 1) q = q.contiguous();  // an expanded matrix
  Tensor out = bytes(q, {rows, up(k, 16)});
  check(ws_fp8_pack(q.const_data_ptr(), q.stride(0), q.stride(1), out.data_ptr(), out.size(1), rows, k, stream_of(q)),
        "ws_fp8_pack");
  return out;
}

struct ScaleOperand {
  Tensor t;
  int64_t ld, rows;  // operand rows per scale row
};
// Scales in the layout the product reads: themselves, or a copy. `vector`: four rows' FP32
// scales are read at a time.
ScaleOperand scale_operand(const Tensor& scale, const Tensor& q, at::ScalarType type, bool vector, const char* name) {
  const int64_t rows = q.size(0), nb = blocks(q.size(1));
  TORCH_CHECK_VALUE(scale.scalar_type() == type && scale.device() == q.device() && scale.dim() == 2, name,
                    " must be a matrix of ", type == at::kFloat ? "float32" : "float8_e8m0fnu", " scales on ",
                    q.device());
  const int64_t n = scale.size(0);
  int64_t block_rows = 1;
  if (n != rows || scale.size(1) != nb) {
    block_rows = kBlock;
    TORCH_CHECK_VALUE(n == blocks(rows) && scale.size(1) == nb, name,
                      " must have one scale per row or per 128 rows and one per 128 columns, [", rows, ", ", nb,
                      "] or [", blocks(rows), ", ", nb, "], not ", scale.sizes());
  }
  const int64_t s0 = scale.stride(0), s1 = scale.stride(1);
  const int64_t size = (int64_t)scale.storage().nbytes(), first = scale.storage_offset();
  const uintptr_t at = reinterpret_cast<uintptr_t>(scale.const_data_ptr());
  if (type != at::kFloat) {
    // The kernel reads whole dwords of a row.
    const int64_t ld = n > 1 ? s0 : up(nb, 4);
    if ((s1 == 1 || nb == 1) && ld % 4 == 0 && ld >= nb && at % 4 == 0 && first + (n - 1) * ld + up(nb, 4) <= size)
      return {scale, ld, block_rows};
    Tensor copy = bytes(scale, {n, up(nb, 4)});
    copy.narrow(1, 0, nb).copy_(scale.view(at::kByte));
    return {copy, copy.size(1), block_rows};
  }
  const int64_t ld = nb > 1 ? s1 : up(n, 4);
  if ((s0 == 1 || n == 1) && ld >= n &&
      (!vector || (ld % 4 == 0 && at % 16 == 0 && 4 * (first + (nb - 1) * ld + up(n, 4)) <= size)))
    return {scale, ld, block_rows};
  Tensor copy = floats(scale, {nb, up(n, 4)});
  copy.narrow(1, 0, n).copy_(scale.t());
  return {copy, copy.size(1), block_rows};
}

Tensor native_fp8_mm(const Tensor& a, const Tensor& a_scale, const Tensor& b, const Tensor& b_scale) {
  check_operand(a, "a");
  check_operand(b, "b");
  const int64_t m = a.size(0), k = a.size(1), n = b.size(0);
  TORCH_CHECK_VALUE(b.size(1) == k && a.device() == b.device(), "Expected a [M, K] and b [N, K] on one device, got ",
                    a.sizes(), " and ", b.sizes());
  const at::ScalarType type = a_scale.scalar_type();
  TORCH_CHECK_VALUE(type == at::kFloat || type == at::kFloat8_e8m0fnu,
                    "Scales are torch.float8_e8m0fnu or torch.float32");
  c10::DeviceGuard guard(a.device());
  const ScaleOperand sa = scale_operand(a_scale, a, type, false, "a_scale");
  const ScaleOperand sb = scale_operand(b_scale, b, type, b_scale.dim() == 2 && b_scale.size(0) == n, "b_scale");
  const Tensor pa = packed(a), pb = packed(b);
  const int64_t wide = up(k, 16);
  Tensor out = at::empty({m, n}, a.options().dtype(at::kBFloat16));
  product(pa, m > 1 ? pa.stride(0) : wide, sa.t, sa.ld, sa.rows, pb, n > 1 ? pb.stride(0) : wide, sb.t, sb.ld,
          sb.rows, type != at::kFloat, out, k);
  return out;
}

// On whole buffers of quantize().
void product_of(const Tensor& a, const Tensor& sa, int64_t rows_a, const Tensor& b, const Tensor& sb,
                int64_t rows_b, bool e8m0, const Tensor& out, int64_t k) {
  product(a, a.size(1), sa, sa.size(1), rows_a, b, b.size(1), sb, sb.size(1), rows_b, e8m0, out, k);
}

FiveTensors linear_forward(const Tensor& x, const Tensor& weight, bool e8m0, bool keep_x, bool keep_w) {
  auto [w, w_scale, wt, wt_scale] = quantize(weight, e8m0, WS_QUANT_BLOCKS, keep_w);
  auto [q, scale, qt, qt_scale] = quantize(x, e8m0, keep_x ? WS_QUANT_ROWS | WS_QUANT_COLUMNS : WS_QUANT_ROWS, false);
  Tensor y = at::empty({x.size(0), weight.size(0)}, x.options());
  product_of(q, scale, 1, w, w_scale, kBlock, e8m0, y, x.size(1));
  auto kept = [&](Tensor& t) { return t.defined() ? t : bytes(x, {0, 0}); };
  return {y, kept(qt), kept(qt_scale), kept(wt), kept(wt_scale)};
}

std::tuple<Tensor, Tensor> linear_backward(const Tensor& grad_in, const Tensor& x, const Tensor& qt,
                                           const Tensor& qt_scale, const Tensor& wt, const Tensor& wt_scale,
                                           int64_t k, bool e8m0, bool want_x, bool want_w, bool master) {
  const Tensor grad = grad_in.contiguous();
  const int64_t m = grad.size(0), n = grad.size(1);
  const int64_t form = (want_x ? WS_QUANT_ROWS : 0) | (want_w && !master ? WS_QUANT_COLUMNS : 0);
  Tensor g, g_scale, gt, gt_scale;
  if (form) std::tie(g, g_scale, gt, gt_scale) = quantize(grad, e8m0, form, false);
  Tensor dx = want_x ? at::empty({m, k}, grad.options()) : at::empty({0}, grad.options());
  if (want_x) product_of(g, g_scale, 1, wt, wt_scale, kBlock, e8m0, dx, n);
  const auto dw_options = grad.options().dtype(master ? at::kFloat : at::kBFloat16);
  if (!want_w) return {dx, at::empty({0}, dw_options)};
  Tensor dw = at::empty({n, k}, dw_options);
  if (master) {
    // fused_execution.mm_f32_group of grad^T and x, FP32 sums unrounded.
    c10::DeviceGuard guard(grad.device());
    const ws_accumulate_problem item{grad.const_data_ptr(), 1, n, x.const_data_ptr(), x.stride(0), x.stride(1),
                                     dw.data_ptr<float>(), k, n, k};
    const int64_t need = ws_mm_accumulate_group_workspace_floats(&item, 1, m);
    Tensor work = need ? floats(grad, {need}) : Tensor();
    check(ws_mm_store_f32_group(&item, 1, m, 0, need ? work.data_ptr<float>() : nullptr, stream_of(grad)),
          "ws_mm_store_f32_group");
  } else {
    product_of(gt, gt_scale, 1, qt, qt_scale, 1, e8m0, dw, m);
  }
  return {dx, dw};
}

struct Fp8LinearFn : Function<Fp8LinearFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, bool e8m0, bool keep_x,
                               bool keep_w) {
    static const auto op = find<FiveTensors(const Tensor&, const Tensor&, bool, bool, bool)>("warpstate::fp8_linear");
    ctx->set_materialize_grads(false);
    auto [y, qt, qt_scale, wt, wt_scale] = below(op, x, weight, e8m0, keep_x, keep_w);
    const bool master = weight.scalar_type() == at::kFloat;
    // x itself only where its weight gradient reads it.
    ctx->save_for_backward({master && weight.requires_grad() ? x : qt, qt, qt_scale, wt, wt_scale});
    ctx->saved_data["k"] = x.sym_size(1);
    ctx->saved_data["e8m0"] = e8m0;
    ctx->saved_data["want_x"] = x.requires_grad();
    ctx->saved_data["want_w"] = weight.requires_grad();
    ctx->saved_data["master"] = master;
    return {y, qt, qt_scale, wt, wt_scale};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    typedef const Tensor& T;
    static const auto op =
        c10::Dispatcher::singleton()
            .findSchemaOrThrow("warpstate::fp8_linear_backward", "")
            .typed<std::tuple<Tensor, Tensor>(T, T, T, T, T, T, c10::SymInt, bool, bool, bool, bool)>();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const auto s = ctx->get_saved_variables();
    const bool want_x = ctx->saved_data["want_x"].toBool(), want_w = ctx->saved_data["want_w"].toBool();
    auto call = [&] {
      return op.call(grads[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["k"].toSymInt(),
                     ctx->saved_data["e8m0"].toBool(), want_x, want_w, ctx->saved_data["master"].toBool());
    };
    std::tuple<Tensor, Tensor> d;
    if (at::GradMode::is_enabled()) {  // the operator's own autograd kernel refuses a second derivative
      d = call();
    } else {
      at::AutoDispatchBelowAutograd guard;
      d = call();
    }
    return {want_x ? std::get<0>(d) : Tensor(), want_w ? std::get<1>(d) : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
FiveTensors linear(const Tensor& x, const Tensor& weight, bool e8m0, bool keep_x, bool keep_w) {
  refuse_tangents("fp8_linear", x, weight);
  if (!records(x, weight)) {
    static const auto op = find<FiveTensors(const Tensor&, const Tensor&, bool, bool, bool)>("warpstate::fp8_linear");
    return below(op, x, weight, e8m0, keep_x, keep_w);
  }
  variable_list v = Fp8LinearFn::apply(x, weight, e8m0, keep_x, keep_w);
  return {v[0], v[1], v[2], v[3], v[4]};
}

// --- token scores ---------------------------------------------------------------------------

// (logprob, entropy, top logprobs, top ids, lse). lse is undefined unless it is kept: small calls
// are bound by the host, so it shares the workspace's allocation instead.
FiveTensors scores_forward(const Tensor& logits, const Tensor& tokens, int64_t top_k, double inv_t, bool keep_lse) {
  c10::DeviceGuard guard(logits.device());
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  Tensor logprob = floats(logits, {rows}), entropy = floats(logits, {rows}), lse;
  if (keep_lse) lse = floats(logits, {rows});
  Tensor top = floats(logits, {rows, top_k});
  Tensor ids = at::empty({rows, top_k}, logits.options().dtype(at::kLong));
  if (rows) {
    const int64_t need = ws_token_scores_workspace_bytes(rows, vocab, top_k), head = keep_lse ? 0 : up(4 * rows, 16);
    Tensor work = need + head ? bytes(logits, {need + head}) : Tensor();
    void* first = ptr(work);
    check(ws_token_scores(logits.const_data_ptr(), row_stride(logits), logits.scalar_type() == at::kFloat,
                          tokens.const_data_ptr<int64_t>(), rows, vocab, (float)inv_t, top_k,
                          need ? static_cast<char*>(first) + head : nullptr,
                          keep_lse ? lse.data_ptr<float>() : static_cast<float*>(first), logprob.data_ptr<float>(),
                          entropy.data_ptr<float>(), top.data_ptr<float>(), ids.data_ptr<int64_t>(),
                          stream_of(logits)),
          "ws_token_scores");
  }
  return {logprob, entropy, top, ids, lse};
}

// An upstream gradient as the kernels read it.
Tensor upstream(const std::optional<Tensor>& g) {
  return g.has_value() && g->defined() ? g->to(at::kFloat).contiguous() : Tensor();
}
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }
const float* float_ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr<float>() : nullptr; }

Tensor scores_backward(const Tensor& logits, const Tensor& tokens, const Tensor& lse, const Tensor& entropy,
                       const std::optional<Tensor>& dlogprob, const std::optional<Tensor>& dentropy, double inv_t) {
  c10::DeviceGuard guard(logits.device());
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  Tensor out = at::empty({rows, vocab}, logits.options());
  if (rows) {
    const Tensor g = upstream(dlogprob), h = upstream(dentropy);
    check(ws_token_scores_backward(logits.const_data_ptr(), row_stride(logits), logits.scalar_type() == at::kFloat,
                                   tokens.const_data_ptr<int64_t>(), rows, vocab, (float)inv_t, float_ptr(lse),
                                   float_ptr(entropy), float_ptr(g), float_ptr(h), out.data_ptr(), vocab,
                                   stream_of(logits)),
          "ws_token_scores_backward");
  }
  return out;
}

// A backward operator: below autograd, unless its own gradient is being recorded (create_graph, a
// functorch transform): then its autograd kernel records a node that refuses to be differentiated.
template <class Op, class... Args>
auto backward_op(const Op& op, Args&&... args) {
  if (at::GradMode::is_enabled()) return op.call(std::forward<Args>(args)...);
  return below(op, std::forward<Args>(args)...);
}
variable_list refuse_second() { TORCH_CHECK(false, "token scores cannot be differentiated twice"); }
bool needs_grad(const std::optional<Tensor>& t) { return t.has_value() && t->defined() && t->requires_grad(); }

typedef Tensor ScoresBackward(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const std::optional<Tensor>&,
                              const std::optional<Tensor>&, double);
const auto& scores_backward_op() {
  static const auto op = find<ScoresBackward>("warpstate::native_token_scores_backward");
  return op;
}
struct ScoresBackwardFn : Function<ScoresBackwardFn> {
  static Tensor forward(AutogradContext*, const Tensor& logits, const Tensor& tokens, const Tensor& lse,
                        const Tensor& entropy, const std::optional<Tensor>& dlogprob,
                        const std::optional<Tensor>& dentropy, double inv_t) {
    return below(scores_backward_op(), logits, tokens, lse, entropy, dlogprob, dentropy, inv_t);
  }
  static variable_list backward(AutogradContext*, variable_list) { return refuse_second(); }
};
Tensor scores_backward_autograd(const Tensor& logits, const Tensor& tokens, const Tensor& lse, const Tensor& entropy,
                                const std::optional<Tensor>& dlogprob, const std::optional<Tensor>& dentropy,
                                double inv_t) {
  if (records(logits, lse, entropy) || (at::GradMode::is_enabled() && (needs_grad(dlogprob) || needs_grad(dentropy))))
    return ScoresBackwardFn::apply(logits, tokens, lse, entropy, dlogprob, dentropy, inv_t);
  return below(scores_backward_op(), logits, tokens, lse, entropy, dlogprob, dentropy, inv_t);
}

struct TokenScoresFn : Function<TokenScoresFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, int64_t top_k,
                               double inv_t) {
    static const auto op =
        find<FiveTensors(const Tensor&, const Tensor&, int64_t, double)>("warpstate::native_token_scores_lse");
    auto [logprob, entropy, top, ids, lse] = below(op, logits, tokens, top_k, inv_t);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, lse, entropy});
    ctx->saved_data["inv_t"] = inv_t;
    ctx->mark_non_differentiable({top, ids});
    return {logprob, entropy, top, ids};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list d(4);
    if (!grads[0].defined() && !grads[1].defined()) return d;
    const auto s = ctx->get_saved_variables();
    d[0] = backward_op(scores_backward_op(), s[0], s[1], s[2], s[3], maybe(grads[0]), maybe(grads[1]),
                       ctx->saved_data["inv_t"].toDouble());
    return d;
  }
};

// A normal FP32 number, and finite times log2 e.
double inverse(double temperature) {
  const double inv_t = 1.0 / temperature;
  TORCH_CHECK_VALUE(inv_t >= 0x1p-126 && inv_t <= 2.3e38,
                    "The temperature must lie between 4.4e-39 and 8.5e37, not ", temperature);
  return inv_t;
}
Tensor checked_tokens(const Tensor& tokens, const Tensor& like) {
  TORCH_CHECK_VALUE(tokens.scalar_type() == at::kLong && tokens.dim() == 1 && tokens.size(0) == like.size(0) &&
                        tokens.device() == like.device(),
                    "Tokens must be an int64 vector, one per row, on the operands' device");
  return tokens.contiguous();
}

// token_scores of ops/token_scores.py, with its checks.
struct CheckedScores {
  Tensor logits, tokens;
  double inv_t;
};
CheckedScores check_scores(const Tensor& logits, const Tensor& tokens, int64_t top_k, double temperature) {
  TORCH_CHECK_VALUE((logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat) &&
                        logits.dim() == 2,
                    "Expected BF16 or FP32 logits [rows, vocab]");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  TORCH_CHECK_VALUE(vocab >= 1 && vocab <= kMaxVocab, "Token scores take 1 to ", kMaxVocab, " logits a row, not ", vocab);
  const int64_t most = std::min(kMaxTopK, vocab);
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= most, "top_k must lie in [0, ", most, "], not ", top_k);
  const bool unit = (logits.stride(1) == 1 || vocab == 1) && (rows <= 1 || logits.stride(0) >= vocab);
  return {unit ? logits : logits.contiguous(), checked_tokens(tokens, logits), inverse(temperature)};
}
FourTensors native_token_scores(const Tensor& logits, const Tensor& tokens, int64_t top_k, double temperature) {
  const auto c = check_scores(logits, tokens, top_k, temperature);
  auto [logprob, entropy, top, ids, lse] = scores_forward(c.logits, c.tokens, top_k, c.inv_t, false);
  return {logprob, entropy, top, ids};
}
FiveTensors scores_with_lse(const Tensor& logits, const Tensor& tokens, int64_t top_k, double inv_t) {
  return scores_forward(logits, tokens, top_k, inv_t, true);
}
FourTensors token_scores_autograd(const Tensor& logits, const Tensor& tokens, int64_t top_k, double temperature) {
  refuse_tangents("token_scores", logits);
  if (!records(logits)) {
    static const auto op =
        find<FourTensors(const Tensor&, const Tensor&, int64_t, double)>("warpstate::native_token_scores");
    return below(op, logits, tokens, top_k, temperature);
  }
  const auto c = check_scores(logits, tokens, top_k, temperature);
  variable_list v = TokenScoresFn::apply(c.logits, c.tokens, top_k, c.inv_t);
  return {v[0], v[1], v[2], v[3]};
}

// hidden and weight as the kernels read them (BF16, 16-byte rows, equal padded widths).
std::tuple<Tensor, Tensor, Tensor> head_forward(const Tensor& h, const Tensor& w, const Tensor& tokens, double inv_t) {
  c10::DeviceGuard guard(h.device());
  const int64_t rows = h.size(0), d = h.size(1), vocab = w.size(0);
  Tensor logprob = floats(h, {rows}), entropy = floats(h, {rows}), lse = floats(h, {rows});
  if (rows) {
    Tensor work = floats(h, {ws_linear_token_scores_workspace_floats(rows, vocab, d)});
    check(ws_linear_token_scores(h.const_data_ptr(), row_stride(h), w.const_data_ptr(), row_stride(w),
                                 tokens.const_data_ptr<int64_t>(), rows, vocab, d, (float)inv_t,
                                 work.data_ptr<float>(), lse.data_ptr<float>(), logprob.data_ptr<float>(),
                                 entropy.data_ptr<float>(), stream_of(h)),
          "ws_linear_token_scores");
  }
  return {logprob, entropy, lse};
}

// (dHidden, dWeight), each empty unless wanted, in the operands' padded width; dWeight in BF16 (of
// one chunk) or FP32.
std::tuple<Tensor, Tensor> head_backward(const Tensor& h, const Tensor& w, const Tensor& tokens, const Tensor& lse,
                                         const Tensor& entropy, const std::optional<Tensor>& dlogprob,
                                         const std::optional<Tensor>& dentropy, double inv_t, int64_t chunk_rows,
                                         bool want_h, bool want_w, bool bf16) {
  c10::DeviceGuard guard(h.device());
  const int64_t rows = h.size(0), width = h.size(1), vocab = w.size(0);
  Tensor dh = at::empty({want_h ? rows : 0, width}, h.options());
  Tensor dw = at::empty({want_w ? vocab : 0, width}, h.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  if (rows) {
    const Tensor g = upstream(dlogprob), e = upstream(dentropy);
    Tensor work = bytes(h, {ws_linear_token_scores_backward_workspace_bytes(rows, vocab, width, chunk_rows)});
    // The dHidden product reads the head weight along the vocabulary.
    Tensor wt;
    if (want_h && rows >= kTransposeMinRows && vocab % 8 == 0) {
      wt = at::empty({width, vocab}, w.options());
      check(ws_transpose_bf16(w.const_data_ptr(), row_stride(w), wt.data_ptr(), vocab, width, stream_of(w)),
            "ws_transpose_bf16");
    }
    check(ws_linear_token_scores_backward(h.const_data_ptr(), row_stride(h), w.const_data_ptr(), row_stride(w),
                                          ptr(wt), tokens.const_data_ptr<int64_t>(), float_ptr(lse),
                                          float_ptr(entropy), float_ptr(g), float_ptr(e), rows, vocab, width,
                                          (float)inv_t, work.data_ptr(), chunk_rows, ptr(dh), width, ptr(dw), width,
                                          bf16, stream_of(h)),
          "ws_linear_token_scores_backward");
  } else if (want_w) {
    dw.zero_();
  }
  return {dh, dw};
}

typedef std::tuple<Tensor, Tensor> HeadBackward(const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                                const Tensor&, const std::optional<Tensor>&,
                                                const std::optional<Tensor>&, double, int64_t, bool, bool, bool);
const auto& head_backward_op() {
  static const auto op = find<HeadBackward>("warpstate::native_head_scores_backward");
  return op;
}
struct HeadBackwardFn : Function<HeadBackwardFn> {
  static variable_list forward(AutogradContext*, const Tensor& h, const Tensor& w, const Tensor& tokens,
                               const Tensor& lse, const Tensor& entropy, const std::optional<Tensor>& dlogprob,
                               const std::optional<Tensor>& dentropy, double inv_t, int64_t chunk_rows, bool want_h,
                               bool want_w, bool bf16) {
    auto [dh, dw] = below(head_backward_op(), h, w, tokens, lse, entropy, dlogprob, dentropy, inv_t, chunk_rows,
                          want_h, want_w, bf16);
    return {dh, dw};
  }
  static variable_list backward(AutogradContext*, variable_list) { return refuse_second(); }
};
std::tuple<Tensor, Tensor> head_backward_autograd(const Tensor& h, const Tensor& w, const Tensor& tokens,
                                                  const Tensor& lse, const Tensor& entropy,
                                                  const std::optional<Tensor>& dlogprob,
                                                  const std::optional<Tensor>& dentropy, double inv_t,
                                                  int64_t chunk_rows, bool want_h, bool want_w, bool bf16) {
  if (records(h, w, lse, entropy) || (at::GradMode::is_enabled() && (needs_grad(dlogprob) || needs_grad(dentropy)))) {
    variable_list v = HeadBackwardFn::apply(h, w, tokens, lse, entropy, dlogprob, dentropy, inv_t, chunk_rows, want_h,
                                            want_w, bf16);
    return {v[0], v[1]};
  }
  return below(head_backward_op(), h, w, tokens, lse, entropy, dlogprob, dentropy, inv_t, chunk_rows, want_h, want_w,
               bf16);
}

struct HeadScoresFn : Function<HeadScoresFn> {
  // Gradients go to the tensors that h and w were made from.
  static variable_list forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& h,
                               const Tensor& w, const Tensor& tokens, double inv_t, int64_t chunk_rows) {
    typedef const Tensor& T;
    static const auto op =
        find<std::tuple<Tensor, Tensor, Tensor>(T, T, T, double)>("warpstate::native_head_scores_lse");
    auto [logprob, entropy, lse] = below(op, h, w, tokens, inv_t);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({h, w, tokens, lse, entropy});
    ctx->saved_data["inv_t"] = inv_t;
    ctx->saved_data["chunk_rows"] = chunk_rows;
    ctx->saved_data["want_h"] = hidden.requires_grad();
    ctx->saved_data["want_w"] = weight.requires_grad();
    ctx->saved_data["width"] = hidden.size(1);
    ctx->saved_data["hidden_type"] = hidden.scalar_type();
    ctx->saved_data["weight_type"] = weight.scalar_type();
    return {logprob, entropy};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list d(7);
    if (!grads[0].defined() && !grads[1].defined()) return d;
    const auto s = ctx->get_saved_variables();
    const bool want_h = ctx->saved_data["want_h"].toBool(), want_w = ctx->saved_data["want_w"].toBool();
    const int64_t rows = s[0].size(0), vocab = s[1].size(0), chunk = ctx->saved_data["chunk_rows"].toInt();
    const auto weight_type = ctx->saved_data["weight_type"].toScalarType();
    // A BF16 weight's gradient is rounded as it is written where one chunk makes all of it.
    const bool bf16 = weight_type == at::kBFloat16 && rows <= chunk && vocab % 8 == 0;
    auto [dh, dw] = backward_op(head_backward_op(), s[0], s[1], s[2], s[3], s[4], maybe(grads[0]), maybe(grads[1]),
                                ctx->saved_data["inv_t"].toDouble(), chunk, want_h, want_w, bf16);
    const int64_t cols = ctx->saved_data["width"].toInt();
    if (want_h) d[0] = dh.narrow(1, 0, cols).to(ctx->saved_data["hidden_type"].toScalarType());
    if (want_w) d[1] = dw.narrow(1, 0, cols).to(weight_type);
    return d;
  }
};
std::tuple<Tensor, Tensor> native_head_scores(const Tensor& hidden, const Tensor& weight, const Tensor& h,
                                              const Tensor& w, const Tensor& tokens, double inv_t,
                                              int64_t chunk_rows) {
  auto [logprob, entropy, lse] = head_forward(h, w, tokens, inv_t);
  return {logprob, entropy};
}
std::tuple<Tensor, Tensor> head_scores_autograd(const Tensor& hidden, const Tensor& weight, const Tensor& h,
                                                const Tensor& w, const Tensor& tokens, double inv_t,
                                                int64_t chunk_rows) {
  refuse_tangents("linear_token_scores", hidden, weight);
  if (!records(hidden, weight)) {
    typedef const Tensor& T;
    static const auto op =
        find<std::tuple<Tensor, Tensor>(T, T, T, T, T, double, int64_t)>("warpstate::native_head_scores");
    return below(op, hidden, weight, h, w, tokens, inv_t, chunk_rows);
  }
  variable_list v = HeadScoresFn::apply(hidden, weight, h, w, tokens, inv_t, chunk_rows);
  return {v[0], v[1]};
}

// Shapes and types only: the logits' operators on fake tensors.
FourTensors scores_meta(const Tensor& logits, const Tensor& tokens, int64_t top_k, double temperature) {
  check_scores(logits, tokens, top_k, temperature);
  const int64_t rows = logits.size(0);
  return {floats(logits, {rows}), floats(logits, {rows}), floats(logits, {rows, top_k}),
          at::empty({rows, top_k}, logits.options().dtype(at::kLong))};
}
FiveTensors scores_with_lse_meta(const Tensor& logits, const Tensor&, int64_t top_k, double) {
  const int64_t rows = logits.size(0);
  return {floats(logits, {rows}), floats(logits, {rows}), floats(logits, {rows, top_k}),
          at::empty({rows, top_k}, logits.options().dtype(at::kLong)), floats(logits, {rows})};
}
Tensor scores_backward_meta(const Tensor& logits, const Tensor&, const Tensor&, const Tensor&,
                            const std::optional<Tensor>&, const std::optional<Tensor>&, double) {
  return at::empty({logits.size(0), logits.size(1)}, logits.options());
}

// Undefined tensors cannot leave an operator: empty ones in the place of forms not wanted.
FourTensors native_quantize(const Tensor& x, bool e8m0, int64_t form, bool transposed) {
  auto [q, scale, qt, scale_t] = quantize(x, e8m0, form, transposed);
  auto known = [&](Tensor& t) { return t.defined() ? t : bytes(x, {0, 0}); };
  return {known(q), known(scale), known(qt), known(scale_t)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(warpstate, m) {
  m.def("native_quantize(Tensor x, bool e8m0, int form, bool transposed) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("native_quantize_rows(Tensor x, bool e8m0) -> (Tensor, Tensor)");
  m.def("native_fp8_mm(Tensor a, Tensor a_scale, Tensor b, Tensor b_scale) -> Tensor");
  m.def(
      "native_token_scores(Tensor logits, Tensor tokens, int top_k, float temperature) -> (Tensor, Tensor, "
      "Tensor, Tensor)");
  m.def(
      "native_token_scores_lse(Tensor logits, Tensor tokens, int top_k, float inv_t) -> (Tensor, Tensor, Tensor, "
      "Tensor, Tensor)");
  m.def(
      "native_token_scores_backward(Tensor logits, Tensor tokens, Tensor lse, Tensor entropy, Tensor? dlogprob, "
      "Tensor? dentropy, float inv_t) -> Tensor");
  m.def("native_head_scores_lse(Tensor h, Tensor w, Tensor tokens, float inv_t) -> (Tensor, Tensor, Tensor)");
  m.def(
      "native_head_scores_backward(Tensor h, Tensor w, Tensor tokens, Tensor lse, Tensor entropy, Tensor? dlogprob, "
      "Tensor? dentropy, float inv_t, int chunk_rows, bool want_h, bool want_w, bool bf16) -> (Tensor, Tensor)");
  m.def(
      "native_head_scores(Tensor hidden, Tensor weight, Tensor h, Tensor w, Tensor tokens, float inv_t, "
      "int chunk_rows) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(warpstate, CUDA, m) {
  m.impl("native_quantize", &native_quantize);
  m.impl("native_quantize_rows", &native_quantize_rows);
  m.impl("native_fp8_mm", &native_fp8_mm);
  m.impl("native_token_scores", &native_token_scores);
  m.impl("native_token_scores_lse", &scores_with_lse);
  m.impl("native_token_scores_backward", &scores_backward);
  m.impl("native_head_scores", &native_head_scores);
  m.impl("native_head_scores_lse", &head_forward);
  m.impl("native_head_scores_backward", &head_backward);
  m.impl("fp8_linear", &linear_forward);
  m.impl("fp8_linear_backward", &linear_backward);
}
TORCH_LIBRARY_IMPL(warpstate, AutogradCUDA, m) {
  m.impl("native_token_scores", &token_scores_autograd);
  m.impl("native_token_scores_backward", &scores_backward_autograd);
  m.impl("native_head_scores", &head_scores_autograd);
  m.impl("native_head_scores_backward", &head_backward_autograd);
  m.impl("fp8_linear", &linear);
}
TORCH_LIBRARY_IMPL(warpstate, Meta, m) {
  m.impl("native_token_scores", &scores_meta);
  m.impl("native_token_scores_lse", &scores_with_lse_meta);
  m.impl("native_token_scores_backward", &scores_backward_meta);
}
