// kaldi-decoder_amd/python/csrc/frames.cc -- torch binding of the operators over rows of logits
// (include/kd_hip.h, kd_token_scores and kd_distill_loss), with their autograd nodes; behind
// kaldi_decoder/frames.py.
//
// Host C++ only.  The smallest of these calls take the GPU 4 us, so what a call does on the host is
// what it costs: checks, three to five allocations and one C call are 4 to 6.5 us here (torch.neg of the
// same row: 4.2), and 15 through ctypes.  With a gradient through autograd 29 or 48 us, from process to
// process, most of it torch's engine (a product of two tensors and its gradient: 27 or 45), and 120.

#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include <optional>
#include <string>
#include <vector>

#include "kd_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int DtypeCode(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KD_DTYPE_F32;
    case at::kHalf: return KD_DTYPE_F16;
    case at::kBFloat16: return KD_DTYPE_BF16;
    default: return -1;
  }
}
int IdBytes(const Tensor &t) {
  return t.scalar_type() == at::kInt ? 4 : t.scalar_type() == at::kLong ? 8 : 0;
}

void Check(int rc) {
  if (rc != KD_OK) throw std::runtime_error(kd_last_error());
}

void *Stream(const Tensor &t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

// (straight from the allocator: through the dispatcher each costs 0.3 us more, of calls of 5 us)
Tensor Empty(at::IntArrayRef sizes, at::ScalarType type, const Tensor &like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

template <class T>
T *Ptr(const OptTensor &t) {
  return t && t->defined() ? static_cast<T *>(t->data_ptr()) : nullptr;
}

// A tangent of forward-mode differentiation would be dropped without a word, a derivative of 0.
void NoTangent(const Tensor &t, const char *what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "kaldi_decoder.frames has no forward-mode derivatives, and ",
                              what, " carries a tangent: detach it");
}

// Rows of logits [N, V] or [B, T, V] as the C entries take them.
struct Rows {
  kd_frame_rows r{};
  std::vector<int64_t> lead;  // the shape without V
  OptTensor lengths;          // (kept alive until the launch)

  Rows(const Tensor &x, const OptTensor &len) {
    NoTangent(x, "the tensor of logits");
    const int dtype = DtypeCode(x);
    TORCH_CHECK_VALUE(x.is_cuda() && dtype >= 0, "logits must be a float32, float16 or bfloat16 CUDA tensor");
    const int64_t dims = x.dim();
    TORCH_CHECK_VALUE(dims == 2 || dims == 3, "logits must be [N, V] or [B, T, V]");
    const int64_t vocab = x.size(-1);
    TORCH_CHECK_VALUE(vocab >= 1 && vocab <= (int64_t(1) << 24), "logits: V must be between 1 and 2^24");
    TORCH_CHECK_VALUE(x.stride(-1) == 1 || vocab == 1, "logits need unit stride over the last (V) dimension");
    TORCH_CHECK_VALUE(!len || !len->defined() || dims == 3, "lengths need logits [B, T, V]");
    lead.assign(x.sizes().begin(), x.sizes().end() - 1);
    r.logits = x.data_ptr();
    r.vocab = vocab;
    r.batch = dims == 3 ? x.size(0) : 1;
    r.steps = x.size(-2);
    r.batch_stride = dims == 3 ? x.stride(0) : 0;
    r.row_stride = x.stride(-2);
    r.dtype = dtype;
    r.device = x.device().index();
    if (len && len->defined()) {
      lengths = Lengths(*len, x);
      r.lengths = lengths->data_ptr<int32_t>();
    }
  }

  static Tensor Lengths(const Tensor &len, const Tensor &x) {
    TORCH_CHECK_VALUE(len.dim() == 1 && x.dim() == 3 && len.size(0) == x.size(0) && IdBytes(len),
                      "lengths must be int32 or int64 [B]");
    return len.to(x.device(), at::kInt).contiguous();
  }
};

// A tensor with a row's values for each row, contiguous; `tail`: how many a row (0: one, no axis of its own).
Tensor PerRow(const Tensor &t, const Rows &rows, int64_t tail, const Tensor &x, bool type_ok, const char *what,
              const char *types) {
  TORCH_CHECK_VALUE(t.defined() && type_ok && t.device() == x.device(), what, " must be a tensor of ", types, " on ",
                    x.device());
  NoTangent(t, what);
  const int64_t n = static_cast<int64_t>(rows.lead.size());
  bool same = t.dim() == n + (tail ? 1 : 0) && (!tail || t.size(n) == tail);
  for (int64_t i = 0; same && i < n; ++i) same = t.size(i) == rows.lead[i];
  TORCH_CHECK_VALUE(same, what, " must have one value a row (", tail ? "and slot, " : "", "shape ",
                    c10::IntArrayRef(rows.lead), tail ? " and the slots" : "", "), not shape ", t.sizes());
  return t.contiguous();
}
Tensor Floats(const Tensor &t, const Rows &rows, int64_t tail, const Tensor &x, const char *what) {
  return PerRow(t, rows, tail, x, t.defined() && t.scalar_type() == at::kFloat, what, "float32");
}
Tensor Ids(const Tensor &t, const Rows &rows, int64_t tail, const Tensor &x, const char *what) {
  return PerRow(t, rows, tail, x, t.defined() && IdBytes(t), what, "int32 or int64");
}

// The gradient's tensor: `out`, or a new one.
Tensor GradOut(const OptTensor &out, const Tensor &x) {
  if (!out || !out->defined()) return Empty(x.sizes(), x.scalar_type(), x);
  TORCH_CHECK_VALUE(out->sizes() == x.sizes() && out->scalar_type() == x.scalar_type() && out->device() == x.device(),
                    "out must have the logits' shape, dtype and device");
  NoTangent(*out, "out");
  TORCH_CHECK(!out->is_inference() || c10::InferenceMode::is_enabled(),
              "out is an inference tensor: it can be written in inference mode alone");
  TORCH_CHECK_VALUE(out->stride(-1) == 1 || out->size(-1) == 1, "out needs unit stride over the last (V) dimension");
  return *out;
}
// (written in place: a graph that saved it must notice)
void Written(const OptTensor &out) {
  if (out && out->defined()) out->unsafeGetTensorImpl()->bump_version();
}

// [B, T] rows that follow each other evenly in every tensor concerned are handed over as one run: no
// division by T in the kernels.
void Join(kd_frame_rows &r, int64_t *grad_batch_stride, int64_t grad_row_stride) {
  if (r.batch == 1 || r.lengths || r.batch_stride != r.steps * r.row_stride) return;
  if (grad_batch_stride && *grad_batch_stride != r.steps * grad_row_stride) return;
  r.steps *= r.batch;
  r.batch = 1;
}

Tensor Workspace(size_t bytes, const Tensor &like) {
  return bytes ? Empty({static_cast<int64_t>(bytes)}, at::kByte, like) : Tensor();
}

// ---- scores ----------------------------------------------------------------------------------

struct Scores {
  Tensor logp, entropy, top_logp, top_ids, stats;  // (undefined: not asked for)
};

Scores TokenScores(const Tensor &x, const OptTensor &tokens, int64_t top, const OptTensor &lengths) {
  Rows rows(x, lengths);
  TORCH_CHECK_VALUE(top >= 0 && top <= 64, "top must be between 0 and 64");
  Scores s;
  Tensor tok;
  if (tokens) {
    tok = Ids(*tokens, rows, 0, x, "tokens");
    s.logp = Empty(rows.lead, at::kFloat, x);
  }
  s.entropy = Empty(rows.lead, at::kFloat, x);
  std::vector<int64_t> wide(rows.lead);
  wide.push_back(2);
  s.stats = Empty(wide, at::kFloat, x);
  if (top) {
    wide.back() = top;
    s.top_logp = Empty(wide, at::kFloat, x);
    s.top_ids = Empty(wide, at::kInt, x);
  }
  Join(rows.r, nullptr, 0);
  const size_t bytes = kd_token_scores_workspace(&rows.r, static_cast<int32_t>(top));
  const Tensor ws = Workspace(bytes, x);
  Check(kd_token_scores(&rows.r, Ptr<void>(tok), tokens ? IdBytes(tok) : 0, static_cast<int32_t>(top),
                        Ptr<float>(s.logp), Ptr<float>(s.entropy), Ptr<float>(s.stats), Ptr<float>(s.top_logp),
                        Ptr<int32_t>(s.top_ids), Ptr<void>(ws), bytes, Stream(x)));
  return s;
}

Tensor TokenScoresGrad(const Tensor &x, const OptTensor &tokens, const OptTensor &lengths, const Tensor &stats,
                       const Tensor &entropy, const OptTensor &g_logp, const OptTensor &g_entropy,
                       const OptTensor &out) {
  Rows rows(x, lengths);
  Tensor tok, gl, gh;
  if (tokens && tokens->defined()) tok = Ids(*tokens, rows, 0, x, "tokens");
  const Tensor st = Floats(stats, rows, 2, x, "stats"), h = Floats(entropy, rows, 0, x, "entropy");
  if (g_logp && g_logp->defined()) gl = Floats(*g_logp, rows, 0, x, "grad_logp");
  if (g_entropy && g_entropy->defined()) gh = Floats(*g_entropy, rows, 0, x, "grad_entropy");
  Tensor dx = GradOut(out, x);
  int64_t bs = dx.dim() == 3 ? dx.stride(0) : 0;
  const int64_t rs = dx.stride(-2);
  Join(rows.r, &bs, rs);
  Check(kd_token_scores_grad(&rows.r, Ptr<void>(tok), tok.defined() ? IdBytes(tok) : 0, Ptr<float>(st), Ptr<float>(h),
                             Ptr<float>(gl), Ptr<float>(gh), dx.data_ptr(), bs, rs, Stream(x)));
  Written(out);
  return dx;
}

// (a backward pass with create_graph would need the gradient's own: refused, not left out)
void OnceOnly() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "kaldi_decoder.frames: differentiable once; no create_graph");
}

struct ScoresNode : torch::autograd::Function<ScoresNode> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &tokens, int64_t top,
                               const OptTensor &lengths) {
    OptTensor len = lengths && lengths->defined() ? OptTensor(Rows::Lengths(*lengths, x)) : std::nullopt;
    const Scores s = TokenScores(x, tokens, top, len);
    variable_list outs{s.entropy, s.stats}, fixed{s.stats};
    if (s.logp.defined()) outs.push_back(s.logp);
    if (top) {
      outs.insert(outs.end(), {s.top_logp, s.top_ids});
      fixed.insert(fixed.end(), {s.top_logp, s.top_ids});
    }
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable(fixed);
    ctx->save_for_backward({x, tokens ? *tokens : Tensor(), len ? *len : Tensor(), s.stats, s.entropy});
    return outs;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    OnceOnly();
    const variable_list v = ctx->get_saved_variables();
    const Tensor gh = grads[0], gl = v[1].defined() ? grads[2] : Tensor();
    Tensor dx;
    if (gh.defined() || gl.defined()) dx = TokenScoresGrad(v[0], v[1], v[2], v[3], v[4], gl, gh, std::nullopt);
    return {dx, Tensor(), Tensor(), Tensor()};
  }
};

bool WantsGrad(const Tensor &x) { return at::GradMode::is_enabled() && x.requires_grad(); }

OptTensor Given(const Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

std::tuple<OptTensor, Tensor, OptTensor, OptTensor, Tensor> PyTokenScores(const Tensor &x, const OptTensor &tokens,
                                                                        int64_t top, const OptTensor &lengths) {
  if (WantsGrad(x)) {
    const variable_list o = ScoresNode::apply(x, tokens, top, lengths);
    const size_t t = tokens ? 3 : 2;
    return {tokens ? OptTensor(o[2]) : std::nullopt, o[0], top ? OptTensor(o[t]) : std::nullopt,
            top ? OptTensor(o[t + 1]) : std::nullopt, o[1]};
  }
  const Scores s = TokenScores(x, tokens, top, lengths);
  return {Given(s.logp), s.entropy, Given(s.top_logp), Given(s.top_ids), s.stats};
}

// ---- distillation ------------------------------------------------------------------------------

// loss (with `want_loss`; writes `stats` where given) and / or gradient (`want_grad`; of `stats` alone
// without a loss).
std::pair<Tensor, Tensor> Distill(const Tensor &x, const Tensor &ids, const Tensor &teacher, const OptTensor &weights,
                                  double temperature, const OptTensor &lengths, bool want_loss, const Tensor &stats,
                                  const Tensor &upstream, bool want_grad, const OptTensor &out) {
  Rows rows(x, lengths);
  TORCH_CHECK_VALUE(ids.dim() == x.dim() && ids.size(-1) >= 1 && ids.size(-1) <= 256,
                    "teacher_ids must be [..., K] with 1 <= K <= 256, beside logits [..., V]");
  const int64_t slots = ids.size(-1);
  const Tensor id = Ids(ids, rows, slots, x, "teacher_ids");
  const Tensor u = PerRow(teacher, rows, slots, x, DtypeCode(teacher) >= 0, "teacher_logits",
                          "float32, float16 or bfloat16");
  Tensor w, up, loss, dx;
  if (weights && weights->defined()) w = Floats(*weights, rows, 0, x, "weights");
  if (upstream.defined()) up = Floats(upstream, rows, 0, x, "the loss's gradient");
  if (want_loss) loss = Empty(rows.lead, at::kFloat, x);
  int64_t bs = 0, rs = 0;
  if (want_grad) {
    dx = GradOut(out, x);
    bs = dx.dim() == 3 ? dx.stride(0) : 0;
    rs = dx.stride(-2);
  }
  Join(rows.r, want_grad ? &bs : nullptr, rs);
  const size_t bytes = want_loss ? kd_distill_loss_workspace(&rows.r, want_grad) : 0;
  const Tensor ws = Workspace(bytes, x);
  kd_teacher_rows t{};
  t.ids = id.data_ptr();
  t.logits = u.data_ptr();
  t.slots = static_cast<int32_t>(slots);
  t.id_bytes = IdBytes(id);
  t.dtype = DtypeCode(u);
  Check(kd_distill_loss(&rows.r, &t, Ptr<float>(w), static_cast<float>(temperature), Ptr<float>(loss),
                        Ptr<float>(stats), Ptr<float>(up), Ptr<void>(dx), bs, rs, Ptr<void>(ws), bytes, Stream(x)));
  Written(out);
  return {loss, dx};
}

struct DistillNode : torch::autograd::Function<DistillNode> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, const Tensor &teacher,
                        const OptTensor &weights, double temperature, const OptTensor &lengths) {
    OptTensor len = lengths && lengths->defined() ? OptTensor(Rows::Lengths(*lengths, x)) : std::nullopt;
    NoTangent(x, "the tensor of logits");
    TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1, "logits must be a float32, float16 or bfloat16 CUDA tensor");
    std::vector<int64_t> wide(x.sizes().begin(), x.sizes().end());
    wide.back() = 2;
    const Tensor stats = Empty(wide, at::kFloat, x);
    const Tensor loss =
        Distill(x, ids, teacher, weights, temperature, len, true, stats, Tensor(), false, std::nullopt).first;
    ctx->save_for_backward({x, ids, teacher, weights ? *weights : Tensor(), len ? *len : Tensor(), stats});
    ctx->saved_data["temperature"] = temperature;
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    OnceOnly();
    const variable_list v = ctx->get_saved_variables();
    const Tensor dx = Distill(v[0], v[1], v[2], v[3], ctx->saved_data["temperature"].toDouble(), v[4], false, v[5],
                              grads[0], true, std::nullopt)
                          .second;
    return {dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor PyDistillLoss(const Tensor &x, const Tensor &ids, const Tensor &teacher, const OptTensor &weights,
                     double temperature, const OptTensor &lengths) {
  TORCH_CHECK_VALUE(!teacher.requires_grad(), "teacher_logits take no gradient here: detach them");
  TORCH_CHECK_VALUE(!weights || !weights->requires_grad(), "weights take no gradient here: detach them");
  if (WantsGrad(x)) return DistillNode::apply(x, ids, teacher, weights, temperature, lengths);
  return Distill(x, ids, teacher, weights, temperature, lengths, true, Tensor(), Tensor(), false, std::nullopt).first;
}

std::pair<Tensor, Tensor> PyDistillLossAndGrad(const Tensor &x, const Tensor &ids, const Tensor &teacher,
                                               const OptTensor &weights, double temperature, const OptTensor &lengths,
                                               const OptTensor &out) {
  at::NoGradGuard no_grad;
  return Distill(x, ids, teacher, weights, temperature, lengths, true, Tensor(), Tensor(), true, out);
}

Tensor PyTokenScoresGrad(const Tensor &x, const OptTensor &tokens, const OptTensor &lengths, const Tensor &stats,
                         const Tensor &entropy, const OptTensor &g_logp, const OptTensor &g_entropy,
                         const OptTensor &out) {
  at::NoGradGuard no_grad;
  return TokenScoresGrad(x, tokens, lengths, stats, entropy, g_logp, g_entropy, out);
}

}  // namespace

PYBIND11_MODULE(_frames, m) {
  m.doc() = "torch binding of the operators over rows of logits (kaldi_decoder.frames)";
  const py::call_guard<py::gil_scoped_release> free_gil;
  m.def("token_scores", &PyTokenScores, free_gil);
  m.def("token_scores_grad", &PyTokenScoresGrad, free_gil);
  m.def("distill_loss", &PyDistillLoss, free_gil);
  m.def("distill_loss_and_grad", &PyDistillLossAndGrad, free_gil);
}
