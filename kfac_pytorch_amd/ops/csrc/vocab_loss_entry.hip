// Entry point of the vocabulary loss on the GPU: checks, autocast, autograd,
// workspaces, streams.
#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "vocab_loss.h"

#include <optional>
#include <vector>

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using vocab_loss::Type;

Type type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return Type::bf16;
    case at::kHalf: return Type::fp16;
    case at::kFloat: return Type::fp32;
    default:
      TORCH_CHECK_TYPE(false, "linear_cross_entropy: bf16, fp16 or fp32 "
                              "expected on the GPU, got ", t.scalar_type());
  }
}

enum Reduction { NONE, MEAN, SUM };

// What a call keeps of its rows, one buffer of 32-bit values: the count, three
// arrays of whole numbers and three of floats.
struct State {
  int *count, *pos, *idx, *tgt;
  float *rowm, *rowi, *ztgt;

  static long size(long rows) { return 4 + 6 * rows; }
  State(const Tensor& t, long rows) {
    count = t.data_ptr<int>();
    pos = count + 4;
    idx = pos + rows;
    tgt = idx + rows;
    rowm = reinterpret_cast<float*>(tgt + rows);
    rowi = rowm + rows;
    ztgt = rowi + rows;
  }
};

// Whether the kernels can load the weight's rows as they lie; otherwise they
// are packed once into rows of whole 16-byte chunks.
bool direct(const Tensor& w) {
  const long size = w.element_size();
  return w.stride(1) == 1 && w.size(1) % 8 == 0 &&
         w.stride(0) >= w.size(1) && w.stride(0) * size % 16 == 0 &&
         w.stride(0) * size < (1l << 22) &&
         reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
}

// The operands as the kernels take them, and what owns them.
struct Call {
  vocab_loss::Operands o{};
  Tensor x, w, b;
  Type type;
  int size;
};

Call make_call(const Tensor& hidden, const Tensor& weight,
               const State& state, double eps, bool keep) {
  Call c;
  c.type = type_of(hidden);
  c.size = (int)hidden.element_size();
  auto& o = c.o;
  o.rows = hidden.size(0);
  o.vocab = weight.size(0);
  o.dim = (int)hidden.size(1);
  o.ldx = (int)vocab_loss::padded(o.dim);
  o.eps = (float)eps;
  o.plan = vocab_loss::plan(o.rows, o.vocab, o.ldx, c.size, keep);
  o.pos = state.pos;
  o.idx = state.idx;
  o.tgt = state.tgt;
  o.count = state.count;
  return c;
}

void pack_weight(Call* c, const Tensor& weight, const Tensor& bias,
                 hipStream_t stream) {
  auto& o = c->o;
  if (direct(weight)) {
    c->w = weight;
    o.ldw = weight.stride(0);
  } else {
    c->w = at::empty({o.vocab, o.ldx}, weight.options());
    vocab_loss::pack(c->type, weight.data_ptr(), weight.stride(0),
                     weight.stride(1), o.vocab, o.dim, nullptr, nullptr,
                     c->w.data_ptr(), o.ldx, stream);
    o.ldw = o.ldx;
  }
  o.w = c->w.data_ptr();
  if (bias.defined()) {
    c->b = bias.contiguous();
    o.bias = c->b.data_ptr();
  }
}

float* floats(const Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The powers of a whole call are kept up to this many bytes (while the call
// lasts); beyond, the backward pass makes the logits again.  Kept, 8192 x
// 128000 x 4096 in bf16 takes 2 GiB and a fifth less time (25.2 against 20.3
// ms).
constexpr long MOST_KEPT = 4l << 30;

bool keeps(long rows, long vocab, int size) {
  const long row = vocab_loss::padded(vocab) * size;
  return row < (1l << 22) && rows * row <= MOST_KEPT;
}

// Whether every launch of a call of these sizes is possible.
bool launches(long rows, long vocab, int ldim, int size) {
  constexpr long MOST = 1l << 32;
  // the smallest tiles and the most cuts: fewer, and no plan need be made
  const long dx = (ldim / 64 + 1) * (rows / 32 + 1) * 64,
             dw = (ldim / 64 + 1) * (vocab / 32 + 1) * 16;
  if (rows < (1l << 25) && vocab < (1l << 25) &&
      (vocab / 64 + 1) * (rows / 32 + 1) * 256 < MOST &&
      (dx + dw) * 256 < MOST) {
    return true;
  }
  for (bool keep : {false, true}) {
    if (keep && !keeps(rows, vocab, size)) continue;
    const auto plan = vocab_loss::plan(rows, vocab, ldim, size, keep);
    if (vocab_loss::work_items(plan, rows, vocab, ldim, size, keep) >= MOST) {
      return false;
    }
  }
  return true;
}

struct Need {
  bool x, w, b;
  bool any() const { return x || w || b; }
};

// What the forward pass leaves for vocab_finish: dw, and the fp32 parts of the
// others in one buffer; undefined where not needed.
struct Kept {
  Tensor parts, dw;
};

// Where what lies in Kept::parts, in floats.
struct Parts {
  long dx = 0, dw = 0, bias = 0;

  Parts(const vocab_loss::Operands& o, Type type, Need need) {
    if (need.x) dx = o.plan.dx_splits * o.rows * o.ldx;
    // fp16 stays in fp32 until the upstream factor, a loss's scale, is known:
    // the type's range is too small to be scaled afterwards.  bf16 that is not
    // cut up is rounded here and once more where the factor is no power of two
    // (relative to the norm, off by 2.4e-3 to 2.6e-3 then and 1.9e-3 else; a
    // layer in bf16 with its loss: 2.4e-3 to 3.6e-3).  In fp32 until the end it
    // would be 1.9e-3 always and cost the usual factor of 1 a second pass: 700
    // x 33278 x 256 takes 109.8 us instead of 101.3, 8192 x 128000 x 4096 21.18
    // ms instead of 20.19, and twice the memory until the backward pass.
    if (need.w && (o.plan.dw_splits > 1 || type == Type::fp16)) {
      dw = o.plan.dw_splits * o.vocab * o.ldx;
    }
    if (need.b) bias = o.plan.parts * o.vocab;
  }
  long all() const { return dx + dw + bias; }
  void set(vocab_loss::Grads* b, const Tensor& parts) const {
    float* at = parts.defined() ? parts.data_ptr<float>() : nullptr;
    if (dx) b->dx_slabs = at;
    if (dw) b->dw_slabs = at + dx;
    if (bias) b->pbias = at + dx + dw;
  }
};

struct Loss {
  Tensor loss, state;
  bool keep;
  Kept kept;
};

// The loss (a scalar, or of every row).  With gradients needed and a reduced
// loss it also makes these, for an upstream factor of 1, if the powers fit.
Loss vocab_forward(const Tensor& hidden, const Tensor& weight,
                   const Tensor& bias, const Tensor& target,
                   int64_t ignore_index, double eps, Reduction reduction,
                   Need need) {
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const auto f32 = hidden.options().dtype(at::kFloat);
  const long rows = hidden.size(0), vocab = weight.size(0);
  const bool mean = reduction == MEAN;
  Loss r;
  r.state = at::empty({State::size(rows)}, f32.dtype(at::kInt));
  const State state(r.state, rows);
  r.keep = reduction != NONE && need.any() &&
           keeps(rows, vocab, (int)hidden.element_size());
  Call c = make_call(hidden, weight, state, eps, r.keep);
  const auto& plan = c.o.plan;

  // packed x, the powers, the bands, and losses that are only added up
  const long xs = (rows * c.o.ldx * c.size + 255) / 256 * 64;
  const long row = vocab_loss::padded(vocab) * c.size;
  const long powers = r.keep ? (rows * row + 255) / 256 * 64 : 0;
  const long bands = rows * plan.bands;
  Tensor work = at::empty(
      {xs + powers + bands * (eps != 0.0 ? 3 : 2) +
       (reduction == NONE ? 0 : rows)}, f32);
  c.o.x = work.data_ptr();
  vocab_loss::prepare(c.type, target.data_ptr(),
                      target.scalar_type() == at::kLong, rows, ignore_index,
                      vocab, state.pos, state.idx, state.tgt, state.count,
                      hidden.data_ptr(), hidden.stride(0), hidden.stride(1),
                      c.o.dim, work.data_ptr(), c.o.ldx, stream);
  pack_weight(&c, weight, bias, stream);

  vocab_loss::Sums f{};
  f.pmax = work.data_ptr<float>() + xs + powers;
  f.psum = f.pmax + bands;
  f.pz = f.psum + bands;
  f.rowm = state.rowm;
  f.rowi = state.rowi;
  f.ztgt = state.ztgt;
  void* grad = r.keep ? work.data_ptr<float>() + xs : nullptr;
  if (reduction == NONE) {
    r.loss = at::empty({rows}, f32);
    f.loss = r.loss.data_ptr<float>();
  } else {
    f.loss = f.pmax + bands * (eps != 0.0 ? 3 : 2);
  }
  vocab_loss::forward(c.type, c.o, f, grad, stream);

  if (reduction != NONE) {
    r.loss = at::empty({}, f32);
    f.total = r.loss.data_ptr<float>();
    if (!r.keep) {
      vocab_loss::total(f.loss, rows, state.count, mean, f.total, stream);
    }
  }
  if (r.keep) {
    const Parts parts(c.o, c.type, need);
    if (parts.all()) r.kept.parts = at::empty({parts.all()}, f32);
    if (need.w && !parts.dw) {
      r.kept.dw = at::empty({vocab, (long)c.o.dim}, weight.options());
    }
    vocab_loss::Grads b{};
    b.mean = mean;
    b.grad = grad;
    b.dw = data(r.kept.dw);
    parts.set(&b, r.kept.parts);
    vocab_loss::gradients_kept(c.type, c.o, f, b, stream);
  }
  return r;
}

struct Gradients {
  Tensor dx, dw, db;  // undefined where not asked for
};

// What vocab_forward kept, times up; uses it up.
Gradients vocab_finish(const Tensor& up, const Tensor& hidden,
                       const Tensor& weight, const Tensor& state_t,
                       double eps, bool mean, Need need, const Kept& k) {
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const State state(state_t, hidden.size(0));
  Call c = make_call(hidden, weight, state, eps, true);
  const Parts parts(c.o, c.type, need);
  Gradients g;
  if (need.x) g.dx = at::empty({c.o.rows, (long)c.o.dim}, hidden.options());
  if (need.w) {
    g.dw = parts.dw ? at::empty({c.o.vocab, (long)c.o.dim}, weight.options())
                    : k.dw;
  }
  if (need.b) g.db = at::empty({c.o.vocab}, weight.options());
  vocab_loss::Grads b{};
  b.mean = mean;
  parts.set(&b, k.parts);
  b.dx = data(g.dx);
  b.dw = data(g.dw);
  b.db = data(g.db);
  vocab_loss::finish_kept(c.type, c.o, b, up.data_ptr<float>(), stream);
  return g;
}

// The gradients from the operands: the logits are made again.
Gradients vocab_backward(const Tensor& up, const Tensor& hidden,
                         const Tensor& weight, const Tensor& bias,
                         const Tensor& state_t, double eps,
                         Reduction reduction, Need need) {
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const auto f32 = hidden.options().dtype(at::kFloat);
  const long rows = hidden.size(0), vocab = weight.size(0);
  const State state(state_t, rows);
  Call c = make_call(hidden, weight, state, eps, false);
  const long dim = c.o.dim, ldx = c.o.ldx;
  c.x = at::empty({rows, ldx}, hidden.options());
  vocab_loss::pack(c.type, hidden.data_ptr(), hidden.stride(0),
                   hidden.stride(1), rows, c.o.dim, c.o.idx, c.o.count,
                   c.x.data_ptr(), c.o.ldx, stream);
  c.o.x = c.x.data_ptr();
  pack_weight(&c, weight, bias, stream);
  const auto& plan = c.o.plan;

  Gradients g;
  Tensor pbias, dx_slabs, dw_slabs;
  if (need.x) {
    g.dx = at::empty({rows, dim}, hidden.options());
    dx_slabs = at::empty({plan.dx_splits, rows, ldx}, f32);
  }
  if (need.w) {
    g.dw = at::empty({vocab, dim}, weight.options());
    if (plan.dw_splits > 1) {
      dw_slabs = at::empty({plan.dw_splits, plan.piece, ldx}, f32);
    }
  }
  if (need.b) {
    g.db = at::empty({vocab}, weight.options());
    pbias = at::empty({plan.parts, vocab}, f32);
  }
  Tensor small = at::empty({4 + rows}, f32);
  Tensor grad =
      at::empty({rows, vocab_loss::padded(plan.piece)}, hidden.options());
  vocab_loss::Sums f{};
  f.rowm = state.rowm;
  f.rowi = state.rowi;
  f.ztgt = state.ztgt;
  vocab_loss::Grads b{};
  b.scale = small.data_ptr<float>();
  b.coef = b.scale + 4;
  b.mean = reduction == MEAN;
  b.pbias = floats(pbias);
  b.dx_slabs = floats(dx_slabs);
  b.dw_slabs = floats(dw_slabs);
  b.grad = data(grad);
  b.dx = data(g.dx);
  b.dw = data(g.dw);
  b.db = data(g.db);
  vocab_loss::coefficients(c.type, c.o, up.data_ptr<float>(),
                           reduction == NONE, b, stream);
  vocab_loss::gradients_again(c.type, c.o, f, b, stream);
  return g;
}

// A reduced loss leaves its gradients for an upstream factor of 1, which the
// first backward pass uses up; a loss of single rows, a second backward pass,
// or a call too large to keep its powers makes the logits again.
class VocabLoss : public torch::autograd::Function<VocabLoss> {
 public:
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden,
                        const Tensor& weight,
                        const std::optional<Tensor>& bias,
                        const Tensor& target, int64_t ignore_index,
                        double eps, int64_t reduction) {
    const Tensor b = bias.value_or(Tensor());
    const Need need{hidden.requires_grad(), weight.requires_grad(),
                    b.defined() && b.requires_grad()};
    const Loss r = vocab_forward(hidden, weight, b, target, ignore_index, eps,
                                 (Reduction)reduction, need);
    ctx->save_for_backward({hidden, weight, b, r.state});
    auto& saved = ctx->saved_data;
    saved["call"] = c10::ivalue::Tuple::create(
        {eps, reduction, (int64_t)(need.x | need.w << 1 | need.b << 2)});
    if (r.keep) saved["parts"] = r.kept.parts;
    if (r.kept.dw.defined()) saved["dw"] = r.kept.dw;
    return r.loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list tensors = ctx->get_saved_variables();
    const Tensor &hidden = tensors[0], &weight = tensors[1],
                 &bias = tensors[2], &state = tensors[3];
    auto& saved = ctx->saved_data;
    const auto call = saved["call"].toTuple();
    const double eps = call->elements()[0].toDouble();
    const auto reduction = (Reduction)call->elements()[1].toInt();
    const int64_t bits = call->elements()[2].toInt();
    const Need need{(bits & 1) != 0, (bits & 2) != 0, (bits & 4) != 0};
    const bool differentiable = at::GradMode::is_enabled();
    Gradients g;
    {
      const at::NoGradGuard none;
      const Tensor up = grads[0].resolve_neg().contiguous();
      const auto parts = saved.find("parts");
      if (parts != saved.end()) {
        Kept kept;
        if (!parts->second.isNone()) kept.parts = parts->second.toTensor();
        saved.erase(parts);
        const auto dw = saved.find("dw");
        if (dw != saved.end()) {
          kept.dw = dw->second.toTensor();
          saved.erase(dw);
        }
        g = vocab_finish(up, hidden, weight, state, eps, reduction == MEAN,
                         need, kept);
      } else {
        g = vocab_backward(up, hidden, weight, bias, state, eps, reduction,
                           need);
      }
    }
    variable_list out = {g.dx,     g.dw,     g.db,    Tensor(),
                         Tensor(), Tensor(), Tensor()};
    if (differentiable) {  // but differentiating these once more is an error
      for (Tensor& t : out) {
        if (!t.defined()) continue;
        const auto error = std::make_shared<torch::autograd::DelayedError>(
            "linear_cross_entropy has no double backward", 1);
        t.requires_grad_();
        t = (*error)({t})[0];
      }
    }
    return out;
  }
};

}  // namespace

// hidden (..., d), weight (V, d), target (...), bias (V,) or none; reduction 0:
// none, 1: mean, 2: sum.  At least one row.
Tensor linear_cross_entropy(Tensor hidden, Tensor weight, Tensor target,
                            std::optional<Tensor> bias, int64_t ignore_index,
                            double eps, int64_t reduction) {
  // a tangent would be lost without a word: nothing below carries it
  const auto dual = [](const Tensor& t) { return t._fw_grad(0).defined(); };
  TORCH_CHECK_NOT_IMPLEMENTED(
      !c10::AutogradState::get_tls_state().get_fw_grad_mode() ||
          !(dual(hidden) || dual(weight) || (bias && dual(*bias))),
      "linear_cross_entropy has no forward-mode derivative on the GPU");
#define CHECK_VALUE(cond, ...) \
  TORCH_CHECK_VALUE(cond, "linear_cross_entropy: ", __VA_ARGS__)
  CHECK_VALUE(eps >= 0.0 && eps <= 1.0,
              "label_smoothing must be in [0, 1], got ", eps);
  CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 &&
                  hidden.size(-1) == weight.size(1),
              "hidden (..., d) and weight (V, d) expected, got ",
              hidden.sizes(), " and ", weight.sizes());
  CHECK_VALUE(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1),
              "target must have hidden's shape without its last dimension, "
              "got ", target.sizes());
  CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == weight.size(0)),
              "bias must have weight's first dimension, got ",
              bias->sizes());
  TORCH_CHECK_TYPE(target.scalar_type() == at::kLong ||
                       target.scalar_type() == at::kInt,
                   "linear_cross_entropy: target must be int64 or int32, "
                   "got ", target.scalar_type());
  CHECK_VALUE(weight.numel() > 0, "weight is empty");
  CHECK_VALUE(hidden.is_cuda() && weight.device() == hidden.device() &&
                  target.device() == hidden.device() &&
                  (!bias || bias->device() == hidden.device()),
              "all tensors must be on ", hidden.device());
  const bool casts = at::autocast::is_autocast_enabled(at::kCUDA);
  const auto cast = at::autocast::get_autocast_dtype(at::kCUDA);
  const int64_t d = hidden.size(-1), n = hidden.numel() / d,
                size = c10::elementSize(casts ? cast : hidden.scalar_type());
  CHECK_VALUE(n > 0 && n < (1l << 30) && weight.size(0) < (1l << 30) &&
                  d * size < (1l << 22) &&
                  launches(n, weight.size(0), (int)vocab_loss::padded(d),
                           (int)size),
              "sizes out of range: ", hidden.sizes(), " and ",
              weight.sizes());
  // sharded or fake tensors name a device and have no memory there
  const auto dense = [](const Tensor& t) {
    return t.layout() == at::kStrided &&
           (t.numel() == 0 || t.const_data_ptr() != nullptr);
  };
  TORCH_CHECK_TYPE(dense(hidden) && dense(weight) && dense(target) &&
                       (!bias || dense(*bias)),
                   "linear_cross_entropy: dense tensors with memory of their "
                   "own expected");
  // the kernels read memory: no sign may be pending on it
  hidden = hidden.resolve_neg();
  weight = weight.resolve_neg();
  if (bias) bias = bias->resolve_neg();
  if (casts) {
    hidden = at::autocast::cached_cast(cast, hidden, at::kCUDA);
    weight = at::autocast::cached_cast(cast, weight, at::kCUDA);
    if (bias) bias = at::autocast::cached_cast(cast, *bias, at::kCUDA);
  }
  TORCH_CHECK_TYPE(hidden.scalar_type() == weight.scalar_type() &&
                       (!bias || bias->scalar_type() == weight.scalar_type()),
                   "linear_cross_entropy: hidden, weight and bias must have "
                   "one dtype, got ", hidden.scalar_type(), ", ",
                   weight.scalar_type(), bias ? ", " : "",
                   bias ? c10::toString(bias->scalar_type()) : "");
  type_of(hidden);
  const Tensor rows =
      hidden.dim() == 2 ? hidden : hidden.reshape({-1, hidden.size(-1)});
  const Tensor flat = target.reshape({-1}).contiguous();
#undef CHECK_VALUE
  const bool grads =
      at::GradMode::is_enabled() &&
      (rows.requires_grad() || weight.requires_grad() ||
       (bias && bias->requires_grad()));
  const Tensor loss =
      grads ? VocabLoss::apply(rows, weight, bias, flat, ignore_index, eps,
                               reduction)
            : vocab_forward(rows, weight, bias.value_or(Tensor()), flat,
                            ignore_index, eps, (Reduction)reduction, Need{})
                  .loss;
  return reduction == NONE ? loss.view(target.sizes()) : loss;
}

// What a call of these sizes is cut into, for tests: logits' and gradients'
// tile, pieces' length, dx's and dw's cuts, tokens to a part of the bias's
// gradient, work items of the largest launch.
std::vector<int64_t> linear_cross_entropy_plan(int64_t rows, int64_t vocab,
                                               int64_t dim, int64_t size,
                                               bool keep) {
  TORCH_CHECK_VALUE(rows > 0 && vocab > 0 && dim > 0 &&
                        (size == 2 || size == 4) && rows < (1l << 30) &&
                        vocab < (1l << 30) && dim * size < (1l << 22),
                    "linear_cross_entropy_plan: sizes out of range");
  const int ldim = (int)vocab_loss::padded(dim);
  const auto p = vocab_loss::plan(rows, vocab, ldim, (int)size, keep);
  return {(int64_t)p.logits, (int64_t)p.grads, p.piece, p.dx_splits,
          p.dw_splits, p.part,
          vocab_loss::work_items(p, rows, vocab, ldim, (int)size, keep)};
}
