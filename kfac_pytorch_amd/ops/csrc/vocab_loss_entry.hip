// Entry points of the vocabulary-loss kernels: checks, workspaces, streams.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "vocab_loss.h"

#include <optional>
#include <tuple>

namespace {

using torch::Tensor;
using vocab_loss::Type;

Type type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return Type::bf16;
    case at::kHalf: return Type::fp16;
    case at::kFloat: return Type::fp32;
    default:
      TORCH_CHECK(false, "linear_cross_entropy: dtype must be bf16, fp16 or "
                         "fp32, got ", t.scalar_type());
  }
}

// The integers of a call, one buffer: count, then three arrays over the rows.
struct Ints {
  int *count, *pos, *idx, *tgt;
  Ints(const Tensor& t, long rows) {
    count = t.data_ptr<int>();
    pos = count + 4;
    idx = pos + rows;
    tgt = idx + rows;
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
               const std::optional<Tensor>& bias, const Tensor& ints_t,
               double eps, bool keep) {
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
  const Ints ints(ints_t, o.rows);
  o.pos = ints.pos;
  o.idx = ints.idx;
  o.tgt = ints.tgt;
  o.count = ints.count;
  return c;
}

void pack_hidden(Call* c, const Tensor& hidden, hipStream_t stream) {
  auto& o = c->o;
  c->x = at::empty({o.rows, o.ldx}, hidden.options());
  vocab_loss::pack(c->type, hidden.data_ptr(), hidden.stride(0),
                   hidden.stride(1), o.rows, o.dim, o.idx, o.count,
                   c->x.data_ptr(), o.ldx, stream);
  o.x = c->x.data_ptr();
}

void pack_weight(Call* c, const Tensor& weight,
                 const std::optional<Tensor>& bias, hipStream_t stream) {
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
  if (bias) {
    c->b = bias->contiguous();
    o.bias = c->b.data_ptr();
  }
}

float* floats(const Tensor& t) {
  return t.defined() ? t.data_ptr<float>() : nullptr;
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// The powers of a whole call are kept up to this many bytes (while the call
// lasts); beyond, the backward pass makes the logits again.  Kept, 8192 x
// 128000 x 4096 in bf16 takes 2 GiB and a quarter less time.
constexpr long MOST_KEPT = 4l << 30;

bool keeps(long rows, long vocab, int size) {
  const long row = vocab_loss::padded(vocab) * size;
  return row < (1l << 22) && rows * row <= MOST_KEPT;
}

vocab_loss::Sums row_state(const Tensor& state, long rows) {
  vocab_loss::Sums f{};
  f.rowm = state.data_ptr<float>();
  f.rowi = f.rowm + rows;
  f.ztgt = f.rowi + rows;
  return f;
}

void check_shapes(const Tensor& hidden, const Tensor& weight,
                  const std::optional<Tensor>& bias) {
  TORCH_CHECK(hidden.is_cuda() && weight.device() == hidden.device(),
              "linear_cross_entropy: hidden and weight must be on one GPU");
  TORCH_CHECK(hidden.dim() == 2 && weight.dim() == 2 &&
                  hidden.size(1) == weight.size(1),
              "linear_cross_entropy: shape mismatch");
  TORCH_CHECK(hidden.scalar_type() == weight.scalar_type() &&
                  (!bias || (bias->scalar_type() == weight.scalar_type() &&
                             bias->device() == weight.device() &&
                             bias->dim() == 1 &&
                             bias->size(0) == weight.size(0))),
              "linear_cross_entropy: hidden, weight and bias must agree");
  TORCH_CHECK(hidden.size(0) > 0 && hidden.size(1) > 0 && weight.size(0) > 0,
              "linear_cross_entropy: empty operand");
  TORCH_CHECK(hidden.size(0) < (1l << 30) && weight.size(0) < (1l << 30) &&
                  hidden.size(1) * hidden.element_size() < (1l << 22),
              "linear_cross_entropy: sizes out of range");
}

}  // namespace

// -> (loss of every row, total or an undefined tensor, state of the kept
// rows, ints, kept).  kept: what vocab_loss_finish needs, empty where the
// gradients are left to vocab_loss_backward.
std::tuple<Tensor, Tensor, Tensor, Tensor, std::vector<std::optional<Tensor>>>
vocab_loss_forward(Tensor hidden, Tensor weight, Tensor target,
                   std::optional<Tensor> bias, int64_t ignore_index,
                   double eps, bool sum, bool mean, bool need_x, bool need_w,
                   bool need_b) {
  check_shapes(hidden, weight, bias);
  const long rows = hidden.size(0), vocab = weight.size(0);
  TORCH_CHECK(target.device() == hidden.device() && target.dim() == 1 &&
                  target.size(0) == rows && target.is_contiguous() &&
                  (target.scalar_type() == at::kLong ||
                   target.scalar_type() == at::kInt),
              "linear_cross_entropy: target must be contiguous int32 or "
              "int64, one for each row, on the same GPU");
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const auto f32 = hidden.options().dtype(at::kFloat);
  Tensor ints_t = at::empty({4 + 3 * rows}, f32.dtype(at::kInt));
  const Ints ints(ints_t, rows);
  const bool keep = (sum || mean) && (need_x || need_w || need_b) &&
                    keeps(rows, vocab, (int)hidden.element_size());
  Call c = make_call(hidden, weight, bias, ints_t, eps, keep);
  c.x = at::empty({rows, (long)c.o.ldx}, hidden.options());
  c.o.x = c.x.data_ptr();
  vocab_loss::prepare(c.type, target.data_ptr(),
                      target.scalar_type() == at::kLong, rows, ignore_index,
                      vocab, ints.pos, ints.idx, ints.tgt, ints.count,
                      hidden.data_ptr(), hidden.stride(0), hidden.stride(1),
                      c.o.dim, c.x.data_ptr(), c.o.ldx, stream);
  pack_weight(&c, weight, bias, stream);
  const auto& plan = c.o.plan;

  Tensor loss = at::empty({rows}, f32);
  Tensor state = at::empty({3, rows}, f32);
  const long bands = rows * plan.bands;
  Tensor work = at::empty({bands * (eps != 0.0 ? 3 : 2)}, f32);
  vocab_loss::Sums f = row_state(state, rows);
  f.pmax = work.data_ptr<float>();
  f.psum = f.pmax + bands;
  f.pz = f.psum + bands;
  f.loss = loss.data_ptr<float>();
  Tensor grad;
  if (keep) {
    grad = at::empty({rows, vocab_loss::padded(vocab)}, hidden.options());
  }
  vocab_loss::forward(c.type, c.o, f, data(grad), stream);

  Tensor total;
  if (sum || mean) {
    total = at::empty({}, f32);
    f.total = total.data_ptr<float>();
    if (!keep) {
      vocab_loss::total(f.loss, rows, ints.count, mean, f.total, stream);
    }
  }
  std::vector<std::optional<Tensor>> kept;
  if (keep) {
    Tensor dx_slabs, dw, dw_slabs, pbias;
    if (need_x) {
      dx_slabs = at::empty({plan.dx_splits, rows, (long)c.o.ldx}, f32);
    }
    // fp16 stays in fp32 until the upstream factor, a loss's scale, is known
    if (need_w && (plan.dw_splits > 1 || c.type == Type::fp16)) {
      dw_slabs = at::empty({plan.dw_splits, vocab, (long)c.o.ldx}, f32);
    } else if (need_w) {
      dw = at::empty({vocab, (long)c.o.dim}, weight.options());
    }
    if (need_b) pbias = at::empty({plan.parts, vocab}, f32);
    vocab_loss::Grads b{};
    b.mean = mean;
    b.pbias = floats(pbias);
    b.dx_slabs = floats(dx_slabs);
    b.dw_slabs = floats(dw_slabs);
    b.grad = data(grad);
    b.dw = data(dw);
    vocab_loss::gradients_kept(c.type, c.o, f, b, stream);
    for (const Tensor& t : {dx_slabs, dw, dw_slabs, pbias}) {
      kept.push_back(t.defined() ? std::optional<Tensor>(t) : std::nullopt);
    }
  }
  return {loss, total, state, ints_t, kept};
}

// The gradients that vocab_loss_forward kept, times up; uses them up.
// -> (dx, dw, db); those not asked for are undefined
std::tuple<Tensor, Tensor, Tensor> vocab_loss_finish(
    Tensor up, Tensor hidden, Tensor weight, Tensor ints_t, bool mean,
    std::vector<std::optional<Tensor>> kept) {
  check_shapes(hidden, weight, std::nullopt);
  TORCH_CHECK(up.device() == hidden.device() && up.numel() == 1 &&
                  up.scalar_type() == at::kFloat && kept.size() == 4 &&
                  ints_t.numel() == 4 + 3 * hidden.size(0),
              "linear_cross_entropy: backward state mismatch");
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  Call c = make_call(hidden, weight, std::nullopt, ints_t, 0.0, true);
  Tensor dx, dw, db;
  Tensor dx_slabs = kept[0].value_or(Tensor());
  Tensor dw_slabs = kept[2].value_or(Tensor());
  Tensor pbias = kept[3].value_or(Tensor());
  if (dx_slabs.defined()) {
    dx = at::empty({c.o.rows, (long)c.o.dim}, hidden.options());
  }
  if (dw_slabs.defined()) {
    dw = at::empty({c.o.vocab, (long)c.o.dim}, weight.options());
  } else if (kept[1]) {
    dw = *kept[1];
  }
  if (pbias.defined()) db = at::empty({c.o.vocab}, weight.options());
  vocab_loss::Grads b{};
  b.mean = mean;
  b.pbias = floats(pbias);
  b.dx_slabs = floats(dx_slabs);
  b.dw_slabs = floats(dw_slabs);
  b.dx = data(dx);
  b.dw = data(dw);
  b.db = data(db);
  vocab_loss::finish_kept(c.type, c.o, b, up.data_ptr<float>(), stream);
  return {dx, dw, db};
}

// -> (dx, dw, db); those not asked for are undefined
std::tuple<Tensor, Tensor, Tensor> vocab_loss_backward(
    Tensor up, Tensor hidden, Tensor weight, std::optional<Tensor> bias,
    Tensor state, Tensor ints_t, double eps, bool each, bool mean,
    bool need_x, bool need_w, bool need_b) {
  check_shapes(hidden, weight, bias);
  const long rows = hidden.size(0), vocab = weight.size(0);
  TORCH_CHECK(up.device() == hidden.device() &&
                  up.scalar_type() == at::kFloat && up.is_contiguous() &&
                  up.numel() == (each ? rows : 1) &&
                  state.numel() == 3 * rows &&
                  ints_t.numel() == 4 + 3 * rows,
              "linear_cross_entropy: backward state mismatch");
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const auto f32 = hidden.options().dtype(at::kFloat);
  Call c = make_call(hidden, weight, bias, ints_t, eps, false);
  pack_hidden(&c, hidden, stream);
  pack_weight(&c, weight, bias, stream);
  const auto& plan = c.o.plan;
  const long dim = c.o.dim, ldx = c.o.ldx;

  Tensor dx, dw, db, pbias, dx_slabs, dw_slabs;
  if (need_x) {
    dx = at::empty({rows, dim}, hidden.options());
    dx_slabs = at::empty({plan.dx_splits, rows, ldx}, f32);
  }
  if (need_w) {
    dw = at::empty({vocab, dim}, weight.options());
    if (plan.dw_splits > 1) {
      dw_slabs = at::empty({plan.dw_splits, plan.piece, ldx}, f32);
    }
  }
  if (need_b) {
    db = at::empty({vocab}, weight.options());
    pbias = at::empty({plan.parts, vocab}, f32);
  }
  Tensor small = at::empty({4 + rows}, f32);
  Tensor grad =
      at::empty({rows, vocab_loss::padded(plan.piece)}, hidden.options());
  vocab_loss::Grads b{};
  b.scale = small.data_ptr<float>();
  b.coef = b.scale + 4;
  b.mean = mean;
  b.pbias = floats(pbias);
  b.dx_slabs = floats(dx_slabs);
  b.dw_slabs = floats(dw_slabs);
  b.grad = data(grad);
  b.dx = data(dx);
  b.dw = data(dw);
  b.db = data(db);
  vocab_loss::coefficients(c.type, c.o, up.data_ptr<float>(), each, b,
                           stream);
  vocab_loss::gradients_again(c.type, c.o, row_state(state, rows), b, stream);
  return {dx, dw, db};
}
