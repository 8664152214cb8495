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

int padded(long dim) { return (int)((dim + 7) / 8 * 8); }

// Whether the kernels can load the weight's rows as they lie; otherwise they
// are packed once into rows of whole 16-byte chunks.
bool direct(const Tensor& w) {
  const long size = w.element_size();
  return w.stride(1) == 1 && w.size(1) % 8 == 0 &&
         w.stride(0) >= w.size(1) && w.stride(0) * size % 16 == 0 &&
         w.stride(0) * size < (1l << 22) &&
         reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
}

struct Operands {
  Tensor x, w, b;  // packed kept rows; weight; contiguous bias
  long ldw;
};

Operands operands(Type type, const Tensor& hidden, const Tensor& weight,
                  const std::optional<Tensor>& bias, const Ints& ints,
                  hipStream_t stream) {
  Operands o;
  const int ld = padded(hidden.size(1));
  o.x = at::empty({hidden.size(0), ld}, hidden.options());
  vocab_loss::pack(type, hidden.data_ptr(), hidden.stride(0),
                   hidden.stride(1), hidden.size(0), (int)hidden.size(1),
                   ints.idx, ints.count, o.x.data_ptr(), ld, stream);
  if (direct(weight)) {
    o.w = weight;
    o.ldw = weight.stride(0);
  } else {
    o.w = at::empty({weight.size(0), ld}, weight.options());
    vocab_loss::pack(type, weight.data_ptr(), weight.stride(0),
                     weight.stride(1), weight.size(0), (int)weight.size(1),
                     nullptr, nullptr, o.w.data_ptr(), ld, stream);
    o.ldw = ld;
  }
  if (bias) o.b = bias->contiguous();
  return o;
}

const void* data_or_null(const Tensor& t) {
  return t.defined() ? t.data_ptr() : nullptr;
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

// -> (loss of every row, total or an undefined tensor, lse, ints)
std::tuple<Tensor, Tensor, Tensor, Tensor> vocab_loss_forward(
    Tensor hidden, Tensor weight, Tensor target, std::optional<Tensor> bias,
    int64_t ignore_index, double eps, bool sum, bool mean) {
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
  const Type type = type_of(hidden);
  const auto f32 = hidden.options().dtype(at::kFloat);
  Tensor ints_t = at::empty({4 + 3 * rows}, f32.dtype(at::kInt));
  const Ints ints(ints_t, rows);
  vocab_loss::scan(target.data_ptr(), target.scalar_type() == at::kLong, rows,
                   ignore_index, vocab, ints.pos, ints.idx, ints.tgt,
                   ints.count, stream);
  const Operands o = operands(type, hidden, weight, bias, ints, stream);

  vocab_loss::Forward f{};
  f.plan = vocab_loss::plan(rows, vocab, (int)o.x.size(1),
                            (int)hidden.element_size());
  Tensor loss = at::empty({rows}, f32);
  Tensor lse = at::empty({rows}, f32);
  const long parts = rows * f.plan.tiles;
  Tensor work = at::empty({rows + parts * (eps != 0.0 ? 3 : 2)}, f32);
  f.w = o.w.data_ptr();
  f.x = o.x.data_ptr();
  f.bias = data_or_null(o.b);
  f.ldw = o.ldw;
  f.rows = rows;
  f.vocab = vocab;
  f.ldx = (int)o.x.size(1);
  f.eps = (float)eps;
  f.pos = ints.pos;
  f.tgt = ints.tgt;
  f.count = ints.count;
  f.ztgt = work.data_ptr<float>();
  f.pmax = f.ztgt + rows;
  f.psum = f.pmax + parts;
  f.pz = f.psum + parts;
  f.lse = lse.data_ptr<float>();
  f.loss = loss.data_ptr<float>();
  vocab_loss::forward(type, f, stream);

  Tensor total;
  if (sum || mean) {
    total = at::empty({}, f32);
    vocab_loss::total(f.loss, rows, ints.count, mean,
                      total.data_ptr<float>(), stream);
  }
  return {loss, total, lse, ints_t};
}

// -> (dx, dw, db); those not asked for are undefined
std::tuple<Tensor, Tensor, Tensor> vocab_loss_backward(
    Tensor up, Tensor hidden, Tensor weight, std::optional<Tensor> bias,
    Tensor lse, Tensor ints_t, double eps, bool each, bool mean, bool need_x,
    bool need_w, bool need_b) {
  check_shapes(hidden, weight, bias);
  const long rows = hidden.size(0), vocab = weight.size(0);
  const int dim = (int)hidden.size(1);
  TORCH_CHECK(up.device() == hidden.device() &&
                  up.scalar_type() == at::kFloat && up.is_contiguous() &&
                  up.numel() == (each ? rows : 1) &&
                  lse.numel() == rows && ints_t.numel() == 4 + 3 * rows,
              "linear_cross_entropy: backward state mismatch");
  const c10::OptionalDeviceGuard guard(hidden.device());
  const hipStream_t stream = c10::hip::getCurrentHIPStream().stream();
  const Type type = type_of(hidden);
  const auto f32 = hidden.options().dtype(at::kFloat);
  const Ints ints(ints_t, rows);
  const Operands o = operands(type, hidden, weight, bias, ints, stream);
  const int ldx = (int)o.x.size(1);

  vocab_loss::Backward b{};
  b.plan = vocab_loss::plan(rows, vocab, ldx, (int)hidden.element_size());
  b.piece = b.plan.piece;
  b.dx_splits = b.plan.dx_splits;
  b.dw_splits = b.plan.dw_splits;
  Tensor dx, dw, db;
  if (need_x) dx = at::empty({rows, dim}, hidden.options());
  if (need_w) dw = at::empty({vocab, dim}, weight.options());
  if (need_b) db = at::empty({vocab}, weight.options());
  Tensor small = at::empty({4 + rows}, f32);
  b.scale = small.data_ptr<float>();
  b.coef = b.scale + 4;
  Tensor grad =
      at::empty({rows, (long)padded(b.piece)}, hidden.options());
  Tensor pbias, dx_slabs, dw_slabs;
  if (need_b) pbias = at::empty({b.plan.row_tiles, vocab}, f32);
  if (need_x) dx_slabs = at::empty({b.dx_splits, rows, (long)ldx}, f32);
  if (need_w && b.dw_splits > 1) {
    dw_slabs = at::empty({b.dw_splits, b.piece, (long)ldx}, f32);
  }
  b.w = o.w.data_ptr();
  b.x = o.x.data_ptr();
  b.bias = data_or_null(o.b);
  b.ldw = o.ldw;
  b.rows = rows;
  b.vocab = vocab;
  b.ldx = ldx;
  b.dim = dim;
  b.eps = (float)eps;
  b.pos = ints.pos;
  b.idx = ints.idx;
  b.tgt = ints.tgt;
  b.count = ints.count;
  b.lse = lse.data_ptr<float>();
  b.up = up.data_ptr<float>();
  b.each = each;
  b.mean = mean;
  b.pbias = need_b ? pbias.data_ptr<float>() : nullptr;
  b.dx_slabs = need_x ? dx_slabs.data_ptr<float>() : nullptr;
  b.dw_slabs = dw_slabs.defined() ? dw_slabs.data_ptr<float>() : nullptr;
  b.grad = grad.data_ptr();
  b.dx = need_x ? dx.data_ptr() : nullptr;
  b.dw = need_w ? dw.data_ptr() : nullptr;
  b.db = need_b ? db.data_ptr() : nullptr;
  vocab_loss::backward(type, b, stream);
  return {dx, dw, db};
}
