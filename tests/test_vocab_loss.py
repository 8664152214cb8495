"""linear_cross_entropy against the formula in float64.

Tolerances.  u is half a step of a type relative to the value (bf16 2^-8,
fp16 2^-11, fp32 2^-24).  With S = sum_d |x||w| + |b|:

* a logit's fp32 sum over d terms is off by at most about (d + 2) 2^-24 S, and
  a loss is a difference and a log-sum of logits: two logits' error, plus the
  exponentials' (a few 2^-23) and the rounding of the loss itself.
* g = c (p - y) is p times (1 + that error), rounded to the inputs' type (fp32:
  not at all) -- twice where the powers were kept in it: p by u, then g by u;
  a gradient is a sum of products of g, off by (2u + logit error + terms
  2^-24) sum (|g| + c eps / V) |w|, plus u of its own rounding, and for dw
  once more, where an upstream factor comes after it.
"""

import math

import pytest
import torch
import torch.nn.functional as F

from kfac_pytorch_amd import ops

IGNORE = -100
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
        torch.float32: 2.0 ** -24}
needs_gpu = pytest.mark.skipif(not torch.cuda.is_available(),
                               reason="needs GPU")


def inputs(rows, dim, vocab, dtype, bias, ignored=0.0, seed=0,
           device="cuda", ints=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g).to(dtype)
    w = (torch.randn(vocab, dim, generator=g) * 2 / math.sqrt(dim)).to(dtype)
    b = torch.randn(vocab, generator=g).to(dtype) if bias else None
    t = torch.randint(vocab, (rows,), generator=g)
    drop = torch.rand(rows, generator=g) < ignored
    t = t.masked_fill(drop, IGNORE).to(ints)
    put = (lambda a: None if a is None else a.to(device))
    return put(x), put(w), put(b), put(t)


def formula(x, w, b, t, eps, up):
    """float64: losses, gradients of sum(up * loss), and the bounds' sums."""
    x, w = x.double().cpu(), w.double().cpu()
    b = torch.zeros(w.size(0), dtype=torch.float64) if b is None \
        else b.double().cpu()
    t = t.long().cpu()
    keep = t != IGNORE
    xs = torch.where(keep[:, None], x, torch.zeros(()).double())
    z = xs @ w.t() + b
    size = (xs.abs() @ w.abs().t() + b.abs()).amax(1)
    y = torch.full_like(z, eps / w.size(0))
    y[torch.arange(len(t)), t.clamp(min=0)] += 1 - eps
    lse = torch.logsumexp(z, 1)
    loss = torch.where(keep, lse - (y * z).sum(1), torch.zeros(()).double())
    g = (z - lse[:, None]).exp() - y
    g = torch.where(keep[:, None], g * up.double().cpu()[:, None],
                    torch.zeros(()).double())
    return {"loss": loss, "size": size, "lse": lse,
            "dx": g @ w, "dw": g.t() @ xs, "db": g.sum(0),
            "sx": g.abs() @ w.abs(), "sw": g.abs().t() @ xs.abs(),
            "sb": g.abs().sum(0), "g": g, "keep": keep,
            "c": torch.where(keep, up.double().cpu().abs(),
                             torch.zeros(()).double()),
            "share": eps / w.size(0)}


def logit_error(ref, dim):
    return (dim + 8) * 2.0 ** -24 * float(ref["size"].max())


def check(name, got, want, bound):
    off = (got.double().cpu() - want).abs()
    assert torch.isfinite(got.double()).all(), name
    worst = (off - bound).max()
    assert worst <= 0, f"{name}: {float(worst)} past the bound, off by up " \
                       f"to {float(off.max())}"


def check_all(ref, loss, grads, x, w, b, dtype, rows, lift=0.0):
    dim, vocab = x.size(1), w.size(0)
    u, e = HALF[dtype], 2 * logit_error(ref, dim)
    if loss is not None:
        check("loss", loss, ref["loss"],
              e + 16 * 2.0 ** -24 * (ref["lse"].abs() + 1)
              + 2.0 ** -23 * ref["size"])
    if grads is None:
        return
    # the smallest steps of fp16 and of exp's flush to zero
    tiny = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -120
    round_g = 0.0 if dtype == torch.float32 else u
    # p = exp(z - lse) is off by the logits' error times p, and by u p where
    # the powers are kept in the inputs' type; off the target p is at most
    # |g| / c + eps / V; at the target, always made from fp32, at most 1
    gabs = ref["g"].abs()
    rel = round_g + 8 * 2.0 ** -24
    wa, xa = w.double().cpu().abs(), x.double().cpu().abs()
    xa = torch.where(ref["keep"][:, None], xa, torch.zeros(()).double())
    p_err = (e + round_g) * (gabs + ref["share"] * ref["c"][:, None])
    at_target = e * ref["c"]
    sx = rel * ref["sx"] + p_err @ wa + (2 * at_target)[:, None] * wa.amax(0)
    sw = rel * ref["sw"] + p_err.t() @ xa \
        + 2 * at_target.max() * xa.amax(0)
    terms = 2.0 ** -24
    check("dx", grads[0], ref["dx"], sx + (vocab + 8) * terms * ref["sx"]
          + u * ref["dx"].abs() + sx * u + tiny)
    check("dw", grads[1], ref["dw"], sw + (rows + 8) * terms * ref["sw"]
          + 2 * u * ref["dw"].abs() + 2 * sw * u + tiny)
    if b is not None:
        sb = 8 * 2.0 ** -24 * ref["sb"] + p_err.sum(0) + 2 * at_target.max()
        check("db", grads[2], ref["db"], sb + (rows + 8) * terms * ref["sb"]
              + u * ref["db"].abs() + sb * u + tiny)


def run(x, w, b, t, eps=0.0, reduction="mean", up=None):
    leaves = [a.detach().requires_grad_() for a in (x, w, b) if a is not None]
    loss = ops.linear_cross_entropy(
        leaves[0], leaves[1], t, bias=leaves[2] if b is not None else None,
        label_smoothing=eps, reduction=reduction)
    grads = torch.autograd.grad(loss, leaves, grad_outputs=up)
    return loss.detach(), grads


SIZES = [
    (1, 8, 2), (1, 64, 1000), (3, 1, 5), (17, 33, 129), (128, 64, 128),
    (129, 72, 257), (35, 256, 3331), (300, 136, 1003), (513, 40, 511),
]


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,dim,vocab", SIZES)
@pytest.mark.parametrize("bias", [False, True])
def test_each_row(rows, dim, vocab, dtype, bias):
    x, w, b, t = inputs(rows, dim, vocab, dtype, bias, 0.2, rows + dim)
    up = torch.linspace(-1.5, 2.0, rows, device="cuda")
    loss, grads = run(x, w, b, t, reduction="none", up=up)
    ref = formula(x, w, b, t, 0.0, up)
    assert loss.dtype == torch.float32 and loss.shape == t.shape
    assert [g.dtype for g in grads] == [dtype] * len(grads)
    check_all(ref, loss, grads, x, w, b, dtype, rows)
    assert not grads[0][t == IGNORE].any() and not loss[t == IGNORE].any()


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("eps", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reduced(dtype, eps, reduction):
    rows, dim, vocab = 200, 96, 700
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.3, 5)
    kept = int((t != IGNORE).sum())
    up = torch.tensor(3.0, device="cuda")
    loss, grads = run(x, w, b, t, eps, reduction, up)
    each = 3.0 / (kept if reduction == "mean" else 1)
    ref = formula(x, w, b, t, eps, torch.full((rows,), each))
    total = ref["loss"].sum() / (kept if reduction == "mean" else 1)
    per = 2 * logit_error(ref, dim) + 2.0 ** -20 * float(ref["lse"].max() + 1)
    check("loss", loss, total,
          per * (1 if reduction == "mean" else kept)
          + 2.0 ** -23 * abs(float(total)))
    check_all(ref, None, grads, x, w, b, dtype, rows)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,dim,vocab,dtype", [
    (2100, 264, 8200, torch.bfloat16),   # more than 256 wide tiles
    (2100, 260, 8200, torch.bfloat16),   # and rows that need packing
    (2100, 264, 8200, torch.float32),
    (2100, 136, 8200, torch.float16),
    (700, 72, 3000, torch.bfloat16),     # tiles of middle size
    (700, 72, 3000, torch.float16),
    (40, 64, 33278, torch.float16),      # a long vocabulary, few rows
    (40, 64, 33278, torch.bfloat16),
    (20, 40, 9000, torch.float32),
])
def test_wide_tiles(rows, dim, vocab, dtype):
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.1, 9)
    up = torch.rand(rows, device="cuda")
    loss, grads = run(x, w, b, t, 0.05, "none", up)
    check_all(formula(x, w, b, t, 0.05, up), loss, grads, x, w, b, dtype,
              rows)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,dim,vocab,dtype", [
    (20000, 8, 40, torch.bfloat16),     # one band, many rows to number
    (20000, 24, 130, torch.float32),
    (70000, 8, 9, torch.float16),
    (3, 8, 1200000, torch.bfloat16),    # a row of more than a million
    (2, 8, 1100000, torch.float32),     # and one whose powers are not kept
])
def test_long_axes(rows, dim, vocab, dtype):
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.3, 41)
    loss, grads = run(x, w, b, t, 0.1, "sum")
    ref = formula(x, w, b, t, 0.1, torch.ones(rows))
    check_all(ref, None, grads, x, w, b, dtype, rows)
    each, _ = run(x, w, b, t, 0.1, "none", torch.ones(rows, device="cuda"))
    check_all(ref, each, None, x, w, b, dtype, rows)
    assert torch.equal(loss, each.double().sum().float())


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_weight_beyond_32_bits(reduction):
    """A weight and its gradient of 4.5 GB, against 64 bits in parts."""
    rows, dim, vocab, part = 3, 12800, 176000, 12000
    u = HALF[torch.bfloat16]
    gen = torch.Generator(device="cuda").manual_seed(43)
    w = torch.randn(vocab, dim, device="cuda", dtype=torch.bfloat16,
                    generator=gen).mul_(2 / math.sqrt(dim))
    assert w.numel() * 2 > 1 << 32
    x = (torch.randn(rows, dim, device="cuda", generator=gen) / 8).bfloat16()
    t = torch.tensor([vocab - 1, 5, vocab - 70001], device="cuda")
    loss, (dx, dw) = run(x, w, None, t, 0.0, reduction,
                         None if reduction == "sum"
                         else torch.ones(rows, device="cuda"))
    xd = x.double()
    z = torch.cat([xd @ p.double().t() for p in w.split(part)], 1)
    size = max(float((xd.abs() @ p.double().abs().t()).max())
               for p in w.split(part))
    each = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    e = 2 * (dim + 8) * 2.0 ** -24 * size  # of a logit less another
    want = each.sum() if reduction == "sum" else each
    assert ((loss.double() - want).abs() <= rows * (e + 2.0 ** -18)).all()
    g = z.softmax(1)
    # an entry: its power and itself rounded, and the logits' errors
    off = g * (e + 2 * u) + 1e-30
    hit = torch.zeros_like(g).scatter_(1, t[:, None], 1.0)
    g -= hit
    off += hit * (e + u)
    sx, ex = torch.zeros_like(xd), torch.zeros_like(xd)
    for k, p in enumerate(w.split(part)):
        cut = slice(k * part, (k + 1) * part)
        p = p.double()
        sx += g[:, cut] @ p
        ex += (off[:, cut] + vocab * 2.0 ** -24 * g[:, cut].abs()) @ p.abs()
        dw_want = g[:, cut].t() @ xd
        bound = off[:, cut].t() @ xd.abs()
        assert ((dw[cut].double() - dw_want).abs()
                <= bound * (1 + u) + u * dw_want.abs()).all()
    assert ((dx.double() - sx).abs() <= ex * (1 + u) + u * sx.abs()).all()


HALVES = [torch.bfloat16, torch.float16]
EACH_TILE = [(*shape, dtype) for shapes, dtypes in [
    ([(660, 8, 21003), (700, 264, 16500),   # 256 x 256 of the logits
      (360, 136, 23600),                    # and of the gradients
      (970, 24, 5010), (2, 264, 6730),      # 128 x 128 of either
      (33, 8, 30505),                       # 128 x 64 of the logits
      (36, 72, 24603), (1, 200, 3372),      # 64 x 64 of either
      (360, 135, 23600), (2, 263, 6730),    # the same with odd rows
      (1, 199, 3371), (360, 134, 23600),    # and rows of whole pairs
      (3, 30, 700)],
     HALVES),
    ([(68, 24, 24900), (2, 520, 8890),      # 128 x 64 of either
      (34, 8, 30505), (1, 264, 11877),      # 64 x 64 of either
      (2, 519, 8890)],
     [torch.float32]),
] for shape in shapes for dtype in dtypes]


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,dim,vocab,dtype", EACH_TILE)
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_each_tile(rows, dim, vocab, dtype, reduction):
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.1, 31)
    up = torch.rand(rows, device="cuda") + 0.5 if reduction == "none" \
        else torch.ones(rows, device="cuda")
    ref = formula(x, w, b, t, 0.05, up)
    loss, grads = run(x, w, b, t, 0.05, reduction,
                      up if reduction == "none" else None)
    check_all(ref, loss if reduction == "none" else None, grads, x, w, b,
              dtype, rows)
    if reduction == "sum":
        each, _ = run(x, w, b, t, 0.05, "none", up)
        assert torch.equal(loss, each.double().sum().float())


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows", [16384, 16385, 20000])
@pytest.mark.parametrize("ignored", [0.0, 0.6])
def test_many_rows(rows, ignored):
    """Either way of numbering the kept rows."""
    x, w, b, t = inputs(rows, 8, 40, torch.float32, False, ignored, rows)
    up = torch.linspace(0.5, 2.0, rows, device="cuda")
    loss, grads = run(x, w, b, t, 0.0, "none", up)
    check_all(formula(x, w, b, t, 0.0, up), loss, grads, x, w, b,
              torch.float32, rows)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_the_targets_factor_is_not_rounded(dtype, reduction):
    """1 - eps lies between two values of the type, u of itself from either;
    with logits of zero and rows of w that add up to zero, dx is
    -(1 - eps) w_t up, here -w_t.  2 - 2 u and 2 are neighbours: with that
    factor rounded, dx would be 2 or less than w_t by as much."""
    u = torch.finfo(dtype).eps / 2
    left = 0.5 + u / 2 * 1.02
    vocab = 65536
    half = (2 - 2 * u) * (torch.randint(0, 2, (vocab // 2, 8), device="cuda")
                          * 2 - 1)
    w = torch.cat([half, -half]).to(dtype)
    x = torch.zeros(64, 8, dtype=dtype, device="cuda")
    t = torch.randint(0, vocab, (64,), device="cuda")
    up = torch.full((64,) if reduction == "none" else (), 1 / left,
                    device="cuda")
    _, grads = run(x, w, None, t, 1 - left, reduction, up)
    # the target's entry is -1 + 1 / vocab of the factor, the others' sum
    # - w_t / vocab: 2^-16 each, together an 8th of fp16's half step below 1
    assert torch.equal(grads[0], -w[t])


@pytest.mark.gpu
@needs_gpu
def test_pieces_of_the_vocabulary():
    """Single rows' losses beyond 256 MB of g: two pieces, against the whole
    call with the same factors kept."""
    rows, dim, vocab = 4100, 16, 17000
    x, w, b, t = inputs(rows, dim, vocab, torch.float32, True, 0.1, 21)
    assert rows * vocab * 4 > 256 << 20
    up = torch.ones(rows, device="cuda")
    loss, grads = run(x, w, b, t, 0.1, "none", up)
    total, kept = run(x, w, b, t, 0.1, "sum")
    # fp32: two orders of summation of the same g
    z = (x.double() @ w.double().t() + b.double())
    z = (z - torch.logsumexp(z, 1, keepdim=True)).exp()
    size = z @ w.double().abs() + w.double().abs()[t.clamp(min=0)] + 1
    bound = (vocab + 64) * 2.0 ** -24 * size
    assert ((grads[0].double() - kept[0].double()).abs() <= bound).all()
    count = torch.bincount(t[t >= 0], minlength=vocab)[:, None]
    size = (z.t() @ x.double().abs()) + (count + 1) * x.double().abs().amax(0)
    bound = (rows + 64) * 2.0 ** -24 * size
    assert ((grads[1].double() - kept[1].double()).abs() <= bound).all()
    size = z.sum(0) + count.squeeze(1) + 1
    bound = (rows + 64) * 2.0 ** -24 * size
    assert ((grads[2].double() - kept[2].double()).abs() <= bound).all()
    assert abs(float(loss.double().sum() - total)) <= 2e-6 * float(total)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
def test_backward_twice(dtype):
    """The first backward pass uses up what the forward pass kept; the second
    makes it again."""
    x, w, b, t = inputs(90, 64, 300, dtype, True, 0.2, 31)
    leaves = [a.requires_grad_() for a in (x, w, b)]
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="sum")
    up = torch.tensor(2.5, device="cuda")
    first = torch.autograd.grad(loss, leaves, up, retain_graph=True)
    second = torch.autograd.grad(loss, leaves, up)
    ref = formula(x.detach(), w.detach(), b.detach(), t, 0.0,
                  torch.full((90,), 2.5))
    for grads in (first, second):
        check_all(ref, None, grads, x.detach(), w.detach(), b.detach(),
                  dtype, 90)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_no_double_backward(reduction):
    x, w, b, t = inputs(9, 16, 30, torch.float32, False)
    x.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, t, reduction=reduction).sum()
    dx, = torch.autograd.grad(loss, x, create_graph=True)
    want, = torch.autograd.grad(
        F.cross_entropy(x @ w.t(), t, reduction=reduction).sum(), x)
    # sums of up to 30 terms of at most 1 * 4
    assert (dx - want).abs().max() <= 64 * 2.0 ** -24 * 4
    with pytest.raises(RuntimeError, match="double backward"):
        dx.sum().backward()


@pytest.mark.gpu
@needs_gpu
def test_ignored_rows_may_hold_anything():
    x, w, b, t = inputs(130, 64, 300, torch.bfloat16, True, 0.4, 3)
    want = run(x, w, b, t)
    dirty = x.clone()
    gone = (t == IGNORE).nonzero().squeeze(1)
    dirty[gone[0::3]] = float("nan")
    dirty[gone[1::3]] = float("inf")
    dirty[gone[2::3]] = torch.finfo(torch.bfloat16).min
    got = run(dirty, w, b, t)
    assert torch.equal(got[0], want[0])
    for a, c in zip(got[1], want[1]):
        assert torch.equal(a, c)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_row_counts(reduction):
    x, w, b, _ = inputs(70, 64, 300, torch.bfloat16, True)
    t = torch.full((70,), IGNORE, device="cuda")
    up = torch.ones(70, device="cuda") if reduction == "none" else None
    loss, grads = run(x, w, b, t, 0.0, reduction, up)
    if reduction == "mean":
        assert torch.isnan(loss)
    else:
        assert not loss.any()
    for g in grads:
        assert not g.any()


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("low", [float("-inf"), "min"])
def test_entries_masked_by_the_bias(low):
    """A bias of -inf, or of the type's lowest value, takes entries out."""
    for dtype in HALF:
        x, w, b, t = inputs(50, 64, 600, dtype, True, 0.1, 4)
        out = torch.arange(600, device="cuda") % 3 == 1
        t = torch.where((t >= 0) & (t % 3 == 1), t - 1, t)
        out[256:384] = True              # all of one tile
        t = torch.where((t >= 256) & (t < 384), 0, t)
        value = torch.finfo(dtype).min if low == "min" else low
        b = b.masked_fill(out, value)
        up = torch.ones(50, device="cuda")
        loss, grads = run(x, w, b, t, 0.0, "none", up)
        kept = ~out
        small = (torch.cumsum(kept, 0) - 1)[t.clamp(min=0)]
        small = torch.where(t == IGNORE, t, small)
        ref = formula(x, w[kept], b[kept], small, 0.0, up)
        check_all(ref, loss, [grads[0], grads[1][kept], grads[2][kept]],
                  x, w[kept], b[kept], dtype, 50)
        assert not grads[1][out].any() and not grads[2][out].any()


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("reduction", ["none", "sum"])
def test_bands_masked_by_large_values(dtype, reduction):
    """Masks of -1e4, -1e9 and the lowest value over whole tiles: what they
    cover weighs nothing, and nothing overflows."""
    x, w, b, t = inputs(50, 64, 900, dtype, True, 0.1, 4)
    lows = [-1e4, -1e9, torch.finfo(dtype).min, float("-inf")]
    for k, low in enumerate(lows):
        low = max(low, torch.finfo(dtype).min) if math.isfinite(low) else low
        b[128 + 128 * k:256 + 128 * k] = low
    kept = torch.ones(900, dtype=torch.bool, device="cuda")
    kept[128:640] = False
    t = torch.where((t >= 128) & (t < 640), 3, t)
    up = torch.ones(50, device="cuda") if reduction == "none" else None
    loss, grads = run(x, w, b, t, 0.0, reduction, up)
    small = torch.where(t >= 640, t - 512, t)
    ref = formula(x, w[kept], b[kept], small, 0.0, torch.ones(50))
    check_all(ref, loss if up is not None else None,
              [grads[0], grads[1][kept], grads[2][kept]], x, w[kept],
              b[kept], dtype, 50)
    assert not grads[1][~kept].any() and not grads[2][~kept].any()


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("base", [-100.0, -200.0])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_masked_bands_beside_low_logits(dtype, base, reduction):
    """Whole bands of -inf in rows whose largest logit is far below zero."""
    x, w, b, t = inputs(50, 64, 900, dtype, True, 0.1, 4)
    b += base
    b[128:640] = float("-inf")
    kept = torch.ones(900, dtype=torch.bool, device="cuda")
    kept[128:640] = False
    t = torch.where((t >= 128) & (t < 640), 3, t)
    up = torch.ones(50, device="cuda") if reduction == "none" else None
    loss, grads = run(x, w, b, t, 0.0, reduction, up)
    each = 1 / int((t != IGNORE).sum()) if reduction == "mean" else 1.0
    small = torch.where(t >= 640, t - 512, t)
    ref = formula(x, w[kept], b[kept], small, 0.0, torch.full((50,), each))
    check_all(ref, loss if up is not None else None,
              [grads[0], grads[1][kept], grads[2][kept]], x, w[kept],
              b[kept], dtype, 50)
    assert not grads[1][~kept].any() and not grads[2][~kept].any()


@pytest.mark.gpu
@needs_gpu
def test_all_entries_masked_alike():
    """A row of nothing but the lowest value is uniform, as in
    F.cross_entropy: the differences are zero."""
    x = torch.zeros(3, 32, device="cuda")
    w = torch.randn(200, 32, device="cuda")
    t = torch.tensor([0, 7, 199], device="cuda")
    for low in (torch.finfo(torch.float32).min, -1e30, -1e9, 1e9, 1e30):
        b = torch.full((200,), low, device="cuda")
        loss, grads = run(x, w, b, t, 0.0, "sum")
        # a loss is log V next to |low|: of the rounding of low alone
        assert abs(float(loss) - 3 * math.log(200)) <= 4 * 2.0 ** -24 * max(
            abs(low) * 3, 64)
        want = torch.full((200,), 3 / 200, device="cuda")
        want[t] -= 1
        assert (grads[2] - want).abs().max() <= 2.0 ** -20


@pytest.mark.gpu
@needs_gpu
def test_infinite_and_nan_logits():
    x, w, b, t = inputs(6, 32, 200, torch.float32, True)
    t = torch.tensor([3, 3, 3, 3, 3, 3], device="cuda")
    x[1, 0] = float("nan")
    x[2, 0] = float("inf")               # logits of both signs: NaN
    b[7] = float("-inf")
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    want = F.cross_entropy(x @ w.t() + b, t, reduction="none")
    assert torch.equal(torch.isnan(loss), torch.isnan(want))
    t[4] = 7                             # a target that cannot be
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    assert loss[4] == float("inf") and torch.isfinite(loss[[0, 3, 5]]).all()
    b[:] = float("-inf")
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    assert torch.isnan(loss).all()


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("bad", [300, -1, 2 ** 40, -2 ** 40])
def test_target_outside_the_vocabulary(bad):
    x, w, b, t = inputs(20, 64, 300, torch.bfloat16, True)
    t[5] = bad
    loss = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    assert torch.isnan(loss[5])
    assert torch.isfinite(loss[torch.arange(20) != 5]).all()
    total, grads = run(x, w, b, t)
    assert torch.isnan(total) and torch.isnan(grads[0][5]).all()


@pytest.mark.gpu
@needs_gpu
def test_layouts():
    """Strided, offset, transposed and expanded operands; int32 targets."""
    dtype = torch.bfloat16
    x, w, b, t = inputs(60, 72, 500, dtype, True, 0.1, 6)
    want = run(x, w, b, t)
    big = torch.zeros(60, 200, device="cuda", dtype=dtype)
    big[:, 3:75] = x
    wt = w.t().contiguous().t()
    off = torch.zeros(500 * 72 + 3, device="cuda", dtype=dtype)[3:]
    off = off.view(500, 72).copy_(w)
    pad = torch.full((500, 90), float("nan"), device="cuda", dtype=dtype)
    pad[:, :72] = w
    half = torch.zeros(1000, device="cuda", dtype=dtype)[::2].copy_(b)
    for xx in (big[:, 3:75], x.t().contiguous().t()):
        for ww in (wt, off, pad[:, :72]):
            got = run(xx, ww, half, t.int())
            assert torch.equal(got[0], want[0])
            for a, c in zip(got[1], want[1]):
                assert torch.equal(a, c)
    row = x[:1].expand(60, 72)
    got = run(row, w, b, t)
    ref = run(row.contiguous(), w, b, t)
    assert torch.equal(got[0], ref[0])
    cube = x.view(5, 12, 72)
    one = ops.linear_cross_entropy(cube, w, t.view(5, 12), bias=b,
                                   reduction="none")
    two = ops.linear_cross_entropy(x, w, t, bias=b, reduction="none")
    assert one.shape == (5, 12) and torch.equal(one.view(-1), two)


@pytest.mark.gpu
@needs_gpu
def test_which_gradients():
    x, w, b, t = inputs(40, 64, 300, torch.bfloat16, True, 0.1, 8)
    full = run(x, w, b, t)[1]
    for k in range(3):
        leaves = [a.clone() for a in (x, w, b)]
        leaves[k].requires_grad_()
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t,
                                        bias=leaves[2])
        got, = torch.autograd.grad(loss, [leaves[k]])
        assert torch.equal(got, full[k])


@pytest.mark.gpu
@needs_gpu
def test_gradient_against_differences():
    x, w, b, t = inputs(12, 16, 40, torch.float32, True, 0.2, 2)
    _, grads = run(x, w, b, t, 0.1, "sum")
    g = torch.Generator().manual_seed(1)
    for k, a in enumerate((x, w, b)):
        step = torch.randn(a.shape, generator=g).double()
        args = [v.double().cpu() for v in (x, w, b)]
        side = []
        for s in (1e-4, -1e-4):
            moved = list(args)
            moved[k] = args[k] + s * step
            z = moved[0] @ moved[1].t() + moved[2]
            side.append(F.cross_entropy(z, t.cpu(), ignore_index=IGNORE,
                                        label_smoothing=0.1,
                                        reduction="sum"))
        slope = (side[0] - side[1]) / 2e-4
        got = (grads[k].double().cpu() * step).sum()
        # third derivatives of a log-sum-exp are at most about |x|^3 <= 1e3
        # along the step: 1e-8 / 6 of that; fp32 sums: 1e-5 of the terms
        bound = 1e-5 + 1e-5 * (grads[k].double().cpu() * step).abs().sum()
        assert abs(got - slope) <= bound


@pytest.mark.gpu
@needs_gpu
def test_autocast_and_shared_weight():
    """bf16 under autocast; one weight as embedding and as projection."""
    torch.manual_seed(0)
    emb = torch.nn.Embedding(90, 32, device="cuda")
    t = torch.randint(90, (3, 7), device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(emb(t), emb.weight, t)
    assert loss.dtype == torch.float32
    loss.backward()
    wide = emb.weight.detach().bfloat16()
    x = wide[t.reshape(-1)]
    ref = formula(x, wide, None, t.reshape(-1), 0.0, torch.full((21,), 1 / 21))
    want = ref["dw"].index_add(0, t.reshape(-1).cpu(), ref["dx"])
    bound = 2.0 ** -6 * (ref["sw"] + ref["dw"].abs()).index_add(
        0, t.reshape(-1).cpu(), ref["sx"] + ref["dx"].abs()) + 1e-6
    check("shared", emb.weight.grad, want, bound)


@pytest.mark.gpu
@needs_gpu
def test_repeats_streams_and_graph():
    """The same bits every time: again, on another stream, and replayed."""
    x, w, b, t = inputs(300, 64, 1100, torch.bfloat16, True, 0.2, 11)
    want = run(x, w, b, t, 0.1)
    again = run(x, w, b, t, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, w, b, t, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    sx, st = torch.zeros_like(x), torch.zeros_like(t)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(sx, w, b, st, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        kept = run(sx, w, b, st, 0.1)
    second = inputs(300, 64, 1100, torch.bfloat16, True, 0.5, 12)
    for xx, tt in ((x, t), (second[0], second[3]), (x, t)):
        sx.copy_(xx)
        st.copy_(tt)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(xx, w, b, tt, 0.1)
        for a, c in zip((kept[0], *kept[1]), (eager[0], *eager[1])):
            assert torch.equal(a, c)
    for got in (again, other):
        for a, c in zip((got[0], *got[1]), (want[0], *want[1])):
            assert torch.equal(a, c)


@pytest.mark.parametrize("device", ["cpu", pytest.param(
    "cuda", marks=[pytest.mark.gpu, needs_gpu])])
def test_refusals(device):
    x, w, b, t = inputs(6, 16, 20, torch.float32, True, device=device)
    call = ops.linear_cross_entropy
    for args, kw in [
            ((x, w, t), {"reduction": "avg"}),
            ((x, w, t), {"label_smoothing": 1.5}),
            ((x, w[:, :8], t), {}), ((x, w[0], t), {}),
            ((x, w, t[:3]), {}), ((x, w, t), {"bias": b[:3]}),
            ((x, w[:0], t), {})]:
        with pytest.raises(ValueError):
            call(*args, **kw)
    with pytest.raises(TypeError):
        call(x, w, t.float())
    with pytest.raises(TypeError):
        call(x, w.bfloat16(), t)
    with pytest.raises(TypeError):
        call(x, w, t, bias=b.bfloat16())
    if device == "cuda":
        with pytest.raises(ValueError):
            call(x, w.cpu(), t)
        with pytest.raises(TypeError):
            call(x.double(), w.double(), t)


@pytest.mark.parametrize("device", ["cpu", pytest.param(
    "cuda", marks=[pytest.mark.gpu, needs_gpu])])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_no_rows_at_all(device, reduction):
    x = torch.empty(0, 16, device=device, requires_grad=True)
    w = torch.randn(20, 16, device=device, requires_grad=True)
    t = torch.empty(0, dtype=torch.int64, device=device)
    loss = ops.linear_cross_entropy(x, w, t, reduction=reduction)
    want = F.cross_entropy(x @ w.t(), t, reduction=reduction)
    assert loss.shape == want.shape
    assert torch.equal(torch.isnan(loss), torch.isnan(want))
    if reduction != "mean":
        loss.sum().backward()
        assert not w.grad.any()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_cpu(reduction, eps):
    x, w, b, t = inputs(30, 24, 70, torch.float32, True, 0.3, 1, "cpu")
    up = torch.rand(30) if reduction == "none" else None
    loss, grads = run(x, w, b, t, eps, reduction, up)
    kept = int((t != IGNORE).sum())
    each = up if up is not None else torch.full(
        (30,), 1.0 / kept if reduction == "mean" else 1.0)
    ref = formula(x, w, b, t, eps, each)
    check_all(ref, loss if reduction == "none" else None, grads, x, w, b,
              torch.float32, 30)
    with pytest.raises(IndexError):
        ops.linear_cross_entropy(x, w, torch.full_like(t, 70))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
def test_ignored_rows_may_hold_anything_on_the_cpu(dtype, eps, reduction):
    x, w, b, t = inputs(24, 16, 70, dtype, True, 0.4, 3, "cpu")
    up = torch.rand(24) if reduction == "none" else None
    want = run(x, w, b, t, eps, reduction, up)
    gone = (t == IGNORE).nonzero().squeeze(1)
    assert len(gone) >= 3
    x[gone[0::3]] = float("nan")
    x[gone[1::3]] = float("inf")
    x[gone[2::3]] = torch.finfo(dtype).min
    got = run(x, w, b, t, eps, reduction, up)
    assert torch.equal(got[0], want[0])
    for a, c in zip(got[1], want[1]):
        assert torch.isfinite(a).all() and torch.equal(a, c)
    assert not got[1][0][gone].any()
    loss, grads = run(x, w, b, torch.full_like(t, IGNORE), eps, reduction, up)
    if reduction == "mean":
        assert torch.isnan(loss)
    else:
        assert not loss.any()
    for g in grads:
        assert not g.any()


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("also", [False, True])
def test_forward_mode_is_refused(which, also):
    """Before any check of devices, so that it can be seen without one; with
    reverse-mode leaves among the inputs too."""
    from torch.autograd import forward_ad
    from kfac_pytorch_amd.ops import _ext
    x, w, b, t = inputs(6, 16, 20, torch.float32, True, device="cpu")
    args = [x, w, b]
    if also:
        args[(which + 1) % 3].requires_grad_()
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which],
                                           torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _ext.linear_cross_entropy(args[0], args[1], t, args[2], IGNORE,
                                      0.0, 1)


@pytest.mark.parametrize("device", ["cpu", pytest.param(
    "cuda", marks=[pytest.mark.gpu, needs_gpu])])
def test_forward_mode(device):
    """The CPU has the tangent, the GPU refuses; without tangents, or with
    forward mode switched off, it answers."""
    from torch.autograd import forward_ad
    x, w, b, t = inputs(6, 16, 20, torch.float32, True, device=device)
    want = ops.linear_cross_entropy(x, w, t, bias=b)
    with forward_ad.dual_level():
        got = ops.linear_cross_entropy(x, w, t, bias=b)
        assert torch.equal(got, want)
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        if device == "cpu":
            loss = ops.linear_cross_entropy(dual, w, t, bias=b)
            slope = forward_ad.unpack_dual(loss).tangent
            leaf = x.clone().requires_grad_()
            dx, = torch.autograd.grad(
                ops.linear_cross_entropy(leaf, w, t, bias=b), leaf)
            # sums of 96 values and of 20 logits' terms, each below 8
            assert abs(slope - dx.sum()) <= 256 * 2.0 ** -24 * 8
        else:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.linear_cross_entropy(dual, w, t, bias=b)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_ignored_rows_beside_a_factor_that_is_not_finite(value, dtype,
                                                         reduction):
    """An overflowed loss scale reaches the rows that count; the ignored
    ones, and all gradients of a call where no row counts, stay zero."""
    x, w, b, t = inputs(70, 64, 300, dtype, True, 0.4, 3)
    up = torch.full((70,) if reduction == "none" else (), value,
                    device="cuda")
    _, grads = run(x, w, b, t, 0.1, reduction, up)
    assert not grads[0][t == IGNORE].any()
    assert not torch.isfinite(grads[0][t != IGNORE]).all()
    _, grads = run(x, w, b, torch.full_like(t, IGNORE), 0.1, reduction, up)
    assert not any(g.any() for g in grads)


class Storageless(torch.Tensor):
    """As a sharded or a fake tensor: a device's name without memory."""

    @staticmethod
    def __new__(cls, like):
        return torch.Tensor._make_wrapper_subclass(
            cls, like.shape, dtype=like.dtype, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} is not for the test")


def test_tensors_without_memory_are_refused():
    """On the host: a kernel would read from address zero."""
    x, w, b, t = inputs(6, 16, 20, torch.float32, True, device="cpu")
    x, w, b, t = (Storageless(a) for a in (x, w, b, t))
    assert x.is_cuda and x.data_ptr() == 0
    for bias in (b, None):
        with pytest.raises(TypeError, match="memory of their own"):
            ops.linear_cross_entropy(x, w, t, bias=bias)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("which", range(4))
def test_one_tensor_without_memory_is_refused(which):
    args = list(inputs(6, 16, 20, torch.float32, True))
    args[which] = Storageless(args[which])
    x, w, b, t = args
    with pytest.raises((TypeError, ValueError)):
        ops.linear_cross_entropy(x, w, t, bias=b)


def test_sparse_tensors_are_refused():
    x, w, b, t = inputs(6, 16, 20, torch.float32, True, device="cpu")
    from kfac_pytorch_amd.ops import _ext
    with pytest.raises((TypeError, ValueError)):
        _ext.linear_cross_entropy(x.to_sparse(), w, t, b, IGNORE, 0.0, 1)


@pytest.mark.parametrize("device", ["cpu", pytest.param(
    "cuda", marks=[pytest.mark.gpu, needs_gpu])])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_operands_with_a_pending_sign(device, reduction):
    """The imaginary part of a lazy conjugate is memory to be negated."""
    args = inputs(20, 16, 70, torch.float32, True, 0.1, 3, device)
    t = args[3]

    def lazy(a):
        a = torch.complex(torch.zeros_like(a), -a).conj().imag
        assert a.is_neg()
        return a

    up = torch.rand(20, device=device) if reduction == "none" else \
        torch.tensor(2.0, device=device)
    want = run(*args, reduction=reduction, up=up)
    got = run(*(lazy(a) for a in args[:3]), t, reduction=reduction,
              up=lazy(up))
    for a, c in zip((got[0], *got[1]), (want[0], *want[1])):
        if device == "cuda":
            assert torch.equal(a, c)
        else:
            # a product's order may go by its operands' layout: sums of up to
            # 70 terms, twice, of at most 16 each
            assert (a - c).abs().max() <= 2 * 78 * 2.0 ** -24 * 70 * 16


EDGES = {"wide": (256, 256, 512), "mid": (128, 128, 512),
         "small": (128, 64, 256), "deep": (64, 64, 256),
         "thin": (64, 32, 256)}


def launched(p, rows, vocab, dim, size, keep):
    """Work items of the largest launch, counted from the plan's tiles."""
    up = lambda a, b: -(-a // b)
    tiles = lambda t, m, n: up(m, EDGES[t][0]) * up(n, EDGES[t][1])
    dim = up(dim, 8) * 8
    logits = tiles(p["logits"], vocab, rows) * EDGES[p["logits"]][2]
    grads = (tiles(p["grads"], dim, rows) * p["dx_splits"]
             + tiles(p["grads"], dim, p["piece"]) * p["dw_splits"]) \
        * EDGES[p["grads"]][2]
    return max(logits, grads, up(rows, 4) * 256)


def test_sizes_that_no_launch_takes_are_refused():
    """The runtime launches fewer than 2^32 work items.  On the host: sizes
    that fit go on to the check of memory, which stands behind it."""
    from kfac_pytorch_amd.ops import _ext
    seen = set()
    for rows, vocab, dim, dtype in [
            (1, 1, 1, torch.bfloat16), (8192, 128000, 4096, torch.bfloat16),
            (1 << 21, 1 << 17, 8, torch.bfloat16),
            (1 << 22, 1 << 17, 8, torch.bfloat16),
            (1 << 23, 1 << 17, 8, torch.bfloat16),
            (1 << 17, 1 << 21, 8, torch.float16),
            (1 << 20, 1 << 20, 64, torch.float16),
            (1 << 19, 1 << 16, 64, torch.float32),
            (1 << 19, 1 << 17, 64, torch.float32),
            ((1 << 26) - 4, 2, 8, torch.bfloat16), (1 << 26, 2, 8,
                                                    torch.bfloat16),
            (2, 1 << 28, 8, torch.bfloat16)]:
        size = dtype.itemsize
        p = _ext.linear_cross_entropy_plan(rows, vocab, dim, size, False)
        count = launched(p, rows, vocab, dim, size, False)
        fits = count < 1 << 32
        assert (p["work_items"] < 1 << 32) == fits and \
            p["work_items"] >= count
        x = Storageless(torch.empty(rows, dim, dtype=dtype, device="meta"))
        w = Storageless(torch.empty(vocab, dim, dtype=dtype, device="meta"))
        t = Storageless(torch.empty(rows, dtype=torch.int64, device="meta"))
        with pytest.raises(TypeError if fits else ValueError,
                           match="memory" if fits else "out of range"):
            ops.linear_cross_entropy(x, w, t)
        seen.add(fits)
    assert seen == {True, False}


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,vocab", [(1 << 23, 1 << 17), (1 << 26, 2)])
def test_large_calls_are_refused_before_anything_is_launched(rows, vocab):
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(vocab, 8, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(rows, dtype=torch.int32, device="cuda")
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="out of range"):
        ops.linear_cross_entropy(x, w, t)
    assert torch.cuda.memory_allocated() == before


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", list(HALF), ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_a_power_of_two_as_upstream_factor_rounds_nothing(dtype, reduction):
    """It scales the gradients' bits; of a factor that is none, bf16 rounds
    the weight's gradient once before it and once after."""
    from kfac_pytorch_amd.ops import _ext
    rows, dim, vocab = 90, 64, 3000
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.2, 31)
    assert _ext.linear_cross_entropy_plan(rows, vocab, dim, dtype.itemsize,
                                          True)["dw_splits"] == 1
    grads = {}
    for up in (1.0, 4.0, 0.25, 3.0):
        grads[up] = run(x, w, b, t, 0.1, reduction,
                        torch.tensor(up, device="cuda"))[1]
    # fp16's smallest steps are lost below 2^-14
    low = 2.0 ** -12 if dtype == torch.float16 else 0.0
    for up in (4.0, 0.25):
        for a, c in zip(grads[up], grads[1.0]):
            assert torch.equal(torch.where(c.abs() >= low, a, 0),
                               torch.where(c.abs() >= low, c * up, 0))
    if dtype == torch.bfloat16:
        assert torch.equal(grads[3.0][1],
                           (grads[1.0][1].float() * 3).bfloat16())


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,dim,vocab,dtype", [
    (700, 256, 33278, torch.bfloat16), (700, 256, 33278, torch.float16),
    (700, 256, 33278, torch.float32), (8192, 256, 9521, torch.bfloat16),
    (4000, 512, 9521, torch.float16), (13, 1000, 20001, torch.bfloat16),
])
def test_memory_until_the_backward_pass(rows, dim, vocab, dtype):
    """What the documentation says: the weight's gradient (fp32 for fp16, or
    partial sums), partial sums of the others, seven numbers for each row."""
    from kfac_pytorch_amd.ops import _ext
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.1, 5)
    leaves = [a.requires_grad_() for a in (x, w, b)]
    size = dtype.itemsize
    p = _ext.linear_cross_entropy_plan(rows, vocab, dim, size, True)
    wide = -(-dim // 8) * 8
    parts = p["dw_splits"] > 1 or dtype == torch.float16
    held = 4 * p["dx_splits"] * rows * wide + 4 * vocab * -(-rows // p["part"])
    held += 4 * p["dw_splits"] * vocab * wide if parts else size * vocab * dim
    assert 1 <= p["dx_splits"] <= 64 and 1 <= p["dw_splits"] <= 16
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    loss = ops.linear_cross_entropy(x, w, t, bias=b)
    # the allocator's blocks are whole 512 bytes, large ones whole 2 MB
    assert torch.cuda.memory_allocated() - before <= held + 28 * rows + (
        4 << 20)
    torch.autograd.grad(loss, leaves)
    del loss
    assert torch.cuda.memory_allocated() - before <= 512


def test_cpu_autocast_casts_as_a_linear_layer():
    """To the autocast type, but for float64."""
    for dtype in (torch.float64, torch.float32, torch.float16):
        x, w, b, t = inputs(9, 16, 20, dtype, True, 0.2, 3, "cpu")
        with torch.autocast("cpu", dtype=torch.bfloat16):
            to = F.linear(x, w, b).dtype
            got = ops.linear_cross_entropy(x, w, t, bias=b)
        want = ops.linear_cross_entropy(x.to(to), w.to(to), t, bias=b.to(to))
        assert torch.equal(got, want) and got.dtype == want.dtype


# tokens enough for dw's k to be cut up, by each of the gradients' tiles
CUT_TOKENS = [(*shape, dtype) for shapes, dtypes in [
    ([(9420, 149, 1919), (9887, 1744, 74),  # 256 x 256, dx cut up and not
      (1697, 8, 8474), (5888, 867, 8),      # 128 x 128
      (6517, 8, 673), (16674, 8, 8),        # 64 x 64
      (1024, 10, 603), (1142, 8, 9)],       # 64 x 32
     HALVES),
    ([(1716, 69, 4269), (9119, 2005, 9),    # 128 x 64
      (5968, 8, 870), (25825, 8, 8),        # 64 x 64
      (1122, 8, 664), (1157, 9, 8)],        # 64 x 32
     [torch.float32]),
] for shape in shapes for dtype in dtypes]


def test_the_lists_reach_every_tile():
    """Which tile a size takes comes of fitted figures: were they fitted
    again, a list here might no longer reach every kernel."""
    from kfac_pytorch_amd.ops import _ext
    for size, logits, grads in [
            (2, {"wide", "mid", "small", "deep", "thin"},
             {"wide", "mid", "deep", "thin"}),
            (4, {"small", "deep", "thin"}, {"small", "deep", "thin"})]:
        shapes = {s[:3] for s in EACH_TILE + CUT_TOKENS
                  if s[3].itemsize == size}
        for keep in (False, True):
            plans = [_ext.linear_cross_entropy_plan(rows, vocab, dim, size,
                                                    keep)
                     for rows, dim, vocab in shapes]
            assert {p["logits"] for p in plans} == logits
            for cut in (False, True):
                assert {p["grads"] for p in plans
                        if (p["dw_splits"] > 1) == cut} == grads
            for tile in grads:
                assert {p["dx_splits"] > 1 for p in plans
                        if p["grads"] == tile} == {False, True}


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("rows,dim,vocab,dtype", CUT_TOKENS)
@pytest.mark.parametrize("reduction", ["sum", "none"])
def test_cut_tokens(rows, dim, vocab, dtype, reduction):
    test_each_tile(rows, dim, vocab, dtype, reduction)


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("dtype", HALVES)
def test_pieces_of_the_vocabulary_in_16_bits(dtype):
    """As in fp32 above: two pieces, against the whole call.  Either way an
    entry of g is off by u of itself, the kept one's power by fp16's too."""
    from kfac_pytorch_amd.ops import _ext
    rows, dim, vocab = 9000, 16, 17000
    piece = _ext.linear_cross_entropy_plan(rows, vocab, dim, 2,
                                           False)["piece"]
    assert piece < vocab
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.1, 21)
    up = torch.ones(rows, device="cuda")
    loss, grads = run(x, w, b, t, 0.1, "none", up)
    total, kept = run(x, w, b, t, 0.1, "sum")
    u = HALF[dtype]
    xd, wd = x.double(), w.double()
    xd[t == IGNORE] = 0
    z = xd @ wd.t()
    z += b.double()
    z -= torch.logsumexp(z, 1, keepdim=True)
    z.exp_()
    z += 0.1 / vocab       # of each entry, |g| at most this, and the target's
    z[t == IGNORE] = 0
    at = t.clamp(min=0)
    # fp16 holds g as g / 2^14 in steps of 2^-24: 2^-39, far below
    off = 2 * u + 2.0 ** -10 + (vocab + rows) * 2.0 ** -24
    size = z @ wd.abs() + wd.abs()[at]
    assert ((grads[0].double() - kept[0].double()).abs()
            <= (off + 2 * u) * size).all()
    size = z.t() @ xd.abs()
    size.index_add_(0, at, xd.abs())
    assert ((grads[1].double() - kept[1].double()).abs()
            <= (off + 2 * u) * size + 2.0 ** -24).all()
    size = z.sum(0) + torch.bincount(t[t >= 0], minlength=vocab)
    assert ((grads[2].double() - kept[2].double()).abs()
            <= (off + 2 * u) * size).all()
    assert abs(float(loss.double().sum() - total)) <= 2e-6 * float(total)


def rounded(v, dtype):
    return torch.tensor(v, dtype=torch.float64).to(dtype).double().item()


def band_of_one_power(bad, ok):
    """(low, vocab): entries of bias 0 at every 32nd place (so in each band),
    `low` elsewhere.  exp(low) as `bad` holds it is off by more than 0.8 2^-8,
    as `ok` by less than 2^-12; its share of the sum lies within a sixth of
    half a step of a bf16 value, and the bad one's is another value."""
    for k in range(1, 2000):
        low = -k / 128.0
        if rounded(low, torch.bfloat16) != low:
            continue
        e = math.exp(low)
        off = bad(e) / e - 1
        if abs(off) < 0.8 * 2.0 ** -8 or abs(ok(e) / e - 1) > 2.0 ** -12:
            continue
        for vocab in range(64, 4096, 32):
            p = e / (vocab // 32 * (1 + 31 * e))
            near = rounded(p, torch.bfloat16)
            step = 2.0 ** (math.floor(math.log2(near)) - 8)  # half of one
            if abs(p - near) <= step / 6 and near > 2 ** -100 and rounded(
                    p * (1 + off), torch.bfloat16) != near:
                return low, vocab, near
    raise AssertionError("no such numbers")


POWERS = {
    "not bf16": lambda e: rounded(e, torch.bfloat16),
    "not fp16 without the lift": lambda e: rounded(e, torch.float16),
}


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("kind", sorted(POWERS))
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_powers_are_kept_as_lifted_fp16_for_bf16(kind, reduction):
    """The bias's gradient is summed before g is rounded: of one row of equal
    powers it shows how these were rounded."""
    low, vocab, want = band_of_one_power(
        POWERS[kind], lambda e: rounded(e * 32768, torch.float16) / 32768)
    b = torch.full((vocab,), low, dtype=torch.bfloat16, device="cuda")
    b[::32] = 0
    x = torch.zeros(1, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(vocab, 8, dtype=torch.bfloat16, device="cuda")
    t = torch.zeros(1, dtype=torch.int64, device="cuda")
    _, grads = run(x, w, b, t, 0.0, reduction)
    db = grads[2].double().cpu()
    db = db[torch.arange(vocab) % 32 != 0]
    assert (db == want).all()


def test_numbers_that_tell_the_powers_types_apart():
    for bad in POWERS.values():
        low, vocab, want = band_of_one_power(
            bad, lambda e: rounded(e * 32768, torch.float16) / 32768)
        e = math.exp(low)
        share = lambda v: rounded(v / (vocab // 32 * (1 + 31 * e)),
                                  torch.bfloat16)
        assert share(e) == want != share(bad(e))


@pytest.mark.gpu
@needs_gpu
def test_calls_of_several_threads():
    """Each on a stream of its own, with sizes in turn: the bits of calls one
    after the other."""
    import threading
    data = [inputs(rows, dim, vocab, dtype, True, 0.2, 7)
            for rows, dim, vocab, dtype in [
                (300, 64, 1100, torch.bfloat16),
                (40, 256, 9000, torch.float16),
                (129, 72, 700, torch.float32),
                (1000, 128, 5000, torch.bfloat16)]]
    want = [run(*a, 0.1) for a in data]
    torch.cuda.synchronize()
    done, errors = [], []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for i in range(12):
                    j = (k + i) % 4
                    got = run(*data[j], 0.1)
                    stream.synchronize()
                    for a, c in zip((got[0], *got[1]),
                                    (want[j][0], *want[j][1])):
                        assert torch.equal(a, c), j
            done.append(k)
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(done) == 4


@pytest.mark.gpu
@needs_gpu
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("rows,dim,vocab,dtype", [
    (2, 2000000, 3, torch.bfloat16), (2, 1999999, 3, torch.float16),
    (3, 1000000, 40, torch.float32), (1, 1, 1, torch.bfloat16),
    (5, 8, 1, torch.float16), (1, 1, 1, torch.float32)])
def test_ends_of_the_sizes(rows, dim, vocab, dtype, reduction):
    x, w, b, t = inputs(rows, dim, vocab, dtype, True, 0.0, 3)
    x = (x / 8).to(dtype)
    up = torch.ones(rows, device="cuda") if reduction == "none" else None
    loss, grads = run(x, w, b, t, 0.05, reduction, up)
    check_all(formula(x, w, b, t, 0.05, torch.ones(rows)),
              loss if up is not None else None, grads, x, w, b, dtype, rows)


@pytest.mark.gpu
@needs_gpu
def test_saved_on_the_cpu_and_checkpointed():
    from torch.utils.checkpoint import checkpoint
    x, w, b, t = inputs(40, 64, 300, torch.bfloat16, True, 0.2, 5)
    want = run(x, w, b, t)
    leaves = [a.clone().requires_grad_() for a in (x, w, b)]
    with torch.autograd.graph.save_on_cpu():
        loss = ops.linear_cross_entropy(leaves[0], leaves[1], t,
                                        bias=leaves[2])
    for a, c in zip(torch.autograd.grad(loss, leaves), want[1]):
        assert torch.equal(a, c)
    loss = checkpoint(
        lambda a, c, d: ops.linear_cross_entropy(a, c, t, bias=d), *leaves,
        use_reentrant=False)
    for a, c in zip(torch.autograd.grad(loss, leaves), want[1]):
        assert torch.equal(a, c)
    with torch.inference_mode():
        assert torch.equal(ops.linear_cross_entropy(x, w, t, bias=b), want[0])


@pytest.mark.gpu
@needs_gpu
def test_step_into_grad_is_captured_and_replayed():
    """projection_loss and its backward pass into .grad, as a user captures
    a step."""
    x, _, _, t = inputs(300, 64, 1100, torch.bfloat16, True, 0.2, 11)
    layer = torch.nn.Linear(64, 1100, device="cuda", dtype=torch.bfloat16)
    x.requires_grad_()
    params = [x, *layer.parameters()]

    def step():
        for p in params:
            p.grad = None
        loss = ops.projection_loss(layer, x, t)
        loss.backward()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(inputs(300, 64, 1100, torch.bfloat16, False, seed=seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = run(x.detach(), layer.weight.detach(), layer.bias.detach(), t)
        assert torch.equal(loss, want[0])
        for p, c in zip(params, want[1]):
            assert torch.equal(p.grad, c)
