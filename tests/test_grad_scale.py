"""global_norm, clip_by_global_norm, clip_grad_norm_ and kl_clip in float64.

Tolerances.  Sums are in double: their error (2^-53 times the square root of
some 10^6 terms) is far below the rounding of the result to fp32, half a step
of 2^-24.  The factor is rounded to fp32 once more, the product once to fp32
and once to the output's type: u + 3 * 2^-24, u half a step of that type
relative to the value (bf16 2^-8, fp16 2^-11, fp32 2^-24), and half its
smallest step (fp16 2^-25, the others' below 2^-130).
"""

import math

import pytest
import torch

from kfac_pytorch_amd import ops

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11,
        torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -24}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
gpu = pytest.param("cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(
    not torch.cuda.is_available(), reason="needs GPU")])
devices = pytest.mark.parametrize("device", ["cpu", gpu])
only_gpu = pytest.mark.parametrize("device", [gpu])


def tensors(shapes, dtype, device, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(device)
            for s in shapes]


def cat(ts):
    return torch.cat([t.double().cpu().reshape(-1) for t in ts])


def near(got, want, rel, small=2.0 ** -130):
    off = (got.double().cpu() - want).abs()
    assert (off <= rel * want.abs() + small).all(), float(off.max())


def near_out(out, want):
    for o, w in zip(out, want):
        near(o, w, HALF[o.dtype] + 3 * 2.0 ** -24,
             2.0 ** -25 if o.dtype == torch.float16 else 2.0 ** -130)


SHAPES = [
    [(1,)], [()], [(0,), (3,)], [(7,), (1, 1), (33, 65)],
    [(2048 * 4,)], [(2048 * 4 + 1,)], [(2048 * 8 - 1,), (5,)],
    [(3, 5, 7, 9), (300, 1000), (70001,)],
    [(k % 7 + 1, 13) for k in range(300)],      # more than one launch
]


@devices
@pytest.mark.parametrize("shapes", SHAPES, ids=range(len(SHAPES)))
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_and_clip(shapes, dtype, device):
    ts = tensors(shapes, dtype, device, len(shapes))
    flat = cat(ts)
    for p in (1.0, 2.0, math.inf):
        want = torch.linalg.vector_norm(flat, p)
        norm = ops.global_norm(ts, p)
        assert norm.dtype == torch.float32 and norm.shape == ()
        near(norm, want, 2.0 ** -23)
        for most in (0.0, 0.3 * float(want), 10 * float(want) + 1):
            out, norm = ops.clip_by_global_norm(ts, most, p)
            near(norm, want, 2.0 ** -23)
            f = min(1.0, most / (float(want) + 1e-6))
            assert [o.shape for o in out] == [t.shape for t in ts]
            assert [o.dtype for o in out] == [t.dtype for t in ts]
            near_out(out, [t.double().cpu() * f for t in ts])
    assert torch.equal(cat(ts), flat)           # inputs as they were


@devices
@pytest.mark.parametrize("clips", [True, False])
def test_in_place(clips, device):
    ts = tensors([(100, 33), (5,), (4097,)], torch.float32, device)
    before = [t.clone() for t in ts]
    norm = torch.linalg.vector_norm(cat(ts))
    most = float(norm) * (0.5 if clips else 2.0)
    out, got = ops.clip_by_global_norm(ts, most, out=ts)
    near(got, norm, 2.0 ** -23)
    assert all(a is b for a, b in zip(out, ts))
    if clips:
        f = most / (float(norm) + 1e-6)
        near_out(ts, [b.double().cpu() * f for b in before])
    else:
        assert all(torch.equal(a, b) for a, b in zip(ts, before))


@devices
def test_written_tensors_are_seen_by_autograd(device):
    a = torch.ones(5, device=device, requires_grad=True)
    b = a * 2
    (b * b).sum().backward(retain_graph=True)
    c = (b * b).sum()
    ops.clip_by_global_norm([b.detach()], 0.1, out=[b.detach()])
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        c.backward()


@devices
def test_layouts(device):
    """Views of a bucket, strides, channels-last, expanded, mixed types."""
    flat, = tensors([(5000,)], torch.float32, device, 3)
    parts = list(flat[1:4800].split([7, 1, 1000, 90, 3701]))
    parts.append(flat[4801:4997:3])
    other = torch.zeros(5003, device=device)
    out = list(other[2:4801].split([7, 1, 1000, 90, 3701]))
    out.append(other[4802:5001:3][:66])
    base, = tensors([(40, 31)], torch.bfloat16, device, 4)
    conv, = tensors([(6, 5, 3, 3)], torch.float16, device, 5)
    conv = conv.contiguous(memory_format=torch.channels_last)
    ts = parts + [base[:, :-1], base[:, -1], base.t()[3:20, ::2], conv,
                  conv[:, 1:, :2], flat[:9].expand(4, 9),
                  flat[:4].view(4, 1).expand(4, 9)]
    outs = out + [torch.zeros(40, 30, device=device, dtype=torch.bfloat16),
                  torch.zeros(40, device=device)] + [
        torch.empty_like(t, memory_format=torch.contiguous_format)
        for t in ts[-5:]]
    assert [t.shape for t in ts] == [o.shape for o in outs]
    want = torch.linalg.vector_norm(cat(ts))
    got, norm = ops.clip_by_global_norm(ts, 1.0, out=outs)
    near(norm, want, 2.0 ** -23)
    f = 1.0 / (float(want) + 1e-6)
    near_out(outs, [t.double().cpu() * f for t in ts])
    # what lies between the views stays
    assert not other[:2].any() and not other[4803::3][:60].any()


@devices
def test_values_that_are_not_finite(device):
    for bad in (math.nan, math.inf):
        for p in (1.0, 2.0, math.inf):
            ts = tensors([(70, 70), (9000,)], torch.float32, device)
            ts[1][8123] = bad
            ts[0][3, 3] = 1e30
            out, norm = ops.clip_by_global_norm(ts, 1.0, p)
            assert (torch.isnan(norm) if bad != bad else
                    norm == math.inf)
            ok = out[0]
            assert torch.isnan(ok).all() if bad != bad else not ok.any()
            assert torch.isnan(out[1][8123])
    big = [torch.full((1000,), 1e25, device=device)]
    near(ops.global_norm(big), torch.tensor(1e25 * math.sqrt(1000)).double(),
         2.0 ** -22)
    tiny = [torch.full((1000,), 1e-30, device=device)]
    near(ops.global_norm(tiny), torch.tensor(1e-30 * math.sqrt(1000)).double(),
         2.0 ** -22, 0.0)


@devices
def test_clip_grad_norm_(device):
    mine = torch.nn.Sequential(torch.nn.Linear(30, 20),
                               torch.nn.Linear(20, 5)).to(device)
    mine[1].bias.requires_grad_(False)
    mine(torch.ones(4, 30, device=device)).square().sum().backward()
    theirs = [p.grad.clone() for p in mine.parameters() if p.grad is not None]
    want = torch.nn.utils.get_total_norm(theirs)
    got = ops.clip_grad_norm_(mine.parameters(), 0.5)
    near(got, want.double().cpu(), 2.0 ** -20)  # theirs sums in fp32
    f = 0.5 / (float(want) + 1e-6)
    for a, b in zip([p.grad for p in mine.parameters()
                     if p.grad is not None], theirs):
        near(a, b.double().cpu() * f, 2.0 ** -19)
    # one tensor, the same parameter twice, no gradient at all
    p = mine[0].weight
    norm = torch.linalg.vector_norm(p.grad.double().cpu())
    near(ops.clip_grad_norm_(p, 1e9), norm, 2.0 ** -23)
    near(ops.clip_grad_norm_([p, p], 1e9), norm, 2.0 ** -23)
    assert ops.clip_grad_norm_(mine[1].bias, 1.0) == 0
    assert ops.clip_grad_norm_([], 1.0) == 0
    p.grad[0, 0] = math.nan
    before = p.grad.clone()
    with pytest.raises(RuntimeError):
        ops.clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad[1:], before[1:])


def trust(us, gs, lr, kl):
    dot = abs(float(torch.dot(cat(us), cat(gs)))) * lr * lr
    return min(1.0, math.sqrt(kl / max(dot, 1e-30)))


@devices
@pytest.mark.parametrize("grad_type", TYPES)
@pytest.mark.parametrize("update_type", TYPES)
@pytest.mark.parametrize("lr", [0.0, 1e-4, 0.1, 3.0])
def test_kl_clip(lr, update_type, grad_type, device):
    shapes = [(64, 33), (64,), (3, 5, 3, 3), (1,), (9001,), (0,)]
    us = tensors(shapes, update_type, device, 1)
    gs = [(u.float() * 0.2 + n).to(grad_type)
          for u, n in zip(us, tensors(shapes, torch.float32, device, 2, 0.1))]
    nu_want = trust(us, gs, lr, 0.001)
    want = [u.double().cpu() * nu_want for u in us]
    out, nu = ops.kl_clip(us, gs, lr=lr, kl_clip=0.001)
    near(nu, torch.tensor(nu_want).double(), 2.0 ** -23)
    assert [o.dtype for o in out] == [grad_type] * len(gs)
    near_out(out, want)
    ops.kl_clip(us, gs, lr=lr, kl_clip=0.001, out=gs)
    assert all(torch.equal(a, b) for a, b in zip(gs, out))


@devices
def test_kl_clip_of_a_bucket_with_bias_columns(device):
    """Updates are [out, in + 1] blocks of one buffer, as K-FAC keeps them;
    written over themselves, the blocks' neighbours stay."""
    dims = [(5, 4), (64, 33), (1, 1), (300, 257), (17, 1)]
    flat, = tensors([(sum(o * (i + 1) for o, i in dims) + 2,)],
                    torch.float32, device, 7)
    us, gs, at = [], [], 1
    for k, (o, i) in enumerate(dims):
        block = flat[at:at + o * (i + 1)].view(o, i + 1)
        at += o * (i + 1)
        us += [block[:, :i], block[:, i:].reshape(o) if k % 2 else block[:, i]]
        gs += tensors([(o, i), (o,)], torch.float32, device, 20 + k)
    before = [u.double().cpu() for u in us]
    nu_want = trust(us, gs, 0.1, 1e-4)
    edge = flat[0].clone(), flat[-1].clone()
    _, nu = ops.kl_clip(us, gs, lr=0.1, kl_clip=1e-4, out=us)
    near(nu, torch.tensor(nu_want).double(), 2.0 ** -23)
    near_out(us, [b * nu_want for b in before])
    assert flat[0] == edge[0] and flat[-1] == edge[1]


@devices
def test_kl_clip_of_nan_and_cancelling(device):
    us = tensors([(50,), (2000,)], torch.float32, device, 1)
    gs = tensors([(50,), (2000,)], torch.float32, device, 2)
    gs[1][77] = math.nan
    out, nu = ops.kl_clip(us, gs, lr=0.1, kl_clip=0.001)
    assert torch.isnan(nu) and torch.isnan(out[0]).all()
    u = torch.ones(4096, device=device)
    g = torch.ones(4096, device=device)
    g[::2] = -1                       # <u, g> = 0: nothing to bound
    out, nu = ops.kl_clip([u], [g], lr=0.1, kl_clip=0.001)
    assert nu == 1 and torch.equal(out[0], u)


@only_gpu
def test_repeats_stream_and_graph(device):
    shapes = [(200, 33), (70001,), (5,)]
    ts = tensors(shapes, torch.float32, device, 1)
    gs = tensors(shapes, torch.float32, device, 2)

    def both(a, b):
        out, norm = ops.clip_by_global_norm(a, 1.0)
        out2, nu = ops.kl_clip(out, b, lr=0.3, kl_clip=0.001)
        return [*out, norm, *out2, nu]

    want = both(ts, gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(ts, gs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = both(ts, gs)
    for seed in (3, 4, 5):
        for t, n in zip(ts, tensors(shapes, torch.float32, device, seed)):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, both(ts, gs)))


@devices
def test_refusals(device):
    a, b = tensors([(4, 3), (5,)], torch.float32, device)
    with pytest.raises(ValueError):
        ops.global_norm([a, b], 3.0)
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a, b], -1.0)
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a, b], math.nan)
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a, b], 1.0, out=[a])
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a, a], 1.0, out=[a, a])
    with pytest.raises(ValueError):
        ops.clip_by_global_norm([a, b], 1.0, out=[b, a])
    with pytest.raises(TypeError):
        ops.global_norm([a.long()])
    with pytest.raises(ValueError):
        ops.kl_clip([a], [b], lr=1.0, kl_clip=0.001)
    with pytest.raises(ValueError):
        ops.kl_clip([a, b], [a], lr=1.0, kl_clip=0.001)
    with pytest.raises(ValueError):
        ops.kl_clip([a], [a], lr=1.0, kl_clip=0.0)
    if device == "cuda":
        with pytest.raises(ValueError):
            ops.global_norm([a, b.cpu()])
        with pytest.raises(TypeError):
            ops.global_norm([a.double()])
        with pytest.raises(ValueError):
            ops.clip_by_global_norm([a], 1.0, out=[a[:1].expand(4, 3)])


@devices
def test_shared_memory(device):
    """An output is its own input or lies apart from all of them."""
    flat = torch.arange(1.0, 41.0, device=device)
    a, b, c = flat[:10], flat[10:20], flat[20:30]
    for out in ([b, a], [b, c], [flat[5:15], c], [c, flat[25:35]],
                [a, flat[1:11]], [a.view(torch.bfloat16)[:10], c]):
        before = flat.clone()
        with pytest.raises(ValueError, match="memory"):
            ops.clip_by_global_norm([a, b], 1.0, out=out)
        with pytest.raises(ValueError, match="memory"):
            ops.kl_clip([a, b], [c, c], lr=1.0, kl_clip=0.001, out=out)
        assert torch.equal(flat, before)
    with pytest.raises(ValueError, match="memory"):
        ops.clip_by_global_norm([a, a], 1.0, out=[a, c])
    # in place beside an output of its own, neighbours, gaps woven together
    want = torch.linalg.vector_norm(flat[:20].double().cpu())
    f = 1.0 / (float(want) + 1e-6)
    wants = [a.double().cpu() * f, b.double().cpu() * f]
    ops.clip_by_global_norm([a, b], 1.0, out=[a, c])
    near_out([a, c], wants)
    grid = torch.arange(1.0, 41.0, device=device).view(10, 4)
    ins = [grid[:, :2], grid[:, 2:]]
    wants = [t.double().cpu() / (float(torch.linalg.vector_norm(
        grid.double())) + 1e-6) for t in ins]
    ops.clip_by_global_norm(ins, 1.0, out=ins)
    near_out(ins, wants)
    # the gradients may be written: they are read before
    us = [flat[:10].clone(), flat[10:20].clone()]
    gs = [flat[20:30], flat[30:40]]
    wants, nu = ops.kl_clip(us, gs, lr=1.0, kl_clip=0.001)
    out, got = ops.kl_clip(us, gs, lr=1.0, kl_clip=0.001, out=gs[::-1])
    assert torch.equal(nu, got)
    assert all(torch.equal(x, y) for x, y in zip(out, wants))


@devices
def test_forward_mode_is_refused(device):
    """A clipped tensor's tangent would lack the norm's part, or be lost."""
    from torch.autograd import forward_ad
    a, b = tensors([(5, 3), (5, 3)], torch.float32, device)
    with forward_ad.dual_level():
        ops.clip_by_global_norm([a], 1.0, out=[b.clone()])
        d = forward_ad.make_dual(a, b)
        for call in (lambda: ops.global_norm([a, d]),
                     lambda: ops.clip_by_global_norm([d], 1.0),
                     lambda: ops.clip_by_global_norm([a], 1.0, out=[d]),
                     lambda: ops.kl_clip([d], [b], lr=1.0, kl_clip=0.001),
                     lambda: ops.kl_clip([a], [d], lr=1.0, kl_clip=0.001)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


class Storageless(torch.Tensor):
    """As a sharded or a fake tensor: a device's name without memory."""

    @staticmethod
    def __new__(cls, shape):
        return torch.Tensor._make_wrapper_subclass(
            cls, shape, dtype=torch.float32, device="cuda")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        assert func is torch.ops.aten.detach.default, func
        return cls(args[0].shape)


class Parameter:
    def __init__(self, grad):
        self.grad = grad


def test_tensors_without_memory_are_refused():
    """On the host: a kernel would read from address zero."""
    a, b, c = (Storageless((5, 3)) for _ in range(3))
    assert a.is_cuda and a.data_ptr() == 0
    for call in (lambda: ops.global_norm([a, b]),
                 lambda: ops.clip_by_global_norm([a], 1.0, out=[a]),
                 lambda: ops.clip_by_global_norm([a], 1.0, out=[b]),
                 lambda: ops.kl_clip([a], [b], lr=1.0, kl_clip=0.001,
                                     out=[c]),
                 lambda: ops.clip_grad_norm_([Parameter(a)], 1.0)):
        with pytest.raises(TypeError, match="memory of their own"):
            call()


@only_gpu
def test_one_tensor_without_memory_is_refused(device):
    a = Storageless((5, 3))
    b = torch.ones(5, 3, device=device)
    for call in (lambda: ops.global_norm([b, a]),
                 lambda: ops.clip_by_global_norm([b], 1.0, out=[a]),
                 lambda: ops.kl_clip([b], [a], lr=1.0, kl_clip=0.001,
                                     out=[b])):
        with pytest.raises((TypeError, ValueError)):
            call()


@devices
def test_tensors_with_a_pending_sign(device):
    """The imaginary part of a lazy conjugate is memory to be negated."""
    def lazy(a):
        a = torch.complex(torch.zeros_like(a), -a).conj().imag
        assert a.is_neg()
        return a

    us = tensors([(64, 33), (5,), (9000,)], torch.float32, device, 1)
    gs = tensors([(64, 33), (5,), (9000,)], torch.float32, device, 2)
    gs = [u + 0.1 * g for u, g in zip(us, gs)]
    clipped, norm = ops.clip_by_global_norm(us, 1.0)
    out, nu = ops.kl_clip(us, gs, lr=1.0, kl_clip=0.001)

    def same(got, want, number, wanted):
        near(number, wanted.double().cpu(), 2.0 ** -23)
        for a, b in zip(got, want):
            assert torch.equal(a, b)

    same(*[[lazy(u) for u in us], us], ops.global_norm(
        [lazy(u) for u in us]), norm)
    got, n = ops.clip_by_global_norm([lazy(u) for u in us], 1.0)
    same(got, clipped, n, norm)
    got, n = ops.clip_by_global_norm(us, 1.0, out=[lazy(u) for u in us])
    same(got, clipped, n, norm)
    both = [lazy(u) for u in us]
    got, n = ops.clip_by_global_norm(both, 1.0, out=both)
    same(both, clipped, n, norm)
    for a, b in (([lazy(u) for u in us], gs), (us, [lazy(g) for g in gs]),
                 ([lazy(u) for u in us], [lazy(g) for g in gs])):
        written = [torch.zeros(g.shape, device=device) for g in gs]
        got, n = ops.kl_clip(a, b, lr=1.0, kl_clip=0.001, out=written)
        same(written, out, n, nu)
    got, n = ops.kl_clip([lazy(u) for u in us], [lazy(g) for g in gs], lr=1.0,
                         kl_clip=0.001)
    same(got, out, n, nu)
    # the sign is pending on one of the two only: written over the gradients
    both = [lazy(g) for g in gs]
    got, n = ops.kl_clip(us, both, lr=1.0, kl_clip=0.001, out=both)
    same(both, out, n, nu)


@devices
@pytest.mark.parametrize("update_order,grad_order", [
    (torch.contiguous_format, torch.channels_last),
    (torch.channels_last, torch.contiguous_format),
    (torch.channels_last, torch.channels_last)])
def test_kl_clip_of_channels_last(update_order, grad_order, device):
    """Convolutions' gradients in one order, the updates in another; written
    apart and over the gradients."""
    shapes = [(6, 5, 3, 3), (16, 16, 1, 1), (33, 7, 5, 5), (4, 1, 3, 3)]
    us = [u.contiguous(memory_format=update_order)
          for u in tensors(shapes, torch.float32, device, 1)]
    gs = [(u * 0.2 + n).contiguous(memory_format=grad_order)
          for u, n in zip(us, tensors(shapes, torch.float32, device, 2, 0.1))]
    nu_want = trust(us, gs, 0.5, 0.001)
    want = [u.double().cpu() * nu_want for u in us]
    strides = [g.stride() for g in gs]
    out, nu = ops.kl_clip(us, gs, lr=0.5, kl_clip=0.001)
    near(nu, torch.tensor(nu_want).double(), 2.0 ** -23)
    near_out(out, want)
    ops.kl_clip(us, gs, lr=0.5, kl_clip=0.001, out=gs)
    near_out(gs, want)
    assert [g.stride() for g in gs] == strides
