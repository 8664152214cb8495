"""The end of a training step as it is used: the model's loss without logits,
clipping, the K-FAC step with its trust region -- and that each gives what the
separate torch calls gave."""

import copy

import pytest
import torch
import torch.nn.functional as F

import kfac_pytorch_amd as kfac
from kfac_pytorch_amd import ops
from kfac_pytorch_amd.models import LSTMLanguageModel, make_transformer
from kfac_pytorch_amd.utils import LabelSmoothLoss

VOCAB = 211
devices = pytest.mark.parametrize("device", ["cpu", pytest.param(
    "cuda", marks=[pytest.mark.gpu, pytest.mark.skipif(
        not torch.cuda.is_available(), reason="needs GPU")])])


def close(got, want, rel):
    """Within rel of the largest of the wanted values."""
    off = (got.double() - want.double()).abs().max()
    assert off <= rel * want.double().abs().max(), float(off)


def lstm(device):
    torch.manual_seed(0)
    model = LSTMLanguageModel(vocab_size=VOCAB, emb=32, hidden=32, layers=1,
                              dropout=0.0).to(device)
    x = torch.randint(VOCAB, (4, 9), device=device)
    y = torch.randint(VOCAB, (4, 9), device=device)
    y[:, -2:] = -100
    return model, x, y


# fp32 models of the same weights: sums of up to 211 products, in another
# order, differ by 211 * 2^-24 = 2^-16 of their terms at most; gradients that
# went through a few such layers are given 2^-12 of their largest value
REL = 2.0 ** -12


@devices
def test_lstm_loss_and_gradients(device):
    model, x, y = lstm(device)
    twin = copy.deepcopy(model)
    loss, hidden = model(x, targets=y)
    logits, hidden2 = twin(x)
    want = F.cross_entropy(logits.reshape(-1, VOCAB), y.reshape(-1))
    close(loss, want, REL)
    close(hidden[0], hidden2[0], REL)
    loss.backward()
    want.backward()
    for a, b in zip(model.parameters(), twin.parameters()):
        close(a.grad, b.grad, REL)


@devices
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_transformer_loss_and_gradients(smoothing, device):
    torch.manual_seed(0)
    model = make_transformer(vocab=VOCAB, d_model=32, nhead=4, num_layers=1,
                             dim_ff=64, max_len=32, dropout=0.0).to(device)
    twin = copy.deepcopy(model)
    src = torch.randint(VOCAB, (3, 7), device=device)
    trg = torch.randint(VOCAB, (3, 6), device=device)
    loss = model(src, trg[:, :-1], targets=trg[:, 1:], smoothing=smoothing)
    want = LabelSmoothLoss(smoothing)(
        twin(src, trg[:, :-1]).reshape(-1, VOCAB), trg[:, 1:].reshape(-1))
    close(loss, want, REL)
    loss.backward()
    want.backward()
    for a, b in zip(model.parameters(), twin.parameters()):
        close(a.grad, b.grad, REL)


@devices
@pytest.mark.parametrize("name", sorted(kfac.kfac_mappers))
def test_step(name, device, single_process_comm):
    """Loss, clip, precondition, update; against the same with torch's own
    calls and the layer-by-layer trust region.  The preconditioners see
    gradients that differ in their last bits and solve in fp32: the updates
    are compared at 2^-7 of their largest value."""
    results = []
    for fused in (True, False):
        model, x, y = lstm(device)
        head = torch.nn.Sequential(
            torch.nn.Linear(32, 24), torch.nn.Tanh(),
            torch.nn.Linear(24, 32)).to(device)
        params = list(model.parameters()) + list(head.parameters())
        whole = torch.nn.ModuleList([model, head])
        pre = kfac.get_kfac_module(name)(
            whole, lr=0.1, damping=0.03, exclude_vocabulary_size=VOCAB)
        if not fused:
            pre._one_pass_update = lambda grads, updates: False
        opt = torch.optim.SGD(params, lr=0.1)
        for _ in range(2):
            opt.zero_grad()
            out, _ = model.lstm(model.embed(x))
            out = out + head(out)
            if fused:
                loss = ops.projection_loss(model.decoder, out, y)
            else:
                loss = F.cross_entropy(
                    model.decoder(out).reshape(-1, VOCAB), y.reshape(-1))
            loss.backward()
            if fused:
                ops.clip_grad_norm_(params, 0.05)
            else:
                torch.nn.utils.clip_grad_norm_(params, 0.05)
            pre.step()
            opt.step()
        results.append([p.grad.clone() for p in params] + [loss.detach()])
    for a, b in zip(*results):
        close(a, b, 2.0 ** -7)


@devices
def test_trust_region_is_the_layerwise_one(device, single_process_comm):
    """The same preconditioned updates through both ways of writing them,
    with convolutions (grouped too), biases and without."""
    torch.manual_seed(1)
    model = torch.nn.Sequential(
        torch.nn.Conv2d(3, 8, 3, bias=False), torch.nn.ReLU(),
        torch.nn.Conv2d(8, 8, 3, groups=2), torch.nn.Flatten(),
        torch.nn.Linear(8 * 16, 5)).to(device)
    pre = kfac.KFAC_EIGEN_DP(model, lr=0.5, damping=0.01, kl_clip=1e-3)
    x = torch.randn(4, 3, 8, 8, device=device)
    model(x).square().sum().backward()
    raw = [p.grad.clone() for p in model.parameters()]
    pre.step()
    first = [p.grad.clone() for p in model.parameters()]
    for p, g in zip(model.parameters(), raw):
        p.grad.copy_(g)
    pre._one_pass_update = lambda grads, updates: False
    pre._update_grad_in_place()
    for p, g in zip(model.parameters(), first):
        # nu's sum is in another precision: 2^-20, and two roundings
        close(g, p.grad, 2.0 ** -19)


def test_hooked_projection_is_refused(single_process_comm):
    model, x, y = lstm("cpu")
    pre = kfac.KFAC_INV_DP(model, damping=0.01)
    with pytest.raises(RuntimeError, match="exclude_vocabulary_size"):
        model(x, targets=y)
    assert len(pre.modules) == 1


def test_trainers_run_fused():
    from tests.test_examples import run_example
    for script, extra in (
            ("examples/train_wikitext_rnn.py",
             ["--vocab-size", "300", "--bptt", "8"]),
            ("examples/train_transformer.py",
             ["--vocab-size", "120", "--layers", "1", "--d-model", "32"])):
        out = run_example(script, extra + [
            "--batch-size", "4", "--iters-per-epoch", "2", "--epochs", "1",
            "--speed", "--display", "1", "--fused-loss", "--clip-grad",
            "0.25"])
        assert "images/s" in out


def test_wikitext_trainer_takes_the_same_loss_fused(monkeypatch):
    """Both ways of the trainer on the same batches, dropout and all: the
    mean loss and the last step's gradients.  Sums of 32 products and losses
    of 32 tokens, in fp32."""
    import sys

    import kfac_pytorch_amd.parallel.comm as comm_mod
    from examples import train_wikitext_rnn as trainer
    from tests.conftest import free_port
    got = []

    def loop(model, *args, **kw):
        loss, times = real(model, *args, **kw)
        got.append([torch.as_tensor(float(loss))]
                   + [p.grad.clone() for p in model.parameters()])
        return loss, times

    real = trainer.train_loop
    monkeypatch.setattr(trainer, "train_loop", loop)
    for name, value in [("RANK", "0"), ("WORLD_SIZE", "1"),
                        ("LOCAL_RANK", "0"), ("MASTER_ADDR", "127.0.0.1")]:
        monkeypatch.setenv(name, value)
    if torch.distributed.is_initialized():
        torch.distributed.destroy_process_group()
    for extra in ([], ["--fused-loss"]):
        monkeypatch.setenv("MASTER_PORT", str(free_port()))
        monkeypatch.setattr(sys, "argv", [
            "train_wikitext_rnn.py", "--vocab-size", "90", "--bptt", "8",
            "--emb", "32", "--hidden", "32", "--batch-size", "4",
            "--iters-per-epoch", "3", "--epochs", "1", *extra])
        comm_mod.reset()
        trainer.main()
        comm_mod.reset()
    assert len(got) == 2
    for a, b in zip(*got):
        close(b, a, REL)


class Adapted(torch.nn.Linear):
    def forward(self, x):
        return super().forward(x) * 0.5


class Counted(torch.nn.Linear):
    def __call__(self, x):
        return super().__call__(x) + 1


@pytest.mark.parametrize("kind", ["subclass", "call", "instance", "other",
                                  "global pre", "global", "global backward"])
def test_projection_that_is_more_than_linear_is_refused(kind):
    """model(x, targets=y) must not be the loss of another model than
    model(x) is."""
    from torch.nn.modules import module as hooks
    model, x, y = lstm("cpu")
    d, handle = model.decoder, None
    if kind in ("subclass", "call"):
        d = (Adapted if kind == "subclass" else Counted)(32, VOCAB)
        d.load_state_dict(model.decoder.state_dict())
    elif kind == "instance":
        d.forward = lambda x: F.linear(x, d.weight) * 2
    elif kind == "other":
        class Head(torch.nn.Module):
            def __init__(self):
                super().__init__()
                self.weight, self.bias = model.decoder.weight, None
                self.out_features = VOCAB

            def forward(self, x):
                return F.linear(x, self.weight).tanh()
        d = Head()
    elif kind == "global pre":
        handle = hooks.register_module_forward_pre_hook(lambda m, a: None)
    elif kind == "global":
        handle = hooks.register_module_forward_hook(lambda m, a, o: None)
    else:
        handle = hooks.register_module_full_backward_hook(
            lambda m, a, o: None)
    model.decoder = d
    try:
        with pytest.raises(RuntimeError, match="loss without logits|loss "
                                               "from the logits"):
            ops.projection_loss(d, torch.randn(4, 32), y[0, :4])
        with pytest.raises(RuntimeError, match="from the logits"):
            model(x, targets=y)
    finally:
        if handle is not None:
            handle.remove()


def test_projections_that_are_linear_are_taken():
    """Parametrised, subclassed without another forward pass, compiled: the
    loss is that of the layer's own output."""
    from torch.nn.utils import parametrize

    class Named(torch.nn.Linear):
        pass

    class Half(torch.nn.Module):
        def forward(self, w):
            return w / 2

    torch.manual_seed(0)
    x, t = torch.randn(6, 16), torch.randint(20, (6,))
    layers = [torch.nn.Linear(16, 20), Named(16, 20, bias=False),
              torch.nn.Linear(16, 20)]
    parametrize.register_parametrization(layers[2], "weight", Half())
    layers.append(torch.compile(torch.nn.Linear(16, 20), backend="eager"))
    for layer in layers:
        plain = getattr(layer, "_orig_mod", layer)
        want = F.cross_entropy(plain(x), t)
        close(ops.projection_loss(layer, x, t), want, REL)


@devices
def test_learning_rate_in_a_tensor_is_not_waited_for(device, monkeypatch,
                                                     single_process_comm):
    """It goes the layer-by-layer way, which leaves it on the device; the
    result is the same."""
    from kfac_pytorch_amd.ops import grad_scale
    calls = []
    real = grad_scale.kl_clip
    monkeypatch.setattr(grad_scale, "kl_clip",
                        lambda *a, **kw: calls.append(1) or real(*a, **kw))
    got = []
    for lr in (0.5, torch.tensor(0.5, device=device)):
        torch.manual_seed(1)
        model = torch.nn.Linear(16, 5).to(device)
        pre = kfac.KFAC_EIGEN_DP(model, lr=0.5, damping=0.01, kl_clip=1e-3)
        pre._one_pass_update = lambda grads, updates: True
        pre.param_groups[0]["lr"] = lr
        model(torch.randn(4, 16, device=device)).square().sum().backward()
        pre.step()
        got.append([p.grad.clone() for p in model.parameters()])
        assert len(calls) == 1
    for a, b in zip(*got):
        close(b, a, 2.0 ** -19)


@devices
def test_lstm_leaves_out_any_padding_number(device):
    model, x, y = lstm(device)
    pad = VOCAB - 1
    y[y == pad] = 0
    want, _ = model(x, targets=y)
    y[y == -100] = pad
    got, _ = model(x, targets=y, ignore_index=pad)
    assert torch.equal(got, want)
    assert not torch.equal(got, model(x, targets=y)[0])


def test_transformer_smoothing_up_to_uniform():
    """1 - 1 / V makes all tokens alike; more raises, as a label smoothing
    past 1 does."""
    torch.manual_seed(0)
    model = make_transformer(vocab=20, d_model=16, nhead=2, num_layers=1,
                             dim_ff=16, max_len=8, dropout=0.0)
    src, trg = torch.randint(20, (2, 5)), torch.randint(20, (2, 5))
    loss = model(src, trg[:, :-1], targets=trg[:, 1:], smoothing=0.95)
    want = LabelSmoothLoss(0.95)(model(src, trg[:, :-1]).reshape(-1, 20),
                                 trg[:, 1:].reshape(-1))
    close(loss, want, REL)
    with pytest.raises(ValueError):
        model(src, trg[:, :-1], targets=trg[:, 1:], smoothing=0.97)
