"""CPU: which layers `int8_inference` converts, with the two 8-bit calls replaced by plain ones over the rounded weights."""
import importlib
from collections import OrderedDict

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import int8_ref as ref
from conftest import load_pkg

pkg = load_pkg()
callers = importlib.import_module("semantic-segmentation_amd.callers")
int8 = importlib.import_module("semantic-segmentation_amd.dcn.int8")


@pytest.fixture
def on_cpu(monkeypatch):
    def quantize(w):
        q, s = ref.quantize(w.detach().numpy())
        return torch.from_numpy(q).to(torch.int8), torch.from_numpy(s)

    def weights(wq, ws):
        return wq.float() * ws[:, None]

    def linear(x, wq, ws, b, relu):
        y = F.linear(x, weights(wq, ws), b)
        return y.relu() if relu else y

    def conv(x, wq, ws, b, stride, relu):
        y = F.conv2d(x, weights(wq, ws)[:, :, None, None], b, stride)
        return y.relu() if relu else y

    for name, f in (("quantize_int8", quantize), ("int8_linear", linear), ("int8_conv1x1", conv)):
        monkeypatch.setattr(int8, name, f)


def _fill_norms(model, seed=0):
    torch.manual_seed(seed)
    with torch.no_grad():
        for m in model.modules():
            if isinstance(m, nn.BatchNorm2d):
                m.running_mean.normal_(), m.running_var.uniform_(0.5, 2), m.weight.normal_(), m.bias.normal_()
    return model.eval()


def _off_by_rounded_weights(before, after, x, w):
    """A product whose weights are off by half a code, 1/254 of a channel's largest, and float32 on top (64 additions)."""
    w = w.detach().flatten(1)
    most = x.abs().sum(1, keepdim=True) * (w.abs().amax(1) / 254)[None, :, None, None]
    return ((before - after).abs() <= most * 1.01 + 2.0 ** -18 * (1 + before.abs())).all()


class Preactivated(nn.Sequential):
    """Registered in another order than it runs."""

    def forward(self, x):
        return self.conv(F.relu(self.norm(x)))


class Taps(nn.Sequential):
    def forward(self, x):
        a = self[0](x)
        return a, self[1](a), self[2](self[1](a))


def test_sequences_that_do_not_run_as_one_are_not_folded(on_cpu):
    """A Sequential with a forward of its own keeps its norms and activations; its layers are converted one by one."""
    model = _fill_norms(Preactivated(OrderedDict(conv=nn.Conv2d(32, 32, 1), norm=nn.BatchNorm2d(32), relu=nn.ReLU())))
    x = torch.randn(2, 32, 5, 6)
    with torch.no_grad():
        want, weight, inner = model(x), model.conv.weight, F.relu(model.norm(x))
        callers.int8_inference(model)
        got = model(x)
    assert type(model.conv).__name__ == "Int8Conv1x1" and isinstance(model.norm, nn.BatchNorm2d) and isinstance(model.relu, nn.ReLU)
    assert not model.conv.relu and _off_by_rounded_weights(want, got, inner, weight)
    taps = _fill_norms(Taps(nn.Conv2d(32, 32, 1), nn.BatchNorm2d(32), nn.ReLU()))
    with torch.no_grad():
        want, weight = taps(x), taps[0].weight
        got = callers.int8_inference(taps)(x)
    assert _off_by_rounded_weights(want[0], got[0], x, weight) and isinstance(taps[1], nn.BatchNorm2d)


def test_a_bottleneck_with_a_forward_of_its_own_is_not_folded(on_cpu):
    class Block(callers.Bottleneck):
        def forward(self, x):
            return self.bn1(self.conv1(self.relu(x)))

    block = _fill_norms(Block(64, 16))
    x = torch.randn(1, 64, 3, 4)
    with torch.no_grad():
        inner, weight, scale = F.relu(x), block.conv1.weight, (block.bn1.weight * torch.rsqrt(block.bn1.running_var + block.bn1.eps))
        want = block(x)
        callers.int8_inference(block)
        got = block(x)
    assert type(block.conv1).__name__ == "Int8Conv1x1" and isinstance(block.bn1, nn.BatchNorm2d) and block.relu1
    assert _off_by_rounded_weights(want, got, inner, weight * scale[:, None, None, None])


def test_plain_sequences_and_bottlenecks_are_folded(on_cpu):
    seq = _fill_norms(nn.Sequential(nn.Conv2d(32, 16, 1), nn.BatchNorm2d(16), nn.ReLU(), nn.Conv2d(16, 8, 1), nn.ReLU()))
    block = _fill_norms(callers.Bottleneck(64, 16))
    callers.int8_inference(seq), callers.int8_inference(block)
    assert [type(m).__name__ for m in seq] == ["Int8Conv1x1", "Identity", "Identity", "Int8Conv1x1", "Identity"]
    assert seq[0].relu and seq[3].relu and isinstance(block.bn1, nn.Identity) and not block.relu1


def test_layers_with_hooks_stay_as_they_are(on_cpu):
    """A hook sees the layer that it was put on: neither is it dropped with the layer, nor does a norm or an activation
    that has one vanish into the layer before it."""
    seen = []
    hook = lambda m, *rest: seen.append(m)                                                         # noqa: E731
    kinds = (lambda m: m.register_forward_hook(hook), lambda m: m.register_forward_pre_hook(hook),
             lambda m: m.register_full_backward_hook(hook), lambda m: m.register_full_backward_pre_hook(hook))
    x = torch.randn(1, 32, 2, 2)
    for put in kinds:
        for at in range(4):
            seq = _fill_norms(nn.Sequential(nn.Conv2d(32, 32, 1), nn.BatchNorm2d(32), nn.ReLU(), nn.Conv2d(32, 16, 1)))
            layer = seq[at]
            put(layer)
            callers.int8_inference(seq)
            assert seq[at] is layer
            names = [type(m).__name__ for m in seq]
            assert names == [["Conv2d", "BatchNorm2d", "ReLU", "Int8Conv1x1"], ["Int8Conv1x1", "BatchNorm2d", "ReLU", "Int8Conv1x1"],
                             ["Int8Conv1x1", "Identity", "ReLU", "Int8Conv1x1"], ["Int8Conv1x1", "Identity", "Identity", "Conv2d"]][at]
            assert seq[0].relu is (at == 3) if at else True
    for name in ("conv1", "bn1", "conv3", "bn3"):
        block = _fill_norms(callers.Bottleneck(64, 16))
        layer = getattr(block, name)
        layer.register_forward_hook(hook)
        callers.int8_inference(block)
        assert getattr(block, name) is layer
        other = "conv3" if name in ("conv1", "bn1") else "conv1"
        assert type(getattr(block, other)).__name__ == "Int8Conv1x1" and type(getattr(block, "conv" + name[-1])) is nn.Conv2d
        assert block.relu1 is (name in ("conv1", "bn1"))
    # weights that a hook makes anew before every call
    linear = torch.nn.utils.spectral_norm(nn.Linear(32, 8))
    model = nn.ModuleDict(dict(fc=linear, other=nn.Linear(32, 8), last=nn.Conv2d(32, 8, 1))).eval()
    model.last.forward = lambda x: x
    callers.int8_inference(model)
    assert model.fc is linear and type(model.other).__name__ == "Int8Linear" and type(model.last) is nn.Conv2d
    alone = nn.Linear(32, 8).eval()
    alone.register_forward_hook(hook)
    assert callers.int8_inference(alone) is alone and x is not None


def test_a_bottleneck_with_another_activation_keeps_it(on_cpu):
    for relu in (nn.ReLU(), nn.SiLU()):
        block = _fill_norms(callers.Bottleneck(64, 16))
        block.relu = relu
        if type(relu) is nn.ReLU:
            relu.register_forward_hook(lambda m, i, o: None)
        callers.int8_inference(block)
        assert block.relu is relu and block.relu1 and not block.conv1.relu and isinstance(block.bn1, nn.Identity)


@pytest.mark.parametrize("make", [lambda: nn.Linear(131073, 4), lambda: nn.Conv2d(131073, 4, 1), lambda: nn.Linear(16, (1 << 20) + 1),
                                  lambda: nn.Conv2d(16, (1 << 20) + 1, 1), lambda: nn.Linear(0, 4)],
                         ids=["inputs", "input channels", "outputs", "output channels", "no inputs"])
def test_layers_that_the_product_does_not_take_stay(on_cpu, make):
    """They were met halfway through a model, after others had been converted."""
    with torch.device("meta"):
        far = make()
    model = nn.Sequential(nn.Linear(32, 8), far).eval()
    callers.int8_inference(model, min_channels=0)
    assert type(model[0]).__name__ == "Int8Linear" and model[1] is far


@pytest.mark.parametrize("make", [lambda: nn.Linear(32, 4), lambda: nn.Conv2d(32, 4, 1)], ids=["linear", "conv"])
def test_double_layers_stay(on_cpu, make):
    model = nn.ModuleList([nn.Linear(32, 8), make().double()]).eval()
    callers.int8_inference(model)
    assert type(model[0]).__name__ == "Int8Linear" and model[1].weight.dtype == torch.float64
    bottleneck = _fill_norms(callers.Bottleneck(64, 16).double())
    layers = list(bottleneck.modules())
    assert list(callers.int8_inference(bottleneck).modules()) == layers
