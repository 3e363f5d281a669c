"""GPU: calls of the 8-bit layers beside the plain ones: sizes that do not fit, gradients asked for, the tiled product's stores at
odd addresses (tests/int8_ref.py)."""
import importlib

import numpy as np
import pytest
import torch

import int8_ref as ref
from conftest import load_pkg

pytestmark = pytest.mark.gpu

pkg = load_pkg()
callers = importlib.import_module("semantic-segmentation_amd.callers")
_lib = importlib.import_module("semantic-segmentation_amd.dcn._lib")
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _np(t):
    return t.detach().float().cpu().numpy()


def _weights(n, k, seed):
    g = torch.Generator().manual_seed(1000 + seed)
    wq = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(DEV)
    return wq, (torch.rand(n, generator=g) * 0.01 + 1e-4).to(DEV), torch.randn(n, generator=g).to(DEV)


def test_sizes_that_32_bits_do_not_hold_are_refused():
    """Before anything is allocated: 2^32 + 5 rows would be 5 in an int.  (Expanded tensors: they take no memory.)"""
    far = (1 << 32) + 5
    wq, ws, b = _weights(6, 8, 1)
    row, byte, one = torch.ones((1, 8), device=DEV), torch.ones((1, 1), dtype=torch.int8, device=DEV), torch.ones(1, device=DEV)
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    for call in (lambda: pkg.int8_linear(row.expand(far, 8), wq, ws, b),
                 lambda: pkg.int8_linear(row.expand(2, 1 << 31, 8), wq, ws, b),
                 lambda: pkg.int8_linear(row.expand(1 << 31, 8), wq, ws, b),
                 lambda: pkg.int8_linear(row[:, :1].expand(1, far), byte.expand(1, far), one),
                 lambda: pkg.int8_linear(row, byte.expand(far, 8), one.expand(far)),
                 lambda: pkg.quantize_int8(row.expand(far, 8)),
                 lambda: pkg.quantize_int8(row[:, :1].expand(1, far)),
                 lambda: pkg.int8_conv1x1(row.view(1, 8, 1, 1).expand(far, 8, 1, 1), wq, ws, b),
                 lambda: pkg.int8_conv1x1(row.view(1, 8, 1, 1).expand(1, 8, far, 1), wq, ws, b),
                 lambda: pkg.int8_conv1x1(row.view(1, 8, 1, 1).expand(1, 8, 1 << 16, 1 << 16), wq, ws, b),
                 lambda: pkg.int8_conv1x1(row[:, :1].view(1, 1, 1, 1).expand(1, far, 1, 1), byte.expand(1, far), one)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            call()
    assert torch.cuda.max_memory_allocated() == before
    y = pkg.int8_conv1x1(row.view(1, 8, 1, 1).expand(1, 8, far, 1), wq, ws, b, stride=far)       # one pixel of it
    assert torch.equal(y.view(6), pkg.int8_linear(row, wq, ws, b).view(6))


def test_gradients_asked_for_are_refused_not_dropped():
    """There is no backward pass: whatever requires a gradient, and forward-mode tangents."""
    from torch.autograd import forward_ad
    wq, ws, b = _weights(6, 8, 1)
    x = torch.randn((3, 8), device=DEV)
    image = torch.randn((1, 8, 2, 2), device=DEV)
    ask = lambda t: t.clone().requires_grad_()                                                     # noqa: E731
    for call in (lambda x, i, ws, b: pkg.int8_linear(x, wq, ws, b), lambda x, i, ws, b: pkg.int8_conv1x1(i, wq, ws, b)):
        for args in ((ask(x), ask(image), ws, b), (x, image, ask(ws), b), (x, image, ws, ask(b))):
            with pytest.raises(RuntimeError, match="no backward"):
                call(*args)
            with torch.no_grad():
                call(*args)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))                               # noqa: E731
        for grad in (True, False):               # (no_grad does not stop forward mode)
            with torch.set_grad_enabled(grad):
                for call in (lambda: pkg.int8_linear(dual(x), wq, ws, b), lambda: pkg.int8_linear(x, wq, dual(ws), b),
                             lambda: pkg.int8_linear(x, wq, ws, dual(b)), lambda: pkg.int8_conv1x1(dual(image), wq, ws, b),
                             lambda: pkg.quantize_int8(dual(x))):
                    with pytest.raises(RuntimeError, match="no backward"):
                        call()
                pkg.int8_linear(x, wq, ws, b)
