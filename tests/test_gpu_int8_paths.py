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
