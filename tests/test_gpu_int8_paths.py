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


# the tiled product (more than 512 tokens, K too short to be split): 64 x 64 tiles, and 128 x 128 where they fill the CUs
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("off", [0, 1, 5])
@pytest.mark.parametrize("images,h,w,k,n,nchw", [(1, 700, 1, 100, 65, 0), (1, 1500, 1, 64, 129, 0), (1, 1003, 1, 200, 523, 0), (1, 601, 1, 65, 7, 0),
                                                 (1, 12503, 1, 130, 265, 0), (1, 13000, 1, 64, 512, 0),
                                                 (2, 23, 25, 100, 33, 1), (2, 23, 25, 64, 130, 1), (3, 15, 15, 65, 64, 1), (90, 3, 3, 64, 40, 1),
                                                 (700, 1, 1, 64, 40, 1), (2, 97, 97, 64, 130, 1), (2, 97, 97, 200, 256, 1), (5, 61, 67, 64, 129, 1),
                                                 (200, 9, 11, 64, 128, 1), (2, 96, 98, 64, 131, 1)])
def test_stores_of_tiles_at_any_address(images, h, w, k, n, nchw, dtype, off):
    """Rows and planes of odd length, images that end inside a run of eight, outputs from any element on: every element, and
    the memory on both sides."""
    t = TYPES[dtype]
    g = torch.Generator().manual_seed(k + n)
    x = torch.randn((images * h * w, k), generator=g).to(t).to(DEV)
    wq, ws, b = _weights(n, k, n)
    total, edge = images * h * w * n, 64
    big = torch.full((edge + off + total + edge,), 7.5, dtype=t, device=DEV)
    y = big[edge + off:edge + off + total]
    if nchw:
        x = x.view(images, h * w, k).transpose(1, 2).contiguous()
        geom = _lib.Int8Geom(images, h, w, k, n, 1, _lib.ELEMENT_TYPES[t], _lib.ELEMENT_TYPES[t], 0, k * h * w, w, 1, h * w, k)
    else:
        geom = _lib.Int8Geom(images, h, w, k, n, 0, _lib.ELEMENT_TYPES[t], _lib.ELEMENT_TYPES[t], 0, 0, k, 0, 1, k)
    size = _lib.lib().ddcn_int8_workspace_bytes(geom)
    work = torch.empty(size, dtype=torch.uint8, device=DEV)
    _lib.check(_lib.lib().ddcn_int8_product(_lib.ptr(x), _lib.ptr(wq), _lib.ptr(ws), _lib.ptr(b), _lib.ptr(y), _lib.ptr(work), size, geom,
                                            _lib.stream_of(0)))
    assert (big[:edge + off] == 7.5).all() and (big[edge + off + total:] == 7.5).all()
    tokens = _np(x.transpose(1, 2).reshape(-1, k) if nchw else x)
    want, tol = ref.product(tokens, _np(wq), _np(ws), _np(b))
    half = torch.finfo(t).eps / 2 if t != torch.float32 else 0.0
    tol = tol + half * (np.abs(want) + tol) + (2.0 ** -25 if t == torch.float16 else 0)
    got = _np(y.view(images, n, h * w).transpose(1, 2) if nchw else y).reshape(-1, n)
    assert (np.abs(got - want) <= tol).all(), np.argwhere(~(np.abs(got - want) <= tol))[:10]
