"""GPU: linear layers and 1x1 convolutions in 8-bit integers against their formulas in 64 bits (tests/int8_ref.py)."""
import importlib

import numpy as np
import pytest
import torch

import int8_ref as ref
from conftest import load_pkg

pytestmark = pytest.mark.gpu

pkg = load_pkg()
callers = importlib.import_module("semantic-segmentation_amd.callers")
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _np(t):
    return t.detach().float().cpu().numpy()


def _make(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g) * 0.5)).to(dtype).to(DEV)


def _weights(n, k, seed, bias=True):
    g = torch.Generator().manual_seed(1000 + seed)
    wq = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8).to(DEV)
    return wq, (torch.rand(n, generator=g) * 0.01 + 1e-4).to(DEV), torch.randn(n, generator=g).to(DEV) if bias else None


def _close(y, want, tol, dtype):
    """y in `dtype` against float64: one rounding to the type on top of what float32 may be off by."""
    half = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    tol = tol + half * (np.abs(want) + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    top = torch.finfo(dtype).max
    got, fine = _np(y).astype(np.float64), np.abs(want) < top * 0.99
    assert (np.abs(got - want)[fine] <= tol[fine]).all(), np.max((np.abs(got - want) - tol)[fine])
    assert fine.mean() > 0.99 or not np.isfinite(want).all()


def _tokens(x):
    """[n, c, h, w] -> [n * h * w, c]"""
    return np.moveaxis(_np(x), 1, 3).reshape(-1, x.shape[1])


def _map(y, n, h, w):
    return np.moveaxis(y.reshape(n, h, w, -1), 3, 1)


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (3, 16), (16, 5), (64, 64), (65, 63), (100, 200), (128, 130), (129, 17), (1000, 98)])
def test_linear_over_sizes(tokens, k, n):
    x = _make((tokens, k), torch.float32, tokens + k)
    wq, ws, b = _weights(n, k, n)
    want, tol = ref.product(_np(x), _np(wq), _np(ws), _np(b))
    _close(pkg.int8_linear(x, wq, ws, b), want, tol, torch.float32)


@pytest.mark.parametrize("tokens,k", [(1030, 40), (1100, 100), (1029, 300), (1100, 1000), (1101, 1500), (2051, 2048), (1100, 3000), (1025, 4100)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shift", [0, 1])
def test_many_tokens_of_any_length(tokens, k, dtype, shift):
    """Rows rounded by a part of a wave, a wave and several, at aligned and other addresses."""
    x = _make((tokens, k + shift), TYPES[dtype], k)[:, shift:]
    wq, ws, b = _weights(70, k, 3)
    want, tol = ref.product(_np(x), _np(wq), _np(ws), _np(b))
    _close(pkg.int8_linear(x, wq, ws, b, out_dtype=torch.float32), want, tol, torch.float32)
    q, s = pkg.quantize_int8(x)
    wq_, ws_ = ref.quantize(_np(x))
    assert np.array_equal(_np(q), wq_) and np.array_equal(_np(s), ws_)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("out", sorted(TYPES))
@pytest.mark.parametrize("tokens,k,n", [(1, 500, 96), (9, 12544, 40), (77, 500, 96), (700, 256, 520)])
def test_linear_over_types(dtype, out, tokens, k, n):
    x = _make((tokens, k), TYPES[dtype], 5)
    wq, ws, b = _weights(n, k, 6)
    for bias, relu in ((None, False), (b, True), (b.to(TYPES[dtype]), False)):
        want, tol = ref.product(_np(x), _np(wq), _np(ws), None if bias is None else _np(bias), relu)
        y = pkg.int8_linear(x, wq, ws, bias, relu=relu, out_dtype=TYPES[out])
        assert y.dtype == TYPES[out]
        _close(y, want, tol, TYPES[out])


@pytest.mark.parametrize("tokens,k,n", [(17, 4096, 64), (70, 4097, 33), (65, 4112, 200), (300, 12544, 130), (64, 9999, 257), (130, 5136, 70),
                                        (600, 2048, 100), (1000, 6000, 700), (513, 1040, 65), (20, 1300, 13000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nchw", [False, True])
def test_long_sums_over_few_tokens(tokens, k, n, dtype, nchw):
    """K split between workgroups, with ends that are no whole turn; the tokens as rows, and as the pixels of a map."""
    x = _make((tokens, k), TYPES[dtype], k + n)
    wq, ws, b = _weights(n, k, n)
    want, tol = ref.product(_np(x), _np(wq), _np(ws), _np(b))
    y = pkg.int8_conv1x1(x.t().contiguous().view(1, k, 1, tokens), wq, ws, b).view(n, tokens).t() if nchw else pkg.int8_linear(x, wq, ws, b)
    _close(y, want, tol, TYPES[dtype])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("images,c,co,h,w", [(1, 3, 64, 7, 5), (2, 64, 64, 9, 11), (1, 130, 40, 1, 1), (3, 17, 3, 13, 1),
                                             (2, 256, 300, 16, 17), (1, 1000, 19, 5, 70), (4, 1, 2, 3, 3)])
@pytest.mark.parametrize("stride", [1, 2, 3])
@pytest.mark.parametrize("layout", ["nchw", "nhwc", "slice"])
def test_conv_over_sizes_strides_and_layouts(dtype, images, c, co, h, w, stride, layout):
    x = _make((images, h, w, c), TYPES[dtype], h + c).permute(0, 3, 1, 2)
    if layout == "nchw":
        x = x.contiguous()
    elif layout == "slice":          # a crop of a larger map: no two dimensions join
        big = torch.zeros((images, c + 1, h + 3, w + 2), dtype=x.dtype, device=DEV)
        big[:, 1:, 2:2 + h, 1:1 + w] = x
        x = big[:, 1:, 2:2 + h, 1:1 + w]
    wq, ws, b = _weights(co, c, co)
    xs = x[:, :, ::stride, ::stride]
    want, tol = ref.product(_tokens(xs), _np(wq), _np(ws), _np(b), True)
    y = pkg.int8_conv1x1(x, wq, ws, b, stride=stride, relu=True)
    shape = (images, co) + tuple(xs.shape[2:])
    assert y.shape == shape and y.dtype == x.dtype
    if layout == "nhwc" and c > 1:
        assert y.is_contiguous(memory_format=torch.channels_last)
    elif layout == "nchw" and h * w > 1:
        assert y.is_contiguous()
    _close(y, _map(want, *[shape[i] for i in (0, 2, 3)]), _map(tol, *[shape[i] for i in (0, 2, 3)]), x.dtype)


@pytest.mark.parametrize("rows,k", [(1, 1), (5, 3), (64, 65), (7, 4097), (300, 128)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_quantize_bit_by_bit(rows, k, dtype):
    x = _make((rows, k), TYPES[dtype], rows)
    x[0] = 0
    q, s = pkg.quantize_int8(x)
    eq, es = ref.quantize(_np(x))
    assert q.shape == (rows, k) and np.array_equal(q.cpu().numpy(), eq) and np.array_equal(_np(s), es)
    q2, s2 = pkg.quantize_int8(x.t().contiguous().t())          # another stride
    assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.parametrize("tokens", [2, 40, 200])
def test_tokens_of_zeros_tiny_values_and_values_that_are_not_finite(tokens):
    x = _make((tokens, 200), torch.float32, 3)
    x[0] = 0
    x[1] = 1e-38
    if tokens > 2:
        x[5, 7], x[9, 0], x[11, 199] = float("nan"), float("inf"), -float("inf")
        x[13] = 3e38
        x[14] = float("nan")
    wq, ws, b = _weights(70, 200, 4)
    want, tol = ref.product(_np(x), _np(wq), _np(ws), _np(b))
    y = pkg.int8_linear(x, wq, ws, b, relu=False)
    bad = [5, 9, 11, 14] if tokens > 2 else []
    good = [i for i in range(tokens) if i not in bad and i != 13]
    assert all(torch.isnan(y[i]).all() for i in bad)
    _close(y[good], want[good], tol[good], torch.float32)
    assert torch.equal(y[0], b)
    if tokens > 2:        # relu keeps a NaN; a map's pixels are tokens alike
        assert torch.isnan(pkg.int8_linear(x, wq, ws, b, relu=True)[5]).all()
        z = pkg.int8_conv1x1(x.t().contiguous().view(1, 200, tokens, 1), wq, ws, b)
        assert all(torch.isnan(z[0, :, i]).all() for i in bad)
        assert torch.equal(z[0, :, good, 0].t(), y[good])


def test_extreme_codes_and_the_longest_token():
    """k = 131072 with every product at its largest: the sum is 127 * 128 * k = 2130706432 < 2^31."""
    k = 131072
    x = torch.ones((3, k), device=DEV)
    x[1] = -1
    wq = torch.full((5, k), -128, dtype=torch.int8, device=DEV)
    ws = torch.ones(5, device=DEV)
    want, tol = ref.product(_np(x), _np(wq), _np(ws))
    _close(pkg.int8_linear(x, wq, ws), want, tol, torch.float32)
    assert float(pkg.int8_linear(x, wq, ws)[1, 0]) == pytest.approx(131072 * 128, rel=1e-6)
    with pytest.raises(RuntimeError, match="outside"):
        pkg.int8_linear(torch.ones((1, k + 1), device=DEV), torch.zeros((2, k + 1), dtype=torch.int8, device=DEV), ws[:2])


@pytest.mark.parametrize("tokens", [1, 20, 150])
def test_weights_of_any_alignment_and_strided_rows_of_input(tokens):
    k, n = 160, 70
    x = _make((tokens, k + 9), torch.bfloat16, 8)
    wide, ws, b = _weights(n, k + 33, 9)
    for start in (0, 1, 16, 33):
        wq = wide[:, start:start + k]                 # rows 193 bytes apart, from an odd address on
        want, tol = ref.product(_np(x[:, 9:]), _np(wq), _np(ws), _np(b))
        _close(pkg.int8_linear(x[:, 9:], wq, ws, b), want, tol, torch.bfloat16)
    wq = wide[:, :k].t().contiguous().t()             # rows that are columns in memory
    want, tol = ref.product(_np(x[:, :k]), _np(wq), _np(ws), _np(b))
    _close(pkg.int8_linear(x[:, :k], wq, ws, b), want, tol, torch.bfloat16)
    flat = torch.zeros(n * k + 16, dtype=torch.int8, device=DEV)
    odd = flat[3:3 + n * k].view(n, k)                # contiguous, 3 bytes off
    odd.copy_(wq)
    _close(pkg.int8_linear(x[:, :k], odd, ws, b), want, tol, torch.bfloat16)


def test_nothing_is_written_beside_the_output():
    """Output tensors inside larger ones, through the C entry point: what lies around them stays."""
    _lib = importlib.import_module("semantic-segmentation_amd.dcn._lib")
    L = _lib.lib()
    for images, c, co, h, w, nchw in ((2, 70, 33, 5, 7, 1), (1, 300, 129, 1, 1, 0), (1, 64, 65, 9, 30, 0), (3, 256, 260, 20, 21, 1)):
        x = _make((images, c, h, w), torch.float32, c)
        wq, ws, b = _weights(co, c, c)
        big = torch.full((64 + images * co * h * w + 64,), 7.5, device=DEV)
        s = x.stride()
        if not nchw:
            x = x.contiguous(memory_format=torch.channels_last)
            s = (c * h * w, 1, c * w, c)
        g = _lib.Int8Geom(images, h, w, c, co, nchw, 0, 0, 0, s[0], s[2], s[3], s[1], c)
        size = L.ddcn_int8_workspace_bytes(g)
        work = torch.full((size + 256,), 77, dtype=torch.uint8, device=DEV)
        _lib.check(L.ddcn_int8_product(_lib.ptr(x), _lib.ptr(wq), _lib.ptr(ws), _lib.ptr(b), _lib.ptr(big[64:]),
                                       _lib.ptr(work), size, g, _lib.current_stream(x.device)))
        assert (big[:64] == 7.5).all() and (big[-64:] == 7.5).all() and (work[size:] == 77).all()
        want, tol = ref.product(_tokens(x), _np(wq), _np(ws), _np(b))
        y = big[64:-64].view(images, co, h, w) if nchw else big[64:-64].view(images, h, w, co).permute(0, 3, 1, 2)
        _close(y, _map(want, images, h, w), _map(tol, images, h, w), torch.float32)


def test_empty_calls_and_refusals():
    wq, ws, b = _weights(6, 8, 1)
    assert pkg.int8_linear(torch.zeros((0, 8), device=DEV), wq, ws, b).shape == (0, 6)
    assert pkg.int8_linear(torch.zeros((3, 0, 8), device=DEV), wq, ws, b).shape == (3, 0, 6)
    assert pkg.int8_conv1x1(torch.zeros((0, 8, 4, 4), device=DEV), wq, ws, b).shape == (0, 6, 4, 4)
    assert pkg.int8_linear(torch.zeros(8, device=DEV), wq, ws, b).shape == (6,)
    x = torch.zeros((3, 8), device=DEV)
    for kw in (dict(weight_q=wq.float()), dict(weight_q=wq[:, :7]), dict(weight_scale=ws[:5]), dict(weight_scale=ws.half()),
               dict(bias=b[:5]), dict(bias=b.int()), dict(out_dtype=torch.float64), dict(input=x.double()),
               dict(input=x.clone().requires_grad_())):
        args = dict(input=x, weight_q=wq, weight_scale=ws, bias=b)
        args.update(kw)
        with pytest.raises(RuntimeError):
            pkg.int8_linear(**args)
    for kw in (dict(weight_q=wq.cpu()), dict(bias=b.cpu())):
        with pytest.raises(NotImplementedError):
            pkg.int8_linear(**dict(dict(input=x, weight_q=wq, weight_scale=ws, bias=b), **kw))
    with pytest.raises(RuntimeError, match="4D"):
        pkg.int8_conv1x1(x, wq, ws)
    for stride in (0, -1, 1.5):
        with pytest.raises(RuntimeError, match="stride"):
            pkg.int8_conv1x1(torch.zeros((1, 8, 2, 2), device=DEV), wq, ws, stride=stride)
    with torch.no_grad():
        pkg.int8_linear(x.clone().requires_grad_(), wq, ws)


@pytest.mark.parametrize("tokens,k,n", [(1, 12544, 1024), (5, 700, 130), (200, 1024, 300), (1500, 256, 256)])
def test_graph_replays_with_new_inputs(tokens, k, n):
    x = _make((tokens, k), torch.bfloat16, 2)
    wq, ws, b = _weights(n, k, 3)
    pkg.int8_linear(x, wq, ws, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pkg.int8_linear(x, wq, ws, b)
        z = pkg.int8_linear(x, wq, ws, None)      # a second call with a workspace of its own
    for i in range(4):
        x.copy_(_make((tokens, k), torch.bfloat16, 50 + i))
        eager = pkg.int8_linear(x, wq, ws, b)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager) and torch.equal(z, pkg.int8_linear(x, wq, ws, None))


def test_two_streams_at_once():
    wq, ws, b = _weights(1024, 12544, 3)
    xs = [_make((t, 12544), torch.bfloat16, t) for t in (1, 40)]
    want = [pkg.int8_linear(x, wq, ws, b) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(20):
        for s, x, l in zip(streams, xs, got):
            with torch.cuda.stream(s):
                l.append(pkg.int8_linear(x, wq, ws, b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for l, w in zip(got, want) for y in l)


def test_layers_from_float_ones():
    torch.manual_seed(0)
    lin = torch.nn.Linear(96, 40).to(DEV)
    x = _make((33, 96), torch.float32, 1)
    layer = pkg.Int8Linear.from_float(lin, relu=True)
    q, s = ref.quantize(_np(lin.weight))
    want, tol = ref.product(_np(x), q, s, _np(lin.bias), True)
    _close(layer(x), want, tol, torch.float32)
    conv, norm = torch.nn.Conv2d(24, 50, 1, stride=2).to(DEV), torch.nn.BatchNorm2d(50).to(DEV).eval()
    with torch.no_grad():
        norm.running_mean.normal_(), norm.running_var.uniform_(0.5, 2), norm.weight.normal_(), norm.bias.normal_()
    x = _make((2, 24, 9, 7), torch.float32, 2)
    layer = pkg.Int8Conv1x1.from_float(conv, norm)
    y, full = _np(layer(x)), _np(norm(conv(x)))
    # codes of 127 steps: a value is off by half a step of its token's or channel's scale, 1/254 of the largest |x| or
    # |w|; 24 such products of both kinds, in the worst case all of one sign
    xs, w = _np(x)[:, :, ::2, ::2], _np(conv.weight)[:, :, 0, 0] * _np(norm.weight * torch.rsqrt(norm.running_var + norm.eps))[:, None]
    bound = 24 / 254 * 2.1 * np.abs(xs).max(1)[:, None] * np.abs(w).max(1)[None, :, None, None]
    assert (np.abs(y - full) <= bound).all()


def test_more_tokens_than_one_pass():
    """2^24 tokens and some: the second pass writes behind the first one's."""
    t, k, n = (1 << 24) + 37, 8, 3
    x = torch.randint(-3, 4, (t, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).to(torch.float16)
    wq, ws, b = _weights(n, k, 5)
    y = pkg.int8_linear(x, wq, ws, b)
    for at in (slice(0, 500), slice((1 << 24) - 200, t)):
        want, tol = ref.product(_np(x[at]), _np(wq), _np(ws), _np(b))
        _close(y[at], want, tol, torch.float16)
    h, images = 1 << 13, 1025                  # images of 2 x 8192: the border between the passes lies inside the last but one
    x = torch.cat([x, x])[:images * 2 * h]
    z = pkg.int8_conv1x1(x.view(images, 2, h, k).permute(0, 3, 1, 2).contiguous(), wq, ws, b).permute(0, 2, 3, 1).reshape(-1, n)
    for at in (slice(0, 500), slice((1 << 24) - 500, (1 << 24) + 500), slice(-500, None)):
        assert torch.equal(z[at], pkg.int8_linear(x[at], wq, ws, b))


def test_passes_of_long_tokens_and_a_pass_that_ends_inside_an_image():
    """Long tokens take a workgroup each: no grid of a pass may reach 2^32 threads.  (All rows of x are one row.)"""
    row = _make((1, 2304), torch.bfloat16, 6)
    wq, ws, b = _weights(2, 2304, 7)
    y = pkg.int8_linear(row.expand((1 << 24) + 5, 2304), wq, ws, b, out_dtype=torch.float32)
    assert (y == pkg.int8_linear(row, wq, ws, b, out_dtype=torch.float32)).all()
    images, h, w, k, n = 3, 4099, 683, 8, 3                # 2^23 tokens end inside the third image
    x = torch.randint(-3, 4, (images, h * w, k), device=DEV, generator=torch.Generator(device=DEV).manual_seed(8)).to(torch.float16)
    wq, ws, b = _weights(n, k, 9)
    z = pkg.int8_conv1x1(x.view(images, h, w, k).permute(0, 3, 1, 2).contiguous(), wq, ws, b).permute(0, 2, 3, 1).reshape(-1, n)
    for at in (slice(0, 500), slice((1 << 23) - 500, (1 << 23) + 500), slice(-500, None)):
        assert torch.equal(z[at], pkg.int8_linear(x.view(-1, k)[at], wq, ws, b))
