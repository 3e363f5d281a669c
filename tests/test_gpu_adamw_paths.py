"""GPU: the optimizer over runs of many steps, and calls of the AdamW entry points beside the plain ones (tests/adamw_ref.py)."""
import importlib

import numpy as np
import pytest
import torch

import adamw_ref as ref
from conftest import load_pkg

pytestmark = pytest.mark.gpu

load_pkg()
callers = importlib.import_module("semantic-segmentation_amd.callers")
_lib = importlib.import_module("semantic-segmentation_amd.dcn._lib")
DEV = "cuda:0"
LR, BETAS, EPS, WD = 1e-2, (0.9, 0.99), 1e-8, 0.05


def _rng(seed):
    return torch.Generator().manual_seed(seed)


def _np(t):
    return t.detach().float().cpu().numpy()


def test_8_bit_moments_of_a_parameter_that_is_trained_later():
    """Parameter a alone, then b alone, in one group.  Half of b's gradients drop by ten after its first steps: its second
    moments follow as they do where every step has another seed (the tolerance of the same experiment with given seeds in
    test_gpu_adamw.py: 25 % is 3 sigma)."""
    a, b = (torch.nn.Parameter(torch.zeros(256, device=DEV)) for _ in range(2))
    beta2, k = 0.999, 1500
    opt = callers.AdamW([a, b], lr=0.0, betas=(0.0, 0.0), weight_decay=0.0, bits=8)
    a.grad = torch.ones_like(a)
    for _ in range(k + 20):
        opt.step()
    a.grad, b.grad = None, torch.ones_like(b)
    opt.step()                                   # v = g^2
    opt.param_groups[0]["betas"] = (0.9, beta2)
    b.grad[128:] = 0.1
    for _ in range(k):
        opt.step()
    s = opt.state[b]
    r = callers.adamw_moments(*(s[name].contiguous() for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")))[1].sqrt()
    want = np.sqrt(beta2 ** k + (1 - beta2 ** k) * 0.01)
    assert abs(float(r[:128].mean()) - 1) < 0.02
    assert abs(float(r[128:].mean()) / want - 1) < 0.25, (float(r[128:].mean()), want)


def test_steps_without_a_seed_round_differently():
    """The default: the step number, or the sum of them."""
    def codes(step, **kw):
        p, m, v = torch.zeros(512, device=DEV), torch.zeros(512, dtype=torch.int8, device=DEV), torch.zeros(512, dtype=torch.uint8, device=DEV)
        g = torch.randn(512, generator=_rng(1)).to(DEV)
        callers.adamw_step([p[:256], p[256:]], [g[:256], g[256:]], m, v, step, 0.0, BETAS, EPS, 0.0, torch.zeros(2, device=DEV),
                           torch.zeros(2, device=DEV), **kw)
        return m
    assert torch.equal(codes(5), codes(5, seed=5)) and torch.equal(codes([5, 9]), codes([5, 9], seed=14))
    assert not torch.equal(codes(5), codes(6))


@pytest.mark.parametrize("bits", [32, 8])
def test_weight_decay_below_half_a_step_of_float32(bits):
    """lr wd = 2.5e-8 (lr 2.5e-4, weight decay 1e-4): 1 - lr wd is 1 in float32, but parameters that move anyway are decayed.
    p in [1, 2), gradients of random signs.  After k steps the mean of p, less what p would be without decay (float64 from the
    moments of a float32 run, or from the decoded ones), is -k lr wd mean(p) = -1.5e-5.  Off by: the rounding of p, 2^-23 /
    sqrt(12) a step and element, its mean over n = 2^16 elements and k = 400 steps 2.7e-9; and the float32 arithmetic of the
    update, 16 half steps of 2^-24 of lr max|m^ / sqrt(v^)| (3 at most here) a step, 2.9e-7 if they all had one sign."""
    n, k, lr, wd = 1 << 16, 400, 2.5e-4, 1e-4
    b1, b2 = BETAS
    g = _rng(5)
    p = (1 + torch.rand(n, generator=g)).to(DEV)
    want = p.double()
    m, v = (torch.zeros(n, device=DEV, dtype=t) for t in ((torch.float32,) * 2 if bits == 32 else (torch.int8, torch.uint8)))
    scales = [] if bits == 32 else [torch.zeros(n // 256, device=DEV) for _ in range(2)]
    for t in range(1, k + 1):
        grad = torch.randn(n, generator=g).to(DEV)
        om, ov = (m, v) if bits == 32 else callers.adamw_moments(m, v, *scales)
        om, ov = om.double() * b1 + (1 - b1) * grad.double(), ov.double() * b2 + (1 - b2) * grad.double() ** 2
        update = om / (1 - b1 ** t) / ((ov / (1 - b2 ** t)).sqrt() + EPS)
        assert float(update.abs().max()) < (3 if bits == 32 else 10)
        want = want * (1 - lr * wd) - lr * update
        callers.adamw_step([p], [grad], m, v, t, lr, BETAS, EPS, wd, *scales, **({} if bits == 32 else dict(seed=t)))
    drift, off = k * lr * wd * 1.5, float((p.double() - want).mean())
    assert drift > 1.4e-5 and abs(off) < (3e-7 if bits == 32 else 1e-6), off


def test_step_of_parameters_that_are_not_finite_or_at_the_end_of_the_range():
    """The decay leaves an infinity what it is, with and without weight decay; so does a NaN stay one, alone."""
    top = torch.finfo(torch.float32).max
    p0 = torch.tensor([float("inf"), -float("inf"), float("nan"), top, -top, 0.0, 1e-40, 3.0], device=DEV)
    for lr, wd in ((1e-3, 0.0), (2.5e-4, 1e-4), (1e-2, 0.05), (1.0, 1.0), (1.0, 1.5), (0.0, 0.1)):
        p = p0.clone()
        callers.adamw_step([p], [torch.zeros(8, device=DEV)], torch.zeros(256, device=DEV), torch.zeros(256, device=DEV), 1, lr, BETAS, EPS, wd)
        d = 1 - lr * wd
        want = (p0.double() * d).float()             # (inf * 0 is NaN)
        assert torch.equal(torch.isnan(p), torch.isnan(want)) and torch.equal(p.nan_to_num(7.0), want.nan_to_num(7.0)), (lr, wd, p)


def _launches(params, grads, steps):
    """Kernel nodes of one C call over float32 tensors (captured, not run)."""
    import ctypes
    from array import array
    numels = [p.numel() for p in params]
    n = callers.adamw_arena(params)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    lists = [array("Q", [p.data_ptr() for p in params]), array("Q", [0 if g is None else g.data_ptr() for g in grads]),
             array("q", numels), array("i", steps)]
    hyper = _lib.AdamwHyper(LR, *BETAS, EPS, WD, 0.0, 1, 0, 32, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        rc = _lib.lib().ddcn_adamw_step(len(params), *(ctypes.c_void_p(a.buffer_info()[0]) for a in lists), _lib.ptr(m), _lib.ptr(v),
                                        None, None, None, hyper, _lib.stream_of(0))
    assert rc == 0
    count = ctypes.c_size_t(0)
    assert _lib.lib().hipGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    return count.value


def test_tensors_without_a_gradient_do_not_split_launches():
    """Convolutions between frozen norm layers: their step numbers stay behind, and no launch needs them."""
    sizes = [4096, 64, 64] * 53
    params = [torch.zeros(n, device=DEV) for n in sizes]
    grads = [torch.zeros(n, device=DEV) if i % 3 == 0 else None for i, n in enumerate(sizes)]
    assert _launches(params, grads, [9 if g is not None else 1 for g in grads]) == 1
    assert _launches(params, [torch.zeros_like(p) for p in params], [9] * 159) == 1
    # two step numbers among those that count: a launch where they change
    assert _launches(params[:9], grads[:9], [3, 1, 1, 3, 2, 7, 5, 1, 1]) == 2
    # more blocks in between than a launch is worth
    far = torch.zeros(8193 * 256, device=DEV)
    for n, launches in ((8192, 1), (8193, 2)):
        assert _launches([params[0], far[:n * 256], params[3]], [grads[0], None, grads[3]], [9, 1, 9]) == launches


@pytest.mark.parametrize("bits", [32, 8])
def test_frozen_parameters_between_others_over_steps(bits):
    """Gradients that come and go (None in turn, stale step numbers): every parameter as if it were alone in its own call."""
    sizes = [300, 7, 256, 5000, 64, 64, 2049, 1, 513] * 3
    g = _rng(8)
    start = [torch.randn(n, generator=g).to(DEV) for n in sizes]
    together, alone = [p.clone() for p in start], [p.clone() for p in start]
    types = (torch.float32,) * 2 if bits == 32 else (torch.int8, torch.uint8)
    new = lambda n: [torch.zeros(n, dtype=t, device=DEV) for t in types] + [torch.zeros(n // 256, device=DEV) for _ in range(2)][:0 if bits == 32 else 2]   # noqa: E731
    state, each = new(callers.adamw_arena(start)), [new(callers.adamw_arena([p])) for p in start]
    at = ref.starts_of(sizes)[0]
    steps = [0] * len(sizes)
    for t in range(5):
        grads = [None if i % 3 == 1 or (i + t) % 4 == 0 or (i > 20 and t > 2) else torch.randn(n, generator=g).to(DEV) for i, n in enumerate(sizes)]
        steps = [s + (x is not None) for s, x in zip(steps, grads)]
        seeds = {} if bits == 32 else dict(seed=t)
        before = [[x.clone() for x in s] for s in each]
        callers.adamw_step(together, grads, state[0], state[1], [max(s, 1) for s in steps], LR, BETAS, EPS, WD, *state[2:], **seeds)
        for i, (p, x, s, b) in enumerate(zip(alone, grads, each, before)):
            if x is not None:          # from the moments that the common call found: codes depend on a tensor's place
                callers.adamw_step([p], [x], s[0], s[1], steps[i], LR, BETAS, EPS, WD, *s[2:], **seeds)
            assert torch.equal(together[i], p), (t, i)
            n = -(-sizes[i] // 256) * 256
            now = [state[0][at[i]:at[i] + n], state[1][at[i]:at[i] + n]] + [q[at[i] // 256:(at[i] + n) // 256] for q in state[2:]]
            if bits == 32 or x is None:
                assert all(torch.equal(c, d) for c, d in zip(now, s)), (t, i)
            else:                      # (the scales do not)
                assert all(torch.equal(c, d) for c, d in zip(now[2:], s[2:])), (t, i)
                for c, d in zip(now, s):
                    d.copy_(c)


def test_gradients_of_any_strides_are_measured_and_clipped():
    """What the optimizer takes without max_norm it takes with it: transposed and expanded gradients."""
    g = _rng(12)
    w, x = torch.randn(40, 30, generator=g).to(DEV), torch.randn(30, 40, generator=g).to(DEV).t()
    e = torch.full((1, 1), 0.25, device=DEV).expand(40, 30)
    part = torch.randn(40, 60, generator=g).to(DEV)[:, ::2]
    for grad in (x, e, part):
        assert not grad.is_contiguous()
        norm = callers.grad_norm([grad, None, w])
        assert float(norm) == float(callers.grad_norm([grad.contiguous(), w]))
        exact = np.sqrt((_np(grad).astype(np.float64) ** 2).sum() + (_np(w).astype(np.float64) ** 2).sum())
        assert abs(float(norm) - exact) <= 2.0 ** -24 * exact * (1 + 1e-6)
        params = [torch.nn.Parameter(w.clone()) for _ in range(2)]
        for p, y in zip(params, (grad, grad.contiguous())):
            opt = callers.AdamW([p], lr=LR, max_norm=0.5)
            p.grad = y
            opt.step()
        assert torch.equal(*params) and not torch.equal(params[0], w)


def test_norm_of_strided_gradients_in_a_graph():
    x = torch.randn(300, 200, generator=_rng(13)).to(DEV)
    callers.grad_norm([x.t()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = callers.grad_norm([x.t(), x])
    for k in range(3):
        x.mul_(1.5 + k)
        eager = float(callers.grad_norm([x.t(), x]))
        graph.replay()
        torch.cuda.synchronize()
        assert float(out) == eager


def test_a_model_that_moves_to_the_gpu_after_a_refused_step():
    model = torch.nn.Linear(7, 5)
    opt = callers.AdamW(model.parameters(), lr=LR)
    for p in model.parameters():
        p.grad = torch.ones_like(p)
    with pytest.raises(NotImplementedError):
        opt.step()
    model.to(DEV)
    before = [p.detach().clone() for p in model.parameters()]
    opt.step()
    assert all((p < b).all() for p, b in zip(model.parameters(), before)) and all(s["step"] == 1 for s in opt.state.values())


def test_step_numbers_that_do_not_fit_change_nothing():
    p, g, m, v = (torch.ones(256, device=DEV) for _ in range(4))
    for step in ((1 << 32) + 1, -(1 << 32) + 1, 1 << 31):
        with pytest.raises(RuntimeError, match="below"):
            callers.adamw_step([p], [g], m, v, step, LR)
    assert all((t == 1).all() for t in (p, m, v))


def test_a_parameter_of_more_than_2_31_elements():
    """It goes in pieces; a small tensor behind it, and one without a gradient before that.  Elements at the ends of the
    pieces against a call over them alone."""
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 60 GB")
    big, small = (1 << 31) + 5000, 700
    p, g = torch.zeros(big, dtype=torch.bfloat16, device=DEV), torch.zeros(big, dtype=torch.bfloat16, device=DEV)
    q, h = (torch.randn(small, generator=_rng(70 + i)).to(torch.bfloat16).to(DEV) for i in range(2))
    parts = [slice(0, 512), slice((1 << 31) - 512, (1 << 31) + 512), slice(big - 904, big)]
    for i, at in enumerate(parts):
        p[at], g[at] = (torch.randn(at.stop - at.start, generator=_rng(80 + 2 * i + j)).to(torch.bfloat16).to(DEV) for j in range(2))
    alone = [p[at].clone() for at in parts] + [q.clone()]
    grads = [g[at].clone() for at in parts] + [h]
    idle = torch.zeros(300, dtype=torch.bfloat16, device=DEV)
    n = callers.adamw_arena([p, idle, q])
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    k = callers.adamw_arena(alone)
    m2, v2 = torch.zeros(k, device=DEV), torch.zeros(k, device=DEV)
    for t in (1, 2):
        callers.adamw_step([p, idle, q], [g, None, h], m, v, t, LR, BETAS, EPS, WD)
        callers.adamw_step(alone, grads, m2, v2, t, LR, BETAS, EPS, WD)
    start = ref.starts_of([big, 300, small])[0]
    places = parts + [slice(start[2], start[2] + small)]
    for at, x, a in zip(places, alone, ref.starts_of([x.numel() for x in alone])[0]):
        size = x.numel()
        assert torch.equal(m[at], m2[a:a + size]) and torch.equal(v[at], v2[a:a + size]) and x.any()
    for at, x in zip(parts, alone):
        assert torch.equal(p[at], x)
    assert torch.equal(q, alone[3]) and not idle.any() and not m[start[1]:start[2]].any() and not p[4096:1 << 20].any()
