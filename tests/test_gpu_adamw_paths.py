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
