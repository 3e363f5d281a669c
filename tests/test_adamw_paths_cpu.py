"""CPU: what `AdamW` hands to `adamw_step` over the life of a run, with the call itself replaced; states that are refused."""
import importlib

import numpy as np
import pytest
import torch

import adamw_ref as ref
from conftest import load_pkg

load_pkg()
callers = importlib.import_module("semantic-segmentation_amd.callers")
optim = importlib.import_module("semantic-segmentation_amd.callers.optim")
_lib = importlib.import_module("semantic-segmentation_amd.dcn._lib")


@pytest.fixture
def calls(monkeypatch):
    """The arguments of every adamw_step that an optimizer makes."""
    seen = []
    monkeypatch.setattr(optim, "adamw_step", lambda params, grads, m, v, step, lr, *a, **kw: seen.append(dict(kw, step=step, grads=grads, arena=m)))
    return seen


def _params(*sizes):
    return [torch.nn.Parameter(torch.zeros(n)) for n in sizes]


def _give(params, which):
    for i, p in enumerate(params):
        p.grad = torch.ones_like(p) if i in which else None


def test_no_two_steps_of_an_arena_share_a_seed(calls):
    """Whichever parameters have a gradient: staged training, branches taken at random, a new group."""
    params = _params(3, 300, 5)
    opt = callers.AdamW(params[:2], bits=8, seed=3)
    turns = [{0}] * 4 + [{1}] * 6 + [{0, 1}, {1}, {0}, {0}, {1}]
    for which in turns:
        _give(params, which)
        opt.step()
    opt.add_param_group(dict(params=params[2:]))
    for which in ({2}, {0, 2}, {1}, {2}):
        _give(params, which)
        opt.step()
    arenas = {}
    for c in calls:
        arenas.setdefault(c["arena"].data_ptr(), []).append(c["seed"] & 0xFFFFFFFF)
    assert [len(s) for s in arenas.values()] == [len(turns) + 2, 3]
    assert all(len(set(s)) == len(s) for s in arenas.values())


def test_seeds_go_on_behind_a_state_dict(calls):
    params = _params(3, 300)
    opt = callers.AdamW(params, bits=8, seed=3)
    for which in ({0}, {0}, {1}):
        _give(params, which)
        opt.step()
    again = callers.AdamW(params, bits=8, seed=3)
    again.load_state_dict(opt.state_dict())
    for o in (opt, again):
        _give(params, {1})
        o.step()
    assert calls[-1]["seed"] == calls[-2]["seed"] and len({c["seed"] for c in calls}) == 4


def test_a_seed_that_repeats_makes_moments_stand_still():
    """Why it matters, from the formulas: second moments of gradients that drop by ten, 1500 steps (beta2 0.999: the mean root
    falls to 0.481); with one seed at every step the rounding is a threshold, and they stop where it says so."""
    def root(seed_of):
        n, b2 = 256, 0.999
        g = np.ones(n, np.float32)
        r = g.copy()
        g[128:] = 0.1
        for t in range(1500):
            r = np.sqrt(ref.moments32(g, g * 0, (r * r).astype(np.float32), 0.9, b2)[1]).astype(np.float32)
            q, s = ref.encode(r, ref.noise(np.arange(n), seed_of(t))[1], 255)
            r = ref.decode_r(np.maximum(q, 1), s)
        return r[128:].mean()

    want = np.sqrt(0.999 ** 1500 + (1 - 0.999 ** 1500) * 0.01)
    assert abs(root(lambda t: t) / want - 1) < 0.25          # as derived in the GPU test of the same experiment
    assert root(lambda t: 7) > 0.9


def test_a_step_without_a_seed_takes_one_from_its_step_number():
    import inspect
    assert inspect.signature(callers.adamw_step).parameters["seed"].default is None


def test_step_numbers_of_parameters_without_a_gradient_do_not_count(calls):
    """One number for the call where all that move share one, whatever the frozen ones' are."""
    params = _params(3, 300, 5)
    opt = callers.AdamW(params)
    for which in ({0, 1, 2}, {0, 2}, {0, 2}, {1, 2}):
        _give(params, which)
        opt.step()
    assert [c["step"] for c in calls] == [1, 2, 3, [3, 2, 4]]
    assert [opt.state[p]["step"] for p in params] == [3, 2, 4]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_dict_that_is_refused_changes_nothing(calls, bits):
    """Whatever is wrong with it, and at whichever parameter: moments, step numbers and settings stay, and steps go on."""
    make = lambda: [torch.nn.Parameter(torch.randn(5, 6, 3, 3)), torch.nn.Parameter(torch.zeros(300))]     # noqa: E731
    params, others = make(), make()
    others[1].data = others[1].data[:300]
    opt, theirs = callers.AdamW(params, bits=bits, lr=0.5), callers.AdamW(others, bits=bits, lr=0.25)
    for o, ps in ((opt, params), (theirs, others)):
        for _ in range(3):
            _give(ps, {0, 1})
            o.step()
    for p in params:
        opt.state[p]["exp_avg"].fill_(3)
    good = theirs.state_dict()

    def with_(index, name, value):
        state = {i: dict(s) for i, s in good["state"].items()}
        if value is None:
            del state[index][name]
        else:
            state[index][name] = value
        return dict(good, state=state)

    last = good["state"][0]["exp_avg"].to(memory_format=torch.channels_last)
    bad = [with_(1, "exp_avg_sq", good["state"][1]["exp_avg_sq"][:1]), with_(1, "exp_avg", good["state"][1]["exp_avg"][:299]),
           with_(1, "exp_avg_sq", None), with_(1, "max_exp_avg_sq", torch.zeros(300)), with_(1, "step", None),
           with_(1, "step", "three"), with_(1, "step", -1), with_(1, "exp_avg", 4.0),
           dict(good, param_groups=good["param_groups"] * 2), dict(good, param_groups=[dict(good["param_groups"][0], params=[0])])]
    if bits == 8:
        bad += [with_(0, "exp_avg", last), with_(1, "exp_avg_scale", good["state"][1]["exp_avg_scale"][:1]),
                with_(1, "exp_avg_sq", good["state"][1]["exp_avg_sq"].float())]
    before = [(id(opt.state[p]["exp_avg"]), opt.state[p]["exp_avg"].clone(), opt.state[p]["step"]) for p in params]
    for state_dict in bad:
        with pytest.raises((ValueError, TypeError)):
            opt.load_state_dict(state_dict)
        for p, (name, m, step) in zip(params, before):
            assert id(opt.state[p]["exp_avg"]) == name and torch.equal(opt.state[p]["exp_avg"], m) and opt.state[p]["step"] == step
        assert opt.param_groups[0]["lr"] == 0.5
    _give(params, {0, 1})
    opt.step()
    assert calls[-1]["step"] == 4
    opt.load_state_dict(good)
    assert opt.param_groups[0]["lr"] == 0.25 and opt.state[params[1]]["step"] == 3 and not opt.state[params[1]]["exp_avg"].any()
    if bits == 32:              # torch.optim.AdamW's own state: a step number in a tensor, any memory format, any type
        opt.load_state_dict(with_(0, "exp_avg", last.double() + 2))
        assert (opt.state[params[0]]["exp_avg"] == 2).all()
    opt.load_state_dict(with_(0, "step", torch.tensor(7.0)))
    assert opt.state[params[0]]["step"] == 7
    empty = callers.AdamW(make(), bits=bits).state_dict()
    opt.load_state_dict(empty)
    assert not opt.state


def test_a_first_step_that_is_refused_leaves_no_state():
    """On a CPU model: NotImplementedError, and the optimizer is as new (the model may move to the GPU next)."""
    params = _params(3, 300)
    opt = callers.AdamW(params)
    _give(params, {0, 1})
    with pytest.raises(NotImplementedError):
        opt.step()
    assert not opt.state and not opt.state_dict()["state"]


def test_a_later_step_that_is_refused_keeps_the_state(calls, monkeypatch):
    params = _params(3, 300)
    opt = callers.AdamW(params)
    _give(params, {0, 1})
    opt.step()

    def refuse(*a, **kw):
        raise RuntimeError("refused")
    monkeypatch.setattr(optim, "adamw_step", refuse)
    with pytest.raises(RuntimeError, match="refused"):
        opt.step()
    assert [opt.state[p]["step"] for p in params] == [1, 1]


def test_step_numbers_beyond_32_bits_are_refused():
    """2^32 + 1 would be step 1 in an int."""
    for step in (1 << 31, (1 << 32) + 1, [1 << 31], -1, -(1 << 32) + 1):
        with pytest.raises((RuntimeError, OverflowError)):
            optim._step_numbers(step, 1)
    assert optim._step_numbers(7, 1) == (None, 7) and optim._step_numbers(np.int64(7), 1) == (None, 7)
    assert list(optim._step_numbers([7, 8], 2)[0]) == [7, 8]


def _list(kind, values):
    import ctypes
    from array import array
    a = array(kind, values)
    return a, ctypes.c_void_p(a.buffer_info()[0])


def test_arena_lengths_do_not_wrap():
    """2^24 tensors of 2^40 elements and one of 256 are 2^64 + 256 together, which 64 bits hold as 256."""
    keep, p = _list("q", [1 << 40] * (1 << 24) + [256])
    assert _lib.lib().ddcn_adamw_arena(len(keep), p) == -5
    keep, p = _list("q", [1 << 40, 1])
    assert _lib.lib().ddcn_adamw_arena(2, p) == -5 and _lib.lib().ddcn_adamw_arena(1, p) == -5
    keep, p = _list("q", [(1 << 40) - 512, 256])
    assert _lib.lib().ddcn_adamw_arena(2, p) == (1 << 40) - 256


def test_norm_workspace_of_a_list_that_is_not_there():
    L = _lib.lib()
    assert L.ddcn_grad_norm_workspace_bytes(3, None) == 0 and L.ddcn_grad_norm_workspace_bytes(-1, None) == 0
    assert L.ddcn_grad_norm_workspace_bytes(0, None) == 256
    keep, p = _list("q", [100])
    assert L.ddcn_grad_norm_workspace_bytes(1, p) == 256


@pytest.mark.parametrize("root", [0.3, 1.5, 10.25, 100.9])
def test_codes_are_right_on_average_and_what_they_stand_for_is_not(root):
    """q = floor(t + u) has the mean t, and q^2 the mean t^2 + f (1 - f), f the fraction of t: what include/ddcn_hip.h states of
    the decoded moments.  Over N places q is n + 1 with probability f, n otherwise: 5 sigma of both means, and u's 2^-16 steps."""
    n, whole = 1 << 16, np.floor(root)
    f = root - whole
    for u in ref.noise(np.arange(n), 11):
        q = np.floor((np.float32(root) + u).astype(np.float32)).astype(np.float64)
        sigma = np.sqrt(f * (1 - f) / n)
        assert abs(q.mean() - root) < 5 * sigma + 2.0 ** -15
        assert abs((q * q).mean() - (root ** 2 + f * (1 - f))) < (2 * whole + 1) * (5 * sigma + 2.0 ** -15)
    assert f * (1 - f) > (2 * whole + 1) * 5 * sigma or root > 100       # it tells the two apart


def test_equal_strides_of_other_shapes_are_not_alike():
    """A step reads as many elements in a row as the parameter has: a gradient of equal strides and number of elements whose
    shape is another one may end before (here after 60 of 108), or lie elsewhere."""
    t = _lib.tensors()
    p = torch.zeros(2, 6, 3, 3).to(memory_format=torch.channels_last)
    g = torch.zeros(200).as_strided((1, 12, 3, 3), p.stride())
    assert g.stride() == p.stride() and g.numel() == p.numel() and t.alike([p], [g]) == 1
    p = torch.zeros(2, 6)
    g = torch.zeros(3, 6)[:, :4]
    assert g.stride() == p.stride() and g.numel() == p.numel() and t.alike([p], [g]) == 1
    assert t.alike([p], [torch.zeros(12)]) == 0 and t.alike([p], [torch.zeros(3, 4)]) == 0       # one run of memory each


@pytest.mark.parametrize("bits", [32, 8])
def test_moments_of_frozen_parameters_of_any_strides_are_their_own(calls, bits):
    """A parameter that is no run of memory can have no step, but it may lie, frozen, beside others."""
    frozen = [torch.zeros(40, 60)[:, ::2], torch.zeros(30, 20).t(), torch.zeros(5, 6, 7, 8)[:, :, 1:5], torch.zeros(1, 1).expand(9, 300)]
    params = [p for t in frozen for p in (*_params(3), torch.nn.Parameter(t))] + _params(5)
    opt = callers.AdamW(params, bits=bits)
    _give(params, {0, 2, 4, 6, 8})
    opt.step()
    for i, p in enumerate(params):
        for k, t in opt.state[p].items():
            if k != "step":
                t.fill_(i + 1)
    for i, p in enumerate(params):
        assert all((t == i + 1).all() and (k.endswith("scale") or t.shape == p.shape) for k, t in opt.state[p].items() if k != "step")
    again = callers.AdamW(params, bits=bits)
    again.load_state_dict(opt.state_dict())
    for i, p in enumerate(params):
        assert all((t == i + 1).all() for k, t in again.state[p].items() if k != "step")
