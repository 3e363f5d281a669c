"""AdamW over all parameters of a model in a few launches, with the moments in float32 or in 8-bit codes, and the
global gradient norm it may clip by.  Not in the reference, whose optimizer is torch.optim.SGD (detseg/apis/train.py:64-105);
the kernels are csrc/ddcn_optim.hip, the arithmetic is written down in include/ddcn_hip.h.

The moments of a step live in one arena per moment: tensor i starts at the next multiple of 256 elements behind tensor
i - 1 (`adamw_arena` gives the length).  In 8 bits `exp_avg` is int8, `exp_avg_sq` uint8, each with one float32 scale per
256 elements: 2.03 bytes a parameter instead of 8.  CPU tensors raise NotImplementedError; there is no fallback.
"""
import ctypes
import operator
from array import array

import torch

from ..dcn import _lib

BLOCK = 256
_Tensor = torch.Tensor


def _address(a):
    return ctypes.c_void_p(a.buffer_info()[0]) if len(a) else None


def _check_device(device, name):
    """The common GPU of tensors that `describe` has seen."""
    if device == -1:
        raise NotImplementedError
    if device == -2:
        raise RuntimeError("ddcn: %s are on more than one device" % name)
    return device


def _dense(t):
    """Contiguous, or channels-last."""
    return t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last)) or \
        (t.dim() == 5 and t.is_contiguous(memory_format=torch.channels_last_3d))


def _same_order(a, b):
    return a.stride() == b.stride() or (a.is_contiguous() and b.is_contiguous())


def _arena_of(count, numels):
    n = _lib.lib().ddcn_adamw_arena(count, numels)
    if n < 0:
        _lib.check(n)
    return n


def adamw_arena(params):
    """Elements of the arena that holds one moment of `params`."""
    numels = array("q", map(_Tensor.numel, params))
    return _arena_of(len(numels), _address(numels))


def grad_norm(grads):
    """sqrt of the sum of squares over all `grads` (entries may be None), a float32 scalar on their GPU: summed in
    float64 in a fixed order, so that it is the same at every call.  Types may be mixed.  Any strides: a gradient that is
    neither contiguous nor channels-last is copied first.  Not differentiable."""
    grads = [g for g in grads if g is not None]
    if not grads:
        raise RuntimeError("ddcn: grad_norm needs at least one gradient")
    pointers, numels, dtypes, dev, dtype, contiguous, _, _ = _lib.tensors().describe(grads)
    _check_device(dev, "gradients")
    if not contiguous and not all(map(_dense, grads)):
        grads = [g if _dense(g) else g.detach().contiguous() for g in grads]
        pointers = _lib.tensors().describe(grads)[0]
    if dtype == -1:
        other = next(g.dtype for g in grads if g.dtype not in _lib.ELEMENT_TYPES)
        raise RuntimeError("ddcn: %s gradients are not supported (float32, float16, bfloat16)" % other)
    L = _lib.lib()
    nbytes = L.ddcn_grad_norm_workspace_bytes(len(grads), numels)
    with _lib.on_device(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=grads[0].device)
        out = torch.empty((), dtype=torch.float32, device=grads[0].device)
        _lib.check(L.ddcn_grad_norm(len(grads), pointers, numels, dtypes, _lib.ptr(out), _lib.ptr(ws), nbytes,
                                    _lib.stream_of(dev)))
    return out


def _check_state(name, t, dtype, numel, device):
    if t.get_device() != device:
        if not t.is_cuda:
            raise NotImplementedError
        raise RuntimeError("ddcn: %s is on another device than the parameters" % name)
    if t.dtype != dtype or t.numel() != numel or not t.is_contiguous():
        raise RuntimeError("ddcn: %s has to be a contiguous %s tensor of %d elements, got %s of %d"
                           % (name, dtype, numel, t.dtype, t.numel()))


def _step_numbers(step, count):
    """-> (None or an array of `count` numbers, one number for all)"""
    if hasattr(step, "__index__"):
        step = operator.index(step)
        if step >> 31:                  # an int of the C call would keep the low bits
            raise RuntimeError("ddcn: step %d is below 1 or not below 2^31" % step)
        return None, step
    steps = array("i", step)
    if len(steps) != count:
        raise RuntimeError("ddcn: %d parameters but %d step numbers" % (count, len(steps)))
    return steps, 1


def adamw_step(params, grads, exp_avg, exp_avg_sq, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               exp_avg_scale=None, exp_avg_sq_scale=None, seed=None, grad_norm=None, max_norm=None):
    """One AdamW step over `params` (list of tensors of one type: float32, bfloat16 or float16), in place.  They are
    contiguous or channels-last and do not overlap.

    `grads`: as many tensors of the same shapes, type and order in memory; None leaves a parameter and its moments as they
    are.  (Moments lie in the arena in the order of the parameter's memory.)
    `exp_avg`, `exp_avg_sq`: the arenas (`adamw_arena(params)` elements): float32, or int8 and uint8 with
    `exp_avg_scale`, `exp_avg_sq_scale` (float32, one per 256 elements) and `seed`, a whole number that has to differ
    from step to step: it drives the random rounding of the codes, and the same seed gives the same codes.  None: the sum
    of the step numbers.  (Under one seed again and again an element is rounded at one fixed threshold, and its moments
    stand still where they should move.)
    `step`: t of the bias corrections, from 1 on, or one for each tensor.  With `max_norm` the gradients are scaled by
    min(1, max_norm / (grad_norm + 1e-6)), `grad_norm` being a float32 scalar on the GPU (see `grad_norm()`): nothing
    waits for it, and if it is not finite the step changes nothing.

    Everything else is as in torch.optim.AdamW: p <- p (1 - lr wd) - lr m^ / (sqrt(v^) + eps), decay and update rounded
    together to the parameter's type (a 16-bit parameter does not see changes below half its step).  The step number, lr and
    seed are fixed when the call is made, so it refuses to be captured into a HIP graph."""
    params, grads = list(params), list(grads)
    if len(params) != len(grads):
        raise RuntimeError("ddcn: %d parameters but %d gradients" % (len(params), len(grads)))
    if not params:
        return
    describe = _lib.tensors().describe
    pointers, numels, _, dev, code, contiguous, distinct, count = describe(params)
    gradients, grad_numels, _, grad_dev, grad_code, grad_contiguous, _, given = describe(grads)
    if count < len(params):
        raise RuntimeError("ddcn: a parameter is None")
    if -1 in (dev, grad_dev) or (grad_norm is not None and not grad_norm.is_cuda):
        raise NotImplementedError
    if dev == -2 or (given and grad_dev != dev) or (grad_norm is not None and grad_norm.get_device() != dev):
        raise RuntimeError("ddcn: parameters and gradients are on more than one device")
    if params[0].dtype not in _lib.ELEMENT_TYPES:
        raise RuntimeError("ddcn: %s parameters are not supported (float32, float16, bfloat16)" % params[0].dtype)
    if code < 0 or (given and grad_code != code):
        raise RuntimeError("ddcn: the parameters and gradients of one step must share a dtype (%s)" % params[0].dtype)
    if given < len(grads) or not contiguous or not grad_contiguous or numels != grad_numels:
        wrong = _lib.tensors().alike(params, grads)
        if wrong == 1:
            raise RuntimeError("ddcn: parameters have to be contiguous (or channels-last), gradients of their shapes in the "
                               "same order")
        if wrong == 2:
            raise RuntimeError("ddcn: a gradient has another number of elements than its parameter")
    if not distinct:
        raise RuntimeError("ddcn: a parameter is listed twice")
    L = _lib.lib()
    arena = _arena_of(len(params), numels)
    bits = 8 if exp_avg.dtype == torch.int8 else 32
    _check_state("exp_avg", exp_avg, torch.int8 if bits == 8 else torch.float32, arena, dev)
    _check_state("exp_avg_sq", exp_avg_sq, torch.uint8 if bits == 8 else torch.float32, arena, dev)
    if bits == 8:
        if exp_avg_scale is None or exp_avg_sq_scale is None:
            raise RuntimeError("ddcn: 8-bit moments need exp_avg_scale and exp_avg_sq_scale")
        _check_state("exp_avg_scale", exp_avg_scale, torch.float32, arena // BLOCK, dev)
        _check_state("exp_avg_sq_scale", exp_avg_sq_scale, torch.float32, arena // BLOCK, dev)
    elif exp_avg_scale is not None or exp_avg_sq_scale is not None:
        raise RuntimeError("ddcn: float32 moments take no scales")
    if (max_norm is None) != (grad_norm is None):
        raise RuntimeError("ddcn: max_norm and grad_norm go together")
    if grad_norm is not None and (grad_norm.dtype != torch.float32 or grad_norm.numel() != 1):
        raise RuntimeError("ddcn: grad_norm has to be one float32 value")
    steps, step = _step_numbers(step, len(params))
    if seed is None:
        seed = step if steps is None else sum(steps)
    hyper = _lib.AdamwHyper(lr, betas[0], betas[1], eps, weight_decay, 0.0 if max_norm is None else max_norm, step,
                            code, bits, int(seed) & 0xFFFFFFFF)
    with _lib.on_device(dev):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ddcn: adamw_step cannot be captured into a HIP graph: a replay would repeat the step "
                               "number, the learning rate and the seed of the capture")
        _lib.check(L.ddcn_adamw_step(len(params), pointers, gradients, numels,
                                     None if steps is None else _address(steps), _lib.ptr(exp_avg),
                                     _lib.ptr(exp_avg_sq), _lib.ptr(exp_avg_scale), _lib.ptr(exp_avg_sq_scale),
                                     _lib.ptr(grad_norm), hyper, _lib.stream_of(dev)))
    # the kernels write behind autograd's back: a backward pass that saved one of these must notice
    changed = _lib.tensors().changed
    changed(params, grads)
    changed([exp_avg, exp_avg_sq] if bits == 32 else [exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale])


def adamw_moments(exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale):
    """(m, v) in float32: what the 8-bit codes of two arenas stand for."""
    dev, n = exp_avg.get_device(), exp_avg.numel()
    if dev < 0:
        raise NotImplementedError
    if n % BLOCK:
        raise RuntimeError("ddcn: an arena has a multiple of %d elements, got %d" % (BLOCK, n))
    _check_state("exp_avg", exp_avg, torch.int8, n, dev)
    _check_state("exp_avg_sq", exp_avg_sq, torch.uint8, n, dev)
    _check_state("exp_avg_scale", exp_avg_scale, torch.float32, n // BLOCK, dev)
    _check_state("exp_avg_sq_scale", exp_avg_sq_scale, torch.float32, n // BLOCK, dev)
    with _lib.on_device(dev):
        m = torch.empty(n, dtype=torch.float32, device=exp_avg.device)
        v = torch.empty_like(m)
        _lib.check(_lib.lib().ddcn_adamw_moments(_lib.ptr(exp_avg), _lib.ptr(exp_avg_sq), _lib.ptr(exp_avg_scale),
                                                 _lib.ptr(exp_avg_sq_scale), _lib.ptr(m), _lib.ptr(v), n,
                                                 _lib.stream_of(dev)))
    return m, v


class _Arena:
    """The moments of one parameter group's tensors of one type on one GPU."""

    def __init__(self, params, bits):
        self.key = self.key_of(params)
        dev, n = params[0].device, adamw_arena(params)
        zeros = lambda k, t: torch.zeros(k, dtype=t, device=dev)                                  # noqa: E731
        self.exp_avg = zeros(n, torch.float32 if bits == 32 else torch.int8)
        self.exp_avg_sq = zeros(n, torch.float32 if bits == 32 else torch.uint8)
        self.scales = {} if bits == 32 else dict(exp_avg_scale=zeros(n // BLOCK, torch.float32),
                                                 exp_avg_sq_scale=zeros(n // BLOCK, torch.float32))

    @staticmethod
    def key_of(params):
        return tuple(map(id, params)), tuple(map(_Tensor.stride, params)), tuple(map(_Tensor.numel, params))

    def views(self, params):
        """For each parameter: its part of the arena, under the names of the state dict."""
        start = 0
        for p in params:
            n = p.numel()
            end = start + -(-n // BLOCK) * BLOCK
            if _dense(p):
                shaped = lambda t: torch.as_strided(t, p.shape, p.stride(), start)               # noqa: E731, B023
            else:                    # it can have no step; its strides may reach beyond its part
                shaped = lambda t: t[start:start + n].view(p.shape)                              # noqa: E731, B023
            state = dict(exp_avg=shaped(self.exp_avg), exp_avg_sq=shaped(self.exp_avg_sq))
            state.update({k: t[start // BLOCK:end // BLOCK] for k, t in self.scales.items()})
            yield state
            start = end


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's interface over `adamw_step`.

    bits=32 or 8: how the moments are held (in 8 bits those of elements far below the largest of their 256 settle too high:
    the first moment by 5 % at a thousandth of it, 30 % at a ten-thousandth; include/ddcn_hip.h).  max_norm: clip all
    gradients by their global norm first (the last norm is kept in `last_grad_norm`, a scalar on the GPU); a step whose norm
    is not finite changes no parameter and no moment, though its step number counts.  seed: of the rounding of 8-bit
    moments; the same seed repeats a run.
    Parameters of one group may have different types (one arena each); all live on one GPU."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, max_norm=None, seed=0):
        if bits not in (32, 8):
            raise ValueError("moments of %r bits: 32 or 8" % (bits,))
        if not lr >= 0 or not eps >= 0 or not weight_decay >= 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr %r, betas %r, eps %r, weight_decay %r" % (lr, betas, eps, weight_decay))
        if max_norm is not None and not max_norm > 0:
            raise ValueError("max_norm %r: above 0, or None" % (max_norm,))
        self.bits, self.max_norm, self.seed, self.last_grad_norm = bits, max_norm, int(seed), None
        self._arenas = {}
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _sets(self, g):
        """(dtype, parameters) of group number g, in the order of its first parameter of each type."""
        sets = {}
        for p in self.param_groups[g]["params"]:
            sets.setdefault(p.dtype, []).append(p)
        return sets.items()

    def _arena(self, g, dtype, params):
        arena = self._arenas.get((g, dtype))
        if arena is not None and arena.key == _Arena.key_of(params):
            return arena
        if arena is not None or any(p in self.state for p in params):
            raise RuntimeError("ddcn: the parameters of a group (or their types or sizes) changed after its first step")
        arena = self._arenas[g, dtype] = _Arena(params, self.bits)
        for p, state in zip(params, arena.views(params)):
            self.state[p] = dict(step=0, **state)
        return arena

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        sets = [(g, dtype, params) for g in range(len(self.param_groups)) for dtype, params in self._sets(g)]
        grads = [[p.grad for p in params] for _, _, params in sets]
        every = [x for l in grads for x in l if x is not None]
        if not every:
            return loss
        norm = self.last_grad_norm = grad_norm(every) if self.max_norm is not None else None
        for number, ((g, dtype, params), gs) in enumerate(zip(sets, grads)):
            if all(x is None for x in gs):
                continue
            if _lib.tensors().alike(params, gs) == 1:
                gs = [x if x is None or _same_order(x, p) else torch.empty_like(p).copy_(x) for p, x in zip(params, gs)]
            first = (g, dtype) not in self._arenas
            group, arena, state = self.param_groups[g], self._arena(g, dtype, params), self.state
            steps = [state[p]["step"] + (x is not None) for p, x in zip(params, gs)]
            counts = {steps[0]} if steps.count(steps[0]) == len(steps) else \
                {s for s, x in zip(steps, gs) if x is not None}          # the others' numbers do not count
            # a seed for every step and arena: the sum of an arena's step numbers grows at each of its steps (their maximum
            # does not, where the gradients belong to tensors that have made fewer), and it comes back with a state dict
            seed = self.seed + 0x10001 * number + 0x3779B1 * sum(steps)
            try:
                adamw_step(params, gs, arena.exp_avg, arena.exp_avg_sq,
                           counts.pop() if len(counts) == 1 else [max(s, 1) for s in steps], group["lr"],
                           group["betas"], group["eps"], group["weight_decay"], seed=seed, grad_norm=norm,
                           max_norm=self.max_norm, **arena.scales)
            except Exception:
                if first:                    # refused: there is no state of it (the parameters may move to a GPU next)
                    del self._arenas[g, dtype]
                    for p in params:
                        del state[p]
                raise
            for p, s in zip(params, steps):
                state[p]["step"] = s
        return loss

    def _check_saved(self, p, saved):
        """Refuses a parameter's saved state that `_take` could not copy."""
        want = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scale", "exp_avg_sq_scale"} if self.bits == 8 else set())
        found = "%s" % {k: getattr(t, "dtype", t) for k, t in saved.items()}
        if set(saved) != want or not all(torch.is_tensor(t) for k, t in saved.items() if k != "step"):
            raise ValueError("the state dict holds %s, not the state of AdamW with bits=%d" % (found, self.bits))
        moments = saved["exp_avg"], saved["exp_avg_sq"]
        scales = [saved[k] for k in sorted(want) if k.endswith("scale")]
        types = all(t.is_floating_point() for t in moments) if self.bits == 32 else \
            [t.dtype for t in moments] == [torch.int8, torch.uint8]
        if not types or any(t.shape != p.shape for t in moments) or any(t.shape != (-(-p.numel() // BLOCK),) for t in scales):
            raise ValueError("the state dict holds %s, not the state of AdamW with bits=%d over these parameters"
                             % (found, self.bits))
        if self.bits == 8 and _dense(p) and not all(_same_order(t, p) for t in moments):      # codes and their scales go by memory
            raise ValueError("8-bit moments of a parameter in another memory format")
        if int(saved["step"]) < 0:
            raise ValueError("step number %r" % (saved["step"],))

    def load_state_dict(self, state_dict):
        """As torch's, but moments keep their types (torch would cast them to the parameter's) and are copied into the
        arenas.  A state of another number of bits, or over other parameters, is refused and changes nothing."""
        saved, order = state_dict["state"], {}
        for group, old in zip(self.param_groups, state_dict["param_groups"]):
            order.update(zip(group["params"], old["params"]))
        loaded = {p: saved[i] for p, i in order.items() if i in saved}
        for p, theirs in loaded.items():
            self._check_saved(p, theirs)
        super().load_state_dict(dict(state_dict, state={}))
        self._take(loaded)

    def _take(self, loaded):
        """Arenas made anew, with the moments of `loaded` (parameter -> state)."""
        self._arenas.clear()
        self.state.clear()
        for g in range(len(self.param_groups)):
            for dtype, params in self._sets(g):
                if not any(p in loaded for p in params):
                    continue
                self._arena(g, dtype, params)
                for p in params:
                    mine = self.state[p]
                    for k, t in loaded.get(p, {}).items():
                        if k == "step":
                            mine[k] = int(t)
                        else:
                            mine[k].copy_(t)

    def __getstate__(self):          # copy.deepcopy and pickle: torch's own leaves a subclass's attributes out
        return dict(super().__getstate__(), settings=(self.bits, self.max_norm, self.seed))

    def __setstate__(self, state):
        state = dict(state)
        settings = state.pop("settings", None)
        super().__setstate__(state)
        if settings is None:         # from load_state_dict, which takes the moments itself
            return
        self.bits, self.max_norm, self.seed = settings
        self._arenas, self.last_grad_norm = {}, None
        with torch.no_grad():
            self._take({p: dict(s) for p, s in self.state.items()})
