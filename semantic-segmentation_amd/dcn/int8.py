"""Linear layers and 1x1 convolutions in 8-bit integers at inference: y = s_token s_channel sum q w (+ bias, ReLU).

Not in the reference; they stand beside the 16-bit inference of the deformable convolutions (deform_conv.py) and take
over the layers around them: a bottleneck's 1x1 convolutions, the depth branch, the fc layers of deformable RoI pooling
(`callers.int8_inference` converts a model).  Weights are rounded once, with one scale per output channel
(`quantize_int8`); every token -- a RoI, a pixel -- is rounded on the way in, with a scale of its own.  The sums are exact.
A token that holds a NaN or an infinity gives NaN in all of its outputs.  Kernels: csrc/ddcn_int8.hip; the arithmetic is
written down in include/ddcn_hip.h.  CPU tensors raise NotImplementedError, tensors that require grad a RuntimeError.
"""
import math

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib


_F32 = torch.float32
_INT8 = torch.int8
MAX_K, MAX_CHANNELS = 131072, 1 << 20         # of ddcn_int8_product


def _element_type(name, t):
    """ddcn element type of a floating-point tensor on the GPU that needs no gradient."""
    if not t.is_cuda:
        raise NotImplementedError
    code = _lib.ELEMENT_TYPES.get(t.dtype)
    if code is None:
        raise RuntimeError("ddcn: %s of %s is not supported (float32, float16, bfloat16)" % (name, t.dtype))
    if t.requires_grad or forward_ad._current_level >= 0:
        _check_no_gradient(name, t)
    return code


def _check_no_gradient(name, t):
    """Neither is a backward pass through t asked for nor does it carry a forward-mode tangent (which no_grad does not stop).
    (Called where one of the two may be: a call more for every tensor costs 0.2 us.)"""
    if t.requires_grad and torch.is_grad_enabled() or \
            forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError("ddcn: the 8-bit layers have no backward pass: call them under torch.no_grad(), or detach %s"
                           % name)


def _check_same_device(name, t, dev, x):
    if t.get_device() != dev:
        if not t.is_cuda:
            raise NotImplementedError
        raise RuntimeError("ddcn: %s is on %s but the input is on %s" % (name, t.device, x.device))


def _refuse_sizes(tokens, k, n):
    """What does not fit 32-bit fields of a struct, which would keep the low bits."""
    raise RuntimeError("ddcn: %d tokens of %d values, %d channels: 2^31 and more are not supported" % (tokens, k, n))


def _check_weight(x, dev, weight_q, weight_scale, bias, tokens, k):
    """-> (channels, weights with contiguous values in a row, the rows' stride in bytes, scales, float32 bias)"""
    _check_same_device("weight_q", weight_q, dev, x)
    _check_same_device("weight_scale", weight_scale, dev, x)
    shape = weight_q.shape
    if weight_q.dtype is not _INT8 or len(shape) != 2 or shape[1] != k:
        raise RuntimeError("ddcn: weight_q has to be int8 [channels, %d], got %s %s" % (k, weight_q.dtype, tuple(shape)))
    n = shape[0]
    if (tokens | k | n) >> 31:
        _refuse_sizes(tokens, k, n)
    if weight_scale.dtype is not _F32 or weight_scale.shape != (n,):
        raise RuntimeError("ddcn: weight_scale has to be float32 [%d], got %s %s" % (n, weight_scale.dtype, tuple(weight_scale.shape)))
    if weight_scale.requires_grad or forward_ad._current_level >= 0:
        _check_no_gradient("weight_scale", weight_scale)
    if bias is not None:
        _check_same_device("bias", bias, dev, x)
        if bias.dtype not in _lib.ELEMENT_TYPES or bias.shape != (n,):
            raise RuntimeError("ddcn: bias has to be floating point [%d], got %s %s" % (n, bias.dtype, tuple(bias.shape)))
        _element_type("bias", bias)
        if bias.dtype is not _F32 or not bias.is_contiguous():
            bias = bias.detach().float().contiguous()
    ldw = k
    if not weight_q.is_contiguous():
        ldw, one = weight_q.stride()
        if one != 1 and k > 1 or n > 1 and ldw < k:
            weight_q, ldw = weight_q.contiguous(), k
        elif n == 1:
            ldw = k
    return n, weight_q, ldw, weight_scale if weight_scale.is_contiguous() else weight_scale.contiguous(), bias


def _product(x, y, dev, weight_q, weight_scale, bias, geom):
    L = _lib.lib()
    ptr = _lib.ptr
    nbytes = L.ddcn_int8_workspace_bytes(geom)
    with _lib.on_device(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        _lib.check(L.ddcn_int8_product(ptr(x), ptr(weight_q), ptr(weight_scale), ptr(bias), ptr(y), ptr(ws), nbytes,
                                       geom, _lib.stream_of(dev)))
    return y


def _out_type(dtype):
    code = _lib.ELEMENT_TYPES.get(dtype)
    if code is None:
        raise RuntimeError("ddcn: output of %s is not supported (float32, float16, bfloat16)" % dtype)
    return code


def quantize_int8(x):
    """(q, scale) of the rows of x [rows, k]: int8 [rows, k] and float32 [rows], x ~ q * scale[:, None].  This is the
    rounding of the tokens of `int8_linear`, and the one to lay a weight [channels, k] out with."""
    code = _element_type("x", x)
    if x.dim() != 2:
        raise RuntimeError("ddcn: 2D tensor expected but got: %d" % x.dim())
    rows, k = x.shape
    if (rows | k) >> 31:
        _refuse_sizes(rows, k, 0)
    if k > 1 and x.stride(1) != 1:
        x = x.contiguous()
    q = torch.empty((rows, k), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    g = _lib.Int8Geom(1, rows, 1, k, 1, 0, code, 0, 0, 0, x.stride(0), 0, 1, k)
    dev = x.get_device()
    with _lib.on_device(dev):
        _lib.check(_lib.lib().ddcn_int8_quantize(_lib.ptr(x), _lib.ptr(q), k, _lib.ptr(scale), g,
                                                 _lib.stream_of(dev)))
    return q, scale


def int8_linear(input, weight_q, weight_scale, bias=None, relu=False, out_dtype=None):
    """input [..., k] (float32, float16 or bfloat16), weight_q int8 [channels, k], weight_scale float32 [channels],
    bias [channels] -> [..., channels] in `out_dtype` (the input's).  Rows of input may be strided.  k up to 131072, channels
    up to 2^20, fewer than 2^31 tokens."""
    code = _element_type("input", input)
    shape = input.shape
    if not shape:
        raise RuntimeError("ddcn: input has no dimension")
    k, dev = shape[-1], input.get_device()
    tokens = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    n, weight_q, ldw, weight_scale, bias = _check_weight(input, dev, weight_q, weight_scale, bias, tokens, k)
    dtype = input.dtype if out_dtype is None else out_dtype
    out = _out_type(dtype)
    y = torch.empty(shape[:-1] + (n,), dtype=dtype, device=input.device)
    if not y.numel():
        return y
    x = input
    if len(shape) != 2:
        x = input.detach().reshape(-1, k)
    rows, step = x.stride()
    g = _lib.Int8Geom(1, x.shape[0], 1, k, n, 0, code, out, int(relu), 0, rows, 0, 1 if k == 1 else step, ldw)
    return _product(x, y, dev, weight_q, weight_scale, bias, g)


def int8_conv1x1(input, weight_q, weight_scale, bias=None, stride=1, relu=False, out_dtype=None):
    """1x1 convolution without padding: input [n, c, h, w] (any strides), weight_q int8 [channels, c] ->
    [n, channels, ceil(h / stride), ceil(w / stride)], in channels-last memory where the input is."""
    code = _element_type("input", input)
    if input.dim() != 4:
        raise RuntimeError("4D input tensor expected but got: %d" % input.dim())
    if int(stride) != stride or stride < 1:
        raise RuntimeError("stride should be greater than zero, but got %r" % (stride,))
    stride = int(stride)
    images, c, h, w = input.shape
    dev = input.get_device()
    ho, wo = -(-h // stride), -(-w // stride)
    n, weight_q, ldw, weight_scale, bias = _check_weight(input, dev, weight_q, weight_scale, bias, images * ho * wo, c)
    dtype = input.dtype if out_dtype is None else out_dtype
    out = _out_type(dtype)
    si, sk, sh, sw = input.stride()
    last = c > 1 and sk == 1
    y = torch.empty((images, n, ho, wo), dtype=dtype, device=input.device,
                    memory_format=torch.channels_last if last else torch.contiguous_format)
    if not y.numel():
        return y
    g = _lib.Int8Geom(images, ho, wo, c, n, 0 if last else 1, code, out, int(relu), si, sh * stride, sw * stride, sk, ldw)
    return _product(input, y, dev, weight_q, weight_scale, bias, g)


class _Int8Layer(nn.Module):
    """Weights in int8 with their scales, as buffers; no parameters."""

    def __init__(self, channels, k, bias):
        super().__init__()
        self.register_buffer("weight_q", torch.zeros((channels, k), dtype=torch.int8))
        self.register_buffer("weight_scale", torch.ones(channels, dtype=torch.float32))
        self.register_buffer("bias", torch.zeros(channels, dtype=torch.float32) if bias else None)

    def _apply(self, fn, recurse=True):
        # .half() / .bfloat16() move a model to 16-bit activations: scales and bias stay float32, unrounded
        before = {name: getattr(self, name) for name in ("weight_scale", "bias")}
        super()._apply(fn, recurse)
        for name, t in before.items():
            now = getattr(self, name)
            if now is not None and now.dtype != torch.float32:
                setattr(self, name, t.to(now.device))
        return self

    @torch.no_grad()
    def _fill(self, weight, bias):
        q, scale = quantize_int8(weight.detach())
        self.weight_q, self.weight_scale = q, scale
        if bias is not None:
            self.bias = bias.detach().float().clone()
        return self


class Int8Linear(_Int8Layer):
    """nn.Linear at inference, in 8 bits; `relu` applies one behind it."""

    def __init__(self, in_features, out_features, bias=True, relu=False):
        super().__init__(out_features, in_features, bias)
        self.in_features, self.out_features, self.relu = in_features, out_features, relu

    @classmethod
    def from_float(cls, layer, relu=False):
        """From an nn.Linear on the GPU."""
        new = cls(layer.in_features, layer.out_features, layer.bias is not None, relu)
        return new._fill(layer.weight, layer.bias)

    def forward(self, x):
        return int8_linear(x, self.weight_q, self.weight_scale, self.bias, self.relu)

    def extra_repr(self):
        return "in_features=%d, out_features=%d, bias=%s, relu=%s" % (self.in_features, self.out_features,
                                                                      self.bias is not None, self.relu)


class Int8Conv1x1(_Int8Layer):
    """nn.Conv2d(kernel_size=1) at inference, in 8 bits, with the batch norm behind it folded in; `relu` applies one."""

    def __init__(self, in_channels, out_channels, stride=1, bias=True, relu=False):
        super().__init__(out_channels, in_channels, bias)
        self.in_channels, self.out_channels, self.stride, self.relu = in_channels, out_channels, stride, relu

    @classmethod
    def from_float(cls, conv, norm=None, relu=False):
        """From an nn.Conv2d on the GPU (1x1, no padding, one group) and, optionally, the nn.BatchNorm2d behind it: its
        running statistics and affine become part of the weights (before they are rounded) and of the bias."""
        if tuple(conv.kernel_size) != (1, 1) or conv.groups != 1 or conv.stride[0] != conv.stride[1] or \
                conv.padding not in ((0, 0), "valid"):
            raise ValueError("not a 1x1 convolution without padding and groups: %r" % (conv,))
        weight, bias = conv.weight.detach().float().flatten(1), conv.bias
        if norm is not None:
            if norm.running_mean is None:
                raise ValueError("the norm layer keeps no running statistics: %r" % (norm,))
            factor = torch.rsqrt(norm.running_var.float() + norm.eps)
            if norm.weight is not None:
                factor = factor * norm.weight.detach().float()
            shift = -norm.running_mean.float() if bias is None else bias.detach().float() - norm.running_mean.float()
            bias = shift * factor
            if norm.bias is not None:
                bias = bias + norm.bias.detach().float()
            weight = weight * factor[:, None]
        new = cls(conv.in_channels, conv.out_channels, conv.stride[0], bias is not None, relu)
        return new._fill(weight, bias)

    def forward(self, x):
        return int8_conv1x1(x, self.weight_q, self.weight_scale, self.bias, self.stride, self.relu)

    def extra_repr(self):
        return "%d, %d, stride=%d, bias=%s, relu=%s" % (self.in_channels, self.out_channels, self.stride,
                                                        self.bias is not None, self.relu)
