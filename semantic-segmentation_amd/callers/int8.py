"""Conversion of a trained model for inference in 8 bits: its 1x1 convolutions (with the batch norm behind them) and fully
connected layers become `Int8Conv1x1` / `Int8Linear`.  Not in the reference; the deformable convolutions, 3x3 convolutions
and the attention products stay as they are (16-bit under .bfloat16() / .half())."""
import torch.nn as nn
from torch.nn.modules.batchnorm import BatchNorm2d

from ..dcn import Int8Conv1x1, Int8Linear
from ..dcn._lib import ELEMENT_TYPES
from ..dcn.deform_conv import _DcnConvBase
from ..dcn.int8 import MAX_CHANNELS, MAX_K
from .resnet import Bottleneck


def _plain(m, kind):
    """A `kind` and no subclass, that runs its forward and nothing beside it: a hook would go with the layer, or see another."""
    return type(m) is kind and "forward" not in vars(m) and \
        not (m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks)


def _taken(m, k, channels, min_channels):
    """The product takes a layer of this size and type."""
    return max(min_channels, 1) <= k <= MAX_K and channels <= MAX_CHANNELS and m.weight.dtype in ELEMENT_TYPES


def _pointwise(m, min_channels):
    return (_plain(m, nn.Conv2d) and tuple(m.kernel_size) == (1, 1) and m.groups == 1 and m.stride[0] == m.stride[1]
            and m.padding in ((0, 0), "valid") and _taken(m, m.in_channels, m.out_channels, min_channels))


def _linear(m, min_channels):
    return _plain(m, nn.Linear) and _taken(m, m.in_features, m.out_features, min_channels)


def _norm(m):
    return _plain(m, BatchNorm2d) and m.running_mean is not None and not m.training


def _runs_as(m, base):
    """m runs `base`'s forward (a subclass with one of its own may take the layers in any other order)."""
    return isinstance(m, base) and type(m).forward is base.forward and "forward" not in vars(m)


def _convert_sequence(seq, min_channels):
    """Conv2d (BatchNorm2d) (ReLU) and Linear (ReLU) runs of a Sequential: one layer, the others become Identity."""
    names = list(seq._modules)
    for i, name in enumerate(names):
        m = seq._modules[name]
        rest = [seq._modules[n] for n in names[i + 1:i + 3]] + [None, None]
        if _pointwise(m, min_channels):
            norm = rest[0] if _norm(rest[0]) else None
            follows = 1 if norm is None else 2
            relu = _plain(rest[follows - 1], nn.ReLU)
            seq._modules[name] = Int8Conv1x1.from_float(m, norm, relu)
        elif _linear(m, min_channels):
            follows, relu = 1, _plain(rest[0], nn.ReLU)
            seq._modules[name] = Int8Linear.from_float(m, relu)
        else:
            continue
        for n in names[i + 1:i + follows + (1 if relu else 0)]:
            seq._modules[n] = nn.Identity()


def _convert(module, min_channels):
    # A deformable convolution's own layers place its samples, in pixels of the map: left exact.  (The fully connected ones of
    # deformable RoI pooling place bins in parts of trans_std times the RoI: their offsets, 0.04 on average, move by 0.0007, and
    # the pooled values by 0.14 %.)
    if isinstance(module, _DcnConvBase):
        return
    if _runs_as(module, Bottleneck):
        if _pointwise(module.conv1, min_channels) and _norm(module.bn1):
            relu = _plain(module.relu, nn.ReLU)
            module.conv1, module.bn1 = Int8Conv1x1.from_float(module.conv1, module.bn1, relu), nn.Identity()
            module.relu1 = not relu
        if _pointwise(module.conv3, min_channels) and _norm(module.bn3):
            module.conv3, module.bn3 = Int8Conv1x1.from_float(module.conv3, module.bn3), nn.Identity()
    elif _runs_as(module, nn.Sequential):
        _convert_sequence(module, min_channels)
    else:
        for name, m in module._modules.items():
            if _pointwise(m, min_channels):
                module._modules[name] = Int8Conv1x1.from_float(m)
            elif _linear(m, min_channels):
                module._modules[name] = Int8Linear.from_float(m)
    for m in module._modules.values():
        if m is not None:
            _convert(m, min_channels)


def int8_inference(model, min_channels=16):
    """Converts `model` in place and returns it.  It has to be on the GPU and in eval mode: running statistics are folded
    into the weights, and the converted layers have no backward pass.  Layers with fewer than `min_channels` inputs are
    left (a token's rounding costs as much as their product), and so are layers with hooks, in float64 or beyond the sizes
    of `int8_linear`.  Norms and ReLUs join the layer before them in an nn.Sequential and in a Bottleneck, but not in
    subclasses with a forward of their own; a Sequential is taken to be called as a whole.  State dicts of the model change
    with its layers."""
    if model.training:
        raise RuntimeError("ddcn: int8_inference folds running statistics: call model.eval() first")
    if _pointwise(model, min_channels):
        return Int8Conv1x1.from_float(model)
    if _linear(model, 0):
        return Int8Linear.from_float(model)
    _convert(model, min_channels)
    return model
