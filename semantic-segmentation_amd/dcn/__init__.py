"""Drop-in for `detseg.ops.dcn`: the names of `detseg/ops/dcn/__init__.py:1-13`, plus the autograd.Functions."""
from . import deform_conv as _conv
from . import deform_pool as _pool
from . import int8 as _int8

_CONV_NAMES = ("DeformConv", "DeformConvPack", "ModulatedDeformConv", "ModulatedDeformConvPack", "DepthawareConv",
               "DepthDeformConvPack", "DeformConvFunction", "ModulatedDeformConvFunction", "DepthawareConvFunction",
               "deform_conv", "modulated_deform_conv", "depthaware_conv")
_POOL_NAMES = ("DeformRoIPooling", "DeformRoIPoolingPack", "ModulatedDeformRoIPoolingPack", "DeformRoIPoolingFunction",
               "deform_roi_pooling")
# not in the reference: 8-bit layers for inference
_INT8_NAMES = ("quantize_int8", "int8_linear", "int8_conv1x1", "Int8Linear", "Int8Conv1x1")

globals().update({n: getattr(_conv, n) for n in _CONV_NAMES})
globals().update({n: getattr(_pool, n) for n in _POOL_NAMES})
globals().update({n: getattr(_int8, n) for n in _INT8_NAMES})

__all__ = list(_CONV_NAMES + _POOL_NAMES + _INT8_NAMES)
