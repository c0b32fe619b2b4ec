"""B200-native (sm_100a) engine for the FP16 NHWC large-kernel depthwise convolution.

Importing the package registers the torch ops of both reference modules
(``depthwise::*`` and ``replknet_dw::*``) plus the generic
``depthwise::conv2d_nhwc`` / ``depthwise::conv2d_nhwc_fused`` ops and the
training ops around them (``norm_ops``: group normalisation with an activation;
``act8_ops``: 8-bit activation checkpoints).  All of them run through the C ABI
of ``libdwconv_b200.so`` (include/dwconv_b200.h).
"""
from . import _lib
from . import dw_ops
from . import act8_ops
from . import norm_ops
from . import depthwise_torch_ops
from . import depthwise_replknet_nhwc_ops
from .dw_ops import conv2d_nhwc, conv2d_nhwc_fused
from .act8_ops import act8_decode, act8_encode, conv2d_nhwc_act8
from .norm_ops import group_norm_act
from ._lib import plan_query, device_error, probe_fma_peak, DwbError

__all__ = ["conv2d_nhwc", "conv2d_nhwc_fused", "act8_encode", "act8_decode", "conv2d_nhwc_act8", "group_norm_act",
           "plan_query", "device_error", "probe_fma_peak", "DwbError",
           "dw_ops", "act8_ops", "norm_ops", "depthwise_torch_ops", "depthwise_replknet_nhwc_ops"]
