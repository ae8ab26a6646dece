"""nnv_amd: MI355X-native star-set reachability (the relax-star methods) behind NNV's API.

The compute path is the HIP library nnv_amd/libnnvhip.so (C ABI in include/nnvhip.h); these Python
classes mirror NNV's MATLAB classes for the path and call it through ctypes.
"""
from ._lib import Context, NNVHipError, NNVHipOutOfMemory, default_context  # noqa: F401
from .layers import Conv2DLayer, FullyConnectedLayer, PosLin, ReluLayer  # noqa: F401
from .layers_affine import (AveragePooling2DLayer, BatchNormalizationLayer, FlattenLayer,  # noqa: F401
                            ImageInputLayer, LayerS)
from .nn import NN  # noqa: F401
from .sets import Box, ImageStar, SetArray, Star, Zono  # noqa: F401
from .verify import HalfSpace, verify_specification  # noqa: F401

# The operators on points work on torch tensors; torch is imported when one of them is first used.
_POINTS = {"layer_norm": "points", "layer_norm_backward": "points", "cross_attention": "points", "cross_attention_backward": "points",
           "clip_gradients": "points", "LayerNormalizationLayer": "points", "CrossAttentionLayer": "points",
           "group_norm": "images", "group_norm_backward": "images", "rotate_positions": "images",
           "differential_attention": "images", "differential_attention_backward": "images", "GroupNormalizationLayer": "images",
           "DifferentialAttentionLayer": "images", "GridAttentionClassifier": "falsify",
           "CrossAttentionClassifier": "falsify", "falsify_point": "falsify", "train_step": "falsify"}


def __getattr__(name):
    if name in _POINTS:
        import importlib
        value = globals()[name] = getattr(importlib.import_module("." + _POINTS[name], __name__), name)
        return value
    raise AttributeError("module %r has no attribute %r" % (__name__, name))


def __dir__():
    return sorted(list(globals()) + list(_POINTS))
