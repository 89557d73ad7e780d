"""firefly_b200 — FireFly's INT8 training hot path, native to NVIDIA B200 (sm_100a).

Drop-in for the reference package's public API (fumitoshi0524/FireFly
``__init__.py:1-10``): ``BitLinear``, ``FireFlyOptim``,
``collect_bitlinear_modules``, ``quantize_fp_to_int8``.  Beside it, new here: MXFP4 layers
(``mxfp4``) and a distillation loss (``distill``).  The compute runs in
libfirefly_b200.so (hand-written sm_100a kernels) through a C ABI
(``include/firefly_b200.h``).
"""
from .fireflykernels import quantize_fp_to_int8
from .bitLinear import BitLinear, collect_bitlinear_modules
from .distill import distillation_loss
from .fireflyoptim import FireFlyOptim, FireFlyOptimSR
from .mxfp4 import (
    MXFP4Linear,
    MXFP4SwiGLU,
    MXFP4Tensor,
    mxfp4_linear,
    mxfp4_matmul,
    mxfp4_swiglu,
    quantize_fp_to_mxfp4,
    quantize_fp_to_mxfp4_dual,
)

__all__ = [
    "BitLinear",
    "FireFlyOptim",
    "FireFlyOptimSR",
    "MXFP4Linear",
    "MXFP4SwiGLU",
    "MXFP4Tensor",
    "collect_bitlinear_modules",
    "distillation_loss",
    "mxfp4_linear",
    "mxfp4_matmul",
    "mxfp4_swiglu",
    "quantize_fp_to_int8",
    "quantize_fp_to_mxfp4",
    "quantize_fp_to_mxfp4_dual",
]
