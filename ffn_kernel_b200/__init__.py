"""B200 (sm_100a) implementation of the routed MaskedLinear / MaskedFFN operators.

Import surface of the reference package (``ffn_kernel/__init__.py:1``):
``from ffn_kernel_b200 import MaskedLinear, MaskedFFN``.
"""
from .ops import MaskedFFN, MaskedLinear  # noqa: F401
from .modules import (GraphedMaskedFFN, MaskedFFNModule, MaskedLinearModule, MXFP4MaskedFFNModule,  # noqa: F401
                      MXFP4MaskedLinearModule, TensorParallelMaskedFFN)
from .mxfp4 import MXFP4MaskedFFN, MXFP4MaskedLinear, MXFP4Tensor, dequantize_mxfp4, quantize_mxfp4  # noqa: F401
from .route import Route, check_status, route  # noqa: F401

__all__ = ["MaskedLinear", "MaskedFFN", "MaskedLinearModule", "MaskedFFNModule", "TensorParallelMaskedFFN", "GraphedMaskedFFN",
           "MXFP4Tensor", "quantize_mxfp4", "dequantize_mxfp4", "MXFP4MaskedLinear", "MXFP4MaskedFFN",
           "MXFP4MaskedLinearModule", "MXFP4MaskedFFNModule",
           "route", "Route", "check_status"]
