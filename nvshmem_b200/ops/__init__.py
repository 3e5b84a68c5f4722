"""Torch-facing operators built on the fused sm_100a kernels."""
from .fused_gemm import (FusedGemmError, gemm, GemmReduceScatter, AllGatherGemm, fused_lib)  # noqa: F401
from .moe import MoeDispatchCombine, MoeError  # noqa: F401
from .norms import rms_norm, block_norms, NormError  # noqa: F401
from .routing import moe_route, balance_loss, RoutingError  # noqa: F401
from .mxfp4 import MxFp4, quantize_mxfp4, gemm_mxfp4  # noqa: F401
