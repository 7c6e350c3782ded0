"""gfx950 HIP kernel implementations of the MoE operations (the
export surface of triton_moe/kernels/__init__.py:18-40 of the reference, and the
operators for a few tokens and the dense operators, which it lacks)."""

from .gather import padded_gather, padded_gather_autograd
from .scatter import padded_scatter, padded_scatter_autograd
from .grouped_gemm import (
    grouped_gemm_up,
    grouped_gemm_down,
    grouped_gemm_up_backward,
    grouped_gemm_down_backward,
    grouped_gemm_up_autograd,
    grouped_gemm_down_autograd,
    precompute_gather_map,
    GroupedGemmUp,
    GroupedGemmDown,
)
from .fused_cumsum import fused_route
from .dense import fused_linear, gated_mlp, layer_norm, layer_norm_max
from .few_tokens import (
    FewTokenExperts,
    QuantizedExperts,
    QuantizedMatrices,
    experts_few_tokens,
    few_token_experts,
    few_tokens_max,
    matvec_q4,
    moe_few_tokens,
    quantize_experts,
    quantize_matrices,
)

__all__ = [
    # Gather/Scatter
    "padded_gather",
    "padded_gather_autograd",
    "padded_scatter",
    "padded_scatter_autograd",
    # Forward kernels
    "grouped_gemm_up",
    "grouped_gemm_down",
    # Backward kernels
    "grouped_gemm_up_backward",
    "grouped_gemm_down_backward",
    # Autograd wrappers
    "grouped_gemm_up_autograd",
    "grouped_gemm_down_autograd",
    # Gather map for fused gather
    "precompute_gather_map",
    # Autograd Function classes
    "GroupedGemmUp",
    "GroupedGemmDown",
    # Routing
    "fused_route",
    # Few tokens (generation): bf16, fp32 and 4-bit expert weights
    "few_token_experts",
    "quantize_experts",
    "quantize_matrices",
    "moe_few_tokens",
    "experts_few_tokens",
    "matvec_q4",
    "few_tokens_max",
    "FewTokenExperts",
    "QuantizedExperts",
    "QuantizedMatrices",
    # Dense operators beside the expert layer
    "layer_norm",
    "layer_norm_max",
    "fused_linear",
    "gated_mlp",
]
