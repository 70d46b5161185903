"""mtp_b200: B200-native (sm_100a) GPTQ-int4 W4A16 mixture-of-experts layer
forward and its MTP-driven expert-prefetch path.

Around them: an int8 (W8A8) expert path, the sort of tokens by expert, and what
training such a layer needs beside that (router with losses, layer norm,
embedding).

The compute runs in ``lib/libmtp_b200.so`` (hand-written CUDA behind a C ABI,
``include/mtp_b200.h``); this package is the host-side mirror of the reference
interfaces. There is no CPU fallback.
"""
from ._lib import MtpError, load as load_library  # noqa: F401
from .ep import ExpertParallelMoE, plan_dispatch  # noqa: F401
from .ops import (  # noqa: F401
    HiddenResidualPredictor,
    MtpPredictor,
    PrefetchSession,
    SharedExpert,
    W4A16Experts,
    dequantize_gptq_projection,
    experts_from_vllm_wna16,
    fused_experts,
    layer_path,
    layer_workspace,
    moe_align_block_size,
    moe_layer_w4a16,
    prefill_workspace,
    topk_softmax,
    vllm_wna16_to_gptq,
)
from .training import (  # noqa: F401
    RoutedTokens,
    embed_tokens,
    layer_norm,
    route_tokens,
)
from .w8a8 import (  # noqa: F401
    SortedTokens,
    int8_grouped_matmul,
    int8_linear,
    int8_matmul,
    moe_layer_w8a8,
    quantize_int8,
    sort_tokens,
    unsort_tokens,
)

__all__ = [
    "ExpertParallelMoE",
    "HiddenResidualPredictor",
    "MtpError",
    "MtpPredictor",
    "PrefetchSession",
    "RoutedTokens",
    "load_library",
    "SharedExpert",
    "SortedTokens",
    "W4A16Experts",
    "dequantize_gptq_projection",
    "embed_tokens",
    "experts_from_vllm_wna16",
    "fused_experts",
    "int8_grouped_matmul",
    "int8_linear",
    "int8_matmul",
    "layer_norm",
    "layer_path",
    "layer_workspace",
    "moe_align_block_size",
    "moe_layer_w4a16",
    "moe_layer_w8a8",
    "plan_dispatch",
    "prefill_workspace",
    "quantize_int8",
    "route_tokens",
    "sort_tokens",
    "topk_softmax",
    "unsort_tokens",
    "vllm_wna16_to_gptq",
]
