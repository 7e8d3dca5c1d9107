"""flashinfer_b200 -- B200-native (sm_100a) fused FP8 block-scale MoE with DeepSeek-V3 routing.

Drop-in for the reference operator ``solution/triton/kernel.py::run`` of the
FlashInfer-Bench ``fused_moe`` solution
(``moe_fp8_block_scale_ds_routing_topk8_ng8_kg4_e32_h7168_i2048``). The compute
path is hand-written CUDA behind the C ABI of ``include/fmoe.h``; expert
parallelism over several GPUs is in ``flashinfer_b200.ep``. The operators around the experts --
tokens sorted by expert and back, products with 8-bit and 4-bit weights, norms, the router's balance
loss -- are in ``tokens``, ``int8``, ``int4``, ``norm`` and ``balance``.
"""
from .moe import run, route, quantize_activations, read_status, workspace_for, WorkspaceView  # noqa: F401,E501

from .balance import balance_loss, expert_counts
from .int4 import (dequantize_int4, int4_expert_matmul, int4_matmul, int4_status,
                   quantize_int4)
from .int8 import int8_expert_matmul, int8_matmul, int8_status, quantize_int8
from .norm import block_norm, layer_norm
from .tokens import ExpertOrder, sort_by_expert, sort_tokens, unsort_tokens

__all__ = ["run", "route", "read_status", "workspace_for", "WorkspaceView",
           "ExpertOrder", "sort_by_expert", "sort_tokens", "unsort_tokens",
           "quantize_int8", "int8_matmul", "int8_expert_matmul", "int8_status", "block_norm",
           "layer_norm", "balance_loss", "expert_counts",
           "quantize_int4", "dequantize_int4", "int4_matmul", "int4_expert_matmul",
           "int4_status"]
