"""The NF4-path pieces of the reference's attention module (solution/attn.py) under its names:
RoPE of q/k (FusedQKRope, solution/attn.py:89-126) and the LoRA dropout helpers (pack_keep,
_lora_inputs, solution/attn.py:183-203) and LoRAPairFromNorm (solution/attn.py:206-273, same
`apply` signature), backed by this package's HIP kernels; with them, under names of their own, the
attention inputs the reference lacks: seeded LoRA dropout, q/k norms, several position axes."""

from .lora import (LoRAPair, LoRAPairFromNorm, LoRAPairSeeded, lora_input_grad, lora_inputs,  # noqa: F401
                   pack_keep)
from .rope import (FusedQKRope, axes_rope, qk_norm_rope, rope_qk_backward, rope_qk_forward)  # noqa: F401


def _lora_inputs(x, bits_q, bits_v, scale_q, scale_v):
    """fp16(x * dropout values) of the q and v branches, [T, W] each (solution/attn.py:183-192)."""
    return lora_inputs(x, bits_q, bits_v, scale_q, scale_v)
