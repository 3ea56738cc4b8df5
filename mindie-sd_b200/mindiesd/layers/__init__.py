from .flash_attn import attention_forward, attention_forward_varlen, attention_forward_host, sparse_attention
from .linear import linear_forward
from .norm import add_rms_norm, add_rms_norm_quant
from .rope import rotary_position_embedding

__all__ = ["attention_forward", "attention_forward_varlen", "attention_forward_host", "sparse_attention",
           "add_rms_norm", "add_rms_norm_quant", "linear_forward", "rotary_position_embedding"]
