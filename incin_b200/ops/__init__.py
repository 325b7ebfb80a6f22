"""Hand-written sm_100a ops (CUDA) with PyTorch-CPU twins."""
from . import functional  # noqa: F401
from .functional import (causal_attention, copy_pages, cross_entropy, decode_attention, embedding, kv_append,  # noqa: F401
                         layer_norm, layernorm_fork, linear, mlp, prompt_attention, rms_norm, rmsnorm_fork, rope, swiglu)
