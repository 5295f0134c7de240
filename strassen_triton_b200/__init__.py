"""B200-native Strassen / Strassen-Winograd matrix multiplication (sm_100a CUDA behind a C ABI).

`strassen_triton_b200.ops.matmul` is the tensor-level entry, with the operators of a training step beside
it (`linear_act`, `layer_norm`, `token_logprobs`, `cross_entropy`, `clip_grad_norm_`); the modules `strassen`,
`strassen_2_layer`, `fixed_strassen`, `fixed_strassen_fp32_agg` and `model.layers` at the
repository root keep the reference project's names and signatures on top of it.
"""
from . import _lib  # noqa: F401
from .grads import clip_grad_norm_, clip_grads_, grad_norm  # noqa: F401
from .loss import TokenLogprobs, cross_entropy, token_logprobs  # noqa: F401
from .norm import LayerNorm, layer_norm  # noqa: F401
from .ops import device_status, linear_act, matmul, matmul_autograd, matmul_out  # noqa: F401

__all__ = ["matmul", "matmul_out", "matmul_autograd", "device_status", "linear_act", "layer_norm", "LayerNorm",
           "token_logprobs", "TokenLogprobs", "cross_entropy", "grad_norm", "clip_grads_", "clip_grad_norm_"]
