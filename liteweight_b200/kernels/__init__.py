"""Drop-in replacements of liteweight's ``kernels`` package (kernels/__init__.py:1-5).

Same names, signatures, dtype/shape assertions and output allocation as the
Triton originals; the work runs in the sm_100a CUDA library through its C ABI.

Beside them, without a counterpart there: the operators of a paged key-value
cache (qk_norm_rope, paged_attention, prompt_attention).
"""

from liteweight_b200.kernels.matmul_fp16 import matmul_fp16
from liteweight_b200.kernels.matmul_int4 import matmul_int4
from liteweight_b200.kernels.matmul_int8 import matmul_int8
from liteweight_b200.kernels.paged import check_device_error, paged_attention, prompt_attention, qk_norm_rope

__all__ = ["matmul_fp16", "matmul_int8", "matmul_int4", "qk_norm_rope", "paged_attention", "prompt_attention",
           "check_device_error"]
