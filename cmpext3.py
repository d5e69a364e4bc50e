"""Drop-in module name for the reference's matmul-path operators.

`import cmpext3` then `cmpext3.linear(...)`, `cmpext3.bmm(...)`,
`cmpext3.attention(...)`, `cmpext3.fp16_matmul(...)` etc. resolve to the
sm_100a implementations in cmp_ext_b200.  Provided: the dense matmul path,
conv2d's 1x1 case (which the reference routes through its matmul),
scaled dot-product attention (its QK^T and PV products), and, beyond the
reference, attention over packed sequences and paged caches with the cache's
write and read; the reference's other operators (general conv, norms, activations) are not part of this
build.
"""
from cmp_ext_b200 import (  # noqa: F401
    attention,
    attention_paged,
    attention_varlen,
    bf16_matmul,
    bmm,
    conv2d,
    fp16_matmul,
    fp32_matmul,
    kv_cache_read,
    kv_cache_write,
    linear,
)

__all__ = ["linear", "bmm", "conv2d", "attention", "attention_varlen", "attention_paged", "kv_cache_write",
           "kv_cache_read", "fp16_matmul", "bf16_matmul", "fp32_matmul"]
