"""Functional wrappers over the native operators."""
from .attention import (  # noqa: F401
    attention_reset,
    attention_set_timeout_ms,
    attention_status,
    cache_append,
    copy_pages,
    paged_attention,
    prompt_attention,
)
from .functional import (  # noqa: F401
    a2a_dispatch_gemm,
    allgather_gemm,
    gemm,
    gemm_allreduce,
    gemm_reducescatter,
    gemm_rmsnorm,
    reorder_rmsnorm,
    rmsnorm,
)
