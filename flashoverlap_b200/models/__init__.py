"""nn.Modules built on the fused operations."""
from .kv_cache import PagedKVCache  # noqa: F401
from .rmsnorm import RMSNorm, ReorderRMSNorm  # noqa: F401
from .row_parallel import (  # noqa: F401
    FusedRowParallelLinear,
    HierarchicalRowParallelLinear,
    OverlapRowParallelLayer,
    RowParallelLayer,
)
