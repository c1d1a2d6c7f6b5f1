"""hydra_amd.attention -- the surface of hydra/attention/__init__.py."""

from .registry import (
    HybridAttentionBackend,
    available_hybrid_attention_backends,
    is_hybrid_attention_backend_available,
    resolve_hybrid_attention_backend,
)
from .backends.ccgqa.attention import CCGQAAttention, CCGQACache
from .factory import build_hybrid_attention_module
from .paged import PagePlan, PagePool, paged_attention, plan_pages, release_pages, store_pages

__all__ = [
    "HybridAttentionBackend",
    "available_hybrid_attention_backends",
    "is_hybrid_attention_backend_available",
    "resolve_hybrid_attention_backend",
    "CCGQAAttention",
    "CCGQACache",
    "build_hybrid_attention_module",
    "PagePlan",
    "PagePool",
    "paged_attention",
    "plan_pages",
    "release_pages",
    "store_pages",
]
