from .attn_engine import AttentionEngine, OnlineFunc
from .cache8 import PagedCache8, PagePlan, plan_pages
from .linear_attn_engine import LinearAttentionEngine

__all__ = ["AttentionEngine", "OnlineFunc", "LinearAttentionEngine", "PagedCache8", "PagePlan", "plan_pages"]
