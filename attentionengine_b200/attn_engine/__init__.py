from .attn_engine import AttentionEngine, OnlineFunc
from .cache8 import PagedCache8, PagePlan, plan_pages
from .linear_attn_engine import LinearAttentionEngine
from .pages import CompactionPlan, ForkPlan, copy_pages, plan_compaction, plan_forks
from .rotary import QKNormRope

__all__ = ["AttentionEngine", "OnlineFunc", "LinearAttentionEngine", "PagedCache8", "PagePlan", "plan_pages", "ForkPlan", "plan_forks",
           "CompactionPlan", "plan_compaction", "copy_pages", "QKNormRope"]
