"""Model adapters (mirrors ``flashgrpo.models``): Medusa heads and the native target model."""
from .medusa_heads import ChainDraftCell, MedusaHeads, MedusaPredictionHead
from .target import KVCache, PagedKVCache, TargetConfig, TargetModel, forward_tree

__all__ = ["ChainDraftCell", "MedusaHeads", "MedusaPredictionHead", "KVCache", "PagedKVCache", "TargetConfig",
           "TargetModel", "forward_tree"]
