from .need import CacheNeed
from .pages import CacheFull, FreeList, PageBook
from .kv8 import LayerKV8
from .kv import TOKENS_PER_PAGE, EntryView, LayerKV, SequenceCache

__all__ = ["CacheNeed", "CacheFull", "FreeList", "PageBook", "TOKENS_PER_PAGE", "EntryView", "LayerKV", "LayerKV8",
           "SequenceCache"]
