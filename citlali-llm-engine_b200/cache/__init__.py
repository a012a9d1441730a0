from .allocators import PageAllocator, SlotAllocator
from .sequence_cache import (PAGE_SIZE, KVRequirement, KVView, Packed4, SequenceCache, StateRequirement, StateView)
