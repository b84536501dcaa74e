from .indexed import IndexedLinear
from .locality import NeighborList
from .norm import LayerNorm

__all__ = ["NeighborList", "LayerNorm", "IndexedLinear"]
