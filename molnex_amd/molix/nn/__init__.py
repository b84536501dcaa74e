from .locality import NeighborList
from .norm import LayerNorm

__all__ = ["NeighborList", "LayerNorm"]
