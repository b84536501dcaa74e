from .locality import get_neighbor_pairs, neighbor_list
from .norm import layer_norm
from .optim import adamw8_moments, adamw8_step, adamw_step, grad_norm
from .pot import pme_direct, pme_reciprocal
from .scatter import batch_add, scatter_sum

__all__ = ["get_neighbor_pairs", "neighbor_list", "pme_direct", "pme_reciprocal", "scatter_sum", "batch_add",
           "layer_norm", "adamw_step", "adamw8_step", "adamw8_moments", "grad_norm"]
