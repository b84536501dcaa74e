"""The AdamW step over lists of tensors (``molix.optim.AdamW`` calls it) and the norm of their gradients."""

from ...training import adamw8_moments, adamw8_step, adamw_step, grad_norm

__all__ = ["adamw_step", "adamw8_step", "adamw8_moments", "grad_norm"]
