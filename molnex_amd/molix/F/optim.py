"""Optimizer steps over lists of tensors: AdamW (``molix.optim.AdamW`` calls it) and the norm of the gradients, Muon
(``molix.optim.Muon``) and the orthogonalisation of its updates."""

from ...training import adamw8_moments, adamw8_step, adamw_step, grad_norm, muon_step, orthogonalize

__all__ = ["adamw_step", "adamw8_step", "adamw8_moments", "grad_norm", "muon_step", "orthogonalize"]
