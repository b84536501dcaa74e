from .adamw import AdamW
from .muon import Muon

__all__ = ["AdamW", "Muon"]
