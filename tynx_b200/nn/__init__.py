"""Neural-network helpers for imported models (``tynx.nn`` subset on CUDA)."""

from . import functional
from .rotary import Rotary

__all__ = ["Rotary", "functional"]
