from .feed_forward import GatedFeedForward
from .sage import SAGE

__all__ = ["SAGE", "GatedFeedForward"]
