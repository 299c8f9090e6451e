"""Layers built on the attention operators."""

from .cross_attention import RotaryCrossAttn
from .msda import MultiScaleDeformAttn2d

__all__ = ["MultiScaleDeformAttn2d", "RotaryCrossAttn"]
