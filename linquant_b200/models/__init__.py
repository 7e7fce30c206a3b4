"""Layers built from the package's operators, for prompts and single tokens."""

from .linear_attention import LinearAttentionLayer  # noqa: F401
from .mamba import Mamba2Layer, MambaLayer  # noqa: F401
