"""Layers built from the package's operators, for prompts and single tokens."""

from .mamba import Mamba2Layer, MambaLayer  # noqa: F401
