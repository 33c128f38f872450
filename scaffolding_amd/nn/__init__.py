"""nn surface of the path: Module, Parameter, Sequential, Linear, LayerNorm,
RMSNorm, Dropout, SiLU, GELU and the functional ops (reference
nn/__init__.py); LinearQ4 (4-bit weights) and MoE (experts)."""
from . import functional
from .layers import GELU, Dropout, LayerNorm, Linear, LinearQ4, MoE, Module, Parameter, RMSNorm, Sequential, SiLU

__all__ = ["functional", "Module", "Parameter", "Sequential", "Linear", "LinearQ4", "MoE", "LayerNorm", "RMSNorm", "Dropout",
           "SiLU", "GELU"]
