"""nn surface of the path: Module, Parameter, Sequential, Linear, LayerNorm,
RMSNorm, Dropout, SiLU, GELU and the functional ops (reference
nn/__init__.py); LinearQ4 (4-bit weights), MoE (experts), and the causal
transformer block's GatedMLP, WindowAttention and DecoderBlock."""
from . import functional
from .layers import (GELU, DecoderBlock, Dropout, GatedMLP, LayerNorm, Linear, LinearQ4, MoE, Module, Parameter, RMSNorm,
                     Sequential, SiLU, WindowAttention)

__all__ = ["functional", "Module", "Parameter", "Sequential", "Linear", "LinearQ4", "MoE", "GatedMLP", "WindowAttention",
           "DecoderBlock", "LayerNorm", "RMSNorm", "Dropout", "SiLU", "GELU"]
