from .attention import attention
from .fmm import fmm
from .fmmv import fdmmv, fmmv
from .layer_norm import layer_norm

__all__ = ("attention", "fmm", "fmmv", "fdmmv", "layer_norm")
