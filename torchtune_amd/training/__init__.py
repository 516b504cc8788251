from . import quantization
from .optim import AdamW

__all__ = ["AdamW", "quantization"]
