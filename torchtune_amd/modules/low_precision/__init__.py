from .mx_linear import FrozenMXLinear
from .nf4_linear import FrozenNF4Linear

__all__ = ["FrozenMXLinear", "FrozenNF4Linear"]
