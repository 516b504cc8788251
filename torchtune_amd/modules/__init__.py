from .low_precision import FrozenMXLinear, FrozenNF4Linear
from .peft import LoRALinear, MXLoRALinear, QATLoRALinear

__all__ = ["FrozenMXLinear", "FrozenNF4Linear", "LoRALinear", "MXLoRALinear", "QATLoRALinear"]
