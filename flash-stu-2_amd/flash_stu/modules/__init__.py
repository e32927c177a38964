from .attention import Attention
from .norm import RMSNorm
from .stu import STU
from .swiglu import FP8MLP, MLP

__all__ = ["STU", "Attention", "MLP", "FP8MLP", "RMSNorm"]
