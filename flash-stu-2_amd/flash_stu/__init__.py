"""Flash STU's inference path on MI355X: the reference's public names
(flash_stu/__init__.py:1-15) backed by libflashstu_hip.so."""
from ._hip import glu_fp8, linear_fp8, quantize_fp8, quantize_weight_fp8, rms_norm_fp8
from .blocks.block import FlashSTUBlock
from .config import FlashSTUConfig
from .model import FlashSTU
from .modules.attention import Attention
from .modules.stu import STU
from .modules.swiglu import FP8MLP
from .utils.stu_utils import convolve, get_spectral_filters

__all__ = ["FlashSTU", "FlashSTUConfig", "FlashSTUBlock", "STU", "Attention", "get_spectral_filters", "convolve",
           "quantize_fp8", "quantize_weight_fp8", "rms_norm_fp8", "linear_fp8", "glu_fp8", "FP8MLP"]
