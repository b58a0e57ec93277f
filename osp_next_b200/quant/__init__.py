"""Fake quantisation: HiF8 linears / attention (the OSP-Next model's quant path, hif8.py)
and the rest of the quant_cy_npu library surface (layers.py); linears that compute in
block-scaled fp8 (fp8.py)."""
from .hif8 import (HIF8Linear, QLinear, QType, hif8_multi_linear, hif8_qkv, quant, quant_dequant_float,  # noqa: F401
                   quant_hif8, replace_linear)
from .layers import BlockFloatFormat, QConv2d, QSLinear, SLinear, quant_block_float, quant_py  # noqa: F401
from .fp8 import FP8Linear, fp8_linear, fp8_multi_linear, freeze_fp8_weights  # noqa: F401
