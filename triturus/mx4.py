"""Import path beside the reference's modules: ``from triturus.mx4 import mm_mx4``."""
from triturus_amd.mx4 import MX4, mm_mx4, mx4_dequantize, mx4_quantize  # noqa: F401
