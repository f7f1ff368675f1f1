"""Approximate convolution layers and their autograd Functions (same exports as approxtorch/nn/__init__.py:4-9,
minus the naive comparison operators), plus a fully connected layer on the same kernels, one on the block-scaled 8-bit
floating point product, and dropout from a counter-based generator."""
from .Conv2d_int8 import Conv2d_int8
from .Conv2d_uint8 import Conv2d_uint8
from .Linear_int8 import Linear_int8
from .Linear_fp8 import Linear_fp8
from .dropout import CounterDropout
from . import bgemm_int8
from . import bgemm_uint8
from . import dropout
from . import gemm_fp8
from . import quantization
