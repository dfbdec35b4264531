"""B200 (sm_100a) decode kernels behind the ``crossdsl_kernels`` op signatures.

Four forward decode ops -- fused residual RMSNorm, the FP32 small-M projection,
fused RoPE + paged K/V append, and the W4A16 INT4 projection -- implemented as
hand-written CUDA in ``libxdk_b200.so`` (C ABI: include/xdk_b200.h) and reached
from Python through ctypes.  There is no CPU or alternative-backend path.  Beside them: paged
decode attention and SwiGLU (``ops``), and a paged K/V cache in 8 bits with its append, attention
and selection of pages (``kv8``).
"""

__version__ = "0.1.0"

__all__ = ["__version__"]
