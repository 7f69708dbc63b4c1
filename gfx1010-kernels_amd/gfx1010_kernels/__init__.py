"""MI355X (gfx950) fused residual-add + dropout + LayerNorm.

Drop-in replacement for the residual LayerNorm surface of the reference
package (gfx1010_kernels/__init__.py:15-19): ``residual_layer_norm``,
``can_use_residual_layer_norm``, ``residual_layer_norm_status`` and
``BackendStatus``, plus the pre-norm integration helpers ``residual_norm``
and ``prenorm_forward`` (the reference's integration recipe,
docs/residual_layer_norm.md:51-83, as code), and the same operator with a
root-mean-square norm (``residual_rms_norm``, its 8-bit output
``residual_rms_norm_quantized`` and ``dequantize``), with norms on both sides of a
block and its gate (``gated_residual_rms_norm``), and the rotary norm of query and
key heads (``rms_norm_rotary``). The reference's attention, patch, linear and Triton
exports are not part of this build.
"""

from ._status import BackendStatus
from .gated_norm import (  # noqa: F401
    can_use_gated_residual_rms_norm,
    gated_residual_rms_norm,
)
from .normalization import (
    can_use_residual_layer_norm,
    residual_layer_norm,
    residual_layer_norm_status,
)
from .prenorm import prenorm_forward, residual_norm
from .rms_norm import (  # noqa: F401
    can_use_residual_rms_norm,
    dequantize,
    residual_rms_norm,
    residual_rms_norm_quantized,
)
from .rotary import (  # noqa: F401
    can_use_rms_norm_rotary,
    rms_norm_rotary,
    rotary_inverse_frequencies,
)

# API version of the reference surface this package reproduces.
__version__ = "0.4.0"

# What a star import of the reference's package surface brings; the names of
# rms_norm.py, gated_norm.py and rotary.py are imported by name (their own __all__
# list them).
__all__ = [
    "__version__",
    "BackendStatus",
    "can_use_residual_layer_norm",
    "prenorm_forward",
    "residual_layer_norm",
    "residual_layer_norm_status",
    "residual_norm",
]
