"""tcgen05_b200 -- a B200-native (sm_100a) batched emulator of NVIDIA
Blackwell tcgen05 MMA arithmetic, bit-exact with the tcgen05_model
reference package and a drop-in for its API.

Scalar and matrix calls (``mma_dot``, ``mma``, ``make_model(...).eval``)
keep the reference's signatures and errors; ``mma_dot_batch`` and
``mma_batch`` evaluate millions of independent dot products or tiles per
kernel launch.  Every result word is computed by hand-written integer CUDA
kernels in ``tcgen05_b200/_lib/libt5e.so``; there is no CPU fallback.

Real tensors meet that arithmetic in ``quantize_blocks`` (tensors to
block-scaled E2M1 rows: the operands of the MXF4, MXF4NVF4 and NVFP4
instructions), ``dequantize_blocks``, ``block_scaled_mm`` (their matrix product
on the tensor cores) and ``block_scaled_linear`` (a linear layer with its
gradients).
"""

import importlib.util as _util

from .formats import bits_to_f32, f32_to_bits
from .model import (
    DotProduct,
    ScalarModel,
    Tcgen05BlockScaledMmaModel,
    Tcgen05I8S32MmaModel,
    Tcgen05MixedRawWindowMmaModel,
    Tcgen05RawWindowNvfp4MmaModel,
    make_model,
    normalize_format,
)
from .simulator import PackedRows, PendingBatch, mma, mma_batch, mma_dot, mma_dot_batch, sparse_active_indices

# in .blocks, which imports PyTorch; the other modules do so when they compute
_BLOCK_SCALED = frozenset((
    "BlockScaledRows",
    "block_multiplier",
    "block_scaled_linear",
    "block_scaled_mm",
    "block_scaled_mm_expired",
    "dequantize_blocks",
    "quantize_blocks",
))


def __getattr__(name: str):
    if name in _BLOCK_SCALED:
        from . import blocks

        globals().update({n: getattr(blocks, n) for n in _BLOCK_SCALED})
        return globals()[name]
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


__all__ = [
    "DotProduct",
    "PackedRows",
    "PendingBatch",
    "ScalarModel",
    "Tcgen05BlockScaledMmaModel",
    "Tcgen05I8S32MmaModel",
    "Tcgen05MixedRawWindowMmaModel",
    "Tcgen05RawWindowNvfp4MmaModel",
    "bits_to_f32",
    "f32_to_bits",
    "make_model",
    "mma",
    "mma_batch",
    "mma_dot",
    "mma_dot_batch",
    "normalize_format",
    "sparse_active_indices",
]

# `from tcgen05_b200 import *` works without PyTorch, as it did before these
if _util.find_spec("torch") is not None:
    __all__ += sorted(_BLOCK_SCALED)
