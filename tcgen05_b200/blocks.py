"""Block-scaled E2M1 tensors: the operands of the MXF4, MXF4NVF4 and NVFP4
instructions made from real tensors, turned back, and multiplied.

``quantize_blocks`` rounds a CUDA tensor to E2M1 codes with one 8-bit scale per
block of 16 or 32 consecutive elements; the result, ``BlockScaledRows``, feeds
the emulator (``packed()`` and ``scale_words()`` are what ``mma_dot_batch``
takes) as well as ``block_scaled_mm``, which multiplies two of them on the
tensor cores.  ``dequantize_blocks`` gives the real values back and
``block_scaled_linear`` is a linear layer whose three products (output, input
gradient, weight gradient) all run in this arithmetic.

``scaling`` and ``scale_vec`` are make_model's: "ue4m3" with 4 (blocks of 16,
NVFP4), "ue8m0" with 2 (blocks of 32, MXF4) or 4 (blocks of 16).  Everything
runs on the current stream of the tensors' device, allocates its results and
workspaces there per call and keeps nothing between calls, so calls may run
side by side on several streams and be captured into CUDA graphs.  There is no
CPU fallback.
"""

from __future__ import annotations

import ctypes

import torch

from . import _native as nat
from . import packing
from .runtime import require_device
from .simulator import PackedRows

# (scaling, scale_vec) -> (scale format, elements per block)
_FORMS = {
    ("ue4m3", 4): (nat.SCALE_UE4M3, 16),
    ("ue8m0", 2): (nat.SCALE_UE8M0, 32),
    ("ue8m0", 4): (nat.SCALE_UE8M0, 16),
}
_ROUNDINGS = {"nearest": nat.SCALE_ROUND_NEAREST, "floor": nat.SCALE_ROUND_FLOOR, "ceil": nat.SCALE_ROUND_CEIL}


_F32_LARGEST, _F32_SMALLEST = torch.finfo(torch.float32).max, torch.finfo(torch.float32).smallest_normal


def _form(scaling, scale_vec) -> tuple[str, int]:
    scaling = str(scaling).lower()
    if scale_vec is None:
        scale_vec = 4 if scaling == "ue4m3" else 2
    if (scaling, scale_vec) not in _FORMS:
        raise ValueError(f"block-scaled E2M1 takes scaling 'ue4m3' with scale_vec 4 or 'ue8m0' with 2 or 4, "
                         f"not {scaling!r} with {scale_vec!r}")
    return scaling, scale_vec


def _rounding(scaling: str, scale_rounding) -> int:
    if scale_rounding is None:
        scale_rounding = "nearest" if scaling == "ue4m3" else "floor"
    if scale_rounding not in _ROUNDINGS or (scale_rounding == "nearest") != (scaling == "ue4m3"):
        raise ValueError(f"scale_rounding is 'floor' or 'ceil' for ue8m0 and 'nearest' for ue4m3, "
                         f"not {scale_rounding!r} for {scaling}")
    return _ROUNDINGS[scale_rounding]


# (scaling, scale_vec, scale_rounding) as a caller gives them -> what they mean
_CHOICES: dict = {}


def _choice(scaling, scale_vec, scale_rounding):
    """(scaling, scale_vec, rounding, scale format, elements per block)."""
    try:
        return _CHOICES[scaling, scale_vec, scale_rounding]
    except (KeyError, TypeError):
        pass
    name, vec = _form(scaling, scale_vec)
    found = (name, vec, _rounding(name, scale_rounding), *_FORMS[name, vec])
    if len(_CHOICES) < 64:
        _CHOICES[scaling, scale_vec, scale_rounding] = found
    return found


_loaded = None


def _ops():
    global _loaded
    if _loaded is None:
        _loaded = nat.torch_ops()
    return _loaded


def tile_scales(words: torch.Tensor) -> torch.Tensor:
    """[rows, blocks] scale bytes -> the tiles of t5e_blocks (include/t5e.h):
    [ceil(rows / 128), ceil(blocks / 4), 512] bytes, zeros where no block is."""
    if words.dim() != 2 or words.dtype != torch.uint8:
        raise ValueError("scale words are a [rows, blocks] uint8 tensor")
    rows, blocks = words.shape
    full = torch.zeros((rows + 127) // 128 * 128, (blocks + 3) // 4 * 4, dtype=torch.uint8, device=words.device)
    full[:rows, :blocks] = words
    tiles = full.view(full.shape[0] // 128, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return tiles.reshape(full.shape[0] // 128, full.shape[1] // 4, 512)


def untile_scales(tiles: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    """Inverse of tile_scales."""
    t = tiles.reshape(tiles.shape[0], tiles.shape[1], 32, 4, 4).permute(0, 3, 2, 1, 4)
    return t.reshape(tiles.shape[0] * 128, tiles.shape[1] * 4)[:rows, :blocks].contiguous()


class BlockScaledRows:
    """Rows of E2M1 codes with a scale per block: what PackedRows are for one
    format, with scales.

    ``data`` is a [rows, stride] uint8 tensor of packed rows (stride a multiple
    of 16, at least ``row_stride(k)``; codes behind k, up to the next multiple
    of 32, zero), ``scales`` the tiled scale bytes (``tile_scales``),
    ``multiplier`` a one-element float32 tensor that the values were
    multiplied by before rounding, or None: element i of row r stands for
    code * scale / multiplier.  The three tensors are held as they are, not
    copied; a call refuses rows whose memory was freed or moved since."""

    __slots__ = ("_rows", "scaling", "scale_vec")

    def __init__(self, data, scales, k: int, *, scaling: str = "ue4m3", scale_vec: int | None = None, multiplier=None):
        self.scaling, self.scale_vec, _, fmt, block = _choice(scaling, scale_vec, None)
        self._rows = _ops().Rows(data, scales, k, fmt, block, multiplier)

    @classmethod
    def _of(cls, rows, choice):
        self = cls.__new__(cls)
        self._rows = rows
        self.scaling, self.scale_vec = choice[0], choice[1]
        return self

    @classmethod
    def from_words(cls, words, scales, *, scaling: str = "ue4m3", scale_vec: int | None = None, multiplier=None):
        """From a [rows, K] CUDA tensor of raw E2M1 container words and
        [rows, blocks] scale bytes, as ``mma_dot_batch`` takes them (K up to
        its 65536)."""
        scaling, scale_vec = _form(scaling, scale_vec)
        _tensor(words, "words"), _tensor(scales, "scales")
        if words.dim() != 2 or words.dtype.is_floating_point or words.dtype.is_complex:
            raise ValueError("words must be a [rows, K] tensor of integers")
        rows, k = words.shape
        if not 1 <= k <= nat.MAX_K:
            raise ValueError(f"K must be between 1 and {nat.MAX_K}, not {k}")
        blocks = -(-k // _FORMS[scaling, scale_vec][1])
        if tuple(scales.shape) != (rows, blocks):
            raise ValueError(f"scales must be [{rows}, {blocks}] bytes")
        if not words.is_cuda or scales.device != words.device:
            raise ValueError("words and scales must be on one CUDA device (there is no CPU fallback)")
        with torch.cuda.device(words.device):
            data = packing.pack_rows_device(words, nat.FMT_E2M1, cls.row_stride(k))
        return cls(data, tile_scales(scales), k, scaling=scaling, scale_vec=scale_vec, multiplier=multiplier)

    @staticmethod
    def row_stride(k: int) -> int:
        """Smallest row stride in bytes: whole groups of 32 elements."""
        return (k + 31) // 32 * 16

    @property
    def rows(self) -> int:
        return self._rows.rows

    @property
    def k(self) -> int:
        return self._rows.k

    @property
    def block(self) -> int:
        """Elements per scale."""
        return self._rows.block

    @property
    def data(self) -> torch.Tensor:
        return self._rows.data

    @property
    def scales(self) -> torch.Tensor:
        return self._rows.scales

    @property
    def multiplier(self):
        return self._rows.multiplier

    @property
    def device(self):
        return self._rows.device

    def packed(self) -> PackedRows:
        """The codes as the emulator's operand rows."""
        return PackedRows(self.data, self.k)

    def scale_words(self) -> torch.Tensor:
        """[rows, blocks] scale bytes, as the emulator takes them."""
        return untile_scales(self.scales, self.rows, -(-self.k // self.block))

    def __repr__(self):
        return (f"BlockScaledRows({self.rows} x {self.k}, {self.scaling}, scale_vec={self.scale_vec}, "
                f"device={self.device})")


def _tensor(x, name: str):
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    return x


def block_multiplier(x) -> torch.Tensor:
    """The power of two that ``quantize_blocks(x, multiplier="auto")``
    multiplies by: the largest m, within 2^-126..2^126, for which every
    |x| * m <= 6 * 448, so that UE4M3 scales use their whole range; 1 where the
    largest |x| is zero or not finite.  A one-element float32 tensor, computed
    without a synchronization."""
    return _ops().multiplier(_tensor(x, "x"))


_AXES = {-1: 1, 0: 2, "both": 3}


def quantize_blocks(x, *, axis=-1, scaling: str = "ue4m3", scale_vec: int | None = None,
                    scale_rounding: str | None = None, multiplier=None):
    """Round a CUDA tensor (float32, bfloat16 or float16, any strides, at least
    one dimension) to block-scaled E2M1 rows.

    ``x`` is taken as a matrix of its last dimension [R, K].  ``axis=-1``
    rounds blocks along its rows (a BlockScaledRows of R rows and K elements),
    ``axis=0`` along its columns (K rows of R elements: the transposed
    operand), ``axis="both"`` returns the pair from one call.

    With u = x * multiplier rounded to float32 and a = max |u| of a block: a
    UE4M3 scale is a / 6 rounded to nearest (at most 448); a UE8M0 scale is
    2^(floor(log2 a) - 2) ("floor", the default) or the smallest power of two
    not below a / 6 ("ceil", nothing exceeds the E2M1 range).  Codes are u /
    scale rounded to nearest even, magnitudes above 6 become 6; both roundings
    are those of the real quotients.  A block that holds a NaN or an infinity
    gets the NaN scale, and everything computed from it is NaN.

    ``multiplier``: None (1), a positive float, a one-element float32 tensor, or
    "auto", ``block_multiplier(x)`` found in the same call.  The result keeps a
    given tensor's value of this call, whatever the tensor holds later; it has
    to be a positive normal number, which is not checked (that would take a
    synchronization).  The result carries no gradient (see
    ``block_scaled_linear``)."""
    choice = _choice(scaling, scale_vec, scale_rounding)
    axes = _AXES.get(axis)
    if axes is None:
        raise ValueError(f"axis is -1, 0 or 'both', not {axis!r}")
    automatic = False
    _tensor(x, "x")
    if multiplier is not None and not isinstance(multiplier, torch.Tensor):
        if isinstance(multiplier, str):
            if multiplier != "auto":
                raise ValueError(f"multiplier is a number, a tensor, 'auto' or None, not {multiplier!r}")
            multiplier, automatic = None, True
        else:
            multiplier = float(multiplier)
            if not _F32_SMALLEST <= multiplier <= _F32_LARGEST:
                raise ValueError(f"multiplier must be positive, finite and a normal float32, not {multiplier!r}")
            multiplier = torch.full((1,), multiplier, dtype=torch.float32, device=x.device)
    got = _ops().quantize(x, axes, choice[3], choice[4], choice[2], multiplier, automatic)
    if axes == 3:
        return BlockScaledRows._of(got[0], choice), BlockScaledRows._of(got[1], choice)
    return BlockScaledRows._of(got, choice)


def _rows_of(q, name: str):
    if not isinstance(q, BlockScaledRows):
        raise ValueError(f"{name} must be BlockScaledRows")
    return q._rows


def dequantize_blocks(blocks: BlockScaledRows, *, dtype=torch.float32, out=None) -> torch.Tensor:
    """The [rows, K] values code * scale / multiplier (times the reciprocal of
    the multiplier, rounded to float32) rounded to ``dtype``; into ``out`` (unit
    column stride) if given, which counts as a change in place."""
    return _ops().dequantize(_rows_of(blocks, "blocks"), dtype, out)


def block_scaled_mm(a: BlockScaledRows, b: BlockScaledRows, c=None, *, alpha: float = 1.0, dtype=torch.bfloat16,
                    out=None) -> torch.Tensor:
    """``D = alpha * A @ B.T + C`` on the tensor cores, in one kernel launch:
    ``a`` [M, K] and ``b`` [N, K] block-scaled rows of the same form (b's rows
    are the columns of B, as in the packed rows of ``mma_batch``); their
    multipliers are divided out.  ``c``: a real tensor that broadcasts to
    [M, N] (a bias, an accumulator), or None.  Returns [M, N] of ``dtype``, or
    ``out`` (unit column stride), which may be ``c`` itself.

    Sums are the instruction's own: float32 accumulators that take K in
    ascending steps of 64, each step truncated as ``mma_dot_batch`` models it
    word for word; where few tiles would leave the GPU idle, K is split into
    parts that are joined in float32.  So a float32 result is off, always toward
    zero, by up to 2^-23 of the running sum per step, about 5e-6 of it in all at
    K = 8192; the rounding of 16-bit results is larger.  alpha divided by the multipliers may
    leave float32's range where the results do not.

    ``c`` may not require a gradient or carry a forward-mode tangent, and the
    result carries neither (see ``block_scaled_linear``); writing to ``out``
    counts as a change in place."""
    return _mm(a, b, c, alpha, dtype, out, 0)


def _mm(a, b, c, alpha, dtype, out, form):
    """block_scaled_mm with t5e_block_mm's `form`."""
    if c is not None:
        _tensor(c, "c")
    return _ops().mm(_rows_of(a, "a"), _rows_of(b, "b"), c, alpha, dtype, out, form)


def block_scaled_mm_expired(device=None) -> bool:
    """Whether a bounded wait inside a product ran out on the device since the
    library was loaded (the tile concerned holds NaN); synchronizes the device."""
    device = require_device(device)
    flag = ctypes.c_int32(0)
    with torch.cuda.device(device):
        nat.check(nat.load().t5e_block_scaled_mm_expired(ctypes.byref(flag)), "t5e_block_scaled_mm_expired")
    return flag.value != 0


def block_scaled_linear(x, w, *, scaling: str = "ue4m3", scale_vec: int | None = None,
                        scale_rounding: str | None = None) -> torch.Tensor:
    """``x @ w.T`` with both rounded to block-scaled E2M1 rows, and its
    gradients in the same arithmetic:

        y  = Q(x) Q(w)^T           blocks along K
        dx = Q(g) Q(w^T)^T         blocks along N
        dw = Q(g^T) Q(x^T)^T       blocks along the tokens

    (the rounding itself passes gradients straight through).  ``x`` [..., K]
    and ``w`` [N, K] are CUDA tensors of one type; y, dx and dw have that type.
    UE4M3 forms take the "auto" multiplier for x, w and g.  x and w are read
    once each; a training step keeps their 4-bit transposes for the backward
    pass, not the tensors.  Differentiable once: under ``create_graph=True`` the
    gradients require gradients, and a backward pass through them is refused.
    Forward-mode tangents are refused."""
    choice = _choice(scaling, scale_vec, scale_rounding)
    return _ops().linear(_tensor(x, "x"), _tensor(w, "w"), choice[3], choice[4], choice[2])
