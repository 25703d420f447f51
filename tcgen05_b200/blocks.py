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
import struct

import torch

from . import _native as nat
from . import packing
from .runtime import require_device
from .simulator import PackedRows

_REAL = {torch.float32: nat.REAL_F32, torch.bfloat16: nat.REAL_BF16, torch.float16: nat.REAL_F16}
# (scaling, scale_vec) -> (scale format, elements per block)
_FORMS = {
    ("ue4m3", 4): (nat.SCALE_UE4M3, 16),
    ("ue8m0", 2): (nat.SCALE_UE8M0, 32),
    ("ue8m0", 4): (nat.SCALE_UE8M0, 16),
}
_pack_blocks = struct.Struct(nat.BLOCKS_FORMAT).pack
_pack_quantize = struct.Struct(nat.QUANTIZE_FORMAT).pack
_pack_mm = struct.Struct(nat.BLOCK_MM_FORMAT).pack
_NO_BLOCKS = (0, 0, 0, 0, 0, 0, 0)
_ROUNDINGS = {"nearest": nat.SCALE_ROUND_NEAREST, "floor": nat.SCALE_ROUND_FLOOR, "ceil": nat.SCALE_ROUND_CEIL}


_MOST = min(nat.MAX_BLOCK_K, nat.MAX_BLOCK_ROWS)
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
    code * scale / multiplier."""

    __slots__ = ("scaling", "scale_vec", "device", "multiplier", "_data", "_scales", "_buffer", "_fields")

    def __init__(self, data, scales, k: int, *, scaling: str = "ue4m3", scale_vec: int | None = None, multiplier=None):
        scaling, scale_vec = _form(scaling, scale_vec)
        fmt, block = _FORMS[scaling, scale_vec]
        k = int(k)
        if not 1 <= k <= nat.MAX_BLOCK_K:
            raise ValueError(f"K={k} outside 1..{nat.MAX_BLOCK_K}")
        if data.dim() != 2 or data.dtype != torch.uint8 or (data.shape[0] and not data.is_contiguous()):
            raise ValueError("data must be a contiguous [rows, stride] uint8 tensor")
        rows, stride = data.shape
        if rows > nat.MAX_BLOCK_ROWS:
            raise ValueError(f"more than {nat.MAX_BLOCK_ROWS} rows")
        if stride % 16 or stride < self.row_stride(k):
            raise ValueError(f"row stride {stride} is not a multiple of 16 of at least {self.row_stride(k)}")
        tiles, groups = (rows + 127) // 128, -(-k // (4 * block))
        if scales.dtype != torch.uint8 or scales.shape != (tiles, groups, 512) or not scales.is_contiguous():
            raise ValueError(f"scales must be a contiguous [{tiles}, {groups}, 512] uint8 tensor (tile_scales)")
        if scales.device != data.device:
            raise ValueError("data and scales are on different devices")
        if multiplier is not None:
            if multiplier.dtype != torch.float32 or multiplier.numel() != 1 or multiplier.device != data.device:
                raise ValueError("multiplier must be a one-element float32 tensor on the data's device")
        at, scales_at = data.data_ptr(), scales.data_ptr()
        if at % 16 or scales_at % 16:
            raise ValueError("data and scales must start on 16-byte boundaries")
        self.scaling, self.scale_vec, self.device, self.multiplier = scaling, scale_vec, data.device, multiplier
        self._data, self._scales, self._buffer = data, scales, None
        self._fields = (at, stride, scales_at, rows, k, fmt, block)  # t5e_blocks

    @classmethod
    def _new(cls, device, rows, k, choice, multiplier):
        """An instance over one new allocation: the rows, then the scale tiles.
        The views are made when they are asked for."""
        self = cls.__new__(cls)
        self.scaling, self.scale_vec, _, fmt, block = choice
        stride = (k + 31) // 32 * 16
        size = rows * stride
        self._buffer = buffer = torch.empty(size + (rows + 127) // 128 * (-(-k // (4 * block)) * 512), dtype=torch.uint8,
                                            device=device)
        self.device, self.multiplier, self._data, self._scales = device, multiplier, None, None
        at = buffer.data_ptr()
        self._fields = (at, stride, at + size, rows, k, fmt, block)
        return self

    @classmethod
    def from_words(cls, words, scales, *, scaling: str = "ue4m3", scale_vec: int | None = None, multiplier=None):
        """From a [rows, K] CUDA tensor of raw E2M1 container words and
        [rows, blocks] scale bytes, as ``mma_dot_batch`` takes them."""
        scaling, scale_vec = _form(scaling, scale_vec)
        if words.dim() != 2:
            raise ValueError("words must be a [rows, K] tensor of words")
        rows, k = words.shape
        blocks = -(-k // _FORMS[scaling, scale_vec][1])
        if tuple(scales.shape) != (rows, blocks):
            raise ValueError(f"scales must be [{rows}, {blocks}] bytes")
        data = packing.pack_rows_device(words, nat.FMT_E2M1, cls.row_stride(k))
        return cls(data, tile_scales(scales), k, scaling=scaling, scale_vec=scale_vec, multiplier=multiplier)

    @staticmethod
    def row_stride(k: int) -> int:
        """Smallest row stride in bytes: whole groups of 32 elements."""
        return (k + 31) // 32 * 16

    @property
    def rows(self) -> int:
        return self._fields[3]

    @property
    def k(self) -> int:
        return self._fields[4]

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            stride = self._fields[1]
            self._data = self._buffer[:self.rows * stride].view(self.rows, stride)
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buffer[self.rows * self._fields[1]:].view(
                (self.rows + 127) // 128, -(-self.k // (4 * self.block)), 512)
        return self._scales

    @property
    def block(self) -> int:
        """Elements per scale."""
        return self._fields[6]

    def packed(self) -> PackedRows:
        """The codes as the emulator's operand rows."""
        return PackedRows(self.data, self.k)

    def scale_words(self) -> torch.Tensor:
        """[rows, blocks] scale bytes, as the emulator takes them."""
        return untile_scales(self.scales, self.rows, -(-self.k // self.block))

    def __repr__(self):
        return (f"BlockScaledRows({self.rows} x {self.k}, {self.scaling}, scale_vec={self.scale_vec}, "
                f"device={self.device})")


def _call(fn, index, *args):
    """A library call on the current stream of the device of index `index`, which
    is made current for it."""
    if torch._C._cuda_getDevice() == index:
        # torch.cuda.current_stream(index).cuda_stream, without building a Stream
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        nat.check(rc, fn.__name__)


def _real_tensor(x, name: str):
    if not isinstance(x, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if x.dtype not in _REAL:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {x.dtype}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device (there is no CPU fallback)")


def _matrix_of(x):
    """(matrix, stride, turned): x as rows of its last dimension with unit column
    stride, or `turned`, the matrix whose columns those rows are (no copy of a
    transposed matrix); other layouts are copied."""
    if x.is_neg():
        x = x.detach().resolve_neg()
    if x.dim() != 2:
        x = x.detach().reshape(-1, x.shape[-1])
    rows, cols = x.shape
    down, across = x.stride()
    if (across == 1 or cols == 1) and (rows == 1 or down >= cols):
        return x, rows, cols, down, False
    if down == 1 and across >= rows:
        return x, cols, rows, across, True
    return x.detach().contiguous(), rows, cols, cols, False


def _partial_count(n: int) -> int:
    """Blocks that look for the largest of n elements: 8192 elements each, up
    to four per multiprocessor."""
    return min(592, -(-n // 8192)) or 1


def block_multiplier(x) -> torch.Tensor:
    """The power of two that ``quantize_blocks(x, multiplier="auto")``
    multiplies by: the largest m, within 2^-126..2^126, for which every
    |x| * m <= 6 * 448, so that UE4M3 scales use their whole range; 1 where the
    largest |x| is zero or not finite.  A one-element float32 tensor, computed
    without a synchronization."""
    _real_tensor(x, "x")
    if x.dim() == 0:
        x = x.reshape(1)
    lib = nat.load()
    n = x.numel()
    if n == 0:
        return torch.ones(1, dtype=torch.float32, device=x.device)
    m, rows, cols, stride, _ = _matrix_of(x)
    count = _partial_count(n)
    work = torch.empty(1 + count, dtype=torch.float32, device=m.device)
    at = work.data_ptr()
    _call(lib.t5e_block_multiplier, x.device.index, _REAL[m.dtype], m.data_ptr(), rows, cols, stride, at + 4, count, at)
    return work[:1]


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
    "auto", ``block_multiplier(x)`` found in the same call.  The result carries
    no gradient (see ``block_scaled_linear``)."""
    choice = _choice(scaling, scale_vec, scale_rounding)
    if axis not in (-1, 0, "both"):
        raise ValueError(f"axis is -1, 0 or 'both', not {axis!r}")
    if multiplier is not None:
        if isinstance(multiplier, str):
            if multiplier != "auto":
                raise ValueError(f"multiplier is a number, a tensor, 'auto' or None, not {multiplier!r}")
        elif not isinstance(multiplier, torch.Tensor):
            multiplier = float(multiplier)
            if not _F32_SMALLEST <= multiplier <= _F32_LARGEST:
                raise ValueError(f"multiplier must be positive, finite and a normal float32, not {multiplier!r}")
    _real_tensor(x, "x")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError("x must have at least one dimension and a non-empty last one")
    if isinstance(multiplier, torch.Tensor) and (multiplier.dtype != torch.float32 or multiplier.numel() != 1
                                                 or multiplier.device != x.device):
        raise ValueError("multiplier must be a one-element float32 tensor on x's device")
    k = shape[-1]
    r = x.numel() // k
    by_rows, by_cols = axis != 0, axis != -1
    if r > _MOST or k > _MOST:
        if (by_rows and k > nat.MAX_BLOCK_K) or (by_cols and r > nat.MAX_BLOCK_K) or max(r, k) > nat.MAX_BLOCK_ROWS:
            raise ValueError(f"x is larger than {nat.MAX_BLOCK_K} elements along a block axis or {nat.MAX_BLOCK_ROWS} rows")
    if by_cols and r == 0:
        raise ValueError("blocks along an empty axis")
    device = x.device
    partials = count = at = 0
    if multiplier is not None:
        if isinstance(multiplier, torch.Tensor):
            at = multiplier.data_ptr()
        elif isinstance(multiplier, float):
            multiplier = torch.full((1,), multiplier, dtype=torch.float32, device=device)
            at = multiplier.data_ptr()
        elif r:
            count = _partial_count(r * k)
            work = torch.empty(1 + count, dtype=torch.float32, device=device)
            at = work.data_ptr()
            partials, multiplier = at + 4, work[:1]
        else:
            multiplier = None
    rows = BlockScaledRows._new(device, r, k, choice, multiplier) if by_rows else None
    cols = BlockScaledRows._new(device, k, r, choice, multiplier) if by_cols else None
    if r:
        m, m_rows, m_cols, stride, turned = _matrix_of(x)
        along = _NO_BLOCKS if rows is None else rows._fields
        across = _NO_BLOCKS if cols is None else cols._fields
        if turned:
            along, across = across, along
        _call(nat.load().t5e_quantize_blocks, device.index,
              _pack_quantize(m.data_ptr(), m_rows, m_cols, stride, _REAL[m.dtype], choice[2], at, partials, count, 0, *along,
                             *across), 1)
    if rows is None:
        return cols
    return rows if cols is None else (rows, cols)


def _check_blocks(q, name: str):
    if not isinstance(q, BlockScaledRows):
        raise ValueError(f"{name} must be BlockScaledRows")
    if q.device.type != "cuda":
        raise ValueError(f"{name} must be on a CUDA device (there is no CPU fallback)")


def _result(out, shape, dtype, device):
    """The result tensor: `out` checked, or a new one."""
    if out is None:
        return torch.empty_strided(shape, (shape[1], 1), dtype=dtype, device=device)
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != device:
        raise ValueError(f"out must be a {tuple(shape)} {dtype} tensor on {device}")
    if out.numel() and ((out.shape[1] > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1])):
        raise ValueError("out must have unit column stride and rows that do not overlap")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out must not require a gradient")
    return out


def dequantize_blocks(blocks: BlockScaledRows, *, dtype=torch.float32, out=None) -> torch.Tensor:
    """The [rows, K] values code * scale / multiplier (times the reciprocal of
    the multiplier, rounded to float32) rounded to ``dtype``; into ``out`` (unit
    column stride) if given."""
    _check_blocks(blocks, "blocks")
    if dtype not in _REAL:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    given = out is not None
    out = _result(out, (blocks.rows, blocks.k), dtype, blocks.device)
    if given:
        _apart(out, blocks, "blocks")
    m = blocks.multiplier
    _call(nat.load().t5e_dequantize_blocks, blocks.device.index, _pack_blocks(*blocks._fields),
          None if m is None else m.data_ptr(), _REAL[dtype], out.data_ptr(),
          out.stride(0) if given and blocks.rows > 1 else blocks.k)
    return out


def _span(t):
    """[first, behind the last) byte of a tensor's elements."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _apart(out, blocks, name):
    """Refuses an `out` that shares memory with the blocks it is computed from."""
    if out.numel():
        d0, d1 = _span(out)
        at, stride, scales, rows, k, _, block = blocks._fields
        for lo, hi in ((at, at + rows * stride), (scales, scales + (rows + 127) // 128 * (-(-k // (4 * block)) * 512))):
            if lo < d1 and d0 < hi:
                raise ValueError(f"out overlaps {name}")


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
    parts that are joined in float32.  The result carries no gradient (see
    ``block_scaled_linear``)."""
    _check_blocks(a, "a")
    _check_blocks(b, "b")
    return _mm(a, b, c, alpha, dtype, out, 0)


def _mm(a, b, c, alpha, dtype, out, form):
    if (a.scaling, a.scale_vec) != (b.scaling, b.scale_vec):
        raise ValueError(f"a and b have different forms: {a!r}, {b!r}")
    if a.k != b.k:
        raise ValueError(f"a has K={a.k} but b has K={b.k}")
    if a.device != b.device:
        raise ValueError("a and b are on different devices")
    if dtype not in _REAL:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, not {dtype}")
    alpha = float(alpha)
    if _F32_LARGEST < abs(alpha) < float("inf"):
        raise ValueError(f"alpha={alpha!r} is not a float32")
    shape = (a.rows, b.rows)
    if c is not None:
        _real_tensor(c, "c")
        if c.device != a.device:
            raise ValueError("c is on another device")
        if c.requires_grad and torch.is_grad_enabled():
            raise ValueError("block_scaled_mm gives c no gradient; detach it or use block_scaled_linear")
        try:
            c = c.detach().resolve_neg().expand(shape)
        except RuntimeError:
            raise ValueError(f"c of shape {tuple(c.shape)} does not broadcast to {shape}") from None
    given = out is not None
    out = _result(out, shape, dtype, a.device)
    if given:
        _apart(out, a, "a")
        _apart(out, b, "b")
    if given and c is not None and out.numel():
        (c0, c1), (d0, d1) = _span(c), _span(out)
        same = c0 == d0 and c.dtype == out.dtype and all(n == 1 or s == t for n, s, t in
                                                         zip(shape, c.stride(), out.stride()))
        if c0 < d1 and d0 < c1 and not same:
            raise ValueError("c overlaps out without being out")
    ma, mb = a.multiplier, b.multiplier
    c_at, c_type, c_rows, c_cols = (0, 0, 0, 0) if c is None else (c.data_ptr(), _REAL[c.dtype], *c.stride())
    _call(nat.load().t5e_block_scaled_mm, a.device.index,
          _pack_mm(*a._fields, *b._fields, 0 if ma is None else ma.data_ptr(), 0 if mb is None else mb.data_ptr(), alpha, form,
                   c_at, c_type, _REAL[dtype], c_rows, c_cols, out.data_ptr(),
                   out.stride(0) if given and shape[0] > 1 else shape[1]))
    return out


def block_scaled_mm_expired(device=None) -> bool:
    """Whether a bounded wait inside a product ran out on the device since the
    library was loaded (the tile concerned holds NaN); synchronizes the device."""
    device = require_device(device)
    flag = ctypes.c_int32(0)
    with torch.cuda.device(device):
        nat.check(nat.load().t5e_block_scaled_mm_expired(ctypes.byref(flag)), "t5e_block_scaled_mm_expired")
    return flag.value != 0


def _part(at, rows, k, fmt, block):
    """(t5e_blocks fields without an address, offset, end) of rows with their
    scales at an offset of an allocation."""
    stride = (k + 31) // 32 * 16
    size = rows * stride
    end = at + size + (rows + 127) // 128 * (-(-k // (4 * block)) * 512)
    return (at, stride, at + size, rows, k, fmt, block), (end + 255) // 256 * 256


def _placed(part, base):
    """The fields of a part of the allocation at `base`."""
    at, stride, scales, rows, k, fmt, block = part
    return base + at, stride, base + scales, rows, k, fmt, block


def _job(x, rounding, multiplier, partials, count, rows, cols):
    """(a tensor that has to live until the launch, t5e_quantize)."""
    m, m_rows, m_cols, stride, turned = _matrix_of(x)
    if turned:
        rows, cols = cols, rows
    return m, _pack_quantize(m.data_ptr(), m_rows, m_cols, stride, _REAL[m.dtype], rounding, multiplier, partials, count, 0,
                             *rows, *cols)


def _product(a, b, ma, mb, rows, cols, dtype, device):
    """block_scaled_mm of t5e_blocks fields."""
    out = torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)
    _call(nat.load().t5e_block_scaled_mm, device.index,
          _pack_mm(*a, *b, ma, mb, 1.0, 0, 0, 0, _REAL[dtype], 0, 0, out.data_ptr(), cols))
    return out


class _Linear(torch.autograd.Function):
    """The three products of block_scaled_linear.  The calls are those of
    quantize_blocks and block_scaled_mm, x and w rounded in the same launches
    and everything a pass needs in one allocation: a small layer's time is
    its launches."""

    @staticmethod
    def forward(ctx, x, w, choice, need_x, need_w):
        (n, k), tokens, device = w.shape, x.numel() // w.shape[1], x.device
        ctx.shapes = x.shape, n, k
        if not tokens:
            ctx.form = None
            return x.new_empty((*x.shape[:-1], n))
        scaling, _, rounding, fmt, block = choice
        auto = scaling == "ue4m3"
        ctx.form = rounding, auto, fmt, block
        # Blocks run along the contraction: K here, the tokens and N in the
        # gradients, so what a gradient needs is rounded along the other axis.
        # Kept for the backward pass: the multipliers, then the columns.
        xt = wt = None
        end = 256
        if need_w:
            xt, end = _part(end, k, tokens, fmt, block)
        if need_x:
            wt, end = _part(end, k, n, fmt, block)
        keep = torch.empty(end, dtype=torch.uint8, device=device)
        xr, end = _part(0, tokens, k, fmt, block)
        wr, partials = _part(end, n, k, fmt, block)
        x_count, w_count = (_partial_count(tokens * k), _partial_count(n * k)) if auto else (0, 0)
        work = torch.empty(partials + 4 * (x_count + w_count), dtype=torch.uint8, device=device)
        base, there = keep.data_ptr(), work.data_ptr()
        xr, wr = _placed(xr, there), _placed(wr, there)
        mx, mw, px, pw = (base, base + 4, there + partials, there + partials + 4 * x_count) if auto else (0, 0, 0, 0)
        x1, x_job = _job(x, rounding, mx, px, x_count, xr, _NO_BLOCKS if xt is None else _placed(xt, base))
        w1, w_job = _job(w, rounding, mw, pw, w_count, wr, _NO_BLOCKS if wt is None else _placed(wt, base))
        _call(nat.load().t5e_quantize_blocks, device.index, x_job + w_job, 2)
        y = _product(xr, wr, mx, mw, tokens, n, x.dtype, device)
        ctx.parts = xt, wt
        ctx.save_for_backward(keep)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], n)

    @staticmethod
    def backward(ctx, g):
        # grad mode is on here only under create_graph=True; the marked form
        # then refuses a second derivative, and costs a few microseconds
        return _marked_backward(ctx, g) if torch.is_grad_enabled() else _Linear._backward(ctx, g)

    @staticmethod
    def _backward(ctx, g):
        x_shape, n, k = ctx.shapes
        need_x, need_w = ctx.needs_input_grad[:2]
        if ctx.form is None:
            return (g.new_zeros(x_shape) if need_x else None, g.new_zeros(n, k) if need_w else None,
                    None, None, None)
        dx = dw = None
        if need_x or need_w:
            rounding, auto, fmt, block = ctx.form
            tokens, device, dtype = g.numel() // n, g.device, g.dtype
            keep, = ctx.saved_tensors
            gr = gt = _NO_BLOCKS
            end = 0
            if need_x:
                gr, end = _part(end, tokens, n, fmt, block)
            if need_w:
                gt, end = _part(end, n, tokens, fmt, block)
            count = _partial_count(tokens * n) if auto else 0
            work = torch.empty(end + 4 * (1 + count), dtype=torch.uint8, device=device)
            base, there = keep.data_ptr(), work.data_ptr()
            gr = _placed(gr, there) if need_x else gr
            gt = _placed(gt, there) if need_w else gt
            mx, mw, mg, pg = (base, base + 4, there + end, there + end + 4) if auto else (0, 0, 0, 0)
            g1, job = _job(g, rounding, mg, pg, count, gr, gt)
            _call(nat.load().t5e_quantize_blocks, device.index, job, 1)
            xt, wt = ctx.parts
            if need_x:
                dx = _product(gr, _placed(wt, base), mg, mw, tokens, k, dtype, device)
                if len(x_shape) != 2:
                    dx = dx.view(x_shape)
            if need_w:
                dw = _product(gt, _placed(xt, base), mg, mx, n, k, dtype, device)
        return dx, dw, None, None, None


@torch.autograd.function.once_differentiable
def _marked_backward(ctx, g):
    return _Linear._backward(ctx, g)


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
    pass, not the tensors.  Differentiable once."""
    choice = _choice(scaling, scale_vec, scale_rounding)
    _real_tensor(x, "x")
    _real_tensor(w, "w")
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x [..., K] and w [N, K] do not fit: {tuple(x.shape)}, {tuple(w.shape)}")
    if w.shape[0] == 0 or w.shape[1] == 0:
        raise ValueError("w must not be empty")
    if x.dtype != w.dtype or x.device != w.device:
        raise ValueError("x and w must have one type and device")
    grad = torch.is_grad_enabled()
    return _Linear.apply(x, w, choice, grad and x.requires_grad, grad and w.requires_grad)
