"""Block-scaled E2M1 tensors: rounding, back, products and the linear layer,
against their definition in 64 bits.

Tolerances.  Codes, scales and (with a power-of-two multiplier) values are
exact and compared as such.  A product's F32 accumulation truncates once per
K=64 instruction: each of its s = ceil(K/64) steps loses less than one unit in
the last place of a running sum that is at most S = sum |a||b|, 2^-23 S, and
joining p parts rounds p - 1 more times by 2^-24 S; the result type rounds once
by half a step.  alpha and the two reciprocals of the multipliers add three
roundings of 2^-24, the final product another.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tcgen05_b200 as t5
from tcgen05_b200 import _native as nat
from tcgen05_b200 import blocks as bk

FORMS = [("ue4m3", 4), ("ue8m0", 2), ("ue8m0", 4)]
BLOCK = {("ue4m3", 4): 16, ("ue8m0", 2): 32, ("ue8m0", 4): 16}
TYPES = [torch.float32, torch.bfloat16, torch.float16]
E2M1 = [0, 0.5, 1, 1.5, 2, 3, 4, 6]


# ------------------------------------------------------- the definition


def e4m3_value(byte: int) -> float:
    e, f = byte >> 3 & 15, byte & 7
    return f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)


E4M3 = np.array([e4m3_value(i) for i in range(0x7F)])


def nearest(values, codes):
    """Index of the nearest of the ascending `codes`, ties to the even index."""
    codes = np.asarray(codes, dtype=np.float64)
    hi = np.clip(np.searchsorted(codes, values), 1, len(codes) - 1)
    lo = hi - 1
    down, up = values - codes[lo], codes[hi] - values
    return np.where(down < up, lo, np.where(up < down, hi, np.where(lo % 2 == 0, lo, hi)))


def define(x, form, multiplier=1.0, ceil=False):
    """(codes [R, K], scale bytes [R, blocks], values [R, K]) of x's rows, by the
    definition, in 64 bits on the host."""
    x = x.detach().cpu().to(torch.float64).numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        u = (x * np.float64(multiplier)).astype(np.float32).astype(np.float64)
    rows, k = u.shape
    block = BLOCK[form]
    n = -(-k // block)
    padded = np.zeros((rows, n * block))
    padded[:, :k] = u
    b = padded.reshape(rows, n, block)
    top = np.abs(b).max(2)
    good = np.isfinite(top)
    a = np.where(good, top, 0.0)
    if form[0] == "ue4m3":
        byte = nearest(np.minimum(a / 6, 448.0), E4M3)
        step = E4M3[byte]
        byte = np.where(good, byte, 0x7F)
    else:
        e = np.frexp(a)[1] - 3
        if ceil:
            e = e + (a > 6 * np.exp2(e.astype(np.float64)))
        e = np.clip(np.where(a > 0, e, -127), -127, 127)
        step = np.exp2(e.astype(np.float64))
        byte = np.where(good, e + 127, 0xFF)
    size = np.where(step[..., None] > 0, np.abs(np.where(good[..., None], b, 0)) / np.where(step > 0, step, 1)[..., None], 0)
    code = nearest(np.minimum(size, 6.0), E2M1)
    sign = np.where(good[..., None], np.signbit(b), False)
    value = np.where(good[..., None], np.where(sign, -1, 1) * np.array(E2M1)[code] * step[..., None], np.nan)
    flat = lambda v: v.reshape(rows, -1)[:, :k]  # noqa: E731
    return flat(code + 8 * sign).astype(np.uint8), byte.astype(np.uint8), flat(value) / multiplier


def codes_of(q):
    d = q.data.cpu().numpy()
    return np.stack([d & 15, d >> 4], axis=2).reshape(d.shape[0], -1)


def check_rows(q, want_codes, want_bytes):
    got = codes_of(q)
    np.testing.assert_array_equal(got[:, :q.k], want_codes)
    assert not got[:, q.k:(q.k + 31) // 32 * 32].any(), "codes behind K"
    np.testing.assert_array_equal(q.scale_words().cpu().numpy(), want_bytes)
    groups = q.scales.shape[1] * 4
    every = bk.untile_scales(q.scales, q.rows, groups).cpu().numpy()
    assert not every[:, want_bytes.shape[1]:].any(), "scales behind the last block"


def make(seed, *shape, dtype=torch.float32, wide=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    if wide:
        x = x * torch.exp(4 * torch.randn(*shape, generator=g, device="cuda"))
    return x.to(dtype)


# ------------------------------------------------------------ on the CPU


def test_scale_tiles_follow_the_documented_order():
    words = torch.randint(0, 256, (300, 13), dtype=torch.uint8)
    tiles = bk.tile_scales(words)
    assert tuple(tiles.shape) == (3, 4, 512)
    flat, groups = tiles.reshape(-1), 4
    for r in (0, 1, 31, 32, 127, 128, 255, 299):
        for b in range(13):
            assert flat[((r // 128) * groups + b // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + b % 4] == words[r, b]
    assert torch.equal(bk.untile_scales(tiles, 300, 13), words)


@pytest.mark.parametrize("kw", [
    dict(scaling="ue4m3", scale_vec=2), dict(scaling="ue5m3"), dict(scaling="ue8m0", scale_vec=1),
    dict(scaling="ue4m3", scale_rounding="floor"), dict(scaling="ue8m0", scale_rounding="nearest"),
    dict(scaling="ue8m0", scale_rounding="up"), dict(axis=1), dict(axis="rows"), dict(multiplier="max"),
    dict(multiplier=0.0), dict(multiplier=-2.0), dict(multiplier=float("nan")), dict(multiplier=float("inf")),
    dict(multiplier=1e300), dict(multiplier=1e-300), dict(multiplier=1e-45),
])
def test_quantize_refuses_bad_arguments(kw):
    with pytest.raises(ValueError):
        t5.quantize_blocks(torch.zeros(4, 64), **kw)


@pytest.mark.parametrize("x", [torch.zeros(4, 64), torch.zeros(4, 64, dtype=torch.float64),
                               torch.zeros(4, 64, dtype=torch.int32), [[1.0]]])
def test_tensors_must_be_real_and_on_the_device(x):
    for call in (t5.quantize_blocks, t5.block_multiplier, lambda v: t5.block_scaled_linear(v, v)):
        with pytest.raises(ValueError):
            call(x)


def _rows(rows=4, k=64, form=("ue4m3", 4), **kw):
    groups = -(-k // (4 * BLOCK[form]))
    return t5.BlockScaledRows(torch.zeros(rows, bk.BlockScaledRows.row_stride(k), dtype=torch.uint8),
                              torch.zeros(-(-rows // 128), groups, 512, dtype=torch.uint8), k, scaling=form[0],
                              scale_vec=form[1], **kw)


def test_block_scaled_rows_checks_its_parts():
    q = _rows(130, 100)
    assert (q.rows, q.k, q.block) == (130, 100, 16) and q.packed().k == 100
    assert tuple(q.scale_words().shape) == (130, 7)
    data, scales = q.data, q.scales
    bad = [
        (data, scales, 0), (data, scales, 129), (data[:, :48].contiguous(), scales, 100), (data[:, :40].contiguous(), scales, 64),
        (data.int(), scales, 100), (data[0], scales, 100), (data, scales[:1], 100), (data, scales[:, :1], 100),
        (data, scales.int(), 100), (data, scales, 40), (data.t().contiguous().t(), scales, 100),
    ]
    for d, s, k in bad:
        with pytest.raises(ValueError):
            t5.BlockScaledRows(d, s, k)
    with pytest.raises(ValueError):
        t5.BlockScaledRows(data, scales, 100, multiplier=torch.ones(2))
    with pytest.raises(ValueError):
        t5.BlockScaledRows(data, scales, 100, multiplier=torch.ones(1, dtype=torch.float64))
    shifted = torch.zeros(130 * 64 + 1, dtype=torch.uint8)[1:].view(130, 64)
    with pytest.raises(ValueError):
        t5.BlockScaledRows(shifted, scales, 100)


def test_products_refuse_what_is_not_on_the_device():
    with pytest.raises(ValueError):
        t5.block_scaled_mm(_rows(), _rows())
    with pytest.raises(ValueError):
        t5.dequantize_blocks(_rows())
    with pytest.raises(ValueError):
        t5.block_scaled_mm(torch.zeros(4, 64), _rows())


def test_c_entry_points_refuse_bad_arguments():
    """Host-side checks: nothing is launched (addresses are never read)."""
    import ctypes

    lib = nat.load()

    def blk(**kw):
        b = nat.Blocks(4096, 64, 4096, 8, 128, nat.SCALE_UE4M3, 16)
        for name, v in kw.items():
            setattr(b, name, v)
        return b

    bad = [dict(k=0), dict(k=nat.MAX_BLOCK_K + 1), dict(stride=48), dict(stride=72), dict(data=4104), dict(scales=4100),
           dict(scale_block=32), dict(scale_format=0), dict(data=None), dict(scales=None),
           dict(rows=nat.MAX_BLOCK_ROWS + 1)]
    none, second = nat.Blocks(), blk()

    def quantize(n=1, **kw):
        q = nat.Quantize(4096, 8, 128, 128, 0, 0, None, None, 0, 0, blk(), none)
        for name, v in kw.items():
            setattr(q, name, v)
        return lib.t5e_quantize_blocks((nat.Quantize * 2)(q, q), n, None)

    for kw in bad:
        b = blk(**kw)
        assert lib.t5e_dequantize_blocks(ctypes.byref(b), None, 0, 4096, 128, None) == nat.ERR_INVALID
        assert quantize(rows=b.rows, cols=max(b.k, 0), by_rows=b) == nat.ERR_INVALID
        mm = nat.BlockMm(b, second, None, None, 1.0, 0, None, 0, 0, 0, 0, 4096, 8)
        assert lib.t5e_block_scaled_mm(ctypes.byref(mm), None) == nat.ERR_INVALID
    good = blk()
    for kw in (dict(type=3), dict(rounding=1), dict(stride=127), dict(x=4098), dict(x=None), dict(partials=4096, count=4),
               dict(partials=4096, multiplier=4096, count=0), dict(rows=9), dict(cols=127), dict(by_rows=none),
               dict(by_cols=blk()), dict(reserved=1), dict(n=0), dict(n=3),
               dict(by_cols=nat.Blocks(4096, 16, 4096, 128, 8, nat.SCALE_UE8M0, 16))):
        assert quantize(**kw) == nat.ERR_INVALID, kw
    assert lib.t5e_quantize_blocks(None, 1, None) == nat.ERR_INVALID
    for partials, count, out in ((4096, 0, 4096), (4096, nat.MAX_PARTIALS + 1, 4096), (None, 4, 4096), (4096, 4, None)):
        assert lib.t5e_block_multiplier(0, 4096, 8, 128, 128, partials, count, out, None) == nat.ERR_INVALID

    def mm(**kw):
        m = nat.BlockMm(good, second, None, None, 1.0, 0, None, 0, 0, 0, 0, 4096, 8)
        for name, v in kw.items():
            setattr(m, name, v)
        return lib.t5e_block_scaled_mm(ctypes.byref(m), None)

    other = blk(scale_format=nat.SCALE_UE8M0)
    for kw in (dict(d=None), dict(d=4098), dict(d_stride=7), dict(d_type=3), dict(c=4096, c_type=5), dict(c=4098),
               dict(form=3), dict(form=16), dict(form=2), dict(b=other), dict(a=none)):
        assert mm(**kw) == nat.ERR_INVALID, kw
    assert lib.t5e_block_scaled_mm_expired(None) == nat.ERR_INVALID


def test_block_structs_match_the_header(tmp_path):
    """The ctypes structures lay t5e_blocks, t5e_quantize and t5e_block_mm out as
    the C compiler does."""
    import ctypes
    import subprocess
    from pathlib import Path

    src = tmp_path / "layout.c"
    src.write_text(
        '#include <stdio.h>\n#include <stddef.h>\n#include "t5e.h"\n'
        'int main(void){printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(t5e_blocks), sizeof(t5e_quantize),'
        ' sizeof(t5e_block_mm), offsetof(t5e_quantize, by_cols), offsetof(t5e_block_mm, c),'
        ' offsetof(t5e_block_mm, d), offsetof(t5e_blocks, scale_block));return 0;}\n')
    exe = tmp_path / "layout"
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(include), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(nat.Blocks), ctypes.sizeof(nat.Quantize), ctypes.sizeof(nat.BlockMm),
                   nat.Quantize.by_cols.offset, nat.BlockMm.c.offset, nat.BlockMm.d.offset, nat.Blocks.scale_block.offset]


def test_empty_calls_launch_nothing():
    import ctypes

    lib = nat.load()
    none = nat.Blocks(None, 64, None, 0, 128, nat.SCALE_UE4M3, 16)
    some = nat.Blocks(4096, 64, 4096, 8, 128, nat.SCALE_UE4M3, 16)
    assert lib.t5e_dequantize_blocks(ctypes.byref(none), None, 0, None, 128, None) == nat.OK
    q = nat.Quantize(None, 0, 128, 128, 0, 0, None, None, 0, 0, nat.Blocks(), nat.Blocks())
    assert lib.t5e_quantize_blocks(ctypes.byref(q), 1, None) == nat.OK
    for a, b in ((none, some), (some, none)):
        m = nat.BlockMm(a, b, None, None, 1.0, 0, None, 0, 0, 0, 0, None, 8)
        assert lib.t5e_block_scaled_mm(ctypes.byref(m), None) == nat.OK


# ------------------------------------------------------------ rounding (GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 15), (1, 16), (2, 17), (3, 32), (5, 33), (7, 100), (130, 64), (33, 257),
                                    (257, 520), (1, 4096), (300, 1000), (300, 1001), (385, 393)])
def test_rows_and_columns_round_as_defined(form, dtype, rows, k):
    x = make(rows * 7919 + k, rows, k, dtype=dtype, wide=True)
    for ceil in ((False, True) if form[0] == "ue8m0" else (False,)):
        kw = dict(scaling=form[0], scale_vec=form[1])
        if form[0] == "ue8m0":
            kw["scale_rounding"] = "ceil" if ceil else "floor"
        q = t5.quantize_blocks(x, **kw)
        qr, qc = t5.quantize_blocks(x, axis="both", **kw)
        q0 = t5.quantize_blocks(x, axis=0, **kw)
        codes, scale, values = define(x, form, ceil=ceil)
        check_rows(q, codes, scale)
        check_rows(qr, codes, scale)
        codes, scale, turned = define(x.t(), form, ceil=ceil)
        check_rows(qc, codes, scale)
        check_rows(q0, codes, scale)
        # E2M1 times the scale has at most 6 significand bits: exact in F32
        got = t5.dequantize_blocks(q)
        np.testing.assert_array_equal(got.cpu().numpy(), values.astype(np.float32))
        for t in (torch.bfloat16, torch.float16):
            # NaN blocks (infinities among F16 inputs) compare equal here
            np.testing.assert_array_equal(t5.dequantize_blocks(q, dtype=t).float().cpu().numpy(),
                                          got.to(t).float().cpu().numpy())
        np.testing.assert_array_equal(t5.dequantize_blocks(q0).cpu().numpy(), turned.astype(np.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_every_tie_and_its_neighbours(form, dtype):
    """Blocks whose largest value sets each scale significand, with elements at
    each rounding border of E2M1 times the scale, and the type's values next to
    it on either side; also with multipliers that shift the whole block."""
    def beside(t, side):
        if side is None:
            return np.asarray(t, dtype=np.float64)
        v = torch.nextafter(torch.as_tensor(t).to(dtype), torch.tensor(side, dtype=dtype))
        return v.double().numpy()

    blocks, block = [], BLOCK[form]
    for m in range(8, 16):
        for e in (-6, 0, 5):
            step = m / 8 * 2.0 ** e if form[0] == "ue4m3" else 2.0 ** e
            ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * step
            for side in (None, np.inf, -np.inf):
                t = ties.astype(np.float32)
                t = t if side is None else np.nextafter(t, np.float32(side))
                for sign in (1, -1):
                    blocks.append(np.concatenate([[6 * step], sign * t, np.zeros(block - 8)]))
    # borders of the scale's own rounding
    for a in (6 * 17 / 16, 6 * 19 / 16, 6 * 2.0 ** -10, 6 * 1.5 * 2.0 ** -9, 6 * 448.0, 6 * 464.0, 1e5):
        for v in (float(beside(a, None)), float(beside(a, np.inf)), float(beside(a, 0.0))):
            blocks.append(np.concatenate([[v, v / 3, -v / 7], np.zeros(block - 3)]))
    x = torch.tensor(np.array(blocks)).to(dtype).cuda()
    for m in (1.0, 0.25, 2.0 ** 70, 1.5):
        codes, scale, _ = define(x, form, m)
        kw = dict(scaling=form[0], scale_vec=form[1], multiplier=None if m == 1 else m)
        check_rows(t5.quantize_blocks(x, **kw), codes, scale)
        check_rows(t5.quantize_blocks(x.t().contiguous(), axis=0, **kw), codes, scale)
        rows, cols = t5.quantize_blocks(x.t(), axis="both", **kw)
        check_rows(cols, codes, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_special_values(form, dtype):
    """Zeros, subnormals, the largest values, infinities and NaN: a block with
    one that is not finite is NaN, its neighbours are not."""
    info = torch.finfo(dtype)
    block = BLOCK[form]
    x = torch.zeros(9, 4 * block)
    x[1, 3] = float("inf")
    x[2, block] = float("-inf")
    x[3, 2 * block + 5] = float("nan")
    x[4] = info.max
    x[5] = -info.max
    x[6] = info.smallest_normal
    x[7, ::3] = info.smallest_normal * info.eps  # the smallest subnormal
    x[8, ::2] = -0.0
    x[1:4, -1] = 2.0
    x = x.to(dtype).cuda()
    for ceil in ((False, True) if form[0] == "ue8m0" else (False,)):
        kw = dict(scaling=form[0], scale_vec=form[1])
        if form[0] == "ue8m0":
            kw["scale_rounding"] = "ceil" if ceil else "floor"
        codes, scale, values = define(x, form, ceil=ceil)
        for q in (t5.quantize_blocks(x, **kw), t5.quantize_blocks(x.t().contiguous(), axis=0, **kw)):
            check_rows(q, codes, scale)
            np.testing.assert_array_equal(t5.dequantize_blocks(q).cpu().numpy(), values.astype(np.float32))
    assert np.isnan(values[1, :block]).all() and np.isfinite(values[1, block:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (3, 5), (1000, 1001), (4, 7, 65)])
def test_multiplier_is_the_largest_fitting_power_of_two(dtype, shape):
    x = make(3, *shape, dtype=dtype) * 0.37
    top = float(x.abs().max().double())
    m = float(t5.block_multiplier(x))
    assert math.log2(m) == int(math.log2(m)) and top * m <= 2688 < top * m * 2
    if x.dim() > 1:
        assert float(t5.block_multiplier(x.t() if x.dim() == 2 else x.transpose(0, 1))) == m
        q = t5.quantize_blocks(x, multiplier="auto")
        assert float(q.multiplier) == m
        codes, scale, values = define(x.reshape(-1, shape[-1]), ("ue4m3", 4), m)
        check_rows(q, codes, scale)
        np.testing.assert_array_equal(t5.dequantize_blocks(q).cpu().numpy(), values.astype(np.float32))
        given = t5.quantize_blocks(x, multiplier=t5.block_multiplier(x))
        assert torch.equal(given.data, q.data) and torch.equal(given.scale_words(), q.scale_words())


@pytest.mark.gpu
def test_multiplier_borders():
    for top, want in ((0.0, 1.0), (float("inf"), 1.0), (float("nan"), 1.0), (2688.0, 1.0), (2689.0, 0.5),
                      (1344.0, 2.0), (1.3125, 2048.0), (1.3126, 1024.0), (1e-45, 2.0 ** 126), (3e38, 2.0 ** -117)):
        x = torch.tensor([[0.0, -top]], device="cuda")
        assert float(t5.block_multiplier(x)) == want, top
    assert float(t5.block_multiplier(torch.empty(0, 4, device="cuda"))) == 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("multiplier", [3.0, 0.1, 1e-3])
def test_any_multiplier_rounds_its_product_to_f32_first(multiplier):
    x = make(11, 40, 200, wide=True)
    m = float(np.float32(multiplier))
    codes, scale, values = define(x, ("ue4m3", 4), m)
    q = t5.quantize_blocks(x, multiplier=multiplier)
    check_rows(q, codes, scale)
    # two roundings: the reciprocal and the product with it
    got = t5.dequantize_blocks(q).cpu().numpy().astype(np.float64)
    assert (np.abs(got - values) <= 2 * 2.0 ** -24 * 1.001 * np.abs(values)).all()


@pytest.mark.gpu
def test_strides_and_alignments():
    base = make(5, 70, 300)
    want = t5.quantize_blocks(base[3:40, 5:202].contiguous())
    pick = [base[3:40, 5:202], base.t().contiguous().t()[3:40, 5:202], base.repeat(1, 2)[3:40, 5:202],
            torch.stack([base, base], 2)[3:40, 5:202, 0]]
    turned = t5.quantize_blocks(base[3:40, 5:202].contiguous(), axis=0)
    for x in pick:
        q, t = t5.quantize_blocks(x, axis="both")
        assert torch.equal(q.data, want.data) and torch.equal(q.scale_words(), want.scale_words())
        assert torch.equal(t.data, turned.data) and torch.equal(t.scale_words(), turned.scale_words())
        assert float(t5.block_multiplier(x)) == float(t5.block_multiplier(x.contiguous()))
    row = base[0, :130]
    a, b = t5.quantize_blocks(row.expand(6, 130)), t5.quantize_blocks(row.repeat(6, 1))
    assert torch.equal(a.data, b.data)
    out = torch.full((40, 256), 7.0, device="cuda")
    t5.dequantize_blocks(want, out=out[1:38, 3:200])
    assert torch.equal(out[1:38, 3:200], t5.dequantize_blocks(want))
    assert bool((out[0] == 7).all() and (out[38:] == 7).all() and (out[:, :3] == 7).all() and (out[:, 200:] == 7).all())
    for bad in (out[:37, :196], out[1:38, 3:397:2], out[1:38, 3:200].double()):
        with pytest.raises(ValueError):
            t5.dequantize_blocks(want, out=bad)


@pytest.mark.gpu
def test_negated_views_and_single_rows():
    z = torch.complex(make(1, 9, 70), make(2, 9, 70))
    neg = torch.conj(z).imag
    assert neg.is_neg()
    assert torch.equal(t5.quantize_blocks(neg).data, t5.quantize_blocks(-z.imag.contiguous()).data)
    a, b = t5.quantize_blocks(make(3, 9, 64)), t5.quantize_blocks(make(4, 70, 64))
    assert torch.equal(t5.block_scaled_mm(a, b, neg), t5.block_scaled_mm(a, b, -z.imag.contiguous()))
    row = make(5, 200)
    q = t5.quantize_blocks(row)
    assert (q.rows, q.k) == (1, 200) and torch.equal(q.data, t5.quantize_blocks(row[None]).data)
    assert torch.equal(t5.quantize_blocks(row[None, ::2]).data, t5.quantize_blocks(row[::2].contiguous()).data)
    w = make(6, 33, 200).requires_grad_()
    x = row.clone().requires_grad_()
    y = t5.block_scaled_linear(x, w)
    assert y.shape == (33,)
    y.sum().backward()
    assert x.grad.shape == (200,) and bool(x.grad.isfinite().all()) and w.grad.shape == (33, 200)


@pytest.mark.gpu
def test_empty_tensors():
    q = t5.quantize_blocks(torch.empty(0, 64, device="cuda"), multiplier="auto")
    assert q.rows == 0 and tuple(t5.dequantize_blocks(q).shape) == (0, 64)
    other = t5.quantize_blocks(make(1, 5, 64))
    assert tuple(t5.block_scaled_mm(q, other).shape) == (0, 5) and tuple(t5.block_scaled_mm(other, q).shape) == (5, 0)
    for x, axis in ((torch.empty(0, 64, device="cuda"), 0), (torch.empty(4, 0, device="cuda"), -1),
                    (torch.tensor(1.0, device="cuda"), -1)):
        with pytest.raises(ValueError):
            t5.quantize_blocks(x, axis=axis)


@pytest.mark.gpu
def test_words_round_trip_through_the_emulators_layout():
    x = make(9, 70, 130)
    q = t5.quantize_blocks(x)
    words = torch.from_numpy(codes_of(q)[:, :q.k].astype(np.int32)).cuda()
    again = t5.BlockScaledRows.from_words(words, q.scale_words())
    assert torch.equal(again.data, q.data) and torch.equal(again.scale_words(), q.scale_words())
    # one dot product per row through the emulator, from the rows as they are
    d = t5.mma_dot_batch(q.packed(), q.packed(), a_format="e2m1", scaling="ue4m3", scale_vec=4,
                         scale_a=q.scale_words(), scale_b=q.scale_words())
    v = t5.dequantize_blocks(q).double()
    got = d.view(torch.float32).double()
    # K = 130 is one instruction of the model: exact products, one truncation per merge
    assert bool(((got - (v * v).sum(1)).abs() <= 4 * 2.0 ** -23 * (v * v).sum(1)).all())


# ------------------------------------------------------------ products (GPU)


def product_bound(a, b, k, out_eps, parts=8):
    """Largest error of a product by the module's account, per element."""
    total = a.abs() @ b.abs().t()
    steps = -(-k // 64)
    return (steps * 2.0 ** -23 + (parts - 1 + 4) * 2.0 ** -24) * total


def check_product(qa, qb, dtype=torch.float32, c=None, alpha=1.0, **kw):
    a, b = t5.dequantize_blocks(qa).double(), t5.dequantize_blocks(qb).double()
    want = alpha * (a @ b.t())
    if c is not None:
        want = want + c.double()
    got = t5.block_scaled_mm(qa, qb, c, dtype=dtype, alpha=alpha, **kw)
    eps = torch.finfo(dtype).eps / 2
    err = product_bound(a, b, qa.k, eps) * abs(alpha)
    # the result's rounding (and the sum's with C), and half a step of the subnormals
    room = err + 1.01 * eps * (want.abs() + err) + (2.0 ** -24 * c.double().abs() if c is not None else 0) \
        + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = (got.double() - want).abs() > room
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outside, first {bad.nonzero()[0].tolist()}"
    return got


SIZES = [(1, 1, 1), (1, 1, 64), (1, 200, 65), (3, 130, 31), (16, 129, 256), (17, 300, 257), (33, 127, 520),
         (64, 128, 1024), (65, 500, 300), (128, 128, 128), (129, 100, 96), (129, 257, 777), (300, 300, 2050),
         (200, 7, 500), (1000, 40, 640), (513, 384, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_matches_its_definition(form, m, n, k):
    kw = dict(scaling=form[0], scale_vec=form[1])
    qa = t5.quantize_blocks(make(m + k, m, k), multiplier="auto" if form[0] == "ue4m3" else None, **kw)
    qb = t5.quantize_blocks(make(n + 3 * k, n, k), **kw)
    for dtype in TYPES:
        check_product(qa, qb, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("m,n,k", [(128, 128, 64), (128, 128, 1024), (40, 200, 130), (300, 260, 700), (5, 130, 2048),
                                   (260, 16, 333)])
def test_product_is_the_emulated_chain_word_for_word(form, m, n, k):
    from tcgen05_b200 import hwcheck

    kw = dict(scaling=form[0], scale_vec=form[1])
    r = hwcheck.cross_check_product(t5.quantize_blocks(make(m, m, k, wide=True), **kw),
                                    t5.quantize_blocks(make(n + 1, n, k), **kw))
    assert r["cases"] == m * n and r["mismatches"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("kernel", [1, 128, 256])
@pytest.mark.parametrize("m,n,k", [(129, 129, 64), (300, 257, 700), (256, 512, 1344), (700, 1030, 2100), (2600, 3000, 300)])
def test_every_kernel_form_is_the_emulated_chain(form, kernel, m, n, k):
    """The tile kernel and both pair kernels, one tile and several per block,
    K that ends in every step of a stage."""
    from tcgen05_b200 import hwcheck

    kw = dict(scaling=form[0], scale_vec=form[1])
    r = hwcheck.cross_check_product(t5.quantize_blocks(make(m, m, k, wide=True), **kw),
                                    t5.quantize_blocks(make(n + 1, n, k), **kw), kernel)
    assert r["mismatches"] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", [1, 128, 256])
@pytest.mark.parametrize("m,n", [(300, 264), (300, 267), (520, 1000)])
def test_every_kernel_forms_outputs(kernel, m, n):
    """Result types, rows on and off 16-byte boundaries, addends, into part of a
    larger tensor."""
    a, b = t5.quantize_blocks(make(m, m, 500), multiplier="auto"), t5.quantize_blocks(make(n, n, 500), multiplier=0.5)
    va, vb = t5.dequantize_blocks(a).double(), t5.dequantize_blocks(b).double()
    exact, err = va @ vb.t(), product_bound(va, vb, 500, 0)
    for dtype in TYPES:
        eps, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        for c in (None, make(1, m, n, dtype=dtype), make(2, n), make(3, n, m).t()):
            for pad in (0, 3, 8):
                big = torch.full((m + 2, n + 2 * pad), 7.0, dtype=dtype, device="cuda")
                out = big[1:m + 1, pad:n + pad]
                got = bk._mm(a, b, c, -0.75, dtype, out, kernel)
                want = -0.75 * exact + (0 if c is None else c.double())
                room = 0.75 * err + 1.01 * eps * (want.abs() + err) + tiny
                if c is not None:
                    room = room + 2.0 ** -24 * c.double().abs()
                assert got.data_ptr() == out.data_ptr()
                assert bool(((got.double() - want).abs() <= room).all())
                out.fill_(7)
                assert bool((big == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("split", [1, 2, 4, 8])
@pytest.mark.parametrize("m,n", [(5, 300), (30, 128), (64, 70), (100, 128), (257, 130)])
def test_split_products(split, m, n):
    a, b = t5.quantize_blocks(make(m, m, 2100)), t5.quantize_blocks(make(n, n, 2100))
    va, vb = t5.dequantize_blocks(a).double(), t5.dequantize_blocks(b).double()
    got = bk._mm(a, b, None, 1.0, torch.float32, None, split)
    want = va @ vb.t()
    room = product_bound(va, vb, 2100, 0, split) + 2.0 ** -24 * 1.01 * want.abs()
    assert bool(((got.double() - want).abs() <= room).all())
    again = bk._mm(a, b, None, 1.0, torch.float32, None, split)
    assert torch.equal(got, again)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(1, 260), (40, 260), (300, 260), (260, 40)])
def test_addends_scale_and_given_outputs(m, n):
    a, b = t5.quantize_blocks(make(m, m, 500), multiplier="auto"), t5.quantize_blocks(make(n, n, 500), multiplier=4.0)
    for dtype in TYPES:
        for c in (make(1, m, n, dtype=dtype), make(2, n), make(3, m, 1), make(4, 1, 1), make(5, n, m, dtype=dtype).t(),
                  make(6, m, n + 9)[:, 4:n + 4]):
            check_product(a, b, dtype, c=c, alpha=-1.75)
    # accumulating in place
    c = make(7, m, n)
    want = t5.block_scaled_mm(a, b, c, dtype=torch.float32)
    got = t5.block_scaled_mm(a, b, c, dtype=torch.float32, out=c)
    assert got.data_ptr() == c.data_ptr() and torch.equal(got, want)
    # into a part of a larger tensor, whose other elements stay
    for dtype in TYPES:
        big = torch.full((m + 3, n + 21), 7.0, dtype=dtype, device="cuda")
        t5.block_scaled_mm(a, b, dtype=dtype, out=big[1:m + 1, 5:n + 5])
        assert torch.equal(big[1:m + 1, 5:n + 5], t5.block_scaled_mm(a, b, dtype=dtype))
        big[1:m + 1, 5:n + 5] = 7
        assert bool((big == 7).all())


@pytest.mark.gpu
def test_product_refusals():
    a, b = t5.quantize_blocks(make(1, 8, 64)), t5.quantize_blocks(make(2, 8, 64))
    other = t5.quantize_blocks(make(2, 8, 64), scaling="ue8m0")
    longer = t5.quantize_blocks(make(2, 8, 65))
    c = torch.zeros(8, 8, device="cuda")
    wide = torch.zeros(8, 17, device="cuda")
    for call in (lambda: t5.block_scaled_mm(a, other), lambda: t5.block_scaled_mm(a, longer),
                 lambda: t5.block_scaled_mm(a, b, torch.zeros(7, 8, device="cuda")),
                 lambda: t5.block_scaled_mm(a, b, torch.zeros(8, 8)),
                 lambda: t5.block_scaled_mm(a, b, c.double()), lambda: t5.block_scaled_mm(a, b, dtype=torch.float64),
                 lambda: t5.block_scaled_mm(a, b, dtype=torch.bfloat16, out=c),
                 lambda: t5.block_scaled_mm(a, b, dtype=torch.float32, out=c.t()),
                 lambda: t5.block_scaled_mm(a, b, dtype=torch.float32, out=torch.zeros(8, 9, device="cuda")),
                 lambda: t5.block_scaled_mm(a, b, wide[:, 1:9], dtype=torch.float32, out=wide[:, 2:10]),
                 lambda: t5.block_scaled_mm(a, b, c.clone().requires_grad_()), lambda: t5.block_scaled_mm(a, b, alpha=1e300),
                 lambda: t5.block_scaled_mm(a, b, dtype=torch.float32, out=a.data.view(torch.float32)[:, :8]),
                 lambda: t5.dequantize_blocks(a, dtype=torch.float16, out=a.scales.view(torch.float16).view(-1)[:8 * 24].view(8, 24)[:, :64])):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_nan_blocks_reach_only_their_rows():
    x, w = make(1, 200, 512), make(2, 150, 512)
    clean = t5.block_scaled_mm(t5.quantize_blocks(x), t5.quantize_blocks(w))
    x[17, 100], w[140, 3] = float("nan"), float("inf")
    d = t5.block_scaled_mm(t5.quantize_blocks(x), t5.quantize_blocks(w))
    assert bool(d[17].isnan().all()) and bool(d[:, 140].isnan().all())
    keep = torch.ones_like(d, dtype=torch.bool)
    keep[17], keep[:, 140] = False, False
    assert torch.equal(d[keep], clean[keep])


@pytest.mark.gpu
def test_waits_never_ran_out():
    t5.block_scaled_mm(t5.quantize_blocks(make(1, 200, 512)), t5.quantize_blocks(make(2, 150, 512)))
    assert t5.block_scaled_mm_expired() is False


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("kernel", [1, 128, 256])
def test_any_words_and_scale_bytes(form, kernel):
    """Operands that no rounding made: every code, every scale byte (NaN among
    them) through the products, the emulator and dequantize_blocks."""
    from tcgen05_b200 import hwcheck

    g = torch.Generator(device="cuda").manual_seed(kernel)
    m, n, k = 200, 150, 190
    blocks = -(-k // BLOCK[form])
    top = 128 if form[0] == "ue4m3" else 256

    def rows(r):
        words = torch.randint(0, 16, (r, k), generator=g, device="cuda", dtype=torch.int32)
        scales = torch.randint(0, top, (r, blocks), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        if form[0] == "ue8m0":  # products that stay finite, and a few NaN
            scales = torch.where(scales == 255, scales, 100 + scales % 50)
        return t5.BlockScaledRows.from_words(words, scales, scaling=form[0], scale_vec=form[1]), words, scales

    (a, words, scales), (b, _, _) = rows(m), rows(n)
    r = hwcheck.cross_check_product(a, b, kernel)
    assert r["mismatches"] == 0 and bool(r["hardware"].isnan().any()) and not bool(r["hardware"].isnan().all())
    value = torch.tensor(E2M1 + [-v for v in E2M1], device="cuda", dtype=torch.float64)[words.long()]
    s = scales.long().cpu().numpy()
    step = np.where(s == 255, np.nan, np.exp2(s - 127.0)) if form[0] == "ue8m0" else \
        np.where(s == 127, np.nan, np.array([e4m3_value(i) for i in range(128)])[s])
    want = value.cpu().numpy() * np.repeat(step, BLOCK[form], axis=1)[:, :k]
    np.testing.assert_array_equal(t5.dequantize_blocks(a).cpu().numpy(), want.astype(np.float32))


@pytest.mark.gpu
def test_many_short_rows():
    """More rows than one launch takes, and offsets that pass 32 bits."""
    free, _ = torch.cuda.mem_get_info()
    rows = (1 << 29) + 200
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    x = torch.zeros(rows, 1, dtype=torch.bfloat16, device="cuda")
    x[-300:, 0] = make(1, 300, dtype=torch.bfloat16)
    x[12345, 0] = 3.0
    q = t5.quantize_blocks(x, scaling="ue8m0", scale_vec=4)
    want = t5.quantize_blocks(x[-300:], scaling="ue8m0", scale_vec=4)
    assert torch.equal(q.data[-300:], want.data) and int(q.data[12345, 0]) == int(t5.quantize_blocks(x[12345:12346], scaling="ue8m0", scale_vec=4).data[0, 0])
    out = t5.dequantize_blocks(q, dtype=torch.bfloat16)
    assert torch.equal(out[-300:], t5.dequantize_blocks(want, dtype=torch.bfloat16)) and float(out[12345, 0]) == 3.0
    assert int(torch.count_nonzero(out)) == int(torch.count_nonzero(out[-300:])) + 1
    w = t5.quantize_blocks(torch.full((3, 1), 2.0, device="cuda"), scaling="ue8m0", scale_vec=4)
    del x, out
    d = t5.block_scaled_mm(q, w)
    assert torch.equal(d[-300:], t5.block_scaled_mm(want, w)) and float(d[12345, 2]) == 6.0


@pytest.mark.gpu
def test_long_rows_and_far_columns():
    """A row of more than 2^31 elements' bytes apart from the next (a view), and
    results that lie beyond 2^32 bytes."""
    wide = torch.zeros(3, 1 << 30, dtype=torch.bfloat16, device="cuda")
    x = wide[:, -70:]
    x.copy_(make(1, 3, 70))
    assert torch.equal(t5.quantize_blocks(x).data, t5.quantize_blocks(x.contiguous()).data)
    assert torch.equal(t5.quantize_blocks(x, axis=0).data, t5.quantize_blocks(x.contiguous(), axis=0).data)
    a, b = t5.quantize_blocks(make(2, 3, 64)), t5.quantize_blocks(make(3, 40, 64))
    for pad in (1, 8):
        t5.block_scaled_mm(a, b, out=wide[:, -40 - pad:-pad])
        assert torch.equal(wide[:, -40 - pad:-pad], t5.block_scaled_mm(a, b))


# ------------------------------------------------------------ the linear layer (GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("shape,n", [((1, 64), 32), ((5, 3, 100), 65), ((257, 130), 300)])
def test_linear_and_its_gradients(form, dtype, shape, n):
    kw = dict(scaling=form[0], scale_vec=form[1])
    k = shape[-1]
    x = make(1, *shape, dtype=dtype).requires_grad_()
    w = (make(2, n, k) / math.sqrt(k)).to(dtype).requires_grad_()
    g = make(3, *shape[:-1], n, dtype=dtype)
    y = t5.block_scaled_linear(x, w, **kw)
    dx, dw = torch.autograd.grad(y, (x, w), g)
    assert y.shape == g.shape and dx.shape == x.shape and dw.shape == w.shape
    assert y.dtype == dx.dtype == dw.dtype == dtype
    m = (lambda t: float(t5.block_multiplier(t))) if form[0] == "ue4m3" else (lambda t: 1.0)
    xf, gf = x.detach().reshape(-1, k), g.reshape(-1, n)
    r = lambda t, mult: torch.from_numpy(define(t, form, mult)[2])  # noqa: E731
    for got, a, b in ((y.reshape(-1, n), r(xf, m(x)), r(w, m(w))), (dx.reshape(-1, k), r(gf, m(g)), r(w.t(), m(w))),
                      (dw, r(gf.t(), m(g)), r(xf.t(), m(x)))):
        want = a @ b.t()
        err = product_bound(a, b, a.shape[1], 0)
        eps = torch.finfo(dtype).eps / 2
        room = err + 1.01 * eps * (want.abs() + err) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        assert bool(((got.detach().cpu().double() - want).abs() <= room).all())


@pytest.mark.gpu
def test_gradient_against_differences():
    """On a grid that rounds to itself the layer is the bilinear product, so
    central differences by whole grid steps are exact up to the products' own
    error."""
    pick = torch.tensor([-6, -4, -2, -1, 0, 1, 2, 4, 6.0], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    draw = lambda *s: pick[torch.randint(0, 9, s, generator=gen, device="cuda")]  # noqa: E731
    x, w, g = draw(32, 32), draw(32, 32), draw(32, 32)
    for t in (x, w, g):  # every block of 32 along either axis has its largest value at 6
        t.fill_diagonal_(6.0)
    x, w = x.requires_grad_(), w.requires_grad_()
    kw = dict(scaling="ue8m0", scale_vec=2)
    loss = lambda a, b: float((t5.block_scaled_linear(a, b, **kw).double() * g).sum())  # noqa: E731
    dx, dw = torch.autograd.grad(t5.block_scaled_linear(x, w, **kw), (x, w), g)
    with torch.no_grad():
        for t, d in ((x, dx), (w, dw)):
            for i, j in ((0, 5), (9, 2), (31, 30)):
                up, down = t.clone(), t.clone()
                up[i, j], down[i, j] = 2.0, -2.0
                at = (lambda v: (v, w)) if t is x else (lambda v: (x, v))
                diff = (loss(*at(up)) - loss(*at(down))) / 4.0
                assert abs(diff - float(d[i, j])) <= 1e-3 * max(1.0, abs(diff))


@pytest.mark.gpu
def test_linear_needs_only_what_is_asked():
    x, w = make(1, 40, 96, dtype=torch.bfloat16), make(2, 50, 96, dtype=torch.bfloat16)
    full_x, full_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = t5.block_scaled_linear(full_x, full_w)
    y.float().sum().backward()
    only_x = x.clone().requires_grad_()
    t5.block_scaled_linear(only_x, w).float().sum().backward()
    only_w = w.clone().requires_grad_()
    t5.block_scaled_linear(x, only_w).float().sum().backward()
    assert torch.equal(only_x.grad, full_x.grad) and torch.equal(only_w.grad, full_w.grad)
    with torch.no_grad():
        assert torch.equal(t5.block_scaled_linear(full_x, full_w), y) and not t5.block_scaled_linear(full_x, w).requires_grad
    # the tensors may change between the passes: their rounded forms are kept
    y = t5.block_scaled_linear(full_x, full_w)
    keep = full_x.grad.clone()
    full_x.grad = full_w.grad = None
    with torch.no_grad():
        full_x.zero_()
    y.float().sum().backward()
    assert torch.equal(full_x.grad, keep)
    # used twice
    z = w.clone().requires_grad_()
    (t5.block_scaled_linear(x, z).float().sum() + t5.block_scaled_linear(x, z).float().sum()).backward()
    assert torch.equal(z.grad.float(), 2 * only_w.grad.float())
    empty = torch.empty(0, 96, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    ze = w.clone().requires_grad_()
    t5.block_scaled_linear(empty, ze).sum().backward()
    assert tuple(empty.grad.shape) == (0, 96) and not bool(ze.grad.any())
    for a, b in ((x, w[:, :64]), (x.float(), w), (x, w[0]), (x, torch.empty(0, 96, dtype=x.dtype, device="cuda"))):
        with pytest.raises(ValueError):
            t5.block_scaled_linear(a, b)


# ------------------------------------------------------------ streams, graphs, devices (GPU)


@pytest.mark.gpu
def test_calls_side_by_side_on_streams():
    xs = [make(i, 60 + 40 * i, 700, dtype=torch.bfloat16) for i in range(4)]
    w = t5.quantize_blocks(make(9, 300, 700), multiplier="auto")
    want = [t5.block_scaled_mm(t5.quantize_blocks(x, multiplier="auto"), w) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(5):
        for i, (s, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(s):
                got[i].append(t5.block_scaled_mm(t5.quantize_blocks(x, multiplier="auto"), w))
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert all(torch.equal(t, v) for t in g)


@pytest.mark.gpu
def test_capture_and_replay():
    """A captured training step replays on new inputs; two graphs of the same
    calls do not share anything."""
    x = make(1, 100, 256, dtype=torch.bfloat16).requires_grad_()
    w = make(2, 130, 256, dtype=torch.bfloat16).requires_grad_()
    g = make(3, 100, 130, dtype=torch.bfloat16)

    def step():
        y = t5.block_scaled_linear(x, w)
        return (y.detach(), *torch.autograd.grad(y, (x, w), g))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in (11, 12):
        with torch.no_grad():
            x.copy_(make(seed, 100, 256))
            g.copy_(make(seed + 5, 100, 130) * 1e-3)
        want = step()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_the_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys

    code = """
import torch, tcgen05_b200 as t5
x = torch.randn(300, 512, device="cuda").bfloat16().requires_grad_(); w = torch.randn(200, 512, device="cuda").bfloat16().requires_grad_()
g = torch.randn(300, 200, device="cuda").bfloat16()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = t5.block_scaled_linear(x, w)
    grads = torch.autograd.grad(y, (x, w), g)
    one = t5.block_scaled_mm(t5.quantize_blocks(x[:1].detach()), t5.quantize_blocks(w.detach()))
    back = t5.dequantize_blocks(t5.quantize_blocks(x.detach(), multiplier="auto"))
graph.replay(); torch.cuda.synchronize()
y2 = t5.block_scaled_linear(x, w)
again = torch.autograd.grad(y2, (x, w), g)
assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, again))
assert torch.equal(one, t5.block_scaled_mm(t5.quantize_blocks(x[:1].detach()), t5.quantize_blocks(w.detach())))
print("captured")
"""
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parents[1])
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_threads_call_at_once():
    import threading

    xs = [make(i, 50 + 70 * i, 600, dtype=torch.bfloat16) for i in range(4)]
    w = make(9, 300, 600, dtype=torch.bfloat16)
    want = [t5.block_scaled_linear(x, w) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(30):
                if not torch.equal(t5.block_scaled_linear(xs[i], w), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.gpu
def test_second_derivative_is_refused():
    x = make(1, 20, 64).requires_grad_()
    w = make(2, 30, 64).requires_grad_()
    y = t5.block_scaled_linear(x, w)
    dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.gpu
def test_the_set_as_a_model_uses_it():
    """Two layers trained a step, then their weights held in 4 bits and served
    token by token: the served tokens are the batch's rows."""
    x = make(1, 96, 256, dtype=torch.bfloat16)
    w1 = (make(2, 384, 256) / 16).to(torch.bfloat16).requires_grad_()
    w2 = (make(3, 128, 384) / 20).to(torch.bfloat16).requires_grad_()
    h = torch.relu(t5.block_scaled_linear(x, w1, scaling="ue8m0"))
    y = t5.block_scaled_linear(h, w2, scaling="ue8m0")
    y.float().square().mean().backward()
    with torch.no_grad():
        for w in (w1, w2):
            assert bool(w.grad.isfinite().all()) and bool(w.grad.any())
            w -= 0.1 * w.grad
        held = [t5.quantize_blocks(w, scaling="ue8m0") for w in (w1, w2)]

        def serve(t):
            t = torch.relu(t5.block_scaled_mm(t5.quantize_blocks(t, scaling="ue8m0"), held[0]))
            return t5.block_scaled_mm(t5.quantize_blocks(t, scaling="ue8m0"), held[1])

        whole = t5.block_scaled_linear(torch.relu(t5.block_scaled_linear(x, w1, scaling="ue8m0")), w2, scaling="ue8m0")
        # K = 256 and 384 are too short to be split, so one token sums in the order of a batch
        one = torch.cat([serve(x[i:i + 1]) for i in range(x.shape[0])])
        assert torch.equal(one, serve(x)) and torch.equal(one, whole)


@pytest.mark.gpu
def test_one_tensor_as_both_operands():
    kw = dict(scaling="ue8m0")
    for rows, k in ((1, 64), (130, 333), (700, 520)):
        x = make(rows, rows, k, dtype=torch.bfloat16)
        q, same = t5.quantize_blocks(x, **kw), t5.quantize_blocks(x.clone(), **kw)
        assert torch.equal(t5.block_scaled_mm(q, q), t5.block_scaled_mm(q, same))
    # one leaf as both: its gradient is the sum of the two
    x = make(5, 96, 200, dtype=torch.float32)
    g = make(6, 96, 96)
    both, a, b = (x.clone().requires_grad_() for _ in range(3))
    t5.block_scaled_linear(both, both).backward(g)
    t5.block_scaled_linear(a, b).backward(g)
    assert torch.equal(both.grad, a.grad + b.grad)


@pytest.mark.gpu
def test_inference_mode():
    x, w = make(1, 70, 96, dtype=torch.bfloat16), make(2, 50, 96, dtype=torch.bfloat16)
    want = t5.block_scaled_linear(x, w)
    product = t5.block_scaled_mm(t5.quantize_blocks(x), t5.quantize_blocks(w))
    with torch.inference_mode():
        assert torch.equal(t5.block_scaled_linear(x, w), want)
        held = t5.quantize_blocks(w)
        assert torch.equal(t5.block_scaled_mm(t5.quantize_blocks(x.clone()), held), product)
    # what was rounded there serves outside
    assert torch.equal(t5.block_scaled_mm(t5.quantize_blocks(x), held), product)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["grad", "backward"])
def test_captured_backward_beside_a_living_graph(how):
    """An eager graph of the same leaves, made on a stream of its own, lives
    while a training step is captured."""
    x = make(1, 64, 256, dtype=torch.bfloat16).requires_grad_()
    w = make(2, 128, 256, dtype=torch.bfloat16).requires_grad_()
    g = make(3, 64, 128, dtype=torch.bfloat16)

    def step():
        y = t5.block_scaled_linear(x, w)
        if how == "grad":
            return torch.autograd.grad(y, (x, w), g)
        x.grad = w.grad = None
        y.backward(g)
        return x.grad, w.grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in step()]
        living = t5.block_scaled_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = torch.autograd.grad(living, (x, w), g)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
