"""Block-scaled calls: what autograd sees of them, extreme factors, aliases and moved memory, and roundings value by
value in the tensors' own types."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import tcgen05_b200 as t5
from tcgen05_b200 import blocks as bk
from test_blocks import BLOCK, E2M1, FORMS, TYPES, check_rows, define, make, product_bound

# ------------------------------------------------------------ autograd


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "w", "both"])
def test_second_derivative_is_refused_whatever_the_incoming_gradient(which):
    """dx depends on w and dw on x even where the incoming gradient is a constant: a loss of them has to refuse its
    backward pass, not to leave the terms out."""
    x, w = make(1, 20, 64), make(2, 30, 64)
    want = torch.autograd.grad(t5.block_scaled_linear(*(p := [t.clone().requires_grad_() for t in (x, w)])).sum(), p)
    x.requires_grad_(which != "w")
    w.requires_grad_(which != "x")
    leaves = [t for t in (x, w) if t.requires_grad]
    for weight in (None, torch.ones(20, 30, device="cuda")):
        y = t5.block_scaled_linear(x, w)
        out = y.sum() if weight is None else y
        got = torch.autograd.grad(out, leaves, weight, create_graph=True)
        for t, g in zip(leaves, got):
            assert g.requires_grad and torch.equal(g, want[0] if t is x else want[1])
            with pytest.raises(RuntimeError, match="differentiable once"):
                (y.square().sum() + g.square().sum()).backward(retain_graph=True)
        # what does not use them is differentiated as ever
        first = torch.autograd.grad(y.square().sum(), leaves)
        assert all(bool(t.isfinite().all()) and not t.requires_grad for t in first)


@pytest.mark.gpu
def test_out_is_seen_as_written():
    """A tensor that autograd saved may not be overwritten behind its back."""
    a, b = t5.quantize_blocks(make(1, 40, 64)), t5.quantize_blocks(make(2, 64, 64))

    def product(out):
        t5.block_scaled_mm(a, b, dtype=torch.float32, out=out)

    def values(out):
        t5.dequantize_blocks(a, out=out)

    for write in (product, values):
        buffer = make(3, 40, 64)
        w = torch.ones(40, 64, device="cuda", requires_grad=True)
        z = w * buffer
        version = buffer._version
        write(buffer)
        assert buffer._version == version + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        # a part of a larger tensor counts for the whole
        big = make(4, 50, 80)
        z = w * big[5:45, 8:72]
        write(big[5:45, 8:72])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.sum().backward()
        # a refused call writes nothing and counts nothing
        version = big._version
        with pytest.raises(ValueError):
            write(big[5:45, 8:71])
        assert big._version == version
        with torch.inference_mode():
            held = torch.zeros(40, 64, device="cuda")
            write(held)
            assert bool(held.any())
            held.zero_()
        with pytest.raises(RuntimeError, match="[Ii]nference tensor"):
            write(held)
        assert not bool(held.any())


@pytest.mark.gpu
def test_forward_mode_tangents_are_refused():
    from torch.autograd import forward_ad

    a, b = t5.quantize_blocks(make(1, 40, 64)), t5.quantize_blocks(make(2, 48, 64))
    x, w = make(3, 40, 64), make(4, 48, 64)
    with forward_ad.dual_level():
        c = forward_ad.make_dual(make(5, 40, 48), make(6, 40, 48))
        with pytest.raises(ValueError, match="tangent"):
            t5.block_scaled_mm(a, b, c)
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):
            t5.block_scaled_mm(a, b, c[0])
        with pytest.raises(ValueError, match="tangent"):
            t5.block_scaled_mm(a, b, dtype=torch.float32, out=c)
        values = forward_ad.make_dual(torch.zeros(40, 64, device="cuda"), x)
        with pytest.raises(ValueError, match="tangent"):
            t5.dequantize_blocks(a, out=values)
        for p, q in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
            with pytest.raises(ValueError, match="tangent"):
                t5.block_scaled_linear(p, q)
        assert torch.equal(t5.block_scaled_mm(a, b, forward_ad.unpack_dual(c).primal),
                           t5.block_scaled_mm(a, b, make(5, 40, 48)))


@pytest.mark.gpu
def test_saved_tensors_pass_through_hooks():
    """What the layer keeps may be moved to the host between the passes; what does not come back as it was is
    refused, not read."""
    x, w = make(1, 33, 96).requires_grad_(), make(2, 50, 96).requires_grad_()
    want = torch.autograd.grad(t5.block_scaled_linear(x, w).square().sum(), (x, w))
    with torch.autograd.graph.save_on_cpu():
        y = t5.block_scaled_linear(x, w).square().sum()
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w)), want))
    for unpack in (lambda t: t.cpu() if t.dtype == torch.uint8 else t, lambda t: t[:-1] if t.dtype == torch.uint8 else t,
                   lambda t: t.float() if t.dtype == torch.uint8 else t,
                   lambda t: torch.cat([t, t])[::2] if t.dtype == torch.uint8 else t,
                   lambda t: torch.cat([t[:1], t])[1:] if t.dtype == torch.uint8 else t):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = t5.block_scaled_linear(x, w).square().sum()
        with pytest.raises(ValueError, match="came back"):
            y.backward()


# ------------------------------------------------------------ what is kept


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [-1, 0, "both"])
@pytest.mark.parametrize("rows", [1, 70, 0])
def test_a_given_multiplier_is_kept_as_it_was(axis, rows):
    """A program that updates its scale in place does not change what was rounded with it before."""
    if rows == 0 and axis != -1:
        pytest.skip("blocks along an empty axis")
    x = make(1, rows, 96)
    scale = torch.full((1,), 8.0, device="cuda")
    got = t5.quantize_blocks(x, axis=axis, multiplier=scale)
    fixed = t5.quantize_blocks(x, axis=axis, multiplier=8.0)
    scale.fill_(0.25)
    for q, f in zip(got if axis == "both" else (got,), fixed if axis == "both" else (fixed,)):
        assert float(q.multiplier) == 8.0 and q.multiplier.shape == (1,)
        assert torch.equal(t5.dequantize_blocks(q), t5.dequantize_blocks(f))
        if rows:
            assert torch.equal(t5.block_scaled_mm(q, q), t5.block_scaled_mm(f, f))
    # any one-element form of it, and a captured call that reads its value at each replay
    for m in (torch.tensor(8.0, device="cuda"), torch.full((1, 1), 8.0, device="cuda"),
              torch.conj(torch.complex(torch.zeros(1, device="cuda"), torch.full((1,), -8.0, device="cuda"))).imag):
        q = t5.quantize_blocks(x, multiplier=m)
        assert float(q.multiplier) == 8.0
        assert torch.equal(q.data, t5.quantize_blocks(x, multiplier=8.0).data)


@pytest.mark.gpu
def test_a_captured_call_keeps_the_multiplier_of_its_replay():
    x = make(1, 33, 200, dtype=torch.bfloat16)
    scale = torch.full((1,), 2.0, device="cuda")
    t5.quantize_blocks(x, multiplier=scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = t5.quantize_blocks(x, multiplier=scale)
    for m in (4.0, 0.5):
        scale.fill_(m)
        graph.replay()
        scale.fill_(77.0)
        assert float(q.multiplier) == m
        assert torch.equal(t5.dequantize_blocks(q), t5.dequantize_blocks(t5.quantize_blocks(x, multiplier=m)))


# ------------------------------------------------------------ extreme factors


def extremes(seed, rows, k, power, dtype=torch.float32):
    """Normal values times 2^power, every third row zeros."""
    x = make(seed, rows, k, dtype=torch.float32).clamp(-3, 3)
    x[::3] = 0
    return (x.double() * 2.0 ** power).to(dtype)


def check_factors(qa, qb, alpha, dtype, c, form):
    """A product against its definition in 64 bits, the multipliers powers of two."""
    bare = [t5.BlockScaledRows(q.data, q.scales, q.k, scaling=q.scaling, scale_vec=q.scale_vec) for q in (qa, qb)]
    a, b = (t5.dequantize_blocks(q).double() for q in bare)
    factor = float(np.float32(alpha))
    for q in (qa, qb):
        factor /= 1.0 if q.multiplier is None else float(q.multiplier)
    want = factor * (a @ b.t()) + (0 if c is None else c.double())
    got = bk._mm(qa, qb, c, alpha, dtype, None, form).double()
    info = torch.finfo(dtype)
    err = abs(factor) * product_bound(a, b, qa.k, 0) + 2.0 ** -24 * (0 if c is None else c.double().abs())
    room = err + 1.01 * info.eps / 2 * (want.abs() + err) + info.smallest_normal * info.eps
    inside = want.abs() + room < info.max
    beyond = want.abs() - room > 2 * info.max
    assert bool(((got - want).abs() <= room)[inside].all())
    assert torch.equal(got[beyond], torch.sign(want[beyond]) * math.inf)
    assert not bool(got.isnan().any())
    return inside, beyond


@pytest.mark.gpu
@pytest.mark.parametrize("form", [0, 1, 2, 4, 8, 128, 256])
@pytest.mark.parametrize("m,n", [(300, 264), (260, 130), (5, 300)])
def test_factors_whose_product_leaves_f32(form, m, n):
    """alpha and the two reciprocals are no single F32 number: zero rows stay zero beside ones that overflow, and
    results within F32 keep their digits."""
    if m == 5 and form >= 128:
        pytest.skip("few rows take no such tile")
    k = 2100
    cases = [(76, 76, 1.0), (100, 100, 1.0), (115, 20, 1.0), (-65, -65, 1.0), (-66, -60, 1.0), (-60, -60, 1.37e-5),
             (66, -66, 2.0 ** 100), (-66, 66, 2.0 ** 100), (-40, 66, 1.37 * 2.0 ** -100), (50, 50, -1.37 * 2.0 ** -120),
             (-50, -50, 1.37 * 2.0 ** 120), (60, 60, 0.0)]
    for pa, pb, alpha in cases:
        qa = t5.quantize_blocks(extremes(1, m, k, pa), multiplier="auto")
        qb = t5.quantize_blocks(extremes(2, n, k, pb), multiplier="auto")
        for dtype in (torch.float32, torch.bfloat16):
            for c in (None, make(3, m, n), make(4, n, dtype=torch.bfloat16), make(5, n, m).t()):
                check_factors(qa, qb, alpha, dtype, c, form)


@pytest.mark.gpu
def test_a_sum_with_c_that_only_the_sum_brings_into_range():
    """alpha * sum beyond F32 and C of the other sign: one rounding, of the sum."""
    a = t5.quantize_blocks(torch.full((200, 64), 6.0, device="cuda"), scaling="ue8m0")
    b = t5.quantize_blocks(torch.full((200, 64), 6.0, device="cuda"), scaling="ue8m0")
    c = torch.full((200, 200), -1.5 * 2.0 ** 127, device="cuda")
    alpha = 2.0 ** 127 / 1152  # 64 * 36 = 2304: the product is 2^128
    for form in (1, 128, 256):
        got = bk._mm(a, b, c, alpha, torch.float32, None, form)
        assert bool((got.double() - 2.0 ** 126).abs().max() <= 2.0 ** 126 * 2.0 ** -20)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_of_large_and_small_tensors(dtype):
    """Zero rows beside values whose products overflow; small values whose products do not vanish."""
    for power in (80, -64):
        x, w, g = (extremes(i, 66, 128, power, dtype).requires_grad_(i < 2) for i in range(3))
        g = g[:, :66].contiguous()
        y = t5.block_scaled_linear(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), g)
        assert not bool(y[::3].any()) and not bool(y[:, ::3].any())
        for t in (y, dx, dw):
            assert not bool(t.isnan().any())
        if power < 0:
            r = [t5.dequantize_blocks(t5.quantize_blocks(t.detach(), multiplier="auto")).double() for t in (x, w)]
            want = r[0] @ r[1].t()
            room = product_bound(*r, 128, 0) + 1.01 * torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -133
            assert bool(want.any()) and bool(((y.double() - want).abs() <= room).all())


@pytest.mark.gpu
@pytest.mark.parametrize("vec", [2, 4])
def test_values_whose_scale_alone_leaves_f32(vec):
    """code * scale / multiplier where code * scale is beyond F32 and the value is not."""
    k = 96
    words = torch.arange(16, dtype=torch.int32, device="cuda").repeat(255, k // 16)
    scales = torch.arange(255, dtype=torch.uint8, device="cuda")[:, None].repeat(1, k // (32 if vec == 2 else 16))
    value = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device="cuda")[words.long()]
    exact = value * torch.exp2(torch.arange(255, dtype=torch.float64, device="cuda") - 127)[:, None]
    for m in (None, 1.0, 4.0, 2.0 ** 100, 2.0 ** -100, 2.0 ** 126, 2.0 ** -126, 3.0, 1e-30, 7e37):
        mult = None if m is None else torch.full((1,), m, device="cuda")
        q = t5.BlockScaledRows.from_words(words, scales, scaling="ue8m0", scale_vec=vec, multiplier=mult)
        back = 1.0 if m is None else float(np.float32(1) / np.float32(m))
        want = exact * back
        for dtype in (torch.float32, torch.bfloat16):
            out = torch.zeros(255, k + 3, dtype=dtype, device="cuda")[:, 1:k + 1]
            for got in (t5.dequantize_blocks(q, dtype=dtype), t5.dequantize_blocks(q, dtype=dtype, out=out)):
                # F32 first, then the type, by the definition
                np.testing.assert_array_equal(got.double().cpu().numpy(), want.float().to(dtype).double().cpu().numpy())


# ------------------------------------------------------------ aliases and moved memory


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(40, 131), (300, 267), (700, 1027)])
def test_chains_without_a_pause(m, n):
    """Each call reads what the one before has just written, in rows that share lines of memory; the same as with the
    device idle between them."""
    a, b = t5.quantize_blocks(make(1, m, 96)), t5.quantize_blocks(make(2, n, 96))
    x = make(3, m, n)

    def chain(pause):
        c, back, out = x.clone(), torch.empty(m, n, device="cuda"), []
        for i in range(40):
            for call in (lambda: t5.block_scaled_mm(a, b, c, alpha=0.25, dtype=torch.float32, out=c),
                         lambda: out.append(t5.quantize_blocks(c, axis="both", multiplier="auto")),
                         lambda: t5.dequantize_blocks(out[-1][0], out=back),
                         lambda: out.append(t5.quantize_blocks(back, scaling="ue8m0")),
                         lambda: t5.dequantize_blocks(out[-1], out=c)):
                call()
                if pause:
                    torch.cuda.synchronize()
        return c, back, out[-2][0].data, out[-2][1].data, out[-1].data

    want = chain(True)
    for _ in range(3):
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(chain(False), want))


@pytest.mark.gpu
def test_out_may_not_hold_a_multiplier():
    x = make(1, 40, 64)
    q = t5.quantize_blocks(x)
    big = torch.ones(40, 64, device="cuda")
    held = t5.BlockScaledRows(q.data, q.scales, 64, multiplier=big[3, 5:6])
    other = t5.quantize_blocks(make(2, 64, 64))
    for call in (lambda: t5.dequantize_blocks(held, out=big),
                 lambda: t5.block_scaled_mm(held, other, dtype=torch.float32, out=big),
                 lambda: t5.block_scaled_mm(other, held, dtype=torch.float32, out=torch.as_strided(big, (64, 40), (40, 1)))):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    assert bool((big == 1).all())


def held_parts(device):
    data = torch.zeros(130, 48, dtype=torch.uint8, device=device)
    scales = torch.zeros(2, 2, 512, dtype=torch.uint8, device=device)
    return data, scales, torch.ones(1, device=device)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("part", [0, 1, 2])
@pytest.mark.parametrize("how", ["free", "grow", "set"])
def test_rows_whose_memory_was_moved_are_refused(device, part, how):
    """The parts' storage freed (as sharded training does between uses), grown, or exchanged: no call may use the
    addresses of before."""
    parts = held_parts(device)
    q = t5.BlockScaledRows(parts[0], parts[1], 96, multiplier=parts[2])
    t = parts[part]
    if how == "free":
        t.untyped_storage().resize_(0)
    elif how == "grow":
        t.resize_(1 << 20)
    else:
        t.set_(torch.zeros_like(t))
    for call in (lambda: t5.dequantize_blocks(q), lambda: t5.block_scaled_mm(q, q)):
        with pytest.raises(ValueError, match="moved"):
            call()


@pytest.mark.gpu
def test_rounded_rows_whose_memory_was_freed_are_refused():
    q = t5.quantize_blocks(make(1, 40, 64))
    t5.block_scaled_mm(q, q)
    q.data.untyped_storage().resize_(0)
    for call in (lambda: t5.dequantize_blocks(q), lambda: t5.block_scaled_mm(q, q), lambda: q.scales, lambda: q.data):
        with pytest.raises(ValueError, match="moved"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 16])
def test_tensors_whose_memory_was_freed_are_refused(offset):
    def freed(*shape):
        n = math.prod(shape)
        t = torch.zeros(n + offset, device="cuda")[offset:].view(*shape)
        t.untyped_storage().resize_(0)
        return t

    a, b = t5.quantize_blocks(make(1, 40, 64)), t5.quantize_blocks(make(2, 48, 64))
    x, w = make(1, 40, 64), make(2, 48, 64)
    for call in (lambda: t5.quantize_blocks(freed(40, 64)), lambda: t5.block_multiplier(freed(40, 64)),
                 lambda: t5.quantize_blocks(x, multiplier=freed(1)), lambda: t5.block_scaled_mm(a, b, freed(40, 48)),
                 lambda: t5.block_scaled_mm(a, b, dtype=torch.float32, out=freed(40, 48)),
                 lambda: t5.dequantize_blocks(a, out=freed(40, 64)), lambda: t5.block_scaled_linear(freed(40, 64), w),
                 lambda: t5.block_scaled_linear(x, freed(48, 64))):
        with pytest.raises(ValueError, match="was freed"):
            call()


# ------------------------------------------------------------ roundings, value by value


def steps_of(form):
    return [m / 8 * 2.0 ** e for m in range(8, 16) for e in (-6, 0, 5)] if form[0] == "ue4m3" else \
        [2.0 ** e for e in (-6, 0, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
def test_ties_and_the_types_own_neighbours(form, dtype):
    """Elements at every border of E2M1 times a scale and the type's next values on either side, which are other
    values than the border."""
    blocks = []
    for step in steps_of(form):
        ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64) * step
        tie = ties.to(dtype)
        assert torch.equal(tie.double(), ties)
        for side in (None, math.inf, 0.0):
            t = tie if side is None else torch.nextafter(tie, torch.full_like(tie, side))
            assert side is None or not bool((t == tie).any())
            for sign in (1, -1):
                blocks.append(torch.cat([torch.tensor([6 * step]).to(dtype), sign * t,
                                         torch.zeros(BLOCK[form] - 8, dtype=dtype)]))
    x = torch.stack(blocks).cuda()
    for m in (1.0, 0.25, 2.0 ** 60, 2.0 ** -60, 2.0 ** 70, 1.5):
        codes, scale, _ = define(x, form, m)
        kw = dict(scaling=form[0], scale_vec=form[1], multiplier=None if m == 1 else m)
        check_rows(t5.quantize_blocks(x, **kw), codes, scale)
        check_rows(t5.quantize_blocks(x.t().contiguous(), axis=0, **kw), codes, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES[1:], ids=lambda t: str(t)[6:])
def test_every_16_bit_element_against_every_significand_of_a_scale(form, dtype):
    block = BLOCK[form]
    every = torch.arange(1, 0x7F80 if dtype == torch.bfloat16 else 0x7C00, dtype=torch.int16).view(dtype)
    rows = []
    for step in steps_of(form)[1::3]:  # every significand, the middle exponent
        v = every[(every.double() >= 0.05 * step) & (every.double() <= 6 * step)]
        v = torch.nn.functional.pad(v, (0, -v.numel() % (block - 1))).view(-1, block - 1)
        rows.append(torch.cat([torch.full((v.shape[0], 1), 6 * step, dtype=dtype), v], 1))
    x = torch.cat(rows).cuda()
    for m in (1.0, 2.0 ** 7, 2.0 ** 60, 2.0 ** -60):
        # the elements' quotients are those of m = 1 with a scale that is m times larger
        kw = dict(scaling=form[0], scale_vec=form[1], multiplier=None if m == 1 else m)
        codes, scale, _ = define(x, form, m)
        check_rows(t5.quantize_blocks(x, **kw), codes, scale)
    codes, scale, _ = define(-x, form)
    check_rows(t5.quantize_blocks(-x.t(), axis=0, scaling=form[0], scale_vec=form[1]), codes, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}-{f[1]}")
@pytest.mark.parametrize("dtype", TYPES[1:], ids=lambda t: str(t)[6:])
def test_every_16_bit_value_as_a_blocks_largest(form, dtype):
    every = torch.arange(0, 0x8000, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(every.numel(), BLOCK[form], dtype=dtype)
    x[:, 3] = every
    x[:, 5] = -(every.double() / 3).to(dtype)
    x = x.cuda()
    for ceil in ((False, True) if form[0] == "ue8m0" else (False,)):
        for m in (1.0, 2.0 ** 11, 2.0 ** -20):
            codes, scale, _ = define(x, form, m, ceil)
            kw = dict(scaling=form[0], scale_vec=form[1], multiplier=None if m == 1 else m)
            if form[0] == "ue8m0":
                kw["scale_rounding"] = "ceil" if ceil else "floor"
            check_rows(t5.quantize_blocks(x, **kw), codes, scale)


# ------------------------------------------------------------ refusals, each by its own words (CPU)


@pytest.mark.parametrize("kw,words", [
    (dict(scaling="ue4m3", scale_vec=2), "takes scaling"), (dict(scaling="ue5m3"), "takes scaling"),
    (dict(scaling="ue8m0", scale_vec=1), "takes scaling"), (dict(scaling="ue4m3", scale_rounding="floor"), "scale_rounding is"),
    (dict(scaling="ue8m0", scale_rounding="nearest"), "scale_rounding is"),
    (dict(scaling="ue8m0", scale_rounding="up"), "scale_rounding is"), (dict(axis=1), "axis is"),
    (dict(axis="rows"), "axis is"), (dict(multiplier="max"), "multiplier is a number"),
    *[(dict(multiplier=m), "multiplier must be positive") for m in (0.0, -2.0, math.nan, math.inf, 1e300, 1e-300, 1e-45)],
    (dict(), "must be a dense tensor on a CUDA device"),
])
def test_each_bad_argument_is_named(kw, words):
    with pytest.raises(ValueError, match=words):
        t5.quantize_blocks(torch.zeros(4, 64), **kw)


def test_each_bad_tensor_is_named():
    calls = (t5.quantize_blocks, t5.block_multiplier, lambda v: t5.block_scaled_linear(v, v))
    for call in calls:
        for dtype in (torch.float64, torch.int32, torch.float8_e4m3fn):
            with pytest.raises(ValueError, match="must be float32, bfloat16 or float16"):
                call(torch.zeros(4, 64, dtype=dtype))
        with pytest.raises(ValueError, match="on a CUDA device"):
            call(torch.zeros(4, 64))
        with pytest.raises(ValueError, match="must be a torch tensor"):
            call([[1.0]])


def test_each_bad_word_tensor_is_named():
    words, scales = torch.zeros(4, 70, dtype=torch.int32), torch.zeros(4, 5, dtype=torch.uint8)
    make_rows = t5.BlockScaledRows.from_words
    for w, s, message in ((words, scales, "on one CUDA device"), (words.float(), scales, "tensor of integers"),
                          (words[0], scales, "tensor of integers"), (words, scales[:, :4], r"scales must be \[4, 5\]"),
                          (words[:, :0], scales[:, :0], "K must be between"), ([[1]], scales, "words must be a torch tensor"),
                          (words, [[1]], "scales must be a torch tensor"),
                          (words[:1].expand(1, 70).repeat(1, 1000), scales, "K must be between 1 and 65536, not 70000")):
        with pytest.raises(ValueError, match=message):
            make_rows(w, s)
