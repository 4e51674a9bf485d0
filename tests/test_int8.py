"""Experts in 8-bit integers (int8.quantize_rows, grouped_mm_int8, int8_moe) against 64-bit restatements, and their
refusals."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from test_experts import BF16, DEV, F16, F32, ROUND, SIZES, device_word, normal, offsets_of  # noqa: F401
from test_experts_edges import HALF_STEP

from blackhole_b200 import _lib, int8, router
from blackhole_b200 import hex_data as hd


def quantized(x):
    """Whole numbers (float64) and scales of x's rows in 64 bits; and |127 x / max| itself."""
    x = x.double()
    largest = x.abs().amax(-1, keepdim=True)
    t = torch.where(largest > 0, x * 127 / largest, 0.0)
    return torch.round(t), (largest / 127)[..., 0], t


def int8_stack(shape, seed):
    """Any 8-bit values (-128 among them), rows on 16 bytes, and scales."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-128, 128, shape, generator=g, dtype=torch.int16).to(torch.int8)
    return w, torch.rand(shape[:-1], generator=g) * 0.02 + 1e-3


def product(q, x_scale, w, w_scale, offsets, rows):
    """out [R, N] in 64 bits and the sum of magnitudes, zero for rows of no group."""
    want = torch.zeros(rows, w.shape[1], dtype=torch.float64)
    mass = torch.zeros_like(want)
    off = offsets.tolist()
    for e in range(w.shape[0]):
        a, m = q[off[e]:off[e + 1]].double(), w[e].double()
        s = x_scale[off[e]:off[e + 1], None].double() * w_scale[e].double()
        want[off[e]:off[e + 1]], mass[off[e]:off[e + 1]] = (a @ m.t()) * s, (a.abs() @ m.abs().t()) * s
    return want, mass


def assert_product(got, want, mass, dtype):
    """Exact sums: the scales' product, the whole number in f32 and their product are rounded (3 x 2^-24), and where a
    reduction is split each of up to 16 parts, with the additions (19 x 2^-24 of the magnitudes); then the type."""
    assert got.dtype == dtype and got.shape == want.shape
    f32 = 2.0 ** -24 * (4 * want.abs() + 19 * mass)
    bound = f32 + 1.01 * ROUND[dtype] * (want.abs() + f32) + HALF_STEP[dtype]
    worst = ((got.double().cpu() - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert torch.isfinite(got).all() and worst <= 0, f"{float(worst)} over the bound"


# ------------------------------------------------------------------ rows to 8 bits
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("width", [1, 7, 8, 64, 100, 513, 768, 2048, 2049, 4096, 8192, 20000, 40008])
def test_quantize_rows(width, dtype):
    x = normal((19, width), dtype, width, 3.0)
    x[3] = 0
    x[4] *= 0
    x[4, width // 2] = -1
    x[5] = x[5].abs().clamp(max=1)      # plenty of 127 x / max = 63.5
    x[5, ::3] = 0.5
    x[5, 0] = 1
    q, scale = int8.quantize_rows(x.to(DEV))
    want, want_scale, _ = quantized(x)
    assert q.dtype == torch.int8 and q.stride(0) % 16 == 0 and torch.equal(q.cpu().double(), want)
    assert ((scale.double().cpu() - want_scale).abs() <= 2.0 ** -24 * want_scale).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_quantize_rows_far_from_one(dtype):
    """Rows at the ends of the type's range, subnormal ones, and rows that hold no numbers."""
    base = normal((9, 96), F32, 3)
    for i, factor in enumerate([1e38, 3e-38, 1e-40, 1e-44, 1e30, 1e-30]):
        base[i] = base[i] / base[i].abs().max() * factor * (1 if i else 3)
    x = base.to(dtype)
    x[6, 5], x[7, 9], x[8, 11] = math.inf, -math.inf, math.nan
    q, scale = int8.quantize_rows(x.to(DEV))
    want, want_scale, _ = quantized(x[:6])
    assert torch.equal(q[:6].cpu().double(), want)
    assert ((scale[:6].double().cpu() - want_scale).abs() <= 2.0 ** -24 * want_scale + 2.0 ** -150).all()
    assert not q[6:].any() and scale[6:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_quantize_rows_at_borders(dtype):
    """Values next to every border n + 1/2 of many largest ones, and on them, above and below."""
    g = torch.Generator().manual_seed(4)
    largest = (torch.rand(300, 1, generator=g).double() + 0.5) * 2.0 ** torch.randint(-12, 8, (300, 1), generator=g)
    largest = largest.to(dtype).double()
    near = ((torch.arange(127) + 0.5) / 127 * largest).to(dtype)
    step = torch.finfo(dtype).eps * near
    x = torch.cat([largest.to(dtype), near, near + step, -(near - step), -near, near + step / 2], 1)
    q, _ = int8.quantize_rows(x.to(DEV))
    assert torch.equal(q.cpu().double(), quantized(x)[0])


@pytest.mark.gpu
def test_quantize_rows_of_views_and_stacks():
    x = normal((40, 300), BF16, 5).to(DEV)
    for view in (x[:, 3:250], x[::2, 8:136], x.t(), x[0], x[:1, :64], x[:, :1].expand(40, 32), x[:0]):
        q, scale = int8.quantize_rows(view)
        want, want_scale, _ = quantized(view.cpu()) if len(view) else (view.cpu().double(), scale.cpu().double(), None)
        assert q.shape == view.shape and scale.shape == view.shape[:-1]
        assert torch.equal(q.cpu().double(), want) and torch.allclose(scale.double().cpu(), want_scale, rtol=2.0 ** -23, atol=0)
    w = normal((3, 20, 50), F32, 6).to(DEV)
    q, scale = int8.quantize_rows(w)
    each = [int8.quantize_rows(m) for m in w]
    assert all(torch.equal(q[e], a) and torch.equal(scale[e], s) for e, (a, s) in enumerate(each))


# ------------------------------------------------------------------ products
@pytest.mark.gpu
@pytest.mark.parametrize("widths", [(8, 16), (136, 72), (256, 128), (264, 200), (512, 64), (13, 7), (101, 67), (40, 1000)], ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_grouped_mm_int8(sizes, widths):
    sizes, (n, k) = SIZES[sizes], widths
    dtype = (BF16, F16, F32)[(n + k + len(sizes)) % 3]
    rows = sum(sizes)
    x, x_scale = int8_stack((rows, k), 1)
    w, w_scale = int8_stack((len(sizes), n, k), 2)
    off = offsets_of(sizes)
    want, mass = product(x, x_scale, w, w_scale, off, rows)
    got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), w_scale.to(DEV), off.to(DEV), x_scale=x_scale.to(DEV), out_dtype=dtype)
    assert_product(got, want, mass, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows", [1, 8, 40, 300, 2000])
@pytest.mark.parametrize("widths", [(1536, 2048), (2048, 768), (776, 1032)], ids=str)
def test_grouped_mm_int8_of_rows_quantized_on_the_way(widths, rows, dtype):
    """The widths of the 96-expert layer and odd multiples of 8; the product of quantize_rows' numbers, bit for bit."""
    (n, k), E = widths, 5
    sizes = np.bincount(np.random.RandomState(rows).randint(0, E, rows), minlength=E)
    x = normal((rows, k), dtype, 3)
    wd, wd_scale = int8.quantize_rows(normal((E, n, k), F32, 4, 0.02).to(DEV))
    off = offsets_of(sizes, dtype=torch.int64)
    q, scale, _ = quantized(x)
    want, mass = product(q, scale, wd.cpu(), wd_scale.cpu(), off, rows)
    got = int8.grouped_mm_int8(x.to(DEV), wd, wd_scale, off.to(DEV))
    assert_product(got, want, mass * (1 + 2.0 ** -20), dtype)
    xq, x_scale = int8.quantize_rows(x.to(DEV))
    assert torch.equal(int8.grouped_mm_int8(xq, wd, wd_scale, off.to(DEV), x_scale=x_scale, out_dtype=dtype), got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(1, 512, 4096), (7, 776, 1624), (300, 512, 4096), (129, 24, 8000), (5, 2049, 33)])
def test_one_matrix_for_all_rows(rows, n, k):
    """Without offsets; few tiles of a long reduction are split over more pairs."""
    x, x_scale = int8_stack((rows, k), 5)
    w, w_scale = int8_stack((n, k), 6)
    want, mass = product(x, x_scale, w[None], w_scale[None], torch.tensor([0, rows]), rows)
    for dtype in (BF16, F32):
        got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), w_scale.to(DEV), x_scale=x_scale.to(DEV), out_dtype=dtype)
        assert_product(got, want, mass, dtype)
    same = int8.grouped_mm_int8(x.to(DEV), w[None].to(DEV), w_scale[None].to(DEV), torch.tensor([0, rows], device=DEV),
                                x_scale=x_scale.to(DEV), out_dtype=F32)
    assert torch.equal(same, got)


@pytest.mark.gpu
def test_largest_sums():
    """Sums at the ends of int32: products of -128 and -128 over the longest reduction, and their negatives."""
    k = int8.MAX_K
    x, w = torch.full((2, k), -128, dtype=torch.int8), torch.full((8, k), -128, dtype=torch.int8)
    w[1::2] = 127
    one = torch.ones(8)
    want, mass = product(x, one[:2], w[None], one[None], torch.tensor([0, 2]), 2)
    assert want.max() == 16384 * k and want.max() < 2 ** 31
    got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), one.to(DEV), x_scale=one[:2].to(DEV), out_dtype=F32)
    assert_product(got, want, mass, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("widths", [(72, 264), (9, 11)], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
def test_strides_gaps_and_out(widths, dtype):
    """Rows of no group are zero, whatever their scales; every operand may be a part of a larger array; what stands
    around `out` stays."""
    (n, k), sizes = widths, [40, 0, 300, 17]
    E, first = len(sizes), 5
    rows = first + sum(sizes) + 9
    x, x_scale = int8_stack((rows, k + 21), 7)
    x_scale[:first], x_scale[-9:] = math.nan, math.inf
    w, w_scale = int8_stack((E, n + 3, k + 16), 8)
    off = offsets_of(sizes, first)
    want, mass = product(x[:, 5:5 + k], torch.nan_to_num(x_scale, 0, 0, 0), w[:, :n, :k], w_scale[:, :n], off, rows)
    big = torch.full((rows, n + 24), 7.0, dtype=dtype, device=DEV)
    xd, wd, sd = x.to(DEV)[:, 5:5 + k], w.to(DEV)[:, :n, :k], w_scale.to(DEV)[:, :n]
    for lo in (8, 3):
        big.fill_(7.0)
        got = int8.grouped_mm_int8(xd, wd, sd, off.to(DEV), x_scale=x_scale.to(DEV), out=big[:, lo:lo + n])
        assert got.data_ptr() == big[:, lo:].data_ptr()
        assert_product(got, want, mass, dtype)
        assert (big[:, :lo] == 7).all() and (big[:, lo + n:] == 7).all()
    turned = torch.empty(n, rows, dtype=dtype, device=DEV).t()
    assert torch.equal(int8.grouped_mm_int8(xd, wd, sd, off.to(DEV), x_scale=x_scale.to(DEV), out=turned), got)


@pytest.mark.gpu
def test_rows_behind_the_last_group_and_bad_offsets():
    from blackhole_b200.hex_moe import device_status
    x, x_scale = int8_stack((64, 32), 9)
    w, w_scale = int8_stack((3, 48, 32), 10)
    args = (x.to(DEV), w.to(DEV), w_scale.to(DEV))
    for off in ([0, 10, 10, 64], [0, 40, 30, 64], [-5, 10, 90, 64]):
        got = int8.grouped_mm_int8(*args, torch.tensor(off, device=DEV), x_scale=x_scale.to(DEV))
        assert torch.isfinite(got).all()
        assert device_status(0) == (0 if off[1] == 10 and off[0] == 0 else 8)


@pytest.mark.gpu
def test_rows_that_are_no_numbers_stay_among_themselves():
    x = normal((10, 64), BF16, 11)
    x[3, 5] = math.nan
    x[7, 1] = math.inf
    w, w_scale = int8_stack((24, 64), 12)
    got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), w_scale.to(DEV))
    bad = torch.tensor([3, 7])
    assert got[bad].isnan().all() and torch.isfinite(got[[0, 1, 2, 4, 5, 6, 8, 9]]).all()


# ------------------------------------------------------------------ the layer
def layer_reference(x, weights, ids, w13, s13, w2, s2):
    """The layer in 64 bits, and how far f32 arithmetic may take it: a value of the activation that lies within its
    error of a border may land on the next whole number."""
    T, k = ids.shape
    inter = w2.shape[2]
    q, scale, _ = quantized(x)
    out = torch.zeros(T, x.shape[1], dtype=torch.float64)
    slack = torch.zeros_like(out)
    y_round = ROUND[F16 if x.dtype == F16 else BF16]
    for e in range(w13.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if not len(t):
            continue
        h = q[t] @ w13[e].double().t() * s13[e].double() * scale[t][:, None]
        g, u = h[:, :inter], h[:, inter:]
        act = g * torch.sigmoid(g) * u
        # silu and the products in f32: a few roundings, and a fast exponential (2 + 1.2 |g| units)
        off = act.abs() * (16 + 3 * g.abs()) * 2.0 ** -23
        aq, a_scale, at = quantized(act)
        doubt = 127 * (off + off.amax(1, keepdim=True)) / act.abs().amax(1, keepdim=True).clamp(min=1e-300) + 2.0 ** -15
        flips = (((at.abs() - at.abs().floor()) - 0.5).abs() <= doubt).double()
        w = weights[t, j].double()[:, None]
        y = aq @ w2[e].double().t() * s2[e].double() * a_scale[:, None] * w
        rel = (off.amax(1, keepdim=True) / act.abs().amax(1, keepdim=True).clamp(min=1e-300)) + 2.0 ** -21
        off_y = flips @ w2[e].double().abs().t() * s2[e].double() * a_scale[:, None] * w.abs() + rel * y.abs()
        out.index_add_(0, t, y)
        slack.index_add_(0, t, off_y + 1.01 * y_round * (y.abs() + off_y) + 2.0 ** -23 * k * y.abs() + HALF_STEP[F16])
    return out, slack


def layer_inputs(E, H, I, dtype, tokens, k, seed):
    weights, ids = hd.synth_routing(tokens, E, k, seed=seed)
    x = normal((tokens, H), dtype, seed + 1)
    w13 = int8.quantize_rows(normal((E, 2 * I, H), F32, seed + 2, H ** -0.5).to(DEV))
    w2 = int8.quantize_rows(normal((E, H, I), F32, seed + 3, I ** -0.5).to(DEV))
    return x, weights.float(), ids, w13, w2


def assert_layer(got, x, weights, ids, w13, w2):
    want, slack = layer_reference(x, weights, ids, *(t.cpu() for t in (*w13, *w2)))
    assert got.dtype == x.dtype and got.shape == x.shape
    bound = slack + 1.01 * ROUND[x.dtype] * (want.abs() + slack) + HALF_STEP[x.dtype]
    worst = ((got.double().cpu() - want).abs() - bound).max()
    assert torch.isfinite(got).all() and worst <= 0, f"{float(worst)} over the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("tokens,E,k,H,I", [(1, 4, 2, 64, 32), (37, 6, 3, 128, 96), (200, 12, 4, 272, 208), (700, 3, 1, 48, 16),
                                            (33, 96, 8, 2048, 768), (2500, 5, 2, 64, 48)])
def test_int8_moe(tokens, E, k, H, I, dtype):
    x, weights, ids, w13, w2 = layer_inputs(E, H, I, dtype, tokens, k, 60)
    ids[ids == 1] = 0                             # an expert without rows, one reached twice by a token
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), *w13, *w2)
    assert_layer(got, x, weights, ids, w13, w2)
    assert torch.equal(int8.int8_moe(x.to(DEV), weights.to(DEV), ids.int().to(DEV), *w13, *w2), got)


@pytest.mark.gpu
def test_int8_moe_without_tokens_and_with_bad_ids():
    from blackhole_b200.hex_moe import device_status
    x, weights, ids, w13, w2 = layer_inputs(4, 64, 32, BF16, 300, 2, 70)
    xd, wd = x.to(DEV), weights.to(DEV)
    assert int8.int8_moe(xd[:0], wd[:0], ids[:0].to(DEV), *w13, *w2).shape == (0, 64)
    bad = ids.clone()
    bad[::7, 0], bad[3], bad[5, 1] = -1, 4, 2 ** 40
    got = int8.int8_moe(xd, wd, bad.to(DEV), *w13, *w2)
    assert device_status(0) & 2
    good = (bad >= 0) & (bad < 4)
    same = int8.int8_moe(xd, torch.where(good, weights, 0.0).to(DEV), bad.clamp(0, 3).to(DEV), *w13, *w2)
    assert torch.equal(same, got) and not got[3].any()
    nobody = int8.int8_moe(xd, wd, torch.full_like(bad, -1).to(DEV), *w13, *w2)
    assert device_status(0) & 2 and not nobody.any()


@pytest.mark.gpu
def test_tokens_that_are_no_numbers_stay_among_themselves():
    x, weights, ids, w13, w2 = layer_inputs(4, 64, 32, BF16, 40, 2, 75)
    x[7, 3], x[20] = math.nan, math.inf
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), *w13, *w2)
    fine = torch.ones(40, dtype=torch.bool)
    fine[[7, 20]] = False
    assert got[7].isnan().all() and got[20].isnan().all()
    assert_layer(got.cpu()[fine], x[fine], weights[fine], ids[fine], w13, w2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_scales_whose_product_is_no_normal_number(dtype):
    x = (normal((40, 512), F32, 130) * 1e-35).to(dtype)
    w, ws = int8_stack((2, 96, 512), 131)
    ws, off = torch.full_like(ws, 1e-5), offsets_of([17, 23])
    q, scale, _ = quantized(x)
    assert float((scale.max() * ws.max())) < 2.0 ** -130
    want, mass = product(q, scale, w, ws, off, 40)
    got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), ws.to(DEV), off.to(DEV), out_dtype=dtype)
    assert_product(got, want, mass, dtype)


@pytest.mark.gpu
def test_a_stack_that_streams_through_l2():
    """Matrices of more than 64 MB read once, and the same product of a part of them that is not: bit for bit."""
    E, n, k = 40, 1024, 2048
    w = torch.randint(-127, 128, (E, n, k), dtype=torch.int8, device=DEV)
    ws = torch.rand(E, n, device=DEV)
    x = normal((80, k), BF16, 120).to(DEV)
    off = torch.arange(0, 81, 2, dtype=torch.int32, device=DEV)
    got = int8.grouped_mm_int8(x, w, ws, off)
    for e in (0, 7, 39):
        rows = slice(2 * e, 2 * e + 2)
        one = int8.grouped_mm_int8(x[rows], w[e:e + 1], ws[e:e + 1], torch.tensor([0, 2], device=DEV), out_dtype=F32)
        q, scale, _ = quantized(x[rows].cpu())
        want, mass = product(q, scale, w[e:e + 1].cpu(), ws[e:e + 1].cpu(), torch.tensor([0, 2]), 2)
        assert_product(one, want, mass, F32)
        assert_product(got[rows], want, mass, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,E,n,k", [(3, 5, 96, 160), (300, 40, 320, 1104), (2500, 7, 512, 256)])
def test_operands_written_just_before(rows, E, n, k):
    """Rows, matrices, scales and offsets rewritten on the stream before each product, by calls not waited for."""
    g = torch.Generator().manual_seed(rows)
    sets = []
    for i in range(4):
        cuts = torch.randint(0, rows + 1, (E - 1,), generator=g).sort().values
        off = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([rows])]).int()
        sets.append((normal((rows, k), BF16, 200 + i), torch.randint(-127, 128, (E, n, k), generator=g).to(torch.int8),
                     torch.rand(E, n, generator=g), off))
    sets = [tuple(t.to(DEV) for t in s) for s in sets]
    alone = []
    for s in sets:
        alone.append(int8.grouped_mm_int8(*(t.clone() for t in s)))
        torch.cuda.synchronize()
    q, scale, _ = quantized(sets[0][0].cpu())
    want, mass = product(q, scale, sets[0][1].cpu(), sets[0][2].cpu(), sets[0][3].long().cpu(), rows)
    assert_product(alone[0], want, mass, BF16)
    held = [torch.empty_like(t) for t in sets[0]]
    order = [i % 4 for i in range(0, 60, 3)] + [0, 0, 2, 1, 3, 1]
    got = []
    for i in order:
        for h, t in zip(held, sets[i]):
            h.copy_(t)
        got.append(int8.grouped_mm_int8(*held))
    for i, y in zip(order, got):
        assert torch.equal(y, alone[i])


@pytest.mark.gpu
def test_int8_moe_written_just_before():
    args = [layer_inputs(6, 128, 64, BF16, 64, 3, seed) for seed in (90, 95)]
    a, b = ([x.to(DEV), w.to(DEV), ids.to(DEV), *(t.to(DEV) for t in (*w13, *w2))] for x, w, ids, w13, w2 in args)
    alone = [int8.int8_moe(*(t.clone() for t in s)) for s in (a, b)]
    torch.cuda.synchronize()
    held = [torch.empty_like(t) for t in a]
    got = []
    for i in (0, 1) * 10:
        for h, t in zip(held, (a, b)[i]):
            h.copy_(t)
        got.append(int8.int8_moe(*held))
    for i, y in enumerate(got):
        assert torch.equal(y, alone[i % 2])


@pytest.mark.gpu
def test_int8_moe_views_streams_and_graphs():
    x, weights, ids, w13, w2 = layer_inputs(6, 128, 64, BF16, 90, 3, 80)
    xd, wd, idd = x.to(DEV), weights.to(DEV), ids.to(DEV)
    want = int8.int8_moe(xd, wd, idd, *w13, *w2)
    wide = torch.zeros(90, 136, dtype=BF16, device=DEV)
    wide[:, 3:131] = xd
    part = torch.zeros(6, 130, 160, dtype=torch.int8, device=DEV)
    part[:, :128, 5:133] = w13[0]
    assert torch.equal(int8.int8_moe(wide[:, 3:131], wd.bfloat16().float(), idd, part[:, :128, 5:133], *w13[1:], *w2),
                       int8.int8_moe(xd, wd.bfloat16(), idd, *w13, *w2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = int8.int8_moe(xd, wd, idd, *w13, *w2)
    side.synchronize()
    assert torch.equal(other, want)
    held, held_ids = torch.zeros_like(xd), torch.zeros_like(idd)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(int8.int8_moe(held, wd, held_ids, *w13, *w2))
    held.copy_(xd)
    held_ids.copy_(idd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):                        # both graphs at once
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.gpu
def test_ordinary_calls_and_the_checked_ones_agree():
    """What _call takes and what goes through Python's checks is the same call: an `out`, or ids that are not
    contiguous, send it there."""
    x, weights, ids, w13, w2 = layer_inputs(6, 128, 64, F16, 70, 3, 100)
    xd, wd, idd = x.to(DEV), weights.to(DEV), ids.to(DEV)
    want = int8.int8_moe(xd, wd, idd, *w13, *w2)
    assert torch.equal(int8.int8_moe(xd, wd, idd.t().contiguous().t(), *w13, *w2), want)
    assert torch.equal(int8.int8_moe(xd, wd.double(), idd.short(), *w13, *w2), want)
    off = offsets_of([20, 0, 50, 0, 0, 0]).to(DEV)
    out = torch.empty(70, 128, dtype=F16, device=DEV)
    assert torch.equal(int8.grouped_mm_int8(xd, *w13, off), int8.grouped_mm_int8(xd, *w13, off, out=out))


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,E,k,H,I", [(31, 5, 4, 1024, 32), (32, 5, 4, 1024, 32), (33, 5, 4, 1024, 32), (8, 5, 33, 64, 32), (1, 3, 200, 32, 16)])
def test_few_tokens_quantized_with_the_plan(tokens, E, k, H, I):
    """Up to 32 tokens whose slots' rows are up to 128 KB go through the plan's kernel, the next ones through two; more
    slots a token than a warp has lanes."""
    g = torch.Generator().manual_seed(110)
    x, weights = normal((tokens, H), BF16, 111), torch.rand(tokens, k, generator=g) / k
    ids = torch.randint(0, E, (tokens, k), generator=g)
    w13 = int8.quantize_rows(normal((E, 2 * I, H), F32, 112, H ** -0.5).to(DEV))
    w2 = int8.quantize_rows(normal((E, H, I), F32, 113, I ** -0.5).to(DEV))
    for rows in (x.to(DEV), torch.cat([x, x], 1).to(DEV)[:, 1:H + 1]):     # and rows that do not begin on 16 bytes
        got = int8.int8_moe(rows, weights.to(DEV), ids.to(DEV), *w13, *w2)
        assert_layer(got, rows.cpu(), weights, ids, w13, w2)


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [1, 2047, 2048, 2049, 9001, 40000])
def test_plan_of_many_slots_and_experts(slots):
    """Routing to up to 2048 experts, from one slot to more than one block counts: every token finds its expert."""
    E, H, I = 2048, 16, 16
    g = torch.Generator().manual_seed(slots)
    x, ids = normal((slots, H), F32, 90), torch.randint(0, E, (slots, 1), generator=g)
    w13 = int8.quantize_rows(normal((E, 2 * I, H), F32, 91).to(DEV))
    w2 = int8.quantize_rows(normal((E, H, I), F32, 92).to(DEV))
    some = torch.arange(0, slots, max(1, slots // 200))
    weights = torch.ones(slots, 1)
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), *w13, *w2)
    assert_layer(got.cpu()[some], x[some], weights[some], ids[some], w13, w2)


@pytest.mark.gpu
def test_from_tiers_through_router_to_output():
    """As it is served: HEX tiers become 8-bit stacks, logits are routed, the layer runs; against 64 bits, and near the HEX layer."""
    from blackhole_b200.hex_moe import HexTier, dequant_all, hex_moe
    E, H, I, k, T = 8, 256, 128, 2, 50
    L = hd.synth_layer(E, H, I, "mixed", 32, seed=70, device=DEV)
    tiers = [HexTier(t["bits"], t["experts"], t["gate_proj"], t["up_proj"], t["down_proj"]).prepare(E) for t in L.tiers]
    w13, w2 = (int8.quantize_rows(w) for w in dequant_all(tiers, F32))
    x, logits = hd.synth_x(T, H, seed=72, device=DEV).to(BF16), normal((T, E), F32, 73).to(DEV)
    weights, ids = router.route(logits, k, scoring="sigmoid", bias=normal((E,), F32, 74, 0.1).to(DEV), groups=4, topk_groups=2)
    got = int8.int8_moe(x, weights, ids, *w13, *w2)
    assert_layer(got, x.cpu(), weights.cpu(), ids.cpu(), w13, w2)
    hexed = hex_moe(x, weights, ids, tiers).float()
    # each 8-bit rounding is off by 1 / (127 sqrt(12)) of its row's largest value, some four times its rms: 1 % of
    # the result for each of x, w13, the activation and w2
    assert float((got.float() - hexed).norm()) <= 0.04 * float(hexed.norm())


# ------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    L, P, odd, off16 = _lib.lib, ctypes.c_void_p(256), ctypes.c_void_p(257), ctypes.c_void_p(264)
    base = dict(x=P, dt=1, ld=32, rows=4, cols=32, q=P, ldq=32, s=P, st=None)
    rows = lambda **a: L.hexmoe_quantize_rows(*{**base, **a}.values())  # noqa: E731
    for bad in (dict(x=None), dict(q=None), dict(s=None), dict(x=odd), dict(s=odd), dict(ld=31), dict(ldq=31), dict(rows=-1), dict(cols=0)):
        assert rows(**bad) == _lib.HEXMOE_E_ARG, bad
    assert rows(dt=3) == _lib.HEXMOE_E_DTYPE and rows(rows=0) == _lib.HEXMOE_OK
    base2 = dict(x=P, dt=3, ldx=32, xs=P, w=P, ldw=32, sw=256, ws=P, rows=4, E=2, n=8, k=32, off=P, odt=0, out=P, ldo=8, outdt=1,
                 work=None, nwork=0, st=None)
    mm = lambda **a: L.hexmoe_grouped_mm_int8(*{**base2, **a}.values())  # noqa: E731
    for bad in (dict(x=None), dict(xs=None), dict(w=None), dict(ws=None), dict(out=None), dict(off=None), dict(x=off16), dict(w=off16),
                dict(ldx=40), dict(ldw=40), dict(sw=200), dict(ldx=16), dict(ldw=16), dict(ldo=7), dict(rows=-1), dict(E=0), dict(E=2049),
                dict(n=0), dict(k=0), dict(k=131072, ldx=131072, ldw=131072), dict(dt=1), dict(dt=1, work=P, nwork=128), dict(off=odd),
                dict(work=off16), dict(rows=2 ** 31), dict(out=odd)):
        assert mm(**bad) == _lib.HEXMOE_E_ARG, bad
    for bad in (dict(dt=4), dict(outdt=3), dict(odt=2)):
        assert mm(**bad) == _lib.HEXMOE_E_DTYPE, bad
    assert mm(rows=0) == _lib.HEXMOE_OK
    need = L.hexmoe_int8_forward_workspace_bytes(4, 2, 2, 32, 16)
    base3 = dict(x=P, dt=1, ldx=32, T=4, H=32, I=16, k=2, tw=P, ids=P, idt=0, E=2, w13=P, ld13=32, st13=1024, s13=P, w2=P, ld2=16, st2=512,
                 s2=P, out=P, outdt=1, work=P, nwork=need, st=None)
    moe = lambda **a: L.hexmoe_int8_forward(*{**base3, **a}.values())  # noqa: E731
    for bad in (dict(x=None), dict(tw=None), dict(ids=None), dict(w13=None), dict(s13=None), dict(w2=None), dict(s2=None), dict(out=None),
                dict(H=40), dict(I=24), dict(H=0), dict(ldx=31), dict(ld13=16), dict(ld2=0), dict(st13=1000), dict(w2=off16), dict(out=off16),
                dict(work=None), dict(nwork=need - 1), dict(work=off16), dict(T=-1), dict(k=0), dict(E=0), dict(T=2 ** 31)):
        assert moe(**bad) == _lib.HEXMOE_E_ARG, bad
    for bad in (dict(dt=3), dict(outdt=2), dict(idt=7)):
        assert moe(**bad) == _lib.HEXMOE_E_DTYPE, bad
    assert moe(T=0) == _lib.HEXMOE_OK and need > 0
    assert L.hexmoe_int8_forward_workspace_bytes(0, 2, 2, 32, 16) == 0


def test_cpu_tensors_are_refused():
    x, w, s = torch.zeros(4, 32), torch.zeros(2, 8, 32, dtype=torch.int8), torch.zeros(2, 8)
    for call in (lambda: int8.quantize_rows(x), lambda: int8.grouped_mm_int8(x, w, s, torch.zeros(3)), lambda: int8.int8_moe(x, x, x, w, s, w, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, off = torch.zeros(4, 32, dtype=BF16, device=DEV), offsets_of([1, 3]).to(DEV)
    w, s = torch.zeros(2, 8, 32, dtype=torch.int8, device=DEV), torch.zeros(2, 8, device=DEV)
    xq, xs = torch.zeros(4, 32, dtype=torch.int8, device=DEV), torch.zeros(4, device=DEV)
    mm = int8.grouped_mm_int8
    bad = [lambda: int8.quantize_rows(xq), lambda: int8.quantize_rows(x.double()), lambda: int8.quantize_rows(x[:, :0]),
           lambda: mm(x, w, s), lambda: mm(x, w[0], s[0], off), lambda: mm(x, w, s[:, :7], off), lambda: mm(x, w.float(), s, off),
           lambda: mm(x, w, s.bfloat16(), off), lambda: mm(x, w, s, off[:2]), lambda: mm(x[:, :31], w, s, off), lambda: mm(x, w, s, off, x_scale=xs),
           lambda: mm(xq, w, s, off), lambda: mm(xq, w, s, off, x_scale=xs[:3]), lambda: mm(xq, w, s, off, x_scale=xs.half()),
           lambda: mm(x, w, s, off, out_dtype=torch.int8), lambda: mm(x, w, s, off, out=torch.zeros(4, 9, dtype=BF16, device=DEV)),
           lambda: mm(x, w.cpu(), s, off), lambda: mm(x, w, s, off.cpu()), lambda: mm(x.double(), w, s, off),
           lambda: mm(x, w, s, off, out_dtype=F32, out=torch.zeros(4, 8, dtype=BF16, device=DEV))]
    tw, ids = torch.zeros(4, 2, device=DEV), torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    w13, s13, w2, s2 = w.new_zeros(2, 32, 32), s.new_zeros(2, 32), w.new_zeros(2, 32, 16), s.new_zeros(2, 32)
    good = dict(x=x, tw=tw, ids=ids, w13=w13, s13=s13, w2=w2, s2=s2)
    moe = lambda **a: (lambda: int8.int8_moe(*{**good, **a}.values()))  # noqa: E731
    bad += [moe(x=x[:, :16]), moe(x=x.double()), moe(tw=tw[:3]), moe(ids=ids[:3]), moe(ids=ids.cpu()), moe(tw=tw.cpu()), moe(w13=w13[:, :30]),
            moe(s13=s13[:1]), moe(w2=w2[:1]), moe(w13=w13.float()), moe(x=x[:, :24], w13=w13[:, :, :24], w2=w2[:, :24], s2=s2[:, :24])]
    moe()()
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was taken")
    for call in (lambda: mm(x.requires_grad_(), w, s, off), lambda: int8.int8_moe(x, tw, ids, w13, s13, w2, s2)):
        with pytest.raises(RuntimeError, match="differentiable"):
            call()
    with torch.no_grad():
        mm(x, w, s, off)


@pytest.mark.gpu
def test_sizes_past_32_bits_are_refused():
    """Views without the memory: none of these sizes may be cut to its low bits, or allocated first."""
    wide = 2 ** 32 + 16
    one = torch.zeros(1, 1, dtype=BF16, device=DEV)
    w, s, off = torch.zeros(1, 1, 1, dtype=torch.int8, device=DEV), torch.zeros(1, 1, device=DEV), offsets_of([1]).to(DEV)
    tw, ids = torch.zeros(1, 1, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    x, w13, s13, w2, s2 = one.expand(1, 16), w.expand(1, 32, 16), s.expand(1, 32), w.expand(1, 16, 16), s.expand(1, 16)
    bad = [lambda: int8.quantize_rows(one.expand(1, wide)), lambda: int8.grouped_mm_int8(one.expand(1, wide), w.expand(1, 1, wide), s, off),
           lambda: int8.grouped_mm_int8(one.expand(1, 131072), w.expand(1, 1, 131072), s, off),
           lambda: int8.grouped_mm_int8(x, w.expand(1, wide, 16), s.expand(1, wide), off),
           lambda: int8.int8_moe(x, tw.expand(1, wide), ids.expand(1, wide), w13, s13, w2, s2),
           lambda: int8.int8_moe(x, tw, ids, w.expand(1, 2 * wide, 16), s.expand(1, 2 * wide), w.expand(1, 16, wide), s2),
           lambda: int8.int8_moe(one.expand(1, wide), tw, ids, w.expand(1, 32, wide), s13, w.expand(1, wide, 16), s.expand(1, wide))]
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was taken")
    assert torch.cuda.max_memory_allocated() <= before + (1 << 20)
