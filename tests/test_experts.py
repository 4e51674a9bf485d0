"""The operators of experts.py (grouped products and their gradients, SwiGLU, gradient clipping,
expert_mlp) against plain 64-bit restatements, and their refusals."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch
from conftest import ROOT

from blackhole_b200 import _lib, experts
from blackhole_b200 import hex_data as hd

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
# half a unit in the last place, relative: the one rounding of a result to its type
ROUND = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 0.0, F16: 2.0 ** -25, F32: 0.0}   # half the smallest f16 subnormal: absolute below the normal range


@pytest.fixture(autouse=True)
def device_word(request):
    yield
    if request.node.get_closest_marker("gpu"):
        from blackhole_b200.hex_moe import device_status
        assert device_status(0) == 0


def offsets_of(sizes, first=0, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]) + first, dtype=dtype)


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def assert_sum(got, want, mass, terms, dtype):
    """got: a sum of `terms` products in fp32 (each addition off by at most 2^-23 of the sum of
    magnitudes, whether it rounds or cuts), rounded once to dtype."""
    got, want, mass = got.double().cpu(), want.double(), mass.double()
    assert got.shape == want.shape
    sums = (terms + 2) * 2.0 ** -23 * mass
    bound = sums + 1.01 * ROUND[dtype] * (want.abs() + sums) + TINY[dtype]
    worst = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert torch.isfinite(got).all() and worst <= 0, f"{float(worst)} over the bound"


def mm_reference(x, w, offsets, transpose, rows):
    out_width = w.shape[2] if transpose else w.shape[1]
    want, mass = torch.zeros(rows, out_width, dtype=torch.float64), torch.zeros(rows, out_width, dtype=torch.float64)
    off = offsets.tolist()
    for e in range(w.shape[0]):
        a, m = x[off[e]:off[e + 1]].double(), w[e].double()
        m = m if transpose else m.t()
        want[off[e]:off[e + 1]], mass[off[e]:off[e + 1]] = a @ m, a.abs() @ m.abs()
    return want, mass


def wgrad_reference(dy, x, offsets):
    off = offsets.tolist()
    E = len(off) - 1
    want = torch.zeros(E, dy.shape[1], x.shape[1], dtype=torch.float64)
    mass = torch.zeros_like(want)
    for e in range(E):
        a, b = dy[off[e]:off[e + 1]].double().t(), x[off[e]:off[e + 1]].double()
        want[e], mass[e] = a @ b, a.abs() @ b.abs()
    return want, mass


# group sizes at which a tile, a block or a walk over the groups can go wrong
SIZES = {
    "one row": [1],
    "none": [0, 0, 0],
    "tile edges": [63, 64, 65, 0, 1, 127, 128, 129],
    "pair edges": [255, 256, 257, 0, 31, 32, 33],
    "empty ends": [0, 0, 5, 0, 16, 0],
    "large": [700, 3],
    "many": [(7 * e) % 5 for e in range(70)],
}
# (N, K): below, at and past tile and step sizes; odd widths leave the 16-byte strides
WIDTHS = [(8, 8), (136, 72), (256, 128), (264, 200), (512, 64), (13, 7), (101, 67)]


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("widths", WIDTHS, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_grouped_mm(sizes, widths, transpose):
    sizes, (n, k) = SIZES[sizes], widths
    dtype = BF16 if (n + k + len(sizes)) % 3 else F16
    rows = sum(sizes)
    x = normal((rows, n if transpose else k), dtype, 1)
    w = normal((len(sizes), n, k), dtype, 2, 0.1)
    off = offsets_of(sizes)
    want, mass = mm_reference(x, w, off, transpose, rows)
    got = experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose)
    assert got.dtype == dtype
    assert_sum(got, want, mass, n if transpose else k, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows", [1, 8, 40, 300])
@pytest.mark.parametrize("widths", [(1536, 2048), (2048, 768), (776, 1032)], ids=str)
def test_grouped_mm_model_widths(widths, rows, transpose):
    """The widths of the 96-expert layer and odd multiples of 8, rows from one token's to several hundred."""
    n, k = widths
    E = 5
    r = np.random.RandomState(rows)
    sizes = np.bincount(r.randint(0, E, rows), minlength=E)
    x, w = normal((rows, n if transpose else k), BF16, 3), normal((E, n, k), BF16, 4, 0.02)
    off = offsets_of(sizes, dtype=torch.int64)
    want, mass = mm_reference(x, w, off, transpose, rows)
    assert_sum(experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose), want, mass,
               n if transpose else k, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("widths", [(72, 264), (9, 11)], ids=str)
def test_grouped_mm_strides_gaps_and_f32(widths, transpose):
    """Rows of no group are zero whatever they hold, groups do not see each other's rows, and every
    operand may be a part of a larger array; f32 output; a stack held transposed."""
    (n, k), sizes = widths, [40, 0, 300, 17]
    E, first, rows = len(sizes), 5, 5 + sum(sizes) + 9
    width = n if transpose else k
    x = torch.full((rows, width + 8), float("nan"), dtype=BF16)
    x[first:first + sum(sizes), :width] = normal((sum(sizes), width), BF16, 5)
    x[first + 40 + 300 + 3] = float("nan")      # one row of the last group
    w = normal((E, n + 3, k + 16), BF16, 6, 0.1)
    off = offsets_of(sizes, first)
    xd, wd = x.to(DEV)[:, :width], w.to(DEV)[:, :n, :k]
    clean = torch.nan_to_num(x[:, :width], nan=0.0)
    want, mass = mm_reference(clean, w[:, :n, :k], off, transpose, rows)
    got = experts.grouped_mm(xd, wd, off.to(DEV), transpose=transpose, out_dtype=F32)
    assert got.dtype == F32
    bad = first + 40 + 300 + 3
    assert got[bad].isnan().all()
    got[bad] = want[bad].float()
    assert not got[:first].any() and not got[first + sum(sizes):].any()
    assert_sum(got, want, mass, width, F32)
    held = wd.transpose(1, 2).contiguous().transpose(1, 2)
    again = experts.grouped_mm(xd, held, off.to(DEV), transpose=transpose)
    again[bad] = 0
    assert_sum(again, torch.where(torch.arange(rows)[:, None] == bad, 0, want), mass, width, BF16)
    into = torch.zeros(rows, want.shape[1] + 3, dtype=BF16, device=DEV)
    assert experts.grouped_mm(xd, wd, off.to(DEV), transpose=transpose, out=into[:, :-3]).data_ptr() == into.data_ptr()
    into[bad] = 0
    assert not into[:, -3:].any() and torch.equal(into[:, :-3], torch.where(
        (torch.arange(rows, device=DEV) == bad)[:, None], 0, got).to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("widths", WIDTHS, ids=str)
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_grouped_wgrad(sizes, widths):
    sizes, (n, k) = SIZES[sizes], widths
    dtype = F16 if (n + k + len(sizes)) % 3 == 0 else BF16
    rows = sum(sizes)
    dy, x, off = normal((rows, n), dtype, 7), normal((rows, k), dtype, 8), offsets_of(sizes)
    want, mass = wgrad_reference(dy, x, off)
    got = experts.grouped_wgrad(dy.to(DEV), x.to(DEV), off.to(DEV))
    assert got.dtype == dtype
    assert_sum(got, want, mass, max(sizes), dtype)
    base = normal((len(sizes), n, k), F32, 9)
    out = base.to(DEV)
    assert experts.grouped_wgrad(dy.to(DEV), x.to(DEV), off.to(DEV), out=out, accumulate=True) is out
    assert_sum(out, want + base.double(), mass + base.double().abs(), max(sizes) + 1, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("widths", [(72, 264), (9, 11)], ids=str)
def test_grouped_wgrad_rows_outside_and_parts(widths):
    """Rows of no group and of other groups never enter a sum, whatever they hold."""
    (n, k), sizes, first = widths, [3, 0, 37, 130, 1], 7
    rows = first + sum(sizes) + 5
    dy = torch.full((rows, n + 8), float("inf"), dtype=F16)
    x = torch.full((rows, k), float("nan"), dtype=F16)
    dy[first:first + sum(sizes), :n] = normal((sum(sizes), n), F16, 10)
    x[first:first + sum(sizes)] = normal((sum(sizes), k), F16, 11)
    off = offsets_of(sizes, first, torch.int64)
    want, mass = wgrad_reference(dy[:, :n], x, off)
    got = experts.grouped_wgrad(dy.to(DEV)[:, :n], x.to(DEV), off.to(DEV), out_dtype=F32)
    assert_sum(got, want, mass, max(sizes), F32)
    x[first + 40:first + 170] = float("nan")      # the fourth group whole: only its gradient follows
    got2 = experts.grouped_wgrad(dy.to(DEV)[:, :n], x.to(DEV), off.to(DEV), out_dtype=F32)
    assert got2[3].isnan().all()
    assert torch.equal(got2[[0, 1, 2, 4]], got[[0, 1, 2, 4]])
    into = torch.zeros(len(sizes), n + 2, k + 5, dtype=F16, device=DEV)
    experts.grouped_wgrad(dy.to(DEV)[:, :n], torch.nan_to_num(x).to(DEV), off.to(DEV), out=into[:, :n, :k])
    assert not into[:, n:].any() and not into[:, :, k:].any()
    assert_sum(into[:3, :n, :k], want[:3], mass[:3], max(sizes), F16)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1000, 2600])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("sizes", ["tile edges", "pair edges", "large"], ids=str)
def test_grouped_mm_of_many_tiles(sizes, transpose, width):
    """More tiles than pairs of SMs at one width of tile or another; what surrounds the groups is not a number."""
    sizes, red, first = SIZES[sizes], 136, 3
    n, k = (red, width) if transpose else (width, red)
    rows = first + sum(sizes) + 2
    x, w = normal((rows, red), BF16, 61), normal((len(sizes), n, k), BF16, 62, 0.1)
    x[:first], x[-2:] = float("nan"), float("inf")
    off = offsets_of(sizes, first)
    want, mass = mm_reference(x, w, off, transpose, rows)
    got = experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose)
    assert not got[:first].any() and not got[-2:].any()
    assert_sum(got, want, mass, red, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [F16, F32], ids=str)
@pytest.mark.parametrize("sizes", ["tile edges", "pair edges", "empty ends"], ids=str)
def test_grouped_wgrad_of_many_tiles(sizes, out_dtype):
    """More tiles than pairs of SMs; each group's neighbours are not numbers when its turn comes."""
    sizes, n, k, first = SIZES[sizes], 520, 584, 5
    rows = first + sum(sizes) + 70
    dy, x = torch.full((rows, n), float("inf"), dtype=F16), torch.full((rows, k), float("nan"), dtype=F16)
    dy[first:first + sum(sizes)], x[first:first + sum(sizes)] = normal((sum(sizes), n), F16, 63), normal((sum(sizes), k), F16, 64)
    off = offsets_of(sizes, first)
    want, mass = wgrad_reference(dy, x, off)
    got = experts.grouped_wgrad(dy.to(DEV), x.to(DEV), off.to(DEV), out_dtype=out_dtype)
    assert_sum(got, want, mass, max(sizes), out_dtype)
    bad = max(range(len(sizes)), key=lambda e: sizes[e])
    x[off[bad]:off[bad + 1]] = float("nan")
    got2 = experts.grouped_wgrad(dy.to(DEV), x.to(DEV), off.to(DEV), out_dtype=out_dtype)
    rest = [e for e in range(len(sizes)) if e != bad]
    assert got2[bad].isnan().all() and torch.equal(got2[rest], got[rest])


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [1096, 1091])
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("n,k", [(72, 1088), (264, 1000), (300, 1091)])
def test_grouped_wgrad_with_x_on_the_wide_side(n, k, out_dtype, ld):
    """A narrow n beside a wide k, in more tiles than pairs: rows of k by TMA and by element, summed, with empty groups."""
    sizes = [3, 0, 65, 200, 16, 1, 130, 0, 64, 9, 17, 33]
    dy, x = normal((sum(sizes) + 2, n), BF16, 65), normal((sum(sizes) + 2, k), BF16, 66)
    dy[-2:], x[-2:] = float("nan"), float("inf")
    off = offsets_of(sizes)
    want, mass = wgrad_reference(dy, x, off)
    out = torch.full((len(sizes), n, ld), 5.0, dtype=out_dtype, device=DEV)
    xd = torch.zeros(sum(sizes) + 2, 1096, dtype=BF16, device=DEV)
    dyd = torch.zeros(sum(sizes) + 2, (n + 7) // 8 * 8, dtype=BF16, device=DEV)
    dyd[:, :n], xd[:, :k] = dy.to(DEV), x.to(DEV)
    experts.grouped_wgrad(dyd[:, :n], xd[:, :k], off.to(DEV), out=out[:, :, :k])
    assert_sum(out[:, :, :k], want, mass, max(sizes), out_dtype)
    assert (out[:, :, k:] == 5).all()
    base = out[:, :, :k].double().cpu()
    experts.grouped_wgrad(dyd[:, :n], xd[:, :k], off.to(DEV), out=out[:, :, :k], accumulate=True)
    assert_sum(out[:, :, :k], want + base, mass + base.abs(), max(sizes) + 1, out_dtype)
    assert (out[:, :, k:] == 5).all()


def padded(t, fill):
    """t as a view into rows that are some elements longer (a multiple of 16 bytes), which hold `fill`."""
    width = t.shape[-1] // 8 * 8 + 8
    buf = torch.full((*t.shape[:-1], width), fill, dtype=t.dtype, device=DEV)
    view = buf[..., :t.shape[-1]]
    view.copy_(t)
    return buf, view


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("E,rows,n,k", [(3, 70, 301, 67), (2, 900, 45, 133), (9, 2000, 1501, 99), (20, 6000, 2100, 77)])
def test_grouped_mm_of_odd_widths_in_padded_rows(E, rows, n, k, transpose):
    """Rows of an odd width, 16-byte strides and not-a-number between them: neither read nor written over."""
    r = np.random.RandomState(E)
    sizes = np.bincount(r.randint(0, E, rows), minlength=E)
    if transpose:
        n, k = k, n
    x, w = normal((rows, n if transpose else k), BF16, 67), normal((E, n, k), BF16, 68, 0.1)
    off = offsets_of(sizes)
    want, mass = mm_reference(x, w, off, transpose, rows)
    buf, out = padded(torch.zeros(rows, k if transpose else n, dtype=BF16), 5.0)
    experts.grouped_mm(padded(x, float("nan"))[1], padded(w, float("nan"))[1], off.to(DEV), transpose=transpose, out=out)
    assert_sum(out, want, mass, n if transpose else k, BF16)
    assert (buf[:, out.shape[1]:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("E,rows,n,k", [(2, 70, 129, 67), (12, 700, 301, 355), (40, 1500, 77, 499), (1, 5000, 97, 131)])
def test_grouped_wgrad_of_odd_widths_in_padded_rows(E, rows, n, k, out_dtype):
    """The same of gradients: what stands between the rows of a view is nobody's."""
    r = np.random.RandomState(E)
    sizes = np.bincount(r.randint(0, E, rows), minlength=E)
    dy, x, off = normal((rows, n), BF16, 69), normal((rows, k), BF16, 70), offsets_of(sizes)
    want, mass = wgrad_reference(dy, x, off)
    buf, out = padded(torch.zeros(E, n, k, dtype=out_dtype), 5.0)
    ins = padded(dy, float("nan"))[1], padded(x, float("nan"))[1]
    experts.grouped_wgrad(*ins, off.to(DEV), out=out)
    assert_sum(out, want, mass, max(sizes), out_dtype)
    assert (buf[..., k:] == 5).all()
    experts.grouped_wgrad(*ins, off.to(DEV), out=out, accumulate=True)
    assert (buf[..., k:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("n,k", [(200, 2056), (2056, 200), (1000, 1048)])
def test_grouped_mm_long_reduction_of_few_tiles(n, k, transpose, out_dtype):
    """Few tiles share the reduction (a workspace is asked for); rows before and after the groups stay zero."""
    sizes, first, rows = [70, 0, 1], 3, 80
    width = n if transpose else k
    if width >= 2000:
        assert _lib.lib.hexmoe_grouped_mm_workspace_bytes(rows, 3, n, k, transpose) > 0
    x, w = normal((rows, width), BF16, 25), normal((3, n, k), BF16, 26, 0.05)
    off = offsets_of(sizes, first)
    want, mass = mm_reference(x, w, off, transpose, rows)
    got = experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose, out_dtype=out_dtype)
    assert not got[:first].any() and not got[first + 71:].any()
    assert_sum(got, want, mass, width, out_dtype)
    assert torch.equal(got, experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose, out_dtype=out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("sizes", [[5000], [4000, 0, 3], [2111, 2050]], ids=str)
def test_grouped_wgrad_long_reduction_of_few_tiles(sizes, out_dtype):
    """One group's rows shared by several runs, groups shorter than the runs are many, sums added to out."""
    E, n, k = len(sizes), 72, 130
    assert _lib.lib.hexmoe_grouped_wgrad_workspace_bytes(sum(sizes), E, n, k) > 0
    dy, x = normal((sum(sizes), n), BF16, 27), normal((sum(sizes), k + 6), BF16, 28)
    off = offsets_of(sizes)
    want, mass = wgrad_reference(dy, x[:, :k], off)
    xd = x.to(DEV)[:, :k]
    assert_sum(experts.grouped_wgrad(dy.to(DEV), xd, off.to(DEV), out_dtype=out_dtype), want, mass, max(sizes), out_dtype)
    base = normal((E, n, k), out_dtype, 29)
    out = experts.grouped_wgrad(dy.to(DEV), xd, off.to(DEV), out=base.to(DEV), accumulate=True)
    assert_sum(out, want + base.double(), mass + base.double().abs(), max(sizes) + 1, out_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("sizes", [[1], [0, 3, 0, 1], [32], [9, 17, 6], [1] * 20, [0] * 40 + [8] + [0] * 30 + [16]], ids=str)
def test_grouped_mm_few_rows(sizes, transpose):
    """A decode step's rows, past one pass over a matrix, with gaps on both sides; fp16; widths off the block sizes."""
    n, k, first = 200, 1352, 32 - sum(sizes) if sum(sizes) > 30 else 1
    rows = min(32, first + sum(sizes) + 1)
    width = n if transpose else k
    x, w = normal((rows, width), F16, 38), normal((len(sizes), n, k), F16, 39, 0.1)
    x[:first] = float("nan")
    off = offsets_of(sizes, first)
    want, mass = mm_reference(x, w, off, transpose, rows)
    for out_dtype in (F16, F32):
        got = experts.grouped_mm(x.to(DEV), w.to(DEV), off.to(DEV), transpose=transpose, out_dtype=out_dtype)
        assert_sum(got, want, mass, width, out_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
def test_grouped_mm_uneven_groups_of_a_training_step(transpose):
    """Mean group sizes between 257 and 512, groups far from the mean: tiles of two accumulators, the
    last of a group ending within the first (1, 256), at its end and just past it."""
    E, n, k = 80, 264, 72     # two 256-row M sides an expert: enough tiles to fill the machine
    if transpose:
        n, k = k, n
    sizes = [4097, 4096, 513, 512, 511, 257, 256, 255, 1, 0, 769, 1025, 1024, 300, 2049, 641] + [205] * 64
    assert 256 * E < sum(sizes) <= 512 * E
    rows, width = sum(sizes), n if transpose else k
    g = torch.Generator(device=DEV).manual_seed(82)
    x = torch.randn(rows, width, generator=g, device=DEV).to(BF16)
    w = torch.randn(E, n, k, generator=g, device=DEV).mul(0.1).to(BF16)
    off = offsets_of(sizes)
    got = experts.grouped_mm(x, w, off.to(DEV), transpose=transpose)
    xd, wd, at = x.double(), w.double(), off.tolist()
    want, mass = torch.zeros_like(got, dtype=torch.float64), torch.zeros_like(got, dtype=torch.float64)
    for e in range(E):
        r, m = slice(at[e], at[e + 1]), wd[e] if transpose else wd[e].t()
        want[r], mass[r] = xd[r] @ m, xd[r].abs() @ m.abs()
    assert_sum(got, want.cpu(), mass.cpu(), width, BF16)


@pytest.mark.gpu
def test_grouped_products_repeat_bit_for_bit():
    sizes = [0, 300, 41, 5, 600]
    off = offsets_of(sizes).to(DEV)
    x, dy, w = normal((sum(sizes), 256), BF16, 12).to(DEV), normal((sum(sizes), 520), BF16, 13).to(DEV), normal((5, 520, 256), BF16, 14).to(DEV)
    for f in (lambda: experts.grouped_mm(x, w, off), lambda: experts.grouped_mm(dy, w, off, transpose=True),
              lambda: experts.grouped_wgrad(dy, x, off, out_dtype=F32), lambda: experts.grouped_mm(x[:8], w, off.clamp(max=8))):
        first = f()
        assert all(torch.equal(first, f()) for _ in range(3))


@pytest.mark.gpu
def test_grouped_mm_in_a_graph_follows_its_offsets():
    """A captured product reads offsets and rows anew at every replay (no size is kept on the host)."""
    E, n, k, rows = 4, 264, 128, 200
    w = normal((E, n, k), BF16, 15, 0.1)
    x, off = normal((rows, k), BF16, 16), offsets_of([50, 50, 50, 50])
    xd, wd, offd = x.to(DEV), w.to(DEV), off.to(DEV)
    experts.grouped_mm(xd, wd, offd)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        got = experts.grouped_mm(xd, wd, offd)
        dw = experts.grouped_wgrad(got, xd, offd, out_dtype=F32)
    for sizes in ([0, 200, 0, 0], [3, 100, 90, 1]):
        new = offsets_of(sizes)
        offd.copy_(new)
        graph.replay()
        want, mass = mm_reference(x, w, new, False, rows)
        assert_sum(got, want, mass, k, BF16)
        want, mass = wgrad_reference(got.cpu(), x, new)
        assert_sum(dw, want, mass, max(sizes), F32)


@pytest.mark.gpu
def test_offsets_that_do_not_fit_are_clamped_and_reported():
    from blackhole_b200.hex_moe import device_status
    x, w = normal((32, 64), BF16, 17).to(DEV), normal((3, 72, 64), BF16, 18).to(DEV)
    for off in ([0, 20, 10, 32], [0, 8, 16, 40], [-4, 8, 16, 32], [0, 2 ** 40, 7, 9]):
        off = torch.tensor(off)
        got = experts.grouped_mm(x, w, off.to(DEV))
        assert device_status(0) == 8
        experts.grouped_wgrad(x, x, off.to(DEV))
        assert device_status(0) == 8
        fixed = torch.cummax(off.clamp(0, 32), 0).values
        assert torch.equal(got, experts.grouped_mm(x, w, fixed.to(DEV)))


@pytest.mark.gpu
def test_grouped_mm_past_2_to_the_31_values():
    """Row offsets and output offsets that pass 32 bits: sampled rows of 1.1 million x 2048."""
    rows, n, k = 1_100_000, 2048, 64
    sizes = [300_000, 0, 500_001, rows - 800_001]
    off = offsets_of(sizes)
    g = torch.Generator(device=DEV).manual_seed(19)
    x = torch.randn(rows, k, generator=g, device=DEV).to(BF16)
    w = torch.randn(4, n, k, generator=g, device=DEV).mul(0.1).to(BF16)
    got = experts.grouped_mm(x, w, off.to(DEV))
    pick = torch.tensor([0, 299_999, 300_000, 800_000, 800_001, 1_048_575, 1_048_576, rows - 1])
    expert = torch.tensor([0, 0, 2, 2, 3, 3, 3, 3])
    xs, ws = x[pick].double().cpu(), w.double().cpu()[expert]
    assert_sum(got[pick], torch.einsum("rk,rnk->rn", xs, ws), torch.einsum("rk,rnk->rn", xs.abs(), ws.abs()), k, BF16)
    back = experts.grouped_mm(got, w, off.to(DEV), transpose=True)   # and as an operand
    gs = got[pick].double().cpu()
    assert_sum(back[pick], torch.einsum("rn,rnk->rk", gs, ws), torch.einsum("rn,rnk->rk", gs.abs(), ws.abs()), n, BF16)


@pytest.mark.gpu
def test_grouped_mm_difference_is_its_gradient():
    """The products are linear: differences of the f32 forward along a step equal the transpose
    product and the weight gradient, up to the f32 sums."""
    sizes, n, k = [33, 0, 150], 136, 72
    off = offsets_of(sizes)
    x, w, dy = normal((183, k), BF16, 20), normal((3, n, k), BF16, 21), normal((183, n), BF16, 22)
    sx, sw = normal((183, k), BF16, 23), normal((3, n, k), BF16, 24)
    f = lambda a, b: experts.grouped_mm(a.to(DEV), b.to(DEV), off.to(DEV), out_dtype=F32).double().cpu()  # noqa: E731
    dx = experts.grouped_mm(dy.to(DEV), w.to(DEV), off.to(DEV), transpose=True, out_dtype=F32).double().cpu()
    dw = experts.grouped_wgrad(dy.to(DEV), x.to(DEV), off.to(DEV), out_dtype=F32).double().cpu()
    # the steps are exact in bf16 arithmetic only one operand at a time: f is linear in each
    lhs_x, lhs_w = (f(sx, w) * dy.double()).sum(), (f(x, sw) * dy.double()).sum()
    mass_x = (mm_reference(sx, w, off, False, 183)[1] * dy.double().abs()).sum()
    mass_w = (mm_reference(x, sw, off, False, 183)[1] * dy.double().abs()).sum()
    assert abs(lhs_x - (dx * sx.double()).sum()) <= (n + k + 4) * 2.0 ** -23 * mass_x
    assert abs(lhs_w - (dw * sw.double()).sum()) <= (150 + k + 4) * 2.0 ** -23 * mass_w


# ------------------------------------------------------------------ SwiGLU
def swiglu_reference(h, weight, dact=None):
    h = h.double()
    gate, up = h.chunk(2, 1)
    w = torch.ones(h.shape[0], dtype=torch.float64) if weight is None else weight.double()
    sig = torch.sigmoid(gate)
    silu = gate * sig
    if dact is None:
        return w[:, None] * silu * up
    d = dact.double()
    dgate = w[:, None] * d * up * (sig + silu * (1 - sig))
    return torch.cat([dgate, w[:, None] * d * silu], 1), (d * silu * up).sum(1), (d * silu * up).abs().sum(1), \
        w[:, None].abs() * d.abs() * up.abs() * (sig + silu.abs() * (1 - sig))


# fp32 evaluation: the exponential, the divide and a handful of products, each within 2^-21 relative
# (CUDA's fast exponential errs by 2 + 1.16 |x| units of its result, |x| below 16 here)
EVAL = 32 * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (1, 768), (3, 8), (5, 33), (7, 96), (9, 200), (31, 517), (300, 768), (2, 5000),
                                   (8200, 104)], ids=str)
def test_swiglu(shape, dtype, weights):
    rows, inter = shape
    h, dact = normal((rows, 2 * inter), dtype, 30, 2.0), normal((rows, inter), dtype, 31)
    weight = normal((rows,), F32, 32) if weights else None
    wd = None if weight is None else weight.to(DEV)
    act = experts.swiglu(h.to(DEV), wd)
    want = swiglu_reference(h, weight)
    assert ((act.double().cpu() - want).abs() <= (EVAL + 1.01 * ROUND[dtype]) * want.abs() + TINY[dtype]).all()
    dh, dw = experts.swiglu_backward(dact.to(DEV), h.to(DEV), wd)
    want, want_dw, mass_dw, mass_gate = swiglu_reference(h, weight, dact)
    # s + silu (1 - s) cancels for negative gates: its error goes by the two terms, not by their sum
    slack = torch.cat([mass_gate, want[:, inter:].abs()], 1)
    assert ((dh.double().cpu() - want).abs() <= EVAL * slack + 1.01 * ROUND[dtype] * want.abs() + TINY[dtype]).all()
    if weights:
        assert ((dw.double().cpu() - want_dw).abs() <= (EVAL + (inter + 2) * 2.0 ** -24) * mass_dw).all()
    else:
        assert dw is None


@pytest.mark.gpu
def test_swiglu_extremes_strides_and_in_place():
    """Gates far out on both sides, weights of zero, rows cut from a wider array, dh over h itself."""
    gate = torch.tensor([0.0, -0.0, 1e-30, 88.0, 200.0, -88.0, -104.0, -200.0, 3e38, -3e38])
    h = torch.stack([torch.cat([gate, torch.full((10,), 2.0)])] * 3)
    weight = torch.tensor([1.0, 0.0, -0.5])
    act = experts.swiglu(h.to(DEV), weight.to(DEV)).cpu()
    want = swiglu_reference(h, weight)
    assert torch.allclose(act.double(), want.clamp(-3.4028e38, 3.4028e38), rtol=EVAL * 8, atol=1e-35) or act[0, 8] == math.inf
    assert not act[1].any() and act[0, 8] == math.inf and not act[0, 5:8].abs().gt(1e-30).any()
    wide = normal((40, 2 * 96 + 16), BF16, 33)
    hd_, dact = wide.to(DEV)[:, :192], normal((40, 96), BF16, 34).to(DEV)
    plain = hd_.contiguous()
    assert torch.equal(experts.swiglu(hd_), experts.swiglu(plain))
    want_dh, _ = experts.swiglu_backward(dact, plain)
    dh, _ = experts.swiglu_backward(dact, plain, out=plain)
    assert dh.data_ptr() == plain.data_ptr() and torch.equal(plain, want_dh)
    assert experts.swiglu(hd_[:0]).shape == (0, 96)


@pytest.mark.gpu
def test_swiglu_gradient_against_differences():
    """f32 kernel gradient against central differences of the 64-bit formula."""
    h, dact, weight = normal((6, 2 * 20), F32, 35), normal((6, 20), F32, 36), normal((6,), F32, 37)
    dh, dw = experts.swiglu_backward(dact.to(DEV), h.to(DEV), weight.to(DEV))
    loss = lambda a, w: float((swiglu_reference(a, w) * dact.double()).sum())  # noqa: E731
    step = 1e-5
    for i, j in [(0, 0), (1, 7), (3, 19), (0, 20), (5, 39), (2, 25)]:
        d = torch.zeros(6, 40, dtype=torch.float64)
        d[i, j] = step
        slope = (loss(h.double() + d, weight.double()) - loss(h.double() - d, weight.double())) / (2 * step)
        # step^2 times a third derivative below 4, and 1e-16 of the loss (below 1e3) over the step
        assert abs(slope - float(dh[i, j])) <= 4 * step ** 2 * 10 + 1e-16 * 1e3 / step + EVAL * 20
    for i in range(6):
        d = torch.zeros(6, dtype=torch.float64)
        d[i] = step
        slope = (loss(h, weight.double() + d) - loss(h, weight.double() - d)) / (2 * step)
        assert abs(slope - float(dw[i])) <= 1e-16 * 1e3 / step + EVAL * 100


# ------------------------------------------------------------------ clipping
def clip_reference(grads, max_norm, norm_type):
    flat = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(0, dtype=torch.float64)
    norm = flat.square().sum().sqrt() if norm_type == 2 else flat.abs().max() if flat.numel() else torch.tensor(0.0)
    return float(norm), min(1.0, max_norm / (float(norm) + 1e-6))


def assert_clipped(got, grads, scale):
    for o, g in zip(got, grads):
        want = g.double() * scale
        # the factor: the norm's f32 rounding, the sum and the divide (4 units); then the product's own rounding
        assert ((o.double().cpu() - want).abs() <= (8 * 2.0 ** -24 + 1.01 * ROUND[o.dtype]) * want.abs()
                + max(TINY[o.dtype], 2.0 ** -149)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0, math.inf])
@pytest.mark.parametrize("counts", [[1], [0, 5, 0], [8191, 8192, 8193, 1], [3, 100_003, 16, 64_000], list(range(1, 90))], ids=["1", "empty", "chunks", "mixed", "many"])
def test_clip_grad_norm(counts, max_norm, norm_type):
    types = [F32, BF16, F16]
    grads = [normal((c,), types[i % 3], 40 + i) for i, c in enumerate(counts)]
    norm, scale = clip_reference(grads, max_norm if max_norm != math.inf else 1e300, norm_type)
    on = [g.to(DEV) for g in grads]
    out = [torch.full_like(g, 7.0) for g in on]
    got = experts.clip_grad_norm(on, max_norm, norm_type, out=out)
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - norm) <= 2.0 ** -22 * norm   # squares summed in f32 by eights, then in 64 bits
    assert all(torch.equal(a.cpu(), b) for a, b in zip(on, grads))
    assert_clipped(out, grads, scale)
    assert torch.equal(experts.clip_grad_norm(on, max_norm, norm_type), got)   # in place
    assert all(torch.equal(a, b) for a, b in zip(on, out))


@pytest.mark.gpu
def test_clip_grad_norm_magnitudes_and_non_finite():
    """Values whose squares leave the f32 range on either side; infinities and NaN."""
    for scale in (1e30, 1e-30, 3e-42):
        g = normal((5000,), F32, 50, scale)
        want = float(g.double().square().sum().sqrt())
        assert abs(float(experts.clip_grad_norm(g.to(DEV), 1e38)) - want) <= 2.0 ** -22 * want + 2.0 ** -149
    assert float(experts.clip_grad_norm(torch.zeros(100, device=DEV), 1.0)) == 0.0
    for value, norm_type in [(math.inf, 2.0), (-math.inf, math.inf), (math.nan, 2.0), (math.nan, math.inf)]:
        g = normal((20_000,), BF16, 51).to(DEV)
        g[12_345] = value
        before = g.clone()
        norm = float(experts.clip_grad_norm([g], 1.0, norm_type))
        if math.isnan(value):
            assert math.isnan(norm) and g.isnan().all()
        else:
            assert norm == math.inf and g[12_345].isnan() and int(g.count_nonzero()) == 1
        torch.testing.assert_close(experts.clip_grad_norm(before.nan_to_num(1.0, 1.0, 1.0), math.inf).isfinite().item(), True)


@pytest.mark.gpu
def test_clip_grad_norm_views_and_types():
    """Parts of flat buffers at every alignment, transposed and sliced tensors, copies to other types,
    more tensors than one launch's list."""
    flat = normal((4000,), BF16, 52).to(DEV)
    cuts, at = [], 0
    for size in (1, 2, 7, 16, 129, 1000, 3, 800):
        cuts.append(flat[at:at + size])
        at += size
    keep = flat.clone()
    norm, scale = clip_reference([c.cpu() for c in cuts], 1.0, 2)
    assert abs(float(experts.clip_grad_norm(cuts, 1.0)) - norm) <= 2.0 ** -22 * norm
    assert_clipped([flat[:at]], [keep[:at].cpu()], scale)
    assert torch.equal(flat[at:], keep[at:])
    big = normal((6, 10, 12), F32, 53)
    d = big.to(DEV)
    views = [d[:2].transpose(1, 2), d[2:4, :, 3:7], d[4:, ::2, ::3]]
    parts = [big[:2], big[2:4, :, 3:7], big[4:, ::2, ::3]]
    norm, scale = clip_reference(parts, 2.0, 2)
    assert abs(float(experts.clip_grad_norm(views, 2.0)) - norm) <= 2.0 ** -22 * norm
    assert_clipped([d[:2], d[2:4, :, 3:7], d[4:, ::2, ::3]], parts, scale)
    assert torch.equal(d.cpu()[2:4, :, :3], big[2:4, :, :3]) and torch.equal(d.cpu()[4:, 1::2], big[4:, 1::2])
    grads = [normal((c,), t, 54 + c) for t in (F32, BF16, F16) for c in (5, 999, 20_000)]
    norm, scale = clip_reference(grads, 3.0, 2)
    for dtype in (F32, BF16, F16):
        for shift in (0, 1):
            out = [torch.zeros(g.numel() + shift, dtype=dtype, device=DEV)[shift:] for g in grads]
            experts.clip_grad_norm([g.to(DEV) for g in grads], 3.0, out=out)
            assert_clipped(out, grads, scale)
    many = [normal((1 + i % 7,), F32, i).to(DEV) for i in range(2100)]
    host = [m.cpu() for m in many]
    norm, scale = clip_reference(host, 1.0, 2)
    assert abs(float(experts.clip_grad_norm(many, 1.0)) - norm) <= 2.0 ** -22 * norm
    assert_clipped(many, host, scale)


# ------------------------------------------------------------------ the layer
def layer_reference(x, weights, ids, w13, w2, dout):
    """Output and gradients in 64 bits from the formulas, expert by expert; and the norm of the terms that
    the gradients of the routing weights are sums of."""
    x, weights, w13, w2 = (t.double().requires_grad_() for t in (x, weights, w13, w2))
    out = torch.zeros(x.shape[0], x.shape[1], dtype=torch.float64)
    inter, terms = w2.shape[2], 0.0
    for e in range(w13.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if len(t):
            h = x[t] @ w13[e].t()
            act = torch.nn.functional.silu(h[:, :inter]) * h[:, inter:]
            terms += float((act * (dout[t].double() @ w2[e])).square().sum())
            out = out.index_add(0, t, act * weights[t, j][:, None] @ w2[e].t())
    out.backward(dout.double())
    return out.detach(), x.grad, weights.grad, w13.grad, w2.grad, terms ** 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,E,k,H,I", [(1, 4, 2, 64, 32), (37, 6, 3, 128, 96), (200, 12, 4, 256, 200)])
def test_expert_mlp(tokens, E, k, H, I):
    weights, ids = hd.synth_routing(tokens, E, k, seed=60)
    ids[ids == 1] = 0                             # an expert without rows, one reached twice by a token
    x, dout = normal((tokens, H), BF16, 61), normal((tokens, H), BF16, 62)
    w13, w2 = normal((E, 2 * I, H), BF16, 63, H ** -0.5), normal((E, H, I), BF16, 64, I ** -0.5)
    leaves = [t.to(DEV).requires_grad_() for t in (x, weights.float(), w13, w2)]
    out = experts.expert_mlp(leaves[0], leaves[1], ids.to(DEV), leaves[2], leaves[3])
    out.backward(dout.to(DEV))
    want = layer_reference(x, weights.float(), ids, w13, w2, dout)
    # every result passes at most five bf16 roundings (2^-9 each, in norm); a gradient of a routing weight is
    # a sum of rounded terms that may cancel: its error goes by their norm
    for i, (got, w) in enumerate(zip([out.detach()] + [t.grad for t in leaves], want)):
        size = want[5] if i == 2 else float(w.norm())
        assert float((got.double().cpu() - w).norm()) <= 5 * 2.0 ** -9 * size
    assert not leaves[2].grad[1].any() and not leaves[3].grad[1].any()
    # differences of the 64-bit loss along a step of all four inputs
    steps = [normal(tuple(t.shape), F32, 65 + i, 0.1).double() for i, t in enumerate((x, weights, w13, w2))]
    loss = lambda s: float((layer_reference(*(a.double() + s * b for a, b in ((x, steps[0]), (weights.float(), steps[1]))), ids,  # noqa: E731
                                            *(a.double() + s * b for a, b in ((w13, steps[2]), (w2, steps[3]))), dout)[0] * dout.double()).sum())
    slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
    mine = sum(float((t.grad.double().cpu() * s).sum()) for t, s in zip(leaves, steps))
    size = sum(float(w.norm() * s.norm()) for w, s in zip(want[1:5], steps))
    assert abs(slope - mine) <= 5 * 2.0 ** -9 * size


@pytest.mark.gpu
def test_expert_mlp_without_tokens_and_with_bad_ids():
    """No tokens; ids of no expert: they add nothing, have no gradient, and set the device error word."""
    from blackhole_b200.hex_moe import device_status
    w13, w2 = normal((4, 64, 32), BF16, 73).to(DEV).requires_grad_(), normal((4, 32, 32), BF16, 74).to(DEV).requires_grad_()
    out = experts.expert_mlp(torch.zeros(0, 32, dtype=BF16, device=DEV), torch.zeros(0, 2, device=DEV),
                             torch.zeros(0, 2, dtype=torch.int64, device=DEV), w13, w2)
    out.sum().backward()
    assert out.shape == (0, 32) and not w13.grad.any() and not w2.grad.any()
    x, weights = normal((5, 32), BF16, 75).to(DEV).requires_grad_(), torch.rand(5, 2, device=DEV).requires_grad_()
    ids = torch.tensor([[0, 1], [2, -1], [4, 3], [3, 0], [9, -7]], device=DEV)
    out = experts.expert_mlp(x, weights, ids, w13, w2)
    out.backward(torch.ones_like(out).expand_as(out))
    assert device_status(0) & 2
    good = (ids >= 0) & (ids < 4)
    assert not weights.grad[~good].any() and weights.grad[good].all() and not out[4].any() and not x.grad[4].any()
    same = experts.expert_mlp(x, torch.where(good, weights, 0), ids.clamp(0, 3), w13, w2)
    assert torch.equal(same, out)


@pytest.mark.gpu
def test_ordinary_calls_and_the_checked_ones_agree():
    """What _call takes and what goes through Python's checks is the same call: an `out` sends it there."""
    off = offsets_of([40, 0, 88]).to(DEV)
    x, w, dy = normal((128, 72), BF16, 76).to(DEV), normal((3, 136, 72), BF16, 77).to(DEV), normal((128, 136), BF16, 78).to(DEV)
    out = torch.empty(128, 136, dtype=BF16, device=DEV)
    assert torch.equal(experts.grouped_mm(x, w, off), experts.grouped_mm(x, w, off, out=out))
    dw = torch.empty(3, 136, 72, device=DEV)
    assert torch.equal(experts.grouped_wgrad(dy, x, off, out_dtype=F32), experts.grouped_wgrad(dy, x, off, out=dw))
    weight, dact = torch.rand(128, device=DEV), dy[:, :68].contiguous()
    dh, dweight = experts.swiglu_backward(dact, dy, weight)
    again, dweight2 = experts.swiglu_backward(dact, dy, weight, out=torch.empty_like(dy))
    assert torch.equal(dh, again) and torch.equal(dweight, dweight2)
    strided = torch.randn(256, device=DEV)[::2]
    assert torch.equal(experts.swiglu(dy, strided), experts.swiglu(dy, strided.contiguous()))
    a, b = torch.randn(50, device=DEV), torch.randn(7, 9, device=DEV)
    want = experts.clip_grad_norm([a.clone(), b.clone()], 1.0)
    got = experts.clip_grad_norm([a, b.t().contiguous().t()], 1.0)
    assert abs(float(want) - float(got)) <= 2.0 ** -22 * float(want)


@pytest.mark.gpu
def test_expert_mlp_equals_hex_moe_on_dequantized_stacks():
    """On the stacks that dequant_all makes, the training layer and the HEX layer agree to the layer's tolerance."""
    from blackhole_b200.hex_moe import HexTier, dequant_all, hex_moe
    E, H, I, k, T = 8, 256, 128, 2, 50
    L = hd.synth_layer(E, H, I, "mixed", 32, seed=70, device=DEV)
    tiers = [HexTier(t["bits"], t["experts"], t["gate_proj"], t["up_proj"], t["down_proj"]).prepare(E) for t in L.tiers]
    w, ids = hd.synth_routing(T, E, k, seed=71)
    x = hd.synth_x(T, H, seed=72, device=DEV).to(BF16)
    want = hex_moe(x, w.to(DEV), ids.to(DEV), tiers).float()
    got = experts.expert_mlp(x, w.to(DEV), ids.to(DEV), *dequant_all(tiers)).float()
    assert ((got - want).abs() <= 1e-2 + 2e-2 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("block_m", [1, 16])
def test_group_offsets(block_m):
    from blackhole_b200.hex_moe import align
    E = 300
    ids = torch.tensor(np.random.RandomState(3).randint(0, E, 700) // 3 * 3, device=DEV)
    _, eid, npp = align(ids, E, block_m)
    off = torch.full((E + 1,), -5, dtype=torch.int32, device=DEV)
    _lib.check(_lib.lib.hexmoe_group_offsets(eid.data_ptr(), eid.numel(), npp.data_ptr(), block_m, E, off.data_ptr(),
                                             torch.cuda.current_stream().cuda_stream))
    counts = torch.bincount(ids.cpu(), minlength=E)
    want = torch.cat([torch.zeros(1, dtype=torch.long), ((counts + block_m - 1) // block_m * block_m).cumsum(0)])
    assert off.cpu().tolist() == want.tolist()


@pytest.mark.gpu
def test_operators_on_another_stream():
    """Calls follow the current stream: a side stream's results are ready after that stream alone."""
    off = offsets_of([100, 28]).to(DEV)
    x, w = normal((128, 64), BF16, 80).to(DEV), normal((2, 72, 64), BF16, 81).to(DEV)
    want = experts.grouped_mm(x, w, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = x * 1
        got = experts.grouped_mm(held, w, off)
        norm = experts.clip_grad_norm([got], 1.0)
        side.synchronize()
        assert float(norm) > 1.0 and float(got.float().norm()) < 1.01
    side.synchronize()
    assert abs(float(want.float().norm()) - float(norm)) <= 2.0 ** -20 * float(norm)


@pytest.mark.gpu
def test_healing_example():
    """The operators together: what training and the Hessians are for shows on held-out rows."""
    import importlib.util
    spec = importlib.util.spec_from_file_location("heal_experts", ROOT / "examples" / "heal_experts.py")
    heal = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(heal)
    got = heal.main(steps=80)
    assert got["pruned and healed"] < got["pruned"]
    assert got["pruned, healed and quantized"] < got["pruned and quantized"] < got["pruned and quantized to the nearest level"]


# ------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    L, P = _lib.lib, ctypes.c_void_p(256)
    odd = ctypes.c_void_p(257)
    mm = lambda **a: L.hexmoe_grouped_mm(*{**dict(x=P, ldx=8, w=P, ldw=8, sw=64, dt=1, rows=4, E=2, n=8, k=8, tr=0, off=P,  # noqa: E731
                                                  odt=0, out=P, ldo=8, outdt=1, ws=None, nws=0, st=None), **a}.values())
    for bad in (dict(n=0), dict(k=-1), dict(rows=-1), dict(E=0), dict(E=2049), dict(ldx=7), dict(ldw=7), dict(ldo=7),
                dict(x=None), dict(w=None), dict(out=None), dict(off=None), dict(x=odd), dict(off=odd), dict(rows=2 ** 31)):
        assert mm(**bad) == _lib.HEXMOE_E_ARG, bad
    for bad in (dict(dt=0), dict(dt=7), dict(outdt=2), dict(odt=5)):
        assert mm(**bad) == _lib.HEXMOE_E_DTYPE, bad
    assert mm(rows=0) == _lib.HEXMOE_OK
    wg = lambda **a: L.hexmoe_grouped_wgrad(*{**dict(dy=P, lddy=8, x=P, ldx=8, dt=1, rows=4, E=2, n=8, k=8, off=P, odt=0,  # noqa: E731
                                                     out=P, ldo=8, so=64, outdt=1, acc=0, ws=None, nws=0, st=None), **a}.values())
    for bad in (dict(n=0), dict(rows=-1), dict(E=0), dict(lddy=7), dict(ldx=7), dict(ldo=7), dict(so=63), dict(out=None),
                dict(dy=None), dict(off=None), dict(out=odd)):
        assert wg(**bad) == _lib.HEXMOE_E_ARG, bad
    assert wg(dt=0) == _lib.HEXMOE_E_DTYPE and wg(outdt=2) == _lib.HEXMOE_E_DTYPE
    assert L.hexmoe_swiglu(P, 1, 4, 0, 8, None, P, 8, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_swiglu(P, 1, 4, 8, 15, None, P, 8, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_swiglu(P, 4, 4, 8, 16, None, P, 8, None) == _lib.HEXMOE_E_DTYPE
    assert L.hexmoe_swiglu(None, 1, 4, 8, 16, None, P, 8, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_swiglu(odd, 1, 4, 8, 16, None, P, 8, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_swiglu(None, 1, 0, 8, 16, None, None, 8, None) == _lib.HEXMOE_OK
    assert L.hexmoe_swiglu_backward(P, 7, P, 16, 1, 4, 8, None, P, 16, None, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_swiglu_backward(None, 8, P, 16, 1, 4, 8, None, P, 16, None, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_group_offsets(P, 4, None, 1, 8, P, None) == _lib.HEXMOE_E_ARG
    assert L.hexmoe_group_offsets(P, 4, P, 0, 8, P, None) == _lib.HEXMOE_E_ARG
    one = lambda v, t: (t * 1)(v)  # noqa: E731
    need = L.hexmoe_clip_grad_norm_workspace_bytes(1)
    clip = lambda max_norm=1.0, ws=P, nbytes=need, norm=P, ptr=256, count=8, dt=0: L.hexmoe_clip_grad_norm(  # noqa: E731
        1, one(ptr, ctypes.c_void_p), one(count, ctypes.c_int64), one(dt, ctypes.c_int32), None, None, max_norm, 0, norm,
        ws, nbytes, None)
    for bad in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(ws=None), dict(nbytes=need - 1), dict(norm=None)):
        assert clip(**bad) == _lib.HEXMOE_E_ARG, bad
    assert need > 0 and L.hexmoe_clip_grad_norm_workspace_bytes(-1) == 0


def test_cpu_tensors_and_types_are_refused():
    x, w, off = torch.zeros(4, 8, dtype=BF16), torch.zeros(2, 16, 8, dtype=BF16), offsets_of([1, 3])
    for call in (lambda: experts.grouped_mm(x, w, off), lambda: experts.grouped_wgrad(x, x, off),
                 lambda: experts.swiglu(x), lambda: experts.swiglu_backward(x, x), lambda: experts.clip_grad_norm([x], 1.0),
                 lambda: experts.expert_mlp(x, x, x, w, w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for bad in (dict(max_norm=-1.0), dict(max_norm=math.nan), dict(max_norm=1.0, norm_type=1.0)):
        with pytest.raises(ValueError):
            experts.clip_grad_norm([x], **bad)
    with pytest.raises(ValueError, match="no gradients"):
        experts.clip_grad_norm([None], 1.0)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w = torch.zeros(4, 8, dtype=BF16, device=DEV), torch.zeros(2, 16, 8, dtype=BF16, device=DEV)
    off = offsets_of([1, 3]).to(DEV)
    bad = [lambda: experts.grouped_mm(x, w[0], off), lambda: experts.grouped_mm(x[0], w, off),
           lambda: experts.grouped_mm(x, w, off[:2]), lambda: experts.grouped_mm(x, w, off.float()),
           lambda: experts.grouped_mm(x, w, off.cpu()), lambda: experts.grouped_mm(x, w.to(F16), off),
           lambda: experts.grouped_mm(x.float(), w.float(), off), lambda: experts.grouped_mm(x, w, off, transpose=True),
           lambda: experts.grouped_mm(x, w, off, out_dtype=F16),
           lambda: experts.grouped_mm(x, w, off, out=torch.zeros(4, 15, dtype=BF16, device=DEV)),
           lambda: experts.grouped_wgrad(x, x[:3], off), lambda: experts.grouped_wgrad(x, x, off, accumulate=True),
           lambda: experts.grouped_wgrad(x, x, off, out=torch.zeros(2, 8, 8, dtype=F16, device=DEV)),
           lambda: experts.swiglu(x[:, :7]), lambda: experts.swiglu(x.double()), lambda: experts.swiglu(x, off.float()),
           lambda: experts.swiglu_backward(x, x), lambda: experts.swiglu_backward(x[:, :4].float(), x),
           lambda: experts.clip_grad_norm([x, x], 1.0), lambda: experts.clip_grad_norm([x, x[:1]], 1.0),
           lambda: experts.clip_grad_norm([x[:1].expand(4, 8)], 1.0), lambda: experts.clip_grad_norm([x.double()], 1.0),
           lambda: experts.clip_grad_norm([x], 1.0, out=[]), lambda: experts.clip_grad_norm([x], 1.0, out=[x[:2]]),
           lambda: experts.clip_grad_norm([x[:2], x[2:]], 1.0, out=[x[2:], x[:2]])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"case {i} was taken")


def test_header_names_every_operator():
    src = (ROOT / "include" / "hexmoe.h").read_text()
    for name in ("hexmoe_grouped_mm", "hexmoe_grouped_wgrad", "hexmoe_swiglu_backward", "hexmoe_clip_grad_norm"):
        assert name in src and name in _lib.EXPORTS
