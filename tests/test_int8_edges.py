"""Experts in 8-bit integers where rounding, splits, offsets and far gates show: against whole numbers and 64 bits."""

from __future__ import annotations

import pytest
import torch
from test_experts import BF16, DEV, F16, F32, ROUND, device_word, normal, offsets_of  # noqa: F401
from test_experts_edges import HALF_STEP
from test_int8 import assert_layer, int8_stack, layer_inputs, product, quantized  # noqa: F401

from blackhole_b200 import int8


# ------------------------------------------------------------------ a token's slots
def whole_layer(T, E, k, H, I, dtype, seed):
    """A layer whose activation f32 holds exactly: rows of whole numbers with a largest one of 127 (scale 1), gates of at
    least 64 (whose sigmoid is 1 in f32), and products of gate and up below 2^24."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(1, 16, (T, H), generator=g).to(dtype)
    x[:, 0] = 127
    w13 = torch.randint(-8, 9, (E, 2 * I, H), generator=g).to(torch.int8)
    w13[:, :I] = w13[:, :I].abs() + 1
    w2, _ = int8_stack((E, H, I), seed + 1)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    weights = torch.rand(T, k, generator=g) + 0.25
    return x, weights, ids, w13, w2


def slots_of(x, ids, w13, s13, w2, s2):
    """Every slot's row [T, k, H] in 64 bits, from the whole numbers of the activation."""
    w13, w2, s13, s2 = w13.double(), w2.double(), s13.double(), s2.double()
    I = w2.shape[2]
    h = torch.einsum("th,tkih->tki", x.double(), w13[ids]) * s13[ids]
    gate, up = h[..., :I], h[..., I:]
    assert (gate >= 64).all() and (gate * up).abs().max() < 2 ** 24
    q, scale, _ = quantized(gate * up)
    return torch.einsum("tki,tkhi->tkh", q, w2[ids]) * s2[ids] * scale[..., None]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("T,E,k,H,I", [(1, 3, 2, 16, 16), (40, 7, 5, 48, 32), (700, 4, 4, 32, 96), (9, 12, 9, 64, 16)])
def test_slots_are_summed_before_they_are_rounded(T, E, k, H, I, dtype):
    """Nothing between the products and a token's sum has fewer than 32 bits: whole sums are exact, scales, the scaled
    values and their products with a weight are rounded (4 x 2^-24, and one of the activation's scale), k sums add one each."""
    x, weights, ids, w13, w2 = whole_layer(T, E, k, H, I, dtype, 7)
    s13, s2 = torch.ones(E, 2 * I), torch.full((E, H), 2.0 ** -20)
    y = slots_of(x, ids, w13, s13, w2, s2) * weights.double()[..., None]
    want, mass = y.sum(1), y.abs().sum(1)
    assert mass.max() < 6e4
    q13, q2 = (torch.zeros(*w.shape[:2], 128, dtype=torch.int8, device=DEV)[..., :w.shape[2]].copy_(w) for w in (w13, w2))
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), q13, s13.to(DEV), q2, s2.to(DEV))
    f32 = (k + 6) * 2.0 ** -24 * mass
    assert got.dtype == dtype
    assert ((got.double().cpu() - want).abs() <= f32 + 1.01 * ROUND[dtype] * (want.abs() + f32) + HALF_STEP[dtype]).all()


@pytest.mark.gpu
def test_slots_past_the_range_of_16_bits():
    """Two experts whose rows are each other's negatives: the sum of slots that fp16 cannot hold is 0."""
    x, weights, ids, w13, w2 = whole_layer(20, 2, 2, 32, 16, F16, 9)
    w13[1], w2[1], weights[:, 1] = w13[0], (-w2[0].clamp(min=-127)).to(torch.int8), weights[:, 0]
    w2[0] = w2[0].clamp(min=-127)
    s13, s2 = torch.ones(2, 32), torch.ones(2, 32)
    assert (slots_of(x, ids, w13, s13, w2, s2) * weights.double()[..., None]).abs().max() > 1e6
    got = int8.int8_moe(*(t.to(DEV) for t in (x, weights, ids, w13, s13, w2, s2)))
    assert not got.any()


@pytest.mark.gpu
def test_routing_weights_of_any_size():
    """An activation's scale times a routing weight that is no normal number, under a result that is one."""
    x, weights, ids, w13, w2 = whole_layer(20, 4, 2, 32, 16, F32, 11)
    s13, s2 = torch.ones(4, 32), torch.full((4, 32), 2.0 ** 100)
    y = slots_of(x, ids, w13, s13, w2, s2) * 2.0 ** -100 * 2.0 ** -60 * weights.double()[..., None]
    s13[:, 16:] = 2.0 ** -100
    got = int8.int8_moe(*(t.to(DEV) for t in (x, weights * 2.0 ** -60, ids, w13, s13, w2, s2)))
    assert ((got.double().cpu() - y.sum(1)).abs() <= 9 * 2.0 ** -24 * y.abs().sum(1)).all()


# ------------------------------------------------------------------ split reductions
def assert_exact(got, want, dtype):
    """Sums are whole numbers, exact; one becomes f32, is multiplied by two scales (3 roundings of 2^-24) and rounded to
    the type, whatever number of pairs its reduction was split over."""
    f32 = 3.01 * 2.0 ** -24 * want.abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert ((got.double().cpu() - want).abs() <= f32 + 1.01 * ROUND[dtype] * (want.abs() + f32) + HALF_STEP[dtype]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("rows,n,k", [(1, 512, 4096), (7, 776, 1624), (300, 512, 4096), (129, 24, 8000), (5, 2049, 33), (3, 7, 131071),
                                      (900, 700, 640)])
def test_sums_of_parts_are_whole_numbers(rows, n, k, dtype):
    """Parts that cancel: halves of every sum with opposite signs, but for what the last values add."""
    x, x_scale = int8_stack((rows, k), 21)
    w, w_scale = int8_stack((n, k), 22)
    half = k // 2
    x[:, half:2 * half], w[:, half:2 * half] = x[:, :half], -w[:, :half].clamp(min=-127)
    w[:, :half] = w[:, :half].clamp(min=-127)
    w[:, :3] += (w[:, :3] < 100).to(torch.int8)
    x_scale, w_scale = x_scale * 0.01, w_scale * 0.01     # fp16 holds the results
    want, mass = product(x, x_scale, w[None], w_scale[None], torch.tensor([0, rows]), rows)
    assert k < 100 or float(want.abs().median()) < 1e-3 * float(mass.median())
    got = int8.grouped_mm_int8(x.to(DEV), w.to(DEV), w_scale.to(DEV), x_scale=x_scale.to(DEV), out_dtype=dtype)
    assert_exact(got, want, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("sizes,first,n,k", [([3, 0, 20, 5, 1], 4, 200, 4096), ([40, 1, 90], 0, 136, 2048), ([1] * 40, 2, 64, 1500)], ids=str)
def test_rows_alone_and_among_others(sizes, first, n, k, dtype):
    """The same row in batches that split differently, in groups with gaps before and behind: the same bits."""
    rows = first + sum(sizes) + 3
    x, x_scale = int8_stack((rows, k), 23)
    w, w_scale = int8_stack((len(sizes), n, k), 24)
    if first:
        x_scale[:first] = float("nan")
    x_scale[-3:] = float("inf")
    off = offsets_of(sizes, first)
    xd, sd, wd, ws = x.to(DEV), x_scale.to(DEV), w.to(DEV), w_scale.to(DEV)
    got = int8.grouped_mm_int8(xd, wd, ws, off.to(DEV), x_scale=sd, out_dtype=dtype)
    want, _ = product(x, torch.nan_to_num(x_scale, 0, 0, 0), w, w_scale, off, rows)
    assert_exact(got, want, dtype)
    for e, size in enumerate(sizes):
        part = slice(int(off[e]), int(off[e + 1]))
        many = torch.cat([xd[part]] * 30), torch.cat([sd[part]] * 30)
        assert torch.equal(int8.grouped_mm_int8(xd[part], wd[e], ws[e], x_scale=sd[part], out_dtype=dtype), got[part])
        assert torch.equal(int8.grouped_mm_int8(many[0], wd[e], ws[e], x_scale=many[1], out_dtype=dtype)[:size], got[part])


@pytest.mark.gpu
def test_matrices_that_stream_through_l2_bit_for_bit():
    """Matrices of more than 64 MB read once, and each of them alone, which stays in L2."""
    E, n, k = 40, 1024, 2048
    w = torch.randint(-127, 128, (E, n, k), dtype=torch.int8, device=DEV)
    ws = torch.rand(E, n, device=DEV)
    x = normal((80, k), BF16, 120).to(DEV)
    got = int8.grouped_mm_int8(x, w, ws, torch.arange(0, 81, 2, dtype=torch.int32, device=DEV))
    for e in range(E):
        rows = slice(2 * e, 2 * e + 2)
        one = int8.grouped_mm_int8(x[rows], w[e:e + 1], ws[e:e + 1], torch.tensor([0, 2], device=DEV))
        assert torch.equal(one, got[rows])


# ------------------------------------------------------------------ gates far below zero
@pytest.mark.gpu
def test_gates_far_below_zero():
    """silu is a normal f32 number down to gates of -91, where 1 + e^-gate is none; one column of the activation, so that
    its 8-bit value is 127 whatever its error (a fast exponential's, 1.2 |g| + 2 units of 2^-23, twice over)."""
    gates = torch.tensor([-1.0, -40, -80, -87, -88, -88.5, -89, -90, -91])
    x, w13, w2 = torch.zeros(1, 16), torch.zeros(9, 32, 16, dtype=torch.int8), torch.zeros(9, 16, 16, dtype=torch.int8)
    x[0, 0], w13[:, 0, 0], w13[:, 16, 0], w2[:, :, 0] = 127, 1, 1, 1
    s13, s2 = torch.ones(9, 32), torch.ones(9, 16)
    s13[:, 0], s13[:, 16] = gates / 127, 2.0 ** 20 / 127
    weights, ids = torch.ones(9, 1), torch.arange(9)[:, None]
    g = (s13[:, 0].double() * 127)
    want = g * torch.sigmoid(g) * (s13[:, 16].double() * 127)
    got = int8.int8_moe(*(t.to(DEV) for t in (x.expand(9, 16), weights, ids, w13, s13, w2, s2))).double().cpu()
    assert ((got - want[:, None]).abs() <= (16 + 3 * g.abs()[:, None]) * 2.0 ** -23 * want.abs()[:, None]).all(), (got[:, 0], want)


# ------------------------------------------------------------------ groups and plans
def clamped(offsets, rows):
    """The groups that any offsets stand for: each entry within 0..rows and no less than the one before."""
    return torch.cummax(offsets.clamp(0, rows), 0).values


@pytest.mark.gpu
@pytest.mark.parametrize("k", [32, 4096])
@pytest.mark.parametrize("at", [0, 1, 30, 31, 32, 33, 63, 64, 65, 69, 70])
def test_offsets_that_are_none(at, k):
    """One bad entry among 70 groups, before, at and behind a step of 32: the clamped groups' products, and the error word."""
    from blackhole_b200.hex_moe import device_status
    E, n, rows = 70, 48, 210
    x, x_scale = int8_stack((rows, k), 31)
    w, w_scale = int8_stack((E, n, k), 32)
    args = x.to(DEV), w.to(DEV), w_scale.to(DEV)
    for bad in (-7, 500, 2 ** 40, 0, 209):
        off = torch.arange(0, rows + 1, 3)
        if int(off[at]) == bad:
            continue
        off[at] = bad
        real = clamped(off, rows)
        want, mass = product(x, x_scale, w, w_scale, real, rows)
        got = int8.grouped_mm_int8(*args, off.to(DEV), x_scale=x_scale.to(DEV), out_dtype=F32)
        assert ((got.double().cpu() - want).abs() <= 2.0 ** -24 * (4 * want.abs() + 19 * mass)).all()
        assert device_status(0) == (0 if torch.equal(real, off) else 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("H", [16, 512, 528, 2048, 2064, 4112, 16400, 20000])
def test_tokens_of_any_length(H, dtype):
    """Rows that 8, 32, 64 and 256 threads take, at the borders between them, and rows longer than their registers."""
    x, weights, ids, w13, w2 = layer_inputs(3, H, 16, dtype, 6, 2, 41)
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), *w13, *w2)
    assert_layer(got, x, weights, ids, w13, w2)
    wide = torch.cat([x, x], 1).to(DEV)[:, 1:H + 1]      # rows that do not begin on 16 bytes, read one by one
    assert_layer(int8.int8_moe(wide, weights.to(DEV), ids.to(DEV), *w13, *w2), wide.cpu(), weights, ids, w13, w2)


@pytest.mark.gpu
@pytest.mark.parametrize("T,k", [(1, 1), (1024, 2), (683, 3), (4097, 2), (5, 1024)])
def test_slots_on_both_sides_of_a_cluster(T, k):
    """2048 slots are placed by one block, the next ones by eight; as many slots a token as there may be."""
    x, weights, ids, w13, w2 = layer_inputs(7, 32, 16, BF16, T, min(k, 7), 51)
    if k > 7:
        ids, weights = ids.repeat(1, k // 7 + 1)[:, :k], weights.repeat(1, k // 7 + 1)[:, :k] / (k / 7)
    some = torch.arange(0, T, max(1, T // 150))
    got = int8.int8_moe(x.to(DEV), weights.to(DEV), ids.to(DEV), *w13, *w2)
    assert_layer(got.cpu()[some], x[some], weights[some], ids[some], w13, w2)
