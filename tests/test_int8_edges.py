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
