"""Edges of the operators of experts.py beyond test_experts.py: gates far from zero in every type, sums long enough
to lose a row in, what happens to a call that fails half way, and what autograd is told."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch
from test_experts import (BF16, DEV, F16, F32, ROUND, assert_sum, device_word, normal, offsets_of,  # noqa: F401
                          swiglu_reference, wgrad_reference)

from blackhole_b200 import experts

# smallest distance between values, halved: what a result near zero may be off by
HALF_STEP = {BF16: 2.0 ** -134, F16: 2.0 ** -25, F32: 2.0 ** -150}
LARGEST = {BF16: 3.3895e38, F16: 65504.0, F32: 3.4028234e38}


def far_gates(dtype):
    """Gates at both ends of where exp(-|g|) is a normal f32 value, is none, and is zero."""
    g = torch.cat([torch.tensor([0.0, -0.0, 1e-6, -1e-6]), torch.arange(1.0, 80.0, 3.0), torch.arange(80.0, 112.0, 0.5)])
    return torch.cat([g, -g]).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("up", [1.0, -1.5, 1e3])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_swiglu_of_gates_far_from_zero(dtype, up):
    """exp(-|g|) comes from an exponential off by 2 + 1.173 |g| units and, below the normal range, by a step
    (2^-149); the sum, the divide and the products add some units."""
    gate = far_gates(dtype)
    n = len(gate)
    h = torch.cat([gate, torch.full((n,), up).to(dtype)])[None].expand(3, -1).contiguous()
    weight = torch.tensor([1.0, 0.0, -0.5])
    g, u, w = gate.double().abs(), abs(h[0, -1].double()), weight.double().abs()[:, None]
    units, step = (32 + 2 * 1.173 * g) * 2.0 ** -23, 2.0 ** -149
    slack = lambda want, scale: units * want + scale * step + 1.01 * ROUND[dtype] * want + HALF_STEP[dtype]  # noqa: E731

    def check(got, want, bound):
        largest = LARGEST[got.dtype]
        got, want = got.double().cpu(), want.double()
        inside = want.abs() <= largest
        assert ((got - want).abs() <= bound)[inside].all(), float(((got - want).abs() / bound)[inside].max())
        assert inside.any() and (got[~inside].abs() >= largest).all()

    want = swiglu_reference(h, weight)
    check(experts.swiglu(h.to(DEV), weight.to(DEV)), want, slack(want.abs(), w * u * g))
    dact = torch.full((3, n), 0.75).to(dtype)
    dh, dw = experts.swiglu_backward(dact.to(DEV), h.to(DEV), weight.to(DEV))
    want, want_dw, mass_dw, mass_gate = swiglu_reference(h, weight, dact)
    check(dh[:, :n], want[:, :n], slack(mass_gate, w * 0.75 * u * (1 + g)))
    check(dh[:, n:], want[:, n:], slack(want[:, n:].abs(), w * 0.75 * g))
    check(dw, want_dw, (float(units.max()) + (n + 2) * 2.0 ** -24) * mass_dw + n * u * 112 * step)
    assert not dh[1].any() and not experts.swiglu(h.to(DEV), weight.to(DEV))[1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_swiglu_of_infinite_and_undefined_gates(dtype):
    gate = torch.tensor([math.inf, -math.inf, math.nan, 1.0])
    h = torch.cat([gate, torch.full((4,), 2.0)])[None].to(dtype)
    act = experts.swiglu(h.to(DEV))[0].float().cpu()
    assert act[0] == math.inf and act[2].isnan() and act[3].isfinite() and not act[1].abs() > 0   # 0 or, as inf / inf, NaN


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_swiglu_of_tiny_gates(dtype):
    """silu(g) is g / 2 near zero, down to the type's smallest values."""
    tiny = torch.tensor([2.0 ** -e for e in (list(range(10, 150, 7)) if dtype != F16 else list(range(5, 25)))])
    gate = torch.cat([tiny, -tiny]).to(dtype)
    h = torch.cat([gate, torch.ones_like(gate)])[None]
    want = swiglu_reference(h, None)
    got = experts.swiglu(h.to(DEV)).double().cpu()
    assert ((got - want).abs() <= (32 * 2.0 ** -23 + 1.01 * ROUND[dtype]) * want.abs() + HALF_STEP[dtype] + 2.0 ** -149).all()
    dh, _ = experts.swiglu_backward(torch.ones(1, len(gate), dtype=dtype, device=DEV), h.to(DEV))
    want = swiglu_reference(h, None, torch.ones(1, len(gate), dtype=dtype))[0]
    assert ((dh.double().cpu() - want).abs() <= (32 * 2.0 ** -23 + 1.01 * ROUND[dtype]) * want.abs() + HALF_STEP[dtype] + 2.0 ** -149).all()
