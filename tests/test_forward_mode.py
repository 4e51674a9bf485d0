"""Forward-mode differentiation: no operator of experts, router or int8 drops a tangent without a word."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from test_experts import BF16, DEV, F32, device_word, normal, offsets_of  # noqa: F401

from blackhole_b200 import experts, int8, router


def test_a_tangent_is_seen():
    x, plain = normal((4, 8), F32, 1), normal((4, 8), F32, 2)
    assert not experts._recorded(x, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert experts._recorded(plain, None, dual) and not experts._recorded(plain, forward_ad.unpack_dual(dual).primal)
        with torch.no_grad():
            assert experts._recorded(dual)
        with torch.inference_mode():
            assert not experts._recorded(plain)
    assert not experts._recorded(dual)


@pytest.mark.gpu
def test_operators_refuse_tangents():
    x, off = normal((4, 32), BF16, 3).to(DEV), offsets_of([1, 3]).to(DEV)
    w16, row_weights = normal((2, 8, 32), BF16, 4).to(DEV), torch.ones(4, device=DEV)
    w8, s8 = int8.quantize_rows(w16)
    w13, s13 = int8.quantize_rows(normal((2, 32, 32), BF16, 5).to(DEV))
    w2, s2 = int8.quantize_rows(normal((2, 32, 16), BF16, 6).to(DEV))
    logits, tw = normal((4, 8), F32, 7).to(DEV), torch.ones(4, 2, device=DEV)
    ids = torch.zeros(4, 2, dtype=torch.int64, device=DEV)
    calls = {
        "route": (logits, lambda t: router.route(t, 2)),
        "grouped_mm_int8 x": (x, lambda t: int8.grouped_mm_int8(t, w8, s8, off)),
        "grouped_mm_int8 scale": (s8, lambda t: int8.grouped_mm_int8(x, w8, t, off)),
        "int8_moe x": (x, lambda t: int8.int8_moe(t, tw, ids, w13, s13, w2, s2)),
        "int8_moe weights": (tw, lambda t: int8.int8_moe(x, t, ids, w13, s13, w2, s2)),
        "grouped_mm x": (x, lambda t: experts.grouped_mm(t, w16, off)),
        "grouped_mm w": (w16, lambda t: experts.grouped_mm(x, t, off)),
        "grouped_wgrad": (x, lambda t: experts.grouped_wgrad(x, t, off)),
        "swiglu": (x, lambda t: experts.swiglu(t)),
        "swiglu weights": (row_weights, lambda t: experts.swiglu(x, t)),
        "expert_mlp": (tw, lambda t: experts.expert_mlp(x, t, ids, w13.bfloat16(), w2.bfloat16())),
    }
    for name, (t, call) in calls.items():
        call(t)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t, torch.ones_like(t))
            for recording in (True, False):
                with torch.set_grad_enabled(recording), pytest.raises(RuntimeError):   # NotImplementedError is one
                    call(dual)
                    pytest.fail(f"{name} took a dual tensor")
            call(forward_ad.unpack_dual(dual).primal)
