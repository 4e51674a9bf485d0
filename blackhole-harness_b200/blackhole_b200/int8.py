"""A MoE layer's experts in 8-bit integers, on B200 (sm_100a).

The tensor cores take 8-bit integers at twice the rate of 16 bits, and the stacks are half the bytes: a layer
whose memory allows 8 bits for an expert's value (HEX takes 3 or 4) runs its prefill on these.

  quantize_rows      rows in 8 bits with a scale each: activations by token, and a stack of matrices by channel
  grouped_mm_int8    rows in expert order times their expert's 8-bit matrix (or all rows times one)
  int8_moe           the routed-expert output of 8-bit stacks: hex_moe and expert_mlp for such experts

Stacks come from 16-bit ones (hex_moe.dequant_all, or what expert_mlp has trained):

    w13, w2 = (quantize_rows(w) for w in dequant_all(tiers))
    out = int8_moe(x, *router.route(logits, 8), *w13, *w2)

Inputs must be CUDA tensors on an sm_100 device; there is no CPU path.  Calls run on the current stream of the
inputs' device, synchronise nothing and can be captured in CUDA graphs.  Nothing here is differentiable: the products
refuse inputs that require a gradient or have a tangent; what quantize_rows returns has neither.
"""

from __future__ import annotations

import torch

from blackhole_b200 import _lib
from blackhole_b200.experts import _INDEX, _call, _check_groups, _recorded, _rows2d, _run, _workspace, _written
from blackhole_b200.hex_moe import _DT, _ptr

MAX_K = 131071   # longest sum of products of 8-bit integers that int32 holds
MAX_SIZE = 1 << 24   # of every other dimension of a stack
MAX_ROW = 1 << 30

_quantize_rows, _grouped_mm_int8, _int8_forward = (_lib.lib.hexmoe_quantize_rows, _lib.lib.hexmoe_grouped_mm_int8,
                                                   _lib.lib.hexmoe_int8_forward)


def _pitched(shape: tuple, dev: torch.device) -> torch.Tensor:
    """An int8 tensor whose rows begin on multiples of 16 bytes."""
    k = shape[-1]
    return torch.empty(*shape[:-1], (k + 15) // 16 * 16, dtype=torch.int8, device=dev)[..., :k]


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """t (2 or 3 dimensions, int8) with rows that begin on multiples of 16 bytes: a copy where they do not."""
    *outer, ld, step = t.stride()
    k = t.shape[-1]
    if (step == 1 or k == 1) and ld % 16 == 0 and ld >= k and t.data_ptr() % 16 == 0 and (
            not outer or t.shape[0] == 1 or (outer[0] % 16 == 0 and outer[0] >= ld)):
        return t
    return _pitched(t.shape, t.device).copy_(t)


def _check_stack(what: str, w: torch.Tensor, scale: torch.Tensor, dev: torch.device, name: str) -> None:
    if w.dim() and (w.shape[-1] > MAX_K or max(w.shape) > MAX_SIZE):
        raise ValueError(f"{what}: {name} {tuple(w.shape)}: rows have at most {MAX_K} values, every other size is at most {MAX_SIZE}")
    if w.dtype != torch.int8 or w.device != dev:
        raise ValueError(f"{what}: {name} must be int8 on {dev}, got {w.dtype} on {w.device}")
    if scale.dtype != torch.float32 or scale.shape != w.shape[:-1] or scale.device != dev:
        raise ValueError(f"{what}: the scales of {name} must be float32 {list(w.shape[:-1])} on {dev}, got {scale.dtype} "
                         f"{tuple(scale.shape)} on {scale.device}")


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of x [..., K] (f32, bf16 or fp16) in 8 bits: q int8 [..., K] and scale float32 [...], with
    scale = max |x| / 127 and q = round(127 x / max |x|), ties to even, as exact arithmetic has it.  The rows of q begin
    on multiples of 16 bytes, as the products want them.  A row of zeros has scale 0; one that holds an infinity or
    NaN has scale NaN and zeros."""
    if not x.is_cuda:
        raise ValueError("quantize_rows runs on CUDA only")
    if x.dtype not in _DT:
        raise ValueError(f"quantize_rows: unsupported dtype {x.dtype}")
    if x.dim() == 0 or not 0 < x.shape[-1] <= MAX_ROW:
        raise ValueError(f"quantize_rows: x must have rows of values, got {tuple(x.shape)}")
    shape, K = x.shape, x.shape[-1]
    rows, ld = _rows2d(x.detach().reshape(-1, K), "x")
    q, scale = _pitched(shape, x.device), torch.empty(shape[:-1], dtype=torch.float32, device=x.device)
    _run(_quantize_rows, x.device, rows.data_ptr(), _DT[x.dtype], ld, rows.shape[0], K, q.data_ptr(), (K + 15) // 16 * 16,
         scale.data_ptr())
    return q, scale


def grouped_mm_int8(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, offsets: torch.Tensor | None = None,
                    x_scale: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r, n] = x_scale[r] w_scale[e, n] sum_k x[r, k] w[e, n, k] for every row r of group e, rows offsets[e] ..
    offsets[e + 1] - 1: x [R, K], w int8 [E, N, K] with w_scale float32 [E, N] -> [R, N].  Without offsets w is one
    matrix [N, K] for all rows.  x is int8 with x_scale float32 [R], or f32, bf16 or fp16 and quantized on the way
    (quantize_rows).  The result is in out_dtype (f32, bf16 or fp16; x's, or bf16 for an int8 x): sums are exact (K at
    most 131071), become f32, are multiplied by both scales there and rounded to the type.  Rows of no group come back as
    zero.  `out` overlaps no input.  Stacks whose rows do not begin on multiples of 16 bytes are copied at each call;
    quantize_rows makes them so that they do."""
    if out is None and out_dtype is None and x_scale is None and offsets is not None:
        res = _call.grouped_mm_int8(x, w, w_scale, offsets)
        if res is not None:
            return res
    if not x.is_cuda:
        raise ValueError("grouped_mm_int8 runs on CUDA only")
    dev = x.device
    given = x.dtype == torch.int8
    if not given and x.dtype not in _DT:
        raise ValueError(f"grouped_mm_int8: x must be int8, f32, bf16 or fp16, got {x.dtype}")
    if given != (x_scale is not None):
        raise ValueError("grouped_mm_int8: x_scale goes with an int8 x")
    if _recorded(x, w_scale, x_scale):
        raise RuntimeError("grouped_mm_int8 is not differentiable: call it under torch.no_grad() or on detached tensors")
    if w.dim() != (2 if offsets is None else 3):
        raise ValueError(f"w must be [E, N, K], or [N, K] without offsets, got {tuple(w.shape)}")
    _check_stack("grouped_mm_int8", w, w_scale, dev, "w")
    if offsets is None:
        w, w_scale, index = w[None], w_scale[None], _lib.I32
    else:
        offsets, index = _check_groups(offsets, w.shape[0], dev)
    E, N, K = w.shape
    if x.dim() != 2 or x.shape[1] != K:
        raise ValueError(f"x must be [R, {K}], got {tuple(x.shape)}")
    R = x.shape[0]
    if given:
        if x_scale.dtype != torch.float32 or x_scale.shape != (R,) or x_scale.device != dev:
            raise ValueError(f"x_scale must be float32 [{R}] on {dev}, got {x_scale.dtype} {tuple(x_scale.shape)} on {x_scale.device}")
        x, x_scale = _aligned_rows(x), x_scale.contiguous()
        ld_x = max(x.stride(0), K)
    else:
        x, ld_x = _rows2d(x, "x")
    w, w_scale = _aligned_rows(w), w_scale.contiguous()
    dtype = out_dtype or (out.dtype if out is not None else torch.bfloat16 if given else x.dtype)
    if dtype not in _DT:
        raise ValueError(f"grouped_mm_int8: out_dtype must be f32, bf16 or fp16, got {dtype}")
    if out is not None and (out.shape != (R, N) or out.device != dev or out.dtype != dtype):
        raise ValueError(f"grouped_mm_int8: out must be {dtype} {[R, N]} on {dev}")
    direct = out is not None and (out.stride(1) == 1 or N == 1) and (out.stride(0) >= N or R == 1)
    to = out if direct else torch.empty(R, N, dtype=dtype, device=dev)
    code = _lib.I8 if given else _DT[x.dtype]
    ws, nbytes = _workspace(_lib.lib.hexmoe_grouped_mm_int8_workspace_bytes(R, E, N, K, code), x)
    _run(_grouped_mm_int8, dev, x.data_ptr(), code, ld_x, _ptr(x_scale), w.data_ptr(), max(w.stride(1), K), w.stride(0),
         w_scale.data_ptr(), R, E, N, K, _ptr(offsets), index, to.data_ptr(), max(to.stride(0), N), _DT[dtype], _ptr(ws), nbytes)
    if direct:
        _written(out)
    elif out is not None:
        out.copy_(to)
    return to if out is None else out


def int8_moe(x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor,
             w2: torch.Tensor, w2_scale: torch.Tensor) -> torch.Tensor:
    """Routed-expert output [T, H] of a SwiGLU MoE layer whose experts are 8-bit stacks with a scale for every
    channel: w13 int8 [E, 2I, H] (gate rows, then up) with w13_scale float32 [E, 2I], w2 int8 [E, H, I] with w2_scale
    [E, H] (quantize_rows makes them).  x [T, H] f32, bf16 or fp16; topk_weights and topk_ids [T, k] as hex_moe takes
    them: an id of no expert adds nothing and sets the device error word.  H and I are multiples of 16.  The rows of x
    and of the activation are quantized on the way."""
    out = _call.int8_moe(x, topk_weights, topk_ids, w13, w13_scale, w2, w2_scale)
    if out is not None:
        return out
    if not x.is_cuda:
        raise ValueError("int8_moe runs on CUDA only")
    dev = x.device
    if x.dtype not in _DT:
        raise ValueError(f"int8_moe: unsupported activation dtype {x.dtype}")
    if _recorded(x, topk_weights, w13_scale, w2_scale):
        raise RuntimeError("int8_moe is not differentiable: call it under torch.no_grad() or on detached tensors")
    _check_stack("int8_moe", w13, w13_scale, dev, "w13")
    _check_stack("int8_moe", w2, w2_scale, dev, "w2")
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[0] != w2.shape[0] or w13.shape[1] != 2 * w2.shape[2] or \
            w13.shape[2] != w2.shape[1]:
        raise ValueError(f"w13 must be [E, 2I, H] and w2 [E, H, I], got {tuple(w13.shape)} and {tuple(w2.shape)}")
    E, H, I = w2.shape
    if H % 16 or I % 16 or not H or not I:
        raise ValueError(f"int8_moe: H ({H}) and I ({I}) must be multiples of 16")
    if x.dim() != 2 or x.shape[1] != H:
        raise ValueError(f"x must be [T, {H}], got {tuple(x.shape)}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_weights / topk_ids / x disagree on T or k")
    if topk_ids.shape[1] > 1024:
        raise ValueError(f"int8_moe: topk {topk_ids.shape[1]}, at most 1024")
    if topk_weights.device != dev or topk_ids.device != dev:
        raise ValueError(f"int8_moe: x is on {dev}, topk_weights on {topk_weights.device}, topk_ids on {topk_ids.device}")
    T, k = topk_ids.shape
    out = torch.empty(T, H, dtype=x.dtype, device=dev)
    if T == 0 or k == 0:
        return out.zero_()
    x, ld_x = _rows2d(x, "x")
    weights = topk_weights.float().contiguous()
    ids = (topk_ids if topk_ids.dtype in _INDEX else topk_ids.long()).contiguous()
    w13, w2 = _aligned_rows(w13), _aligned_rows(w2)
    w13_scale, w2_scale = w13_scale.contiguous(), w2_scale.contiguous()
    ws, nbytes = _workspace(_lib.lib.hexmoe_int8_forward_workspace_bytes(T, k, E, H, I), x)
    _run(_int8_forward, dev, x.data_ptr(), _DT[x.dtype], ld_x, T, H, I, k, weights.data_ptr(), ids.data_ptr(), _INDEX[ids.dtype], E,
         w13.data_ptr(), w13.stride(1), w13.stride(0), w13_scale.data_ptr(), w2.data_ptr(), w2.stride(1), w2.stride(0),
         w2_scale.data_ptr(), out.data_ptr(), _DT[x.dtype], _ptr(ws), nbytes)
    return out
