"""Training the experts of a MoE layer in 16 bits, on B200 (sm_100a).

What stands between hex_moe.dequant_all (the 16-bit stacks w13 [E, 2I, H] and
w2 [E, H, I] of a layer's HEX tiers) and quant.quantize_stack (which takes the
trained matrices back, with the Hessians of GPTQ rounding):

  expert_mlp         the routed-expert output of 16-bit stacks, differentiable in the
                     rows, the routing weights and both stacks (hex_moe's training twin)
  grouped_mm         rows in expert order times their expert's matrix, and the
                     gradient of the rows (transpose=True)
  grouped_wgrad      the experts' weight gradients; with dy = x their Hessians
  swiglu, swiglu_backward   the activation between the two products, times the routing weight
  clip_grad_norm     the global norm of a list of gradients, and the clipping

Rows lie in expert order: group e is rows offsets[e] .. offsets[e + 1] - 1
(expert_plan makes them from a router's ids).  Inputs must be CUDA tensors on an
sm_100 device; there is no CPU path.  Calls run on the current stream of the
inputs' device, synchronise nothing and can be captured in CUDA graphs.
"""

from __future__ import annotations

import math
from array import array

import torch

from blackhole_b200 import _lib
from blackhole_b200.hex_moe import _DT, _aligned, _ptr, align, combine_rows

_16BIT = (torch.bfloat16, torch.float16)
_INDEX = {torch.int32: _lib.I32, torch.int64: _lib.I64}


_raw_stream = torch._C._cuda_getCurrentRawStream   # current_stream() without building a Stream object


def _run(name: str, dev: torch.device, *args) -> None:
    """One C call on dev's current stream (with dev current), its status raised as an exception."""
    fn = getattr(_lib.lib, name)
    index = dev.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _rows2d(t: torch.Tensor, what: str) -> torch.Tensor:
    """t as a matrix whose rows are contiguous (a copy only where they are not)."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be a matrix, got {tuple(t.shape)}")
    # a row stride shorter than a row (an expanded or overlapping view) is no stride the kernels take
    return t if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) >= t.shape[1] else t.contiguous()


def _check_groups(offsets: torch.Tensor, experts: int, dev: torch.device) -> torch.Tensor:
    if offsets.dtype not in _INDEX or offsets.dim() != 1 or offsets.shape[0] != experts + 1:
        raise ValueError(f"offsets must be int32 or int64 [{experts + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if offsets.device != dev:
        raise ValueError(f"offsets are on {offsets.device}, the rows on {dev}")
    return offsets.contiguous()


def _check_16bit(what: str, *tensors: torch.Tensor) -> None:
    t0 = tensors[0]
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{what} runs on CUDA only")
        if t.device != t0.device:
            raise ValueError(f"{what}: tensors on {t0.device} and {t.device}")
        if t.dtype not in _16BIT or t.dtype != t0.dtype:
            raise ValueError(f"{what} takes bf16 or fp16 tensors of one type, got {t0.dtype} and {t.dtype}")


def _output(out, shape: tuple, dtype, out_dtype, dev, what: str) -> torch.Tensor:
    """The caller's `out`, checked, or a new tensor of out_dtype (dtype unless given)."""
    if out is None:
        out_dtype = out_dtype or dtype
        if out_dtype not in (dtype, torch.float32):
            raise ValueError(f"{what}: out_dtype must be {dtype} or float32")
        return torch.empty(shape, dtype=out_dtype, device=dev)
    if tuple(out.shape) != shape or out.device != dev or out.dtype not in (dtype, torch.float32) or (
            out_dtype is not None and out_dtype != out.dtype):
        raise ValueError(f"{what}: out must be {dtype} or float32 {list(shape)} on {dev}")
    return out


def grouped_mm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, transpose: bool = False,
               out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x[r] W[e]^T for every row r of group e: x [R, K], w [E, N, K] -> [R, N]; with transpose
    x[r] W[e]: x [R, N] -> [R, K].  Rows of no group come back as zero.  bf16 or fp16, the
    result in the same type or (out_dtype, out) float32."""
    if w.dim() != 3:
        raise ValueError(f"w must be [E, N, K], got {tuple(w.shape)}")
    _check_16bit("grouped_mm", x, w)
    x = _rows2d(x, "x")
    E, N, K = w.shape
    offsets = _check_groups(offsets, E, x.device)
    R, width = x.shape
    if width != (N if transpose else K):
        raise ValueError(f"x has {width} columns, w is {tuple(w.shape)} (transpose={transpose})")
    if w.stride(2) != 1 or w.stride(1) < K:
        # a transposed view of [E, K, N] is that stack, used the other way round
        if w.stride(1) == 1 and w.stride(2) >= N:
            w, N, K, transpose = w.transpose(1, 2), K, N, not transpose
        else:
            w = w.contiguous()
    res = _output(out, (R, K if transpose else N), x.dtype, out_dtype, x.device, "grouped_mm")
    to = res if res.stride(1) == 1 and res.stride(0) >= res.shape[1] else torch.empty_like(
        res, memory_format=torch.contiguous_format)
    _run("hexmoe_grouped_mm", x.device, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(1), w.stride(0), _DT[x.dtype],
         R, E, N, K, transpose, offsets.data_ptr(), _INDEX[offsets.dtype], to.data_ptr(), to.stride(0), _DT[to.dtype])
    return res if to is res else res.copy_(to)


def grouped_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, out_dtype: torch.dtype | None = None,
                  out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """dW[e] = dy_e^T x_e over the rows of every group: dy [R, N], x [R, K] -> [E, N, K] (zero for
    an empty group), in their type or float32.  accumulate adds to `out`.  With dy = x these
    are the Hessians that quant.quantize_stack(H=...) takes."""
    _check_16bit("grouped_wgrad", dy, x)
    dy, x = _rows2d(dy, "dy"), _rows2d(x, "x")
    if dy.shape[0] != x.shape[0]:
        raise ValueError(f"dy has {dy.shape[0]} rows, x {x.shape[0]}")
    if accumulate and out is None:
        raise ValueError("accumulate adds to out, which is not given")
    E = offsets.shape[0] - 1 if offsets.dim() == 1 else 0
    if E < 1:
        raise ValueError("offsets must be [experts + 1]")
    offsets = _check_groups(offsets, E, x.device)
    R, N, K = x.shape[0], dy.shape[1], x.shape[1]
    res = _output(out, (E, N, K), x.dtype, out_dtype, x.device, "grouped_wgrad")
    if res.stride(2) == 1 and res.stride(1) >= K and res.stride(0) >= (N - 1) * res.stride(1) + K:
        to = res
    elif accumulate:
        to = res.contiguous()
    else:
        to = torch.empty_like(res, memory_format=torch.contiguous_format)
    _run("hexmoe_grouped_wgrad", x.device, dy.data_ptr(), dy.stride(0), x.data_ptr(), x.stride(0), _DT[x.dtype], R, E, N,
         K, offsets.data_ptr(), _INDEX[offsets.dtype], to.data_ptr(), to.stride(1), to.stride(0), _DT[to.dtype],
         accumulate)
    return res if to is res else res.copy_(to)


def _check_row_weights(row_weights, rows: int, dev: torch.device):
    if row_weights is None:
        return None
    if row_weights.dtype != torch.float32 or row_weights.shape != (rows,) or row_weights.device != dev:
        raise ValueError(f"row_weights must be float32 [{rows}] on {dev}")
    return row_weights.contiguous()


def swiglu(h: torch.Tensor, row_weights: torch.Tensor | None = None) -> torch.Tensor:
    """silu(gate) * up * row_weights of rows h [R, 2I] = [gate | up] -> [R, I] (f32, bf16 or fp16)."""
    if not h.is_cuda:
        raise ValueError("swiglu runs on CUDA only")
    if h.dtype not in _DT:
        raise ValueError(f"unsupported dtype {h.dtype}")
    h = _rows2d(h, "h")
    R, width = h.shape
    if width % 2 or not width:
        raise ValueError(f"h must be [R, 2 * I], got {tuple(h.shape)}")
    row_weights = _check_row_weights(row_weights, R, h.device)
    act = torch.empty(R, width // 2, dtype=h.dtype, device=h.device)
    _run("hexmoe_swiglu", h.device, h.data_ptr(), _DT[h.dtype], R, width // 2, h.stride(0), _ptr(row_weights),
         act.data_ptr(), width // 2)
    return act


def swiglu_backward(dact: torch.Tensor, h: torch.Tensor, row_weights: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradient of swiglu(h, row_weights) for dact [R, I]: dh [R, 2I], and that of row_weights
    (float32 [R]; None without them).  out takes dh; it may be h itself."""
    if not h.is_cuda or not dact.is_cuda:
        raise ValueError("swiglu_backward runs on CUDA only")
    if h.dtype not in _DT or dact.dtype != h.dtype or dact.device != h.device:
        raise ValueError(f"dact ({dact.dtype}, {dact.device}) and h ({h.dtype}, {h.device}) must agree")
    if h.dim() != 2 or h.shape[1] % 2 or not h.shape[1] or dact.shape != (h.shape[0], h.shape[1] // 2):
        raise ValueError(f"h must be [R, 2 * I] and dact [R, I], got {tuple(h.shape)} and {tuple(dact.shape)}")
    R, I = dact.shape
    if out is not None and (out.shape != h.shape or out.dtype != h.dtype or out.device != h.device
                            or out.stride(1) != 1 or out.stride(0) < 2 * I):
        raise ValueError(f"out must be {h.dtype} {list(h.shape)} with contiguous rows")
    row_weights = _check_row_weights(row_weights, R, h.device)
    h, dact = _rows2d(h, "h"), _rows2d(dact, "dact")
    dh = torch.empty(R, 2 * I, dtype=h.dtype, device=h.device) if out is None else out
    dw = None if row_weights is None else torch.empty(R, dtype=torch.float32, device=h.device)
    _run("hexmoe_swiglu_backward", h.device, dact.data_ptr(), dact.stride(0), h.data_ptr(), h.stride(0), _DT[h.dtype], R,
         I, _ptr(row_weights), dh.data_ptr(), dh.stride(0), _ptr(dw))
    return dh, dw


def _dense(t: torch.Tensor) -> bool:
    """Whether t's values fill one run of memory, in any order of its dimensions."""
    if t.is_contiguous():
        return True
    need = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != need:
            return False
        need *= size
    return True


def _runs(t: torch.Tensor):
    """Tensors that cover t's values, each one run of memory (t itself where it is dense)."""
    if t.numel() == 0 or _dense(t):
        yield t
        return
    if 0 in t.stride():
        raise ValueError("clip_grad_norm: an expanded tensor holds a value more than once")
    d = max(range(t.dim()), key=lambda i: t.stride(i) if t.shape[i] > 1 else -1)
    for i in range(t.shape[d]):
        yield from _runs(t.select(d, i))


_CLIP_RUNS = 1 << 16


def clip_grad_norm(grads, max_norm: float, norm_type: float = 2.0, out=None) -> torch.Tensor:
    """The norm of all values of `grads` (a tensor or a list of tensors; f32, bf16 or fp16, mixed;
    None entries are skipped), and the values scaled by min(1, max_norm / (norm + 1e-6)): in
    place, or into `out` (tensors of the same shapes and strides, of any of these types).  norm_type
    2 or inf.  Returns the norm before clipping, float32 [] on the device.  A norm that is not finite
    is not refused (that would synchronise): it scales by 0 or NaN."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if norm_type not in (2, 2.0, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    if out is not None:
        out = [out] if isinstance(out, torch.Tensor) else list(out)
        if len(out) != len(grads) or any((g is None) != (o is None) for g, o in zip(grads, out)):
            raise ValueError("out must hold a tensor for every gradient")
        out = [o for o in out if o is not None]
    grads = [g for g in grads if g is not None]
    if not grads:
        raise ValueError("clip_grad_norm: no gradients")
    dev = grads[0].device
    if dev.type != "cuda":
        raise ValueError("clip_grad_norm runs on CUDA only")
    held = grads if out is None else grads + out
    if {t.get_device() for t in held} != {dev.index}:
        raise ValueError(f"clip_grad_norm: not every tensor is on {dev}")
    if out is not None and [g.shape for g in grads] != [o.shape for o in out]:
        raise ValueError("every tensor of out must have its gradient's shape")
    if not all([t.is_contiguous() for t in held]):
        if out is not None and [g.stride() for g in grads] != [o.stride() for o in out]:
            raise ValueError("every tensor of out must have its gradient's strides")
        grads = [r for g in grads for r in _runs(g)]
        if len(grads) > _CLIP_RUNS:
            raise ValueError(f"clip_grad_norm: the tensors fall into {len(grads)} runs of memory (at most {_CLIP_RUNS})")
        if out is not None:
            out = [r for o in out for r in _runs(o)]
    n = len(grads)
    try:
        types = array("i", [_DT[g.dtype] for g in grads])
        out_types = None if out is None else array("i", [_DT[o.dtype] for o in out])
    except KeyError as e:
        raise ValueError(f"clip_grad_norm: unsupported dtype {e.args[0]}") from None
    ptrs, counts = array("Q", [g.data_ptr() for g in grads]), array("q", [g.numel() for g in grads])
    out_ptrs = None if out is None else array("Q", [o.data_ptr() for o in out])
    norm = torch.empty((), dtype=torch.float32, device=dev)
    nbytes = _lib.lib.hexmoe_clip_grad_norm_workspace_bytes(n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    at = lambda a: None if a is None else a.buffer_info()[0]  # noqa: E731
    _run("hexmoe_clip_grad_norm", dev, n, at(ptrs), at(counts), at(types), at(out_ptrs), at(out_types), max_norm,
         norm_type == math.inf, norm.data_ptr(), ws.data_ptr(), nbytes)
    return norm


def expert_plan(topk_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, tuple]:
    """The expert order of routed slots (topk_ids [T, k]): offsets int32 [E + 1], slot int32 [P] (the
    slot of every row, T * k where a row has none), rows int32 [T * k] (the row of every slot, -1
    for an id outside 0..E-1), and the plan for the gather.  P = T * k + min(E, T * k)."""
    if topk_ids.dim() != 2:
        raise ValueError(f"topk_ids must be [T, k], got {tuple(topk_ids.shape)}")
    sid, eid, npp = align(topk_ids.reshape(-1), num_experts, 1)
    S, dev = topk_ids.numel(), sid.device
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    _run("hexmoe_group_offsets", dev, _ptr(eid), eid.numel(), _ptr(npp), 1, num_experts, _ptr(offsets))
    rows = torch.full((S + 1,), -1, dtype=torch.int32, device=dev)
    rows[sid.long()] = torch.arange(sid.numel(), dtype=torch.int32, device=dev)
    return offsets, sid, rows[:S], (sid, eid, npp)


def _gather(x: torch.Tensor, topk: int, num_experts: int, plan: tuple) -> torch.Tensor:
    """x[slot / topk] for every row of an expert_plan (16-bit).  Rows past the last
    group's are not written: no product reads them."""
    sid, _, npp = plan
    x = _aligned(x)
    xs = torch.empty(sid.numel(), x.shape[1], dtype=x.dtype, device=x.device)
    _run("hexmoe_gather", x.device, _ptr(x), _DT[x.dtype], x.shape[0], x.shape[1], topk, num_experts, _ptr(sid), _ptr(npp),
         1, _ptr(xs))
    return xs


class _ExpertMLP(torch.autograd.Function):
    """y_r = (w_r silu(Wg x) * (Wu x)) Wd^T per routed row, summed per token.  The routing weight
    enters at the activation, so its gradient falls out of the activation's."""

    @staticmethod
    def forward(ctx, x, topk_weights, topk_ids, w13, w2):
        T, k = topk_ids.shape
        E = w13.shape[0]
        offsets, slot, rows, plan = expert_plan(topk_ids, E)
        xs = _gather(x, k, E, plan)
        flat = torch.cat([topk_weights.float().reshape(-1), topk_weights.new_zeros(1, dtype=torch.float32)])
        weight = flat[slot.long()]
        h = grouped_mm(xs, w13, offsets)
        act = swiglu(h, weight)
        ctx.save_for_backward(xs, h, act, weight, offsets, rows, w13, w2, *plan)
        ctx.tokens, ctx.topk, ctx.weights_dtype = T, k, topk_weights.dtype
        return combine_rows(grouped_mm(act, w2, offsets), T, k, rows)

    @staticmethod
    def backward(ctx, dout):
        xs, h, act, weight, offsets, rows, w13, w2, *plan = ctx.saved_tensors
        T, k = ctx.tokens, ctx.topk
        dy = _gather(dout, k, w13.shape[0], tuple(plan))
        need = ctx.needs_input_grad
        dw2 = grouped_wgrad(dy, act, offsets, out_dtype=w2.dtype) if need[4] else None
        dx = dweights = dw13 = None
        if need[0] or need[1] or need[3]:
            dh, dweight = swiglu_backward(grouped_mm(dy, w2, offsets, transpose=True), h, weight)
            if need[3]:
                dw13 = grouped_wgrad(dh, xs, offsets, out_dtype=w13.dtype)
            if need[0]:
                dx = combine_rows(grouped_mm(dh, w13, offsets, transpose=True), T, k, rows)
            if need[1]:
                held = rows >= 0   # a slot whose id names no expert has no row, and no gradient
                dweights = torch.where(held, dweight[rows.clamp(min=0).long()], 0).view(T, k).to(ctx.weights_dtype)
        return dx, dweights, None, dw13, dw2


def expert_mlp(x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, w13: torch.Tensor,
               w2: torch.Tensor) -> torch.Tensor:
    """Routed-expert output [T, H] of a SwiGLU MoE layer with 16-bit experts, differentiable in
    x, topk_weights, w13 and w2: what hex_moe computes for HEX tiers, on the stacks that
    dequant_all makes of them (w13 [E, 2I, H]: gate rows, then up; w2 [E, H, I])."""
    _check_16bit("expert_mlp", x, w13, w2)
    if w13.dim() != 3 or w2.dim() != 3 or w13.shape[0] != w2.shape[0] or w13.shape[1] != 2 * w2.shape[2] or \
            w13.shape[2] != w2.shape[1]:
        raise ValueError(f"w13 must be [E, 2I, H] and w2 [E, H, I], got {tuple(w13.shape)} and {tuple(w2.shape)}")
    if x.dim() != 2 or x.shape[1] != w13.shape[2] or x.shape[1] % 32:
        raise ValueError(f"x must be [T, {w13.shape[2]}] (a multiple of 32), got {tuple(x.shape)}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0] or topk_weights.shape != topk_ids.shape:
        raise ValueError("topk_weights / topk_ids / x disagree on T or k")
    return _ExpertMLP.apply(x, topk_weights, topk_ids, w13, w2)
