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

grouped_mm, grouped_wgrad, swiglu and expert_mlp are differentiable (once).  What is written
into an `out` stays outside autograd's graph, as do swiglu_backward and clip_grad_norm, and
an `out` overlaps no input (swiglu_backward's may be h).
"""

from __future__ import annotations

import math
from array import array
from operator import attrgetter

import torch

from blackhole_b200 import _lib
from blackhole_b200.hex_moe import _DT, _aligned, _ptr, align, combine_rows

try:
    from blackhole_b200 import _call   # the same calls without Python's share, None where it passes
except ImportError:   # not built, or built for another torch: every call goes through Python and libhexmoe.so
    class _call:
        grouped_mm = grouped_wgrad = swiglu = swiglu_backward = clip_grad_norm = staticmethod(lambda *args: None)

_16BIT = (torch.bfloat16, torch.float16)
_INDEX = {torch.int32: _lib.I32, torch.int64: _lib.I64}


_raw_stream = torch._C._cuda_getCurrentRawStream   # current_stream() without building a Stream object
_current_device = torch.cuda.current_device
_written = torch.autograd.graph.increment_version   # tells autograd, which may hold the tensor, that it changed


def _run(fn, dev: torch.device, *args) -> None:
    """One C call on dev's current stream (with dev current), its status raised as an exception."""
    index = dev.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, fn.__name__)


def _rows2d(t: torch.Tensor, what: str) -> tuple[torch.Tensor, int]:
    """t as a matrix whose rows are contiguous (a copy only where they are not), and its row stride."""
    if t.dim() != 2:
        raise ValueError(f"{what} must be a matrix, got {tuple(t.shape)}")
    ld, step = t.stride()
    # a row stride shorter than a row (an expanded or overlapping view) is no stride the kernels take
    if ld < t.shape[1] or (step != 1 and t.shape[1] != 1):
        t = t.contiguous()
        ld = max(t.stride(0), t.shape[1])
    return t, ld


def _check_groups(offsets: torch.Tensor, experts: int, dev: torch.device) -> tuple[torch.Tensor, int]:
    """offsets, checked, and their type's code."""
    code = _INDEX.get(offsets.dtype)
    if code is None or offsets.shape != (experts + 1,):
        raise ValueError(f"offsets must be int32 or int64 [{experts + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    if offsets.device != dev:
        raise ValueError(f"offsets are on {offsets.device}, the rows on {dev}")
    return offsets.contiguous(), code


def _check_16bit(what: str, *tensors: torch.Tensor) -> int:
    """The code of the tensors' type, which is one."""
    t0 = tensors[0]
    dtype, dev = t0.dtype, t0.device
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{what} runs on CUDA only")
        if t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")
        if t.dtype != dtype:
            raise ValueError(f"{what} takes bf16 or fp16 tensors of one type, got {dtype} and {t.dtype}")
    if dtype not in _16BIT:
        raise ValueError(f"{what} takes bf16 or fp16 tensors, got {dtype}")
    return _DT[dtype]


def _output(out, shape: tuple, like: torch.Tensor, out_dtype, what: str) -> torch.Tensor:
    """The caller's `out`, checked, or a new tensor of out_dtype (like's unless given)."""
    dtype = like.dtype
    if out is None:
        if out_dtype is None or out_dtype == dtype:
            return like.new_empty(shape)
        if out_dtype != torch.float32:
            raise ValueError(f"{what}: out_dtype must be {dtype} or float32")
        return like.new_empty(shape, dtype=out_dtype)
    if out.shape != shape or out.device != like.device or out.dtype not in (dtype, torch.float32) or (
            out_dtype is not None and out_dtype != out.dtype):
        raise ValueError(f"{what}: out must be {dtype} or float32 {list(shape)} on {like.device}")
    return out


def _recorded(*tensors) -> bool:
    """Whether autograd is to see the call."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _workspace(nbytes: int, like: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    return (torch.empty(nbytes, dtype=torch.uint8, device=like.device), nbytes) if nbytes else (None, 0)


_grouped_mm, _grouped_wgrad = _lib.lib.hexmoe_grouped_mm, _lib.lib.hexmoe_grouped_wgrad
_swiglu, _swiglu_backward = _lib.lib.hexmoe_swiglu, _lib.lib.hexmoe_swiglu_backward


class _GroupedMM(torch.autograd.Function):
    """y = x W^T: dx = dy W, dW[e] = dy_e^T x_e; with transpose y = x W: dx = dy W^T, dW[e] = x_e^T dy_e.  The
    gradient of an f32 result is rounded to the 16 bits that the products take."""

    @staticmethod
    def forward(ctx, x, w, offsets, transpose, out_dtype):
        ctx.save_for_backward(x, w, offsets)
        ctx.transpose = transpose
        return grouped_mm(x, w, offsets, transpose, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dy = dy.to(x.dtype)
        dx = grouped_mm(dy, w, offsets, not ctx.transpose) if ctx.needs_input_grad[0] else None
        dw = None
        if ctx.needs_input_grad[1]:
            dw = grouped_wgrad(x, dy, offsets) if ctx.transpose else grouped_wgrad(dy, x, offsets)
        return dx, dw, None, None, None


class _GroupedWgrad(torch.autograd.Function):
    """dW[e] = dy_e^T x_e: with its gradient G, ddy = x G^T and dx = dy G.  G is rounded as above."""

    @staticmethod
    def forward(ctx, dy, x, offsets, out_dtype):
        ctx.save_for_backward(dy, x, offsets)
        return grouped_wgrad(dy, x, offsets, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        dy, x, offsets = ctx.saved_tensors
        g = g.to(x.dtype)
        ddy = grouped_mm(x, g, offsets) if ctx.needs_input_grad[0] else None
        return ddy, grouped_mm(dy, g, offsets, transpose=True) if ctx.needs_input_grad[1] else None, None, None


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, row_weights):
        ctx.save_for_backward(h, row_weights)
        return swiglu(h, row_weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dact):
        return swiglu_backward(dact, *ctx.saved_tensors)


def grouped_mm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, transpose: bool = False,
               out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """x[r] W[e]^T for every row r of group e: x [R, K], w [E, N, K] -> [R, N]; with transpose
    x[r] W[e]: x [R, N] -> [R, K].  Rows of no group come back as zero.  bf16 or fp16, the
    result in the same type or (out_dtype, out) float32.  Differentiable in x and w; with
    `out`, where they require grad, an error."""
    if out is None and out_dtype is None:
        res = _call.grouped_mm(x, w, offsets, transpose)
        if res is not None:
            return res
    if _recorded(x, w):
        if out is not None:
            raise RuntimeError("grouped_mm: x or w requires grad, and what is written into out is not differentiable")
        return _GroupedMM.apply(x, w, offsets, transpose, out_dtype)
    code = _check_16bit("grouped_mm", x, w)
    if w.dim() != 3:
        raise ValueError(f"w must be [E, N, K], got {tuple(w.shape)}")
    x, ld_x = _rows2d(x, "x")
    E, N, K = w.shape
    dev = x.device
    offsets, index_code = _check_groups(offsets, E, dev)
    R, width = x.shape
    if width != (N if transpose else K):
        raise ValueError(f"x has {width} columns, w is {tuple(w.shape)} (transpose={transpose})")
    stride_w, ld_w, step = w.stride()
    if step != 1 or ld_w < K:
        # a transposed view of [E, K, N] is that stack, used the other way round
        if ld_w == 1 and step >= N:
            ld_w, N, K, transpose = step, K, N, not transpose
        else:
            w = w.contiguous()
            stride_w, ld_w = N * K, K
    width = K if transpose else N
    res = to = _output(out, (R, width), x, out_dtype, "grouped_mm")
    ld = width
    if out is not None:
        ld = res.stride(0)
        if ld < width or res.stride(1) != 1:
            to, ld = torch.empty_like(res, memory_format=torch.contiguous_format), width
    ws, nbytes = _workspace(_lib.lib.hexmoe_grouped_mm_workspace_bytes(R, E, N, K, transpose), x)
    _run(_grouped_mm, dev, x.data_ptr(), ld_x, w.data_ptr(), ld_w, stride_w, code, R, E, N, K, transpose,
         offsets.data_ptr(), index_code, to.data_ptr(), ld, _DT[to.dtype], _ptr(ws), nbytes)
    if to is not res:
        res.copy_(to)
    elif out is not None:
        _written(out)
    return res


def grouped_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, out_dtype: torch.dtype | None = None,
                  out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """dW[e] = dy_e^T x_e over the rows of every group: dy [R, N], x [R, K] -> [E, N, K] (zero for
    an empty group), in their type or float32.  accumulate adds to `out`.  With dy = x these
    are the Hessians that quant.quantize_stack(H=...) takes.  Differentiable without `out`; sums
    in `out` are statistics or gradients, and keep no graph."""
    if out is None and not accumulate and (out_dtype is None or out_dtype in (torch.float32, x.dtype)):
        res = _call.grouped_wgrad(dy, x, offsets, out_dtype == torch.float32)
        if res is not None:
            return res
    if out is None and not accumulate and _recorded(dy, x):
        return _GroupedWgrad.apply(dy, x, offsets, out_dtype)
    code = _check_16bit("grouped_wgrad", dy, x)
    (dy, ld_dy), (x, ld_x) = _rows2d(dy, "dy"), _rows2d(x, "x")
    if dy.shape[0] != x.shape[0]:
        raise ValueError(f"dy has {dy.shape[0]} rows, x {x.shape[0]}")
    if accumulate and out is None:
        raise ValueError("accumulate adds to out, which is not given")
    E = offsets.shape[0] - 1 if offsets.dim() == 1 else 0
    if E < 1:
        raise ValueError("offsets must be [experts + 1]")
    dev = x.device
    offsets, index_code = _check_groups(offsets, E, dev)
    (R, K), N = x.shape, dy.shape[1]
    res = to = _output(out, (E, N, K), x, out_dtype, "grouped_wgrad")
    stride, ld = N * K, K
    if out is not None:
        stride, ld, step = res.stride()
        if step != 1 or ld < K or stride < (N - 1) * ld + K:
            to = res.contiguous() if accumulate else torch.empty_like(res, memory_format=torch.contiguous_format)
            stride, ld = N * K, K
    ws, nbytes = _workspace(_lib.lib.hexmoe_grouped_wgrad_workspace_bytes(R, E, N, K), x)
    _run(_grouped_wgrad, dev, dy.data_ptr(), ld_dy, x.data_ptr(), ld_x, code, R, E, N, K, offsets.data_ptr(), index_code,
         to.data_ptr(), ld, stride, _DT[to.dtype], accumulate, _ptr(ws), nbytes)
    if to is not res:
        res.copy_(to)
    elif out is not None:
        _written(out)
    return res


def _check_row_weights(row_weights, rows: int, dev: torch.device):
    if row_weights is None:
        return None
    if row_weights.dtype != torch.float32 or row_weights.shape != (rows,) or row_weights.device != dev:
        raise ValueError(f"row_weights must be float32 [{rows}] on {dev}")
    return row_weights.contiguous()


def swiglu(h: torch.Tensor, row_weights: torch.Tensor | None = None) -> torch.Tensor:
    """silu(gate) * up * row_weights of rows h [R, 2I] = [gate | up] -> [R, I] (f32, bf16 or fp16),
    differentiable in both."""
    act = _call.swiglu(h, row_weights)
    if act is not None:
        return act
    if _recorded(h, row_weights):
        return _SwiGLU.apply(h, row_weights)
    if not h.is_cuda:
        raise ValueError("swiglu runs on CUDA only")
    if h.dtype not in _DT:
        raise ValueError(f"unsupported dtype {h.dtype}")
    h, ld = _rows2d(h, "h")
    R, width = h.shape
    if width % 2 or not width:
        raise ValueError(f"h must be [R, 2 * I], got {tuple(h.shape)}")
    dev, inter = h.device, width // 2
    row_weights = _check_row_weights(row_weights, R, dev)
    act = h.new_empty((R, inter))
    _run(_swiglu, dev, h.data_ptr(), _DT[h.dtype], R, inter, ld, _ptr(row_weights), act.data_ptr(), inter)
    return act


def swiglu_backward(dact: torch.Tensor, h: torch.Tensor, row_weights: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradient of swiglu(h, row_weights) for dact [R, I]: dh [R, 2I], and that of row_weights
    (float32 [R]; None without them).  out takes dh; it may be h itself.  Not differentiable itself."""
    if out is None:
        both = _call.swiglu_backward(dact, h, row_weights)
        if both is not None:
            return both
    if not h.is_cuda or not dact.is_cuda:
        raise ValueError("swiglu_backward runs on CUDA only")
    if h.dtype not in _DT or dact.dtype != h.dtype or dact.device != h.device:
        raise ValueError(f"dact ({dact.dtype}, {dact.device}) and h ({h.dtype}, {h.device}) must agree")
    if h.dim() != 2 or h.shape[1] % 2 or not h.shape[1] or dact.shape != (h.shape[0], h.shape[1] // 2):
        raise ValueError(f"h must be [R, 2 * I] and dact [R, I], got {tuple(h.shape)} and {tuple(dact.shape)}")
    R, I = dact.shape
    if out is not None and (out.shape != h.shape or out.dtype != h.dtype or out.device != h.device
                            or out.stride(1) != 1 or (R > 1 and out.stride(0) < 2 * I)):
        raise ValueError(f"out must be {h.dtype} {list(h.shape)} with contiguous rows")
    dev = h.device
    row_weights = _check_row_weights(row_weights, R, dev)
    (h, ld_h), (dact, ld_dact) = _rows2d(h, "h"), _rows2d(dact, "dact")
    dh = h.new_empty((R, 2 * I)) if out is None else out
    dw = None if row_weights is None else row_weights.new_empty(R)
    _run(_swiglu_backward, dev, dact.data_ptr(), ld_dact, h.data_ptr(), ld_h, _DT[h.dtype], R, I, _ptr(row_weights),
         dh.data_ptr(), 2 * I if out is None else max(out.stride(0), 2 * I), _ptr(dw))
    if out is not None:
        _written(out)
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
    if 0 in (st for st, size in zip(t.stride(), t.shape) if size > 1):
        raise ValueError("clip_grad_norm: an expanded tensor holds a value more than once")
    d = max(range(t.dim()), key=lambda i: t.stride(i) if t.shape[i] > 1 else -1)
    for i in range(t.shape[d]):
        yield from _runs(t.select(d, i))


def _places(t: torch.Tensor) -> list:
    """Where t's values stand: the strides of the dimensions that have any."""
    return [(st, size) for st, size in zip(t.stride(), t.shape) if size != 1] if t.numel() else []


def _type_codes(tensors: list) -> array:
    dtypes = list(map(_get_dtype, tensors))
    try:
        if dtypes.count(dtypes[0]) == len(dtypes):
            return array("i", [_DT[dtypes[0]]]) * len(dtypes)
        return array("i", [_DT[t] for t in dtypes])
    except KeyError as e:
        raise ValueError(f"clip_grad_norm: unsupported dtype {e.args[0]}") from None


_CLIP_RUNS = 1 << 16
# called by map() over a model's gradients: the host's share of a small model's clipping
_get_device, _is_contiguous, _data_ptr, _numel = (torch.Tensor.get_device, torch.Tensor.is_contiguous,
                                                  torch.Tensor.data_ptr, torch.Tensor.numel)
_get_shape, _get_dtype = attrgetter("shape"), attrgetter("dtype")
_clip_grad_norm, _clip_workspace_bytes = _lib.lib.hexmoe_clip_grad_norm, _lib.lib.hexmoe_clip_grad_norm_workspace_bytes


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
    norm = _call.clip_grad_norm(grads, out, max_norm, norm_type == math.inf)
    if norm is not None:
        return norm
    dev = grads[0].device
    if dev.type != "cuda":
        raise ValueError("clip_grad_norm runs on CUDA only")
    held, written = grads if out is None else grads + out, grads if out is None else out
    if set(map(_get_device, held)) != {dev.index}:
        raise ValueError(f"clip_grad_norm: not every tensor is on {dev}")
    if out is not None and list(map(_get_shape, grads)) != list(map(_get_shape, out)):
        raise ValueError("every tensor of out must have its gradient's shape")
    if not all(map(_is_contiguous, held)):
        if out is not None and list(map(_places, grads)) != list(map(_places, out)):
            raise ValueError("every tensor of out must have its gradient's strides")
        grads = [r for g in grads for r in _runs(g)]
        if len(grads) > _CLIP_RUNS:
            raise ValueError(f"clip_grad_norm: the tensors fall into {len(grads)} runs of memory (at most {_CLIP_RUNS})")
        if out is not None:
            out = [r for o in out for r in _runs(o)]
    n = len(grads)
    types = _type_codes(grads)
    ptrs, counts = array("Q", map(_data_ptr, grads)), array("q", map(_numel, grads))
    if out is None:
        out_ptr = out_types_ptr = None
    else:
        out_types, out_ptrs = _type_codes(out), array("Q", map(_data_ptr, out))
        out_ptr, out_types_ptr = out_ptrs.buffer_info()[0], out_types.buffer_info()[0]
    nbytes = _clip_workspace_bytes(n)
    ws = torch.empty(nbytes // 4 + 1, dtype=torch.float32, device=dev)   # the partial sums, then the norm
    _run(_clip_grad_norm, dev, n, ptrs.buffer_info()[0], counts.buffer_info()[0], types.buffer_info()[0], out_ptr,
         out_types_ptr, max_norm, norm_type == math.inf, ws.data_ptr() + nbytes, ws.data_ptr(), nbytes)
    _written(written)
    return ws[nbytes // 4]


def expert_plan(topk_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, tuple]:
    """The expert order of routed slots (topk_ids [T, k]): offsets int32 [E + 1], slot int32 [P] (the
    slot of every row, T * k where a row has none), rows int32 [T * k] (the row of every slot, -1
    for an id outside 0..E-1), and the plan for the gather.  P = T * k + min(E, T * k)."""
    if topk_ids.dim() != 2:
        raise ValueError(f"topk_ids must be [T, k], got {tuple(topk_ids.shape)}")
    sid, eid, npp = align(topk_ids.reshape(-1), num_experts, 1)
    S, dev = topk_ids.numel(), sid.device
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    _run(_lib.lib.hexmoe_group_offsets, dev, _ptr(eid), eid.numel(), _ptr(npp), 1, num_experts, _ptr(offsets))
    rows = torch.full((S + 1,), -1, dtype=torch.int32, device=dev)
    rows[sid.long()] = torch.arange(sid.numel(), dtype=torch.int32, device=dev)
    return offsets, sid, rows[:S], (sid, eid, npp)


def _gather(x: torch.Tensor, topk: int, num_experts: int, plan: tuple) -> torch.Tensor:
    """x[slot / topk] for every row of an expert_plan (16-bit).  Rows past the last
    group's are not written: no product reads them."""
    sid, _, npp = plan
    x = _aligned(x)
    xs = torch.empty(sid.numel(), x.shape[1], dtype=x.dtype, device=x.device)
    _run(_lib.lib.hexmoe_gather, x.device, _ptr(x), _DT[x.dtype], x.shape[0], x.shape[1], topk, num_experts, _ptr(sid), _ptr(npp),
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
    @torch.autograd.function.once_differentiable
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
