"""The operators that train the 16-bit experts of a MoE layer, as they are measured.

A layer's experts are dequantized to 16-bit stacks (`dequant_all`), trained on routed rows, and
quantized again.  What that takes beside the routing, gather and combine of the layer itself:

  mm      products of ragged row groups with their experts' matrices: y = x W[e]^T (forward), or
          dx = dy W[e] ("transpose", the gradient of the rows)
  wgrad   the experts' weight gradients dW[e] = dy_e^T x_e, a reduction over each group's rows
  swiglu  act = weight * silu(gate) * up on rows [gate | up], forward and backward, the backward
          with the gradient of the routing weight
  clip    the global norm of a list of gradients, and the gradients scaled to a largest norm

Rows are in expert order, group e at rows offsets[e] .. offsets[e + 1] - 1.  `own` selects the
framework's operators; otherwise `run` computes the same in 32 bits from elementary operations.
"""

import math
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one new token through the gate/up stack of the 96-expert layer: 8 rows, 8 of 96 experts read
        dict(name="mm decode 1", op="mm", tokens=1, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # a batch of 64 sequences, one token each: nearly every expert is read for about five rows
        dict(name="mm decode 64", op="mm", tokens=64, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # a training or calibration step of 4096 tokens, gate/up
        dict(name="mm gate up 4096", op="mm", tokens=4096, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # the gradient of the rows of the down projection with skewed routing (Zipf 1.2), an odd number of tokens
        dict(name="mm down grad skew", op="mm", tokens=2047, topk=8, experts=96, n=2048, k=768, skew=1.2, type="bf16",
             transpose=True),
        # the gate/up weight gradients of the 4096-token step, in the weights' type
        dict(name="wgrad gate up 4096", op="wgrad", tokens=4096, topk=8, experts=96, n=1536, k=2048, skew=0.0,
             type="bf16", out="bf16"),
        # a slice of 16 large experts (hidden 4096, intermediate 1536): down weight gradients kept in 32 bits
        dict(name="wgrad down large f32", op="wgrad", tokens=1023, topk=8, experts=16, n=4096, k=1536, skew=0.5,
             type="bf16", out="f32"),
        # the activation of a decode batch, an odd number of rows
        dict(name="swiglu small", op="swiglu", rows=509, inter=768, type="bf16", weights=False),
        # the activation of the 4096-token step, with the routing weights
        dict(name="swiglu 32768", op="swiglu", rows=32768, inter=768, type="bf16", weights=True),
        # its gradient, with that of the routing weights
        dict(name="swiglu grad 32768", op="swiglu_grad", rows=32768, inter=768, type="bf16", weights=True),
        # the gradient of a small batch with an odd width, f16
        dict(name="swiglu grad odd", op="swiglu_grad", rows=1021, inter=517, type="f16", weights=True),
        # a small model's gradients in 32 bits: 40 tensors, odd sizes among them
        dict(name="clip small f32", op="clip", tensors=40, values=1_500_001, spread=2.0, type="f32", norm=1.0),
        # expert stacks of several layers: 24 tensors of 25 million values each
        dict(name="clip stacks bf16", op="clip", tensors=24, values=604_000_000, spread=0.0, type="bf16", norm=1.0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["mm", "mm", "mm", "wgrad", "wgrad", "swiglu", "swiglu_grad", "clip"])
    if op in ("mm", "wgrad"):
        while True:
            experts = _log(rng, 1, 128)
            case = dict(op=op, tokens=_log(rng, 1, 8192), topk=min(experts, rng.randint(1, 8)), experts=experts,
                        n=8 * _log(rng, 8, 512), k=8 * _log(rng, 8, 512), skew=rng.choice([0.0, 0.0, 0.5, 1.2]),
                        type=rng.choice(["bf16", "bf16", "f16"]))
            rows = case["tokens"] * case["topk"]
            stack = case["n"] * case["k"]
            if rows * stack <= 32768 * 1536 * 2048 and experts * stack <= 96 * 1536 * 2048:
                break
        if op == "mm":
            case["transpose"] = rng.random() < 0.4
        else:
            case["out"] = rng.choice([case["type"], "f32"])
        return case
    if op in ("swiglu", "swiglu_grad"):
        inter = _log(rng, 32, 4096)
        if rng.random() < 0.75:
            inter = max(8, inter // 8 * 8)
        return dict(op=op, rows=min(_log(rng, 1, 65536), 32768 * 768 // inter), inter=inter,
                    type=rng.choice(["bf16", "bf16", "f16", "f32"]), weights=rng.random() < 0.6)
    kind = rng.choice(["bf16", "f32"])
    return dict(op="clip", tensors=rng.randint(1, 60), values=_log(rng, 1000, 300_000_000), spread=rng.choice([0.0, 1.0, 3.0]),
                type=kind, norm=rng.choice([1.0, 1.0, 1e6]))


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, kind, g, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(TYPES[kind])


def _sizes(case, seed):
    """Rows of every expert, routed as the layer routes: the top k of N(0, 1) logits with a Zipf bias."""
    r = np.random.RandomState(seed % (1 << 31))
    bias = -case["skew"] * np.log(np.arange(1, case["experts"] + 1))
    logits = r.standard_normal((case["tokens"], case["experts"])) + r.permutation(bias)
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :case["topk"]]
    return np.bincount(ids.reshape(-1), minlength=case["experts"])


def _blocks(sizes):
    """The plan of the plain form: each group cut into blocks of `height` rows, every block with its expert.
    Returns height, and as device tensors the blocks' experts, the rows of each block, which of them exist,
    and the place of every row in the blocks."""
    mean = sizes.sum() / max(1, (sizes > 0).sum())
    height = int(min(256, max(1, 2 ** math.ceil(math.log2(max(1.0, mean / 2))))))
    counts = -(-sizes // height)
    expert = np.repeat(np.arange(len(sizes)), counts)
    first = np.concatenate([[0], np.cumsum(sizes)])[:-1]
    within = np.arange(counts.sum()) - np.repeat(np.cumsum(counts) - counts, counts)
    rows = (first[expert] + within * height)[:, None] + np.arange(height)
    exists = rows < (first + sizes)[expert][:, None]
    place = np.flatnonzero(exists.reshape(-1))
    as_device = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    return as_device(expert), as_device(np.minimum(rows, sizes.sum() - 1)), as_device(exists), as_device(place)


def prepare(case, seed):
    g = _generator(seed)
    op, kind = case["op"], case["type"]
    if op in ("mm", "wgrad"):
        sizes = _sizes(case, seed)
        n, k, rows = case["n"], case["k"], int(sizes.sum())
        s = {"op": op, "sizes": sizes.tolist(),
             "offsets": torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).cuda(),
             "blocks": _blocks(sizes), "case": dict(case)}
        if op == "mm":
            s["transpose"] = bool(case.get("transpose"))
            s["x"] = _normal((rows, n if s["transpose"] else k), kind, g)
            s["w"] = _normal((case["experts"], n, k), kind, g, 0.02)
        else:
            s["dy"] = _normal((rows, n), kind, g, 0.01)
            s["x"] = _normal((rows, k), kind, g)
        return s
    if op in ("swiglu", "swiglu_grad"):
        rows, inter = case["rows"], case["inter"]
        s = {"op": op, "h": _normal((rows, 2 * inter), kind, g),
             "weights": torch.rand(rows, generator=g, device="cuda") if case["weights"] else None}
        if op == "swiglu_grad":
            s["dact"] = _normal((rows, inter), kind, g, 0.01)
        return s
    r = np.random.RandomState(case["values"] % (1 << 31))  # the tensors of a model keep their sizes
    share = np.exp(case["spread"] * r.standard_normal(case["tensors"]))
    counts = np.maximum(1, (case["values"] * share / share.sum()).astype(np.int64))
    grads = [_normal((int(c),), kind, g, 0.01) for c in counts]
    return {"op": op, "grads": grads, "out": [torch.empty_like(t) for t in grads], "norm": float(case["norm"])}


def _experts():
    """The framework's operators (its package lies beside this file's folder)."""
    if "blackhole_b200" not in sys.modules:
        sys.path.insert(0, "blackhole-harness_b200")
    from blackhole_b200 import experts
    return experts


def _mm_plain(s):
    expert, rows, _, place = s["blocks"]
    w = s["w"][expert].float()
    y = torch.matmul(s["x"].float()[rows], w if s["transpose"] else w.transpose(1, 2))
    return y.flatten(0, 1)[place].to(s["x"].dtype)


def _wgrad_plain(s):
    expert, rows, exists, _ = s["blocks"]
    case = s["case"]
    part = torch.matmul((s["dy"].float()[rows] * exists[..., None]).transpose(1, 2), s["x"].float()[rows])
    out = torch.zeros(case["experts"], case["n"], case["k"], device="cuda")
    return out.index_add_(0, expert, part).to(TYPES[case["out"]])


def _swiglu_plain(s):
    gate, up = s["h"].float().chunk(2, dim=1)
    act = gate / (1 + torch.exp(-gate)) * up
    if s["weights"] is not None:
        act = act * s["weights"][:, None]
    return act.to(s["h"].dtype)


def _swiglu_grad_plain(s):
    gate, up = s["h"].float().chunk(2, dim=1)
    d = s["dact"].float()
    sig = 1 / (1 + torch.exp(-gate))
    silu = gate * sig
    dweights = None
    if s["weights"] is not None:
        dweights = (d * silu * up).sum(1)
        d = d * s["weights"][:, None]
    dgate = d * up * (sig + silu * (1 - sig))
    return {"dh": torch.cat([dgate, d * silu], 1).to(s["h"].dtype), "dweights": dweights}


def _clip_plain(s):
    flat = torch.cat(s["grads"]).float()
    norm = flat.square().sum().sqrt()
    flat *= (s["norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "grads": list(flat.to(s["grads"][0].dtype).split([t.numel() for t in s["grads"]]))}


def run(state):
    s = state
    if not own:
        return {"mm": _mm_plain, "wgrad": _wgrad_plain, "swiglu": _swiglu_plain, "swiglu_grad": _swiglu_grad_plain,
                "clip": _clip_plain}[s["op"]](s)
    experts = _experts()
    if s["op"] == "mm":
        return experts.grouped_mm(s["x"], s["w"], s["offsets"], transpose=s["transpose"])
    if s["op"] == "wgrad":
        return experts.grouped_wgrad(s["dy"], s["x"], s["offsets"], out_dtype=TYPES[s["case"]["out"]])
    if s["op"] == "swiglu":
        return experts.swiglu(s["h"], s["weights"])
    if s["op"] == "swiglu_grad":
        dh, dweights = experts.swiglu_backward(s["dact"], s["h"], s["weights"])
        return {"dh": dh, "dweights": dweights}
    return {"norm": experts.clip_grad_norm(s["grads"], s["norm"], out=s["out"]), "grads": s["out"]}


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    op, z = case["op"], size[case["type"]]
    if op in ("mm", "wgrad"):
        rows, stack = case["tokens"] * case["topk"], case["n"] * case["k"]
        ends = rows * (case["n"] + case["k"]) * z
        if op == "mm":  # only the matrices of experts that have rows are read
            used = int((_sizes(case, 1) > 0).sum())
            return {"bytes": ends + used * stack * z, "flops": 2 * rows * stack}
        return {"bytes": ends + case["experts"] * stack * size[case["out"]], "flops": 2 * rows * stack}
    if op == "clip":
        return {"bytes": 2 * case["values"] * z, "flops": 3 * case["values"]}
    values, weights = case["rows"] * case["inter"], 4 * case["rows"] * bool(case["weights"])
    if op == "swiglu":
        return {"bytes": 3 * values * z + weights, "flops": 6 * values}
    return {"bytes": 5 * values * z + 2 * weights, "flops": 12 * values}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("mm", "wgrad"):
        ends = np.cumsum(s["sizes"])
        rows = [slice(int(end) - size, int(end)) for end, size in zip(ends, s["sizes"])]
        if op == "wgrad":
            out = torch.empty(case["experts"], case["n"], case["k"], dtype=torch.float64, device="cuda")
            for e, r in enumerate(rows):
                torch.mm(s["dy"][r].double().t(), s["x"][r].double(), out=out[e])
            return out
        parts = [s["x"][r].double() @ (s["w"][e].double() if s["transpose"] else s["w"][e].double().t())
                 for e, r in enumerate(rows) if s["sizes"][e]]
        return torch.cat(parts)
    if op == "clip":
        total = sum(float(t.double().square().sum()) for t in s["grads"])
        norm = math.sqrt(total)
        scale = min(1.0, s["norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "grads": [t.double() * scale for t in s["grads"]]}
    inter = case["inter"]
    gate, up = s["h"][:, :inter].double(), s["h"][:, inter:].double()
    weight = torch.ones(case["rows"], 1, dtype=torch.float64, device="cuda")
    if s["weights"] is not None:
        weight = s["weights"].double()[:, None]
    sig = torch.sigmoid(gate)
    if op == "swiglu":
        return weight * gate * sig * up
    d = s["dact"].double()
    dh = torch.empty(case["rows"], 2 * inter, dtype=torch.float64, device="cuda")
    dh[:, :inter] = weight * d * up * sig * (1 + gate * (1 - sig))
    dh[:, inter:] = weight * d * gate * sig
    return {"dh": dh, "dweights": (d * gate * sig * up).sum(1) if s["weights"] is not None else None}
