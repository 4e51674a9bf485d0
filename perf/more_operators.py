"""The router of a MoE layer and its experts in 8-bit integers, as they are measured.

  route       every token's k experts: softmax or sigmoid scores, a bias that balances the choice, groups of
              which a token may use a few, the weights renormalised and scaled
  route_grad  the gradient of the logits for that of the weights
  mm8         products of ragged row groups with their experts' 8-bit matrices, the rows quantized on the way:
              q = round(127 x / max |x|) of every row, y[r, n] = x_scale[r] w_scale[e, n] sum_k q[r, k] w[e, n, k]
  moe8        a SwiGLU layer of such experts on routed tokens, the activation quantized per row as well

The order of experts, groups and 8-bit values is decided in 64 bits: a border that 32 bits miss gives another
whole number.  `own` selects the framework's operators; otherwise `run` computes the same from elementary operations.
"""

import math
import sys

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one new token among 256 experts in 8 groups, four of them open to it: sigmoid scores with the balancing bias
        dict(name="route 1 sigmoid groups", op="route", tokens=1, experts=256, topk=8, scoring="sigmoid", bias=True, groups=8,
             topk_groups=4, group_top=2, renormalize=True, scale=2.5, type="f32"),
        # a prefill of 8192 tokens through the same router
        dict(name="route 8192 sigmoid groups", op="route", tokens=8192, experts=256, topk=8, scoring="sigmoid", bias=True,
             groups=8, topk_groups=4, group_top=2, renormalize=True, scale=2.5, type="f32"),
        # the 96-expert layer's softmax router on 4096 tokens with a balancing bias, 16-bit logits
        dict(name="route 4096 softmax bias", op="route", tokens=4096, experts=96, topk=8, scoring="softmax", bias=True, groups=1,
             topk_groups=1, group_top=2, renormalize=True, scale=1.0, type="bf16"),
        # a training step's gradient of the 96-expert router: 4096 tokens, plain softmax weights
        dict(name="route grad 4096 softmax", op="route_grad", tokens=4096, experts=96, topk=8, scoring="softmax", bias=False,
             groups=1, topk_groups=1, group_top=1, renormalize=False, scale=1.0, type="f32"),
        # the gradient of an odd number of tokens through the router with groups
        dict(name="route grad 8191 sigmoid", op="route_grad", tokens=8191, experts=256, topk=8, scoring="sigmoid", bias=True,
             groups=8, topk_groups=4, group_top=2, renormalize=True, scale=2.5, type="f32"),
        # one new token through the gate/up stack of the 96-expert layer: 8 rows, 8 of 96 experts read
        dict(name="mm8 decode 1", op="mm8", tokens=1, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # a batch of 64 sequences, one token each
        dict(name="mm8 decode 64", op="mm8", tokens=64, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # a prefill of 4096 tokens, gate/up
        dict(name="mm8 gate up 4096", op="mm8", tokens=4096, topk=8, experts=96, n=1536, k=2048, skew=0.0, type="bf16"),
        # the down projection with skewed routing (Zipf 1.2), an odd number of tokens, f16
        dict(name="mm8 down skew", op="mm8", tokens=2047, topk=8, experts=96, n=2048, k=768, skew=1.2, type="f16"),
        # a decode step of 16 sequences through the whole layer
        dict(name="moe8 decode 16", op="moe8", tokens=16, topk=8, experts=96, hidden=2048, inter=768, skew=0.0, type="bf16"),
        # a prefill of 4096 tokens through the whole layer
        dict(name="moe8 4096", op="moe8", tokens=4096, topk=8, experts=96, hidden=2048, inter=768, skew=0.0, type="bf16"),
        # a slice of 16 large experts on a ragged batch
        dict(name="moe8 large experts 1023", op="moe8", tokens=1023, topk=8, experts=16, hidden=4096, inter=1536, skew=0.5,
             type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "route", "route_grad", "mm8", "mm8", "moe8", "moe8"])
    if op in ("route", "route_grad"):
        groups = rng.choice([1, 1, 2, 4, 8, 8, 12, 16])
        experts = max(groups, _log(rng, 4, 512) // groups * groups)
        open_groups = rng.randint(1, groups)
        topk = rng.randint(1, min(16, experts // groups * open_groups))
        return dict(op=op, tokens=_log(rng, 1, 8192 * 256 // max(256, experts)), experts=experts, topk=topk,
                    scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6, groups=groups, topk_groups=open_groups,
                    group_top=rng.choice([1, 2]), renormalize=topk > 1 and rng.random() < 0.7,   # one weight alone is 1
                    scale=rng.choice([1.0, 2.5]), type=rng.choice(["f32", "f32", "bf16", "f16"]))
    while True:
        experts = _log(rng, 1, 128)
        case = dict(op=op, tokens=_log(rng, 1, 8192), topk=min(experts, rng.randint(1, 8)), experts=experts)
        rows = case["tokens"] * case["topk"]
        if op == "mm8":
            k = 16 * _log(rng, 4, 256)
            case |= dict(n=8 * _log(rng, 8, 512), k=k if rng.random() < 0.75 else k + rng.randint(1, 15))
            stack, most = case["n"] * case["k"], 1536 * 2048
        else:
            case |= dict(hidden=32 * _log(rng, 4, 128), inter=16 * _log(rng, 4, 128))
            stack, most = case["hidden"] * case["inter"], 2048 * 768
        case |= dict(skew=rng.choice([0.0, 0.0, 0.5, 1.2]), type=rng.choice(["bf16", "bf16", "f16"]))
        if rows * stack <= 32768 * most and experts * stack <= 96 * most:
            return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ids(case, seed):
    """Every token's experts, routed as the layer routes: the top k of N(0, 1) logits with a Zipf bias."""
    r = np.random.RandomState(seed % (1 << 31))
    bias = -case["skew"] * np.log(np.arange(1, case["experts"] + 1))
    logits = r.standard_normal((case["tokens"], case["experts"])) + r.permutation(bias)
    return np.argsort(-logits, axis=1, kind="stable")[:, :case["topk"]]


def _sizes(case, seed):
    return np.bincount(_ids(case, seed).reshape(-1), minlength=case["experts"])


def _on_device(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _blocks(sizes):
    """The plan of the plain form: each group cut into blocks of `height` rows, every block with its expert.
    Returns as device tensors the blocks' experts, the rows of each block, and the place of every row in them."""
    mean = sizes.sum() / max(1, (sizes > 0).sum())
    height = int(min(256, max(1, 2 ** math.ceil(math.log2(max(1.0, mean / 2))))))
    counts = -(-sizes // height)
    expert = np.repeat(np.arange(len(sizes)), counts)
    first = np.concatenate([[0], np.cumsum(sizes)])[:-1]
    within = np.arange(counts.sum()) - np.repeat(np.cumsum(counts) - counts, counts)
    rows = (first[expert] + within * height)[:, None] + np.arange(height)
    place = np.flatnonzero((rows < (first + sizes)[expert][:, None]).reshape(-1))
    return _on_device(expert), _on_device(np.minimum(rows, sizes.sum() - 1)), _on_device(place)


def _stack8(experts, n, k, g):
    """A stack of N(0, 0.02) matrices in 8 bits with a scale for each of their rows, on a row pitch of whole
    16 bytes as quantize_rows lays it out."""
    q = torch.zeros(experts, n, (k + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :, :k]
    scale = torch.empty(experts, n, device="cuda")
    for e in range(experts):
        w = torch.randn(n, k, generator=g, device="cuda") * 0.02
        largest = w.abs().amax(1)
        q[e] = torch.round(w.double() * 127 / largest.double()[:, None]).to(torch.int8)
        scale[e] = largest / 127
    return q, scale


def prepare(case, seed):
    g = _generator(seed)
    op, kind = case["op"], TYPES[case["type"]]
    s = {"op": op, "case": dict(case)}
    if op in ("route", "route_grad"):
        T, E = case["tokens"], case["experts"]
        s["logits"] = (torch.randn(T, E, generator=g, device="cuda") * 1.5).to(kind)
        s["bias"] = torch.randn(E, generator=g, device="cuda") * 0.1 if case["bias"] else None
        if op == "route_grad":
            s["ids"] = _route_plain(s)["ids"]
            s["dweights"] = torch.randn(T, case["topk"], generator=g, device="cuda") * 0.01
        return s
    ids = _ids(case, seed)
    sizes = np.bincount(ids.reshape(-1), minlength=case["experts"])
    s["sizes"], s["blocks"] = sizes.tolist(), _blocks(sizes)
    if op == "mm8":
        s["offsets"] = _on_device(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32))
        s["x"] = torch.randn(int(sizes.sum()), case["k"], generator=g, device="cuda").to(kind)
        s["w"], s["w_scale"] = _stack8(case["experts"], case["n"], case["k"], g)
        return s
    s["x"] = torch.randn(case["tokens"], case["hidden"], generator=g, device="cuda").to(kind)
    weights = torch.rand(case["tokens"], case["topk"], generator=g, device="cuda") + 0.1
    s["weights"], s["ids"] = weights / weights.sum(1, keepdim=True), _on_device(ids.astype(np.int32))
    s["order"] = _on_device(np.argsort(ids.reshape(-1), kind="stable"))     # the slot of every row in expert order
    s["w13"], s["s13"] = _stack8(case["experts"], 2 * case["inter"], case["hidden"], g)
    s["w2"], s["s2"] = _stack8(case["experts"], case["hidden"], case["inter"], g)
    return s


def _framework():
    """The framework's operators (its package lies beside this file's folder)."""
    if "blackhole_b200" not in sys.modules:
        sys.path.insert(0, "blackhole-harness_b200")
    from blackhole_b200 import int8, router
    return int8, router


def _scores(s):
    logits = s["logits"].double()
    return 1 / (1 + torch.exp(-logits)) if s["case"]["scoring"] == "sigmoid" else torch.softmax(logits, 1)


def _route_plain(s):
    case = s["case"]
    T, E, G = case["tokens"], case["experts"], case["groups"]
    scores = _scores(s)
    biased = scores if s["bias"] is None else scores + s["bias"].double()
    choice = s["logits"].double() if s["bias"] is None else biased      # without a bias the logits have the scores' order
    if G > 1:
        best = biased.view(T, G, E // G).sort(2, descending=True).values[:, :, :case["group_top"]].sum(2)
        shut = best.sort(dim=1, descending=True, stable=True).indices[:, case["topk_groups"]:]
        choice = choice.view(T, G, E // G).scatter(1, shut[:, :, None].expand(-1, -1, E // G), -math.inf).view(T, E)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :case["topk"]]
    weights = scores.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    return {"weights": (weights * case["scale"]).float(), "ids": ids.int()}


def _route_grad_plain(s):
    case, ids, scores = s["case"], s["ids"].long(), _scores(s)    # 64 bits: a few large scores leave small differences
    chosen, d = scores.gather(1, ids), s["dweights"].double() * case["scale"]
    if case["renormalize"]:
        total = chosen.sum(1, keepdim=True)
        d = (d - (d * chosen).sum(1, keepdim=True) / total) / total
    d = torch.zeros_like(scores).scatter_(1, ids, d)
    if case["scoring"] == "sigmoid":
        return (d * scores * (1 - scores)).to(s["logits"].dtype)
    return (scores * (d - (d * scores).sum(1, keepdim=True))).to(s["logits"].dtype)


def _quantized(x):
    """The rows of x as whole numbers in 32 bits, and their scales."""
    largest = x.abs().amax(1, keepdim=True)
    return torch.round(x.double() * 127 / largest.double().clamp(min=1e-300)).float(), largest / 127


def _product_plain(q, scale, w, w_scale, blocks):
    """Quantized rows in expert order times their expert's matrix."""
    expert, rows, place = blocks
    y = torch.matmul(q[rows], w[expert].float().transpose(1, 2)) * w_scale[expert][:, None]
    return y.flatten(0, 1)[place] * scale


def _mm8_plain(s):
    return _product_plain(*_quantized(s["x"].float()), s["w"], s["w_scale"], s["blocks"]).to(s["x"].dtype)


def _moe8_plain(s):
    (T, k), order = s["ids"].shape, s["order"]
    q, scale = _quantized(s["x"].float())
    rows = order // k
    gate, up = _product_plain(q[rows], scale[rows], s["w13"], s["s13"], s["blocks"]).chunk(2, dim=1)
    y = _product_plain(*_quantized(gate / (1 + torch.exp(-gate)) * up), s["w2"], s["s2"], s["blocks"])
    slots = torch.empty_like(y).index_copy_(0, order, y * s["weights"].reshape(-1)[order][:, None])
    return slots.view(T, k, -1).sum(1).to(s["x"].dtype)


def run(state):
    s = state
    if not own:
        return {"route": _route_plain, "route_grad": _route_grad_plain, "mm8": _mm8_plain, "moe8": _moe8_plain}[s["op"]](s)
    int8, router = _framework()
    case = s["case"]
    if s["op"] == "route":
        weights, ids = router.route(s["logits"], case["topk"], scoring=case["scoring"], bias=s["bias"], groups=case["groups"],
                                    topk_groups=case["topk_groups"], group_top=case["group_top"],
                                    renormalize=case["renormalize"], scale=case["scale"])
        return {"weights": weights, "ids": ids}
    if s["op"] == "route_grad":
        return router.route_backward(s["dweights"], s["logits"], s["ids"], scoring=case["scoring"],
                                     renormalize=case["renormalize"], scale=case["scale"])
    if s["op"] == "mm8":
        return int8.grouped_mm_int8(s["x"], s["w"], s["w_scale"], s["offsets"])
    return int8.int8_moe(s["x"], s["weights"], s["ids"], s["w13"], s["s13"], s["w2"], s["s2"])


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    op, z = case["op"], size[case["type"]]
    if op in ("route", "route_grad"):
        values, slots = case["tokens"] * case["experts"], case["tokens"] * case["topk"]
        if op == "route":
            return {"bytes": values * z + 4 * case["experts"] * case["bias"] + 8 * slots, "flops": 8 * values}
        dense = case["scoring"] == "softmax" and not case["renormalize"]    # else the chosen logits are enough
        return {"bytes": values * z * (2 if dense else 1) + slots * (8 if dense else 8 + z), "flops": 8 * values}
    used, rows = int((_sizes(case, 1) > 0).sum()), case["tokens"] * case["topk"]    # only experts that have rows are read
    if op == "mm8":
        n, k = case["n"], case["k"]
        return {"bytes": rows * (n + k) * z + used * n * (k + 4), "flops": 2 * rows * n * k}
    H, I = case["hidden"], case["inter"]
    return {"bytes": 2 * case["tokens"] * H * z + 8 * rows + used * (3 * I * H + 4 * (2 * I + H)), "flops": 6 * rows * I * H}


def _exact_rows(x):
    x = x.double()
    scale = torch.max(x.abs(), dim=1, keepdim=True).values
    return torch.where(scale > 0, x * 127 / scale, 0).round(), scale / 127


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        logits, E = s["logits"].double(), case["experts"]
        scores = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else (logits - logits.logsumexp(1, keepdim=True)).exp()
        biased = scores.clone()
        if case["bias"]:
            biased += s["bias"].double()
        per = E // case["groups"]
        groups = biased.view(-1, case["groups"], per)
        value = groups.topk(min(case["group_top"], per), dim=2).values.sum(2)
        # a group is open where fewer than topk_groups others come before it
        index = torch.arange(case["groups"], device="cuda")
        ahead = (value[:, None, :] > value[:, :, None]) | (
            (value[:, None, :] == value[:, :, None]) & (index[None, None, :] < index[None, :, None]))
        is_open = (ahead.sum(2) < case["topk_groups"]).repeat_interleave(per, dim=1)
        rank = torch.where(is_open, biased if case["bias"] else logits, -math.inf)
        picked = torch.argsort(rank, dim=1, descending=True, stable=True)[:, :case["topk"]]
        weights = torch.take_along_dim(scores, picked, 1)
        if case["renormalize"]:
            weights /= weights.sum(1, keepdim=True)
        return {"weights": weights * case["scale"], "ids": picked.int()}
    if op == "route_grad":
        logits = s["logits"].double().requires_grad_()
        scores = torch.sigmoid(logits) if case["scoring"] == "sigmoid" else torch.softmax(logits, 1)
        weights = torch.take_along_dim(scores, s["ids"].long(), 1)
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True)
        (weights * case["scale"] * s["dweights"].double()).sum().backward()
        return logits.grad
    ends = np.cumsum(s["sizes"])
    if op == "mm8":
        q, scale = _exact_rows(s["x"])
        parts = [q[end - size:end] @ s["w"][e].double().t() * s["w_scale"][e].double()
                 for e, (end, size) in enumerate(zip(ends, s["sizes"])) if size]
        return torch.cat(parts) * scale
    q, scale = _exact_rows(s["x"])
    out = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    for e, (end, size) in enumerate(zip(ends, s["sizes"])):
        if not size:
            continue
        slots = s["order"][end - size:end]
        token = slots // case["topk"]
        h = q[token] @ s["w13"][e].double().t() * s["s13"][e].double() * scale[token]
        gate, up = h[:, :case["inter"]], h[:, case["inter"]:]
        a, a_scale = _exact_rows(gate * torch.sigmoid(gate) * up)
        y = a @ s["w2"][e].double().t() * s["s2"][e].double() * a_scale
        out.index_add_(0, token, y * s["weights"].double().reshape(-1)[slots][:, None])
    return out
