"""Edges of the operators of experts.py beyond test_experts.py: gates far from zero in every type, sums long enough
to lose a row in, what happens to a call that fails half way, and what autograd is told."""

from __future__ import annotations

import math
import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch
from conftest import ROOT
from test_experts import (BF16, DEV, F16, F32, ROUND, assert_sum, device_word, mm_reference, normal, offsets_of, padded,  # noqa: F401
                          swiglu_reference, wgrad_reference)

from blackhole_b200 import experts

PACKAGE = ROOT / "blackhole-harness_b200"
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


# ------------------------------------------------------------------ long sums
RUN = 2048   # the most products that one accumulator of an f32 result sums (16 at a time)


def run_bound(terms):
    """Of a sum of `terms` positive products of even size, relative.  One addition of 16 products is off by at most a unit
    in the last place (2^-23) of a sum that has grown to half on average; the runs are added in f32 (2^-24 each, on half
    the sum on average); some units for the ends."""
    return (min(terms, RUN) / 16 / 2 + 8) * 2.0 ** -23 + (terms / RUN / 2 + 1) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("hessian", [False, True])
@pytest.mark.parametrize("rows", [500, 8000, 60_000])
@pytest.mark.parametrize("E,n,k", [(1, 72, 136), (40, 256, 512), (90, 72, 264), (2, 9, 11)])
def test_f32_gradients_do_not_lose_bits_with_length(E, n, k, rows, hessian):
    """The error of a sum of one sign stays below what a lost row would take from it, however long the group: tiles alone
    and shared, x on either side, by TMA and by element."""
    if hessian:
        n = k
    sizes = [rows] + [17] * (E - 1)
    g = torch.Generator(device=DEV).manual_seed(83)
    draw = lambda width: (1 + torch.rand(sum(sizes), width, generator=g, device=DEV) / 4).to(BF16)  # noqa: E731
    x = draw(k)
    dy = x if hessian else draw(n)
    off = offsets_of(sizes).to(DEV)
    assert run_bound(rows) < 0.7 / rows
    want = dy[:rows].double().t() @ x[:rows].double()
    out = experts.grouped_wgrad(dy, x, off, out_dtype=F32)
    assert float(((out[0].double() - want).abs() / want).max()) <= run_bound(rows)
    base = torch.full_like(out, 1000.0)
    experts.grouped_wgrad(dy, x, off, out=base, accumulate=True)
    assert float(((base[0].double() - want - 1000).abs() / (want + 1000)).max()) <= run_bound(rows) + 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("rows", [3, 100, 700, 40_000])
@pytest.mark.parametrize("width", [2048, 32768, 32766])
def test_f32_row_products_do_not_lose_bits_with_width(rows, width, transpose):
    """The same along the reduction of the row products."""
    out_width = 72
    g = torch.Generator(device=DEV).manual_seed(84)
    draw = lambda *shape: (1 + torch.rand(*shape, generator=g, device=DEV) / 4).to(BF16)  # noqa: E731
    x, w = draw(rows, width), draw(2, *((width, out_width) if transpose else (out_width, width)))
    off = offsets_of([rows // 2, rows - rows // 2]).to(DEV)
    got = experts.grouped_mm(x, w, off, transpose=transpose, out_dtype=F32)
    for e, (a, b) in enumerate([(0, rows // 2), (rows // 2, rows)]):
        want = x[a:b].double() @ (w[e].double() if transpose else w[e].double().t())
        assert not len(want) or float(((got[a:b].double() - want).abs() / want).max()) <= run_bound(width)


# whole numbers: every sum is exact in f32, so a row that is lost or taken twice shows whatever the length
@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("n,k", [(72, 130), (264, 520), (88, 1336)])
@pytest.mark.parametrize("sizes", [[5000], [4000, 0, 3], [2111, 2050], [1, 15, 16, 17, 63, 64, 65, 2047, 2048, 2049, 2064, 4097],
                                   [33] * 70], ids=lambda s: f"{len(s)} groups of {s[0]}")
def test_whole_numbers_keep_every_row(sizes, n, k, out_dtype):
    g = torch.Generator().manual_seed(85)
    first, rows = 3, sum(sizes) + 70
    dy, x = (torch.randint(-3, 4, (rows, w), generator=g).float() for w in (n, k))
    dy[:first], x[:first] = math.nan, math.inf      # what no group holds
    dy[first + sum(sizes):], x[first + sum(sizes):] = math.inf, math.nan
    off = offsets_of(sizes, first)
    want, _ = wgrad_reference(dy, x, off)
    assert want.abs().max() < 2 ** 24
    dyd, xd, offd = dy.to(BF16).to(DEV), x.to(BF16).to(DEV), off.to(DEV)
    got = experts.grouped_wgrad(dyd, xd, offd, out_dtype=out_dtype)
    assert torch.equal(got.cpu(), want.to(out_dtype))
    base = torch.randint(-100, 101, want.shape, generator=g).to(out_dtype)
    out = experts.grouped_wgrad(dyd, xd, offd, out=base.to(DEV), accumulate=True)
    assert torch.equal(out.cpu(), (want + base.double()).to(out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("n,k", [(200, 2056), (2056, 200), (1000, 3004)])
@pytest.mark.parametrize("sizes", [[1], [70, 0, 1], [300, 257, 512, 2]], ids=str)
def test_whole_numbers_keep_every_column(sizes, n, k, out_dtype, transpose):
    g = torch.Generator().manual_seed(86)
    rows = sum(sizes)
    x = torch.randint(-3, 4, (rows, n if transpose else k), generator=g).float()
    w = torch.randint(-3, 4, (len(sizes), n, k), generator=g).float()
    off = offsets_of(sizes)
    want, _ = mm_reference(x, w, off, transpose, rows)
    got = experts.grouped_mm(x.to(BF16).to(DEV), w.to(BF16).to(DEV), off.to(DEV), transpose=transpose, out_dtype=out_dtype)
    assert torch.equal(got.cpu(), want.to(out_dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [BF16, F32], ids=str)
@pytest.mark.parametrize("E,rows,n,k", [(2, 70, 129, 67), (12, 700, 301, 355), (40, 1500, 77, 499), (1, 5000, 97, 131)])
def test_gradients_are_added_to_odd_rows(E, rows, n, k, out_dtype):
    """What stands in rows whose width is no multiple of 16 bytes is added to, exactly (whole numbers), and nothing beside."""
    g = torch.Generator().manual_seed(87)
    sizes = np.bincount(np.random.RandomState(E).randint(0, E, rows), minlength=E)
    dy, x = (torch.randint(-3, 4, (rows, w), generator=g).to(BF16) for w in (n, k))
    off = offsets_of(sizes)
    base = torch.randint(-100, 101, (E, n, k), generator=g).to(out_dtype)
    want = (wgrad_reference(dy, x, off)[0] + base.double()).to(out_dtype)
    buf, out = padded(base, 5.0)
    ins = padded(dy, math.nan)[1], padded(x, math.nan)[1]
    experts.grouped_wgrad(*ins, off.to(DEV), out=out, accumulate=True)
    assert torch.equal(out.cpu(), want) and (buf[..., k:] == 5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("off", [[0, 20, 10, 32], [0, 8, 16, 40], [-4, 8, 16, 32], [0, 2 ** 40, 7, 9]], ids=str)
def test_gradients_of_offsets_that_do_not_fit(off):
    """The gradient of offsets that are clamped is that of the clamped ones."""
    from blackhole_b200.hex_moe import device_status
    x, off = normal((32, 64), BF16, 88).to(DEV), torch.tensor(off)
    got = experts.grouped_wgrad(x, x, off.to(DEV), out_dtype=F32)
    assert device_status(0) == 8
    fixed = torch.cummax(off.clamp(0, 32), 0).values
    assert torch.equal(got, experts.grouped_wgrad(x, x, fixed.to(DEV), out_dtype=F32))
    want, mass = wgrad_reference(x.cpu(), x.cpu(), fixed)
    assert_sum(got, want, mass, 32, F32)


# ------------------------------------------------------------------ calls and autograd
FAILING = r"""
extern "C" int hexmoe_clip_grad_norm() { return 3; }                         // HEXMOE_E_CUDA
extern "C" const char* hexmoe_last_error() { return "a launch that failed"; }
"""


@pytest.mark.gpu
def test_a_failed_clipping_is_not_made_again(tmp_path):
    """After a launch that failed some lists may have been scaled: the call raises and is not repeated."""
    (tmp_path / "failing.cpp").write_text(FAILING)
    lib = tmp_path / "failing.so"
    subprocess.run(["g++", "-shared", "-fPIC", "-o", lib, tmp_path / "failing.cpp"], check=True)
    code = ("import torch\nfrom blackhole_b200 import experts\ng = torch.ones(4, device='cuda')\n"
            "try:\n    experts.clip_grad_norm([g], 0.5)\nexcept RuntimeError as e:\n    assert 'a launch that failed' in str(e), e\n"
            "else:\n    raise SystemExit('the call was made again')\nassert g.tolist() == [1.0] * 4, g\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=PACKAGE,
                          env={**os.environ, "LD_PRELOAD": str(lib)})
    assert done.returncode == 0, done.stdout + done.stderr


def test_the_operators_import_without_the_call_module():
    """_call.so is bound to one torch and one Python; libhexmoe.so is not, and every call has a path to it in Python."""
    code = ("import sys\nsys.modules['blackhole_b200._call'] = None\nimport torch\nfrom blackhole_b200 import experts\n"
            "try:\n    experts.swiglu(torch.zeros(2, 4))\nexcept ValueError as e:\n    assert 'CUDA' in str(e)\nelse:\n    raise SystemExit(1)\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=PACKAGE)
    assert done.returncode == 0, done.stderr


def test_the_library_builds_without_headers_of_python_and_torch():
    done = subprocess.run(["make", "-n", "-B", "PYTHON=false", "all"], capture_output=True, text=True, timeout=60, cwd=PACKAGE)
    assert done.returncode == 0 and "libhexmoe.so" in done.stdout and "call.cpp" not in done.stdout, done.stderr
    done = subprocess.run(["make", "-n", "-B", f"PYTHON={sys.executable}", "all"], capture_output=True, text=True, timeout=120, cwd=PACKAGE)
    assert done.returncode == 0 and "call.cpp" in done.stdout, done.stderr


@pytest.mark.gpu
def test_calls_without_the_call_module_are_the_same(monkeypatch):
    off = offsets_of([40, 0, 88]).to(DEV)
    x, w, dy = normal((128, 72), BF16, 89).to(DEV), normal((3, 136, 72), BF16, 90).to(DEV), normal((128, 136), BF16, 91).to(DEV)
    weight, grads = torch.rand(128, device=DEV), [normal((300, 7), F32, 92).to(DEV), normal((9,), BF16, 93).to(DEV)]

    def calls():
        out = [torch.empty_like(t) for t in grads]
        norm = experts.clip_grad_norm(grads, 1.0, out=out)
        return [experts.grouped_mm(x, w, off), experts.grouped_mm(dy, w, off, transpose=True), experts.grouped_wgrad(dy, x, off),
                experts.grouped_wgrad(dy, x, off, out_dtype=F32), experts.swiglu(dy, weight),
                *experts.swiglu_backward(dy[:, :68].contiguous(), dy, weight), norm, *out]

    with_it = calls()
    none = type("none", (), {name: staticmethod(lambda *args: None) for name in
                             ("grouped_mm", "grouped_wgrad", "swiglu", "swiglu_backward", "clip_grad_norm")})
    monkeypatch.setattr(experts, "_call", none)
    assert all(torch.equal(a, b) for a, b in zip(with_it, calls(), strict=True))


@pytest.mark.gpu
def test_autograd_sees_what_is_written():
    """A tensor that is written to has a new version, so that a backward pass that kept its old values refuses them."""
    off = offsets_of([40, 0, 88]).to(DEV)
    x, w, dy = normal((128, 72), BF16, 94).to(DEV), normal((3, 136, 72), BF16, 95).to(DEV), normal((128, 136), BF16, 96).to(DEV)
    wide, grads = torch.zeros(128, 140, dtype=BF16, device=DEV), [torch.ones(9, device=DEV), torch.ones(5, dtype=BF16, device=DEV)]
    strided = torch.ones(6, 8, device=DEV)[:, :5]
    with torch.inference_mode():
        kept = torch.ones(4, device=DEV)
    cases = [([wide], lambda: experts.grouped_mm(x, w, off, out=wide[:, :136])),
             ([w], lambda: experts.grouped_wgrad(dy, x, off, out=w, accumulate=True)),
             ([dy], lambda: experts.swiglu_backward(dy[:, :68].contiguous(), dy, out=dy)),
             (grads, lambda: experts.clip_grad_norm(grads, 1.0)), ([strided], lambda: experts.clip_grad_norm([strided], 1.0)),
             (grads, lambda: experts.clip_grad_norm([torch.ones_like(t) for t in grads], 1.0, out=grads))]
    for written, call in cases:
        before = [t._version for t in written]
        call()
        assert all(t._version > v for t, v in zip(written, before))
    experts.clip_grad_norm([kept], 1.0)      # a tensor without versions
    assert float(kept.norm()) < 1.01
    source = [torch.ones(9, device=DEV)]
    experts.clip_grad_norm(source, 1.0, out=[torch.empty(9, device=DEV)])
    assert source[0]._version == 0           # only read
    leaf = torch.zeros(9, device=DEV, requires_grad=True)
    held = leaf.exp()
    experts.clip_grad_norm([held.detach()], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        held.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["grouped_mm", "transpose", "grouped_wgrad"])
def test_a_product_may_be_a_threads_first_call(name):
    """A host thread that has launched nothing has no CUDA context of its own (autograd's and a server's worker threads)."""
    off = offsets_of([40, 0, 88]).to(DEV)
    x, w, dy = normal((128, 72), BF16, 104).to(DEV), normal((3, 136, 72), BF16, 105).to(DEV), normal((128, 136), BF16, 106).to(DEV)
    call = {"grouped_mm": lambda: experts.grouped_mm(x, w, off), "transpose": lambda: experts.grouped_mm(dy, w, off, transpose=True),
            "grouped_wgrad": lambda: experts.grouped_wgrad(dy, x, off)}[name]
    want = call().clone()     # and its memory is at hand: the thread's call allocates nothing from the driver
    torch.cuda.synchronize()
    with ThreadPoolExecutor(1) as pool:
        got = pool.submit(call).result()
    assert torch.equal(got, want)


def grads_of(call, *inputs):
    """The call's result, its gradient for a drawn one of the result, and that."""
    leaves = [t.detach().clone().requires_grad_() for t in inputs]
    out = call(*leaves)
    assert out.requires_grad
    d = normal(tuple(out.shape), out.dtype, 97).to(DEV)
    return [out.detach(), *torch.autograd.grad(out, leaves, d)], d


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [None, F32], ids=str)
def test_operators_inside_a_graph(out_dtype):
    """Called on inputs that require grad, the operators hand on gradients: those of the operators themselves."""
    sizes = [40, 0, 88]
    off = offsets_of(sizes).to(DEV)
    x, w, dy = normal((130, 72), BF16, 98).to(DEV), normal((3, 136, 72), BF16, 99, 0.1).to(DEV), normal((130, 136), BF16, 100).to(DEV)
    (y, dx, dw), d = grads_of(lambda a, b: experts.grouped_mm(a, b, off, out_dtype=out_dtype), x, w)
    d = d.to(BF16)
    assert torch.equal(y, experts.grouped_mm(x, w, off, out_dtype=out_dtype)) and dx.dtype == dw.dtype == BF16
    assert torch.equal(dx, experts.grouped_mm(d, w, off, transpose=True)) and torch.equal(dw, experts.grouped_wgrad(d, x, off))
    want, mass = wgrad_reference(d.cpu(), x.cpu(), off.cpu())
    assert_sum(dw, want, mass, max(sizes), BF16)
    (y, dx, dw), d = grads_of(lambda a, b: experts.grouped_mm(a, b, off, transpose=True, out_dtype=out_dtype), dy, w)
    d = d.to(BF16)
    assert torch.equal(dx, experts.grouped_mm(d, w, off)) and torch.equal(dw, experts.grouped_wgrad(dy, d, off))
    want, mass = mm_reference(d.cpu(), w.cpu(), off.cpu(), False, 130)
    assert_sum(dx, want, mass, 72, BF16)
    (dw, ddy, dx), g = grads_of(lambda a, b: experts.grouped_wgrad(a, b, off, out_dtype=out_dtype), dy, x)
    g = g.to(BF16)
    assert torch.equal(ddy, experts.grouped_mm(x, g, off)) and torch.equal(dx, experts.grouped_mm(dy, g, off, transpose=True))
    # one of the inputs alone, and one input twice: H = x^T x has the gradient x (G + G^T)
    leaf = x.clone().requires_grad_()
    experts.grouped_mm(leaf, w, off).float().sum().backward()
    assert torch.equal(leaf.grad, experts.grouped_mm(torch.ones_like(dy), w, off, transpose=True))
    (h, dx), g = grads_of(lambda a: experts.grouped_wgrad(a, a, off, out_dtype=F32), x)
    want, mass = mm_reference(x.cpu(), (g.to(BF16).double() + g.to(BF16).double().transpose(1, 2)).cpu(), off.cpu(), False, 130)
    # two products, each rounded to bf16, and their sum
    both, mass2 = mm_reference(x.cpu().abs(), (g.abs().double() + g.abs().double().transpose(1, 2)).cpu(), off.cpu(), False, 130)
    assert ((dx.double().cpu() - want).abs() <= 3 * 2.0 ** -8 * mass2).all()


@pytest.mark.gpu
def test_swiglu_inside_a_graph():
    h, weight = normal((50, 96), BF16, 101).to(DEV), torch.rand(50, device=DEV)
    (act, dh, dw), d = grads_of(experts.swiglu, h, weight)
    assert torch.equal(act, experts.swiglu(h, weight))
    assert all(torch.equal(a, b) for a, b in zip((dh, dw), experts.swiglu_backward(d, h, weight)))
    (act, dh), d = grads_of(experts.swiglu, h)
    assert torch.equal(dh, experts.swiglu_backward(d, h)[0])
    leaf = weight.clone().requires_grad_()
    experts.swiglu(h, leaf).float().sum().backward()
    assert torch.equal(leaf.grad, experts.swiglu_backward(torch.ones_like(d), h, weight)[1])


@pytest.mark.gpu
def test_calls_outside_the_graph():
    """Without grad mode nothing is recorded; a product into `out` says that it cannot be; sums in `out` are not."""
    off = offsets_of([40, 0, 88]).to(DEV)
    x, w = normal((128, 72), BF16, 102).to(DEV).requires_grad_(), normal((3, 136, 72), BF16, 103).to(DEV)
    out, h = torch.empty(128, 136, dtype=BF16, device=DEV), torch.zeros(3, 72, 72, device=DEV)
    with pytest.raises(RuntimeError, match="requires grad"):
        experts.grouped_mm(x, w, off, out=out)
    assert experts.grouped_wgrad(x, x, off, out=h, accumulate=True) is h and not h.requires_grad
    with torch.no_grad():
        assert not experts.grouped_mm(x, w, off).requires_grad and not experts.grouped_mm(x, w, off, out=out).requires_grad
        assert torch.equal(h, experts.grouped_wgrad(x, x, off, out_dtype=F32))
    assert not experts.grouped_mm(x.detach(), w, off).requires_grad


@pytest.mark.gpu
def test_the_library_alone_plans_the_workspace(monkeypatch):
    """Whatever the size, the library is asked, and gets what it asks for: no rule of its plan is kept on this side."""
    from blackhole_b200 import _lib
    sizes = [3] * 120
    off, asked, given = offsets_of(sizes).to(DEV), [], []
    x, dy = normal((360, 264), BF16, 107).to(DEV), normal((360, 520), BF16, 108).to(DEV)
    w = normal((120, 520, 264), BF16, 109).to(DEV)
    want = experts.grouped_mm(x, w, off), experts.grouped_wgrad(dy, x, off)
    for name in ("hexmoe_grouped_mm_workspace_bytes", "hexmoe_grouped_wgrad_workspace_bytes"):
        monkeypatch.setattr(_lib.lib, name, lambda *args: asked.append(args) or 4096)
    held = experts._workspace
    monkeypatch.setattr(experts, "_workspace", lambda nbytes, like: given.append(nbytes) or held(nbytes, like))
    outs = torch.empty_like(want[0]), torch.empty_like(want[1])
    experts.grouped_mm(x, w, off, out=outs[0])
    experts.grouped_wgrad(dy, x, off, out=outs[1])
    assert [a[:4] for a in asked] == [(360, 120, 520, 264)] * 2 and given == [4096] * 2
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
def test_clipping_does_not_look_at_strides_of_single_entries():
    """The stride of a dimension of one entry, or of a tensor without values, says nothing about where values stand."""
    base, into = normal((4, 6), F32, 110).to(DEV), torch.full((4, 6), 9.0, device=DEV)
    grads = [base.as_strided((1, 4, 1, 3), (0, 6, 0, 2)), torch.empty(0, 6, device=DEV)[:, ::2]]
    out = [into.as_strided((1, 4, 1, 3), (7, 6, 1, 2)), torch.empty(0, 3, device=DEV)]
    part = base[:, ::2].clone()
    norm = experts.clip_grad_norm(grads, 1.0, out=out)
    assert abs(float(norm) - float(part.double().norm())) <= 2.0 ** -22 * float(norm)
    torch.testing.assert_close(into[:, ::2], part / part.norm(), rtol=1e-5, atol=0)
    assert (into[:, 1::2] == 9).all() and torch.equal(base[:, ::2], part)
    assert torch.equal(experts.clip_grad_norm(grads, 1.0), norm) and torch.equal(base[:, ::2], into[:, ::2])
    with pytest.raises(ValueError, match="strides"):
        experts.clip_grad_norm([base[:, ::2]], 1.0, out=[torch.empty(4, 3, device=DEV)])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 1])
def test_swiglu_backward_into_a_single_row(rows):
    """A single row has no row stride to be refused for."""
    h, dact, weight = normal((rows, 48), BF16, 111).to(DEV), normal((rows, 24), BF16, 112).to(DEV), torch.rand(rows, device=DEV)
    out = torch.zeros(48, dtype=BF16, device=DEV).as_strided((rows, 48), (1, 1))
    dh, dw = experts.swiglu_backward(dact, h, weight, out=out)
    want = experts.swiglu_backward(dact, h, weight)
    assert dh is out and torch.equal(dh, want[0]) and torch.equal(dw, want[1])
