"""What the pair kernel's warps owe one another, read from its source: faults here would show as a hang or
as a race, which no run may be made to show."""

from __future__ import annotations

import re

from conftest import ROOT

CSRC = ROOT / "blackhole-harness_b200" / "csrc"


def kernel_lines():
    """The lines of grouped_pair_kernel, without comments."""
    src = (CSRC / "grouped.cu").read_text()
    body = src[src.index("grouped_pair_kernel(const __grid_constant__"):src.index("encode_fn()")]
    return [re.sub(r"//.*", "", line) for line in body.splitlines()]


def test_a_warp_gives_up_as_one():
    """Lanes that disagree on a wait that ran out must not part ways before a warp-wide operation: every wait
    of a whole warp votes, and a bare wait stands only where a single lane runs."""
    lines = kernel_lines()
    bare = [i for i, line in enumerate(lines) if re.search(r"(?<!\w)mbar_wait\(", line)]
    for i in bare:
        assert any("lane == 0" in line for line in lines[max(0, i - 5):i]), lines[i]
    assert sum("warp_wait(" in line for line in lines) >= 5
    helper = (CSRC / "pair.cuh").read_text()
    assert re.search(r"bool warp_wait\([^{]*\{\s*return __all_sync\(0xffffffffu, mbar_wait\(", helper)


def test_a_kernel_that_gives_up_waits_for_its_copies():
    """After a wait that ran out neither CTA may leave while copies still land in its shared memory: the leader, on whose
    barriers both CTAs' copies complete, waits for the steps and for the tails."""
    text = "\n".join(kernel_lines())
    for barrier, guard in (("full", r"\*abort && lane == 0 && leader"), ("tail", r"\*abort && lane == 0 && leader")):
        assert re.search(guard + r"[^}]*mbar_wait\(&c->" + barrier + r"\[[^}]*&ignore", text), barrier


def test_shared_arrays_read_as_words_are_aligned():
    """An array of 16-bit elements is only sure of 2 bytes: one that is read as wider words says its alignment."""
    for name in ("grouped.cu", "train.cu"):
        src = re.sub(r"//.*", "", (CSRC / name).read_text())
        for line in re.findall(r"(?<!extern )__shared__[^;]*\buint(?:8|16)_t\b[^;]*;", src):
            assert "__align__(16)" in line, line


def test_zeroed_rows_are_published_to_the_product():
    """The rows that are cleared are read by a product that the leader issues.  No arrival here releases to the other CTA,
    so the leader's warps clear them in both, behind copies that complete in the leader, and arrive in the leader."""
    text = "\n".join(kernel_lines())
    assert ".release.cluster" not in (CSRC / "pair.cuh").read_text().split("cluster_sync")[1].split("}", 1)[1]
    assert re.search(r"peer_addr\(fix \? &c->tail\[st\] : &c->full\[st\], 0\)", text)
    role = text[text.index("(warp == 2 || warp == 3) && MODE >= kWgrad && leader"):text.index("warp >= 4")]
    assert re.search(r"warp_wait\(&c->tail\[st\].*pair_store_zeros.*if \(cta == 0\) fence_proxy_async_smem\(\);\s*"
                     r"else fence_proxy_async\(\);\s*__syncwarp\(\);\s*if \(ok && lane == 0\) mbar_arrive\(&c->full\[st\]\)", role, re.S)
