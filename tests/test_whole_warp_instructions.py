"""Barriers and allocations in inline PTX that need all lanes of a warp at once bring their warp barrier along.

Where one lane took a branch before (a barrier set up, a sum handed over), nothing else promises that the others have not gone ahead. Whether they do is the
compiler's choice, so no run shows it: the sources are read.
"""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "csrc"
NEEDS = re.compile(r'"[^"]*\b(barrier\.cluster\.arrive[\w.:]*\.aligned|tcgen05\.(?:alloc|dealloc)\.[\w.:]+|bar\.(?:sync|red|arrive)|barrier\.(?:cta\.)?(?:sync|red)[\w.:]*\.aligned)')


def functions_with_them():
    for path in sorted([*CSRC.rglob("*.cuh"), *CSRC.rglob("*.cu")]):
        text = path.read_text()
        for m in NEEDS.finditer(text):
            start = max(text.rfind("__device__", 0, m.start()), text.rfind("__global__", 0, m.start()))
            yield path.name, m.group(1), text[start:m.start()]


def test_every_one_of_them_is_found():
    found = [f"{name}: {what}" for name, what, _ in functions_with_them()]
    assert len(found) >= 6, found  # the cluster's barrier, tensor memory taken and given back by one CTA and by a pair, a row's barrier


def test_a_warp_barrier_comes_first():
    for name, what, before in functions_with_them():
        assert "__syncwarp()" in before, f"{name}: {what} without a warp barrier before it"
