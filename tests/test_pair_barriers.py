"""Barriers by which one CTA of a pair gives shared memory back to the other order what was read before what is written next.

No run shows it when they do not (a slot that is read late has to be overtaken by a store from the other CTA): the sources are read.
"""
import re
from pathlib import Path

KERNELS = Path(__file__).resolve().parent.parent / "csrc" / "kernels"
SOURCES = {path.name: path.read_text() for path in sorted([*KERNELS.glob("*.cu"), *KERNELS.glob("*.cuh")])}


def body(text, name):
    """A function's, from its name to the brace that closes it."""
    start = text.index("{", re.search(rf"\b{name}\(const Shared& s, (?:uint32_t rank, )?Ring&", text).start())
    return text[start:text.index("\n}\n", start)]


def test_arrivals_without_memory_are_for_accumulators():
    uses = [(name, line) for name, text in SOURCES.items() for line in text.splitlines() if "mbar_arrive_only(" in line and "void mbar_arrive_only" not in line]
    assert len(uses) >= 2
    for name, line in uses:
        assert re.search(r"mbar_arrive_only\(.*\bacc_empty\[", line), f"{name}: {line.strip()}"


def test_slots_of_tasks_change_hands_in_the_cluster():
    text = SOURCES["linear_ce.cu"]
    tell, read = (body(text, name) for name in ("tell_task", "read_task"))
    # written in both CTAs: what is waited for before, and told behind, reaches as far
    assert tell.index("warp_wait<true>(&s.task_empty[") < tell.index("store_cluster(") < tell.index("mbar_arrive_at(cluster_address(&s.task_full[")
    # read, and given back: rank 0, which waits for it, has its own warps in its CTA; the others' reads have to be ordered across CTAs
    assert read.index("warp_wait<true>(&s.task_full[") < read.index("s.task[ring.stage]") < read.index("__syncwarp()") < read.index("if (rank == 0)")
    assert re.search(r"if \(rank == 0\) mbar_arrive\(&s\.task_empty\[ring\.stage\]\);\s*else mbar_arrive_at\(rank0_address\(&s\.task_empty\[", read)
    header = SOURCES["ptx_sm100.cuh"]
    for instruction in ("mbarrier.arrive.release.cta.shared::cta", "mbarrier.arrive.release.cluster.shared::cluster", "mbarrier.try_wait.parity.acquire.cluster.shared::cta"):
        assert instruction in header
    assert re.search(r"CLUSTER \? mbar_try_wait_cluster\(bar, parity\) : mbar_try_wait\(bar, parity\)", text)
