"""Block-scaled e4m3 linears and the norms around them: what can be held to without a GPU."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fastworld_b200", "csrc")


def source(name):
    return re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())


def test_arrivals_at_another_cta_are_at_cluster_scope():
    """mbarrier.arrive without a scope has CTA scope: a thread of another CTA that waits for it observes nothing."""
    seen = 0
    for path in glob.glob(os.path.join(CSRC, "*.cu*")):
        for op in re.findall(r"mbarrier\.arrive\.[^ ]*", source(os.path.basename(path))):
            if "shared::cluster" in op:
                seen += 1
                assert ".cluster.shared::cluster" in op, (path, op)
    assert seen >= 2


def test_waits_for_another_cta_are_at_cluster_scope():
    """The pair kernel's barriers that work of the other CTA completes are waited for at cluster scope."""
    waits = re.findall(r"wait_on(<true>)?\((\w+)", source("gemm_block_wide.cu"))
    assert {b for _, b in waits} >= {"empty", "full", "tfull", "tfree", "sf_full", "sf_free", "sf_used"}
    for scope, bar in waits:
        if bar in ("empty", "full", "tfull", "tfree"):
            assert scope, bar


def test_no_wait_hides_the_one_before():
    """A wait that ran out ends the loop: its result is looked at before the next wait's takes its place."""
    for name in ("gemm_block.cu", "gemm_block_wide.cu"):
        src = source(name)
        at = [m for m in re.finditer(r"[^\n]*\bok = (?:__all_sync\([^,]*, )?wait_on", src)]
        assert len(at) >= 4
        for one, two in zip(at, at[1:]):
            if "bool ok" in two.group():      # another role's
                continue
            between = src[one.end():two.end()]
            assert "!ok" in between or "if (ok" in two.group(), (name, two.group())


def test_a_split_joins_only_what_every_rank_staged():
    """Partials of other ranks are added only behind a look at every rank's abort flag."""
    src = source("gemm_block.cu")
    load, add = src.index("ld_cluster4(mapa_cluster(st"), src.index("u[0].x += u[k].x")
    assert "cluster_abort_flag(abort_flag, splits)" in src[:load] and "__any_sync(0xffffffffu, gave_up)" in src[load:add]
