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
