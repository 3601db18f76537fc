"""Block-scaled e4m3 linears and the norms around them: what can be held to without a GPU."""
import ctypes
import glob
import os
import re

import pytest
import torch

from test_block8_host import EALIGN, EINVAL, ESHAPE, L, P  # noqa: F401

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
        at = [m for m in re.finditer(r"(?:if \([^\n]*\n)?[^\n]*\bok = (?:__all_sync\([^,]*, )?wait_on", src)]
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


def test_status_entry(L):
    """The entry with a status word turns away what the plain one does, and a word that is not aligned."""
    def call(status=None, **kw):
        a = dict(A=P, sa=P, B=P, sb=P, bias=P, out=P, out_s=None, M=4, N=8, K=128, epi=0, dt=0)
        a.update(kw)
        return L.fw_gemm_e4m3_block_status(*a.values(), status, None)
    assert call(M=0) == 0 and call(M=0, status=P) == 0
    assert call(A=None, status=P) == EINVAL and call(K=0, status=P) == ESHAPE and call(out=P + 8, status=P) == EALIGN
    assert call(status=P + 2) == EALIGN


def test_every_wait_of_the_products_has_a_status():
    for name in ("gemm_block.cu", "gemm_block_wide.cu"):
        waits = re.findall(r"\b(?:wait_on(?:<true>)?|mbar_wait)\(([^;{]*)", source(name))
        assert len(waits) >= 6
        for w in waits:
            assert re.search(r"a\.status,\s+DEV_TIMEOUT_", w), (name, w)


# ---------------------------------------------------------------- sizes
def test_sizes_past_32_bits_are_refused_not_cut(L):
    """2^32 + n would reach the library as n."""
    cut = (1 << 32) + 128
    for call in (lambda: L.fw_quant_e4m3_block(P, 0, 0, cut, P, P, None),
                 lambda: L.fw_quant_e4m3_block(P, 0, 1 << 32, 128, P, P, None),
                 lambda: L.fw_gemm_e4m3_block(P, P, P, P, P, P, None, 0, 8, cut, 0, 0, None),
                 lambda: L.fw_gemm_e4m3_block_status(P, P, P, P, P, P, None, 1 << 32, 8, 128, 0, 0, None, None),
                 lambda: L.fw_gemm_bf16(None, P, P, P, 1, 8, cut, 0, 0, None),
                 lambda: L.fw_quant_e4m3(None, 1, -cut, P, P, None)):
        with pytest.raises(ctypes.ArgumentError, match="does not fit an int"):
            call()
    assert L.fw_quant_e4m3_block(P, 0, 0, 2 ** 31 - 1, P, P, None) == ESHAPE


class Fake:
    """A tensor's face without its memory: what the wrappers look at before a launch."""

    def __init__(self, *shape, dtype=torch.float32):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, "cuda:0"

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def stride(self):
        return (self.shape[-1], 1)


def test_wrappers_refuse_sizes_that_the_kernels_do_not_take():
    from fastworld_b200 import ops
    u8, top = torch.uint8, 1 << 24
    s = Fake(1, 1, 4, dtype=u8)
    for name, call in (("x", lambda: ops.quant_e4m3_block(Fake(1, (1 << 32) + 128, dtype=torch.bfloat16))),
                       ("x", lambda: ops.quant_e4m3_block(Fake(1, top + 1))),
                       ("a8", lambda: ops.gemm_e4m3_block(Fake(1, (1 << 32) + 128, dtype=u8), s, s, s)),
                       ("a8", lambda: ops.gemm_e4m3_block(Fake(1, top + 128, dtype=u8), s, s, s)),
                       ("b8", lambda: ops.gemm_e4m3_block(Fake(1, 128, dtype=u8), s, Fake(top + 1, 128, dtype=u8), s)),
                       ("resid", lambda: ops.norm_gate_resid_(Fake(1 << 31, 1))),
                       ("resid", lambda: ops.norm_gate_resid_(Fake(1, (1 << 32) + 1)))):
        with pytest.raises(ValueError, match=name + ": expected"):
            call()


def test_rows_per_frame_is_a_whole_number():
    """2.5 rows are not 2."""
    from fastworld_b200 import ops
    for rows in (2.5, 0.5, -1, 0):
        with pytest.raises(ValueError, match="rows_per_frame"):
            ops.norm_gate_resid_(Fake(4, 128), rows_per_frame=rows)


def test_calls_go_to_the_tensors_device_and_its_stream(monkeypatch):
    """Tensors of another device than the current one: that device is made the current one around the launch, and its
    current stream taken."""
    from fastworld_b200 import ops
    current, log = [0], []

    class device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.back, current[0] = current[0], self.index

        def __exit__(self, *_):
            current[0] = self.back

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)

    def fn(a, stream):
        log.append((a, stream, current[0]))
        return 0
    ops._on(1, fn, "f", "x")
    ops._on(0, fn, "f", "y")
    assert log == [("x", 101, 1), ("y", 100, 0)] and current == [0]
    with pytest.raises(RuntimeError):
        ops._on(1, lambda *_: EINVAL, "f")
    assert current == [0]
