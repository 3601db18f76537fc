"""Block-scaled e4m3 linears and the norms around them at their edges.  Tolerances as in test_block8_gpu.py."""
import math

import pytest
import torch

from test_block8_gpu import is_nan_code, norm_ref, operands, rand, value

from test_failure_gpu import DEV_TIMEOUT_TEST, LIMIT_NS, gemm_still_correct, run_selftest

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- products
@pytest.mark.parametrize("M,N,K", [(2640, 4608, 5000), (2640, 1536, 8960)])
@pytest.mark.parametrize("out", ["f32", "e4m3"])
def test_wide_products_are_the_same_on_every_run(M, N, K, out):
    """Many groups of scales through the ring between the CTAs of a pair, beside traffic on another stream: the same
    bits each time, and the sums right."""
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(M, N, K, seed=13)
    flat = lambda r: r if out == "e4m3" else (r,)
    first = [t.clone() for t in flat(ops.gemm_e4m3_block(a8, sa, b8, sb, out=out))]
    other, buf = torch.cuda.Stream(), torch.empty(1 << 27, device="cuda", dtype=torch.uint8)
    other.wait_stream(torch.cuda.current_stream())
    for i in range(12):
        with torch.cuda.stream(other):
            buf.fill_(i)
        for t, r in zip(flat(ops.gemm_e4m3_block(a8, sa, b8, sb, out=out)), first):
            assert torch.equal(t, r)
    torch.cuda.synchronize()
    if out == "f32":
        rows = torch.arange(0, M, 7, device="cuda")
        va, vb = value(a8, sa)[rows], value(b8, sb)
        err = (first[0][rows].double() - va @ vb.t()).abs() / (va.abs() @ vb.abs().t())
        assert err.max().item() <= (K + 4) * 2.0 ** -24


def test_a_split_without_one_part_is_seen_by_every_rank():
    """One rank's wait runs out: all warps of all ranks of its cluster know, none of another cluster."""
    status, scratch, ms = run_selftest(2)
    assert int(status[0]) == DEV_TIMEOUT_TEST
    assert scratch[:4 * 16].view(torch.int32).tolist() == [2] * 8 + [1] * 8
    assert LIMIT_NS / 1e6 <= ms < 1000.0
    assert gemm_still_correct() < 6e-3


@pytest.mark.parametrize("M,N,K", [(1, 640, 1536), (300, 512, 4096), (2640, 4608, 640)])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_status_of_a_product(M, N, K, out):
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(M, N, K, seed=2)
    status = torch.zeros(4, device="cuda", dtype=torch.int32)
    got = ops.gemm_e4m3_block(a8, sa, b8, sb, out=out, status=status)
    ref = ops.gemm_e4m3_block(a8, sa, b8, sb, out=out)
    assert all(torch.equal(g, r) for g, r in (zip(got, ref) if out == "e4m3" else [(got, ref)]))
    assert not status.any()
    for bad in (status.long(), status.cpu(), status[:0], status[::2]):
        with pytest.raises(ValueError, match="status"):
            ops.gemm_e4m3_block(a8, sa, b8, sb, out=out, status=bad)


# ---------------------------------------------------------------- norms
@pytest.mark.parametrize("D", [100, 300, 1283, 1535, 1536, 2050])
@pytest.mark.parametrize("post,pre", [("layer", "rms"), ("rms", "layer"), (None, "layer"), ("layer", None), (None, None)])
def test_norm_of_rows_that_are_not_finite(D, post, pre):
    """A NaN or an infinity stays in its row, and where the formula has it; codes behind D are zero in every row."""
    from fastworld_b200 import ops
    M = 9
    resid, y = rand(M, D, seed=1, dtype=torch.float32), rand(M, D, seed=2)
    resid[1, 3], resid[3, D - 1], y[5, 0], y[7, D - 2] = math.nan, math.inf, math.nan, -math.inf
    odd = torch.zeros(M, dtype=torch.bool, device="cuda")
    odd[1::2] = True
    x, h = norm_ref(resid, y, post, None, None, None, 1, 1, pre, None, None, None, None, M, 1e-6)
    work = resid.clone()
    q, s = ops.norm_gate_resid_(work, y, post=post, pre=pre, out="e4m3")
    assert torch.equal(work.isnan(), x.isnan()) and torch.equal(work.isinf(), x.isinf())
    assert torch.equal(is_nan_code(q[:, :D]), ~h.isfinite())       # infinities are held as the NaN code too
    assert not q[:, D:].any()
    clean, cy = resid[~odd].clone(), y[~odd].clone()
    cq, cs = ops.norm_gate_resid_(clean, cy, post=post, pre=pre, out="e4m3")
    assert torch.equal(q[~odd], cq) and torch.equal(s[:, ~odd], cs) and torch.equal(work[~odd], clean)
    work = resid.clone()
    b = ops.norm_gate_resid_(work, y, post=post, pre=pre)
    assert torch.equal(b.isnan(), h.isnan()) and torch.equal(b.isinf(), h.isinf())
