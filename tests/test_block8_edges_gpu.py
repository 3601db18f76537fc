"""Block-scaled e4m3 linears and the norms around them at their edges.  Tolerances as in test_block8_gpu.py."""
import pytest
import torch

from test_block8_gpu import operands, rand, value  # noqa: F401

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
