"""Block-scaled e4m3 linears and the norms around them at their edges.  Tolerances as in test_block8_gpu.py."""
import math

import pytest
import torch

from test_block8_gpu import (is_nan_code, norm64, norm_ref, operands, pow2, rand, test_gemm_epilogues as epilogues,
                             test_norm_gate_resid as norms, value)

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


# tiles of 64 and of 128 rows whose k-blocks a cluster shares; the pair kernel's rows of C that no 16-byte store can
# address (4500 bf16: the time model is far from the border at 4680 rows)
@pytest.mark.parametrize("M,N,K", [(300, 1000, 4096), (512, 1536, 4096), (513, 1535, 4000), (4680, 4500, 2000)])
@pytest.mark.parametrize("epi", ["none", "gelu_tanh", "gelu_erf"])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_split_and_wide_epilogues(M, N, K, epi, out):
    epilogues(M, N, K, epi, out)


def test_e4m3_result_past_32_bits():
    """The last rows of codes of more than 2^31 bytes."""
    from fastworld_b200 import ops
    M, N, last = 1100001, 2048, slice(-300, None)
    a8, sa, b8, sb = operands(M, N, 128)
    q, s = ops.gemm_e4m3_block(a8, sa, b8, sb, out="e4m3")
    q, s = q[last].contiguous(), s[:, last].contiguous()
    va, vb = value(a8[last], sa[:, last]), value(b8, sb)
    ref, tol = va @ vb.t(), 132 * 2.0 ** -24 * (va.abs() @ vb.abs().t())
    unit = pow2(s.permute(1, 0, 2).reshape(300, -1).double() - 127).repeat_interleave(128, 1)
    step = torch.maximum(ref.abs() * 2.0 ** -4, unit * 2.0 ** -10)
    assert ((value(q, s) - ref).abs() <= step * (1 + 1e-6) + 1.07 * tol).all()


# ---------------------------------------------------------------- norms
# with test_norm_widths, every number of warps per row and of blocks per warp over rows aligned to four elements and not
@pytest.mark.parametrize("D", [383, 511, 1283, 1535, 2816, 2948])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_norm_more_widths(D, out):
    norms(21, D, 8, "layer", "rms", torch.bfloat16, out)
    norms(3, D, 1, "rms", "layer", torch.float32, out)


@pytest.mark.parametrize("D", [5, 384, 1535, 1536, 5120, 16384])
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e-3])
def test_norm_statistics_in_fp32(D, kind, eps):
    """Rows whose mean square is about eps or far below, and a row of zeros, as the norm after a block (fp32 out) and as
    the one before the next (bf16 out).

    A row's sums are added up by lane (at most 2 * 8 + 1 terms in a chain), across a warp (5) and across at most 16
    warps, each a rounding: 38 of 2^-24.  1 / D, its product and eps add 4, so the reciprocal root is off by (38 + 4) / 2
    and its own 4 (two units in the last place), the product with it by 1: 26, rounded up to 32.  LayerNorm's mean is off by
    the 38 + 2 of mean|v| and the subtraction by 1, against the root: 42 r mean|v|."""
    from fastworld_b200 import ops
    u = 2.0 ** -24
    y = rand(24, D, seed=3, dtype=torch.float32) * torch.tensor([0.0, 1e-4, 1e-3, 3e-3, 1e-2, 1.0],
                                                                device="cuda").repeat(4)[:, None]
    y[12:] += 0.5 * y[12:].abs().amax(1, keepdim=True)      # means that are not small
    ref = norm64(y.double(), kind, eps)
    v = y.double() - (y.double().mean(1, keepdim=True) if kind == "layer" else 0)
    r = 1 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    tol = 32 * u * ref.abs() + (42 * u * r * y.double().abs().mean(1, keepdim=True) if kind == "layer" else 0)
    x = torch.zeros(24, D, device="cuda")
    assert ops.norm_gate_resid_(x, y, post=kind, eps=eps, out=None) is None
    assert ((x.double() - ref).abs() <= tol).all()
    assert not x[::6].any()
    h = ops.norm_gate_resid_(y, pre=kind, eps=eps)
    assert ((h.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * tol).all()
    assert not h[::6].any()


@pytest.mark.parametrize("D", [384, 1535, 5120])
def test_norm_of_the_residual_itself(D):
    """y may be the residual's own memory."""
    from fastworld_b200 import ops
    x = rand(50, D, seed=1, dtype=torch.float32)
    kw = dict(post="rms", post_w=rand(D, seed=2), resid_scale=0.5, branch_scale=2.0, pre="layer")
    apart = x.clone()
    ref = ops.norm_gate_resid_(apart, x.clone(), **kw)
    h = ops.norm_gate_resid_(x, x, **kw)
    assert torch.equal(h, ref) and torch.equal(x, apart)


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


# ---------------------------------------------------------------- long and wide ones, and the feed-forward pair
def test_longest_sum():
    """2^24 columns of ones: every partial sum is a whole number that fp32 holds."""
    from fastworld_b200 import ops
    K = 1 << 24
    a8, sa = ops.quant_e4m3_block(torch.ones(2, K, device="cuda", dtype=torch.bfloat16))
    b8, sb = ops.quant_e4m3_block(torch.ones(3, K, device="cuda", dtype=torch.bfloat16))
    assert (ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32") == K).all()


def test_many_columns():
    from fastworld_b200 import ops
    M, N, K = 3, (1 << 20) + 5, 200
    a8, sa, b8, sb = operands(M, N, K)
    va, vb = value(a8, sa), value(b8, sb)
    ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
    out = ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32")
    assert ((out.double() - ref).abs() <= (K + 4) * 2.0 ** -24 * mag).all()


def test_feed_forward_pair():
    """The pair's result is the product of the codes between, which are right one by one: a hidden value on the other
    side of a rounding border is a step of the format, and all that a plain form's result may differ by.  Alternating
    inputs give each its own result, the same bits every time."""
    from fastworld_b200 import ops
    M, D, F = 2640, 1536, 8960
    epilogues(M, F, D, "gelu_tanh", "e4m3")
    up, down = operands(4, F, D, seed=21)[2:], operands(4, D, F, seed=22)[2:]
    b1, b2 = rand(F, seed=23, size=0.1), rand(D, seed=24, size=0.1)

    def pair(x):
        h8, sh = ops.gemm_e4m3_block(*x, *up, b1, epilogue="gelu_tanh", out="e4m3")
        return h8, sh, ops.gemm_e4m3_block(h8, sh, *down, b2)
    xs = [operands(M, 4, D, seed=25 + i)[:2] for i in range(2)]
    first = [pair(x) for x in xs]
    assert not torch.equal(first[0][2], first[1][2])
    for _ in range(5):
        for x, ref in zip(xs, first):
            assert all(torch.equal(g, r) for g, r in zip(pair(x), ref))
    for h8, sh, got in first:
        vh, vd = value(h8, sh), value(*down)
        ref = vh @ vd.t() + b2.double()
        mag = vh.abs() @ vd.abs().t() + b2.double().abs()
        assert ((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * (F + 4) * 2.0 ** -24 * mag).all()
