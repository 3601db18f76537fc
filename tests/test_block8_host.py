"""Refusals of the block-scaled e4m3 linears and the norms around them (no GPU: every call is turned away
on the host before a launch, or has nothing to do)."""
import ctypes

import pytest
import torch

EINVAL, ESHAPE, EALIGN = -1, -2, -3
P = 1 << 20            # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    import os

    from fastworld_b200 import _lib, build
    if not os.path.exists(_lib.LIB_PATH):
        build.build()
    return _lib.lib()


def test_quant_refusals(L):
    f = L.fw_quant_e4m3_block
    assert f(P, 0, 0, 128, P, P, None) == 0                      # no rows: nothing to do
    assert f(None, 0, 1, 128, P, P, None) == EINVAL
    assert f(P, 0, 1, 128, None, P, None) == EINVAL
    assert f(P, 0, 1, 128, P, None, None) == EINVAL
    assert f(P, 2, 1, 128, P, P, None) == EINVAL                 # int32 rows
    assert f(P, 0, -1, 128, P, P, None) == ESHAPE
    assert f(P, 0, 1, 0, P, P, None) == ESHAPE
    assert f(P, 0, 1, (1 << 24) + 1, P, P, None) == ESHAPE
    assert f(P, 0, 1, 128, P + 8, P, None) == EALIGN
    assert f(P, 0, 1, 128, P, P + 2, None) == EALIGN
    assert f(P + 1, 0, 1, 128, P, P, None) == EALIGN             # x not at an element


def gemm(L, A=P, sa=P, B=P, sb=P, bias=P, out=P, out_s=None, M=4, N=8, K=128, epi=0, dt=0):
    return L.fw_gemm_e4m3_block(A, sa, B, sb, bias, out, out_s, M, N, K, epi, dt, None)


def test_gemm_refusals(L):
    assert gemm(L, M=0, A=None, out=None) == 0 and gemm(L, N=0) == 0
    for k in ("A", "sa", "B", "sb", "out"):
        assert gemm(L, **{k: None}) == EINVAL, k
    for k in ("A", "B", "out"):
        assert gemm(L, **{k: P + 8}) == EALIGN, k
    assert gemm(L, sa=P + 2) == EALIGN and gemm(L, sb=P + 1) == EALIGN and gemm(L, bias=P + 1) == EALIGN
    assert gemm(L, dt=3, out_s=P + 2) == EALIGN
    for k in ("M", "N", "K"):
        assert gemm(L, **{k: -1}) == ESHAPE, k
    assert gemm(L, K=0) == ESHAPE
    assert gemm(L, K=(1 << 24) + 1) == ESHAPE and gemm(L, N=(1 << 24) + 1) == ESHAPE
    assert gemm(L, epi=2) == EINVAL and gemm(L, epi=3) == EINVAL and gemm(L, epi=5) == EINVAL
    assert gemm(L, dt=2) == EINVAL and gemm(L, dt=4) == EINVAL
    assert gemm(L, dt=3) == EINVAL                                # codes without a place for exponents
    assert gemm(L, dt=0, out_s=P) == EINVAL                       # exponents of a bf16 result


def norm(L, **kw):
    from fastworld_b200 import _lib
    a = dict(resid=P, y=P, y_dtype=0, post=0, pre=1, post_w=0, post_b=0, pre_w=0, pre_b=0, gate=0, shift=0, scale=0,
             resid_scale=1.0, branch_scale=1.0, eps=1e-6, M=2, D=128, rows_per_frame=1, out=P, out_s=0)
    a.update(kw)
    return L.fw_norm_gate_resid(ctypes.byref(_lib.FwNormArgs(*a.values())), None)


def test_norm_refusals(L):
    assert L.fw_norm_gate_resid(None, None) == EINVAL
    assert norm(L, M=0, resid=0) == 0
    assert norm(L, resid=0) == EINVAL
    assert norm(L, M=-1) == ESHAPE and norm(L, D=0) == ESHAPE and norm(L, D=16385) == ESHAPE
    assert norm(L, rows_per_frame=0) == ESHAPE
    assert norm(L, post=3) == EINVAL and norm(L, pre=-1) == EINVAL
    assert norm(L, y_dtype=4) == EINVAL
    assert norm(L, shift=P) == EINVAL and norm(L, scale=P) == EINVAL
    assert norm(L, y=0, out=0) == EINVAL and norm(L, out=0, out_s=P) == EINVAL
    assert norm(L, out=P + 8, out_s=P) == EALIGN
    for k in ("resid", "gate"):
        assert norm(L, **{k: P + 2}) == EALIGN, k
    for k in ("y", "post_w", "post_b", "pre_w", "pre_b", "out"):
        assert norm(L, **{k: P + 1}) == EALIGN, k
    assert norm(L, y=P + 2, y_dtype=1) == EALIGN


def test_wrappers_refuse_what_is_not_on_a_gpu():
    from fastworld_b200 import ops
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 128, dtype=torch.uint8), torch.zeros(1, 2, 4, dtype=torch.uint8)
    for call in (lambda: ops.quant_e4m3_block(x), lambda: ops.quant_e4m3_block(x.int()),
                 lambda: ops.gemm_e4m3_block(q, s, q, s), lambda: ops.gemm_e4m3_block(q, s, q, s, epilogue="relu"),
                 lambda: ops.gemm_e4m3_block(q, s, q, s, out="f16"),
                 lambda: ops.norm_gate_resid_(x.float()), lambda: ops.norm_gate_resid_(x.float(), x)):
        with pytest.raises(ValueError):
            call()
