"""Block-scaled e4m3 linears and the norms around them against 64-bit PyTorch references.

Tolerances.  The quantiser is exact: every code and exponent follows from the definition.  A product's operands
are exact in fp64, so its error is the fp32 accumulation, at most K 2^-24 of sum|a b| in any order of summation
(measured far below), then the activation (a few fp32 roundings) and half a step of the output type.  Where
a result is quantised, a value may fall on the other side of a rounding border, which
moves it by one step of its block: 2^-3 of the value, or 2^-9 of the block's scale at the bottom."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def exponents(x):
    """Unbiased exponents [R, blocks] by the definition, in fp64 (finite elements only)."""
    r, k = x.shape
    nb = -(-k // 128)
    w = torch.nn.functional.pad(x.double(), (0, nb * 128 - k)).view(r, nb, 128).abs()
    top = torch.where(torch.isfinite(w), w, torch.zeros_like(w)).amax(-1)
    e = torch.full_like(top, -127)
    for b in range(-126, 122):       # the smallest that holds the maximum (host powers of two are exact)
        e = torch.where(top > 448 * 2.0 ** (b - 1), torch.full_like(e, b), e)
    return e


def pow2(e):
    """2^e in fp64 from the exponent field."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def ref_quant(x):
    r, k = x.shape
    nb = -(-k // 128)
    e = exponents(x)
    w = torch.nn.functional.pad(x.double(), (0, nb * 128 - k)).view(r, nb, 128)
    c = (w * pow2(-e)[..., None]).float()          # exact, or below every code
    q = torch.where(torch.isfinite(w), c, torch.full_like(c, math.nan)).to(F8).view(torch.uint8).view(r, nb * 128)
    s = torch.full((r, -(-nb // 4) * 4), 127, dtype=torch.uint8, device=x.device)
    s[:, :nb] = (e + 127).to(torch.uint8)
    return q, s.view(r, -1, 4).permute(1, 0, 2).contiguous()


def value(q, s):
    """fp64 values of codes and exponents."""
    r, kp = q.shape
    e = s.permute(1, 0, 2).reshape(r, -1)[:, :kp // 128].double() - 127
    return (q.view(F8).double().view(r, -1, 128) * pow2(e)[..., None]).view(r, kp)


def powers(lo, hi, *shape, seed=0):
    """Random powers of two, exponents in [lo, hi)."""
    g = torch.Generator(device="cuda").manual_seed(seed + 91)
    return torch.exp2(torch.randint(lo, hi, shape, device="cuda", generator=g).float())


def rand(*shape, seed=0, dtype=torch.bfloat16, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + sum(shape) * 7)
    return (torch.randn(*shape, device="cuda", generator=g) * size).to(dtype)


def is_nan_code(q):
    return (q & 0x7f) == 0x7f


# ---------------------------------------------------------------- quantiser
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (1, 1536), (3, 127), (9, 129), (257, 1283), (8, 512), (7, 516),
                                 (300, 2050),
                                 (1001, 640)])
def test_quant_exact(M, K, dtype):
    from fastworld_b200 import ops
    x = rand(M, K, dtype=dtype) * powers(-12, 12, M, 1).to(dtype)
    q, s = ops.quant_e4m3_block(x)
    rq, rs = ref_quant(x)
    assert torch.equal(s, rs)
    assert torch.equal(q, rq)


def test_quant_borders_and_specials():
    from fastworld_b200 import ops
    x = torch.zeros(16, 256, device="cuda")
    x[1, 0] = 448.0                                   # exactly the largest code
    x[2, 0] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    x[3, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    x[4, 0] = 3.4028234663852886e38
    x[5, 0] = 1e-45                                   # subnormal
    x[6, 0] = 2.0 ** -119
    x[7, :] = math.nan
    x[8, :3] = torch.tensor([448.0, 17.0, 19.0])      # ties of 16 and 18 and 20: to even
    x[9, :] = -0.0
    q, s = ops.quant_e4m3_block(x)
    rq, rs = ref_quant(x)
    assert torch.equal(s, rs)
    nan = is_nan_code(rq)
    assert torch.equal(is_nan_code(q), nan) and torch.equal(q[~nan], rq[~nan])
    assert s[0, 1, 0] == 127 and s[0, 2, 0] == 128 and s[0, 0, 0] == 0


def test_quant_unaligned_view_and_empty():
    from fastworld_b200 import ops
    flat = rand(5 * 516 + 3, size=2.0)
    x = flat[3:].view(5, 516)                         # 6 bytes past an aligned address
    q, s = ops.quant_e4m3_block(x)
    rq, rs = ref_quant(x)
    assert torch.equal(q, rq) and torch.equal(s, rs)
    q, s = ops.quant_e4m3_block(torch.empty(0, 300, device="cuda"))
    assert q.shape == (0, 384) and s.shape == (1, 0, 4)


# ---------------------------------------------------------------- product
def act64(v, name):
    if name == "gelu_tanh":
        # 0.5 (1 + tanh u) = sigmoid(2u): the sum cancels below u = -18 even in fp64
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5)) if name == "gelu_erf" else v


def operands(M, N, K, seed=0):
    from fastworld_b200 import ops
    a = rand(M, K, seed=seed, size=1.0) * powers(-3, 4, M, 1, seed=seed).bfloat16()
    b = rand(N, K, seed=seed + 1, size=1 / math.sqrt(K))
    # blocks of very different size, so that a wrong scale shows
    blk = powers(-4, 5, -(-K // 128), seed=seed + 1).repeat_interleave(128)[:K]
    a, b = (a * blk).bfloat16(), (b * blk.flip(0)).bfloat16()
    return (*ops.quant_e4m3_block(a), *ops.quant_e4m3_block(b))


SHAPES = [(1, 9216, 1536), (1, 1, 1), (2, 130, 129), (16, 256, 512), (17, 300, 640), (32, 128, 2048), (33, 77, 130),
          (64, 512, 1024), (65, 1000, 1283), (128, 128, 128), (129, 260, 384), (257, 1536, 1280), (300, 777, 896),
          (512, 1536, 4096), (1001, 777, 1283), (2640, 1536, 1536), (2640, 4608, 640)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_f32(M, N, K):
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(M, N, K)
    bias = rand(N, seed=5)
    va, vb = value(a8, sa), value(b8, sb)
    ref = va @ vb.t() + bias.double()
    mag = va.abs() @ vb.abs().t() + bias.double().abs()
    out = ops.gemm_e4m3_block(a8, sa, b8, sb, bias, out="f32")
    assert out.shape == (M, N) and out.dtype == torch.float32
    err = ((out.double() - ref).abs() / mag).max().item()
    assert err <= (K + 4) * 2.0 ** -24, err
    again = ops.gemm_e4m3_block(a8, sa, b8, sb, bias, out="f32")
    assert torch.equal(out, again)


@pytest.mark.parametrize("M,N,K", [(1, 640, 512), (40, 129, 256), (200, 384, 1280), (700, 1000, 512),
                                   (2640, 1536, 256)])
@pytest.mark.parametrize("epi", ["none", "gelu_tanh", "gelu_erf"])
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
def test_gemm_epilogues(M, N, K, epi, out):
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(M, N, K, seed=3)
    bias = rand(N, seed=9, size=0.3)
    va, vb = value(a8, sa), value(b8, sb)
    pre = va @ vb.t() + bias.double()
    mag = va.abs() @ vb.abs().t() + bias.double().abs()
    ref = act64(pre, epi)
    # |act'| <= 1.13; the activation itself: a few roundings of its value, and of v for tiny results
    tol = 1.13 * (K + 4) * 2.0 ** -24 * mag + 16 * 2.0 ** -24 * pre.abs()
    got = ops.gemm_e4m3_block(a8, sa, b8, sb, bias, epilogue=epi, out=out)
    if out == "e4m3":
        q, s = got
        Np = -(-N // 128) * 128
        assert q.shape == (M, Np) and s.shape == (-(-Np // 512), M, 4)
        assert not q[:, N:].any()
        rs = ref_quant(ref)[1]
        assert (s.int() - rs.int()).abs().max() <= 1 and (s != rs).float().mean() < 1e-2
        nb = Np // 128
        assert (s.permute(1, 0, 2).reshape(M, -1)[:, nb:] == 127).all()
        e = s.permute(1, 0, 2).reshape(M, -1)[:, :nb].double() - 127
        unit = pow2(e).repeat_interleave(128, 1)[:, :N]
        v = value(q, s)[:, :N]
        step = torch.maximum(ref.abs() * 2.0 ** -4, unit * 2.0 ** -10)     # half a step
        assert ((v - ref).abs() <= step * (1 + 1e-6) + 1.07 * tol).all()
        assert (ref.abs().amax(1) <= 448 * unit.amax(1) * (1 + 1e-5)).all()
    else:
        half = 2.0 ** -8 if out == "bf16" else 2.0 ** -24
        assert ((got.double() - ref).abs() <= half * ref.abs() + 1.01 * tol + 1e-38).all()


def test_gemm_scales_at_the_ends():
    """Exponents far from one another multiply exactly; a NaN reaches its row and no other."""
    from fastworld_b200 import ops
    M, N, K = 40, 200, 640
    a8, sa, b8, sb = operands(M, N, K, seed=11)
    base = ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32")
    out = ops.gemm_e4m3_block(a8, sa + 60, b8, sb - 70, out="f32")
    assert torch.equal(out, base * 2.0 ** -10)
    a8[3, 5] = 0x7f
    got = ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32")
    assert got[3].isnan().all()
    keep = torch.arange(M, device="cuda") != 3
    assert torch.equal(got[keep], base[keep])


@pytest.mark.parametrize("M,N,K", [(20, 300, 256), (600, 300, 256), (1500, 1000, 640)])
@pytest.mark.parametrize("out", ["f32", "e4m3"])
def test_gemm_infinities(M, N, K, out):
    """A result that overflows fp32 is an infinity, the NaN code in e4m3; its block is scaled by what is finite.
    All terms are positive: partial sums of both signs may overflow to infinities that add up to NaN."""
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(M, N, K, seed=5)
    a8, b8 = a8 & 0x7f, b8 & 0x7f
    sa[:, 7] = 127 + 70
    sb[:, N - 3:] = 127 + 70                           # (7, N - 3 ...): 2^140 times a sum; 2^70 elsewhere
    v = ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32")
    assert v[7, N - 3:].isinf().all() and v[:7].isfinite().all() and v[8:].isfinite().all()
    if out == "e4m3":
        q, s = ops.gemm_e4m3_block(a8, sa, b8, sb, out="e4m3")
        rq, rs = ref_quant(v)
        assert torch.equal(s, rs) and torch.equal(is_nan_code(q), is_nan_code(rq))
        keep = ~is_nan_code(rq)
        assert torch.equal(q[keep], rq[keep])


# several waves of 256 x 256 tiles on CTA pairs: rows and columns that end inside a tile, a group of scales that
# K does not fill, rows of C that no 16-byte store can address (4500 bf16, 4503)
@pytest.mark.parametrize("M,N,K", [(2600, 4504, 768), (2601, 4500, 769), (2640, 4503, 1400)])
@pytest.mark.parametrize("epi", ["none", "gelu_tanh", "gelu_erf"])
@pytest.mark.parametrize("out", ["bf16", "f32", "e4m3"])
def test_gemm_large_epilogues(M, N, K, epi, out):
    test_gemm_epilogues(M, N, K, epi, out)


@pytest.mark.parametrize("out", ["f32", "e4m3"])
def test_gemm_large_infinities(out):
    test_gemm_infinities(2600, 4504, 768, out)


@pytest.mark.parametrize("M,N,K", [(3, 200, 70001), (300, 520, 20000), (1000, 900, 9000)])
def test_gemm_long_sums(M, N, K):
    test_gemm_f32(M, N, K)


def test_offsets_past_32_bits():
    """The last rows of tensors of more than 2^31 elements are what they are alone."""
    from fastworld_b200 import ops
    M, D, last = 1100001, 2048, slice(-300, None)
    x = torch.zeros(M, D, device="cuda", dtype=torch.bfloat16)
    x[last] = rand(300, D, seed=1)
    q, s = ops.quant_e4m3_block(x)
    rq, rs = ops.quant_e4m3_block(x[last])
    assert torch.equal(q[last], rq) and torch.equal(s[:, last], rs) and not q[:-300].any()
    del q, s
    resid = torch.zeros(M, D, device="cuda")
    resid[last] = rand(300, D, seed=2, dtype=torch.float32)
    alone = resid[last].clone()
    ref = ops.norm_gate_resid_(alone, x[last], post="rms", pre="layer")
    out = ops.norm_gate_resid_(resid, x, post="rms", pre="layer")
    assert torch.equal(out[last], ref) and torch.equal(resid[last], alone) and not resid[:-300].any()
    del out, resid, x
    a8, sa, b8, sb = operands(M, D, 128)
    got = ops.gemm_e4m3_block(a8, sa, b8, sb, out="f32")[last]
    va, vb = value(a8[last], sa[:, last]), value(b8, sb)
    assert ((got.double() - va @ vb.t()).abs() <= 132 * 2.0 ** -24 * (va.abs() @ vb.abs().t())).all()


def test_gemm_no_rows():
    from fastworld_b200 import ops
    _, _, b8, sb = operands(4, 100, 300)
    a8, sa = ops.quant_e4m3_block(torch.empty(0, 300, device="cuda"))
    assert ops.gemm_e4m3_block(a8, sa, b8, sb).shape == (0, 100)
    q, s = ops.gemm_e4m3_block(a8, sa, b8, sb, out="e4m3")
    assert q.shape == (0, 128) and s.shape == (1, 0, 4)


# ---------------------------------------------------------------- norms
def norm64(v, kind, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def norm_ref(resid, y, post, post_w, post_b, gate, rs, bs, pre, pre_w, pre_b, shift, scale, rpf, eps):
    M = resid.shape[0]
    f = torch.arange(M, device=resid.device) // rpf
    x = resid.double()
    if y is not None:
        b = norm64(y.double(), post, eps)
        b = b * (1 if post_w is None else post_w.double()) + (0 if post_b is None else post_b.double())
        x = rs * x + bs * b * (1 if gate is None else gate.double().view(-1, x.shape[1])[f])
    h = norm64(x, pre, eps) * (1 if pre_w is None else pre_w.double()) + (0 if pre_b is None else pre_b.double())
    if scale is not None:
        h = h * (1 + scale.double().view(-1, x.shape[1])[f]) + shift.double().view(-1, x.shape[1])[f]
    return x, h


NORM_SHAPES = [(1, 1536, 1), (1, 1, 1), (5, 3, 2), (2, 128, 1), (7, 129, 3), (3, 500, 3), (880, 1536, 293), (33, 1538, 20),
               (64, 5120, 32), (9, 6146, 4), (4, 16384, 2), (1200, 384, 400)]


@pytest.mark.parametrize("M,D,rpf", NORM_SHAPES)
@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms"), (None, "layer"), ("rms", None)])
@pytest.mark.parametrize("ydt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("out", ["bf16", "e4m3", None])
def test_norm_gate_resid(M, D, rpf, post, pre, ydt, out):
    from fastworld_b200 import ops
    fr = -(-M // rpf)
    resid = rand(M, D, seed=1, dtype=torch.float32, size=3.0) + 0.5
    y = (rand(M, D, seed=2, dtype=torch.float32, size=2.0) - 0.3).to(ydt)
    post_w, post_b = rand(D, seed=3) + 1, rand(D, seed=4, size=0.2)
    pre_w, pre_b = rand(D, seed=5, size=0.2) + 1, rand(D, seed=6, size=0.2)
    gate, shift, scale = (rand(fr, D, seed=7 + i, dtype=torch.float32, size=0.5) for i in range(3))
    kw = dict(post=post, post_w=post_w, post_b=post_b, gate=gate, resid_scale=0.75, branch_scale=1.25, eps=1e-5)
    if out is not None:
        kw.update(pre_w=pre_w, pre_b=pre_b, shift=shift, scale=scale)
    x, h = norm_ref(resid, y, post, post_w, post_b, gate, 0.75, 1.25, pre, pre_w, pre_b, shift, scale, rpf, 1e-5)
    work = resid.clone()
    got = ops.norm_gate_resid_(work, y, pre=pre, rows_per_frame=rpf, out=out, **kw)
    # the row sums: D roundings at worst, half of them count in 1 / sqrt; a few products behind them
    eps_x = (D / 2 + 16) * 2.0 ** -24
    mag = 0.75 * resid.double().abs() + (x - 0.75 * resid.double()).abs() + post_b.abs().double() * 4
    assert ((work.double() - x).abs() <= eps_x * (mag + 8)).all()
    if out is None:
        assert got is None
        return
    tol = 8 * eps_x * (h.abs() + 8) * (16 if D < 4 else 1)
    if pre == "layer" and D == 1:        # the deviation is exactly zero on both sides
        tol = torch.full_like(h, 1e-5)
    if out == "bf16":
        assert ((got.double() - h).abs() <= 2.0 ** -8 * h.abs() + 1.01 * tol).all()
    else:
        q, s = got
        Dp = -(-D // 128) * 128
        assert not q[:, D:].any()
        e = s.permute(1, 0, 2).reshape(M, -1).double() - 127
        assert (e[:, Dp // 128:] == 0).all()
        unit = pow2(e[:, :Dp // 128]).repeat_interleave(128, 1)[:, :D]
        step = torch.maximum(h.abs() * 2.0 ** -4, unit * 2.0 ** -10)
        assert ((value(q, s)[:, :D] - h).abs() <= step * (1 + 1e-6) + 1.07 * tol).all()
        rs = ref_quant(h)[1]
        assert (s.int() - rs.int()).abs().max() <= 1 and (s != rs).float().mean() < 0.02


# every number of warps per row and of blocks per warp, rows aligned to four elements and not
@pytest.mark.parametrize("D", [200, 255, 300, 512, 701, 768, 1001, 1024, 1151, 1152, 1900, 1919, 2300, 2301, 2561, 2688,
                               3001, 4000, 4095, 5119, 6143, 6144, 8191, 8192, 9001])
@pytest.mark.parametrize("out", ["bf16", "e4m3"])
def test_norm_widths(D, out):
    test_norm_gate_resid(21, D, 8, "layer", "rms", torch.bfloat16, out)
    test_norm_gate_resid(3, D, 1, "rms", "layer", torch.float32, out)


def test_norm_plain_forms():
    """No y: the norm alone, the residual untouched; no options: the plain residual sum."""
    from fastworld_b200 import ops
    M, D = 37, 384
    resid = rand(M, D, seed=1, dtype=torch.float32)
    keep = resid.clone()
    h = ops.norm_gate_resid_(resid)
    assert torch.equal(resid, keep)
    ref = norm64(keep.double(), "layer", 1e-6)
    assert ((h.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-5).all()
    y = rand(M, D, seed=2)
    assert ops.norm_gate_resid_(resid, y, out=None) is None
    assert torch.equal(resid, keep + y.float())
    w = rand(D, seed=3)
    one = ops.norm_gate_resid_(resid, pre="rms", pre_w=w, shift=torch.zeros(D, device="cuda"),
                               scale=torch.zeros(D, device="cuda"))
    assert torch.equal(one, ops.norm_gate_resid_(resid, pre="rms", pre_w=w))
    assert ops.norm_gate_resid_(torch.empty(0, D, device="cuda"), out="e4m3")[0].shape == (0, 384)


# ---------------------------------------------------------------- together, streams, graphs
def _block(x, y, W, ops):
    """norm -> q/k/v-like product; feed-forward pair; norm and residual: one block's linears."""
    h8, sh = ops.norm_gate_resid_(x, y, post="rms", gate=W["gate"], pre="layer", shift=W["shift"], scale=W["scale"],
                                  out="e4m3")
    u8, su = ops.gemm_e4m3_block(h8, sh, *W["up"], W["b1"], epilogue="gelu_tanh", out="e4m3")
    v = ops.gemm_e4m3_block(u8, su, *W["down"], W["b2"])
    return ops.norm_gate_resid_(x, v, post="layer", gate=W["gate"], pre="rms")


def _weights(D, F):
    from fastworld_b200 import ops
    return {"gate": rand(1, D, seed=1, dtype=torch.float32), "shift": rand(1, D, seed=2, dtype=torch.float32),
            "scale": rand(1, D, seed=3, dtype=torch.float32), "b1": rand(F, seed=4, size=0.1),
            "b2": rand(D, seed=5, size=0.1),
            "up": ops.quant_e4m3_block(rand(F, D, seed=6, size=D ** -0.5)),
            "down": ops.quant_e4m3_block(rand(D, F, seed=7, size=F ** -0.5))}


@pytest.mark.parametrize("M", [1, 50, 700])
def test_block_of_linears(M):
    from fastworld_b200 import ops
    D, F = 384, 1000
    W = _weights(D, F)
    x, y = rand(M, D, seed=8, dtype=torch.float32), rand(M, D, seed=9)
    x0 = x.clone()
    got = _block(x, y, W, ops)
    r, h = norm_ref(x0, y, "rms", None, None, W["gate"], 1, 1, "layer", None, None, W["shift"], W["scale"], M, 1e-6)
    q = value(*ref_quant(h.float()))[:, :D]
    u = act64(q @ value(*W["up"])[:, :D].t() + W["b1"].double(), "gelu_tanh")
    v = value(*ref_quant(u.float()))[:, :F] @ value(*W["down"])[:, :F].t() + W["b2"].double()
    r, h = norm_ref(r, v, "layer", None, None, W["gate"], 1, 1, "rms", None, None, None, None, M, 1e-6)
    # two bf16 roundings (v and the output); the few codes on the other side of a border are far below them
    assert float((got.double() - h).norm() / h.norm()) < 2 * 2.0 ** -8
    assert float((x.double() - r).norm() / r.norm()) < 2.0 ** -8


def test_two_streams_and_a_graph_give_the_same():
    from fastworld_b200 import ops
    D, F, M = 512, 1024, 300
    W = _weights(D, F)
    xs = [rand(M, D, seed=20 + i, dtype=torch.float32) for i in range(2)]
    ys = [rand(M, D, seed=30 + i) for i in range(2)]
    refs = [_block(x.clone(), y, W, ops) for x, y in zip(xs, ys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    work = [x.clone() for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                work[i].copy_(xs[i])
                got[i] = _block(work[i], ys[i], W, ops)
    torch.cuda.synchronize()
    for g, r in zip(got, refs):
        assert torch.equal(g, r)
    buf, src = xs[0].clone(), ys[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _block(buf, src, W, ops)
    for i in range(2):
        buf.copy_(xs[i])
        src.copy_(ys[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, refs[i])


def test_refusals():
    """Wrong types, shapes, strides and combinations raise before a launch."""
    from fastworld_b200 import ops
    a8, sa, b8, sb = operands(4, 100, 300)
    x = torch.zeros(4, 384, device="cuda")
    y, w, v = x.bfloat16(), torch.ones(384, device="cuda", dtype=torch.bfloat16), torch.ones(384, device="cuda")
    bad = [lambda: ops.quant_e4m3_block(x.double()), lambda: ops.quant_e4m3_block(x[:, :128]),
           lambda: ops.quant_e4m3_block(x[0]), lambda: ops.quant_e4m3_block(x[:, :0]),
           lambda: ops.gemm_e4m3_block(a8, sa[:, :3], b8, sb), lambda: ops.gemm_e4m3_block(a8[:, :256], sa, b8, sb),
           lambda: ops.gemm_e4m3_block(a8[:, :256].contiguous(), sa, b8, sb),
           lambda: ops.gemm_e4m3_block(a8[:, :100].contiguous(), sa, b8, sb),
           lambda: ops.gemm_e4m3_block(a8, sa.int(), b8, sb), lambda: ops.gemm_e4m3_block(a8, sa, b8, sb, w),
           lambda: ops.gemm_e4m3_block(a8, sa, b8, sb, v[:100]), lambda: ops.gemm_e4m3_block(a8.cpu(), sa, b8, sb),
           lambda: ops.gemm_e4m3_block(a8, sa.cpu(), b8, sb), lambda: ops.gemm_e4m3_block(a8, sa, b8, sb, out="e5m2"),
           lambda: ops.gemm_e4m3_block(a8, sa, b8, sb, epilogue="silu"),
           lambda: ops.norm_gate_resid_(y), lambda: ops.norm_gate_resid_(x, y[:3]),
           lambda: ops.norm_gate_resid_(x, y.half()),
           lambda: ops.norm_gate_resid_(x, y, post="batch"), lambda: ops.norm_gate_resid_(x, y, post_w=v),
           lambda: ops.norm_gate_resid_(x, y, post_w=w[:100]), lambda: ops.norm_gate_resid_(x, y, gate=w),
           lambda: ops.norm_gate_resid_(x, y, gate=v.view(1, -1), rows_per_frame=3),
           lambda: ops.norm_gate_resid_(x, y, gate=v, rows_per_frame=3), lambda: ops.norm_gate_resid_(x, y, shift=v),
           lambda: ops.norm_gate_resid_(x, y, rows_per_frame=0), lambda: ops.norm_gate_resid_(x, out=None),
           lambda: ops.norm_gate_resid_(x, gate=v), lambda: ops.norm_gate_resid_(x, resid_scale=2.0),
           lambda: ops.norm_gate_resid_(x, y, pre_w=w, out=None), lambda: ops.norm_gate_resid_(x, y, out="f16"),
           lambda: ops.norm_gate_resid_(x[:, :128], y[:, :128])]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("accepted:", i)
    with pytest.raises(RuntimeError):
        ops.norm_gate_resid_(torch.zeros(2, 16385, device="cuda"))
