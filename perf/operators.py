"""Cases of the block-scaled e4m3 linears and of the norms around them, with their plain forms.

Operators (all of ``fastworld_b200.ops``):

* ``quant_e4m3_block(x)``: rows of x in e4m3 with one power-of-two scale per row and 128 columns;
* ``gemm_e4m3_block(a8, sa, b8, sb, bias, epilogue, out)``: the matrix product of two such operands,
  its result in bf16, fp32, or e4m3 with block scales again (the next product's operand);
* ``norm_gate_resid_(resid, y, ...)``: the norm after a block, its gate and the residual update, and
  the norm and modulation before the next block, in one pass.

The format.  x [R, K] is held as codes q [R, Kp] (uint8 holding e4m3; Kp = K rounded up to 128, zeros
behind K) and exponents s [ceil(Kp / 512), R, 4] (uint8): s[g, r, j] - 127 is the exponent of row r's
columns [128 (4 g + j), 128 (4 g + j + 1)); places behind the last block hold 127.  A block's exponent is
the smallest e (at least -127) with max|x| <= 448 * 2^e, so a stored value is code * 2^e.
"""
import math

import torch

own = False
BLK = 128


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # quantisation: a single row, the FFN hidden rows of one chunk, context rows of an odd width
        {"name": "quant_row", "kind": "quant", "M": 1, "K": 1536, "dtype": "bf16"},
        {"name": "quant_hidden", "kind": "quant", "M": 2640, "K": 8960, "dtype": "bf16"},
        {"name": "quant_ragged_f32", "kind": "quant", "M": 257, "K": 1283, "dtype": "f32"},
        # products: the time projection of one timestep (one row), the text embedding of a prompt, the packed
        # q/k/v projection of a chunk, the FFN-up of the 14B shape, and odd sizes
        {"name": "gemm_row", "kind": "gemm", "M": 1, "N": 9216, "K": 1536, "epilogue": "none", "out": "f32"},
        {"name": "gemm_text_gelu", "kind": "gemm", "M": 512, "N": 1536, "K": 4096, "epilogue": "gelu_tanh", "out": "bf16"},
        {"name": "gemm_qkv", "kind": "gemm", "M": 2640, "N": 4608, "K": 1536, "epilogue": "none", "out": "bf16"},
        {"name": "gemm_14b_up", "kind": "gemm", "M": 4680, "N": 13824, "K": 5120, "epilogue": "gelu_tanh", "out": "bf16"},
        {"name": "gemm_ragged", "kind": "gemm", "M": 1001, "N": 777, "K": 1283, "epilogue": "gelu_erf", "out": "f32"},
        # the feed-forward pair of a chunk: the up product leaves its GELU in e4m3, which the down product reads
        {"name": "ffn_pair", "kind": "ffn", "M": 2640, "D": 1536, "F": 8960},
        # norms: one row, a chunk's sandwich (RMS after the block, LayerNorm and modulation before the next), and the
        # 14B rows with the e4m3 output feeding the q/k/v product
        {"name": "norm_row", "kind": "norm", "M": 1, "D": 1536, "post": "rms", "pre": "rms", "frames": 1},
        {"name": "norm_chunk", "kind": "norm", "M": 2640, "D": 1536, "post": "rms", "pre": "layer", "frames": 3},
        {"name": "norm_then_qkv", "kind": "entry", "M": 4680, "D": 5120, "N": 7680, "post": "layer", "pre": "layer", "frames": 3},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "gemm", "gemm", "gemm", "ffn", "norm", "norm", "entry"])
    if kind == "quant":
        return {"kind": kind, "M": _log(rng, 1, 6032), "K": _log(rng, 60, 13824), "dtype": rng.choice(["bf16", "f16", "f32"])}
    if kind == "gemm":
        while True:
            m, n, k = _log(rng, 1, 6032), _log(rng, 30, 13824), _log(rng, 60, 8960)
            if m * n * k <= 3.3e11:
                break
        return {"kind": kind, "M": m, "N": n, "K": k, "epilogue": rng.choice(["none", "gelu_tanh", "gelu_erf"]),
                "out": rng.choice(["bf16", "f32"])}
    if kind == "ffn":
        d, r = _log(rng, 120, 2048), rng.uniform(1.5, 6.0)
        return {"kind": kind, "M": _log(rng, 1, 4680), "D": d, "F": int(d * r)}
    m, d = _log(rng, 1, 6032), _log(rng, 120, 5120)
    c = {"kind": kind, "M": m, "D": d, "post": rng.choice(["rms", "layer"]), "pre": rng.choice(["rms", "layer"]),
         "frames": rng.randint(1, min(m, 4))}
    return c if kind == "norm" else {**c, "N": _log(rng, 30, 7680)}


# ---------------------------------------------------------------------------------- inputs
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _acts(g, m, k, dtype):
    """Activations: rows of differing size, channels of differing size, a few of them far larger."""
    x = torch.randn(m, k, device="cuda", generator=g)
    ch = torch.exp(0.5 * torch.randn(k, device="cuda", generator=g))
    ch = torch.where(torch.rand(k, device="cuda", generator=g) < 0.005, ch * 20, ch)
    row = torch.exp(0.3 * torch.randn(m, 1, device="cuda", generator=g))
    return (x * ch * row).to(dtype)


def _pack(x):
    """x in the block-scaled format: what a user's program holds of its weights, or got from the call before."""
    m, k = x.shape
    nb = -(-k // BLK)
    xp = torch.nn.functional.pad(x.float(), (0, nb * BLK - k)).view(m, nb, BLK)
    e = _exponents(xp.abs().amax(-1))
    q = (xp * _pow2(-e)[..., None]).to(torch.float8_e4m3fn).view(torch.uint8).view(m, nb * BLK)
    return q.contiguous(), _layout(e)


def _exponents(amax):
    """Smallest e >= -127 with amax <= 448 * 2^e."""
    f, e = torch.frexp(amax)                     # amax = f * 2^e, f in [0.5, 1); 448 = 0.875 * 2^9
    e = e - 9 + (f > 0.875).to(e.dtype)
    return torch.where(amax > 0, e.clamp_min(-127), torch.full_like(e, -127))


def _pow2(e):
    """2^e in fp32 for e in [-126, 127], from the exponent field."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _layout(e):
    """Exponents [R, blocks] as s [ceil(blocks / 4), R, 4]."""
    r, nb = e.shape
    ng = -(-nb // 4)
    s = torch.full((r, ng * 4), 127, dtype=torch.uint8, device=e.device)
    s[:, :nb] = (e + 127).to(torch.uint8)
    return s.view(r, ng, 4).permute(1, 0, 2).contiguous()


def _frames(case):
    return -(-case["M"] // case["frames"])      # rows of a frame


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, m = case["kind"], case["M"]

    def weight(n, k):
        return _pack((torch.randn(n, k, device="cuda", generator=g) / math.sqrt(k)).to(torch.bfloat16))

    def vec(n, size, mean=0.0, dtype=torch.float32, rows=None):
        shape = (n,) if rows is None else (rows, n)
        return (torch.randn(*shape, device="cuda", generator=g) * size + mean).to(dtype)

    s = {"case": case}
    if kind == "quant":
        s["x"] = _acts(g, m, case["K"], DT[case["dtype"]])
    elif kind == "gemm":
        s["a8"], s["sa"] = _pack(_acts(g, m, case["K"], torch.bfloat16))
        s["b8"], s["sb"] = weight(case["N"], case["K"])
        s["bias"] = vec(case["N"], 0.1, dtype=torch.bfloat16)
    elif kind == "ffn":
        s["a8"], s["sa"] = _pack(_acts(g, m, case["D"], torch.bfloat16))
        s["up8"], s["sup"] = weight(case["F"], case["D"])
        s["down8"], s["sdown"] = weight(case["D"], case["F"])
        s["b1"], s["b2"] = vec(case["F"], 0.1, dtype=torch.bfloat16), vec(case["D"], 0.1, dtype=torch.bfloat16)
    else:
        d, fr = case["D"], -(-m // _frames(case))
        s["resid"] = _acts(g, m, d, torch.float32)
        s["y"] = _acts(g, m, d, torch.bfloat16)
        s["post_w"] = vec(d, 0.2, 1.0, torch.bfloat16)
        s["gate"], s["shift"], s["scale"] = (vec(d, 0.3, mu, rows=fr) for mu in (0.5, 0.0, 0.0))
        if kind == "entry":
            s["w8"], s["sw"] = weight(case["N"], d)
            s["bias"] = vec(case["N"], 0.1, dtype=torch.bfloat16)
    return s


# ---------------------------------------------------------------------------------- one pass
def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from fastworld_b200 import ops
    c = s["case"]
    if c["kind"] == "quant":
        q, e = ops.quant_e4m3_block(s["x"])
        return q.view(torch.float8_e4m3fn), e
    if c["kind"] == "gemm":
        return ops.gemm_e4m3_block(s["a8"], s["sa"], s["b8"], s["sb"], s["bias"], epilogue=c["epilogue"], out=c["out"])
    if c["kind"] == "ffn":
        h8, sh = ops.gemm_e4m3_block(s["a8"], s["sa"], s["up8"], s["sup"], s["b1"], epilogue="gelu_tanh", out="e4m3")
        return ops.gemm_e4m3_block(h8, sh, s["down8"], s["sdown"], s["b2"])
    h = ops.norm_gate_resid_(s["resid"], s["y"], post=c["post"], post_w=s["post_w"], gate=s["gate"], branch_scale=0.5,
                             pre=c["pre"], shift=s["shift"], scale=s["scale"], rows_per_frame=_frames(c),
                             out="bf16" if c["kind"] == "norm" else "e4m3")
    if c["kind"] == "norm":
        return s["resid"], h
    return s["resid"], ops.gemm_e4m3_block(h[0], h[1], s["w8"], s["sw"], s["bias"])


def _deq(q, s):
    """fp32 values [R, Kp] of codes and exponents."""
    r, kp = q.shape
    e = s.permute(1, 0, 2).reshape(r, -1)[:, :kp // BLK].to(torch.int32) - 127
    v = q.view(torch.float8_e4m3fn).float().view(r, kp // BLK, BLK)
    return (v * torch.exp2(e.double()).float()[..., None]).view(r, kp)


def _plain_quant(x):
    m, k = x.shape
    nb = -(-k // BLK)
    xp = torch.zeros(m, nb * BLK, device=x.device)
    xp[:, :k] = x
    xp = xp.view(m, nb, BLK)
    e = _exponents(xp.abs().amax(-1))
    return (xp * _pow2(-e)[..., None]).to(torch.float8_e4m3fn).view(m, nb * BLK), _layout(e)


def _act(v, name):
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _plain_norm(v, kind):
    """fp32 statistics over the row; eps = 1e-6."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6)


def _plain(s):
    c = s["case"]
    if c["kind"] == "quant":
        return _plain_quant(s["x"])
    if c["kind"] == "gemm":
        v = _deq(s["a8"], s["sa"]) @ _deq(s["b8"], s["sb"]).t() + s["bias"].float()
        return _act(v, c["epilogue"]).to(DT[c["out"]])
    if c["kind"] == "ffn":
        h = _act(_deq(s["a8"], s["sa"]) @ _deq(s["up8"], s["sup"]).t() + s["b1"].float(), "gelu_tanh")
        q, e = _plain_quant(h)
        return (_deq(q.view(torch.uint8), e) @ _deq(s["down8"], s["sdown"]).t() + s["b2"].float()).to(torch.bfloat16)
    frame = torch.arange(c["M"], device="cuda") // _frames(c)
    branch = _plain_norm(s["y"].float(), c["post"]) * s["post_w"].float() * s["gate"][frame]
    s["resid"] += 0.5 * branch
    h = _plain_norm(s["resid"], c["pre"]) * (1 + s["scale"][frame]) + s["shift"][frame]
    if c["kind"] == "norm":
        return s["resid"], h.to(torch.bfloat16)
    q, e = _plain_quant(h)
    return s["resid"], (_deq(q.view(torch.uint8), e) @ _deq(s["w8"], s["sw"]).t() + s["bias"].float()).to(torch.bfloat16)


# ---------------------------------------------------------------------------------- in 64 bits
def _exact_codes(v):
    """Codes (as the e4m3 values they stand for, fp64) and unbiased exponents of fp64 rows, by the definition of the
    formats: the nearest multiple of the step 2^max(floor(log2|c|) - 3, -9), ties to the even multiple."""
    r, k = v.shape
    nb = (k + BLK - 1) // BLK
    w = torch.cat([v, v.new_zeros(r, nb * BLK - k)], 1).reshape(r, nb, BLK)
    top = w.abs().max(-1).values
    e = torch.ceil(torch.log2(top / 448)).nan_to_num(neginf=-127).clamp_min(-127)
    e = torch.where(top > 448 * torch.exp2(e), e + 1, e)                       # where log2 rounded
    e = torch.where((e > -127) & (top <= 448 * torch.exp2(e - 1)), e - 1, e)
    c = w * torch.exp2(-e)[..., None]
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(c.abs().clamp_min(1e-300))), min=-6) - 3)
    return (torch.round(c / step) * step).reshape(r, nb * BLK), e


def _exact_values(q, s):
    bits = q.to(torch.int64)
    ex, mant = (bits >> 3) & 15, (bits & 7).double()
    mag = torch.where(ex > 0, torch.exp2((ex - 7).double()) * (1 + mant / 8), torch.exp2(mant.new_tensor(-6.0)) * mant / 8)
    v = torch.where(bits >= 128, -mag, mag)
    e = torch.cat(list(s), 1)[:, :q.shape[1] // BLK].double() - 127            # groups of four side by side
    return v * torch.exp2(e).repeat_interleave(BLK, 1)


def _exact_act(v, name):
    if name == "gelu_tanh":
        u = math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)
        return v * torch.sigmoid(u)                                            # (1 + tanh(u / 2)) / 2
    return v * 0.5 * torch.special.erfc(-v / math.sqrt(2)) if name == "gelu_erf" else v


def _exact_norm(v, kind):
    mu = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    var = ((v - mu) ** 2).mean(1, keepdim=True)
    return (v - mu) / torch.sqrt(var + 1e-6)


def exact(case, seed):
    s = prepare(case, seed)
    kind, m = case["kind"], case["M"]
    if kind == "quant":
        c, e = _exact_codes(s["x"].double())
        nb = e.shape[1]
        full = e.new_zeros(m, (nb + 3) // 4 * 4)
        full[:, :nb] = e
        return c, torch.stack(full.split(4, 1)).add(127).to(torch.uint8)
    if kind == "gemm":
        v = _exact_values(s["a8"], s["sa"]) @ _exact_values(s["b8"], s["sb"]).T + s["bias"].double()
        return _exact_act(v, case["epilogue"])
    if kind == "ffn":
        h = _exact_act(_exact_values(s["a8"], s["sa"]) @ _exact_values(s["up8"], s["sup"]).T + s["b1"].double(), "gelu_tanh")
        c, e = _exact_codes(h)
        h = c * torch.exp2(e).repeat_interleave(BLK, 1)
        return h @ _exact_values(s["down8"], s["sdown"]).T + s["b2"].double()
    rows = _frames(case)
    gate, shift, scale = (s[n].double().repeat_interleave(rows, 0)[:m] for n in ("gate", "shift", "scale"))
    x = s["resid"].double() + _exact_norm(s["y"].double(), case["post"]) * s["post_w"].double() * gate / 2
    h = _exact_norm(x, case["pre"]) * (scale + 1) + shift
    if kind == "norm":
        return x, h
    c, e = _exact_codes(h)
    h = c * torch.exp2(e).repeat_interleave(BLK, 1)
    return x, h @ _exact_values(s["w8"], s["sw"]).T + s["bias"].double()


# ---------------------------------------------------------------------------------- what a pass cannot do without
def _packed_bytes(r, k):
    """Codes and the exponents in use."""
    return r * k + r * -(-k // BLK)


def work(case):
    kind, m = case["kind"], case["M"]
    if kind == "quant":
        k = case["K"]
        return {"bytes": m * k * (4 if case["dtype"] == "f32" else 2) + _packed_bytes(m, k), "flops": 3 * m * k}
    if kind == "gemm":
        n, k = case["N"], case["K"]
        return {"bytes": _packed_bytes(m, k) + _packed_bytes(n, k) + 2 * n + m * n * (4 if case["out"] == "f32" else 2),
                "flops": 2 * m * n * k}
    if kind == "ffn":
        d, f = case["D"], case["F"]
        return {"bytes": _packed_bytes(m, d) + _packed_bytes(f, d) + _packed_bytes(d, f) + 2 * (d + f) + 2 * m * d,
                "flops": 4 * m * d * f}
    d = case["D"]
    params = 2 * d + 12 * d * case["frames"]
    if kind == "norm":
        return {"bytes": m * d * (4 + 4 + 2 + 2) + params, "flops": 16 * m * d}
    n = case["N"]
    return {"bytes": m * d * (4 + 4 + 2) + params + _packed_bytes(n, d) + 2 * n + 2 * m * n, "flops": 16 * m * d + 2 * m * n * d}
