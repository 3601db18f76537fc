"""Torch-facing wrappers of the op-level C ABI (device tensors in, device tensors out).

These call the sm_100a kernels directly; there is no fallback: a tensor on the wrong device
or with the wrong dtype/layout raises.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check, lib, ptr, stream_ptr

EPILOGUES = {"none": _lib.EPI_BF16, "gelu_tanh": _lib.EPI_GELU_BF16, "f32": _lib.EPI_F32,
             "gelu_erf": _lib.EPI_GELU_ERF_BF16}


BLOCK_EPILOGUES = {"none": _lib.EPI_BF16, "gelu_tanh": _lib.EPI_GELU_BF16, "gelu_erf": _lib.EPI_GELU_ERF_BF16}
BLOCK_OUTPUTS = {"bf16": (_lib.DT_BF16, torch.bfloat16), "f32": (_lib.DT_F32, torch.float32),
                 "e4m3": (_lib.DT_U8, torch.uint8)}
NORMS = {None: _lib.NORM_NONE, "layer": _lib.NORM_LAYER, "rms": _lib.NORM_RMS}
_DTYPES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16, torch.float32: _lib.DT_F32}


def _req(t, dtype, name):
    if not (t.is_cuda and t.dtype == dtype and t.is_contiguous()):
        raise ValueError(f"{name}: expected a contiguous CUDA {dtype} tensor, got {t.dtype} on {t.device}")


def gemm(a: torch.Tensor, b: torch.Tensor, bias=None, epilogue: str = "none", tile_n: int = 0) -> torch.Tensor:
    """a [M, K] @ b[N, K]^T (+ bias) with fp32 accumulation; bf16 (or fp32 for 'f32') output."""
    _req(a, torch.bfloat16, "a")
    _req(b, torch.bfloat16, "b")
    if bias is not None:
        _req(bias, torch.bfloat16, "bias")
    M, K = a.shape
    N = b.shape[0]
    out = torch.empty(M, N, device=a.device, dtype=torch.float32 if epilogue == "f32" else torch.bfloat16)
    check(lib().fw_gemm_bf16(ptr(a), ptr(b), ptr(bias), ptr(out), M, N, K, EPILOGUES[epilogue], tile_n,
                             stream_ptr()), "gemm")
    return out


def quant_e4m3(x: torch.Tensor):
    """Per-row e4m3 quantisation: returns (q [M, K] uint8 e4m3 bits, scale [M] fp32)."""
    _req(x, torch.bfloat16, "x")
    M, K = x.shape
    q = torch.empty(M, K, device=x.device, dtype=torch.uint8)
    sc = torch.empty(M, device=x.device, dtype=torch.float32)
    check(lib().fw_quant_e4m3(ptr(x), M, K, ptr(q), ptr(sc), stream_ptr()), "quant_e4m3")
    return q, sc


def gemm_e4m3(a8: torch.Tensor, sa: torch.Tensor, b8: torch.Tensor, sw: torch.Tensor, bias=None,
              epilogue: str = "none", tile_n: int = 0) -> torch.Tensor:
    """(a8 [M, K] e4m3 * sa[M]) @ (b8 [N, K] e4m3 * sw[N])^T (+ bias), fp32 accumulation."""
    for n, t, d in (("a8", a8, torch.uint8), ("b8", b8, torch.uint8), ("sa", sa, torch.float32),
                    ("sw", sw, torch.float32)):
        _req(t, d, n)
    M, K = a8.shape
    N = b8.shape[0]
    out = torch.empty(M, N, device=a8.device, dtype=torch.float32 if epilogue == "f32" else torch.bfloat16)
    check(lib().fw_gemm_e4m3(ptr(a8), ptr(sa), ptr(b8), ptr(sw), ptr(bias), ptr(out), M, N, K, EPILOGUES[epilogue],
                             tile_n, stream_ptr()), "gemm_e4m3")
    return out


def gemm_resid_(resid: torch.Tensor, a: torch.Tensor, b: torch.Tensor, bias=None, gate=None,
                rows_per_frame: int = 1 << 30) -> torch.Tensor:
    """resid (fp32, in place) += gate[row // rows_per_frame] * (a @ b^T + bias)."""
    _req(resid, torch.float32, "resid")
    _req(a, torch.bfloat16, "a")
    _req(b, torch.bfloat16, "b")
    if gate is not None:
        _req(gate, torch.float32, "gate")
    M, K = a.shape
    N = b.shape[0]
    check(lib().fw_gemm_bf16_resid(ptr(a), ptr(b), ptr(bias), ptr(resid), ptr(gate), rows_per_frame, M, N, K,
                                   stream_ptr()), "gemm_resid")
    return resid


def attention(q: torch.Tensor, k0: torch.Tensor, v0: torch.Tensor, k1: torch.Tensor, v1: torch.Tensor,
              meta: torch.Tensor, status: torch.Tensor = None) -> torch.Tensor:
    """Non-causal attention of q [Lq, H, 128] over keys [k0[:n0] | k1[:n1]] with
    meta = device int32 (n0, n1).  Returns [Lq, H * 128] bf16."""
    for n, t in (("q", q), ("k0", k0), ("v0", v0), ("k1", k1), ("v1", v1)):
        _req(t, torch.bfloat16, n)
    _req(meta, torch.int32, "meta")
    Lq, H, Dh = q.shape
    assert Dh == 128
    out = torch.empty(Lq, H * Dh, device=q.device, dtype=torch.bfloat16)
    check(lib().fw_attention(ptr(q), Lq, H, ptr(k0), ptr(v0), k0.shape[0], ptr(k1), ptr(v1), k1.shape[0], ptr(meta),
                             ptr(out), ptr(status), stream_ptr()), "attention")
    return out


def copy_(dst: torch.Tensor, src: torch.Tensor) -> torch.Tensor:
    """Byte copy src -> dst with the vectorised copy kernel (same byte size)."""
    nb = dst.numel() * dst.element_size()
    if src.numel() * src.element_size() != nb or not (dst.is_contiguous() and src.is_contiguous()):
        raise ValueError("copy_: contiguous tensors of equal byte size required")
    check(lib().fw_copy(ptr(dst), ptr(src), nb, stream_ptr()), "copy")
    return dst


def layernorm(x: torch.Tensor, eps: float = 1e-6, shift=None, scale=None, w=None, b=None, out=None) -> torch.Tensor:
    """bf16 LN(x) of fp32 rows x [M, D], then * (1 + scale) + shift (fp32 [D]) or * w + b (bf16 [D])."""
    _req(x, torch.float32, "x")
    for n, t, d in (("shift", shift, torch.float32), ("scale", scale, torch.float32), ("w", w, torch.bfloat16),
                    ("b", b, torch.bfloat16)):
        if t is not None:
            _req(t, d, n)
    M, D = x.shape
    out = torch.empty(M, D, device=x.device, dtype=torch.bfloat16) if out is None else out
    _req(out, torch.bfloat16, "out")
    check(lib().fw_layernorm(ptr(x), M, D, float(eps), ptr(shift), ptr(scale), ptr(w), ptr(b), ptr(out),
                             stream_ptr()), "layernorm")
    return out


def rms_rope(x: torch.Tensor, w: torch.Tensor, rope=None, head_dim: int = 128, eps: float = 1e-6,
             out=None) -> torch.Tensor:
    """bf16 RMSNorm(x) * w over the full row of x [M, D], then RoPE of every head's (even, odd)
    pairs by rope [M, head_dim // 2, 2] (cos, sin) fp32 when given."""
    _req(x, torch.bfloat16, "x")
    _req(w, torch.bfloat16, "w")
    if rope is not None:
        _req(rope, torch.float32, "rope")
    M, D = x.shape
    out = torch.empty_like(x) if out is None else out
    check(lib().fw_rms_rope(ptr(x), M, D, float(eps), ptr(w), ptr(rope), head_dim, ptr(out), stream_ptr()),
          "rms_rope")
    return out


# ---------------------------------------------------------------- block-scaled e4m3
# An operand x [R, K] is a pair (q, s): e4m3 codes q [R, Kp] (uint8; Kp = K rounded up to 128, zeros behind
# K) and exponents s [ceil(Kp / 512), R, 4] (uint8): s[g, r, j] - 127 is the power of two that scales
# row r's columns [128 (4 g + j), + 128); places behind the last block hold 127.
def _on(dev, fn, what, *args):
    """fn(*args, stream) on dev's current stream, with dev as the current device."""
    if torch.cuda.current_device() == dev.index:
        check(fn(*args, stream_ptr()), what)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, stream_ptr()), what)


def _same_device(dev, **tensors):
    for n, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{n}: on {t.device}, expected {dev}")


def _shape(t, shape, name):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")


def _block_empty(rows, cols, dev):
    """Uninitialised codes and exponents of a [rows, cols] operand."""
    kp = -(-cols // 128) * 128
    return (torch.empty(rows, kp, device=dev, dtype=torch.uint8),
            torch.empty(-(-kp // 512), rows, 4, device=dev, dtype=torch.uint8))


def _block_req(q, s, name):
    """Checks an operand's codes and exponents; returns its rows and padded columns."""
    _req(q, torch.uint8, name + "8")
    _req(s, torch.uint8, "s" + name)
    if q.ndim != 2 or q.shape[1] == 0 or q.shape[1] % 128:
        raise ValueError(f"{name}8: shape {tuple(q.shape)}, expected [rows, a positive multiple of 128]")
    _shape(s, (-(-q.shape[1] // 512), q.shape[0], 4), "s" + name)
    return q.shape


def quant_e4m3_block(x: torch.Tensor):
    """x [M, K] (bf16, fp16 or fp32) in block-scaled e4m3: (q [M, Kp], s [ceil(Kp / 512), M, 4]), both
    uint8.  Each row's 128 columns share the smallest power of two 2^e (e >= -127) with
    max|x| <= 448 * 2^e over the finite elements; NaN and infinities become the NaN code."""
    if x.dtype not in _DTYPES:
        raise ValueError(f"x: expected bf16, fp16 or fp32, got {x.dtype}")
    _req(x, x.dtype, "x")
    if x.ndim != 2 or x.shape[1] == 0:
        raise ValueError(f"x: shape {tuple(x.shape)}, expected [M, K] with K > 0")
    M, K = x.shape
    q, s = _block_empty(M, K, x.device)
    _on(x.device, lib().fw_quant_e4m3_block, "quant_e4m3_block", ptr(x), _DTYPES[x.dtype], M, K, ptr(q), ptr(s))
    return q, s


def gemm_e4m3_block(a8: torch.Tensor, sa: torch.Tensor, b8: torch.Tensor, sb: torch.Tensor, bias=None,
                    epilogue: str = "none", out: str = "bf16"):
    """act(A @ B^T + bias) of block-scaled e4m3 A [M, K] and B [N, K] (quant_e4m3_block), fp32 accumulation.
    epilogue: 'none', 'gelu_tanh' or 'gelu_erf'; bias bf16 [N].  out: 'bf16' or 'f32' [M, N], or 'e4m3': the
    pair (q, s) of the result, quantised from fp32, as the next product takes it."""
    if epilogue not in BLOCK_EPILOGUES:
        raise ValueError(f"epilogue: {epilogue!r}, expected one of {sorted(BLOCK_EPILOGUES)}")
    if out not in BLOCK_OUTPUTS:
        raise ValueError(f"out: {out!r}, expected one of {sorted(BLOCK_OUTPUTS)}")
    M, K = _block_req(a8, sa, "a")
    N, Kb = _block_req(b8, sb, "b")
    if K != Kb:
        raise ValueError(f"a8 and b8 have {K} and {Kb} columns")
    if bias is not None:
        _req(bias, torch.bfloat16, "bias")
        _shape(bias, (N,), "bias")
    _same_device(a8.device, sa=sa, b8=b8, sb=sb, bias=bias)
    code, dtype = BLOCK_OUTPUTS[out]
    if out == "e4m3":
        if N == 0:
            raise ValueError("out: e4m3 of no columns")
        o, so = _block_empty(M, N, a8.device)
    else:
        o, so = torch.empty(M, N, device=a8.device, dtype=dtype), None
    _on(a8.device, lib().fw_gemm_e4m3_block, "gemm_e4m3_block", ptr(a8), ptr(sa), ptr(b8), ptr(sb), ptr(bias), ptr(o),
        ptr(so), M, N, K, BLOCK_EPILOGUES[epilogue], code)
    return o if so is None else (o, so)


def norm_gate_resid_(resid: torch.Tensor, y=None, post=None, post_w=None, post_b=None, gate=None,
                     resid_scale: float = 1.0, branch_scale: float = 1.0, pre="layer", pre_w=None, pre_b=None,
                     shift=None, scale=None, rows_per_frame=None, eps: float = 1e-6, out="bf16"):
    """The norm after a block, its gate and the residual update, and the norm before the next block:

        resid = resid_scale * resid + branch_scale * gate[f] * (post(y) * post_w + post_b)      (in place)
        h = (pre(resid) * pre_w + pre_b) * (1 + scale[f]) + shift[f]                            (returned)

    resid fp32 [M, D]; y bf16 or fp32 [M, D], or None (no residual update); post and pre 'layer', 'rms' or None,
    fp32 statistics; weights bf16 [D]; gate, shift and scale fp32 [frames, D] (or [D], one frame) with
    f = row // rows_per_frame (None: all rows are one frame).  out: 'bf16', 'e4m3' (the pair (q, s) of
    quant_e4m3_block, quantised from fp32) or None (h is not computed)."""
    _req(resid, torch.float32, "resid")
    if resid.ndim != 2 or resid.shape[1] == 0:
        raise ValueError(f"resid: shape {tuple(resid.shape)}, expected [M, D] with D > 0")
    M, D = resid.shape
    if post not in NORMS or pre not in NORMS:
        raise ValueError(f"post, pre: {post!r}, {pre!r}, expected 'layer', 'rms' or None")
    if out not in ("bf16", "e4m3", None):
        raise ValueError(f"out: {out!r}, expected 'bf16', 'e4m3' or None")
    if y is None and out is None:
        raise ValueError("nothing to do: no y and no output")
    if y is None and not (post is None and post_w is None and post_b is None and gate is None and resid_scale == 1.0
                          and branch_scale == 1.0):
        raise ValueError("post, post_w, post_b, gate, resid_scale and branch_scale need y")
    if out is None and not (pre_w is None and pre_b is None and shift is None and scale is None):
        raise ValueError("pre_w, pre_b, shift and scale need an output")
    if (shift is None) != (scale is None):
        raise ValueError("shift and scale come together")
    rpf = max(M, 1) if rows_per_frame is None else int(rows_per_frame)
    if rpf <= 0:
        raise ValueError(f"rows_per_frame: {rows_per_frame}")
    if y is not None:
        if y.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"y: expected bf16 or fp32, got {y.dtype}")
        _req(y, y.dtype, "y")
        _shape(y, (M, D), "y")
    for n, t in (("post_w", post_w), ("post_b", post_b), ("pre_w", pre_w), ("pre_b", pre_b)):
        if t is not None:
            _req(t, torch.bfloat16, n)
            _shape(t, (D,), n)
    frames = -(-M // rpf)
    for n, t in (("gate", gate), ("shift", shift), ("scale", scale)):
        if t is not None:
            _req(t, torch.float32, n)
            rows = 1 if t.ndim == 1 else t.shape[0]
            if t.ndim not in (1, 2) or t.shape[-1] != D or rows < frames:
                raise ValueError(f"{n}: shape {tuple(t.shape)}, expected [{frames}, {D}]" + (f" or [{D}]" * (frames <= 1)))
    _same_device(resid.device, y=y, post_w=post_w, post_b=post_b, gate=gate, pre_w=pre_w, pre_b=pre_b, shift=shift,
                 scale=scale)
    h = s = None
    if out == "e4m3":
        h, s = _block_empty(M, D, resid.device)
    elif out == "bf16":
        h = torch.empty(M, D, device=resid.device, dtype=torch.bfloat16)
    a = _lib.FwNormArgs(ptr(resid), ptr(y), _DTYPES[torch.bfloat16 if y is None else y.dtype], NORMS[post], NORMS[pre],
                        ptr(post_w), ptr(post_b), ptr(pre_w), ptr(pre_b), ptr(gate), ptr(shift), ptr(scale),
                        resid_scale, branch_scale, eps, M, D, min(rpf, 2**31 - 1), ptr(h), ptr(s))
    _on(resid.device, lib().fw_norm_gate_resid, "norm_gate_resid", ctypes.byref(a))
    return (h, s) if out == "e4m3" else h
