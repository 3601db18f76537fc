"""Torch-facing wrappers of the op-level C ABI (device tensors in, device tensors out).

These call the sm_100a kernels directly; there is no fallback: a tensor on the wrong device
or with the wrong dtype/layout raises.
"""
from __future__ import annotations

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
def _on(index, fn, what, *args):
    """fn(*args, stream) on the current stream of device `index`, with that device as the current one."""
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, what)


def _block_empty(rows, cols, dev):
    """Uninitialised codes and exponents of a [rows, cols] operand."""
    kp = -(-cols // 128) * 128
    return (torch.empty(rows, kp, device=dev, dtype=torch.uint8),
            torch.empty(-(-kp // 512), rows, 4, device=dev, dtype=torch.uint8))


def _is(t, dtype, index):
    return t.dtype is dtype and t.get_device() == index and t.is_contiguous()


def _refuse(name, t, dtype, index, shape):
    where = f"cuda:{index}" if index >= 0 else "a CUDA device"
    raise ValueError(f"{name}: expected a contiguous {dtype} tensor of shape {shape} on {where}, got {t.dtype} "
                     f"{tuple(t.shape)} with strides {t.stride()} on {t.device}")


def quant_e4m3_block(x: torch.Tensor):
    """x [M, K] (bf16, fp16 or fp32) in block-scaled e4m3: (q [M, Kp], s [ceil(Kp / 512), M, 4]), both
    uint8.  Each row's 128 columns share the smallest power of two 2^e (e >= -127) with
    max|x| <= 448 * 2^e over the finite elements; NaN and infinities become the NaN code."""
    dtype, index, shape = _DTYPES.get(x.dtype), x.get_device(), x.shape
    if (dtype is None or index < 0 or len(shape) != 2 or not 0 < shape[1] <= _lib.BLOCK_MAX_COLS
            or not x.is_contiguous()):
        _refuse("x", x, "bf16, fp16 or fp32", index, f"[M, 0 < K <= {_lib.BLOCK_MAX_COLS}]")
    M, K = shape
    q, s = _block_empty(M, K, x.device)
    _on(index, lib().fw_quant_e4m3_block, "quant_e4m3_block", x.data_ptr(), dtype, M, K, q.data_ptr(), s.data_ptr())
    return q, s


def gemm_e4m3_block(a8: torch.Tensor, sa: torch.Tensor, b8: torch.Tensor, sb: torch.Tensor, bias=None,
                    epilogue: str = "none", out: str = "bf16", status: torch.Tensor = None):
    """act(A @ B^T + bias) of block-scaled e4m3 A [M, K] and B [N, K] (quant_e4m3_block), fp32 accumulation.
    epilogue: 'none', 'gelu_tanh' or 'gelu_erf'; bias bf16 [N].  out: 'bf16' or 'f32' [M, N], or 'e4m3': the
    pair (q, s) of the result, quantised from fp32, as the next product takes it.  status: int32, zeroed by the caller;
    where a wait of the kernel runs out, its first word receives a code and parts of the result are not written."""
    if epilogue not in BLOCK_EPILOGUES:
        raise ValueError(f"epilogue: {epilogue!r}, expected one of {sorted(BLOCK_EPILOGUES)}")
    if out not in BLOCK_OUTPUTS:
        raise ValueError(f"out: {out!r}, expected one of {sorted(BLOCK_OUTPUTS)}")
    u8, index, shape = torch.uint8, a8.get_device(), a8.shape
    if (index < 0 or len(shape) != 2 or not 0 < shape[1] <= _lib.BLOCK_MAX_COLS or shape[1] % 128
            or not _is(a8, u8, index)):
        _refuse("a8", a8, u8, index, f"[M, a multiple of 128 from 128 to {_lib.BLOCK_MAX_COLS}]")
    M, K = shape
    shape = b8.shape
    if len(shape) != 2 or shape[0] > _lib.BLOCK_MAX_COLS or shape[1] != K or not _is(b8, u8, index):
        _refuse("b8", b8, u8, index, f"[N <= {_lib.BLOCK_MAX_COLS}, {K}]")
    N, groups = shape[0], -(-K // 512)
    if sa.shape != (groups, M, 4) or not _is(sa, u8, index):
        _refuse("sa", sa, u8, index, [groups, M, 4])
    if sb.shape != (groups, N, 4) or not _is(sb, u8, index):
        _refuse("sb", sb, u8, index, [groups, N, 4])
    if bias is not None and (bias.shape != (N,) or not _is(bias, torch.bfloat16, index)):
        _refuse("bias", bias, torch.bfloat16, index, [N])
    if status is not None and (status.numel() == 0 or not _is(status, torch.int32, index)):
        _refuse("status", status, torch.int32, index, "[at least 1]")
    code, dtype = BLOCK_OUTPUTS[out]
    if out == "e4m3":
        if N == 0:
            raise ValueError("out: e4m3 of no columns")
        o, so = _block_empty(M, N, a8.device)
    else:
        o, so = torch.empty(M, N, device=a8.device, dtype=dtype), None
    _on(index, lib().fw_gemm_e4m3_block_status, "gemm_e4m3_block", a8.data_ptr(), sa.data_ptr(), b8.data_ptr(),
        sb.data_ptr(), ptr(bias), o.data_ptr(), ptr(so), M, N, K, BLOCK_EPILOGUES[epilogue], code, ptr(status))
    return o if so is None else (o, so)


def _weight(name, t, D, index):
    if t.dtype is not torch.bfloat16 or t.shape != (D,) or t.get_device() != index or not t.is_contiguous():
        _refuse(name, t, torch.bfloat16, index, [D])


def _per_frame(name, t, frames, D, index):
    """fp32 [at least frames, D], or [D] for one frame."""
    shape = t.shape
    if (t.dtype is not torch.float32 or shape[-1:] != (D,) or t.get_device() != index or not t.is_contiguous()
            or not (len(shape) == 2 and shape[0] >= frames or len(shape) == 1 and frames <= 1)):
        _refuse(name, t, torch.float32, index, f"[{frames}, {D}]" + (f" or [{D}]" if frames <= 1 else ""))


def norm_gate_resid_(resid: torch.Tensor, y=None, post=None, post_w=None, post_b=None, gate=None,
                     resid_scale: float = 1.0, branch_scale: float = 1.0, pre="layer", pre_w=None, pre_b=None,
                     shift=None, scale=None, rows_per_frame=None, eps: float = 1e-6, out="bf16"):
    """The norm after a block, its gate and the residual update, and the norm before the next block:

        resid = resid_scale * resid + branch_scale * gate[f] * (post(y) * post_w + post_b)      (in place)
        h = (pre(resid) * pre_w + pre_b) * (1 + scale[f]) + shift[f]                            (returned)

    resid fp32 [M, D]; y bf16 or fp32 [M, D], or None (no residual update); post and pre 'layer', 'rms' or None,
    fp32 statistics; weights bf16 [D]; gate, shift and scale fp32 [frames, D] (or [D], one frame) with
    f = row // rows_per_frame (None: all rows are one frame).  out: 'bf16', 'e4m3' (the pair (q, s) of
    quant_e4m3_block, quantised from fp32) or None (h is not computed).  resid's memory may be y's as a whole
    (fp32), and otherwise overlaps no argument."""
    f32, b16, index, shape = torch.float32, torch.bfloat16, resid.get_device(), resid.shape
    if (index < 0 or len(shape) != 2 or shape[1] == 0 or max(shape) > 0x7fffffff or resid.dtype is not f32
            or not resid.is_contiguous()):
        _refuse("resid", resid, f32, index, f"[M, 0 < D <= {_lib.NORM_MAX_COLS}], M below 2^31")
    M, D = shape
    if post not in NORMS or pre not in NORMS:
        raise ValueError(f"post, pre: {post!r}, {pre!r}, expected 'layer', 'rms' or None")
    if out not in ("bf16", "e4m3", None):
        raise ValueError(f"out: {out!r}, expected 'bf16', 'e4m3' or None")
    rpf = (M or 1) if rows_per_frame is None else int(rows_per_frame)
    if rpf <= 0 or rows_per_frame is not None and rpf != rows_per_frame:
        raise ValueError(f"rows_per_frame: {rows_per_frame}, expected a positive whole number")
    frames = -(-M // rpf)
    if y is None:
        if out is None:
            raise ValueError("nothing to do: no y and no output")
        if not (post is None and post_w is None and post_b is None and gate is None and resid_scale == 1.0
                and branch_scale == 1.0):
            raise ValueError("post, post_w, post_b, gate, resid_scale and branch_scale need y")
    else:
        if ((y.dtype is not b16 and y.dtype is not f32) or y.shape != shape or y.get_device() != index
                or not y.is_contiguous()):
            _refuse("y", y, "bf16 or fp32", index, [M, D])
        if post_w is not None:
            _weight("post_w", post_w, D, index)
        if post_b is not None:
            _weight("post_b", post_b, D, index)
        if gate is not None:
            _per_frame("gate", gate, frames, D, index)
    if out is None and not (pre_w is None and pre_b is None and shift is None and scale is None):
        raise ValueError("pre_w, pre_b, shift and scale need an output")
    if (shift is None) != (scale is None):
        raise ValueError("shift and scale come together")
    if shift is not None:
        _per_frame("shift", shift, frames, D, index)
        _per_frame("scale", scale, frames, D, index)
    if pre_w is not None:
        _weight("pre_w", pre_w, D, index)
    if pre_b is not None:
        _weight("pre_b", pre_b, D, index)
    h = s = None
    if out == "e4m3":
        h, s = _block_empty(M, D, resid.device)
    elif out == "bf16":
        h = torch.empty(M, D, device=resid.device, dtype=b16)
    args = _lib.NORM_ARGS.pack(
        resid.data_ptr(), 0 if y is None else y.data_ptr(),
        _lib.DT_F32 if y is not None and y.dtype is f32 else _lib.DT_BF16,
        NORMS[post], NORMS[pre], 0 if post_w is None else post_w.data_ptr(), 0 if post_b is None else post_b.data_ptr(),
        0 if pre_w is None else pre_w.data_ptr(), 0 if pre_b is None else pre_b.data_ptr(),
        0 if gate is None else gate.data_ptr(), 0 if shift is None else shift.data_ptr(),
        0 if scale is None else scale.data_ptr(), resid_scale, branch_scale, eps, M, D, min(rpf, 2**31 - 1),
        0 if h is None else h.data_ptr(), 0 if s is None else s.data_ptr())
    _on(index, lib().fw_norm_gate_resid, "norm_gate_resid", args)
    return h if s is None else (h, s)
