"""Operators of a feed-forward layer around the fp8 products of ops.py:

    gemm_epilogue(a, b, ...)        act(A @ B * scales + bias) + residual in one kernel
    epilogue_backward(grad, pre)    gradients of that epilogue
    moe_route(logits, top_k, ...)   experts and weights of each token;  moe_route_backward
    moe_dispatch(x, experts, E)     rows sorted by expert, quantized to fp8
    moe_gemm(x, w, offsets, ...)    the experts' products over those rows;  moe_gemm_swiglu (gate+up -> fp8 h)
    moe_combine(y, rows, weights)   weighted sum back to tokens;  moe_combine_backward

A mixture-of-experts layer is route -> dispatch -> moe_gemm_swiglu -> moe_gemm -> combine: no step waits for the host, so
the whole run can be captured into a CUDA graph.  All arithmetic happens in the sm_100a kernels of libb2x.so (C ABI in
include/b2x.h); there is no CPU path.  The calls run on the current stream of their tensors' device and keep no state
between them.

A new result whose rows are no multiple of 8 values (16 of float8) is a view of rows padded to one: not contiguous.
float8 operands whose rows do not start on 16-byte boundaries are copied to padded rows in every call; a weight that is
kept spares that where it is stored padded: torch.empty(N, -(-K // 16) * 16)[:, :K].
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .ops import FP8_DTYPES, IN_DTYPES, OUT_DTYPES

FLOAT_DTYPES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


class MoePlan(NamedTuple):
    """Where dispatch put the (token, slot) pairs: rows[t, j] is the pair's row or -1, expert e owns the rows
    [offsets[e], offsets[e + 1])."""
    offsets: torch.Tensor  # int32 [experts + 1]
    rows: torch.Tensor     # int32 [tokens, top_k]


_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream
_byref = ctypes.byref


def _device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> torch.device:
    """The one CUDA device of all tensors."""
    if not first.is_cuda:
        raise ValueError("b2x ops take CUDA tensors only (there is no CPU path)")
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"all tensors must be on {dev}, got one on {t.device}")
    return dev


def _call(dev: torch.device, fn, *args) -> None:
    """fn(*args, stream) with `dev` current and its current stream."""
    i = dev.index
    if i == _current_device():
        st = fn(*args, _current_stream(i))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _current_stream(i))
    if st:
        L.check(st)


def _matrix(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D, got shape {tuple(t.shape)}")
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements; a single row (or column) may have any."""
    rows, cols = t.shape
    return max(t.stride(0), cols) if rows <= 1 else t.stride(0)


def _rows(t: torch.Tensor, what: str) -> torch.Tensor:
    """A 2-D tensor with unit column stride and rows that do not overlap."""
    if t.dim() == 2 and t.is_contiguous():
        return t
    t = _matrix(t, what)
    return t if t.shape[0] <= 1 or t.stride(0) >= t.shape[1] else t.contiguous()


def _output(out: Optional[torch.Tensor], shape, dtype, like: torch.Tensor, what: str, pad: int = 8) -> torch.Tensor:
    """`out` checked, or a new tensor on like's device whose row pitch is a multiple of `pad` elements."""
    dev = like.device
    if out is None:
        n = shape[1]
        if n % pad == 0:
            return like.new_empty(shape, dtype=dtype)
        return like.new_empty((shape[0], -(-n // pad) * pad), dtype=dtype)[:, :n]
    if tuple(out.shape) != tuple(shape) or out.dtype != dtype or out.device != dev:
        raise ValueError(f"{what} must be a {dtype} tensor of shape {tuple(shape)} on {dev}")
    if (out.stride(1) != 1 and out.shape[1] > 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1]):
        raise ValueError(f"{what} must have unit column stride and rows that do not overlap")
    return out


def _scale(t: Optional[torch.Tensor], what: str, *counts: int) -> Optional[torch.Tensor]:
    """A contiguous fp32 vector of one of the given lengths."""
    if t is None:
        return None
    if t.numel() not in counts:
        raise ValueError(f"{what} must have {' or '.join(str(c) for c in dict.fromkeys(counts))} elements, got {t.numel()}")
    if t.dtype is torch.float32 and t.is_contiguous():
        return t
    return t.reshape(-1).to(torch.float32).contiguous()


def _ints(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
    if t.dtype is torch.int64:
        t = t.clamp(-1, 2**31 - 1).to(torch.int32)  # what int32 cannot hold stays out of range instead of wrapping
    return t if t.is_contiguous() else t.contiguous()


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """float8 t [..., rows, cols] with 16-byte aligned rows that do not overlap: t itself or, where TMA could not address
    it, a copy with padded rows."""
    shape, strides = t.shape, t.stride()
    rows, cols = shape[-2:]
    sr, sc = strides[-2:]
    one = len(shape) == 2 or shape[0] == 1
    if t.data_ptr() % 16 == 0 and (sc == 1 or cols == 1) and (rows == 1 or (sr % 16 == 0 and sr >= cols)) and (
            one or (strides[0] % 16 == 0 and strides[0] >= rows * sr)):
        return t
    if (sc != 1 and cols > 1) or sr < cols or not (one or strides[0] == rows * sr):
        t = t.contiguous()
        sr = cols
    out = t.new_empty((*t.shape[:-1], -(-cols // 16) * 16))
    n = t.numel() // cols if cols else 0  # rows of all experts lie one stride apart
    _call(t.device, L.lib().b2x_pad_rows, t.data_ptr(), max(sr, cols), n, cols, out.data_ptr(), out.shape[-1])
    return out[..., :cols]


def _pitch(t: torch.Tensor) -> int:
    """Row stride of an _aligned matrix; a single row may have any."""
    rows, cols = t.shape[-2:]
    return t.stride(-2) if rows > 1 else max(-(-cols // 16) * 16, 16)


# ----------------------------------------------------------------------------
# dense product with its epilogue


def gemm_epilogue(a: torch.Tensor, b: torch.Tensor, *, scale_a: Optional[torch.Tensor] = None,
                  scale_b: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                  activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
                  out_dtype: torch.dtype = torch.bfloat16, return_pre: bool = False):
    """C = act(scale_a * scale_b * (A @ B) + bias) + residual for float8 A [M, K] and B [K, N] (as for matmul: a
    K-major weight is w.t()), in fp32 and rounded once; see include/b2x.h b2x_fp8_gemm_epilogue.

    bias [N] fp32 / bf16 / fp16; activation None, "relu", "gelu" (erf), "gelu_tanh" or "silu"; residual [M, N] of
    out_dtype.  return_pre=True returns (C, pre) with pre = what the activation was given, for epilogue_backward."""
    dev = _device(a, b, scale_a, scale_b, bias, residual)
    if a.dtype not in FP8_DTYPES or b.dtype not in FP8_DTYPES:
        raise TypeError(f"gemm_epilogue takes float8 A and B, got {a.dtype} and {b.dtype}")
    if out_dtype not in OUT_DTYPES:
        raise TypeError(f"gemm_epilogue output must be bfloat16 or float16, got {out_dtype}")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[0]:
        raise ValueError(f"A {tuple(a.shape)} and B {tuple(b.shape)} are not [M, K] and [K, N]")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of {[k for k in ACTIVATIONS if k]}")
    if (scale_a is None) != (scale_b is None):
        raise ValueError("pass both scales or neither")
    M, K = a.shape
    N = b.shape[1]
    if bias is not None:
        if tuple(bias.shape) != (N,):
            raise ValueError(f"bias must have shape ({N},), got {tuple(bias.shape)}")
        if bias.dtype not in FLOAT_DTYPES:
            raise TypeError(f"bias must be float32, bfloat16 or float16, got {bias.dtype}")
        bias = bias.contiguous()
    if residual is not None:
        if tuple(residual.shape) != (M, N):
            raise ValueError(f"residual must have shape {(M, N)}, got {tuple(residual.shape)}")
        if residual.dtype != out_dtype:
            raise TypeError(f"residual must be {out_dtype} like the output, got {residual.dtype}")
        residual = _rows(residual, "residual")
    sa, sb = _scale(scale_a, "scale_a", 1), _scale(scale_b, "scale_b", 1)
    c = _output(None, (M, N), out_dtype, a, "out")
    pre = _output(None, (M, N), out_dtype, a, "pre") if return_pre else None
    if M and N:
        if K == 0:
            raise ValueError("gemm_epilogue needs K > 0")
        a = _aligned(a)
        if b.stride(0) == 1 or K == 1:  # a K-major weight
            b = _aligned(b.t())
            ldb = (1, _pitch(b))
        else:
            b = _aligned(b)
            ldb = (_pitch(b), 1)
        g = L.GemmArgs(a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K, _pitch(a), *ldb, _ld(c), FP8_DTYPES[a.dtype],
                       FP8_DTYPES[b.dtype], OUT_DTYPES[out_dtype])
        if sa is not None:
            g.scale_mode, g.scale_a, g.scale_b = L.SCALE_TENSOR, sa.data_ptr(), sb.data_ptr()
        ep = L.Epilogue(activation=ACTIVATIONS[activation])
        if bias is not None:
            ep.bias, ep.bias_type = bias.data_ptr(), FLOAT_DTYPES[bias.dtype]
        if residual is not None:
            ep.residual, ep.ld_residual = residual.data_ptr(), _ld(residual)
        if pre is not None:
            ep.pre, ep.ld_pre = pre.data_ptr(), _ld(pre)
        _call(dev, L.lib().b2x_fp8_gemm_epilogue, _byref(g), _byref(ep))
    return (c, pre) if return_pre else c


def epilogue_backward(grad: torch.Tensor, pre: torch.Tensor, activation: Optional[str] = None, *, bias_grad: bool = True):
    """(d_pre, d_bias) of gemm_epilogue: d_pre = grad * act'(pre) in grad's dtype, d_bias [N] fp32 = its column sums
    before rounding (None if not bias_grad).  grad and pre [M, N] share a dtype (bf16, fp16 or fp32).  The residual's
    gradient is grad.  relu'(0) = 0."""
    dev = _device(grad, pre)
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of {[k for k in ACTIVATIONS if k]}")
    if grad.dim() != 2 or grad.shape != pre.shape:
        raise ValueError(f"grad {tuple(grad.shape)} and pre {tuple(pre.shape)} must be 2-D and of one shape")
    if grad.dtype not in FLOAT_DTYPES or pre.dtype != grad.dtype:
        raise TypeError(f"grad and pre must both be float32, bfloat16 or float16, got {grad.dtype} and {pre.dtype}")
    M, N = grad.shape
    grad, pre = _rows(grad, "grad"), _rows(pre, "pre")
    out = _output(None, (M, N), grad.dtype, grad, "d_pre")
    db = grad.new_empty(N, dtype=torch.float32) if bias_grad else None
    _call(dev, L.lib().b2x_epilogue_backward, grad.data_ptr(), _ld(grad), pre.data_ptr(), _ld(pre), out.data_ptr(), _ld(out),
          db.data_ptr() if db is not None else None, FLOAT_DTYPES[grad.dtype], M, N, ACTIVATIONS[activation])
    return out, db


# ----------------------------------------------------------------------------
# routing


SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 0, "top2": 1}


def _choice(table: dict, value, what: str) -> int:
    if value not in table:
        raise ValueError(f"{what} must be {' or '.join(map(repr, table))}, got {value!r}")
    return table[value]


def _count(value: int, what: str) -> int:
    """A number that the C ABI takes as int, which would wrap past 32 bits."""
    if not -2**31 <= value < 2**31:
        raise ValueError(f"{what} must fit 32 bits, got {value}")
    return value


def moe_route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None,
              num_groups: int = 1, top_groups: int = 1, group_score: str = "max", renormalize: bool = True,
              scale: float = 1.0):
    """(weights fp32 [T, top_k], experts int32 [T, top_k]) for router logits [T, E] (fp32, bf16 or fp16).

    score "softmax" or "sigmoid" gives s; experts are chosen by s + bias (bias [E], for balance) and weighed by s, divided
    by the chosen ones' sum if renormalize, times scale.  With num_groups > 1 only the experts of the top_groups best
    groups take part; a group scores its largest ("max") or the sum of its two largest ("top2") choices.  The slots fall
    in choice, equal choices go to the lower expert.  An expert with logit or bias -inf is masked; slots that no expert
    is left for hold expert -1 and weight 0, which moe_dispatch drops.  Sigmoid scores that are 0 in 64 bits (logits of the
    type's lowest value) weigh 0 also where renormalized.  E <= 1024, top_k <= 32."""
    dev = _device(logits, bias)
    if logits.dtype not in FLOAT_DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    logits = _rows(logits, "logits")
    T, E = logits.shape
    bias = _scale(bias, "bias", E)
    k = max(_count(top_k, "top_k"), 0)
    weights = logits.new_empty((T, k), dtype=torch.float32)
    experts = logits.new_empty((T, k), dtype=torch.int32)
    a = L.MoeRouteArgs(logits.data_ptr(), FLOAT_DTYPES[logits.dtype], T, E, _ld(logits), top_k, _choice(SCORES, score, "score"),
                       None if bias is None else bias.data_ptr(), _count(num_groups, "num_groups"), _count(top_groups, "top_groups"),
                       _choice(GROUP_SCORES, group_score, "group_score"), bool(renormalize), scale, weights.data_ptr(),
                       experts.data_ptr())
    _call(dev, L.lib().b2x_moe_route, _byref(a))
    return weights, experts


def moe_route_backward(grad_weights: torch.Tensor, logits: torch.Tensor, experts: torch.Tensor, *, score: str = "softmax",
                       renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """Gradient of the logits [T, E] (their dtype) from that of moe_route's weights; logits, experts, score, renormalize
    and scale as in the forward call.  The choice of experts has no gradient, nor has the bias."""
    dev = _device(logits, grad_weights, experts)
    if logits.dtype not in FLOAT_DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    logits = _rows(logits, "logits")
    T, E = logits.shape
    if experts.dim() != 2 or experts.shape[0] != T or grad_weights.shape != experts.shape:
        raise ValueError(f"experts {tuple(experts.shape)} and grad_weights {tuple(grad_weights.shape)} must be [{T}, top_k]")
    experts = _ints(experts, "experts")
    d = grad_weights if grad_weights.dtype == torch.float32 and grad_weights.is_contiguous() else grad_weights.to(torch.float32).contiguous()
    out = logits.new_empty((T, E))
    a = L.MoeRouteArgs(logits.data_ptr(), FLOAT_DTYPES[logits.dtype], T, E, _ld(logits), experts.shape[1],
                       _choice(SCORES, score, "score"), None, 1, 1, 0, bool(renormalize), scale, None, experts.data_ptr())
    _call(dev, L.lib().b2x_moe_route_backward, _byref(a), d.data_ptr(), out.data_ptr(), E)
    return out


# ----------------------------------------------------------------------------
# dispatch and combine


def moe_dispatch(x: torch.Tensor, experts: torch.Tensor, num_experts: int, *, dtype: torch.dtype = torch.float8_e4m3fn,
                 scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None):
    """(q, scales, plan) for tokens x [T, H] (fp32 or bf16) and experts [T, top_k]: the pairs stably sorted by expert,
    row plan.rows[t, j] of q [T * top_k, H] being x[t] in fp8 (the recipe of quantize).

    scale None: one scale per row, scales [T * top_k] fp32.  scale given (one fp32): used for every row and returned.
    Pairs whose expert lies outside [0, num_experts) are dropped (row -1); rows of q and scales from plan.offsets[-1] on
    are not written (q may be given as `out`, which keeps what it held there)."""
    dev = _device(x, experts, scale, out)
    if x.dtype not in IN_DTYPES:
        raise TypeError(f"moe_dispatch takes float32 or bfloat16, got {x.dtype}")
    if dtype not in FP8_DTYPES:
        raise TypeError(f"moe_dispatch output must be float8_e4m3fn or float8_e5m2, got {dtype}")
    x = _rows(x, "x")
    T, H = x.shape
    if experts.dim() != 2 or experts.shape[0] != T:
        raise ValueError(f"experts must be [{T}, top_k], got {tuple(experts.shape)}")
    experts = _ints(experts, "experts")
    k = experts.shape[1]
    given = _scale(scale, "scale", 1)
    q = _output(out, (T * k, H), dtype, x, "out", 16)
    scales = x.new_empty(T * k, dtype=torch.float32) if given is None else given
    offsets = x.new_empty(max(num_experts, 0) + 1, dtype=torch.int32)
    rows = x.new_empty((T, k), dtype=torch.int32)
    a = L.MoeDispatchArgs(x.data_ptr(), IN_DTYPES[x.dtype], T, H, _ld(x), experts.data_ptr(), k, num_experts, q.data_ptr(),
                          FP8_DTYPES[dtype], _ld(q), scales.data_ptr() if given is None else None,
                          None if given is None else given.data_ptr(), offsets.data_ptr(), rows.data_ptr())
    _call(dev, L.lib().b2x_moe_dispatch, _byref(a))
    return q, scales, MoePlan(offsets, rows)


def _pair_tensors(rows, weights):
    if rows.dim() != 2:
        raise ValueError(f"rows must be [tokens, top_k], got {tuple(rows.shape)}")
    if weights is not None:
        if weights.shape != rows.shape:
            raise ValueError(f"weights must have the shape of rows {tuple(rows.shape)}, got {tuple(weights.shape)}")
        weights = weights if weights.dtype == torch.float32 and weights.is_contiguous() else weights.to(torch.float32).contiguous()
    return _ints(rows, "rows"), weights


def moe_combine(y: torch.Tensor, rows: torch.Tensor, weights: Optional[torch.Tensor] = None, *,
                residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * y[rows[t, j]] + residual[t] for the experts' outputs y [R, H] (bf16, fp16 or fp32)
    and plan.rows, in fp32 in the order of the slots.  weights None counts every row once (the gradient of the
    dispatch's gather).  A dropped pair (row -1) adds nothing."""
    dev = _device(y, rows, weights, residual)
    if y.dtype not in FLOAT_DTYPES:
        raise TypeError(f"y must be float32, bfloat16 or float16, got {y.dtype}")
    y = _rows(y, "y")
    rows, weights = _pair_tensors(rows, weights)
    T, k = rows.shape
    R, H = y.shape
    if residual is not None:
        if tuple(residual.shape) != (T, H) or residual.dtype != y.dtype:
            raise ValueError(f"residual must be a {y.dtype} tensor of shape {(T, H)}")
        residual = _rows(residual, "residual")
    out = _output(None, (T, H), y.dtype, y, "out")
    _call(dev, L.lib().b2x_moe_combine, y.data_ptr(), R, _ld(y), rows.data_ptr(), weights.data_ptr() if weights is not None else None,
          T, k, H, residual.data_ptr() if residual is not None else None, _ld(residual) if residual is not None else 0,
          out.data_ptr(), _ld(out), FLOAT_DTYPES[y.dtype])
    return out


def moe_combine_backward(grad: torch.Tensor, y: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, *,
                         out: Optional[torch.Tensor] = None):
    """(d_y [R, H], d_weights fp32 [T, top_k]) of moe_combine for grad [T, H] of y's dtype.  The residual's gradient is
    grad.  No row may be named by two pairs, as in a plan of moe_dispatch.  Rows of d_y that no pair names are not written
    (d_y may be given as `out`)."""
    dev = _device(y, grad, rows, weights, out)
    if y.dtype not in FLOAT_DTYPES or grad.dtype != y.dtype:
        raise TypeError(f"y and grad must both be float32, bfloat16 or float16, got {y.dtype} and {grad.dtype}")
    y, grad = _rows(y, "y"), _rows(grad, "grad")
    rows, weights = _pair_tensors(rows, weights)
    T, k = rows.shape
    R, H = y.shape
    if tuple(grad.shape) != (T, H):
        raise ValueError(f"grad must have shape {(T, H)}, got {tuple(grad.shape)}")
    dy = _output(out, (R, H), y.dtype, y, "out")
    dw = y.new_empty((T, k), dtype=torch.float32)
    _call(dev, L.lib().b2x_moe_combine_backward, grad.data_ptr(), _ld(grad), y.data_ptr(), R, _ld(y), rows.data_ptr(),
          weights.data_ptr(), T, k, H, dy.data_ptr(), _ld(dy), dw.data_ptr(), FLOAT_DTYPES[y.dtype])
    return dy, dw


# ----------------------------------------------------------------------------
# the experts' products


def _moe_gemm_args(x, w, offsets, scale_x, scale_w, who, kmajor):
    if x.dtype not in FP8_DTYPES or w.dtype not in FP8_DTYPES:
        raise TypeError(f"{who} takes float8 x and w, got {x.dtype} and {w.dtype}")
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[2]:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} are not [R, K] and [E, N, K]")
    E, N, K = w.shape
    if offsets.dim() != 1 or offsets.shape[0] != E + 1:
        raise ValueError(f"offsets must have {E + 1} elements, got {tuple(offsets.shape)}")
    if K == 0:
        raise ValueError(f"{who} needs K > 0")
    offsets = _ints(offsets, "offsets")
    x = _aligned(x)
    if w.stride(2) != 1 and w.stride(1) == 1 and not kmajor:  # a transposed view of [E, K, N]
        w = _aligned(w.transpose(1, 2))
        ldw = (w.stride(0), 1, _pitch(w))
    else:
        w = _aligned(w)
        ldw = (w.stride(0), _pitch(w), 1)
    sx, sw = _scale(scale_x, "scale_x", 1, x.shape[0]), _scale(scale_w, "scale_w", 1, E)
    R = x.shape[0]
    a = L.MoeGemmArgs(x.data_ptr(), FP8_DTYPES[x.dtype], R, K, _pitch(x), w.data_ptr(), FP8_DTYPES[w.dtype],
                      E, N, *ldw, offsets.data_ptr(), None if sx is None else sx.data_ptr(), 0 if sx is None else sx.numel(),
                      None if sw is None else sw.data_ptr(), 0 if sw is None else sw.numel())
    return a, (x, w, offsets, sx, sw)


def moe_gemm(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, *, scale_x: Optional[torch.Tensor] = None,
             scale_w: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y[r] = scale_x[r] * scale_w[e] * (w[e] @ x[r]) for the rows r in [offsets[e], offsets[e + 1]) of float8 x [R, K],
    with one float8 weight [N, K] per expert in w [E, N, K].

    w may be K-major or a transposed view of [E, K, N] storage (so that w.transpose(1, 2) of the same weights gives the
    gradient of the rows).  scale_x: one or one per row; scale_w: one or one per expert.  offsets (int32, on the device)
    rise from 0 to at most R; rows from offsets[-1] on are not written (y may be given as `out`)."""
    dev = _device(x, w, offsets, scale_x, scale_w, out)
    if out_dtype not in OUT_DTYPES:
        raise TypeError(f"moe_gemm output must be bfloat16 or float16, got {out_dtype}")
    a, keep = _moe_gemm_args(x, w, offsets, scale_x, scale_w, "moe_gemm", False)
    y = _output(out, (a.rows, a.N), out_dtype, x, "out")
    if a.rows and a.N:
        _call(dev, L.lib().b2x_moe_gemm, _byref(a), y.data_ptr(), OUT_DTYPES[out_dtype], _ld(y))
    return y


def moe_gemm_swiglu(x: torch.Tensor, w_gu: torch.Tensor, offsets: torch.Tensor, h_scale: torch.Tensor, *,
                    scale_x: Optional[torch.Tensor] = None, scale_w: Optional[torch.Tensor] = None,
                    h_dtype: torch.dtype = torch.float8_e4m3fn, h_amax: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h = fp8(silu(gate) * up / h_scale) [R, I] of the experts' gate and up products over rows sorted by expert, for
    w_gu [E, 2I, K] interleaved per expert (interleave_gate_up); I a multiple of 128.  h_scale: one fp32, as for
    gemm_swiglu's mode "given"; h_amax (one fp32, zeroed by the caller) collects max |h|.  Scales and offsets as for
    moe_gemm, whose x the result is (with scale_x=h_scale)."""
    dev = _device(x, w_gu, offsets, h_scale, scale_x, scale_w, h_amax, out)
    if h_dtype not in FP8_DTYPES:
        raise TypeError(f"moe_gemm_swiglu produces float8 h, got {h_dtype}")
    if w_gu.dim() == 3 and w_gu.shape[1] % 256:
        raise ValueError(f"w_gu must have 2I rows with I a multiple of 128, got {w_gu.shape[1]}")
    if h_amax is not None and (h_amax.numel() != 1 or h_amax.dtype != torch.float32):
        raise ValueError("h_amax must be one float32")
    if w_gu.dim() == 3 and w_gu.shape[0] > 1 and w_gu.stride(0) != w_gu.shape[1] * w_gu.stride(1):
        w_gu = w_gu.contiguous()
    a, keep = _moe_gemm_args(x, w_gu, offsets, scale_x, scale_w, "moe_gemm_swiglu", True)
    hs = _scale(h_scale, "h_scale", 1)
    h = _output(out, (a.rows, a.N // 2), h_dtype, x, "out", 16)
    if a.rows and a.N:
        _call(dev, L.lib().b2x_moe_gemm_swiglu, _byref(a), h.data_ptr(), FP8_DTYPES[h_dtype], _ld(h), hs.data_ptr(),
              h_amax.data_ptr() if h_amax is not None else None)
    return h
