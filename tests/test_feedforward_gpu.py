"""GPU checks of the feed-forward operators (b2x/feedforward.py) against plain implementations in 64 bits.

Tolerances, from the arithmetic:
  products   fp8 products are exact in fp32; K additions, each off by at most 2^-23 of the running sum (truncation counted),
             give |err| <= K 2^-23 sum |a||b|.  Scales, bias and activation add a few 2^-24 of their values; activations
             have slope <= 1.2 and are computed to 4e-6 relative (activations.cuh).
  rounding   half a step of the output type: eps / 2 of the value (and half the smallest subnormal).
  sums       n additions in fp32: n 2^-24 sum |x|.
  fp8 codes  equal to the quantization of the exact value, a neighbouring code only where the exact value lies within the
             product's error of the border between the two.
Choices of experts, row numbers and quantized rows of the dispatch are exact."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D = torch.float64
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
FMAX = {E4: 448.0, E5: 57344.0}
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=F32, std=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * std).to(dtype)


def fp8(*shape, seed=0, dtype=E4, std=40.0):
    return randn(*shape, seed=seed, std=std).clamp(-FMAX[dtype], FMAX[dtype]).to(dtype)


def rounded(dtype, ref):
    """Half a step of dtype at ref."""
    tiny = {BF: 2.0 ** -134, HF: 2.0 ** -25, F32: 2.0 ** -150}[dtype]
    return torch.finfo(dtype).eps / 2 * ref.abs() + tiny


def check(got, ref, tol, what=""):
    got = got.to(D)
    assert got.shape == ref.shape, (got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} out of tolerance, first at {i}: got {got[i].item()} "
                             f"want {ref[i].item()} tolerance {(tol if not torch.is_tensor(tol) or tol.dim() == 0 else tol.expand_as(ref)[i])}")


def act(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "gelu":
        return 0.5 * x * torch.erfc(-x * 0.5 ** 0.5)
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / np.pi) ** 0.5 * (x + 0.044715 * x ** 3)))
    if name == "silu":
        return x / (1 + torch.exp(-x))
    return x


def teardown_module():
    import b2x
    torch.cuda.synchronize()
    assert b2x.read_device_status() == 0


# ------------------------------------------------------------------------------------------------- gemm_epilogue

LINEAR = [  # M, N, K, activation, bias, residual, out, pre, layout
    (1, 128, 128, None, None, False, BF, False, "nk"),
    (1, 1, 16, "relu", F32, True, BF, True, "nk"),
    (3, 200, 144, "gelu", BF, True, BF, True, "nk"),
    (16, 640, 4096, "silu", HF, False, HF, False, "nk"),
    (17, 130, 100, "gelu_tanh", F32, True, HF, True, "nk"),
    (33, 72, 2000, "silu", F32, True, BF, False, "kn"),
    (64, 256, 512, "relu", None, True, BF, True, "kn"),
    (65, 2049, 640, "gelu", F32, False, BF, True, "nk"),
    (128, 1000, 1024, None, BF, True, HF, False, "kn"),
    (129, 264, 272, "gelu_tanh", F32, False, BF, True, "nk"),
    (300, 513, 384, "gelu", F32, True, BF, True, "kn"),
    (700, 1032, 256, "silu", BF, True, HF, True, "nk"),
    (1025, 2304, 1040, "gelu_tanh", F32, True, BF, True, "nk"),
    (2000, 3968, 512, "relu", F32, True, BF, False, "kn"),
    (4500, 1100, 272, "gelu", F32, True, BF, True, "nk"),     # more than one band of token tiles, half a weight tile over
    (257, 19000, 128, "silu", None, False, HF, False, "nk"),
    (5000, 1039, 300, "gelu_tanh", BF, True, HF, True, "nk"),
]


def linear_ref(a, b, sa, sb, bias, name, residual, out):
    K = a.shape[1]
    al, bl = a.to(D), b.to(D)
    alpha = 1.0 if sa is None else sa.to(D) * sb.to(D)
    z, size = (al @ bl) * alpha, (al.abs() @ bl.abs()) * alpha
    err = (K + 4) * 2.0 ** -23 * size
    if bias is not None:
        z = z + bias.to(D)
        err = err + 2.0 ** -23 * (size + bias.to(D).abs())
    y = act(z, name)
    e = 1.2 * err + 4e-6 * y.abs()
    if residual is not None:
        y = y + residual.to(D)
        e = e + 2.0 ** -23 * y.abs()
    return z, err + rounded(out, z.abs() + err), y, e + rounded(out, y.abs() + e)


@pytest.mark.parametrize("M,N,K,name,bias,residual,out,pre,layout", LINEAR)
def test_gemm_epilogue(M, N, K, name, bias, residual, out, pre, layout):
    import b2x
    a = fp8(M, K, seed=1)
    b = fp8(N, K, seed=2).t() if layout == "nk" else fp8(K, N, seed=2)
    sa, sb = torch.tensor([0.02], device="cuda"), torch.tensor([K ** -0.5 / 30], device="cuda")
    bias = None if bias is None else randn(N, seed=3, dtype=bias)
    res = randn(M, N, seed=4, dtype=out) if residual else None
    got = b2x.gemm_epilogue(a, b, scale_a=sa, scale_b=sb, bias=bias, activation=name, residual=res, out_dtype=out, return_pre=pre)
    z, ztol, y, tol = linear_ref(a, b, sa, sb, bias, name, res, out)
    c = got[0] if pre else got
    assert c.dtype == out
    check(c, y, tol, "C")
    if pre:
        check(got[1], z, ztol, "pre")
    again = b2x.gemm_epilogue(a, b, scale_a=sa, scale_b=sb, bias=bias, activation=name, residual=res, out_dtype=out)
    assert torch.equal(again.view(torch.int16), c.view(torch.int16)), "the same call gave other bits"


@pytest.mark.parametrize("da,db", [(E4, E5), (E5, E4), (E5, E5)])
def test_gemm_epilogue_formats_without_scales(da, db):
    import b2x
    a, b = fp8(70, 256, seed=1, dtype=da, std=1.0), fp8(96, 256, seed=2, dtype=db, std=1.0).t()
    _, _, y, tol = linear_ref(a, b, None, None, None, None, None, BF)
    check(b2x.gemm_epilogue(a, b), y, tol)


def test_gemm_epilogue_small_integers_are_exact():
    """Sums of small integers fit 8 bits of bf16: nothing may be lost or added."""
    import b2x
    a = torch.randint(-1, 2, (40, 200), device="cuda", generator=gen(1)).to(F32).to(E4)
    b = torch.randint(-1, 2, (200, 136), device="cuda", generator=gen(2)).to(F32).to(E4)
    ref = a.to(D) @ b.to(D)
    assert ref.abs().max() <= 256
    assert torch.equal(b2x.gemm_epilogue(a, b).to(D), ref)


def test_gemm_epilogue_strided_operands():
    import b2x
    wide = fp8(50, 512, seed=1)
    a = wide[:, 100:356]                                    # not 16-byte aligned: copied
    a2 = wide[:, 128:384]                                   # aligned rows with a longer pitch
    b = fp8(260, 256, seed=2)[4:, :].t()
    res = randn(50, 999, seed=3, dtype=BF)[:, 1:257]        # odd pitch and base
    for x in (a, a2, wide[:1, :256].expand(50, 256)):
        _, _, y, tol = linear_ref(x, b, None, None, None, "relu", res, BF)
        check(b2x.gemm_epilogue(x, b, activation="relu", residual=res), y, tol)


@pytest.mark.parametrize("rows,cols,ld,first", [(1, 1, 1, 0), (3, 15, 15, 1), (7, 33, 40, 3), (100, 257, 257, 0), (50, 1001, 1003, 2), (2, 64, 64, 5)])
def test_pad_rows(rows, cols, ld, first):
    """Byte for byte, zeros up to the next 16, nothing else written."""
    import b2x
    from b2x import _lib as L
    src = torch.randint(0, 256, (rows * ld + 64,), device="cuda", generator=gen(1), dtype=torch.uint8)[first:]
    pitch = -(-cols // 16) * 16 + 32
    dst = torch.full((rows, pitch), 7, device="cuda", dtype=torch.uint8)
    L.check(L.lib().b2x_pad_rows(src.data_ptr(), ld, rows, cols, dst.data_ptr(), pitch, torch.cuda.current_stream().cuda_stream))
    want = torch.full_like(dst, 7)
    want[:, :-(-cols // 16) * 16] = 0
    want[:, :cols] = torch.as_strided(src, (rows, cols), (ld, 1))
    assert torch.equal(dst, want)


def test_gemm_epilogue_nan_and_inf_reach_the_output():
    import b2x
    a, b = torch.ones((4, 128), device="cuda").to(E4), torch.ones((128, 128), device="cuda").to(E4)
    bias = torch.zeros(128, device="cuda")
    bias[3], bias[5] = float("nan"), float("inf")
    for name in (None, "relu", "gelu", "gelu_tanh", "silu"):
        c = b2x.gemm_epilogue(a, b, bias=bias, activation=name)
        assert torch.isnan(c[:, 3]).all() and torch.isinf(c[:, 5]).all(), name
        assert torch.isfinite(c[:, :3]).all()


def test_gemm_epilogue_empty():
    import b2x
    b = torch.zeros((128, 64), device="cuda").to(E4)
    assert b2x.gemm_epilogue(torch.zeros((0, 128), device="cuda").to(E4), b, activation="gelu").shape == (0, 64)


# ------------------------------------------------------------------------------------------------- epilogue_backward


def slope(x, name):
    x = x.clone().requires_grad_()
    act(x, name).sum().backward()
    return x.grad


@pytest.mark.parametrize("M,N", [(1, 8), (1, 1), (5, 7), (64, 256), (257, 264), (513, 33), (4100, 64), (2049, 520)])
@pytest.mark.parametrize("name,dtype", [(None, BF), ("relu", HF), ("gelu", BF), ("gelu_tanh", F32), ("silu", BF)])
def test_epilogue_backward(M, N, name, dtype):
    import b2x
    g, z = randn(M, N, seed=1, dtype=dtype), randn(M, N, seed=2, dtype=dtype, std=2.0)
    d, db = b2x.epilogue_backward(g, z, name)
    s = slope(z.to(D), name)
    ref = g.to(D) * s
    # the slope is a sum of terms of size <= 1 + |x|, each to 4e-6
    err = g.to(D).abs() * 4e-6 * (1 + z.to(D).abs())
    assert d.dtype == dtype and db.dtype == F32
    check(d, ref, err + rounded(dtype, ref.abs() + err), "d_pre")
    check(db, ref.sum(0), err.sum(0) + M * 2.0 ** -24 * ref.abs().sum(0) + 1e-30, "d_bias")
    d2, none = b2x.epilogue_backward(g, z, name, bias_grad=False)
    assert none is None and torch.equal(d2, d)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "silu"])
def test_epilogue_backward_against_differences(name):
    """(act(x + h) - act(x - h)) / 2h in fp64: off by h^2 / 6 of the third derivative, which is below 3."""
    import b2x
    x = torch.linspace(-8, 8, 4096, device="cuda").view(64, 64)
    d, _ = b2x.epilogue_backward(torch.ones_like(x), x, name)
    h = 1e-4
    ref = (act(x.to(D) + h, name) - act(x.to(D) - h, name)) / (2 * h)
    check(d, ref, 4e-6 * (1 + x.to(D).abs()) + h * h / 2)


@pytest.mark.parametrize("name,bound", [("gelu", 12), ("gelu_tanh", 16), ("silu", 10), ("relu", 0), (None, 0)])
@pytest.mark.parametrize("N", [512, 257])
def test_epilogue_backward_fp32_to_a_few_units(name, bound, N):
    """u = 2^-24; the exponential is off by 4 u (2 units in the last place, or 2^-22 for the approximate one).
      gelu       erfc(|x|) / 2 <= 0.5: its fit 2 u, the exponential 4 u, the polynomial's rounding 8 u, z^2 1 u; x phi(x) <=
                 0.25 by 8 u; the differences and sums 2 u
      silu       e^-|x| 4 u, 1 / (1 + e) 4 u, their product 9 u; x q <= 0.28 and the sum by 10 u and u, the product by s
      gelu_tanh  the exponent y by 5 u y, y e^-y <= 0.37: sigma 5 u; x p q 2u' <= 0.35 by 21 u + 5 u y; the sum 1.1 u"""
    import b2x
    u = 2.0 ** -24
    z = torch.linspace(-20, 20, 300 * N, device="cuda").view(300, N)
    z = torch.cat([z, z * 2.0 ** -8])
    g = randn(600, N, seed=1)
    d, db = b2x.epilogue_backward(g, z, name)
    ref = g.to(D) * (slope(z.to(D), name) if name else 1.0)
    tol = bound * u * g.to(D).abs() + u * ref.abs() + 2.0 ** -126
    check(d, ref, tol, "d_pre")
    check(db, ref.sum(0), tol.sum(0) + 600 * u * ref.abs().sum(0), "d_bias")


ENDS = [-3.3e38, -1e20, -1e18, -2e13, -1e12, -1e6, -60.0, 60.0, 1e6, 1e12, 2e13, 1e20]


@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("N", [24, 23])
def test_epilogue_backward_of_large_values(name, dtype, N):
    """Finite pre-activations however large: the slope is 0 or 1 (silu's at -60 is -5e-25), in d_bias too."""
    import b2x
    lim = torch.finfo(dtype).max
    z = torch.tensor(ENDS + ENDS[::-1], device="cuda").clamp(-lim, lim).to(dtype)[:N].repeat(40, 1)
    g = randn(40, N, seed=1, dtype=dtype)
    d, db = b2x.epilogue_backward(g, z, name)
    ref = g.to(D) * (1.0 if name is None else (z > 0).to(D))
    check(d, ref, rounded(dtype, ref) + 1e-20, "d_pre")
    check(db, ref.sum(0), 40 * 2.0 ** -24 * ref.abs().sum(0) + 1e-18, "d_bias")


@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_gemm_epilogue_of_large_values(name):
    """The activations themselves there: 0 or the value."""
    import b2x
    bias = torch.tensor(ENDS, device="cuda").repeat(11)
    zero = torch.zeros((5, 128), device="cuda").to(E4)
    c, pre = b2x.gemm_epilogue(zero, torch.zeros((132, 128), device="cuda").to(E4).t(), bias=bias, activation=name, return_pre=True)
    check(pre, bias.to(D).expand(5, -1), rounded(BF, bias.to(D)), "pre")
    ref = bias.to(D).clamp_min(0).expand(5, -1)
    check(c, ref, rounded(BF, ref) + 1e-20, "C")


# wide enough for 8 and for 32 threads side by side (296 and 1184 runs of 16 bytes on 148 SMs), the last block partly empty,
# several rounds of the ring, rows split over a cluster or not
@pytest.mark.parametrize("M,N,name,dtype", [(4100, 2400, "gelu", BF), (300, 2400, "silu", HF), (301, 9480, "gelu_tanh", BF), (1, 9480, "relu", HF),
                                            (1300, 9480, None, BF), (70, 4800, "silu", F32), (900, 1200, "gelu_tanh", F32),
                                            (3, 19000, "gelu", BF)])
def test_epilogue_backward_wide(M, N, name, dtype):
    test_epilogue_backward(M, N, name, dtype)


@pytest.mark.parametrize("M,N", [(1100, 2400), (600, 9480), (257, 264), (130, 33)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_epilogue_backward_in_place(M, N, dtype):
    """d_pre may be grad or pre: the bits of the call with an output of its own."""
    import b2x
    from b2x import _lib as L
    g, z = randn(M, N, seed=1, dtype=dtype), randn(M, N, seed=2, dtype=dtype)
    kind = {BF: L.BF16, F32: L.F32}[dtype]
    for act_id, name in ((0, None), (2, "gelu"), (3, "gelu_tanh")):
        want, db = b2x.epilogue_backward(g, z, name)
        for over in ("grad", "pre"):
            a, b = g.clone(), z.clone()
            out = a if over == "grad" else b
            got = torch.empty_like(db)
            L.check(L.lib().b2x_epilogue_backward(a.data_ptr(), N, b.data_ptr(), N, out.data_ptr(), N, got.data_ptr(), kind, M, N, act_id,
                                                  torch.cuda.current_stream().cuda_stream))
            assert torch.equal(out, want) and torch.equal(got, db), (name, over)


@pytest.mark.parametrize("M,N,K", [(5, 256, 4096), (70, 520, 512), (1025, 2304, 512), (700, 1037, 256)])
@pytest.mark.parametrize("out", [BF, HF])
def test_gemm_epilogue_onto_its_residual(M, N, K, out):
    """The residual may be C itself, on either product kernel and with rows off the 8-byte grid."""
    import b2x
    from b2x import _lib as L
    a, b, bias = fp8(M, K, seed=1, std=1.0), fp8(N, K, seed=2, std=0.1), randn(N, seed=3)
    c = randn(M, N, seed=4, dtype=out)
    want = b2x.gemm_epilogue(a, b.t(), bias=bias, activation="gelu", residual=c, out_dtype=out)
    g = L.GemmArgs(a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K, K, 1, K, N, L.E4M3, L.E4M3, L.BF16 if out == BF else L.F16)
    ep = L.Epilogue(bias=bias.data_ptr(), bias_type=L.F32, activation=2, residual=c.data_ptr(), ld_residual=N)
    L.check(L.lib().b2x_fp8_gemm_epilogue(L.ctypes.byref(g), L.ctypes.byref(ep), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(c, want)


def test_epilogue_backward_strided_and_in_place_buffers():
    import b2x
    g, z = randn(70, 300, seed=1, dtype=BF)[:, 3:200], randn(197, 70, seed=2, dtype=BF).t()
    d, db = b2x.epilogue_backward(g, z, "silu")
    d2, db2 = b2x.epilogue_backward(g.contiguous(), z.contiguous(), "silu")
    assert torch.equal(d, d2)
    check(db, db2.to(D), 70 * 2.0 ** -23 * (g.to(D).abs() * 1.2).sum(0))
    d, db = b2x.epilogue_backward(torch.empty((0, 16), device="cuda"), torch.empty((0, 16), device="cuda"))
    assert d.shape == (0, 16) and torch.equal(db, torch.zeros(16, device="cuda"))


def test_epilogue_backward_of_the_forwards_pre():
    """The two together: gradients of sum(C * w) by the bias, against differences of the 64-bit forward."""
    import b2x
    M, N, K = 24, 64, 128
    a, b = fp8(M, K, seed=1, std=1.0), fp8(K, N, seed=2, std=0.1)
    bias, w = randn(N, seed=3), randn(M, N, seed=4, dtype=BF)
    _, pre = b2x.gemm_epilogue(a, b, bias=bias, activation="gelu", return_pre=True)
    _, db = b2x.epilogue_backward(w, pre, "gelu")
    z = a.to(D) @ b.to(D)
    h = 1e-4
    f = lambda s: (act(z + bias.to(D) + s, "gelu") * w.to(D)).sum(0)  # noqa: E731
    # pre is rounded to bf16 (2^-8 of it); the slope of the slope is below 0.8
    slack = (w.to(D).abs() * (0.8 * 2.0 ** -8 * (z + bias.to(D)).abs() + 1e-5)).sum(0)
    check(db, (f(h) - f(-h)) / (2 * h), slack)


# ------------------------------------------------------------------------------------------------- routing


def route_ref(logits, k, score, bias, groups, top_groups, gscore, renorm, scale):
    l = logits.to(D).cpu().numpy()
    T, E = l.shape
    b = None if bias is None else bias.to(D).cpu().numpy()
    W, I = np.zeros((T, k)), np.full((T, k), -1, np.int64)
    for t in range(T):
        x = l[t]
        off = np.isneginf(x) | (np.isneginf(b) if b is not None else False)
        with np.errstate(all="ignore"):
            if score == "sigmoid":
                s = 1 / (1 + np.exp(-x))
            elif np.isneginf(x).all():
                s = np.zeros(E)
            else:
                e = np.exp(x - np.nanmax(x))
                s = e / e.sum()
        c = s + b if b is not None else x.copy()  # without a bias s rises with x
        g = s + b if b is not None else s
        rank = lambda v: np.where(np.isnan(v), np.inf, v)  # noqa: E731
        if groups > 1 and top_groups < groups:
            gs = E // groups
            val = []
            for q in range(groups):
                m = [v for v, o in zip((g if gscore == "top2" else c)[q * gs:(q + 1) * gs], off[q * gs:(q + 1) * gs]) if not o]
                m = sorted(m, key=lambda v: np.inf if np.isnan(v) else v)[::-1]
                val.append(None if not m else sum(m[:2 if gscore == "top2" else 1]))
            order = sorted([q for q in range(groups) if val[q] is not None], key=lambda q: (-rank(val[q]), q))
            keep = set(order[:top_groups])
            off = off | np.array([e // gs not in keep for e in range(E)])
        order = sorted([e for e in range(E) if not off[e]], key=lambda e: (-rank(c[e]), e))[:k]
        w = s[order]
        if renorm and len(order):
            total = w.sum()
            w = w / total if total != 0 else w * 0
        W[t, :len(order)] = w * scale
        I[t, :len(order)] = order
    return W, I


def check_route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, gscore="max", renorm=True, scale=1.0):
    import b2x
    w, e = b2x.moe_route(logits, k, score=score, bias=bias, num_groups=groups, top_groups=top_groups, group_score=gscore,
                         renormalize=renorm, scale=scale)
    W, I = route_ref(logits, k, score, bias, groups, top_groups, gscore, renorm, scale)
    assert w.dtype == F32 and e.dtype == torch.int32
    assert np.array_equal(e.cpu().numpy(), I)
    got = w.cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(W))
    # exp to 2e-6 (|x| 2^-24 for |x| <= 20), sums of up to 1024 positive terms to 1024 2^-24 at worst
    tol = (8e-6 + logits.shape[1] * 2.0 ** -24) * np.abs(W) + 1e-37
    assert np.all(np.isnan(W) | (np.abs(got - W) <= tol)), np.nanmax(np.abs(got - W) / (np.abs(W) + 1e-30))
    return w, e


ROUTE = [  # T, E, k, score, bias, groups, top_groups, gscore, renorm, dtype
    (1, 8, 2, "softmax", False, 1, 1, "max", True, F32),
    (1, 1, 1, "sigmoid", True, 1, 1, "max", False, F32),
    (5, 60, 4, "softmax", False, 1, 1, "max", False, BF),
    (33, 64, 8, "sigmoid", False, 8, 3, "max", True, F32),
    (17, 160, 6, "softmax", False, 8, 3, "max", False, BF),
    (65, 256, 8, "sigmoid", True, 8, 4, "top2", True, F32),
    (40, 256, 8, "softmax", True, 8, 4, "top2", True, F32),
    (31, 384, 8, "sigmoid", True, 1, 1, "max", True, HF),
    (9, 1000, 32, "softmax", True, 10, 5, "max", False, F32),
    (9, 1024, 5, "sigmoid", False, 32, 7, "top2", True, BF),
    (20, 33, 33 - 1, "softmax", False, 1, 1, "max", True, F32),
    (12, 24, 24, "sigmoid", True, 3, 2, "top2", True, F32),
    (100, 96, 6, "softmax", True, 96, 48, "max", True, F32),
]


@pytest.mark.parametrize("T,E,k,score,bias,groups,top_groups,gscore,renorm,dtype", ROUTE)
def test_route(T, E, k, score, bias, groups, top_groups, gscore, renorm, dtype):
    l = randn(T, E, seed=T + E, std=1.5, dtype=dtype)
    b = randn(E, seed=7, std=0.1) if bias else None
    check_route(l, k, score, b, groups, top_groups, gscore, renorm, 2.5)
    l[:, ::5] = float("-inf")  # masked experts; in small groups whole groups
    l[T // 2, :] = float("-inf")  # a row that leaves nothing
    if E > 3:
        l[0, 2:] = float("-inf")  # a row that leaves fewer than k
    check_route(l, k, score, b, groups, top_groups, gscore, renorm, 1.0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_lowest_value_and_nan(score):
    l = randn(6, 40, seed=1)
    l[1, :] = torch.finfo(F32).min          # all at the lowest value of the type: an ordinary tie
    l[2, 5:] = torch.finfo(F32).min
    l[3, 7] = float("nan")
    l[4, 3], l[4, 9] = float("nan"), float("-inf")
    check_route(l, 6, score)
    check_route(l, 6, score, renorm=False)


def test_route_masked_by_bias():
    l = randn(8, 32, seed=3)
    b = torch.zeros(32, device="cuda")
    b[4:] = float("-inf")
    w, e = check_route(l, 6, "sigmoid", b)
    assert (e[:, 4:] == -1).all() and (w[:, 4:] == 0).all()


def test_route_ties_take_the_lower_expert():
    l = (randn(64, 128, seed=5) * 2).round().to(BF)  # a handful of different values
    for score in ("softmax", "sigmoid"):
        check_route(l, 8, score)
        check_route(l, 8, score, groups=8, top_groups=3)
        check_route(l, 8, score, bias=torch.zeros(128, device="cuda"))
        check_route(l, 8, score, bias=torch.full((128,), 0.25, device="cuda"), groups=8, top_groups=3, gscore="top2")


@pytest.mark.parametrize("E,groups", [(64, 1), (256, 8)])
def test_route_choices_that_fp32_cannot_tell_apart(E, groups):
    """s + b is the same number for all experts but for the rounding of b to fp32: the order lies below fp32's step of
    the sum and has to be that of 64 bits."""
    l = randn(1, E, seed=11)
    s = torch.sigmoid(l.to(D))
    b = (0.9 - s).to(F32).view(-1)
    l = l.repeat(20, 1)
    l[10:] += randn(10, E, seed=12, std=1e-7)
    spread = (torch.sigmoid(l[0].to(D)) + b.to(D))
    assert (spread.max() - spread.min()) < 1e-6
    check_route(l, 8, "sigmoid", b, groups, max(1, groups // 2), "top2" if groups > 1 else "max")


@pytest.mark.parametrize("E,k", [(64, 6), (64, 32), (256, 8), (24, 3), (1024, 1)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties_that_only_64_bits_tell_apart(E, k, score):
    """Scores that are one number in fp32: at the border of the choice stand experts that are the same, and behind them
    others, some of them better in 64 bits."""
    zero = torch.zeros(E, device="cuda")
    l = torch.zeros((40, E), device="cuda")
    l[:20] = -600.0 if score == "sigmoid" else -200.0   # all of them 0 in fp32, but for an expert that is not
    l[:20, 1] = 1.0
    l[20:] = 1e-4                                       # 1 ulp of the score apart, or less
    step = torch.where(torch.arange(40, device="cuda") < 20, 4.0, 2e-8)
    for t in range(40):
        n = 1 + t % 10
        at = torch.randperm(E, device="cuda", generator=gen(t))[:n]
        if t < 20:
            at = at[at != 1]
        l[t, at] += step[t]                             # a few above the rest
        l[t, at[::3]] += step[t]
    check_route(l, k, score, zero)
    check_route(l, k, score, zero + 0.25)
    if E >= 64:
        check_route(l, k, score, zero, groups=4, top_groups=2, gscore="top2")
        check_route(l.to(BF), k, score, zero)


def test_route_ties_at_the_border_are_not_always_alike():
    """The last chosen expert and the next one are the same, a third lies within fp32's error of them and is better."""
    l = torch.full((60, 96), -4.0, device="cuda")
    for t in range(60):
        at = torch.randperm(96, device="cuda", generator=gen(t))[:8]
        l[t, at[:4]] = torch.tensor([3.0, 2.5, 2.0, 1.5], device="cuda")
        l[t, at[4:7]] = 1.0
        l[t, at[7]] = 1.0 + (1 + t % 3) * 2.0 ** -23
    for k in (4, 5, 6, 7, 8):
        check_route(l, k, "sigmoid", torch.full((96,), 4.0, device="cuda"))
        check_route(l, k, "softmax", torch.full((96,), 4.0, device="cuda"))


def route_choice_64(l, bias, k, score, groups, top_groups):
    """Experts by top-2 group scores, in 64 bits on the GPU (many rows)."""
    s = torch.sigmoid(l.to(D)) if score == "sigmoid" else torch.softmax(l.to(D), 1)
    c = s + bias.to(D)
    T, E = l.shape
    two = torch.sort(c.view(T, groups, -1), dim=2, descending=True)[0][:, :, :2].sum(2)
    best = torch.sort(two, dim=1, descending=True, stable=True)[1][:, :top_groups]
    kept = torch.zeros_like(two, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(E // groups, 1)
    return torch.sort(c.masked_fill(~kept, float("-inf")), dim=1, descending=True, stable=True)[1][:, :k].to(torch.int32)


@pytest.mark.parametrize("E,groups", [(256, 128), (256, 32), (1024, 16), (96, 16), (24, 12)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups_whose_two_choices_cancel(E, groups, score):
    """Biases +b and -b in every group: the sum of the two is small beside the roundings of its terms."""
    import b2x
    gs = E // groups
    for b in (0.5, 4.0, 16.0, 100.0, 1e4):
        bias = torch.full((groups, gs), -3.0 * b, device="cuda")
        bias[:, 0], bias[:, 1] = b, -b
        l = randn(8000, E, seed=int(b), std=1.5)
        k = min(8, groups // 2)
        _, e = b2x.moe_route(l, k, score=score, bias=bias.view(-1), num_groups=groups, top_groups=k, group_score="top2")
        ref = route_choice_64(l, bias.view(-1), k, score, groups, k)
        assert int((e != ref).any(1).sum()) == 0, b


def test_route_groups_with_one_far_larger_bias():
    """The uncertain group need not be the next one: one of large terms may stand far behind it in fp32."""
    import b2x
    E, groups = 64, 8
    l = randn(8000, E, seed=5, std=1e-2)
    bias = torch.zeros((groups, 8), device="cuda")
    bias[::2, 0], bias[::2, 1], bias[::2, 2:] = 3e4, -3e4, -1e5   # half of the groups: s1 + s2 after cancellation
    _, e = b2x.moe_route(l, 4, score="softmax", bias=bias.view(-1), num_groups=groups, top_groups=4, group_score="top2")
    assert torch.equal(e, route_choice_64(l, bias.view(-1), 4, "softmax", groups, 4))


@pytest.mark.parametrize("E,groups", [(32, 8), (256, 8), (96, 16), (60, 5)])
def test_route_groups_of_the_lowest_bias(E, groups):
    """Experts that a bias of the type's lowest value puts last are still experts: their groups are not empty."""
    l = randn(9, E, seed=1)
    bias = torch.zeros((groups, E // groups), device="cuda")
    bias[2:] = torch.finfo(F32).min
    k = min(32, 3 * (E // groups) - 1)
    for score in ("softmax", "sigmoid"):
        _, e = check_route(l, k, score, bias.view(-1), groups, 4, "top2")
        check_route(l, k, score, bias.view(-1), groups, 4, "max")
        assert (e >= 0).all()


@pytest.mark.parametrize("E,k", [(24, 4), (64, 8), (256, 8), (1024, 32)])
@pytest.mark.parametrize("std,base", [(1.5, 0.0), (15.0, 0.0), (3.0, -20.0), (1.5, -80.0), (30.0, 7.3)])
def test_route_weights_to_a_few_units(E, k, std, base):
    """u = 2^-24.  The exponential is off by 2 units in the last place (4 u), with the difference put back 5 u; 1 + e by
    3 u; each division, product and level of the warp's sum by u.
      sigmoid              8 u, scale u                                               9 u
      sigmoid, quotient    9 u above; 9 u and 5 levels below; division, scale         25 u
      softmax of the k     5 u above; 5 u and 5 levels below; division, scale         17 u
      softmax of all       5 u above; below each term by 4 u (2^-22, the approximate exponential) and by 3 u of its distance
                           from the maximum, which in the mean over the softmax is at most ln E; levels 5 and experts a
                           lane at most 2 ceil(E / 32); division, scale               (16 + 5 + 3 ln E + 2 ceil(E / 32)) u"""
    import b2x
    u = 2.0 ** -24
    l = randn(200, E, seed=E, std=std) + base
    for score, renorm, bound in (("sigmoid", False, 9), ("sigmoid", True, 25), ("softmax", True, 17),
                                 ("softmax", False, 21 + 3 * np.log(E) + 2 * -(-E // 32))):
        w, e = b2x.moe_route(l, k, score=score, renormalize=renorm, scale=1.7)
        s = torch.sigmoid(l.to(D)) if score == "sigmoid" else torch.softmax(l.to(D), 1)
        c = s.gather(1, e.long())
        ref = float(np.float32(1.7)) * (c / c.sum(1, keepdim=True) if renorm else c)
        check(w, ref, bound * u * ref + 2.0 ** -146, (score, renorm))


def test_route_strided_logits_and_no_tokens():
    import b2x
    l = randn(30, 200, seed=1)
    check_route(l[:, 5:69], 4)
    check_route(l.t()[:100, :], 3)
    w, e = b2x.moe_route(l[:0], 4)
    assert w.shape == e.shape == (0, 4)


@pytest.mark.parametrize("base", [-20.0, -60.0, -88.0, -100.0, -200.0, -600.0])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_route_sigmoid_of_low_logits(base, dtype):
    """Renormalised weights sum to the scale however small the scores, and so do their gradients' parts."""
    import b2x
    l = (randn(33, 64, seed=3, std=1.5) + base).to(dtype)
    l[1, 2:] = float("-inf")                     # fewer than k are left
    l[2, 5] = base / 2                           # one far above the others
    l[3, 7] = 1.0                                # and one that is not small
    w, e = check_route(l, 6, "sigmoid", scale=1.7)
    assert (w.sum(1) - 1.7).abs().max() < 1e-5
    check_route(l, 6, "sigmoid", groups=8, top_groups=3)
    g = randn(33, 6, seed=4)
    got = b2x.moe_route_backward(g, l, e, score="sigmoid", scale=1.7)
    z = l.to(D).requires_grad_()
    c = torch.where(e >= 0, torch.sigmoid(z).gather(1, e.clamp_min(0).long()), torch.zeros((), dtype=D, device="cuda"))
    (1.7 * c / c.sum(1, keepdim=True) * g.to(D)).sum().backward()
    ref = torch.nan_to_num(z.grad, nan=0.0)
    check(got, ref, 1e-5 * 1.7 * g.to(D).abs().sum(1, keepdim=True) + rounded(dtype, ref))
    assert got[4:].abs().amax(1).min() > 1e-7  # nothing vanished


def test_route_sigmoid_of_the_lowest_value():
    """Scores that are 0 in 64 bits too: weights and gradients 0, no NaN; a NaN among them stays one."""
    import b2x
    l = torch.full((3, 16), torch.finfo(F32).min, device="cuda")
    l[1, 4] = float("nan")
    w, e = check_route(l, 4, "sigmoid")
    assert (w[0] == 0).all() and torch.isnan(w[1]).all()
    w, e = check_route(l, 1, "sigmoid")
    assert torch.isnan(w[1]).all()
    d = b2x.moe_route_backward(torch.ones((3, 1), device="cuda"), l, e, score="sigmoid")
    assert (d[0] == 0).all() and (d[2] == 0).all()


@pytest.mark.parametrize("E", [192, 320, 352, 512, 768])
@pytest.mark.parametrize("score,dtype", [("sigmoid", F32), ("softmax", BF)])
def test_route_of_other_widths(E, score, dtype):
    """6, 10, 12, 16 and 32 experts a lane, with and without bias and groups, forward and backward."""
    test_route(20, E, 8, score, True, 16, 5, "top2", True, dtype)
    test_route(20, E, 8, score, False, 16, 5, "max", False, dtype)
    test_route(20, E, 31, score, True, 1, 1, "max", False, dtype)
    test_route_backward(20, E, 8, score, True, dtype)
    test_route_backward(20, E, 8, score, False, dtype)


@pytest.mark.parametrize("T,E,k,score,renorm,dtype", [
    (1, 8, 2, "softmax", True, F32), (33, 64, 8, "softmax", False, F32), (17, 160, 6, "sigmoid", True, BF),
    (9, 1000, 32, "sigmoid", False, F32), (40, 60, 1, "softmax", True, HF), (65, 128, 8, "softmax", False, BF),
    (3, 5, 5, "softmax", True, F32)])
def test_route_backward(T, E, k, score, renorm, dtype):
    import b2x
    l = randn(T, E, seed=3, std=1.5, dtype=dtype)
    if E > 20:
        l[:, ::7] = float("-inf")
    w, e = b2x.moe_route(l, k, score=score, renormalize=renorm, scale=1.7)
    e[T // 2, k - 1] = -1  # an empty slot
    g = randn(T, k, seed=4)
    got = b2x.moe_route_backward(g, l, e, score=score, renormalize=renorm, scale=1.7)
    z = l.to(D).requires_grad_()
    s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
    c = torch.where(e >= 0, s.gather(1, e.clamp_min(0).long()), torch.zeros((), dtype=D, device="cuda"))
    w64 = 1.7 * (c / c.sum(1, keepdim=True) if renorm else c)
    (w64 * g.to(D)).sum().backward()
    ref = torch.nan_to_num(z.grad, nan=0.0)
    # each term of the gradient has size <= 1.7 sum |g| (the weights sum to at most scale or, sigmoid without
    # renormalizing, each is at most scale) and 1e-5 relative error; rounding of the type on top
    size = 1.7 * g.to(D).abs().sum(1, keepdim=True)
    assert got.dtype == dtype and got.shape == l.shape
    check(got, ref, 1e-5 * size + rounded(dtype, ref))


def test_route_backward_against_differences():
    import b2x
    l, g = randn(4, 12, seed=1), randn(4, 3, seed=2)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            _, e = b2x.moe_route(l, 3, score=score, renormalize=renorm)
            got = b2x.moe_route_backward(g, l, e, score=score, renormalize=renorm)

            def f(z):
                s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
                c = s.gather(1, e.long())
                return ((c / c.sum(1, keepdim=True) if renorm else c) * g.to(D)).sum(1)

            for i in range(12):
                h = torch.zeros((4, 12), dtype=D, device="cuda")
                h[:, i] = 1e-5
                ref = (f(l.to(D) + h) - f(l.to(D) - h)) / 2e-5
                check(got[:, i], ref, 1e-5 * g.to(D).abs().sum(1) + 1e-8)


def test_route_backward_same_expert_twice():
    """Two slots that name one expert: the gradient of the sum of both weights."""
    import b2x
    l = randn(2, 6, seed=1)
    e = torch.tensor([[1, 1, 4], [0, 5, 0]], device="cuda", dtype=torch.int32)
    g = randn(2, 3, seed=2)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = b2x.moe_route_backward(g, l, e, score=score, renormalize=renorm)
            z = l.to(D).requires_grad_()
            s = torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)
            c = s.gather(1, e.long())
            ((c / c.sum(1, keepdim=True) if renorm else c) * g.to(D)).sum().backward()
            check(got, z.grad, 1e-5 * g.to(D).abs().sum(1, keepdim=True))


# ------------------------------------------------------------------------------------------------- dispatch


def quant_rows(x, dtype, given=None):
    """The framework's cast recipe, row by row, in fp32 on the CPU."""
    x = x.float().cpu()
    m = torch.nan_to_num(x.abs(), nan=0.0, posinf=float("inf")).amax(1) if x.shape[1] else torch.zeros(x.shape[0])
    s = m / FMAX[dtype] if given is None else given.float().cpu().expand(x.shape[0])
    inv = torch.where(s == 0, torch.zeros_like(s), 1 / s)
    y = x * inv[:, None]
    y = torch.where(torch.isnan(y), torch.full_like(y, FMAX[dtype]), y.clamp(-FMAX[dtype], FMAX[dtype]))
    return y.to(dtype), s


def check_dispatch(x, e, E, dtype=E4, given=None):
    import b2x
    T, k = e.shape
    H = x.shape[1]
    out = torch.full((T * k, H), 3.0, device="cuda").to(dtype)
    q, s, plan = b2x.moe_dispatch(x, e, E, dtype=dtype, scale=given, out=out)
    flat = e.reshape(-1).cpu().long()
    ok = (flat >= 0) & (flat < E)
    order = [i for i in torch.sort(torch.where(ok, flat, torch.full_like(flat, E)), stable=True)[1].tolist() if ok[i]]
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    for r, i in enumerate(order):
        rows[i] = r
    counts = torch.bincount(flat[ok], minlength=E)
    assert torch.equal(plan.offsets.cpu(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]).to(torch.int32))
    assert torch.equal(plan.rows.cpu(), rows.view(T, k))
    Q, S = quant_rows(x, dtype, given)
    token = torch.tensor([i // k for i in order], dtype=torch.long)
    n = len(order)
    assert torch.equal(q[:n].cpu().view(torch.uint8), Q[token].view(torch.uint8))
    assert torch.equal(q[n:].float(), torch.full((T * k - n, H), 3.0, device="cuda")), "rows behind the last were written"
    if given is None:
        assert torch.equal(s[:n].cpu(), S[token])
    else:
        assert torch.equal(s.cpu(), given.cpu().float().view(1))
    return q, s, plan


@pytest.mark.parametrize("T,H,E,k", [(1, 16, 1, 1), (1, 100, 8, 2), (7, 33, 5, 3), (16, 2048, 64, 8), (100, 7000, 16, 4), (256, 272, 128, 8),
                                     (257, 48, 128, 8), (1000, 72, 1000, 3), (3001, 16, 64, 6), (5, 9000, 4, 2), (4, 20001, 3, 2)])
@pytest.mark.parametrize("dtype,q", [(BF, E4), (F32, E5)])
def test_dispatch(T, H, E, k, dtype, q):
    x = randn(T, H, seed=T, dtype=dtype)
    e = torch.randint(0, E, (T, k), device="cuda", generator=gen(5), dtype=torch.int32)
    check_dispatch(x, e, E, q)
    e[::3, 0] = -1           # dropped pairs
    e[::4, k - 1] = E + 5
    check_dispatch(x, e, E, q, torch.tensor([0.013], device="cuda"))
    e[:] = E - 1             # every pair to one expert
    check_dispatch(x, e, E, q)
    e[:] = -1                # nothing left
    check_dispatch(x, e, E, q)


@pytest.mark.parametrize("T,k", [(8193, 8), (16385, 8), (140000, 1)])
def test_dispatch_of_many_pairs(T, k):
    """More than 65536 pairs: the plan's warps take several rounds."""
    e = torch.randint(-2, 70, (T, k), device="cuda", generator=gen(5), dtype=torch.int32)
    check_dispatch(randn(T, 16, seed=T, dtype=BF), e, 64)


def test_dispatch_special_values_strides_and_wide_integers():
    x = randn(12, 300, seed=1)
    x[0] = 0.0
    x[1, 5] = float("nan")
    x[2, 6] = float("inf")
    x[3] = torch.finfo(F32).max
    x[4] = 1e-42
    e = torch.randint(0, 6, (12, 2), device="cuda", generator=gen(1))
    assert e.dtype == torch.int64
    check_dispatch(x, e, 6)
    check_dispatch(x[:, 1:200], e, 6)                  # rows off the 16-byte grid
    check_dispatch(x[:, 8:264], e.int().t().contiguous().t(), 6)
    check_dispatch(x.t()[:12, :12].to(BF), e, 6)


def test_dispatch_no_tokens():
    import b2x
    q, s, plan = b2x.moe_dispatch(torch.empty((0, 64), device="cuda"), torch.empty((0, 2), device="cuda", dtype=torch.int32), 5)
    assert q.shape == (0, 64) and s.shape == (0,) and plan.rows.shape == (0, 2)
    assert torch.equal(plan.offsets, torch.zeros(6, device="cuda", dtype=torch.int32))


# ------------------------------------------------------------------------------------------------- experts' products


def offsets_of(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), device="cuda", dtype=torch.int32)


def experts_ref(x, w, counts, sx, sw):
    """(y, size): exact products and sum |x||w|, both scaled."""
    Y, S, lo = [], [], 0
    for e, c in enumerate(counts):
        xe, we = x[lo:lo + c].to(D), w[e].to(D)
        f = torch.ones((c, 1), dtype=D, device="cuda")
        if sx is not None:
            f = f * (sx[lo:lo + c] if sx.numel() > 1 else sx.expand(c)).to(D)[:, None]
        if sw is not None:
            f = f * (sw[e] if sw.numel() > 1 else sw[0]).to(D)
        Y.append(xe @ we.t() * f)
        S.append(xe.abs() @ we.abs().t() * f)
        lo += c
    return torch.cat(Y), torch.cat(S)


EXPERTS = [  # counts, N, K, layout, rows behind
    ([1], 128, 128, "nk", 0),
    ([0, 1, 0, 3], 200, 144, "nk", 0),
    ([2, 1, 0, 5, 1, 0, 0, 7], 1000, 512, "nk", 3),
    ([17, 0, 30, 5], 264, 1040, "kn", 0),
    ([64, 100, 1, 47], 384, 640, "nk", 9),
    ([300, 0, 129, 257], 130, 272, "kn", 2),
    ([0, 0, 0, 700], 1152, 256, "nk", 0),
    ([5] * 70, 256, 384, "nk", 1),
    ([0, 0, 0], 128, 128, "nk", 4),
    ([513, 511, 256, 2, 1000], 520, 1024, "nk", 5),
    ([9, 8], 40, 100, "nk", 0),
    ([5] * 70, 1100, 384, "nk", 1),
    ([1, 0, 300, 33, 513] * 14, 640, 144, "nk", 3),
    ([0, 70, 17, 256, 31, 1, 257] * 10, 528, 272, "kn", 3),
    ([0] * 999 + [4200], 1300, 128, "nk", 6),
    ([3] * 1000, 300, 256, "nk", 0),
]


@pytest.mark.parametrize("counts,N,K,layout,behind", EXPERTS)
@pytest.mark.parametrize("out", [BF, HF])
def test_moe_gemm(counts, N, K, layout, behind, out):
    import b2x
    E, n = len(counts), sum(counts)
    R = n + behind
    x = fp8(R, K, seed=1)
    w = fp8(E, N, K, seed=2) if layout == "nk" else fp8(E, K, N, seed=2).transpose(1, 2)
    sx = torch.rand(R, device="cuda", generator=gen(3)) * 0.02 + 0.01
    sw = (torch.rand(E, device="cuda", generator=gen(4)) + 0.5) * K ** -0.5 / 30
    y = torch.full((R, N), 5.0, device="cuda", dtype=out)
    r = b2x.moe_gemm(x, w, offsets_of(counts), scale_x=sx, scale_w=sw, out_dtype=out, out=y)
    assert r is y
    ref, size = experts_ref(x, w, counts, sx, sw)
    err = (K + 4) * 2.0 ** -23 * size
    check(y[:n], ref, err + rounded(out, ref.abs() + err))
    assert (y[n:] == 5).all(), "rows behind the last expert's were written"
    y2 = b2x.moe_gemm(x, w, offsets_of(counts), scale_x=sx, scale_w=sw, out_dtype=out)
    assert torch.equal(y2[:n], y[:n])


@pytest.mark.parametrize("da,dw,one", [(E4, E5, True), (E5, E4, False)])
def test_moe_gemm_formats_and_single_scales(da, dw, one):
    import b2x
    counts = [3, 40, 0, 21]
    x, w = fp8(64, 256, seed=1, dtype=da, std=2.0), fp8(4, 136, 256, seed=2, dtype=dw, std=2.0)
    sx, sw = (torch.tensor([0.5], device="cuda"), torch.tensor([0.25], device="cuda")) if one else (None, None)
    ref, size = experts_ref(x, w, counts, sx, sw)
    err = 260 * 2.0 ** -23 * size
    check(b2x.moe_gemm(x, w, offsets_of(counts), scale_x=sx, scale_w=sw), ref, err + rounded(BF, ref.abs() + err))


def test_moe_gemm_gradient_of_the_rows():
    """dX = dY W with the forward's weights, by a transposed view."""
    import b2x
    counts, N, K = [20, 0, 45, 3], 144, 272
    dy, w = fp8(68, N, seed=1), fp8(4, N, K, seed=2)
    got = b2x.moe_gemm(dy, w.transpose(1, 2), offsets_of(counts))
    ref, size = experts_ref(dy, w.transpose(1, 2), counts, None, None)
    err = (N + 4) * 2.0 ** -23 * size
    check(got, ref, err + rounded(BF, ref.abs() + err))


def test_moe_gemm_strided_x_and_out():
    import b2x
    counts = [7, 12, 31]
    x, w = fp8(50, 400, seed=1)[:, 16:272], fp8(3, 300, 256, seed=2)[:, 10:210]
    y = torch.full((50, 333), 2.0, device="cuda", dtype=BF)
    b2x.moe_gemm(x, w, offsets_of(counts), out=y[:, 7:207])
    ref, size = experts_ref(x, w, counts, None, None)
    err = 260 * 2.0 ** -23 * size
    check(y[:, 7:207], ref, err + rounded(BF, ref.abs() + err))
    assert (y[:, :7] == 2).all() and (y[:, 207:] == 2).all()


def test_moe_gemm_offsets_past_the_rows_stay_inside():
    """Offsets that claim more rows than there are: only those that are there are written."""
    import b2x
    x, w = fp8(20, 128, seed=1), fp8(2, 128, 128, seed=2)
    buf = torch.full((40, 128), 9.0, device="cuda", dtype=BF)
    b2x.moe_gemm(x, w, torch.tensor([0, 8, 4000], device="cuda", dtype=torch.int32), out=buf[:20])
    ref, size = experts_ref(x, w, [8, 12], None, None)
    err = 132 * 2.0 ** -23 * size
    check(buf[:20], ref, err + rounded(BF, ref.abs() + err))
    assert (buf[20:] == 9).all()


def interleaved(E, I, K, seed):
    import b2x
    wg, wu = fp8(E, I, K, seed=seed), fp8(E, I, K, seed=seed + 1)
    return wg, wu, torch.stack([b2x.interleave_gate_up(wg[e], wu[e]) for e in range(E)])


def check_codes(q, ref, err, dtype):
    """fp8 codes of ref (error err before rounding): the nearest, or its neighbour where the border is within err."""
    lim = FMAX[dtype]
    lo, hi = (ref - err).clamp(-lim, lim), (ref + err).clamp(-lim, lim)
    got = q.to(D)
    a, b = lo.float().to(dtype).to(D), hi.float().to(dtype).to(D)
    bad = (got < a) | (got > b)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} codes"


@pytest.mark.parametrize("counts,I,K,behind", [([1], 128, 128, 0), ([3, 0, 1, 9], 256, 400, 2), ([40, 64, 0, 21], 128, 272, 0),
                                               ([300, 129, 1], 384, 512, 5), ([1024, 700, 0, 513], 256, 1024, 1),
                                               ([7, 0, 290, 1] * 20, 384, 272, 4)])
@pytest.mark.parametrize("dtype", [E4, E5])
def test_moe_gemm_swiglu(counts, I, K, behind, dtype):
    import b2x
    E, n = len(counts), sum(counts)
    R = n + behind
    x = fp8(R, K, seed=1)
    wg, wu, w = interleaved(E, I, K, 2)
    sx = torch.rand(R, device="cuda", generator=gen(3)) * 0.02 + 0.01
    sw = (torch.rand(E, device="cuda", generator=gen(4)) + 0.5) * K ** -0.5 / 30
    hs = torch.tensor([0.02 if dtype == E4 else 0.002], device="cuda")
    amax = torch.zeros(1, device="cuda")
    out = torch.full((R, I), 1.0, device="cuda").to(dtype)
    h = b2x.moe_gemm_swiglu(x, w, offsets_of(counts), hs, scale_x=sx, scale_w=sw, h_dtype=dtype, h_amax=amax, out=out)
    g, gs = experts_ref(x, wg, counts, sx, sw)
    u, us = experts_ref(x, wu, counts, sx, sw)
    ref = act(g, "silu") * u
    ge, ue = (K + 4) * 2.0 ** -23 * gs, (K + 4) * 2.0 ** -23 * us
    err = 1.2 * ge * (u.abs() + ue) + act(g, "silu").abs() * ue + 4e-6 * ref.abs()
    check_codes(h[:n], ref / hs.to(D), err / hs.to(D), dtype)
    assert (h[n:].float() == 1).all()
    top = ref.abs().max()
    assert abs(amax.to(D).item() - top.item()) <= err.max().item()


# ------------------------------------------------------------------------------------------------- combine


@pytest.mark.parametrize("T,k,H,dtype", [(1, 1, 8, BF), (1, 1, 1, F32), (5, 3, 7, BF), (64, 8, 256, BF), (33, 9, 1000, HF), (100, 2, 2050, F32),
                                         (17, 32, 520, BF)])
def test_combine_and_backward(T, k, H, dtype):
    import b2x
    R = T * k + 3
    y = randn(R, H, seed=1, dtype=dtype)
    rows = torch.randperm(R, device="cuda", generator=gen(2))[:T * k].view(T, k).to(torch.int32)
    rows[::2, k - 1] = -1
    rows[T // 2, :] = -1                       # a token that lost every pair
    w = torch.rand((T, k), device="cuda", generator=gen(3))
    res = randn(T, H, seed=4, dtype=dtype)
    live = (rows >= 0)[:, :, None]
    yr = torch.where(live, y.to(D)[rows.clamp_min(0).long()], torch.zeros((), dtype=D, device="cuda"))
    for wt, r in ((w, res), (None, None), (w, None)):
        got = b2x.moe_combine(y, rows, wt, residual=r)
        terms = yr if wt is None else yr * wt.to(D)[:, :, None]
        ref, size = terms.sum(1), terms.abs().sum(1)
        if r is not None:
            ref, size = ref + r.to(D), size + r.to(D).abs()
        check(got, ref, (k + 1) * 2.0 ** -24 * size + rounded(dtype, size))
    g = randn(T, H, seed=5, dtype=dtype)
    dy = torch.full((R, H), 7.0, device="cuda", dtype=dtype)
    dy2, dw = b2x.moe_combine_backward(g, y, rows, w, out=dy)
    assert dy2 is dy
    ref = torch.full((R, H), 7.0, dtype=D, device="cuda")
    sel = rows.view(-1) >= 0
    ref[rows.view(-1)[sel].long()] = (w.to(D)[:, :, None] * g.to(D)[:, None, :]).view(T * k, H)[sel]
    check(dy, ref, rounded(dtype, ref) + 2.0 ** -24 * ref.abs(), "d_y")
    prod = yr * g.to(D)[:, None, :]
    check(dw, prod.sum(2), H * 2.0 ** -24 * prod.abs().sum(2) + 1e-30, "d_weights")


# several column steps and several CTAs a token; more of them than go side by side (the second and the last two)
@pytest.mark.parametrize("T,k,H,dtype", [(60, 8, 7168, BF), (22000, 2, 2056, BF), (50, 9, 7168, HF), (33, 3, 4500, F32), (3000, 4, 2049, BF),
                                         (2500, 1, 1030, F32)])
def test_combine_and_backward_wide(T, k, H, dtype):
    test_combine_and_backward(T, k, H, dtype)


def test_combine_backward_against_differences():
    import b2x
    y, w = randn(6, 16, seed=1), torch.rand((3, 2), device="cuda", generator=gen(2))
    rows = torch.tensor([[4, 0], [1, 5], [3, -1]], device="cuda", dtype=torch.int32)
    g = randn(3, 16, seed=3)
    dy, dw = b2x.moe_combine_backward(g, y, rows, w, out=torch.zeros_like(y))

    def f(yy, ww):
        t = torch.where((rows >= 0)[:, :, None], yy[rows.clamp_min(0).long()], torch.zeros((), dtype=D, device="cuda"))
        return ((t * ww[:, :, None]).sum(1) * g.to(D)).sum()

    for idx in ((0, 1), (2, 0), (2, 1)):
        h = torch.zeros((3, 2), dtype=D, device="cuda")
        h[idx] = 1e-3
        ref = (f(y.to(D), w.to(D) + h) - f(y.to(D), w.to(D) - h)) / 2e-3
        assert abs(dw[idx].item() - ref.item()) <= 16 * 2.0 ** -24 * 16 * 9 + 1e-9
    for idx in ((4, 3), (5, 0), (2, 2)):
        h = torch.zeros((6, 16), dtype=D, device="cuda")
        h[idx] = 1e-3
        ref = (f(y.to(D) + h, w.to(D)) - f(y.to(D) - h, w.to(D))) / 2e-3
        assert abs(dy[idx].item() - ref.item()) <= 1e-6


def test_combine_strided_and_rows_outside():
    import b2x
    y = randn(20, 300, seed=1, dtype=BF)[:, 1:130]
    rows = torch.tensor([[0, 19], [20, 3], [1 << 30, -5]], device="cuda", dtype=torch.int64)
    w = torch.rand((3, 2), device="cuda", generator=gen(2)).to(BF)
    got = b2x.moe_combine(y, rows, w)
    ref = torch.stack([w[0, 0].to(D) * y[0].to(D) + w[0, 1].to(D) * y[19].to(D), w[1, 1].to(D) * y[3].to(D), torch.zeros(129, dtype=D, device="cuda")])
    check(got, ref, rounded(BF, ref) + 1e-6)
    assert b2x.moe_combine(y, rows[:0]).shape == (0, 129)


# ------------------------------------------------------------------------------------------------- together


def layer(x, router, w_gu, w_down, sgu, sdown, hs, k, mask=None):
    """A mixture-of-experts layer as it is used: every step on the device."""
    import b2x
    logits = x.float() @ router
    if mask is not None:
        logits = logits.masked_fill(mask[:, None], float("-inf"))  # a padded batch
    w, e = b2x.moe_route(logits, k, score="sigmoid", renormalize=True)
    q, s, plan = b2x.moe_dispatch(x, e, w_gu.shape[0])
    h = b2x.moe_gemm_swiglu(q, w_gu, plan.offsets, hs, scale_x=s, scale_w=sgu)
    y = b2x.moe_gemm(h, w_down, plan.offsets, scale_x=hs, scale_w=sdown)
    return b2x.moe_combine(y, plan.rows, w, residual=x), (logits, w, e, q, s, plan, h, y)


def layer_weights(E, H, I, seed=10):
    wg, wu, w_gu = interleaved(E, I, H, seed)
    w_down = fp8(E, H, I, seed=seed + 5)
    sgu = torch.full((E,), H ** -0.5 / 40, device="cuda")
    sdown = torch.full((E,), I ** -0.5 / 40, device="cuda")
    router = randn(H, E, seed=seed + 6, std=H ** -0.5)
    return wg, wu, w_gu, w_down, sgu, sdown, router, torch.tensor([0.02], device="cuda")


@pytest.mark.parametrize("T,E,H,I,k", [(1, 8, 256, 128, 2), (50, 8, 384, 256, 2), (600, 16, 512, 128, 4)])
def test_layer(T, E, H, I, k):
    import b2x
    wg, wu, w_gu, w_down, sgu, sdown, router, hs = layer_weights(E, H, I)
    x = randn(T, H, seed=1, dtype=BF)
    mask = torch.zeros(T, dtype=torch.bool, device="cuda")
    mask[T // 2 + 1:] = T > 1
    before = b2x.launch_count()
    out, (logits, w, e, q, s, plan, h, y) = layer(x, router, w_gu, w_down, sgu, sdown, hs, k, mask)
    assert b2x.launch_count() > before
    assert (e[mask] == -1).all() and torch.equal(out[mask], x[mask])  # padding passes through
    # in 64 bits from the quantized rows on (h's codes are one step off at most, and only at borders)
    ref = x.to(D)
    tol = torch.zeros_like(ref)
    n = int(plan.offsets[-1])
    counts = (plan.offsets[1:] - plan.offsets[:-1]).tolist()
    g, _ = experts_ref(q, wg, counts, s, sgu)
    u, _ = experts_ref(q, wu, counts, s, sgu)
    href = (act(g, "silu") * u / hs.to(D)).clamp(-448, 448)
    assert ((h[:n].to(D) - href).abs() <= 2.0 ** -4 * href.abs() * 1.01 + 2.0 ** -10).all()
    yref, size = experts_ref(h, w_down, counts, hs, sdown)
    for t in range(T):
        for j in range(k):
            r = int(plan.rows[t, j])
            if r >= 0:
                ref[t] += w[t, j].to(D) * yref[r]
                tol[t] += w[t, j].to(D) * (2.0 ** -8 * yref[r].abs() + (I + 8) * 2.0 ** -23 * size[r]) + 2.0 ** -23 * yref[r].abs()
    check(out, ref, tol + rounded(BF, ref.abs() + tol) + 2.0 ** -22 * ref.abs())


@pytest.mark.parametrize("T", [40, 700, 9000])
def test_layer_captured_and_replayed(T):
    """Two graphs of one layer, two sets of inputs: the replays follow the new routing with the bits of the eager run."""
    wg, wu, w_gu, w_down, sgu, sdown, router, hs = layer_weights(8, 256, 128)
    x = randn(T, 256, seed=1, dtype=BF)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer(x, router, w_gu, w_down, sgu, sdown, hs, 2)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs of the same calls
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, _ = layer(x, router, w_gu, w_down, sgu, sdown, hs, 2)
        graphs.append((g, out))
    for seed in (2, 3):
        x.copy_(randn(T, 256, seed=seed, dtype=BF))
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        for st, (g, _) in zip((a, b), graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        want, _ = layer(x.clone(), router, w_gu, w_down, sgu, sdown, hs, 2)
        for _, out in graphs:
            assert torch.equal(out, want)


def test_gemm_epilogue_captured_and_on_two_streams():
    import b2x
    a, b = fp8(5, 4096, seed=1), fp8(512, 4096, seed=2).t()
    want = b2x.gemm_epilogue(a, b, activation="silu")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(b2x.gemm_epilogue(a, b, activation="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = b2x.gemm_epilogue(a, b, activation="silu")
    out.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_layer_gradients_against_differences():
    """Backward of route and combine around fixed experts' outputs: the layer's gradient by the router's logits."""
    import b2x
    T, E, k, H = 6, 8, 2, 32
    logits, y, g = randn(T, E, seed=1), randn(T * k, H, seed=2), randn(T, H, seed=3)
    w, e = b2x.moe_route(logits, k)
    _, _, plan = b2x.moe_dispatch(randn(T, H, seed=4), e, E)
    dy, dw = b2x.moe_combine_backward(g, y, plan.rows, w)
    dl = b2x.moe_route_backward(dw, logits, e)

    def f(z):
        ww = torch.softmax(z, 1).gather(1, e.long())
        ww = ww / ww.sum(1, keepdim=True)
        return ((y.to(D)[plan.rows.long()] * ww[:, :, None]).sum(1) * g.to(D)).sum(1)

    for i in range(E):
        h = torch.zeros((T, E), dtype=D, device="cuda")
        h[:, i] = 1e-5
        ref = (f(logits.to(D) + h) - f(logits.to(D) - h)) / 2e-5
        check(dl[:, i], ref, 1e-5 * dw.to(D).abs().sum(1) + 1e-7)
    # the gather's gradient: every row counted once
    rows = randn(T * k, H, seed=5)
    dx = b2x.moe_combine(rows, plan.rows)
    check(dx, rows.to(D)[plan.rows.long()].sum(1), 1e-5)
