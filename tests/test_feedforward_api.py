"""CPU tests of the feed-forward operators' boundary: ctypes structs match the header, the C ABI refuses bad arguments
with a status and a message before touching a GPU, and the Python calls refuse what they do not take.  No kernel is
launched here."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # a 16-byte aligned stand-in for a device pointer: nothing reads it


def _L():
    from b2x import _lib as L
    return L


def refused(name, status, *args):
    L = _L()
    st = getattr(L.lib(), name)(*args, None)
    assert st == getattr(L, status), (st, L.lib().b2x_last_error())
    assert L.lib().b2x_last_error()


def test_struct_layouts_match_header(tmp_path):
    L = _L()
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    names = {"b2x_epilogue": L.Epilogue, "b2x_moe_route_args": L.MoeRouteArgs, "b2x_moe_dispatch_args": L.MoeDispatchArgs,
             "b2x_moe_gemm_args": L.MoeGemmArgs}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "p.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "b2x.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    exe = str(tmp_path / "p")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for py in names.values():
        want.append(ctypes.sizeof(py))
        want += [getattr(py, f).offset for f, _ in py._fields_]
    assert got == want


def gemm(**kw):
    L = _L()
    g = L.GemmArgs()
    g.a, g.b, g.c = P, 2 * P, 3 * P
    g.M, g.N, g.K = 64, 256, 256
    g.lda, g.ldb_k, g.ldb_n, g.ldc = 256, 1, 256, 256
    g.a_type = g.b_type = L.E4M3
    g.c_type = L.BF16
    for k, v in kw.items():
        setattr(g, k, v)
    return ctypes.byref(g)


def epi(**kw):
    e = _L().Epilogue()
    for k, v in kw.items():
        setattr(e, k, v)
    return ctypes.byref(e)


@pytest.mark.parametrize("g,e,status", [
    (dict(a_type=1), {}, "ERR_UNSUPPORTED"),
    (dict(c_type=0), {}, "ERR_UNSUPPORTED"),
    (dict(K=0), {}, "ERR_UNSUPPORTED"),
    (dict(M=-1), {}, "ERR_INVALID_ARG"),
    (dict(M=1 << 31), {}, "ERR_UNSUPPORTED"),
    (dict(a=0), {}, "ERR_INVALID_ARG"),
    (dict(a=P + 8), {}, "ERR_INVALID_ARG"),
    (dict(lda=200), {}, "ERR_INVALID_ARG"),
    (dict(lda=264), {}, "ERR_INVALID_ARG"),
    (dict(ldb_k=2), {}, "ERR_INVALID_ARG"),
    (dict(ldb_n=264), {}, "ERR_INVALID_ARG"),
    (dict(ldc=255), {}, "ERR_INVALID_ARG"),
    (dict(scale_mode=1), {}, "ERR_INVALID_ARG"),
    (dict(scale_mode=3, scale_a=P, scale_b=P), {}, "ERR_UNSUPPORTED"),
    ({}, dict(activation=9), "ERR_INVALID_ARG"),
    ({}, dict(bias=P, bias_type=3), "ERR_UNSUPPORTED"),
    ({}, dict(residual=P, ld_residual=10), "ERR_INVALID_ARG"),
    ({}, dict(pre=P, ld_pre=10), "ERR_INVALID_ARG"),
])
def test_gemm_epilogue_refuses(g, e, status):
    refused("b2x_fp8_gemm_epilogue", status, gemm(**g), epi(**e))


def test_null_arguments():
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", None, epi())
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", gemm(), None)
    for name, more in (("b2x_moe_route", ()), ("b2x_moe_dispatch", ()), ("b2x_moe_gemm", (P, 1, 8)),
                       ("b2x_moe_gemm_swiglu", (P, 3, 128, P, None)), ("b2x_moe_route_backward", (P, P, 8))):
        refused(name, "ERR_INVALID_ARG", None, *more)


def route(**kw):
    L = _L()
    a = L.MoeRouteArgs()
    a.logits, a.logits_type, a.tokens, a.experts, a.ld_logits = P, L.F32, 4, 64, 64
    a.top_k, a.num_groups, a.top_groups, a.scale, a.weights, a.indices = 8, 1, 1, 1.0, P, P
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,status", [
    (dict(logits_type=3), "ERR_UNSUPPORTED"), (dict(tokens=-1), "ERR_INVALID_ARG"), (dict(experts=0), "ERR_INVALID_ARG"),
    (dict(ld_logits=63), "ERR_INVALID_ARG"), (dict(experts=1025, ld_logits=1025), "ERR_UNSUPPORTED"), (dict(top_k=0), "ERR_INVALID_ARG"),
    (dict(top_k=33), "ERR_UNSUPPORTED"), (dict(experts=4, top_k=5), "ERR_INVALID_ARG"), (dict(num_groups=5), "ERR_INVALID_ARG"),
    (dict(num_groups=8, top_groups=9), "ERR_INVALID_ARG"), (dict(num_groups=8, top_groups=0), "ERR_INVALID_ARG"),
    (dict(logits=0), "ERR_INVALID_ARG"), (dict(weights=0), "ERR_INVALID_ARG"), (dict(indices=0), "ERR_INVALID_ARG")])
def test_route_refuses(kw, status):
    refused("b2x_moe_route", status, route(**kw))


def test_route_backward_refuses():
    refused("b2x_moe_route_backward", "ERR_INVALID_ARG", route(), P, P, 63)
    refused("b2x_moe_route_backward", "ERR_INVALID_ARG", route(), None, P, 64)
    refused("b2x_moe_route_backward", "ERR_INVALID_ARG", route(indices=0), P, P, 64)


def dispatch(**kw):
    L = _L()
    a = L.MoeDispatchArgs()
    a.x, a.x_type, a.tokens, a.cols, a.ld_x, a.indices, a.top_k, a.experts = P, L.BF16, 4, 64, 64, P, 2, 8
    a.q, a.q_type, a.ld_q, a.scale, a.offsets, a.rows = P, L.E4M3, 64, P, P, P
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,status", [
    (dict(x_type=2), "ERR_UNSUPPORTED"), (dict(q_type=1), "ERR_UNSUPPORTED"), (dict(ld_x=63), "ERR_INVALID_ARG"),
    (dict(ld_q=63), "ERR_INVALID_ARG"), (dict(top_k=0), "ERR_INVALID_ARG"), (dict(experts=0), "ERR_INVALID_ARG"),
    (dict(experts=1025), "ERR_UNSUPPORTED"), (dict(tokens=1 << 30, top_k=2), "ERR_UNSUPPORTED"), (dict(offsets=0), "ERR_INVALID_ARG"),
    (dict(rows=0), "ERR_INVALID_ARG"), (dict(scale=0), "ERR_INVALID_ARG"), (dict(q=0), "ERR_INVALID_ARG")])
def test_dispatch_refuses(kw, status):
    refused("b2x_moe_dispatch", status, dispatch(**kw))


def experts(**kw):
    L = _L()
    a = L.MoeGemmArgs()
    a.x, a.x_type, a.rows, a.K, a.ld_x = P, L.E4M3, 16, 256, 256
    a.w, a.w_type, a.experts, a.N, a.ldw_e, a.ldw_n, a.ldw_k, a.offsets = P, L.E4M3, 4, 256, 256 * 256, 256, 1, P
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,status", [
    (dict(x_type=1), "ERR_UNSUPPORTED"), (dict(rows=-1), "ERR_INVALID_ARG"), (dict(experts=0), "ERR_INVALID_ARG"),
    (dict(experts=1025), "ERR_UNSUPPORTED"), (dict(K=0), "ERR_UNSUPPORTED"), (dict(offsets=0), "ERR_INVALID_ARG"),
    (dict(ld_x=255), "ERR_INVALID_ARG"), (dict(ld_x=264), "ERR_INVALID_ARG"), (dict(x=P + 1), "ERR_INVALID_ARG"),
    (dict(ldw_n=255), "ERR_INVALID_ARG"), (dict(ldw_n=264), "ERR_INVALID_ARG"), (dict(ldw_e=100), "ERR_INVALID_ARG"),
    (dict(ldw_k=2), "ERR_INVALID_ARG"), (dict(scale_x=P, scale_x_count=3), "ERR_INVALID_ARG"),
    (dict(scale_w=P, scale_w_count=3), "ERR_INVALID_ARG")])
def test_moe_gemm_refuses(kw, status):
    refused("b2x_moe_gemm", status, experts(**kw), P, 1, 256)
    refused("b2x_moe_gemm_swiglu", status, experts(**kw), P, 3, 128, P, None)


def test_moe_gemm_refuses_outputs():
    refused("b2x_moe_gemm", "ERR_UNSUPPORTED", experts(), P, 0, 256)
    refused("b2x_moe_gemm_swiglu", "ERR_UNSUPPORTED", experts(), P, 1, 128, P, None)
    refused("b2x_moe_gemm_swiglu", "ERR_UNSUPPORTED", experts(N=128, ldw_e=128 * 256), P, 3, 128, P, None)
    refused("b2x_moe_gemm_swiglu", "ERR_UNSUPPORTED", experts(ldw_e=256 * 256 + 16), P, 3, 128, P, None)
    refused("b2x_moe_gemm_swiglu", "ERR_UNSUPPORTED", experts(ldw_n=1, ldw_k=256), P, 3, 128, P, None)


def test_combine_and_backward_refuse():
    ok = [P, 8, 64, P, P, 4, 2, 64, None, 0, P, 64, 1]
    for at, v, status in ((12, 3, "ERR_UNSUPPORTED"), (2, 63, "ERR_INVALID_ARG"), (6, 0, "ERR_INVALID_ARG"), (3, None, "ERR_INVALID_ARG"),
                          (0, None, "ERR_INVALID_ARG"), (10, None, "ERR_INVALID_ARG"), (11, 63, "ERR_INVALID_ARG"), (5, -1, "ERR_INVALID_ARG")):
        refused("b2x_moe_combine", status, *[v if i == at else a for i, a in enumerate(ok)])
    ok = [P, 64, P, 8, 64, P, P, 4, 2, 64, P, 64, P, 1]
    for at, v, status in ((13, 4, "ERR_UNSUPPORTED"), (1, 63, "ERR_INVALID_ARG"), (6, None, "ERR_INVALID_ARG"), (12, None, "ERR_INVALID_ARG"),
                          (8, 0, "ERR_INVALID_ARG"), (11, 63, "ERR_INVALID_ARG")):
        refused("b2x_moe_combine_backward", status, *[v if i == at else a for i, a in enumerate(ok)])
    ok = [P, 64, P, 64, P, 64, P, 1, 4, 64, 0]
    for at, v, status in ((7, 5, "ERR_UNSUPPORTED"), (10, 5, "ERR_INVALID_ARG"), (1, 63, "ERR_INVALID_ARG"), (0, None, "ERR_INVALID_ARG"),
                          (8, -1, "ERR_INVALID_ARG")):
        refused("b2x_epilogue_backward", status, *[v if i == at else a for i, a in enumerate(ok)])


def test_pad_rows_refuses():
    for args, status in (((P, 10, -1, 10, P, 16), "ERR_INVALID_ARG"), ((P, 9, 4, 10, P, 16), "ERR_INVALID_ARG"),
                         ((P, 10, 4, 10, P + 8, 16), "ERR_INVALID_ARG"), ((P, 10, 4, 10, P, 24), "ERR_INVALID_ARG"),
                         ((None, 10, 4, 10, P, 16), "ERR_INVALID_ARG"), ((P, 20, 4, 20, P, 16), "ERR_INVALID_ARG"),
                         ((P, 16, 1 << 40, 16, P, 16), "ERR_UNSUPPORTED")):
        refused("b2x_pad_rows", status, *args)


def test_python_calls_refuse_cpu_tensors():
    import b2x
    f8 = torch.zeros((4, 128)).to(torch.float8_e4m3fn)
    w = torch.zeros((2, 256, 128)).to(torch.float8_e4m3fn)
    off, one = torch.zeros(3, dtype=torch.int32), torch.ones(1)
    x, i = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)
    for f in (lambda: b2x.gemm_epilogue(f8, f8.t()), lambda: b2x.epilogue_backward(x, x), lambda: b2x.moe_route(x, 2),
              lambda: b2x.moe_route_backward(x[:, :2], x, i), lambda: b2x.moe_dispatch(x, i, 2), lambda: b2x.moe_gemm(f8, w, off),
              lambda: b2x.moe_gemm_swiglu(f8, w, off, one), lambda: b2x.moe_combine(x, i), lambda: b2x.moe_combine_backward(x, x, i, x[:, :2])):
        with pytest.raises(ValueError, match="CUDA tensors only"):
            f()


@pytest.mark.gpu
def test_python_calls_refuse_bad_arguments():
    import b2x
    c = "cuda"
    a, b = torch.zeros((4, 128), device=c).to(torch.float8_e4m3fn), torch.zeros((128, 64), device=c).to(torch.float8_e4m3fn)
    x, i = torch.zeros((4, 8), device=c), torch.zeros((4, 2), dtype=torch.int32, device=c)
    w, off = torch.zeros((2, 256, 128), device=c).to(torch.float8_e4m3fn), torch.zeros(3, dtype=torch.int32, device=c)
    one = torch.ones(1, device=c)
    bf = torch.bfloat16
    bad = [
        lambda: b2x.gemm_epilogue(x, b), lambda: b2x.gemm_epilogue(a, b[:64]), lambda: b2x.gemm_epilogue(a, b, activation="tanh"),
        lambda: b2x.gemm_epilogue(a, b, scale_a=one), lambda: b2x.gemm_epilogue(a, b, bias=torch.zeros(63, device=c)),
        lambda: b2x.gemm_epilogue(a, b, bias=torch.zeros(64, device=c, dtype=torch.int32)),
        lambda: b2x.gemm_epilogue(a, b, residual=torch.zeros((4, 64), device=c)), lambda: b2x.gemm_epilogue(a, b, out_dtype=torch.float32),
        lambda: b2x.gemm_epilogue(a, b, residual=torch.zeros((3, 64), device=c, dtype=bf)), lambda: b2x.gemm_epilogue(a, b.cpu()),
        lambda: b2x.gemm_epilogue(a, b, scale_a=torch.ones(2, device=c), scale_b=one), lambda: b2x.gemm_epilogue(a[:, :0], b[:0]),
        lambda: b2x.epilogue_backward(x, x.to(bf)), lambda: b2x.epilogue_backward(x, x[:3]), lambda: b2x.epilogue_backward(x, x, "tanh"),
        lambda: b2x.moe_route(x, 9), lambda: b2x.moe_route(x, 0), lambda: b2x.moe_route(x, 2, score="relu"),
        lambda: b2x.moe_route(x, 2, num_groups=3), lambda: b2x.moe_route(x, 2, bias=torch.zeros(7, device=c)),
        lambda: b2x.moe_route(x, 2, num_groups=2, group_score="sum"), lambda: b2x.moe_route(x[0], 2), lambda: b2x.moe_route(i, 1),
        lambda: b2x.moe_route_backward(x[:, :3], x, i), lambda: b2x.moe_route_backward(x[:, :2], x, i.float()),
        lambda: b2x.moe_dispatch(x.half(), i, 2), lambda: b2x.moe_dispatch(x, i[:3], 2), lambda: b2x.moe_dispatch(x, i, 0),
        lambda: b2x.moe_dispatch(x, i, 2, dtype=bf), lambda: b2x.moe_dispatch(x, i, 2, scale=torch.ones(2, device=c)),
        lambda: b2x.moe_dispatch(x, i, 2, out=x), lambda: b2x.moe_dispatch(x, i.float(), 2),
        lambda: b2x.moe_gemm(a, w[0], off), lambda: b2x.moe_gemm(a, w, off[:2]), lambda: b2x.moe_gemm(a, w[:, :, :64], off),
        lambda: b2x.moe_gemm(a, w, off, scale_x=torch.ones(3, device=c)), lambda: b2x.moe_gemm(a, w, off, out=x),
        lambda: b2x.moe_gemm(a, w, off, out_dtype=torch.float32), lambda: b2x.moe_gemm(a, w, off.float()),
        lambda: b2x.moe_gemm_swiglu(a, w[:, :128], off, one), lambda: b2x.moe_gemm_swiglu(a, w, off, torch.ones(2, device=c)),
        lambda: b2x.moe_gemm_swiglu(a, w, off, one, h_dtype=bf), lambda: b2x.moe_gemm_swiglu(a, w, off, one, h_amax=one.double()),
        lambda: b2x.moe_combine(x, i, x), lambda: b2x.moe_combine(x, i, residual=x[:3]), lambda: b2x.moe_combine(i, i),
        lambda: b2x.moe_combine(x, i[0]), lambda: b2x.moe_combine_backward(x[:3], x, i, x[:, :2]),
        lambda: b2x.moe_combine_backward(x.to(bf), x, i, x[:, :2]),
    ]
    for n, f in enumerate(bad):
        with pytest.raises((ValueError, TypeError, b2x.B2XError)):
            f()
            print("not refused:", n)
    torch.cuda.synchronize()


def test_indices_past_int32_do_not_wrap():
    """An int64 index outside int32 stays out of range (dropped) instead of becoming another one."""
    from b2x.feedforward import _ints
    t = torch.tensor([[1 << 32, 3], [-(1 << 32) + 1, (1 << 31) + 2], [-1, 0]])
    assert _ints(t, "experts").tolist() == [[(1 << 31) - 1, 3], [-1, (1 << 31) - 1], [-1, 0]]


def test_values_off_their_own_grid_are_refused():
    """A pointer that is no multiple of its element's size would be a misaligned access."""
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", gemm(), epi(residual=P + 1, ld_residual=256))
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", gemm(), epi(pre=P + 1, ld_pre=256))
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", gemm(), epi(bias=P + 2, bias_type=0))
    refused("b2x_fp8_gemm_epilogue", "ERR_INVALID_ARG", gemm(), epi(bias=P + 1, bias_type=1))
    refused("b2x_moe_route", "ERR_INVALID_ARG", route(logits=P + 2))
    refused("b2x_moe_dispatch", "ERR_INVALID_ARG", dispatch(x=P + 1))
    ok = [P, 8, 64, P, P, 4, 2, 64, P, 64, P, 64, 0]
    for at in (0, 8, 10):
        refused("b2x_moe_combine", "ERR_INVALID_ARG", *[P + 2 if i == at else a for i, a in enumerate(ok)])
    ok = [P, 64, P, 8, 64, P, P, 4, 2, 64, P, 64, P, 0]
    for at in (0, 2, 10):
        refused("b2x_moe_combine_backward", "ERR_INVALID_ARG", *[P + 2 if i == at else a for i, a in enumerate(ok)])
    ok = [P, 64, P, 64, P, 64, P, 0, 4, 64, 0]
    for at in (0, 2, 4):
        refused("b2x_epilogue_backward", "ERR_INVALID_ARG", *[P + 2 if i == at else a for i, a in enumerate(ok)])


def test_counts_past_32_bits_are_refused():
    """num_groups = 2^32 + 1 would reach the C ABI as 1."""
    from b2x.feedforward import _count
    for v in (1 << 31, (1 << 32) + 1, -(1 << 31) - 1):
        with pytest.raises(ValueError, match="32 bits"):
            _count(v, "num_groups")
    assert _count(8, "num_groups") == 8 and _count(-1, "top_k") == -1


@pytest.mark.gpu
def test_route_refuses_counts_past_32_bits():
    import b2x
    x = torch.zeros((4, 8), device="cuda")
    for kw in (dict(top_k=(1 << 32) + 2), dict(top_k=2, num_groups=(1 << 32) + 1), dict(top_k=2, num_groups=2, top_groups=(1 << 32) + 1)):
        with pytest.raises(ValueError, match="32 bits"):
            b2x.moe_route(x, **kw)
