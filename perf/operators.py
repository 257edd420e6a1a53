"""Cases of the feed-forward operators: the dense fp8 product with its epilogue, and the mixture-of-experts operators
(routing, dispatch, the experts' products, combine), each with its plain form in elementary torch operations.

Sizes are those of this repository's own benchmark: 8192 and 28672 are its dense layers', 7168 (hidden) and 4096 (gate and up
of 2048) those of its grouped expert products. The rest is generic."""
import sys

import torch

own = False

FMAX = 448.0  # largest finite float8_e4m3fn
FLOATS = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SQRT_HALF = 0.7071067811865476
GELU_A, GELU_B = 0.7978845608028654, 0.044715  # sqrt(2 / pi) and the cubic term of the tanh form


def listed():
    return [
        # One token through a row-parallel output projection: all of it is reading the weights.
        {"name": "linear one token", "op": "linear", "M": 1, "N": 8192, "K": 28672, "act": "none", "bias": "bf16",
         "residual": True, "pre": False, "out": "bf16", "layout": "nk"},
        # A prefill or training batch of ragged length through the first layer of a feed-forward block; the pre-activation
        # is kept for the backward pass.
        {"name": "linear batch", "op": "linear", "M": 4000, "N": 28672, "K": 8192, "act": "gelu_tanh", "bias": "fp32",
         "residual": False, "pre": True, "out": "bf16", "layout": "nk"},
        # The backward pass of that layer's epilogue.
        {"name": "linear gradient", "op": "linear_grad", "M": 4000, "N": 28672, "act": "gelu_tanh", "out": "bf16"},
        # Routing of a decode step: a handful of tokens, latency counts.
        {"name": "route decode", "op": "route", "T": 8, "E": 128, "k": 8, "score": "softmax", "bias": False, "groups": 1,
         "top_groups": 1, "group_score": "max", "renorm": True, "logits": "bf16", "masked": 0},
        # Routing of a prefill or training batch, with a balancing bias and groups of experts.
        {"name": "route batch", "op": "route", "T": 16384, "E": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "top_groups": 4, "group_score": "top2", "renorm": True, "logits": "fp32", "masked": 0},
        # The gradient of a softmax router's logits in training.
        {"name": "route gradient", "op": "route_grad", "T": 16384, "E": 128, "k": 8, "score": "softmax", "renorm": False,
         "logits": "bf16", "masked": 0},
        # Dispatch of a decode step.
        {"name": "dispatch decode", "op": "dispatch", "T": 16, "H": 7168, "E": 64, "k": 8, "x": "bf16"},
        # Dispatch of a batch whose length is odd.
        {"name": "dispatch batch", "op": "dispatch", "T": 8191, "H": 7168, "E": 64, "k": 8, "x": "bf16"},
        # Down projections of a decode step: about half of the experts get a row or two.
        {"name": "experts decode", "op": "experts", "rows": 40, "E": 64, "N": 7168, "K": 2048, "swiglu": False, "out": "bf16"},
        # Gate and up projections of a batch, unevenly spread over the experts, with SwiGLU and fp8 in the epilogue.
        {"name": "experts batch swiglu", "op": "experts", "rows": 20001, "E": 32, "N": 4096, "K": 7168, "swiglu": True, "out": "fp8"},
        # Weighted sum of the experts' outputs of a batch, onto the residual stream.
        {"name": "combine batch", "op": "combine", "T": 8191, "H": 7168, "k": 8, "y": "bf16", "residual": True},
        # Its backward pass.
        {"name": "combine gradient", "op": "combine_grad", "T": 4095, "H": 7168, "k": 8, "y": "bf16"},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], evenly spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "route", "route", "route_grad", "dispatch", "experts", "experts",
                     "combine", "combine_grad"])
    if op == "linear":
        return {"op": op, "M": _log(rng, 1, 4096), "N": _log(rng, 64, 16384), "K": _log(rng, 128, 8192),
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.choice(["none", "fp32", "bf16"]),
                "residual": rng.random() < 0.5, "pre": rng.random() < 0.3, "out": rng.choice(["bf16", "bf16", "fp16"]),
                "layout": rng.choice(["nk", "nk", "kn"])}
    if op == "linear_grad":
        return {"op": op, "M": _log(rng, 1, 8192), "N": _log(rng, 64, 12288),
                "act": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "out": rng.choice(["bf16", "fp16"])}
    if op in ("route", "route_grad"):
        E = rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 256, 384])
        c = {"op": op, "T": _log(rng, 1, 16384), "E": E, "k": rng.randint(1, min(8, E // 4)),
             "score": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.6,
             "logits": rng.choice(["fp32", "bf16"]), "masked": rng.choice([0, 0, E // 8])}
        if op == "route":
            groups = rng.choice([1, 1, 4, 8]) if E % 8 == 0 and E >= 64 else 1
            c.update(bias=rng.random() < 0.5, groups=groups, top_groups=groups // 2 or 1, group_score=rng.choice(["max", "top2"]))
        return c
    if op == "dispatch":
        return {"op": op, "T": _log(rng, 1, 8192), "H": _log(rng, 256, 8192), "E": rng.choice([8, 16, 64, 128, 256]),
                "k": rng.randint(1, 8), "x": rng.choice(["bf16", "fp32"])}
    if op == "experts":
        swiglu = rng.random() < 0.5
        return {"op": op, "rows": _log(rng, 1, 16384), "E": rng.choice([4, 8, 16, 32, 64]),
                "N": 256 * _log(rng, 1, 16) if swiglu else _log(rng, 128, 4096), "K": 16 * _log(rng, 16, 256),
                "swiglu": swiglu, "out": "fp8" if swiglu else rng.choice(["bf16", "fp16"])}
    return {"op": op, "T": _log(rng, 1, 8192), "H": _log(rng, 256, 7168), "k": rng.randint(1, 8), "y": "bf16",
            **({"residual": rng.random() < 0.5} if op == "combine" else {})}


# ---------------------------------------------------------------------------------------------------------------- inputs


def _fp8(shape, gen, std=96.0):
    """Normal values as a per-tensor quantization leaves them: the largest of some millions near 448."""
    q = torch.empty(shape, dtype=torch.float8_e4m3fn, device="cuda")
    flat = q.view(-1)
    step = 1 << 26
    for i in range(0, flat.numel(), step):
        n = min(step, flat.numel() - i)
        flat[i:i + n] = (torch.randn(n, device="cuda", generator=gen) * std).clamp_(-FMAX, FMAX).to(torch.float8_e4m3fn)
    return q


def _choices(T, E, k, gen):
    """k different experts for each token, some experts more popular than others."""
    popular = torch.randn(E, device="cuda", generator=gen) * 0.5
    noise = torch.rand((T, E), device="cuda", generator=gen).clamp_min_(1e-9).log_().neg_().log_().neg_()
    return torch.sort(popular + noise, dim=1, descending=True)[1][:, :k].to(torch.int32).contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)

    def randn(*shape, dtype=torch.float32, std=1.0):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)

    s, op = {"case": case}, case["op"]
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        s["a"] = _fp8((M, K), g)
        s["b"] = _fp8((N, K), g).t() if case["layout"] == "nk" else _fp8((K, N), g)
        s["scale_a"] = torch.full((1,), 1 / 96.0, device="cuda")
        s["scale_b"] = torch.full((1,), K ** -0.5 / 96.0, device="cuda")
        s["bias"] = None if case["bias"] == "none" else randn(N, dtype=FLOATS[case["bias"]], std=0.5)
        s["residual"] = randn(M, N, dtype=FLOATS[case["out"]]) if case["residual"] else None
    elif op == "linear_grad":
        s["grad"] = randn(case["M"], case["N"], dtype=FLOATS[case["out"]])
        s["pre"] = randn(case["M"], case["N"], dtype=FLOATS[case["out"]], std=1.2)
    elif op in ("route", "route_grad"):
        T, E = case["T"], case["E"]
        s["logits"] = randn(T, E, std=1.5).to(FLOATS[case["logits"]])
        if case["masked"]:  # experts that are out of service
            s["logits"][:, torch.randperm(E, device="cuda", generator=g)[:case["masked"]]] = float("-inf")
        if op == "route":
            s["bias"] = randn(E, std=0.05) if case["bias"] else None
        else:
            s["experts"] = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)[1][:, :case["k"]].to(torch.int32).contiguous()
            s["grad"] = randn(T, case["k"])
    elif op == "dispatch":
        s["x"] = randn(case["T"], case["H"], dtype=FLOATS[case["x"]])
        s["experts"] = _choices(case["T"], case["E"], min(case["k"], case["E"]), g)
    elif op == "experts":
        E, R, N, K = case["E"], case["rows"], case["N"], case["K"]
        share = torch.softmax(torch.randn(E, device="cuda", generator=g) * 0.5, 0)
        of = torch.multinomial(share, R, replacement=True, generator=g)
        count = torch.bincount(of, minlength=E)
        s["offsets"] = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), count.cumsum(0)]).to(torch.int32)
        s["most"] = int(count.max())  # used by the plain form alone
        s["x"] = _fp8((R, K), g)
        s["scale_x"] = torch.rand(R, device="cuda", generator=g) * 0.01 + 0.005
        s["w"] = _fp8((E, N, K), g)
        s["scale_w"] = (torch.rand(E, device="cuda", generator=g) * 0.01 + 0.005) * K ** -0.5
        s["h_scale"] = torch.full((1,), 0.02, device="cuda")
    else:
        T, H, k = case["T"], case["H"], case["k"]
        s["y"] = randn(T * k, H, dtype=FLOATS[case["y"]])
        s["weights"] = torch.softmax(randn(T, k), 1)
        # rows as a dispatch to 64 experts leaves them: sorted by expert, by token inside one
        of = torch.randint(0, 64, (T * k,), device="cuda", generator=g)
        order = torch.sort(of, stable=True)[1]
        rows = torch.empty(T * k, device="cuda", dtype=torch.int32)
        rows[order] = torch.arange(T * k, device="cuda", dtype=torch.int32)
        s["rows"] = rows.view(T, k)
        if op == "combine":
            s["residual"] = randn(T, H, dtype=FLOATS[case["y"]]) if case["residual"] else None
        else:
            s["grad"] = randn(T, H, dtype=FLOATS[case["y"]])
    return s


# ---------------------------------------------------------------------------------------------------------------- plain forms


def _act(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "gelu":
        return 0.5 * x * torch.erfc(x * -SQRT_HALF)
    if name == "gelu_tanh":
        return x * torch.sigmoid(2 * GELU_A * (x + GELU_B * x * x * x))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def _slope(x, name):
    """Derivative of _act at x."""
    if name == "relu":
        return (x > 0).to(x.dtype)
    if name == "gelu":
        return 0.5 * torch.erfc(x * -SQRT_HALF) + x * torch.exp(-0.5 * x * x) * (GELU_A / 2)
    if name == "gelu_tanh":
        p = torch.sigmoid(2 * GELU_A * (x + GELU_B * x * x * x))
        return p + x * p * (1 - p) * (2 * GELU_A * (1 + 3 * GELU_B * x * x))
    if name == "silu":
        p = torch.sigmoid(x)
        return p + x * p * (1 - p)
    return torch.ones_like(x)


def _linear(s):
    c = s["case"]
    pre = (s["a"].float() @ s["b"].float()) * (s["scale_a"] * s["scale_b"])
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    y = _act(pre, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"out": y.to(FLOATS[c["out"]])}
    if c["pre"]:
        out["pre"] = pre.to(FLOATS[c["out"]])
    return out


def _linear_grad(s):
    d = s["grad"].float() * _slope(s["pre"].float(), s["case"]["act"])
    return {"pre": d.to(s["grad"].dtype), "bias": d.sum(0, dtype=torch.float64).float()}


def _scores(l, kind):
    masked = l == float("-inf")
    if kind == "sigmoid":
        return torch.sigmoid(l), masked
    e = torch.exp(l - l.amax(1, keepdim=True))
    return e / e.sum(1, keepdim=True), masked


def _route(s):
    c = s["case"]
    l = s["logits"].double()  # choices next to a border
    score, masked = _scores(l, c["score"])
    choice = score if s["bias"] is None else score + s["bias"].double()
    choice = choice.masked_fill(masked, float("-inf"))
    T, E = l.shape
    if c["groups"] > 1:
        g = choice.view(T, c["groups"], -1)
        if c["group_score"] == "max":
            of = g.amax(2)
        else:
            best = torch.sort(g, dim=2, descending=True)[0][:, :, :2]
            of = best.masked_fill(best == float("-inf"), 0).sum(2).masked_fill(best[:, :, 0] == float("-inf"), float("-inf"))
        rank = torch.sort(of, dim=1, descending=True, stable=True)[1][:, :c["top_groups"]]
        kept = torch.zeros_like(of, dtype=torch.bool).scatter_(1, rank, True)
        choice = choice.masked_fill(~kept.repeat_interleave(E // c["groups"], 1), float("-inf"))
    best, at = torch.sort(choice, dim=1, descending=True, stable=True)
    best, at = best[:, :c["k"]], at[:, :c["k"]]
    w = score.gather(1, at).masked_fill(best == float("-inf"), 0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    return {"weights": w.float(), "experts": at.masked_fill(best == float("-inf"), -1).to(torch.int32)}


def _route_grad(s):
    c = s["case"]
    l, at, d = s["logits"].float(), s["experts"].long(), s["grad"]
    score, _ = _scores(l, c["score"])
    w = score.gather(1, at)
    if c["renorm"]:
        total = w.sum(1, keepdim=True)
        d = (d - (d * w).sum(1, keepdim=True) / total) / total
    ds = torch.zeros_like(l).scatter_(1, at, d)
    if c["score"] == "sigmoid":
        out = ds * score * (1 - score)
    else:
        out = score * (ds - (ds * score).sum(1, keepdim=True))
    return {"logits": out.to(s["logits"].dtype)}


def _dispatch(s):
    x, experts, E = s["x"].float(), s["experts"], s["case"]["E"]
    T, k = experts.shape
    flat = experts.reshape(-1).long()
    order = torch.sort(flat, stable=True)[1]
    count = torch.zeros(E + 1, device=x.device, dtype=torch.int64).index_add_(0, flat + 1, torch.ones_like(flat))
    rows = torch.empty_like(flat)
    rows[order] = torch.arange(T * k, device=x.device)
    scale = x.abs().amax(1) / FMAX
    inv = torch.where(scale == 0, torch.zeros_like(scale), 1 / scale)
    q = (x * inv[:, None]).clamp(-FMAX, FMAX).to(torch.float8_e4m3fn)
    token = order // k
    return {"q": q.view(torch.uint8)[token].view(torch.float8_e4m3fn), "scale": scale[token],
            "offsets": count.cumsum(0).to(torch.int32), "rows": rows.view(T, k).to(torch.int32)}


def _by_expert(x, offsets, most):
    """Rows in a padded [E, most, ...] tensor, and where each went."""
    E, R = offsets.numel() - 1, x.shape[0]
    r = torch.arange(R, device=x.device)
    e = torch.searchsorted(offsets[1:].long(), r, right=True)
    at = e * most + r - offsets[e].long()
    return torch.zeros((E * most, x.shape[1]), device=x.device, dtype=x.dtype).index_copy_(0, at, x).view(E, most, -1), e, at


def _experts(s):
    c = s["case"]
    x, e, at = _by_expert(s["x"].float(), s["offsets"], s["most"])
    y = torch.bmm(x, s["w"].float().transpose(1, 2)).view(-1, c["N"])[at]
    y = y * (s["scale_x"] * s["scale_w"][e])[:, None]
    if not c["swiglu"]:
        return {"out": y.to(FLOATS[c["out"]])}
    y = y.view(y.shape[0], -1, 2, 128)  # 128 gate columns, then their 128 up columns
    h = (y[:, :, 0] * torch.sigmoid(y[:, :, 0]) * y[:, :, 1]).reshape(y.shape[0], -1)
    return {"out": (h * (1 / s["h_scale"])).clamp(-FMAX, FMAX).to(torch.float8_e4m3fn)}


def _combine(s):
    out = (s["y"][s["rows"].long()].float() * s["weights"][:, :, None]).sum(1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(s["y"].dtype)}


def _combine_grad(s):
    rows, d = s["rows"].long(), s["grad"].float()
    dy = torch.empty_like(s["y"])
    dy[rows.view(-1)] = (d[:, None, :] * s["weights"][:, :, None]).to(dy.dtype).view(-1, dy.shape[1])
    return {"y": dy, "weights": (d[:, None, :] * s["y"][rows].float()).sum(2)}


PLAIN = {"linear": _linear, "linear_grad": _linear_grad, "route": _route, "route_grad": _route_grad, "dispatch": _dispatch,
         "experts": _experts, "combine": _combine, "combine_grad": _combine_grad}


# ---------------------------------------------------------------------------------------------------------------- the framework's calls


def _own(s):
    if "triton-ext_b200" not in sys.path:
        sys.path.insert(0, "triton-ext_b200")
    import b2x

    c = s["case"]
    op = c["op"]
    if op == "linear":
        r = b2x.gemm_epilogue(s["a"], s["b"], scale_a=s["scale_a"], scale_b=s["scale_b"], bias=s["bias"], activation=c["act"],
                              residual=s["residual"], out_dtype=FLOATS[c["out"]], return_pre=c["pre"])
        return {"out": r[0], "pre": r[1]} if c["pre"] else {"out": r}
    if op == "linear_grad":
        d, bias = b2x.epilogue_backward(s["grad"], s["pre"], c["act"])
        return {"pre": d, "bias": bias}
    if op == "route":
        w, e = b2x.moe_route(s["logits"], c["k"], score=c["score"], bias=s["bias"], num_groups=c["groups"], top_groups=c["top_groups"],
                             group_score=c["group_score"], renormalize=c["renorm"])
        return {"weights": w, "experts": e}
    if op == "route_grad":
        return {"logits": b2x.moe_route_backward(s["grad"], s["logits"], s["experts"], score=c["score"], renormalize=c["renorm"])}
    if op == "dispatch":
        q, scale, plan = b2x.moe_dispatch(s["x"], s["experts"], c["E"])
        return {"q": q, "scale": scale, "offsets": plan.offsets, "rows": plan.rows}
    if op == "experts":
        if c["swiglu"]:
            return {"out": b2x.moe_gemm_swiglu(s["x"], s["w"], s["offsets"], s["h_scale"], scale_x=s["scale_x"], scale_w=s["scale_w"])}
        return {"out": b2x.moe_gemm(s["x"], s["w"], s["offsets"], scale_x=s["scale_x"], scale_w=s["scale_w"], out_dtype=FLOATS[c["out"]])}
    if op == "combine":
        return {"out": b2x.moe_combine(s["y"], s["rows"], s["weights"], residual=s["residual"])}
    dy, dw = b2x.moe_combine_backward(s["grad"], s["y"], s["rows"], s["weights"])
    return {"y": dy, "weights": dw}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- work


def work(case):
    c, op = case, case["op"]
    size = {"none": 0, "bf16": 2, "fp16": 2, "fp32": 4}
    if op == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": M * K + K * N + N * size[c["bias"]] + M * N * 2 * (1 + c["residual"] + c["pre"]), "flops": 2 * M * N * K}
    if op == "linear_grad":
        return {"bytes": 6 * c["M"] * c["N"] + 4 * c["N"], "flops": 12 * c["M"] * c["N"]}
    if op == "route":
        return {"bytes": c["T"] * (c["E"] * size[c["logits"]] + 8 * c["k"]) + 4 * c["E"] * c["bias"], "flops": 10 * c["T"] * c["E"]}
    if op == "route_grad":
        return {"bytes": c["T"] * (2 * c["E"] * size[c["logits"]] + 8 * c["k"]), "flops": 8 * c["T"] * c["E"]}
    if op == "dispatch":
        T, H, k = c["T"], c["H"], min(c["k"], c["E"])
        return {"bytes": T * H * size[c["x"]] + T * k * (H + 4 + 8) + 4 * c["E"], "flops": 3 * T * H}
    if op == "experts":
        R, E, N, K = c["rows"], c["E"], c["N"], c["K"]
        active = E * (1 - (1 - 1 / E) ** R)  # experts with a row, on average
        out = R * N // 2 if c["swiglu"] else 2 * R * N
        return {"bytes": active * N * K + R * (K + 4) + out, "flops": 2 * R * N * K}
    T, H, k = c["T"], c["H"], c["k"]
    if op == "combine":
        return {"bytes": 2 * T * H * (k + 1 + c["residual"]) + 8 * T * k, "flops": 2 * T * H * k}
    return {"bytes": 2 * T * H * (2 * k + 1) + 12 * T * k, "flops": 3 * T * H * k}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, D = case["op"], torch.float64
    if op == "linear":
        z = torch.mm(s["a"].to(D), s["b"].to(D)).mul_(s["scale_a"].to(D)).mul_(s["scale_b"].to(D))
        if s["bias"] is not None:
            z += s["bias"].to(D)
        out = {"out": _exact_act(z, case["act"])}
        if s["residual"] is not None:
            out["out"] = out["out"] + s["residual"].to(D)
        if case["pre"]:
            out["pre"] = z
        return out
    if op == "linear_grad":
        z = s["pre"].to(D).requires_grad_()
        _exact_act(z, case["act"]).backward(s["grad"].to(D))
        return {"pre": z.grad, "bias": z.grad.sum(0)}
    if op == "route":
        # the weights alone: equal choices are told apart by their number, which the comparison with the plain form holds
        z = s["logits"].to(D)
        p = 1 / (1 + torch.exp(-z)) if case["score"] == "sigmoid" else torch.softmax(z, 1)
        c = torch.where(torch.isinf(z), z, p if s["bias"] is None else p + s["bias"].to(D))
        if case["groups"] > 1:
            parts = c.unflatten(1, (case["groups"], -1))
            two = torch.topk(parts, 1 if case["group_score"] == "max" else 2, dim=2).values
            total = torch.where(torch.isinf(two), torch.zeros_like(two), two).sum(2)
            total = torch.where(torch.isinf(two[:, :, 0]), two[:, :, 0], total)
            top = torch.topk(total, case["top_groups"], dim=1).indices
            c = torch.full_like(parts, -torch.inf).scatter(1, top[:, :, None].expand(-1, -1, parts.shape[2]),
                                                           parts.gather(1, top[:, :, None].expand(-1, -1, parts.shape[2]))).flatten(1)
        c, at = torch.topk(c, case["k"], dim=1)
        w = torch.where(torch.isinf(c), torch.zeros_like(c), p.gather(1, at))
        return {"weights": w / w.sum(1, keepdim=True) if case["renorm"] else w, "experts": None}
    if op == "route_grad":
        z = s["logits"].to(D).requires_grad_()
        p = torch.sigmoid(z) if case["score"] == "sigmoid" else torch.softmax(z, 1)
        w = p.gather(1, s["experts"].long())
        (w / w.sum(1, keepdim=True) if case["renorm"] else w).backward(s["grad"].to(D))
        return {"logits": torch.nan_to_num(z.grad, nan=0.0)}
    if op == "dispatch":
        order = torch.argsort(s["experts"].flatten().long(), stable=True)
        x = s["x"].to(D)[torch.div(order, s["experts"].shape[1], rounding_mode="floor")]
        scale = x.abs().max(1).values / FMAX
        return {"q": x / scale[:, None], "scale": scale, "offsets": None, "rows": None}
    if op == "experts":
        start = s["offsets"].tolist()
        parts = []
        for i in range(case["E"]):
            x = s["x"][start[i]:start[i + 1]].to(D)
            y = x @ s["w"][i].to(D).t() * (s["scale_x"][start[i]:start[i + 1]].to(D) * s["scale_w"][i].to(D))[:, None]
            if case["swiglu"]:
                gate, up = y.unflatten(1, (-1, 256)).split(128, dim=2)
                y = ((gate / (1 + torch.exp(-gate)) * up).flatten(1) / s["h_scale"].to(D)).clamp(-FMAX, FMAX)
            parts.append(y)
        return {"out": torch.cat(parts)}
    T, k = s["rows"].shape
    y, w = s["y"].to(D), s["weights"].to(D)
    if op == "combine":
        out = torch.zeros((T, y.shape[1]), dtype=D, device=y.device) if s["residual"] is None else s["residual"].to(D)
        for j in range(k):
            out = out.addcmul(y.index_select(0, s["rows"][:, j].long()), w[:, j, None])
        return {"out": out}
    d, dy, dw = s["grad"].to(D), torch.zeros_like(y), torch.zeros_like(w)
    for j in range(k):
        r = s["rows"][:, j].long()
        dy.index_copy_(0, r, d * w[:, j, None])
        dw[:, j] = torch.linalg.vecdot(d, y.index_select(0, r))
    return {"y": dy, "weights": dw}


def _exact_act(z, name):
    if name == "relu":
        return torch.relu(z)
    if name == "gelu":
        return torch.nn.functional.gelu(z)
    if name == "gelu_tanh":
        return torch.nn.functional.gelu(z, approximate="tanh")
    if name == "silu":
        return torch.nn.functional.silu(z)
    return z
