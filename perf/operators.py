"""The operators of the quantised transformer block and the cases they are measured on.

``norm``   residual addition + root-mean-square norm, forward and backward (training)
``normq``  the same norm with an 8-bit output and its scales (serving)
``w4``     rows times 4-bit weights with group scales, rows of 16 bits or of 8 bits with scales

``own`` false: plain torch operations in 32 bits. ``own`` true: the package's operators.
"""
import math

import torch

own = False

EPS = 1e-6
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i8": torch.int8,
      "e4m3": torch.float8_e4m3fn}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "i8": 1, "e4m3": 1, "": 0}
QMAX = {"i8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # one token of a running generation: add + norm in front of a 16-bit layer; latency only
        dict(name="norm_token_f16", op="norm", rows=1, cols=2048, x="f16", res="f16", w="f16", back=False),
        # a training step's block input: 8192 tokens, 32-bit residual stream, 16-bit branch
        dict(name="norm_train_bf16_f32", op="norm", rows=8192, cols=4096, x="bf16", res="f32", w="f32", back=True),
        # ragged training batch of an odd width, everything in 16 bits
        dict(name="norm_train_ragged_f16", op="norm", rows=1003, cols=1111, x="f16", res="f16", w="f16", back=True),
        # one token, the 8-bit input of the following 4-bit layer, one scale
        dict(name="normq_token_i8", op="normq", rows=1, cols=8192, x="bf16", res="bf16", w="bf16", out="i8",
             scale="row", group=0),
        # a long prompt, 8-bit floats with a scale for every 128 columns
        dict(name="normq_prompt_e4m3", op="normq", rows=8192, cols=8192, x="bf16", res="bf16", w="bf16", out="e4m3",
             scale="group", group=128),
        # a batch of decoding requests, calibrated (given) scale, odd width, no residual
        dict(name="normq_batch_i8_static", op="normq", rows=250, cols=1301, x="f16", res="", w="f32", out="i8",
             scale="given", group=0),
        # one token through a square projection: the smallest product, launch and latency
        dict(name="w4_token_f16", op="w4", m=1, n=4096, k=4096, group=64, x="f16", out="f16", scale="", bias=False),
        # one token through the widest layer: weight streaming
        dict(name="w4_token_wide_bf16", op="w4", m=1, n=28672, k=8192, group=128, x="bf16", out="bf16", scale="",
             bias=False),
        # a few environments through a layer whose sizes fit no tile
        dict(name="w4_ragged_f16", op="w4", m=5, n=777, k=1002, group=64, x="f16", out="f16", scale="", bias=True),
        # a decoding batch on the norm's int8 rows, one scale a row
        dict(name="w4_batch_i8", op="w4", m=16, n=14336, k=4096, group=128, x="i8", out="bf16", scale="row",
             bias=False),
        # a larger decoding batch on 8-bit floats with a scale a group
        dict(name="w4_batch_e4m3", op="w4", m=64, n=4096, k=14336, group=128, x="e4m3", out="f16", scale="group",
             bias=True),
        # a short prompt: no longer bound by the weights
        dict(name="w4_prompt_f16", op="w4", m=1024, n=4096, k=4096, group=64, x="f16", out="f16", scale="",
             bias=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "normq", "w4", "w4"])
    if op in ("norm", "normq"):
        while True:
            rows, cols = _log(rng, 1, 16384), _log(rng, 32, 16384)
            if rng.random() < 0.6:
                cols = max(16, cols // 16 * 16)
            if rows * cols <= 8192 * 4096:
                break
        x = rng.choice(["f16", "bf16"] if op == "normq" else ["f16", "bf16", "bf16", "f32"])
        res = rng.choice([x, x, "f32", ""])
        w = rng.choice([x, "f32"])
        if op == "norm":
            return dict(op=op, rows=rows, cols=cols, x=x, res=res, w=w, back=rng.random() < 0.7)
        scale = rng.choice(["row", "group", "given"])
        return dict(op=op, rows=rows, cols=cols, x=x, res=res, w=w, out=rng.choice(["i8", "e4m3"]), scale=scale,
                    group=rng.choice([32, 64, 128]) if scale == "group" else 0)
    while True:
        m, n, k = _log(rng, 1, 1024), _log(rng, 16, 16384), 2 * _log(rng, 32, 8192)
        if rng.random() < 0.7:
            n, k = max(16, n // 16 * 16), max(64, k // 64 * 64)
        if m * n * k <= 1024 * 4096 * 4096 and n * k <= 28672 * 8192:
            break
    x = rng.choice(["f16", "bf16", "i8", "e4m3"])
    scale = rng.choice(["row", "group"]) if x in QMAX else ""
    return dict(op=op, m=m, n=n, k=k, group=rng.choice([32, 64, 128]), x=x,
                out=x if x in ("f16", "bf16") else rng.choice(["f16", "bf16"]), scale=scale, bias=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] in ("norm", "normq"):
        R, C = case["rows"], case["cols"]
        train = case.get("back", False)
        # the residual stream of a trained block has a few columns far larger than the others
        loud = 1.0 + 15.0 * (rand(C) < 0.01)
        s["x"] = randn(R, C).to(DT[case["x"]]).requires_grad_(train)
        s["res"] = (3.0 * randn(R, C) * loud).to(DT[case["res"]]).requires_grad_(train) if case["res"] else None
        s["w"] = (1.0 + 0.2 * randn(C)).to(DT[case["w"]]).requires_grad_(train)
        if train:
            s["dy"] = randn(R, C).to(DT[case["x"]])
            s["dh"] = randn(R, C).to(DT[case["res"]]) if case["res"] else None
        if case["op"] == "normq":
            s["given"] = None
            if case["scale"] == "given":
                s["given"] = (4.0 + rand(())) / QMAX[case["out"]]
            s["buf"] = torch.empty(R, C, dtype=DT[case["x"]], device="cuda")
        return s
    M, Nn, K, group = case["m"], case["n"], case["k"], case["group"]
    G = -(-K // group)
    q = (randn(Nn, K) * 2.7).round_().clamp_(-8, 7).to(torch.int8)
    s["packed"] = ((q[:, 0::2] & 15) | ((q[:, 1::2] & 15) << 4)).view(torch.uint8)
    s["scales"] = ((0.5 + rand(Nn, G)) * 0.02).half()
    s["bias"] = randn(Nn).to(DT[case["out"]]) if case["bias"] else None
    s["x_scale"] = None
    if case["x"] == "i8":
        s["x"] = (randn(M, K) * 33.0).round_().clamp_(-127, 127).to(torch.int8)
    elif case["x"] == "e4m3":
        s["x"] = (randn(M, K) * 100.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    else:
        s["x"] = randn(M, K).to(DT[case["x"]])
    if case["x"] in QMAX:
        s["x_scale"] = (0.5 + rand(M, G if case["scale"] == "group" else 1)) * (4.0 / QMAX[case["x"]])
    if own:
        from rl_quant_b200.w4linear import pack_w4

        s["weight"] = pack_w4(s["packed"], s["scales"], group)
    return s


# -- plain forms -------------------------------------------------------------------------------


def _plain_norm(x, w, res):
    """(y unrounded, h as stored or None, 1/rms, h in 32 bits)"""
    h = None
    xf = x.float()
    if res is not None:
        h = (xf + res.float()).to(res.dtype)
        xf = h.float()
    rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    return xf * rstd * w.float(), h, rstd, xf


def _plain_quant(y, case, given):
    Q = QMAX[case["out"]]
    R, C = y.shape
    if case["scale"] == "given":
        s, per = given, given
    else:
        width = case["group"] or C
        G = -(-C // width)
        padded = torch.zeros(R, G * width, device=y.device)
        padded[:, :C] = y
        s = padded.view(R, G, width).abs().amax(-1) / Q
        s = torch.where(s > 0, s, torch.ones_like(s))
        per = s.repeat_interleave(width, dim=1)[:, :C]
    v = (y / per).clamp(-Q, Q)
    return (v.round().to(torch.int8) if case["out"] == "i8" else v.to(torch.float8_e4m3fn)), s


def _unpack(packed):
    q = torch.stack((packed & 15, packed >> 4), dim=-1).view(packed.shape[0], -1).float()
    return q - 16.0 * (q > 7.0)


def _plain_w4(s):
    case = s["case"]
    col = torch.arange(case["k"], device="cuda") // case["group"]
    W = _unpack(s["packed"]) * s["scales"].float()[:, col]
    x = s["x"].float()
    if s["x_scale"] is not None:
        x = x * (s["x_scale"][:, col] if case["scale"] == "group" else s["x_scale"])
    y = x @ W.T
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(DT[case["out"]])


# -- one pass ----------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if case["op"] == "norm":
        x, w, res = s["x"], s["w"], s["res"]
        if own:
            from rl_quant_b200.norm import rms_norm

            if res is None:
                y, h = rms_norm(x, w, eps=EPS), None
            else:
                y, h = rms_norm(x, w, residual=res, eps=EPS)
            if not case["back"]:
                return [y] if h is None else [y, h]
            if h is None:
                return [y.detach(), *torch.autograd.grad(y, (x, w), s["dy"])]
            dx, dw, dr = torch.autograd.grad((y, h), (x, w, res), (s["dy"], s["dh"]))
            return [y.detach(), h.detach(), dx, dw, dr]
        with torch.no_grad():
            y, h, rstd, hf = _plain_norm(x, w, res)
            out = [y.to(x.dtype)] if h is None else [y.to(x.dtype), h]
            if not case["back"]:
                return out
            dy = s["dy"].float()
            g = dy * w.float()
            d = rstd * (g - hf * rstd * rstd * (g * hf).mean(-1, keepdim=True))
            if h is not None:
                d = d + s["dh"].float()
            dw = (dy * hf * rstd).sum(0)
            return out + [d.to(x.dtype), dw.to(w.dtype)] + ([] if h is None else [d.to(res.dtype)])
    if case["op"] == "normq":
        if own:
            from rl_quant_b200.norm import rms_norm_quant

            got = rms_norm_quant(s["x"], s["w"], residual=s["res"], eps=EPS, out_dtype=DT[case["out"]],
                                 group=case["group"], scale=s["given"])
            q, scale, h = got if s["res"] is not None else (*got, None)
        else:
            y, h, _, _ = _plain_norm(s["x"], s["w"], s["res"])
            q, scale = _plain_quant(y, case, s["given"])
        if case["out"] == "i8":  # the values that the codes stand for
            per = scale
            if case["scale"] == "group":
                per = scale.repeat_interleave(case["group"], dim=1)[:, :case["cols"]]
            q = torch.mul(q, per, out=s["buf"])
        out = [q] if case["scale"] == "given" else [q, scale]
        return out if h is None else out + [h]
    if own:
        from rl_quant_b200.w4linear import w4_linear

        return w4_linear(s["x"], s["weight"], bias=s["bias"], x_scale=s["x_scale"], out_dtype=DT[case["out"]])
    return _plain_w4(s)


def work(case):
    if case["op"] in ("norm", "normq"):
        e = case["rows"] * case["cols"]
        xb, rb, wb = BYTES[case["x"]], BYTES[case["res"]], BYTES[case["w"]]
        if case["op"] == "norm":
            b = e * (2 * xb + 2 * rb) + case["cols"] * wb
            if case["back"]:
                b += e * (2 * xb + 2 * rb) + case["cols"] * wb
            return {"bytes": b, "flops": e * (15 if case["back"] else 5)}
        G = {"row": 1, "given": 0, "group": -(-case["cols"] // max(1, case["group"]))}[case["scale"]]
        return {"bytes": e * (xb + 2 * rb + 1) + case["cols"] * wb + 4 * case["rows"] * G, "flops": e * 8}
    m, n, k = case["m"], case["n"], case["k"]
    G = -(-k // case["group"])
    b = n * k // 2 + 2 * n * G + m * k * BYTES[case["x"]] + m * n * BYTES[case["out"]]
    if case["bias"]:
        b += n * BYTES[case["out"]]
    if case["scale"]:
        b += 4 * m * (G if case["scale"] == "group" else 1)
    return {"bytes": b, "flops": 2 * m * n * k}


# -- the definition in 64 bits -----------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    D = torch.float64
    if case["op"] in ("norm", "normq"):
        v, h = s["x"].to(D), None
        if s["res"] is not None:
            v = v + s["res"].to(D)
            h = v.to(s["res"].dtype)      # the sum is an output of its own; the norm is of that output
            v = h.to(D)
        C = case["cols"]
        inv = 1.0 / torch.sqrt(torch.einsum("rc,rc->r", v, v) / C + EPS)
        unit = v * inv[:, None]
        weight = s["w"].to(D)
        y = unit * weight
        hs = [] if h is None else [v]
        if case["op"] == "norm":
            if not case["back"]:
                return [y] + hs
            dy = s["dy"].to(D)
            t = dy * weight
            dh = inv[:, None] * (t - unit * torch.einsum("rc,rc->r", t, unit)[:, None] / C)
            if h is not None:
                dh = dh + s["dh"].to(D)
            return [y] + hs + [dh, torch.einsum("rc,rc->c", dy, unit)] + ([] if h is None else [dh])
        Q = QMAX[case["out"]]
        if case["scale"] == "given":
            step = s["given"].to(D).expand_as(y)
        else:
            parts = y.abs().split(case["group"] or C, dim=1)
            tops = torch.stack([p.amax(dim=1) for p in parts], dim=1) / Q
            tops = tops.masked_fill(tops == 0, 1.0)
            step = torch.cat([tops[:, i:i + 1].expand(-1, p.shape[1]) for i, p in enumerate(parts)], dim=1)
        units = torch.minimum(torch.maximum(y / step, torch.tensor(-Q, device="cuda", dtype=D)),
                              torch.tensor(Q, device="cuda", dtype=D))
        if case["out"] == "i8":
            values = torch.round(units) * step
        else:
            values = units.to(torch.float8_e4m3fn).to(D)
        return [values] + ([] if case["scale"] == "given" else [tops]) + hs
    q = torch.empty(case["n"], case["k"], dtype=D, device="cuda")
    b = s["packed"].to(torch.int32)
    q[:, 0::2] = ((b << 28) >> 28).to(D)
    q[:, 1::2] = ((b << 24) >> 28).to(D)
    x = s["x"].to(D)
    y = torch.zeros(case["m"], case["n"], dtype=D, device="cuda")
    step = case["group"]
    sc = s["scales"].to(D)
    for i, lo in enumerate(range(0, case["k"], step)):
        part = x[:, lo:lo + step]
        if s["x_scale"] is not None:
            part = part * s["x_scale"][:, i if case["scale"] == "group" else 0, None].to(D)
        y += (part @ q[:, lo:lo + step].T) * sc[:, i]
    return y if s["bias"] is None else y + s["bias"].to(D)
