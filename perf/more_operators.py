"""The operators of a PPO update on adapters and tokens, and the cases they are measured on.

``lora``   low-rank adapters of many requests beside a shared projection, forward (serving) and backward (training)
``logp``   log probabilities of given tokens with entropy and top alternatives, forward and backward
``clip``   the global gradient norm over many tensors, and the gradients clipped by it

``own`` false: plain torch operations in 32 bits. ``own`` true: the package's operators.
"""
import math
import random

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}

# the parameters of this package's policy (actor, critic and their encoder): 612,637 elements
POLICY = [29, 1200, 16, 16, 16, 9216, 64, 64, 64, 6144, 64, 6336, 64, 64, 1, 8192, 64, 128, 1, 12288, 192, 4096, 64,
          114688, 512, 131072, 256, 32768, 128, 3712, 29, 116224, 512, 131072, 256, 32768, 128, 128, 1]


def listed():
    return [
        # one token of a running generation through one layer's adapter: latency only
        dict(name="lora_token_f16", op="lora", m=1, k=4096, n=4096, r=16, adapters=4, x="f16", base=True, runs=False,
             back=False),
        # a decoding batch where every request has an adapter of its own, wide layer
        dict(name="lora_batch_bf16", op="lora", m=64, k=4096, n=14336, r=16, adapters=64, x="bf16", base=True,
             runs=False, back=False),
        # prompts of several requests one after the other, high rank
        dict(name="lora_prompt_f16", op="lora", m=2048, k=4096, n=4096, r=64, adapters=6, x="f16", base=True, runs=True,
             back=False),
        # a 32-bit policy with one adapter a task, environments of all tasks mixed, sizes that fit no tile
        dict(name="lora_ragged_f32", op="lora", m=300, k=1002, n=777, r=9, adapters=5, x="f32", base=True, runs=False,
             back=True),
        # a training step's rows through one adapter
        dict(name="lora_train_bf16", op="lora", m=8192, k=4096, n=4096, r=16, adapters=1, x="bf16", base=True,
             runs=True, back=True),
        # one token, log probabilities of it and of five alternatives, with temperature
        dict(name="logp_token_f32", op="logp", rows=1, cols=65536, x="f32", top=5, entropy=True, temp=0.7, masked=False,
             back=False),
        # a decoding batch of an odd vocabulary with twenty alternatives each
        dict(name="logp_batch_bf16", op="logp", rows=61, cols=128001, x="bf16", top=20, entropy=False, temp=1.0,
             masked=False, back=False),
        # 4096 environments x 29 joints with 256 action bins each, some masked: loss and gradient
        dict(name="logp_bins_f16", op="logp", rows=118784, cols=256, x="f16", top=0, entropy=True, temp=1.0, masked=True,
             back=True),
        # a training batch over a large vocabulary: loss and gradient
        dict(name="logp_train_bf16", op="logp", rows=2048, cols=131072, x="bf16", top=0, entropy=True, temp=1.0,
             masked=False, back=True),
        # the policy's own gradients, clipped: launches and latency
        dict(name="clip_policy_f32", op="clip", tensors=0, total=sum(POLICY), x="f32", norm="2", clipped=True,
             packed=False),
        # the gradients of 224 adapter pairs, below the limit as in most steps
        dict(name="clip_adapters_bf16", op="clip", tensors=448, total=20_000_000, x="bf16", norm="2", clipped=False,
             packed=False),
        # a whole model's gradients, clipped
        dict(name="clip_model_bf16", op="clip", tensors=290, total=268_000_000, x="bf16", norm="2", clipped=True,
             packed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lora", "lora", "logp", "logp", "clip"])
    if op == "lora":
        while True:
            m, k, n = _log(rng, 1, 16384), _log(rng, 16, 16384), _log(rng, 16, 16384)
            if rng.random() < 0.7:
                k, n = max(16, k // 16 * 16), max(16, n // 16 * 16)
            r = rng.choice([4, 8, 16, 16, 32, 64, 128, rng.randint(1, 128)])
            adapters = rng.choice([1, 1, _log(rng, 2, 128)])
            if m * (k + n) <= 8192 * 8192 and adapters * r * (k + n) <= 2 ** 28 and \
                    m * adapters * r * (k + n) <= 10 ** 12 and m * r <= 8192 * 16 * 4:
                break
        return dict(op=op, m=m, k=k, n=n, r=r, adapters=adapters, x=rng.choice(["f16", "bf16", "bf16", "f32"]),
                    base=rng.random() < 0.8, runs=rng.random() < 0.5, back=rng.random() < 0.5)
    if op == "logp":
        back = rng.random() < 0.5
        while True:
            rows, cols = _log(rng, 1, 131072), _log(rng, 2, 262144)
            if rng.random() < 0.5:
                cols = max(8, cols // 8 * 8)
            if rows * cols <= (2 ** 27 if back else 2 ** 25):
                break
        top = 0 if back else rng.choice([0, 1, rng.randint(2, 32)])
        return dict(op=op, rows=rows, cols=cols, x=rng.choice(["f16", "bf16", "f32"]), top=min(top, cols),
                    entropy=rng.random() < 0.6, temp=rng.choice([1.0, 1.0, round(rng.uniform(0.3, 2.0), 2)]),
                    masked=cols >= 256 and rng.random() < 0.4, back=back)
    tensors = _log(rng, 1, 1000)
    return dict(op=op, tensors=tensors, total=_log(rng, tensors, 134_000_000), x=rng.choice(["f16", "bf16", "f32"]),
                norm=rng.choice(["2", "2", "inf", "1"]), clipped=rng.random() < 0.6, packed=rng.random() < 0.3)


def _sizes(case):
    """Sizes of the gradients: small and large ones mixed, their sum as stated; the same for every seed."""
    if not case["tensors"]:
        return POLICY
    count, total = case["tensors"], case["total"]
    rng = random.Random(count * 1000003 + total)
    share = [math.exp(rng.uniform(0.0, 5.0)) for _ in range(count)]
    scale = (total - count) / sum(share)
    sizes = [1 + int(v * scale) for v in share]
    sizes[0] += total - sum(sizes)
    return sizes


def _bucket(case):
    """A flat buffer and its parts, the gradients: at 256-byte boundaries each, or one directly after the other."""
    dt, parts, at = DT[case["x"]], [], 0
    step = 1 if case["packed"] else 256 // BYTES[case["x"]]
    for v in _sizes(case):
        parts.append((at, v))
        at += -(-v // step) * step
    flat = torch.zeros(at, dtype=dt, device="cuda")
    return flat, [flat[lo:lo + v] for lo, v in parts]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed + 1))
    dt = DT[case["x"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] == "lora":
        m, k, n, r, L = case["m"], case["k"], case["n"], case["r"], case["adapters"]
        train = case["back"]
        s["x"] = randn(m, k).to(dt).requires_grad_(train)
        s["a"] = (randn(L, r, k) / math.sqrt(k)).to(dt).requires_grad_(train)
        s["b"] = (randn(L, n, r) * 0.05).to(dt).requires_grad_(train)
        s["scale"] = 1.0 + rand(L)
        s["base"] = randn(m, n).to(dt) if case["base"] else None
        s["index"] = None
        if L > 1:
            # every adapter that the rows suffice for, then others; a few rows without one
            i = torch.arange(m, device="cuda") % L
            if m > L:
                i[L:] = torch.randint(L, (m - L,), generator=g, device="cuda")
                i[L:][rand(m - L) < 0.05] = -1
            i = i.sort().values if case["runs"] else i[torch.randperm(m, generator=g, device="cuda")]
            s["index"] = i.int()
        if train:
            s["dy"] = randn(m, n).to(dt)
        return s
    if case["op"] == "logp":
        R, V = case["rows"], case["cols"]
        x = randn(R, V).mul_(2.5)
        x[:, ::max(2, V // 16)] += 4.0          # a few likely tokens
        if case["masked"]:
            mask = rand(1, V) < 0.2
            mask[:, 0] = False
            x.masked_fill_(mask, -math.inf)
        # sampled by exponential races, as a rollout samples
        race = torch.empty_like(x).exponential_(generator=g).clamp_(min=1e-30).log_()
        s["tokens"] = (x / case["temp"]).sub_(race).argmax(-1)
        del race
        if R >= 16:
            s["tokens"][R - R // 16:] = -100    # padding at the end of the batch
        s["x"] = x.to(dt).requires_grad_(case["back"])
        if case["back"]:
            size = 64.0 if case["x"] == "f16" else 1.0 / R      # a mean over the rows; 16-bit floats under a loss scale
            s["g"] = randn(R) * size
            s["gh"] = torch.full((R,), -0.01 * size, device="cuda") if case["entropy"] else None
        return s
    s["flat"], s["grads"] = _bucket(case)
    for i, t in enumerate(s["grads"]):
        t.copy_(randn(t.numel()) * (1e-3 * (1 + i % 7)))
    # a limit well below or well above what such gradients have
    rms = 4.5e-3
    typical = {"2": rms * math.sqrt(case["total"]), "1": 0.8 * rms * case["total"], "inf": 5 * rms}[case["norm"]]
    s["max_norm"] = typical * (0.1 if case["clipped"] else 100.0)
    s["out_flat"], s["out"] = _bucket(case) if case["clipped"] else (None, None)
    return s


# -- plain forms -------------------------------------------------------------------------------


def _plain_lora(s):
    case = s["case"]
    L, r, m = case["adapters"], case["r"], case["m"]
    dt = DT[case["x"]]
    x = s["x"].float()
    a = s["a"].float().reshape(L * r, -1)                       # every adapter's rows, masked to each row's own
    b = s["b"].float().permute(0, 2, 1).reshape(L * r, -1)
    factor = s["scale"].repeat(m, 1)
    if s["index"] is not None:
        factor = factor * (s["index"][:, None] == torch.arange(L, device="cuda"))
    factor = factor.repeat_interleave(r, dim=1)
    u = (x @ a.T) * factor
    y = u @ b
    if s["base"] is not None:
        y = y + s["base"].float()
    out = [y.to(dt)]
    if case["back"]:
        dy = s["dy"].float()
        du = (dy @ b.T) * factor
        out += [(du @ a).to(dt), (du.T @ x).reshape(L, r, -1).to(dt),
                (u.T @ dy).reshape(L, r, -1).permute(0, 2, 1).contiguous().to(dt)]
    return out


def _plain_logp(s):
    case = s["case"]
    T, k = case["temp"], case["top"]
    x, tokens = s["x"].float(), s["tokens"]
    live = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    z = (x - x.amax(-1, keepdim=True)) / T
    e = z.exp()
    total = e.sum(-1, keepdim=True)
    logs = z - total.log()
    out = [torch.where(live, logs.gather(1, at)[:, 0], 0.0)]
    p = e / total
    if case["entropy"]:
        h = -(p * logs.masked_fill(p == 0, 0.0)).sum(-1)
        out.append(torch.where(live, h, 0.0))
    if k:
        order = x.sort(dim=-1, descending=True, stable=True).indices[:, :k]
        out += [torch.where(live[:, None], logs.gather(1, order), 0.0), torch.where(live[:, None], order, -1)]
    if case["back"]:
        d = p * -s["g"][:, None]
        d.scatter_add_(1, at, s["g"][:, None])
        if case["entropy"]:
            d -= s["gh"][:, None] * p * (logs.masked_fill(p == 0, 0.0) + h[:, None])
        out.append((d / T).masked_fill(~live[:, None], 0.0).to(s["x"].dtype))
    return out


def _plain_clip(s):
    case = s["case"]
    if case["norm"] == "2":
        parts = [(t.float() * t.float()).sum() for t in s["grads"]]
        norm = torch.stack(parts).sum().sqrt()
    elif case["norm"] == "1":
        norm = torch.stack([t.float().abs().sum() for t in s["grads"]]).sum()
    else:
        norm = torch.stack([t.float().abs().amax() for t in s["grads"]]).amax()
    c = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    if s["out"] is None:
        for t in s["grads"]:
            t.copy_(t.float() * c)
        return [norm, s["flat"]]
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * c)
    return [norm, s["out_flat"]]


# -- one pass ----------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if case["op"] == "lora":
        if not own:
            with torch.no_grad():
                return _plain_lora(s)
        from rl_quant_b200.lora import lora_linear

        y = lora_linear(s["x"], s["a"], s["b"], index=s["index"], scale=s["scale"], base=s["base"])
        if not case["back"]:
            return [y]
        return [y.detach(), *torch.autograd.grad(y, (s["x"], s["a"], s["b"]), s["dy"])]
    if case["op"] == "logp":
        if not own:
            with torch.no_grad():
                return _plain_logp(s)
        from rl_quant_b200.logprob import token_log_probs

        got = token_log_probs(s["x"], s["tokens"], temperature=case["temp"], entropy=case["entropy"], top=case["top"])
        outs = [got.log_prob] + ([got.entropy] if case["entropy"] else [])
        if case["back"]:
            d, = torch.autograd.grad(outs, s["x"], [s["g"]] + ([s["gh"]] if case["entropy"] else []))
            return [t.detach() for t in outs] + [d]
        return outs + ([got.top_log_prob, got.top_index] if case["top"] else [])
    if not own:
        return _plain_clip(s)
    from rl_quant_b200.gradnorm import clip_grads, clip_grads_

    kind = float(case["norm"])
    if s["out"] is None:            # in place; below the limit, so the gradients stay as they are
        return [clip_grads_(s["grads"], s["max_norm"], norm_type=kind), s["flat"]]
    _, norm = clip_grads(s["grads"], s["max_norm"], norm_type=kind, out=s["out"])
    return [norm, s["out_flat"]]


def work(case):
    e = BYTES[case["x"]]
    if case["op"] == "lora":
        m, k, n, r, L = case["m"], case["k"], case["n"], case["r"], case["adapters"]
        weights = min(m, L) * r * (k + n) * e
        b = m * (k + n * (2 if case["base"] else 1)) * e + weights + (4 * m if L > 1 else 0) + 4 * L
        flops = 2 * m * r * (k + n)
        if case["back"]:                        # dy and x in, dx and the adapters' gradients out
            b += m * (n + 2 * k) * e + weights + L * r * (k + n) * e
            flops *= 3
        return {"bytes": b, "flops": flops}
    if case["op"] == "logp":
        size = case["rows"] * case["cols"]
        live = size - (case["rows"] // 16 * case["cols"] if case["rows"] >= 16 else 0)
        b = live * e + case["rows"] * (8 + 4 + (4 if case["entropy"] else 0) + 12 * case["top"])
        if case["back"]:
            b += live * e + size * e + case["rows"] * 8
        return {"bytes": b, "flops": live * (14 if case["back"] else 6)}
    return {"bytes": case["total"] * e * (2 if case["clipped"] else 1) + 4,
            "flops": case["total"] * (3 if case["clipped"] else 2)}


# -- the definition in 64 bits -----------------------------------------------------------------


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    D = torch.float64
    if case["op"] == "lora":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=D, device="cuda") if s["base"] is None else s["base"].to(D)
        out = [y]
        if case["back"]:
            dx = torch.zeros(m, k, dtype=D, device="cuda")
            da, db = torch.zeros_like(s["a"], dtype=D), torch.zeros_like(s["b"], dtype=D)
            out += [dx, da, db]
        for i in range(case["adapters"]):
            rows = torch.arange(m, device="cuda") if s["index"] is None else (s["index"] == i).nonzero()[:, 0]
            if not len(rows):
                continue
            A, B, c = s["a"][i].to(D), s["b"][i].to(D), float(s["scale"][i])
            X = s["x"][rows].to(D)
            U = torch.einsum("mk,rk->mr", X, A)
            y[rows] += c * torch.einsum("mr,nr->mn", U, B)
            if case["back"]:
                G = s["dy"][rows].to(D)
                V = torch.einsum("mn,nr->mr", G, B)
                dx[rows] = c * torch.einsum("mr,rk->mk", V, A)
                da[i] = c * torch.einsum("mr,mk->rk", V, X)
                db[i] = c * torch.einsum("mn,mr->nr", G, U)
        return out
    if case["op"] == "logp":
        R, k = case["rows"], case["top"]
        parts = []
        step = max(1, 2 ** 26 // case["cols"])
        for lo in range(0, R, step):
            x = s["x"][lo:lo + step].detach().to(D) / case["temp"]
            t = s["tokens"][lo:lo + step]
            row = torch.arange(len(t), device="cuda")
            lse = torch.logsumexp(x, -1)
            lp = x[row, t.clamp(min=0)] - lse
            part = [lp]
            logs = x - lse[:, None]
            p = torch.exp(logs)
            if case["entropy"]:
                h = torch.special.entr(p).sum(-1)
                part.append(h)
            if k:
                part.append(torch.topk(logs, k, dim=-1).values)
            if case["back"]:
                w = s["g"][lo:lo + step].to(D)[:, None]
                d = -w * p
                d[row, t.clamp(min=0)] += w[:, 0]
                if case["entropy"]:
                    d += s["gh"][lo:lo + step].to(D)[:, None] * (torch.special.entr(p) - p * h[:, None])
                part.append(d / case["temp"])
            pad = t < 0
            for v in part:
                v[pad] = 0.0
            parts.append(part)
        out = [torch.cat(v) for v in zip(*parts)]
        return out + [None] if k else out
    p = float(case["norm"])
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(t.to(D), p) for t in s["grads"]]), p)
    c = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return [norm, s["flat"].to(D) * c]
