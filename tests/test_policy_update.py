"""Adapters, log probabilities and clipping together, as a PPO update on action tokens and its rollout use them: normalised
4-bit layers with an adapter a task, a head over action bins, one update step, and the captured rollout step.

The update is compared with the same step in 64-bit torch operators from the same float32 numbers. Tolerance: every operator on the
way keeps its sums in float32, at most a few hundred additions in a row, so gradients agree to 2^-24 times a few hundred of their
largest element; 2^-12 of it is taken, which a wrong term exceeds."""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from rl_quant_b200 import RMSNorm, clip_grad_norm_, grad_norm, swap, token_log_probs

gpu = pytest.mark.gpu
ROWS, OBS, WIDTH, JOINTS, BINS, TASKS = 60, 96, 128, 5, 24, 3
PATHS = ["1", "3"]


def policy(dtype=torch.float32):
    torch.manual_seed(0)
    m = nn.Sequential(RMSNorm(OBS), nn.Linear(OBS, WIDTH), nn.ELU(), nn.Linear(WIDTH, JOINTS * BINS)).cuda().to(dtype)
    quantised = swap.apply(m, {p: {"bits": 4, "group": 32} for p in PATHS})
    layers = swap.apply_lora(m, PATHS, rank=8, adapters=TASKS, alpha=16)
    for mod in layers.values():
        nn.init.normal_(mod.lora_b, std=0.05)
    return m, layers, quantised


def batch():
    g = torch.Generator().manual_seed(1)
    obs = torch.randn(ROWS, OBS, generator=g).cuda()
    task = torch.randint(-1, TASKS, (ROWS,), generator=g).cuda()
    actions = torch.randint(BINS, (ROWS, JOINTS), generator=g).cuda()
    actions[-4:] = -100                                     # padding
    old = torch.full((ROWS, JOINTS), -math.log(BINS)).cuda()
    advantage = torch.randn(ROWS, 1, generator=g).cuda()
    banned = torch.rand(ROWS, JOINTS, BINS, generator=g) < 0.1
    banned.scatter_(2, actions.cpu().clamp(min=0)[..., None], False)
    return obs, task, actions, old, advantage, banned.cuda()


def ppo_loss(lp, entropy, old, advantage, keep):
    ratio = (lp - old).exp()
    gain = torch.minimum(ratio * advantage, ratio.clamp(0.8, 1.2) * advantage)
    return -((gain + 0.01 * entropy) * keep).sum() / keep.sum()


def plain_step(m, layers, obs, task, actions, old, advantage, banned):
    """The same loss and gradients in 64 bits."""
    D = torch.float64
    leaves = [(mod.lora_a.detach().to(D).requires_grad_(), mod.lora_b.detach().to(D).requires_grad_()) for mod in layers.values()]
    h = obs.to(D)
    h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + m[0].eps) * m[0].weight.detach().to(D)
    for j, (mod, (a, b)) in enumerate(zip(layers.values(), leaves)):
        y = F.linear(h, mod.base.weight.detach().to(D), mod.base.bias.detach().to(D))
        on = (task >= 0).to(D)[:, None]
        t = task.clamp(min=0)
        y = y + mod.scale * on * torch.einsum("mnr,mr->mn", b[t], torch.einsum("mrk,mk->mr", a[t], h))
        h = F.elu(y) if j == 0 else y
    logits = h.view(ROWS, JOINTS, BINS).masked_fill(banned, -math.inf)
    logs = logits.log_softmax(-1)
    keep = (actions >= 0).to(D)
    lp = logs.gather(-1, actions.clamp(min=0)[..., None])[..., 0] * keep
    entropy = -(logs.exp() * logs.masked_fill(banned, 0.0)).sum(-1) * keep
    loss = ppo_loss(lp, entropy, old.to(D), advantage.to(D), keep)
    return loss, torch.autograd.grad(loss, [t for pair in leaves for t in pair])


@gpu
def test_update_step():
    m, layers, _ = policy()
    m[0].weight.requires_grad_(False)
    obs, task, actions, old, advantage, banned = batch()
    params = [p for p in m.parameters() if p.requires_grad]
    assert len(params) == 2 * len(layers)
    want_loss, want = plain_step(m, layers, obs, task, actions, old, advantage, banned)
    swap.select_lora(layers, task)

    def back():
        logits = m(obs).view(ROWS, JOINTS, BINS).masked_fill(banned, -math.inf)
        out = token_log_probs(logits, actions, entropy=True)
        loss = ppo_loss(out.log_prob, out.entropy, old, advantage, (actions >= 0).float())
        for p in params:
            p.grad = None
        loss.backward()
        return loss.detach()
    loss = back()
    assert abs(float(loss) - float(want_loss)) <= 2.0 ** -16 * (1 + abs(float(want_loss)))
    order = [p for mod in layers.values() for p in (mod.lora_a, mod.lora_b)]
    for p, w in zip(order, want):
        assert float((p.grad.double() - w).abs().max()) <= 2.0 ** -12 * float(w.abs().max())
        assert float(w.abs().max()) > 0
    n = math.sqrt(sum(float((w * w).sum()) for w in want))
    got = clip_grad_norm_(params, n / 2)
    assert abs(float(got) - n) <= 2.0 ** -12 * n
    assert abs(float(grad_norm([p.grad for p in params])) - n / 2) <= 2.0 ** -11 * n
    before = [p.detach().clone() for p in params]
    torch.optim.SGD(params, lr=0.1).step()
    assert all(not torch.equal(p, q) for p, q in zip(params, before))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rollout_step_in_a_graph(dtype):
    """Norm, 4-bit layers, adapters of the rows' tasks and log probabilities with alternatives, captured once: each replay reads the
    current observations, tasks and adapters."""
    m, layers, _ = policy(dtype)
    obs, task, actions, _, _, _ = batch()
    obs, task = obs.to(dtype), task.clone()
    swap.select_lora(layers, task)

    def step():
        logits = m(obs).view(ROWS, JOINTS, BINS)
        return logits, token_log_probs(logits, actions, temperature=0.8, entropy=True, top=3)
    with torch.no_grad():
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits, out = step()
        for k in range(2):
            obs.mul_(-0.5 - k)
            task.copy_(task.flip(0))
            layers["3"].lora_b.mul_(1.5)
            graph.replay()
            want_logits, want = step()
            assert torch.equal(logits, want_logits)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert (out.top_index[:-4] >= 0).all() and (out.top_index[-4:] == -1).all()
    best = logits[:-4].float().amax(-1)
    assert torch.equal(logits[:-4].float().gather(-1, out.top_index[:-4, :, :1])[..., 0], best)
