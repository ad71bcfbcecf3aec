"""w4_linear / W4Linear against the definition in 64 bits.

Tolerance, fixed before the first run: the products x * q are exact; a tensor-core sum keeps at least 24 bits of its
largest term, so each of at most K/16 steps, 64 joins and scale products is off by at most 2^-23 of the sum of
magnitudes S = sum |x q| s xs seen so far, in all (K/16 + 64) * 2^-23 * S; the result is rounded once (half a step)."""
import contextlib
import threading

import numpy as np
import pytest
import torch
import torch.nn as nn

from rl_quant_b200 import _native as N
from rl_quant_b200 import swap
from rl_quant_b200.fused import DeviceStatusError
from rl_quant_b200.norm import RMSNorm, rms_norm_quant
from rl_quant_b200.w4a16 import quantize_w4
from rl_quant_b200.w4linear import W4Linear, W4Weight, pack_w4, unpack_w4, w4_linear, w4_status

gpu = pytest.mark.gpu
F16, BF16, I8, E4M3 = torch.float16, torch.bfloat16, torch.int8, torch.float8_e4m3fn


def weight(n, k, group, seed, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-8, 8, (n, k), generator=g).to(torch.int8)
    packed = ((q[:, 0::2] & 15) | ((q[:, 1::2] & 15) << 4)).view(torch.uint8)
    s = ((0.5 + torch.rand(n, -(-k // group), generator=g)) * 0.02).half()
    return q.to(device), packed.to(device), s.to(device)


def rows(m, k, t, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g)
    if t == I8:
        return (x * 40).round().clamp(-128, 127).to(I8).cuda()
    if t == E4M3:
        return (x * 90).clamp(-448, 448).to(E4M3).cuda()
    return x.to(t).cuda()


def check(y, x, q, s, group, bias=None, xs=None):
    k = q.shape[1]
    col = torch.arange(k, device=q.device) // group
    W = q.double() * s.double()[:, col]
    xd = x.double()
    if xs is not None:
        xd = xd * (xs.double()[:, col] if xs.dim() == 2 and xs.shape[1] > 1 else xs.double())
    ref, S = xd @ W.T, xd.abs() @ W.abs().T
    if bias is not None:
        ref, S = ref + bias.double(), S + bias.double().abs()
    step = 0.0 if y.dtype == torch.float32 else torch.finfo(y.dtype).eps / 2
    tol = step * ref.abs() + (k / 16 + 64) * 2.0 ** -23 * S * (1 + step) + torch.finfo(y.dtype).smallest_normal * step
    assert torch.isfinite(y).all()
    assert ((y.double() - ref).abs() <= tol).all(), float(((y.double() - ref).abs() / tol.clamp_min(1e-30)).max())


# rows from one to several tiles of every kind, sizes off every tile
M_SIZES = [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 200, 300, 1000]
SHAPES = [(16, 64), (1, 2), (29, 128), (777, 1002), (512, 224), (130, 4096), (4096, 320), (17, 16384)]


@gpu
@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_16_bit_rows(n, k, group):
    q, packed, s = weight(n, k, group, n + k)
    w = pack_w4(packed, s, group)
    for i, m in enumerate(M_SIZES):
        t = (F16, BF16)[i % 2]
        x = rows(m, k, t, m)
        bias = rows(1, n, t, 7)[0] if i % 3 else None
        y = w4_linear(x, w, bias)
        assert y.dtype == t and y.shape == (m, n)
        check(y, x, q, s, group, bias)
    for t in (F16, BF16):
        for m in (1, 20, 150):
            x = rows(m, k, t, m)
            for out in (F16, BF16, torch.float32):
                check(w4_linear(x, w, out_dtype=out), x, q, s, group)


@gpu
@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("t", [I8, E4M3])
def test_8_bit_rows(n, k, group, t):
    q, packed, s = weight(n, k, group, n + k)
    w = pack_w4(packed, s, group)
    G = -(-k // group)
    for i, m in enumerate(M_SIZES):
        x = rows(m, k, t, m)
        for j, xs in enumerate((torch.tensor(0.01, device="cuda"), 0.01 * (0.5 + torch.rand(m, 1, device="cuda")),
                                0.01 * (0.5 + torch.rand(m, G, device="cuda")))):
            out = (F16, BF16, torch.float32)[(i + j) % 3]
            bias = rows(1, n, out, 7)[0] if (i + j) % 2 else None
            check(w4_linear(x, w, bias, x_scale=xs, out_dtype=out), x, q, s, group, bias, xs)


@gpu
def test_every_code_and_extremes():
    """Every weight code at every place of a word; the largest magnitudes of each input type; signed zeros."""
    k, group = 256, 64
    for v in range(-8, 8):
        q = torch.full((16, k), v, dtype=torch.int8)
        q[torch.arange(16), torch.arange(16) * 16 + 3] = -8
        packed = ((q[:, 0::2] & 15) | ((q[:, 1::2] & 15) << 4)).view(torch.uint8).cuda()
        s = torch.full((16, 4), 0.125, dtype=F16, device="cuda")
        w = pack_w4(packed, s, group)
        for m in (3, 40):
            x = rows(m, k, F16, v + 50)
            check(w4_linear(x, w), x, q.cuda(), s, group)
            x8 = rows(m, k, I8, v + 90)
            x8[0] = -128
            x8[1] = 127
            one = torch.tensor(1.0, device="cuda")
            check(w4_linear(x8, w, x_scale=one, out_dtype=torch.float32), x8, q.cuda(), s, group, None, one)
            xe = rows(m, k, E4M3, v)
            xe[0] = torch.full((k,), 448.0, device="cuda").to(E4M3)
            xe[1] = torch.full((k,), 2.0 ** -9, device="cuda").to(E4M3)
            check(w4_linear(xe, w, x_scale=one, out_dtype=torch.float32), xe, q.cuda(), s, group, None, one)


@gpu
def test_identity_rows_pick_weights():
    """A unit row picks one column of the weight exactly, for every column: the layout end to end."""
    n, k, group = 40, 192, 32
    q, packed, s = weight(n, k, group, 5)
    w = pack_w4(packed, s, group)
    W = (q.float() * s.float()[:, torch.arange(k, device="cuda") // group])
    for t in (F16, BF16):
        assert torch.equal(w4_linear(torch.eye(k, device="cuda").to(t), w, out_dtype=torch.float32), W.T)
    one = torch.tensor(1.0, device="cuda")
    for t in (I8, E4M3):
        x = torch.eye(k, device="cuda").to(t)
        for lo, hi in ((0, k), (3, 4), (5, 18)):
            assert torch.equal(w4_linear(x[lo:hi], w, x_scale=one, out_dtype=torch.float32), W.T[lo:hi])


@gpu
def test_nonfinite_rows_stay_apart():
    """A row with NaN or infinities spoils its own outputs only; zero scales give zeros."""
    q, packed, s = weight(48, 320, 64, 1)
    w = pack_w4(packed, s, 64)
    for m in (4, 12, 90, 260):
        x = rows(m, 320, F16, m)
        clean = w4_linear(x, w)
        x[1, 17] = float("nan")
        x[2, 300] = float("inf")
        y = w4_linear(x, w)
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.equal(y[keep], clean[keep])
        assert torch.isnan(y[1]).all() and not torch.isfinite(y[2][q[:, 300] != 0]).any()
    w0 = pack_w4(packed, torch.zeros_like(s), 64)
    assert not w4_linear(rows(5, 320, BF16, 1), w0).any()


@gpu
@pytest.mark.parametrize("t", [F16, I8])
def test_strides_alignment_and_shapes(t):
    q, packed, s = weight(100, 192, 64, 1)
    w = pack_w4(packed, s, 64)
    base = rows(70, 500, t, 2)
    xs = torch.rand(70, 1, device="cuda") if t == I8 else None
    kw = dict(x_scale=xs, out_dtype=F16) if t == I8 else {}
    for at in (0, 1, 2, 8, 16):
        for m in (1, 5, 70):
            k2 = dict(kw, x_scale=xs[:m]) if xs is not None else kw
            x = base[:m, at:at + 192]
            assert torch.equal(w4_linear(x, w, **k2), w4_linear(x.contiguous(), w, **k2))
    x = base[:, :192].t().contiguous().t()
    assert torch.equal(w4_linear(x, w, **kw), w4_linear(x.contiguous(), w, **kw))
    x3 = base[:, :192].reshape(7, 10, 192)
    k3 = dict(kw, x_scale=xs.view(7, 10, 1)) if xs is not None else kw
    assert torch.equal(w4_linear(x3, w, **k3).view(70, 100), w4_linear(base[:, :192], w, **kw))
    k1 = dict(kw, x_scale=xs[0]) if xs is not None else kw
    assert w4_linear(base[0, :192], w, **k1).shape == (100,)
    k0 = dict(kw, x_scale=xs[:0]) if xs is not None else kw
    assert w4_linear(base[:0, :192], w, **k0).shape == (0, 100)
    if xs is not None:
        g = torch.rand(70, 6, device="cuda")[:, ::2]
        assert torch.equal(w4_linear(base[:, :192], w, x_scale=g, out_dtype=F16),
                           w4_linear(base[:, :192], w, x_scale=g.contiguous(), out_dtype=F16))


@gpu
def test_status():
    q, packed, s = weight(512, 2048, 128, 1)
    w = pack_w4(packed, s, 128)
    for m in (1, 24, 200):
        w4_linear(rows(m, 2048, F16, 2), w)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert w4_status() == 0
    assert w4_status("cuda:0") == 0


@gpu
@pytest.mark.parametrize("t", [F16, I8, E4M3])
@pytest.mark.parametrize("m", [20, 40, 100])
@pytest.mark.parametrize("n,k,hold", [(256, 16384, 1), (256, 16384, 2), (256, 16384, 4), (256, 16384, 8), (19200, 2048, 1),
                                      (19200, 2048, 2), (19200, 2048, 4), (100, 250, 1), (256, 2050, 1)])
def test_waits_that_run_out(n, k, hold, m, t):
    """One arrival that never comes (a host switch) and a limit of a millisecond: the kernel gives up, says so in the
    status word, and the next calls are what they were. With blocks that share a tile's inputs (few columns) and
    without, rows that are copied by TMA and rows that are not, and a single unit of inputs."""
    lib = N.load()
    q, packed, s = weight(n, k, 64, 1)
    w = pack_w4(packed, s, 64)
    x = rows(m, k, t, 2)
    kw = {} if t == F16 else dict(x_scale=torch.full((m, -(-k // 64)), 0.01, device="cuda"), out_dtype=F16)
    want = w4_linear(x, w, **kw)
    assert w4_status() == 0
    N.check(lib.glad_debug_w4_wait(hold, 1_000_000))
    try:
        w4_linear(x, w, **kw)
        torch.cuda.synchronize()
    finally:
        N.check(lib.glad_debug_w4_wait(0, 0))
    with pytest.raises(DeviceStatusError):
        w4_status()
    assert w4_status() == 0
    for _ in range(2):
        assert torch.equal(w4_linear(x, w, **kw), want)
    assert w4_status() == 0


@gpu
@pytest.mark.parametrize("m", [5, 40])
def test_broadcast_rows(m):
    q, packed, s = weight(100, 192, 64, 1)
    w = pack_w4(packed, s, 64)
    for t in (F16, I8):
        kw = dict(x_scale=torch.ones(1, 1, device="cuda").expand(m, 1), out_dtype=F16) if t == I8 else {}
        x = rows(1, 192, t, 2).expand(m, 192)
        want = w4_linear(x.contiguous(), w, **kw)
        assert torch.equal(w4_linear(x, w, **kw), want) and torch.equal(want[0], want[-1])
        k3 = dict(kw, x_scale=kw["x_scale"].unsqueeze(0)) if kw else kw
        assert torch.equal(w4_linear(x.unsqueeze(0), w, **k3)[0], want)


@gpu
def test_streams_graph_repeat():
    q, packed, s = weight(512, 2048, 128, 1)
    w = pack_w4(packed, s, 128)
    for m in (1, 24, 200):
        x = rows(m, 2048, BF16, 2)
        want = w4_linear(x, w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [w4_linear(x, w) for _ in range(3)]
        main = [w4_linear(x, w) for _ in range(3)]        # at the same time on two streams
        side.synchronize()
        assert all(torch.equal(y, want) for y in got + main)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = w4_linear(x, w)
            graphs.append((g, y))
        x.copy_(rows(m, 2048, BF16, 3))
        for g, _ in graphs:
            g.replay()
        want = w4_linear(x, w)
        assert all(torch.equal(y, want) for _, y in graphs)


@gpu
def test_64_bit_offsets():
    """An output past 2^31 elements and rows past 2^31 elements apart."""
    q, packed, s = weight(16384, 64, 32, 1)
    w = pack_w4(packed, s, 32)
    x = rows(140000, 64, F16, 1)
    y = w4_linear(x, w)
    check(y[-100:], x[-100:], q, s, 32)
    big = torch.zeros(3, 1 << 30, dtype=F16, device="cuda")
    big[:, :64] = rows(3, 64, F16, 2)
    check(w4_linear(big[:, :64], w), big[:, :64], q, s, 32)
    del y, big


class Block(nn.Module):
    """Residual block of two linears behind a norm, as a policy's trunk has it."""

    def __init__(self, d, f):
        super().__init__()
        self.norm, self.up, self.down = nn.RMSNorm(d, eps=1e-6), nn.Linear(d, f), nn.Linear(f, d)

    def forward(self, x, res):
        y, h = self.norm(x, res)
        return self.down(torch.nn.functional.elu(self.up(y))), h


def block(seed=0):
    torch.manual_seed(seed)
    return Block(256, 640).cuda().half()


@gpu
def test_block_serves_and_trains():
    """The operators together: swapped block at inference (16-bit and int8 rows) and in training, refreshed in place."""
    b = block()
    params = {n: p for n, p in b.named_parameters()}
    swapped = swap.apply(b, {"up": {"bits": 4, "group": 32}, "down": {"bits": 4}})
    norms = swap.apply_norm(b)
    assert isinstance(b.up, W4Linear) and b.up.group == 32 and b.down.group == 64 and isinstance(b.norm, RMSNorm)
    assert all(params[n] is p for n, p in b.named_parameters())
    x, res = rows(5, 256, F16, 1), rows(5, 256, F16, 2)
    with torch.no_grad():
        y, h = b(x, res)
        n16 = b.norm(x, res)[0]
        up = w4_linear(n16, b.up.w4(), b.up.bias)
        assert torch.equal(y, w4_linear(torch.nn.functional.elu(up), b.down.w4(), b.down.bias))
        # the int8 form: the product of the codes is the product of the values they stand for
        q, s, h2 = b.norm.quant(x, res, group=32)
        assert torch.equal(h, h2)
        packed, sc = quantize_w4(b.up.weight, 32)
        codes = torch.stack((packed & 15, packed >> 4), -1).view(640, 256).to(torch.int8)
        codes = torch.where(codes > 7, codes - 16, codes)
        got = b.up(q, x_scale=s)
        assert got.dtype == F16
        check(got, q, codes, sc, 32, b.up.bias, s)
        # ... and near the 16-bit form: a code is off by half a step of s at most
        step = s.float().amax() / 2
        W = (codes.float() * sc.float()[:, torch.arange(256, device="cuda") // 32]).abs().sum(1)
        assert ((got.float() - up.float()).abs() <= step * W + 2.0 ** -9 * up.float().abs() + 0.02).all()
        ptr, before = b.up.tiles.data_ptr(), y.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            yg, _ = b(x, res)
        b.up.weight.mul_(0.5)
        b.up.requantize_()
        g.replay()
        assert b.up.tiles.data_ptr() == ptr
        assert torch.equal(yg, b(x, res)[0]) and not torch.equal(yg, before)
    # training: the plain layers' gradients
    ref = block()
    with torch.no_grad():
        ref.up.weight.mul_(0.5)
    out, h = b(x, res)
    out.float().square().sum().backward()
    yr, hr = ref.norm(x + res), x + res
    ref.down(torch.nn.functional.elu(ref.up(yr))).float().square().sum().backward()
    for (n, p), (_, r) in zip(b.named_parameters(), ref.named_parameters()):
        d = (p.grad.float() - r.grad.float()).norm() / r.grad.float().norm()
        assert d <= 2.0 ** -8, (n, float(d))       # fp16 gradients of fp16 activations, each rounded to 2^-11
    swap.restore(b, swapped)
    swap.restore_norm(b, norms)
    assert type(b.up) is nn.Linear and type(b.norm) is nn.RMSNorm and all(params[n] is p for n, p in b.named_parameters())


@gpu
@pytest.mark.parametrize("bias", [False, True])
def test_float32_rows(bias):
    """W4Linear serves what it trains on. x is split exactly, so the tolerance is that of the sums (module docstring): three
    of them over parts whose magnitudes add up to less than 1.01 |x|, two additions and the bias; what a third part loses below
    bfloat16's smallest number is 2^-134 of each input."""
    torch.manual_seed(0)
    for n, k, group in ((40, 64, 32), (777, 1002, 64), (130, 4096, 128)):
        m = W4Linear(nn.Linear(k, n, bias=bias), group=group).cuda()
        packed, s = quantize_w4(m.weight, group)
        q = torch.stack((packed & 15, packed >> 4), -1).view(n, k).double()
        W = (q - 16 * (q > 7)) * s.double()[:, torch.arange(k, device="cuda") // group]
        b = m.bias.detach().double() if bias else torch.zeros(n, dtype=torch.float64, device="cuda")
        for shape in ((1, k), (7, k), (3, 11, k), (300, k), (k,), (0, k)):
            x = torch.randn(shape, device="cuda") * torch.logspace(-30, 30, k, device="cuda")[torch.randperm(k)].pow(
                torch.rand((), device="cuda") < 0.5)
            with torch.no_grad():
                y = m(x)
                assert y.dtype == torch.float32 and y.shape == shape[:-1] + (n,)
                ref, S = x.double() @ W.T + b, x.double().abs() @ W.abs().T + b.abs()
                tol = 1.01 * (k / 16 + 68) * 2.0 ** -23 * S + 2.0 ** -134 * W.abs().sum(1)
                assert ((y.double() - ref).abs() <= tol).all()
                y16 = m(x, out_dtype=F16)
                assert y16.dtype == F16 and torch.equal(y16, y.half())
        x = torch.randn(9, k, device="cuda")
        with torch.no_grad():
            clean = m(x)
            x[1, 3], x[2, 5], x[3, 5] = float("nan"), float("inf"), -float("inf")
            y = m(x)
            assert torch.isnan(y[1]).all() and torch.equal(y[4:], clean[4:]) and torch.equal(y[0], clean[0])
            nz = W[:, 5] != 0
            for i, sign in ((2, 1.0), (3, -1.0)):
                assert torch.equal(y[i][nz], sign * torch.sign(W[nz, 5]).float() * float("inf")) and torch.isnan(y[i][~nz]).all()
            wide = torch.randn(5, 2 * k, device="cuda")
            assert torch.equal(m(wide[:, ::2]), m(wide[:, ::2].contiguous()))
            same = wide[:1, :k].expand(6, k)
            assert torch.equal(m(same), m(same.contiguous()))
            with pytest.raises(ValueError):
                m(wide)


@gpu
def test_float32_rows_past_a_third_of_the_limit():
    m = W4Linear(nn.Linear(64, 8)).cuda()
    x = torch.randn(400000, 64, device="cuda")
    with torch.no_grad():
        y = m(x)
        assert torch.equal(y[-1000:], m(x[-1000:])) and torch.equal(y[:1000], m(x[:1000]))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("mode", ["eager", "manual-graph"])
def test_runner_acts_through_w4_layers(dtype, mode):
    """InferenceRunner over a policy with 4-bit layers: built, acted with, synchronised with its master and checked. The
    reference is the same policy with the weights that the 4-bit copies stand for: four layers, each off by the tolerance of
    its sums (fp16: and a rounding of 2^-11), of which 1e-3 (fp16: 2^-6) of the largest mean leaves a factor of ten for
    cancellation."""
    from rl_quant_b200 import InferenceRunner, build_glad
    from rl_quant_b200.synthetic import glad_obs

    def policy(seed):
        torch.manual_seed(seed)
        return build_glad().cuda().to(dtype).eval()

    paths = ("actor.0", "actor.2", "actor.4")
    model = policy(0)
    swap.apply(model, {p: {"bits": 4, "group": 32} for p in paths})
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(model, mode=mode)
    obs = glad_obs(33, seed=1).cuda().to(dtype)
    for seed in (0, 1):
        master = policy(seed)
        run.sync_weights_from(master)
        with torch.no_grad():
            for p in paths:
                lin = master.get_submodule(p)
                packed, s = quantize_w4(lin.weight, 32)
                q = torch.stack((packed & 15, packed >> 4), -1).view(lin.weight.shape).float()
                lin.weight.copy_((q - 16 * (q > 7)) * s.float().repeat_interleave(32, 1)[:, :lin.in_features])
            want = master.act_inference({"policy_obs": obs})[0].float()
        got = run.act(obs)
        assert got.dtype == dtype
        assert (got.float() - want).abs().max() <= (1e-3 if dtype == torch.float32 else 2.0 ** -6) * want.abs().max()
    run.check_status()


@gpu
@pytest.mark.parametrize("src_t", [torch.float32, F16, BF16])
@pytest.mark.parametrize("dst_t", [torch.float32, F16, BF16])
def test_runner_syncs_every_type(src_t, dst_t):
    """sync_weights_from between a master and a copy of any two of the types that the layers take: each value is the master's,
    rounded once; 4-bit copies are those of the new weights. Odd and empty sizes, infinities and NaN among them."""
    from rl_quant_b200 import InferenceRunner

    def model(t):
        m = nn.Sequential(nn.RMSNorm(64, eps=1e-6), nn.Linear(64, 33), nn.ELU(), nn.Linear(33, 7)).cuda().to(t)
        m.register_buffer("extra", torch.zeros(5, device="cuda").to(t))
        m.register_buffer("none", torch.zeros(0, device="cuda").to(t))
        return m

    src, dst = model(src_t), model(dst_t)
    swap.apply(dst, {"1": {"bits": 4, "group": 32}})
    swap.apply_norm(dst)
    src.extra.copy_(torch.tensor([float("inf"), -float("inf"), float("nan"), 6e4, 2.0 ** -20]))
    run = InferenceRunner.__new__(InferenceRunner)
    run.model, run._g_sync, run._sync_items = dst, None, None
    run._quant_layers = [m for m in dst.modules() if m is not dst and hasattr(m, "requantize_")]
    for graph in (False, True, True):
        with torch.no_grad():
            for p in src.parameters():
                p.normal_()
        run.sync_weights_from(src, use_graph=graph)
        want = dict(src.named_parameters()) | dict(src.named_buffers())
        have = dict(dst.named_parameters()) | dict(dst.named_buffers())
        for name, t in want.items():
            assert have[name].dtype == dst_t
            assert torch.equal(have[name].detach().nan_to_num(1.5, 1e3, -1e3), t.detach().to(dst_t).nan_to_num(1.5, 1e3, -1e3)), name
        w = pack_w4(*quantize_w4(dst[1].weight, 32), 32)
        assert torch.equal(dst[1].tiles, w.tiles) and torch.equal(dst[1].scales, w.scales)


@gpu
def test_runner_refreshes_w4_layers():
    """InferenceRunner's weight hand-over reaches W4Linear layers (refresh_quant, eager and graphed)."""
    from rl_quant_b200 import InferenceRunner

    class Policy(nn.Module):
        def __init__(self):
            super().__init__()
            self.actor = nn.Sequential(nn.Linear(64, 96), nn.ELU(), nn.Linear(96, 8))

    p = Policy().cuda().half()
    swap.apply(p, {"actor.0": {"bits": 4}})
    run = InferenceRunner.__new__(InferenceRunner)
    run.model, run._g_refresh = p, None
    run._quant_layers = [m for m in p.modules() if m is not p and hasattr(m, "requantize_")]
    for graph in (False, True, True):
        with torch.no_grad():
            p.actor[0].weight.normal_()
        run.refresh_quant(use_graph=graph)
        want = pack_w4(*quantize_w4(p.actor[0].weight, 64), 64)
        assert torch.equal(p.actor[0].tiles, want.tiles) and torch.equal(p.actor[0].scales, want.scales)


# -- no GPU ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("n,k,group", [(1, 2, 32), (16, 64, 64), (29, 130, 128), (140, 192, 32), (33, 100, 64)])
def test_layout(n, k, group):
    """tiles and scales as include/glad_b200.h words them, element by element; the round trip."""
    q, packed, s = weight(n, k, group, 3, "cpu")
    w = pack_w4(packed, s, group)
    lib = N.load()
    assert w.tiles.numel() == lib.glad_w4_tiles_bytes(k, n, group)
    assert w.scales.numel() * 2 == lib.glad_w4_scales_bytes(k, n, group)
    T, U, G = w.tiles.shape[0], w.tiles.shape[1], 128 // group
    words = w.tiles.numpy().view(np.uint32).reshape(T, U, 8, 2, 32, 4).astype(np.int64)
    sc = w.scales.view(T, U, 8, G, 8, 2)
    seen, scales = np.zeros((T * 128, U * 128), np.int64), torch.zeros(T * 128, U * G, dtype=torch.float16)
    for t, u, b, lane in np.ndindex(T, U, 8, 32):
        r, c = lane >> 2, lane & 3
        for kb, j, i in np.ndindex(2, 4, 8):
            row = 128 * t + 16 * b + r + 8 * (i & 1)
            col = 128 * u + 64 * kb + 16 * j + 4 * c + 2 * ((i >> 1) & 1) + (i >> 2)
            v = (words[t, u, b, kb, lane, j] >> (4 * i)) & 15
            seen[row, col] = v - 16 if v > 7 else v
        for gi, h in np.ndindex(G, 2):
            scales[128 * t + 16 * b + r + 8 * h, u * G + gi] = sc[t, u, b, gi, r, h]
    assert np.array_equal(seen[:n, :k], q.numpy()) and not seen[n:].any() and not seen[:, k:].any()
    g = s.shape[1]
    assert torch.equal(scales[:n, :g], s) and not scales[n:].any() and not scales[:, g:].any()
    p2, s2 = unpack_w4(w)
    assert torch.equal(p2, packed) and torch.equal(s2, s)


def test_refusals():
    q, packed, s = weight(24, 128, 64, 1, "cpu")
    w = pack_w4(packed, s, 64)
    x = torch.zeros(3, 128, dtype=F16)
    x8 = x.to(I8)
    one, row, grp = torch.ones(()), torch.ones(3, 1), torch.ones(3, 2)
    for bad, args, kw in (
            (ValueError, (x[:, :126], w), {}), (TypeError, (x.float(), w), {}), (TypeError, (x.to(torch.uint8), w), {}),
            (ValueError, (torch.tensor(1.0), w), {}), (TypeError, (x, w), dict(out_dtype=torch.float64)),
            (ValueError, (x, w), dict(x_scale=one)), (ValueError, (x8, w), dict(out_dtype=F16)),
            (ValueError, (x8, w), dict(x_scale=row)), (TypeError, (x8, w), dict(x_scale=row.half(), out_dtype=F16)),
            (ValueError, (x8, w), dict(x_scale=torch.ones(3), out_dtype=F16)),
            (ValueError, (x8, w), dict(x_scale=torch.ones(3, 3), out_dtype=F16)),
            (ValueError, (x8, w), dict(x_scale=torch.ones(1, 2), out_dtype=F16)),
            (ValueError, (x, w, torch.zeros(23, dtype=F16)), {}), (ValueError, (x, w, torch.zeros(24)), {}),
            (ValueError, (x.to("meta"), w), {}), (RuntimeError, (x, w), {}),
            (RuntimeError, (x8, w), dict(x_scale=grp, out_dtype=F16)),
            (RuntimeError, (x.clone().requires_grad_(), w), {})):
        with pytest.raises(bad):
            w4_linear(*args, **kw)
    for args in ((packed, s, 16), (packed.view(I8), s, 64), (packed, s.float(), 64), (packed, s[:, :1], 64),
                 (packed, s, 32), (packed[:, :0], s[:, :0], 64), (packed[0], s, 64)):
        with pytest.raises(ValueError):
            pack_w4(*args)
    for args in ((w.tiles, w.scales, 127, 24, 64), (w.tiles, w.scales, 128, 24, 48), (w.tiles, w.scales, 128, 133, 64),
                 (w.tiles[..., :512], w.scales, 128, 24, 64), (w.tiles, w.scales.float(), 128, 24, 64)):
        with pytest.raises(ValueError):
            W4Weight(*args)
    with pytest.raises(ValueError):
        W4Linear(nn.Linear(7, 3))
    with pytest.raises(ValueError):
        W4Linear(nn.Linear(8, 3), group=8)
    with pytest.raises(ValueError):
        swap.apply(nn.Sequential(nn.Linear(8, 3)), {"0": {"bits": 3}})
    with pytest.raises(ValueError):
        swap.apply(nn.Sequential(nn.Linear(8, 3)), {"0": {"bits": 4, "s_z": 0.1}})


def test_swap_and_restore_on_cpu():
    m = nn.Sequential(nn.RMSNorm(64, eps=1e-6), nn.Linear(64, 40), nn.ELU(), nn.Linear(40, 3, bias=False)).eval()
    params = list(m.parameters())
    x = torch.randn(5, 64)
    want = m(x)
    sw = swap.apply(m, {"1": {"bits": 4}, "3": {"bits": 4, "group": 128}})
    nm = swap.apply_norm(m, ["0"])
    assert [type(l) for l in m] == [RMSNorm, W4Linear, nn.ELU, W4Linear] and not m[1].training
    assert all(a is b for a, b in zip(params, m.parameters()))
    p, s = unpack_w4(m[1].w4())
    p2, s2 = quantize_w4(m[1].weight, 64)
    assert torch.equal(p, p2) and torch.equal(s, s2)
    swap.restore(m, sw)
    swap.restore_norm(m, nm)
    assert [type(l) for l in m] == [nn.RMSNorm, nn.Linear, nn.ELU, nn.Linear] and torch.equal(m(x), want)
    assert all(a is b for a, b in zip(params, m.parameters())) and m[0].eps == 1e-6


def test_abi_refusals():
    lib = N.load()
    a = np.zeros(8192, np.float32).ctypes.data // 16 * 16 + 16          # an address that no call may reach

    def call(tiles=a, scales=a, k=128, n=24, group=64, x=a, t=N.DTYPE_F16, m=2, ld=128, xs=None, xr=0, xg=0, b=None, y=a,
             yt=N.DTYPE_F16):
        return lib.glad_w4_linear_forward(N.GladW4Weight(tiles, scales, k, n, group), x, t, m, ld, xs, xr, xg, b, y, yt,
                                          None)

    assert call(m=0) == N.GLAD_OK
    for kw in (dict(tiles=None), dict(scales=None), dict(tiles=a + 8), dict(scales=a + 2), dict(k=127), dict(k=0),
               dict(k=1 << 21), dict(n=0), dict(n=1 << 21), dict(group=16), dict(x=None), dict(y=None), dict(x=a + 1),
               dict(y=a + 1), dict(b=a + 1), dict(t=N.DTYPE_F32), dict(t=9), dict(yt=N.DTYPE_I8), dict(m=-1),
               dict(m=(1 << 20) + 1), dict(ld=64), dict(xs=a), dict(t=N.DTYPE_I8), dict(t=N.DTYPE_I8, xs=a + 2),
               dict(t=N.DTYPE_I8, xs=a, xr=1, xg=3), dict(t=N.DTYPE_I8, xs=a, xr=0, xg=2),
               dict(t=N.DTYPE_E4M3, xs=a, xr=2, xg=1)):
        assert call(**kw) == N.GLAD_ERR_INVALID_ARG, kw
        assert lib.glad_last_error()
    assert lib.glad_w4_tiles_bytes(127, 8, 64) == 0 and lib.glad_w4_scales_bytes(128, 8, 48) == 0
    assert lib.glad_w4_linear_status(None, None) == N.GLAD_ERR_INVALID_ARG
    assert lib.glad_debug_w4_wait(16, 0) == lib.glad_debug_w4_wait(1, 2_000_000_001) == N.GLAD_ERR_INVALID_ARG


def test_status_raises(monkeypatch):
    """A status word with a bit set, as a fake of the library reports it."""
    from rl_quant_b200.fused import DeviceStatusError

    class Fake:
        def glad_w4_linear_status(self, word, stream):
            word.value = 1
            return N.GLAD_ERR_DEVICE

    monkeypatch.setattr(N, "load", Fake)
    monkeypatch.setattr(N, "stream_handle", lambda device=None: 0)
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    with pytest.raises(DeviceStatusError):
        w4_status(0)


def test_runner_checks_w4_status(monkeypatch):
    from rl_quant_b200 import w4linear
    from rl_quant_b200.runtime import InferenceRunner
    asked = []
    monkeypatch.setattr(w4linear, "w4_status", asked.append)
    run = InferenceRunner.__new__(InferenceRunner)
    run._fused = run._fused_critic = run._fused_ac = None
    run.model = nn.Sequential(nn.Linear(64, 8))
    run.check_status()
    assert not asked
    swap.apply(run.model, {"0": {"bits": 4}})
    run.check_status()
    assert asked == [torch.device("cpu")]


def test_8_bit_rows_refuse_a_gradient():
    """8-bit rows have no training form: with gradients enabled they are refused, not served without one."""
    q, one = torch.zeros(3, 64, dtype=I8), torch.ones(())
    m = W4Linear(nn.Linear(64, 8))
    with pytest.raises(RuntimeError, match="no gradient"):
        m(q, x_scale=one)
    m.weight.requires_grad_(False)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(q, x_scale=one)                     # the bias
    m.bias.requires_grad_(False)
    with pytest.raises(RuntimeError, match="no gradient"):
        m(q, x_scale=one.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="CUDA"):
        m(q, x_scale=one)                     # nothing asks for one: served (by the kernels only)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        W4Linear(nn.Linear(64, 8))(q, x_scale=one)


def test_rows_of_every_type_refuse_other_outputs():
    m = W4Linear(nn.Linear(64, 8))
    with torch.no_grad():
        for x in (torch.zeros(3, 64), torch.zeros(3, 64, dtype=F16)):
            for out in (torch.float64, torch.int8):
                with pytest.raises(TypeError):
                    m(x, out_dtype=out)
        with pytest.raises(TypeError):
            m(torch.zeros(3, 64, dtype=torch.float64))
        with pytest.raises(RuntimeError, match="CUDA"):
            m(torch.zeros(3, 64))


def test_scales_refuse_a_gradient():
    q, packed, s = weight(24, 128, 64, 1, "cpu")
    w, x = pack_w4(packed, s, 64), torch.zeros(3, 128, dtype=I8)
    for shape in ((), (3, 1), (3, 2)):
        xs = torch.ones(shape, requires_grad=True)
        with pytest.raises(RuntimeError, match="no gradient"):
            w4_linear(x, w, x_scale=xs, out_dtype=F16)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            w4_linear(x, w, x_scale=xs, out_dtype=F16)
    given = torch.ones((), requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quant(torch.zeros(3, 64), scale=given)


def test_forward_mode_is_refused():
    from test_norm import forward_mode
    q, packed, s = weight(24, 128, 64, 1, "cpu")
    w = pack_w4(packed, s, 64)
    forward_mode(lambda x, b: w4_linear(x, w, b), torch.ones(3, 128, dtype=F16), torch.ones(24, dtype=F16))
    forward_mode(lambda xs: w4_linear(torch.ones(3, 128, dtype=I8), w, x_scale=xs, out_dtype=F16), torch.ones(3, 1))
    m, x = W4Linear(nn.Linear(64, 8).half()), torch.ones(3, 64, dtype=F16)
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
        m(forward_ad.make_dual(x, x))
    with forward_ad.dual_level():             # with gradients enabled it is F.linear
        y = m(forward_ad.make_dual(x, x))
        assert torch.equal(forward_ad.unpack_dual(y).tangent, torch.nn.functional.linear(x, m.weight))


def test_cast_copy_refuses_other_types():
    lib = N.load()
    a = np.zeros(64, np.float32).ctypes.data
    for src, dst in ((N.DTYPE_I8, 0), (0, N.DTYPE_E4M3), (-1, 0), (0, 9)):
        assert lib.glad_cast_copy(N.GladCastCopy(a, a, 0, src, dst), 1, None) == N.GLAD_ERR_INVALID_ARG


def test_a_refused_layer_leaves_the_model_as_it_was():
    """A refusal in the middle of a plan: nothing of it is applied, so nothing has to be put back."""
    m = nn.Sequential(nn.RMSNorm(64, eps=1e-6), nn.Linear(64, 7), nn.Linear(7, 5), nn.RMSNorm((1, 5), eps=1e-6),
                      nn.RMSNorm(5, elementwise_affine=False))
    before = list(m)
    for plan, error in (({"1": {"bits": 4}, "2": {"bits": 4}}, ValueError), ({"1": {"bits": 4}, "2": {"bits": 5}}, ValueError),
                        ({"1": {"bits": 4}, "0": {"bits": 4}}, AssertionError), ({"1": {"bits": 4}, "9": {"bits": 4}}, AttributeError)):
        with pytest.raises(error):
            swap.apply(m, plan)
        assert all(a is b for a, b in zip(m, before))
    for paths in (None, ["0", "3"], ["0", "4"]):
        with pytest.raises(ValueError):
            swap.apply_norm(m, paths)
        assert all(a is b for a, b in zip(m, before))
    with pytest.raises(AssertionError):
        swap.apply_norm(m, ["0", "1"])
    assert all(a is b for a, b in zip(m, before))


def bare_runner():
    from rl_quant_b200.runtime import InferenceRunner
    run = InferenceRunner.__new__(InferenceRunner)
    run._fused = run._fused_critic = run._fused_ac = None
    run.model = nn.Sequential(W4Linear(nn.Linear(64, 8)))
    run._device = lambda: 0
    return run


def test_every_reader_learns_of_a_failure(monkeypatch):
    """Two runners and a direct caller on one device: the first to ask clears the device's word, and still all three are
    told, once each, of each failure; another device's readers are not."""
    class Fake:
        bits = {0: 0, 1: 0}

        def glad_w4_linear_status(self, word, stream):
            word.value, self.bits[device[0]] = self.bits[device[0]], 0
            return N.GLAD_ERR_DEVICE if word.value else N.GLAD_OK

    device = [0]

    def select(index):
        device[0] = index
        return contextlib.nullcontext()

    monkeypatch.setattr(N, "load", Fake)
    monkeypatch.setattr(N, "stream_handle", lambda d=None: 0)
    monkeypatch.setattr(torch.cuda, "device", select)
    a, b = bare_runner(), bare_runner()
    for _ in range(2):                       # whatever was found before
        for ask in (a.check_status, b.check_status, lambda: w4_status(0)):
            with contextlib.suppress(DeviceStatusError):
                ask()
    for first in range(3):
        asks = [a.check_status, b.check_status, lambda: w4_status(0)]
        Fake.bits[0] = 1
        assert w4_status(1) == 0
        for ask in asks[first:] + asks[:first]:
            with pytest.raises(DeviceStatusError):
                ask()
        for ask in asks:
            ask()
    a.check_status()
    Fake.bits[0] = 1
    with pytest.raises(DeviceStatusError):
        b.check_status()
    Fake.bits[0] = 1
    with pytest.raises(DeviceStatusError):
        a.check_status()
    with pytest.raises(DeviceStatusError):
        b.check_status()
    with pytest.raises(DeviceStatusError):
        w4_status(0)


@gpu
def test_readers_on_the_device():
    """The same with kernels: one whose wait runs out on a side stream, two runners, a direct caller; calls in other streams
    and threads at the same time get words of their own."""
    lib = N.load()
    q, packed, s = weight(256, 2048, 64, 1)
    w, x = pack_w4(packed, s, 64), rows(40, 2048, F16, 2)
    a, b = bare_runner(), bare_runner()
    for ask in (a.check_status, b.check_status, w4_status):
        with contextlib.suppress(DeviceStatusError):
            ask()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    N.check(lib.glad_debug_w4_wait(1, 1_000_000))
    try:
        with torch.cuda.stream(side):
            w4_linear(x, w)
        side.synchronize()
    finally:
        N.check(lib.glad_debug_w4_wait(0, 0))
    for ask in (b.check_status, a.check_status, w4_status):
        with pytest.raises(DeviceStatusError):
            ask()
    found = []

    def many():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                found.append(w4_status())

    threads = [threading.Thread(target=many) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    a.check_status()
    assert found == [0] * 200


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32, torch.float64])
def test_module_casts(t):
    m = W4Linear(nn.Linear(64, 40)).bfloat16().to(t)
    assert m.weight.dtype == t and m.scales.dtype == F16
    packed, s = unpack_w4(m.w4())
    want, s2 = quantize_w4(m.weight, 64)
    assert torch.equal(packed, want) and torch.equal(s, s2)
