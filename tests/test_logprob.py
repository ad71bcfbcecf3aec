"""token_log_probs against the formula in 64 bits.

Tolerances, fixed before the first run, in units of u = 2^-24. z = (x - m) / T has three roundings: 3 |z| u. A term e^z is
off by the base-2 exponential's 4 u and by its argument's error, (4 |z|) u; a thread adds at most max(64, V / 128) terms and a tree joins at
most 1024 x 16 threads: S is off by A + 4 E|z| relative, A = max(64, V / 128) + 24, with E|z| = sum p |z|, and ln S by that and its own 2 u
and |ln S| u. H = ln S - E z adds E|z| (2 A + 16). Where p underflows (2^-126) nothing counts."""
import math

import pytest
import torch

from rl_quant_b200 import token_log_probs

gpu = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(rows, cols, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * scale).to(dtype).cuda()
    return x, torch.randint(cols, (rows,), generator=g).cuda()


class Ref:
    def __init__(self, x, T=1.0):
        self.x = x.double()
        m = self.x.amax(-1, keepdim=True)
        self.empty = m[:, 0] == -math.inf
        m = m.masked_fill(m == -math.inf, 0.0)
        self.z = (self.x - m) / T
        e = self.z.exp()
        s = e.sum(-1, keepdim=True)
        self.ln_s = s.log()
        self.log = self.z - self.ln_s
        self.p = torch.where(self.empty[:, None], 0.0, e / s)
        zf = self.z.masked_fill(self.p == 0, 0.0).abs()
        lf = self.log.masked_fill(self.p == 0, 0.0)
        self.h = -(self.p * lf).sum(-1)
        ez = (self.p * zf).sum(-1)
        A = max(64, x.shape[1] / 128) + 24
        self.ln_err = (A + 4 * ez + 2 + self.ln_s[:, 0].abs().nan_to_num(posinf=0.0)) * U
        self.h_err = self.ln_err + ez * (2 * A + 16) * U
        self.log_err = self.ln_err[:, None] + 3 * U * self.z.abs() + U * self.log.abs()
        self.T, self.lf = T, lf

    def grad(self, tok, g, gh, ti=None, gt=None):
        """(gradient, bound of its error before it is rounded)"""
        R, V = self.x.shape
        g, gh = (torch.zeros(R, dtype=torch.float64, device="cuda") if t is None else t.double() for t in (g, gh))
        G, mag = g.clone(), g.abs()
        if gt is not None:
            G, mag = G + gt.double().sum(-1), mag + gt.double().abs().sum(-1)
        lh = self.lf + self.h[:, None]
        d = -self.p * (G[:, None] + gh[:, None] * lh)
        rel = self.log_err.masked_fill(self.p == 0, 0.0) + 8 * U
        err = self.p * (rel + 8 * U) * (mag[:, None] + gh.abs()[:, None] * lh.abs())
        err = err + self.p * gh.abs()[:, None] * (self.log_err.masked_fill(self.p == 0, 0.0) + self.h_err[:, None] + 4 * U * lh.abs())
        err = err + self.p * 34 * U * mag[:, None]          # the sum of up to 33 given gradients
        add = torch.zeros_like(d)
        add.scatter_add_(1, tok[:, None], g[:, None])
        top = add.abs()
        if gt is not None:
            add.scatter_add_(1, ti, gt.double())
            top.scatter_add_(1, ti, gt.double().abs())
        live = ~self.empty[:, None]
        return torch.where(live, (d + add) / self.T, 0.0), (err + 4 * U * (top + d.abs())) / self.T


def check_forward(x, tok, T, top):
    r = Ref(x, T)
    got = token_log_probs(x, tok, temperature=T, entropy=True, top=top)
    inf = (x == math.inf).any(-1)           # such rows are NaN, but for the order of their columns
    live = ~r.empty & ~inf
    lp = r.log.gather(1, tok[:, None])[:, 0]
    same = (got.log_prob.double() == lp) | ((got.log_prob.double() - lp).abs() <= r.log_err.gather(1, tok[:, None])[:, 0])
    assert same[live].all() and (got.log_prob[r.empty] == -math.inf).all()
    assert ((got.entropy.double() - r.h).abs() <= r.h_err)[live].all() and (got.entropy[r.empty] == 0).all()
    assert got.log_prob[inf].isnan().all() and got.entropy[inf].isnan().all()
    if top:
        order = r.x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_index, order)
        want, err = r.log.gather(1, order), r.log_err.gather(1, order)
        near = (got.top_log_prob.double() == want) | ((got.top_log_prob.double() - want).abs() <= err)
        assert near[live].all() and (got.top_log_prob[r.empty] == -math.inf).all()
    else:
        assert got.top_log_prob is None and got.top_index is None
    return got


# widths: one column, below a warp, off every vector, one block, several pieces a thread, split rows; few rows and many
SIZES = [(1, 1), (3, 2), (5, 31), (64, 256), (2, 257), (700, 1000), (9, 1024), (3, 1025), (40, 4097), (5, 32768), (1, 65536),
         (2, 128001), (1, 262144), (300, 8200), (150, 50000)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SIZES)
def test_forward(shape, dtype):
    x, tok = make(*shape, dtype, 1)
    for T, top in ((1.0, 0), (0.7, min(5, shape[1])), (1.6, min(32, shape[1]))):
        check_forward(x, tok, T, top)
    got = token_log_probs(x, tok.int())
    assert got.entropy is None and torch.equal(got.log_prob, token_log_probs(x, tok).log_prob)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [33, 300, 1025, 20000, 65537])
def test_ties(cols, dtype):
    """Equal values: the lower index first."""
    g = torch.Generator().manual_seed(2)
    x = torch.randint(-2, 3, (4, cols), generator=g).to(dtype).cuda()
    x[1] = 0.5
    x[2, :] = 0.0
    x[2, ::2] = -0.0
    x[3] = torch.arange(cols).float().cuda().to(dtype)
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    check_forward(x, tok, 1.0, min(20, cols))
    check_forward(x.flip(-1).contiguous(), tok, 1.0, min(32, cols))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_place_holds_all_the_large(dtype):
    """Large values that fall to one thread in any interleaving of its pieces."""
    for cols in (40000, 131072):
        for step in (8, 16, 256, 1024, 2048, 4096, 8192):
            x, tok = make(1, cols, dtype, 3, 1.0)
            at = torch.arange(5, cols, step).cuda()
            x[0, at] = 20.0 + torch.arange(len(at)).cuda().to(dtype) % 64
            check_forward(x, tok, 1.0, 32)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 1000, 9000])
def test_masks(cols, dtype):
    x, tok = make(6, cols, dtype, 4)
    x[0, 1:] = -math.inf
    tok[0] = 0
    x[1] = -math.inf                       # nothing left
    x[2] = torch.finfo(dtype).min          # the lowest value everywhere: uniform
    x[3, 3:] = torch.finfo(dtype).min
    tok[3] = 2
    x[4, : cols // 2] = -math.inf
    tok[4] = 0                             # a masked token
    x[5] = torch.finfo(dtype).max
    got = check_forward(x, tok, 1.0, 8)
    assert float(got.log_prob[0]) == 0.0 and float(got.entropy[0]) == 0.0
    assert float(got.log_prob[4]) == -math.inf
    check_forward(x, tok, 0.3, 0)
    g = x.clone().requires_grad_()
    out = token_log_probs(g, tok, entropy=True, top=3)
    d, = torch.autograd.grad([out.log_prob, out.entropy], g, [torch.ones(6, device="cuda")] * 2)
    assert (d[1] == 0).all() and (d[0] == 0).all() and torch.isfinite(d).all()
    want, err = Ref(x).grad(tok, torch.ones(6, device="cuda"), torch.ones(6, device="cuda"))
    assert ((d.double() - want).abs() <= err + half_step(dtype) * (want.abs() + err) + tiny(dtype)).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [100, 1500, 70000])
def test_bad_rows(cols, dtype):
    """NaN, +inf, tokens outside and ignored ones stay in their rows."""
    x, tok = make(7, cols, dtype, 5)
    clean = x.clone()
    x[1, 7] = math.nan
    x[2, cols - 1] = math.inf
    tok[3], tok[4], tok[5] = cols, -100, -1
    x[4] = math.nan
    g = x.clone().requires_grad_()
    out = token_log_probs(g, tok, entropy=True, top=4)
    assert out.log_prob[[1, 2, 3, 5]].isnan().all() and out.entropy[[1, 2]].isnan().all()
    assert out.log_prob[4] == 0 and out.entropy[4] == 0 and (out.top_index[4] == -1).all() and (out.top_log_prob[4] == 0).all()
    d, = torch.autograd.grad(out.log_prob.nan_to_num().sum() + out.entropy.sum() * 0 + out.log_prob.sum(), g)
    assert (d[4] == 0).all() and d[[1, 2, 3, 5]].isnan().any(-1).all()
    good = [0, 6]
    # the same rows at the same addresses (another alignment of a row adds in another order)
    want = token_log_probs(clean, tok.clamp(0, cols - 1), entropy=True, top=4)
    for a, b in zip(out, want):
        assert torch.equal(a[good], b[good])
    assert torch.isfinite(d[good]).all()
    assert ((out.top_index >= -1) & (out.top_index < cols)).all()
    keep = token_log_probs(clean, tok.clamp(0, cols - 1), ignore_index=int(tok[6]))
    assert float(keep.log_prob[6]) == 0.0


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 100, 300, 1000, 1500])
def test_ignored_rows_have_no_gradient(cols, dtype):
    """Whatever an ignored row holds: its gradient is 0, and its neighbours' is what it is beside clean rows."""
    x, tok = make(20, cols, dtype, 13)
    fills = {1: [math.inf] * cols, 3: [-math.inf] * cols, 4: [math.nan] * cols, 6: [math.inf, math.nan] * (cols // 2), 9: [math.inf, -math.inf] * (cols // 2),
             10: [torch.finfo(dtype).max] * cols, 12: [torch.finfo(dtype).min] * cols, 19: None}
    bad = x.clone()
    for row, fill in fills.items():
        tok[row] = -100
        if fill is None:
            bad[row, cols - 1] = math.inf          # one logit that overflowed
        else:
            bad[row] = torch.tensor(fill)
    rng = torch.Generator().manual_seed(14)
    g, gh, gt = (torch.randn(*s, generator=rng).cuda() for s in ((20,), (20,), (20, 3)))
    for use in ((1, 0, 0), (0, 1, 0), (1, 1, 1)):
        grads = []
        for v in (bad, x):
            leaf = v.clone().requires_grad_()
            out = token_log_probs(leaf, tok, entropy=True, top=3)
            outs = [o for o, u in zip((out.log_prob, out.entropy, out.top_log_prob), use) if u]
            grads += torch.autograd.grad(outs, leaf, [t for t, u in zip((g, gh, gt), use) if u])
        assert not grads[0][list(fills)].any()     # neither a number nor NaN
        assert torch.equal(*grads) and grads[0].any()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [40, 200, 1000, 1500])
@pytest.mark.parametrize("T", [1e-6, 1e-3, 1e-2, 1e3])
def test_masked_columns_have_no_gradient(T, cols, dtype):
    """Masked by -inf or by the type's lowest value, at any temperature and any size of the entropy's gradient (a loss scale): 0 there,
    the formula's elsewhere. Logits are of the temperature's size, so that the distribution is not one column's. Results beyond the type
    are infinite as rounding makes them."""
    x, tok = make(12, cols, dtype, 15, 2.0)
    x = (x.float() * T).to(dtype)
    rng = torch.Generator().manual_seed(16)
    mask = (torch.rand(12, cols, generator=rng) < 0.3).cuda()
    mask[torch.arange(12), tok] = False
    x[mask] = -math.inf
    x[6:][mask[6:]] = torch.finfo(dtype).min
    g = torch.randn(12, generator=rng).cuda()
    r = Ref(x, T)
    edge = float(torch.finfo(dtype).max) * (1 + torch.finfo(dtype).eps / 4)
    for size in (1e-3, 1.0, 400.0, 65536.0):
        gh = torch.full((12,), size, device="cuda")
        for use in ((0, 1), (1, 1)):
            leaf = x.clone().requires_grad_()
            out = token_log_probs(leaf, tok, temperature=T, entropy=True)
            outs = [o for o, u in zip((out.log_prob, out.entropy), use) if u]
            d, = torch.autograd.grad(outs, leaf, [t for t, u in zip((g, gh), use) if u])
            assert not d[mask].any() and not d.isnan().any()
            want, err = r.grad(tok, g if use[0] else None, gh)
            near = (d.double() - want).abs() <= err + half_step(dtype) * (want.abs() + err) + tiny(dtype)
            assert (near | ((d.double() == torch.sign(want) * math.inf) & (want.abs() + err >= edge))).all()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (5, 31), (64, 256), (3, 1025), (700, 1000), (40, 4097), (2, 128001), (300, 8200)])
def test_backward(shape, dtype):
    x, tok = make(*shape, dtype, 6)
    R, V = shape
    k = min(7, V)
    rng = torch.Generator().manual_seed(7)
    g, gh, gt = (torch.randn(*s, generator=rng).cuda() for s in ((R,), (R,), (R, k)))
    for T in (1.0, 0.6):
        r = Ref(x, T)
        for use in ((1, 0, 0), (0, 1, 0), (1, 1, 0), (1, 1, 1), (0, 0, 1)):
            leaf = x.clone().requires_grad_()
            out = token_log_probs(leaf, tok, temperature=T, entropy=True, top=k if use[2] else 0)
            outs = [o for o, u in zip((out.log_prob, out.entropy, out.top_log_prob), use) if u]
            d, = torch.autograd.grad(outs, leaf, [t for t, u in zip((g, gh, gt), use) if u])
            assert d.dtype == dtype and d.shape == x.shape
            want, err = r.grad(tok, g if use[0] else None, gh if use[1] else None, out.top_index, gt if use[2] else None)
            assert ((d.double() - want).abs() <= err + half_step(dtype) * (want.abs() + err) + tiny(dtype)).all()


@gpu
def test_gradient_against_differences():
    x, tok = make(4, 50, torch.float32, 8)
    w = torch.randn(4, 3, generator=torch.Generator().manual_seed(9)).cuda()

    def f(v):       # in 64 bits, from the formula
        r = Ref(v, 0.8)
        return (w[:, 0] * r.log.gather(1, tok[:, None])[:, 0] + w[:, 1] * r.h
                + w[:, 2] * r.log.gather(1, x.argmax(-1)[:, None])[:, 0]).sum()
    leaf = x.clone().requires_grad_()
    out = token_log_probs(leaf, tok, temperature=0.8, entropy=True, top=1)
    d, = torch.autograd.grad((w[:, 0] * out.log_prob + w[:, 1] * out.entropy + w[:, 2] * out.top_log_prob[:, 0]).sum(), leaf)
    base, eps = x.double(), 1e-5
    for i, j in ((0, 3), (1, int(tok[1])), (2, 49), (3, int(x[3].argmax()))):
        hi, lo = base.clone(), base.clone()
        hi[i, j] += eps
        lo[i, j] -= eps
        assert abs(float((f(hi) - f(lo)) / (2 * eps)) - float(d[i, j])) < 1e-5


@gpu
def test_strides_shapes_and_streams():
    x, tok = make(24, 600, torch.bfloat16, 10)
    want = token_log_probs(x, tok, entropy=True, top=3)
    wide = torch.zeros(24, 701, dtype=torch.bfloat16, device="cuda")
    wide[:, 5:605] = x
    turned = x.t().contiguous().t()
    for v in (wide[:, 5:605], turned):
        for a, b in zip(token_log_probs(v, tok, entropy=True, top=3), want):
            # another alignment may add in another order
            assert torch.equal(a, b) if a.dtype == torch.int64 else torch.allclose(a, b, rtol=64 * U, atol=64 * U)
    cube = token_log_probs(x.view(2, 3, 4, 600), tok.view(2, 3, 4), entropy=True, top=3)
    assert cube.top_index.shape == (2, 3, 4, 3) and torch.equal(cube.log_prob.view(-1), want.log_prob)
    spread = torch.zeros(24, 2, dtype=torch.int64, device="cuda")
    spread[:, 0] = tok
    assert torch.equal(token_log_probs(x, spread[:, 0]).log_prob, want.log_prob)
    one = x[:1].expand(24, 600).requires_grad_()
    got = token_log_probs(one, tok).log_prob
    assert torch.equal(got, token_log_probs(x[:1].repeat(24, 1), tok).log_prob)
    assert token_log_probs(x[:0], tok[:0], entropy=True, top=2).top_index.shape == (0, 2)
    leaf = x[:0].clone().requires_grad_()
    assert torch.autograd.grad(token_log_probs(leaf, tok[:0]).log_prob.sum(), leaf)[0].shape == (0, 600)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = token_log_probs(x, tok, entropy=True, top=3)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(again, want))


@gpu
def test_rows_beyond_32_bits():
    """Row offsets past 2^31 elements."""
    cols = 1 << 20
    x = torch.zeros(2100, cols, dtype=torch.bfloat16, device="cuda")
    x[2099, 77] = 3.0
    x[2098, cols - 1] = 2.0
    tok = torch.full((2100,), 77, dtype=torch.int64, device="cuda")
    got = token_log_probs(x, tok, top=2)
    assert got.top_index[2099].tolist() == [77, 0] and got.top_index[2098].tolist() == [cols - 1, 0]
    assert abs(float(got.log_prob[2099]) - (3.0 - math.log(cols - 1 + math.exp(3.0)))) < 1e-4


@gpu
@pytest.mark.parametrize("shape", [(64, 256), (3, 60000)])
def test_graph(shape):
    x, tok = make(*shape, torch.float16, 11)
    leaf = x.clone()
    token_log_probs(leaf, tok, entropy=True, top=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = token_log_probs(leaf, tok, entropy=True, top=4)
        b = token_log_probs(leaf, tok, temperature=0.5)
    leaf.copy_(x.flip(-1))
    for _ in range(3):
        graph.replay()
    want = token_log_probs(x.flip(-1), tok, entropy=True, top=4)
    assert all(torch.equal(u, v) for u, v in zip(a, want))
    assert torch.equal(b.log_prob, token_log_probs(x.flip(-1), tok, temperature=0.5).log_prob)


@gpu
def test_autocast_free_and_modified_inputs():
    x, tok = make(4, 40, torch.float32, 12)
    leaf = x.clone().requires_grad_()
    y = leaf * 1.0
    out = token_log_probs(y, tok)
    y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.log_prob.sum().backward()


def test_refusals():
    x, tok = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int64)
    for bad in (x.double(), x.int()):
        with pytest.raises(TypeError, match="logits"):
            token_log_probs(bad, tok)
    with pytest.raises(TypeError, match="tokens"):
        token_log_probs(x, tok.float())
    with pytest.raises(ValueError, match="match"):
        token_log_probs(x, tok[:2])
    with pytest.raises(ValueError, match="columns"):
        token_log_probs(torch.zeros(3, 0), tok)
    for t in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            token_log_probs(x, tok, temperature=t)
    for top in (-1, 6, 33):
        with pytest.raises(ValueError, match="top"):
            token_log_probs(x, tok, top=top)
    with pytest.raises(ValueError, match="tensors on"):
        token_log_probs(x, torch.zeros(3, dtype=torch.int64, device="meta"))
    with pytest.raises(RuntimeError, match="CUDA"):
        token_log_probs(x, tok)
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            token_log_probs(fwAD.make_dual(x, torch.ones_like(x)), tok)
