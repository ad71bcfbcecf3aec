"""lora_linear and its gradients against the formula in 64 bits.

Tolerances, from the arithmetic of the kernels. One matrix instruction adds up to 17 terms aligned to the largest, each off by at most
2^-24 of it: 2^-20 of the running sum of magnitudes. A warp runs at most K / 64 + 2 of them for u, the tensor-core kernel (16-bit rows, ranks above 32) at most K / 16 (the 16-bit
products are exact; split fp32 ones are off by 2^-20), and the joins of warps and blocks add at most 16 roundings: so u is off by
(K / 64 + 20) 2^-20 sum |x| |A|, or K / 16 for K / 64.
(The gradients of fp16 rows above rank 16 split u and du by a power of two a rank: 2^-22 of each, or 2^-39 of the rank's largest, which
the instructions' 2^-20 of the sum of magnitudes covers where no row's share is 2^-19 of what its neighbours' largest would give it.)
In y each term of u counts with its own error, splitting u is off by 2^-21 (two tf32 numbers) or 2^-17 (two bf16 ones beside
bf16 rows), and at most 3 r / 8 + 2 instructions follow; the rounding to the type is half a step. The gradients are the same sums with other operands; rows of an adapter take the place of K.
Inputs of one sign make the sums of magnitudes the sums themselves."""
import math

import pytest
import torch
import torch.nn as nn

from rl_quant_b200 import LoRALinear, lora_linear, swap
from rl_quant_b200 import lora as lora_mod

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
S = 2.0 ** -20


def half_step(t):
    return 2.0 ** -24 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(m, k, n, r, L, dtype, seed, sign=False, base=True, index="mixed"):
    g = torch.Generator().manual_seed(seed)

    def rnd(*s):
        v = torch.randn(*s, generator=g)
        return v.abs() if sign else v
    x, a, b = rnd(m, k).to(dtype).cuda(), (rnd(L, r, k) / math.sqrt(k)).to(dtype).cuda(), (rnd(L, n, r) * 0.1).to(dtype).cuda()
    base = rnd(m, n).to(dtype).cuda() if base else None
    scale = (0.5 + torch.rand(L, generator=g)).cuda()
    if index is None:
        i = None
    elif index == "one":
        i = torch.full((m,), L - 1, dtype=torch.int64, device="cuda")
    else:
        i = torch.randint(-1, L, (m,), generator=g)
        i = (i.sort().values if index == "runs" else i).cuda()
    return x, a, b, i, scale, base, rnd(m, n).to(dtype).cuda()


def ref(x, a, b, i, scale, base, dy):
    """((y, bound), (dx, bound), (da, bound), (db, bound)); the bounds are of what precedes the last rounding."""
    D = torch.float64
    m, k = x.shape
    L, r, _ = a.shape
    n = b.shape[1]
    new = lambda *s: torch.zeros(*s, dtype=D, device="cuda")  # noqa: E731
    out = [[new(m, n), new(m, n)], [new(m, k), new(m, k)], [new(L, r, k), new(L, r, k)], [new(L, n, r), new(L, n, r)]]
    if base is not None:
        out[0][0] += base.to(D)
        out[0][1] += base.to(D).abs() * S
    for j in range(L):
        rows = torch.arange(m, device="cuda") if i is None else (i == j).nonzero()[:, 0]
        if not len(rows):
            continue
        X, A, B, G = x[rows].to(D), a[j].to(D), b[j].to(D), dy[rows].to(D)
        s = float(scale[j]) if isinstance(scale, torch.Tensor) else scale
        U, V = s * X @ A.T, s * G @ B
        U1, V1 = s * X.abs() @ A.abs().T, s * G.abs() @ B.abs()
        per = 16 if r > 32 and x.dtype != torch.float32 else 64
        eU, eV = (k / per + 21) * S * U1, (n / per + 21) * S * V1
        split = 8 if x.dtype == torch.bfloat16 else 1
        more, many = (3 * r / 8 + 2 + split) * S, (3 * len(rows) / 8 + 19 + split) * S
        out[0][0][rows] += U @ B.T
        out[0][1][rows] += (eU + more * U.abs()) @ B.abs().T
        out[1][0][rows] = V @ A
        out[1][1][rows] = (eV + more * V.abs()) @ A.abs()
        out[2][0][j], out[2][1][j] = V.T @ X, (eV + many * V.abs()).T @ X.abs()
        out[3][0][j], out[3][1][j] = G.T @ U, G.abs().T @ (eU + many * U.abs())
    return out


def close(got, want, dtype):
    value, bound = want
    assert got.dtype == dtype and got.shape == value.shape
    tol = bound + half_step(dtype) * (value.abs() + bound) + tiny(dtype)
    # From half a step above the type's largest number on (fp16: 65520) rounding to nearest gives infinity: expected there, and allowed
    # where the bound reaches that far.
    edge = float(torch.finfo(dtype).max) * (1 + torch.finfo(dtype).eps / 4)
    infinite = got.double() == torch.sign(value) * math.inf
    assert infinite[value.abs() - bound > edge].all()
    value = torch.where(infinite & (value.abs() + bound >= edge), got.double(), value)
    off = torch.where(got.double() == value, 0.0, (got.double() - value).abs() - tol)
    worst = off.max() if got.numel() else torch.tensor(0.0)
    assert float(worst) <= 0.0, float(worst)


def check(x, a, b, i, scale, base, dy, back=True):
    want = ref(x, a, b, i, scale, base, dy)
    y = lora_linear(x, a, b, i, scale, base)
    close(y, want[0], x.dtype)
    if i is not None and base is not None:
        assert torch.equal(y[i < 0], base[i < 0])
    if not back:
        return y
    leaves = [t.detach().clone().requires_grad_() for t in (x, a, b)]
    bl = None if base is None else base.clone().requires_grad_()
    y2 = lora_linear(*leaves, i, scale, bl)
    close(y2.detach(), want[0], x.dtype)
    grads = torch.autograd.grad(y2, leaves + ([] if bl is None else [bl]), dy)
    for g, w in zip(grads, want[1:]):
        close(g, w, x.dtype)
    if bl is not None:
        assert torch.equal(grads[3], dy)
    return y


# rows, inputs, outputs, rank, adapters: one token to many, ranks at and off the tile sizes, sizes off every vector
SIZES = [(1, 64, 64, 16, 1), (1, 4096, 512, 16, 3), (5, 1, 1, 1, 2), (7, 33, 65, 3, 2), (16, 256, 128, 8, 1), (17, 128, 256, 4, 4),
         (64, 512, 1024, 16, 64), (33, 96, 64, 32, 2), (40, 1002, 777, 9, 5), (256, 264, 136, 24, 3), (257, 64, 72, 64, 3),
         (300, 200, 320, 48, 1), (300, 72, 64, 100, 2), (130, 128, 128, 128, 2), (1000, 48, 40, 16, 130), (2050, 520, 264, 16, 2),
         (600, 1024, 1024, 33, 1),
         (8192, 32, 24, 16, 512), (4096, 32, 24, 16, 512), (4097, 40, 24, 8, 3), (8200, 24, 32, 8, 7), (400, 16, 16, 16, 600), (1500, 64, 64, 64, 3),
         # high ranks: one and several tiles of any height, odd counts of chunks and of columns, empty adapters (TC_SIZES below are
         # those that the tensor-core kernel takes)
         (64, 64, 64, 64, 1), (129, 72, 136, 40, 1), (700, 4096, 264, 64, 2), (300, 520, 1032, 128, 1), (2000, 1000, 504, 96, 9),
         (513, 2048, 2048, 128, 4), (3000, 192, 320, 80, 3), (1024, 64, 64, 64, 1), (1025, 72, 136, 40, 1), (1300, 4096, 264, 64, 2), (1300, 64, 64, 64, 1), (1297, 72, 136, 40, 1),
         (1300, 520, 1032, 128, 1), (1030, 128, 640, 128, 16), (9000, 64, 48, 64, 3), (5000, 520, 264, 24, 1),
         (700, 1032, 264, 32, 40), (1000, 776, 1000, 128, 3),
         # as many rows and ranks, off the 16 bytes
         (1200, 72, 64, 100, 2), (1300, 73, 65, 64, 2), (1330, 70, 68, 40, 3),
         (4100, 136, 72, 128, 5), (128, 96, 72, 16, 4), (256, 72, 64, 64, 3), (200, 73, 64, 16, 2), (4100, 70, 72, 100, 2), (1100, 4096, 4096, 72, 3)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_sizes(size, dtype):
    m, k, n, r, L = size
    for seed, (sign, base, index) in enumerate(((True, False, "mixed"), (False, True, "runs"), (False, True, "one"))):
        if index == "one" and L == 1:
            index = None
        check(*make(m, k, n, r, L, dtype, seed, sign, base, index))


# Calls that the tensor-core kernel takes, forward and backward: few and many adapters (some without rows), ranks that are no power of two, inputs and outputs
# of several chunks of 128 and a rest, or of less than one.
TC_SIZES = [(4100, 136, 72, 80, 9), (4096, 264, 392, 96, 16), (5200, 648, 904, 128, 40), (4200, 72, 136, 104, 1), (1100, 4096, 4096, 128, 2),
            (1030, 4104, 4104, 96, 3), (4099, 2184, 136, 72, 12), (8000, 136, 1544, 128, 33), (4224, 128, 128, 120, 66),
            (1300, 392, 264, 64, 9), (2700, 1032, 776, 56, 40), (1500, 8, 8, 40, 5), (1280, 1000, 1160, 48, 20), (1177, 264, 136, 64, 1)]


def test_sizes_of_the_tensor_core_kernel():
    """The workspace of the backward pass, for the adapters transposed, tells which kernel takes a call."""
    from rl_quant_b200 import _native as N
    size = N.load().glad_lora_backward_workspace_size
    for m, k, n, r, L in TC_SIZES:
        for code in (N.DTYPE_F16, N.DTYPE_BF16):
            assert size(m, k, n, L, r, code, L > 1) == 2 * L * r * (k + n)
        assert size(m, k, n, L, r, N.DTYPE_F32, L > 1) == 0
    # the borders: rows, rank, rows an adapter, ranks off 8
    few, many = 1024, 4096
    for at in ((1160, 72, 72, 64, 1), (few, 4096, 4000, 128, 1), (many - 1, 136, 72, 128, 1), (1300, 72, 72, 32, 1), (2700, 72, 72, 64, 43),
               (4100, 72, 72, 100, 1)):
        m, k, n, r, L = at
        assert size(m, k, n, L, r, N.DTYPE_BF16, L > 1) == 0, at


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", TC_SIZES)
def test_tensor_core_kernel(size, dtype):
    m, k, n, r, L = size
    for seed, (sign, base, index) in enumerate(((True, False, "mixed"), (False, True, "runs"), (False, True, "one"))):
        if L == 1:
            index = None
        data = make(m, k, n, r, L, dtype, 20 + seed, sign, base, index)
        if index == "mixed" and L > 4:
            data[3][data[3] % 3 == 1] = 0                # a third of the adapters without rows
        check(*data)


@gpu
@pytest.mark.parametrize("size", [(64, 16384, 24, 8, 1), (70, 16381, 25, 40, 2), (40, 24, 16384, 8, 1), (20000, 8192, 8, 16, 1)])
def test_long_sums_of_float32(size):
    """Sums of thousands of terms of one sign, as a relative norm. The instruction cuts its sum off, so every bit that a long chain of them loses has the
    same sign; 16 terms at most (6 instructions, 2^-23 of their own sum each, and 4 * 2^-23 for the split operands) are summed that way
    and added by rounding, which has no sign: n independent roundings of 2^-24 at most are 2^-24 sqrt(n), of which six are allowed.
    n: a warp's steps of 8 terms, and the joins. Every output is two sums after the other."""
    m, k, n, r, L = size
    data = make(m, k, n, r, L, torch.float32, 30, sign=True, base=False, index=None if L == 1 else "mixed")
    want = [w for w, _ in ref(*data)]
    x, a, b, i, scale, _, dy = data
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = lora_linear(*leaves, i, scale)
    longest = max(m, k, n)
    bound = 2 * (10 * 2.0 ** -23 + 6 * math.sqrt(longest / 64 + 16) * 2.0 ** -24)
    for got, w in zip((y.detach(), *torch.autograd.grad(y, leaves, dy)), want):
        assert float((got.double() - w).norm() / w.norm()) <= bound


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    x, a, b, i, scale, base, dy = make(50, 128, 96, 16, 3, dtype, 4)
    want = lora_linear(x, a, b, i, scale, base)
    wide = torch.zeros(50, 300, dtype=dtype, device="cuda")
    wide[:, 8:136] = x
    wide2 = torch.zeros(50, 201, dtype=dtype, device="cuda")
    wide2[:, 3:99] = base
    # rows off the 16-byte boundaries are added up by another kernel, in another order
    for xs, bs in ((wide[:, 8:136], base), (x, wide2[:, 3:99]), (x.t().contiguous().t(), base.t().contiguous().t())):
        close(lora_linear(xs, a, b, i, scale, bs), ref(x, a, b, i, scale, base, dy)[0], dtype)
    more = torch.zeros(50, 304, dtype=dtype, device="cuda")
    more[:, 8:136] = x
    assert torch.equal(lora_linear(more[:, 8:136], a, b, i, scale, base), want)      # on them: the same
    wide[:, 3:131] = x
    close(lora_linear(wide[:, 3:131], a, b, i, scale, base), ref(x, a, b, i, scale, base, dy)[0], dtype)
    turned = a.transpose(1, 2).contiguous().transpose(1, 2)
    spread = torch.zeros(50, 2, dtype=torch.int32, device="cuda")
    spread[:, 1] = i
    assert torch.equal(lora_linear(x, turned, b, spread[:, 1], scale, base), want)
    cube = lora_linear(x.view(5, 10, 128), a, b, i.view(5, 10), scale, base.view(5, 10, 96))
    assert cube.shape == (5, 10, 96) and torch.equal(cube.view(50, 96), want)
    one = x[:1].expand(50, 128)
    close(lora_linear(one, a, b, i, scale, base), ref(one, a, b, i, scale, base, dy)[0], dtype)
    for leaf, args in ((x.clone().requires_grad_(), ()),):
        y = lora_linear(leaf, a, b, i, scale, base)
        g, = torch.autograd.grad(y, leaf, dy.t().contiguous().t())
        close(g, ref(x, a, b, i, scale, base, dy)[1], dtype)
        g, = torch.autograd.grad(lora_linear(leaf, a, b, i, scale, base).sum(), leaf)
        close(g, ref(x, a, b, i, scale, base, torch.ones_like(dy))[1], dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [20, 400])
def test_index(m, dtype):
    """Outside 0..L-1: no adapter. Adapters without rows: zero gradients. A number as scale."""
    x, a, b, i, scale, base, dy = make(m, 64, 48, 8, 6, dtype, 5)
    i = i.clone()
    i[i == 2] = 3
    i[0], i[1], i[2] = 6, -7, 2 ** 40
    clean = torch.where((i < 0) | (i > 5), -1, i)
    y = check(x, a, b, clean, scale, base, dy)
    assert torch.equal(lora_linear(x, a, b, i, scale, base), y)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    dx, da, db = torch.autograd.grad(lora_linear(*leaves, i, scale, base), leaves, dy)
    assert not dx[:3].any() and not da[2].any() and not db[2].any()
    none = torch.full_like(i, -1)
    assert torch.equal(lora_linear(x, a, b, none, scale, base), base)
    assert not lora_linear(x, a, b, none, scale).any()
    close(lora_linear(x, a, b, clean, 0.75, base), ref(x, a, b, clean, 0.75, base, dy)[0], dtype)
    # rows alone give what they give together, up to the order of the sums
    for j in (3, m - 1):
        close(lora_linear(x[j:j + 1], a, b, i[j:j + 1], scale, base[j:j + 1]),
              [t[j:j + 1] for t in ref(x, a, b, clean, scale, base, dy)[0]], dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(70, 64, 96, 16, 3), (1300, 64, 96, 64, 3), (4100, 520, 72, 128, 1)])
def test_some_gradients_only(size, dtype):
    x, a, b, i, scale, base, dy = make(*size, dtype, 6, index=None if size[4] == 1 else "mixed")
    want = ref(x, a, b, i, scale, base, dy)[1:]
    for use in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
        leaves = [t.clone().requires_grad_(bool(u)) for t, u in zip((x, a, b), use)]
        y = lora_linear(*leaves, i, scale, base)
        for g, w in zip(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy), [w for w, u in zip(want, use) if u]):
            close(g, w, dtype)
    bl = base.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(lora_linear(x, a, b, i, scale, bl), bl, dy)[0], dy)


@gpu
@pytest.mark.parametrize("r", [16, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_keep_to_themselves(dtype, r):
    """A NaN or an infinity in a row of x or of base stays in that row; in an adapter, in its rows."""
    x, a, b, i, scale, base, dy = make(90, 96, 80, 16, 4, dtype, 7) if r == 16 else make(1290, 96, 80, r, 4, dtype, 7)
    want = lora_linear(x, a, b, i, scale, base)
    i[5], i[9] = 1, -1
    want = lora_linear(x, a, b, i, scale, base)
    bad = x.clone()
    bad[5, 3] = math.nan
    bad[9] = math.inf                      # a row without an adapter
    got = lora_linear(bad, a, b, i, scale, base)
    keep = torch.ones(len(x), dtype=torch.bool)
    keep[5] = False
    assert torch.equal(got[keep], want[keep]) and got[5].isnan().all()
    ab = a.clone()
    ab[2] = math.nan
    got = lora_linear(x, ab, b, i, scale, base)
    assert torch.equal(got[i != 2], want[i != 2]) and got[i == 2].isnan().all()
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    g = dy.clone()
    g[5] = math.nan
    dx, da, db = torch.autograd.grad(lora_linear(*leaves, i, scale, base), leaves, g)
    assert torch.isfinite(dx[keep]).all() and torch.isfinite(da[[0, 2, 3]]).all() and torch.isfinite(db[[0, 2, 3]]).all()
    assert dx[5].isnan().all() and da[1].isnan().all()


@gpu
@pytest.mark.parametrize("size", [(90, 96, 80, 16), (90, 97, 81, 15), (300, 96, 80, 128), (300, 96, 80, 72),
                                  (1290, 96, 80, 64), (1290, 96, 80, 40), (4130, 96, 80, 128), (4130, 96, 80, 104)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_infinities_of_16_bit_rows(size, dtype):
    """Positive numbers with an infinity in a row of x and in one of dy: infinite, not NaN, where u and du are, although they are taken as
    pairs of 16-bit numbers; the other rows and adapters as without."""
    m, k, n, r = size
    x, a, b, i, scale, base, dy = make(m, k, n, r, 3, dtype, 17, sign=True)
    a, b = a + 2.0 ** -10, b + 2.0 ** -10                # no zeros, which times an infinity are NaN
    x, dy = x + 2.0 ** -10, dy + 2.0 ** -10
    i[5], i[7] = 1, 2
    clean = [t.clone().requires_grad_() for t in (x, a, b)]
    want = lora_linear(*clean, i, scale, base)
    want = [want.detach(), *torch.autograd.grad(want, clean, dy)]
    x, dy = x.clone(), dy.clone()
    x[5, 3] = math.inf
    dy[7, 4] = math.inf
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    y = lora_linear(*leaves, i, scale, base)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    for j, (g, w) in enumerate(zip(got, want)):
        hit, past = torch.zeros_like(g, dtype=torch.bool), torch.zeros_like(g, dtype=torch.bool)
        if j < 2:
            hit[5 + 2 * j] = True                        # y of the one row, dx of the other
        elif j == 2:
            hit[2], past[1, :, 3] = True, True           # du of row 7; the column of x, times a pair that may have both signs
        else:
            hit[1], past[2, 4] = True, True              # u of row 5; the column of dy
        assert (g[hit] == math.inf).all() and not torch.isfinite(g[past]).any(), j
        hit |= past
        assert torch.equal(g[~hit], w[~hit]), j


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_repeats_streams_and_graphs(dtype):
    for m, r in ((30, 16), (700, 16), (700, 64), (1300, 64)):
        x, a, b, i, scale, base, dy = make(m, 256, 192, r, 5, dtype, 8)
        leaves = [t.clone().requires_grad_() for t in (x, a, b)]

        def once():
            y = lora_linear(*leaves, i, scale, base)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))
        first = once()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            again = once()
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(u, v) for u, v in zip(first, again))
        moving = i.clone()
        with torch.no_grad():
            lora_linear(x, a, b, moving, scale, base)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y1 = lora_linear(x, a, b, moving, scale, base)
                y2 = lora_linear(x, a, b, moving, 2.0)
            moving.copy_(i.flip(0))
            for _ in range(2):
                graph.replay()
            assert torch.equal(y1, lora_linear(x, a, b, i.flip(0), scale, base))
            assert torch.equal(y2, lora_linear(x, a, b, i.flip(0), 2.0))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,r", [(300, 16), (1300, 64), (9000, 32)])
def test_captured_training(m, r, dtype):
    """Forward and backward pass in one graph, replayed twice on other rows, adapters and gradients; two graphs of one pool in turn."""
    x, a, b, i, scale, base, dy = make(m, 136, 72, r, 3, dtype, 13)
    x2, a2, b2, i2, _, base2, dy2 = make(m, 136, 72, r, 3, dtype, 14)

    def once(x, a, b, i, base, dy):
        leaves = [t.clone().requires_grad_() for t in (x, a, b)]
        y = lora_linear(*leaves, i, scale, base)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    held = [t.clone() for t in (x, a, b, i, base, dy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once(*held)
    torch.cuda.current_stream().wait_stream(s)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once(*held)
    with torch.cuda.graph(other, pool=graph.pool()):
        got2 = once(*held)
    for given in ((x2, a2, b2, i2, base2, dy2), (x, a, b, i, base, dy)):
        for h, t in zip(held, given):
            h.copy_(t)
        want = once(*given)
        for g, outs in ((graph, got), (graph, got), (other, got2)):
            g.replay()
            assert all(torch.equal(u, v) for u, v in zip(outs, want))


@gpu
@pytest.mark.parametrize("m,r", [(300, 16), (1300, 64), (4100, 128)])
def test_two_at_once(m, r):
    """Calls on two streams whose kernels share the GPU."""
    sets = [make(m, 520, 264, r, 3, torch.bfloat16, 15 + j) for j in range(2)]

    def once(x, a, b, i, scale, base, dy):
        leaves = [t.clone().requires_grad_() for t in (x, a, b)]
        y = lora_linear(*leaves, i, scale, base)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = [once(*q) for q in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(once(*sets[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for g in got[j]:
            assert all(torch.equal(u, v) for u, v in zip(g, want[j]))


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ranges_of_the_split(dtype):
    """Rows of u of very different magnitudes, and of one large number beside small ones: rows keep their relative accuracy."""
    for m, r in ((40, 16), (300, 64), (300, 128), (1300, 64), (4130, 128)):
        x, a, b, i, scale, base, dy = make(m, 256, 128, r, 1, dtype, 11, sign=True, base=False, index=None)
        x = x * torch.logspace(-3, 2, m).to(dtype).cuda()[:, None]
        a = a.clone()
        a[:, 1::2] *= 2.0 ** -9
        check(x, a, b, i, scale, base, dy * torch.logspace(0, -3, m).to(dtype).cuda()[:, None])


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_waits_that_run_out(dtype):
    """Arrivals that never come (a host switch) and a limit of a millisecond: the kernel gives up, says so in the status word, and
    the next calls are what they were."""
    from rl_quant_b200 import DeviceStatusError, w4_status
    from rl_quant_b200 import _native as N
    lib = N.load()
    x, a, b, i, scale, base, dy = make(1300, 512, 384, 64, 2, dtype, 12)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]

    def once():
        y = lora_linear(*leaves, i, scale, base)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    want = once()
    assert w4_status() == 0
    N.check(lib.glad_debug_lora_wait(1, 1_000_000))
    try:
        once()
        torch.cuda.synchronize()
    finally:
        N.check(lib.glad_debug_lora_wait(0, 0))
    with pytest.raises(DeviceStatusError):
        w4_status()
    assert w4_status() == 0
    for _ in range(2):
        assert all(torch.equal(u, v) for u, v in zip(once(), want))
    assert w4_status() == 0


@gpu
def test_gradients_against_differences():
    x, a, b, i, scale, base, dy = make(9, 20, 12, 4, 2, torch.float32, 9)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    grads = torch.autograd.grad(lora_linear(*leaves, i, scale, base), leaves, dy)
    data = [t.double() for t in (x, a, b)]

    def f(x_, a_, b_):
        total = 0.0
        for m in range(9):
            j = int(i[m])
            if j >= 0:
                total = total + (float(scale[j]) * (b_[j] @ (a_[j] @ x_[m])) * dy[m].double()).sum()
        return total
    for t in range(3):
        for at in ((0,) * data[t].dim(), tuple(v - 1 for v in data[t].shape)):
            hi, lo = [v.clone() for v in data], [v.clone() for v in data]
            hi[t][at] += 1e-4
            lo[t][at] -= 1e-4
            d = float(f(*hi) - f(*lo)) / 2e-4 if not isinstance(f(*hi), float) else 0.0
            assert abs(d - float(grads[t][at])) < 1e-4 * (1 + abs(d))


@gpu
def test_empty_and_large_offsets():
    x, a, b, i, scale, base, dy = make(4, 64, 64, 16, 2, torch.bfloat16, 10)
    assert lora_linear(x[:0], a, b, i[:0], scale, base[:0]).shape == (0, 64)
    leaves = [t.clone().requires_grad_() for t in (x[:0], a, b)]
    dx, da, db = torch.autograd.grad(lora_linear(*leaves, i[:0], scale).sum(), leaves)
    assert dx.shape == (0, 64) and not da.any() and not db.any()
    # rows whose offsets pass 2^31 elements
    m = 70000
    big = torch.zeros(m, 32768, dtype=torch.bfloat16, device="cuda")
    big[m - 1] = 1.0
    one = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for r in (16, 64):
        a, b = one(1, r, 32768) * 2.0 ** -15, one(1, 64, r)
        y = lora_linear(big, a, b)
        assert (y[m - 1] == r).all() and not y[:m - 1].any()
        leaf = a.clone().requires_grad_()
        da, = torch.autograd.grad(lora_linear(big, leaf, b), leaf, one(m, 64))
        assert (da == 64.0).all()
    # outputs whose offsets do
    for r in (16, 64):
        y = lora_linear(big[:, :64], one(1, r, 64) / 64, one(1, 32768, r), base=big)
        assert (y[m - 1] == r + 1).all() and not y[:m - 1].any()


FIRST_CALLS = """
import sys, threading
import torch
sys.path.insert(0, ".")
from rl_quant_b200 import lora_linear
sets = []
for L in (16384, 600, 1023, 4095):
    g = torch.Generator().manual_seed(L)
    x, a, b = torch.randn(5000, 16, generator=g).cuda(), torch.randn(L, 4, 16, generator=g).cuda(), torch.randn(L, 8, 4, generator=g).cuda()
    i = torch.randint(-1, L, (5000,), generator=g).cuda()
    j = i.clamp(min=0)
    want = torch.einsum("mnr,mr->mn", b[j].double(), torch.einsum("mrk,mk->mr", a[j].double(), x.double())) * (i >= 0)[:, None]
    sets.append((x, a, b, i, want))
torch.cuda.synchronize()
gate, bad = threading.Barrier(len(sets)), []
def work(x, a, b, i, want):
    try:
        gate.wait()
        for _ in range(3):
            assert torch.allclose(lora_linear(x, a, b, i).double(), want, rtol=1e-4, atol=1e-4)
    except Exception as e:
        bad.append(repr(e))
for order in range(2):
    threads = [threading.Thread(target=work, args=s) for s in sets]
    [t.start() for t in threads]
    [t.join() for t in threads]
assert not bad, bad
"""


@gpu
def test_first_calls_of_several_threads():
    """The shared memory that the plan's kernel is allowed does not depend on which thread's first call comes last: in a process of its
    own, four threads whose calls need between 79 and 197 KB."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=root, check=True, timeout=300)


def net(dtype, device):
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(96, 128), nn.ELU(), nn.Linear(128, 64)).to(device=device, dtype=dtype)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_module_over_4_bit_layers(dtype):
    m = net(dtype, "cuda")
    plain = net(dtype, "cuda")
    q = swap.apply(m, {"0": {"bits": 4, "group": 32}, "2": {"bits": 4, "group": 32}})
    x = torch.randn(40, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    with torch.no_grad():
        before = m(x)
    layers = swap.apply_lora(m, ["0", "2"], rank=8, adapters=3, alpha=16)
    index = torch.arange(40, device="cuda") % 4 - 1
    swap.select_lora(layers, index)
    with torch.no_grad():
        assert torch.equal(m(x), before)                 # new adapters change nothing
        for mod in layers.values():
            mod.lora_b.normal_(std=0.05)
        y = m(x)
        assert torch.equal(y[index < 0], before[index < 0]) and not torch.equal(y, before)
        for j in range(3):
            swap.select_lora(layers, j)
            assert torch.allclose(m(x)[index == j].float(), y[index == j].float(), rtol=2 ** -6, atol=2 ** -6)
        swap.select_lora(layers, None)
        assert torch.equal(m(x), before)
    swap.select_lora(layers, index)
    out = m(x)                                           # training: the source layers' own weights below
    out.float().square().sum().backward()
    assert all(mod.lora_a.grad is not None and mod.lora_b.grad is not None for mod in layers.values())
    assert all(mod.base.weight.grad is None for mod in layers.values())
    swap.restore_lora(m, layers)
    assert m[0] is q["0"]
    swap.restore(m, q)
    assert torch.equal(m[0].weight, plain[0].weight)


@gpu
@pytest.mark.parametrize("mode", ["eager", "manual-graph"])
def test_runner_with_adapters(mode):
    """InferenceRunner over a policy with adapters on a plain and on a 4-bit layer: sync_weights_from masters without and with
    adapters, and the actions are those of the policy itself."""
    from rl_quant_b200 import InferenceRunner, build_glad
    from rl_quant_b200.synthetic import glad_obs
    paths = ["actor.0", "actor.2"]

    def policy(seed, dtype):
        torch.manual_seed(seed)
        return build_glad().cuda().to(dtype).eval()
    copy = policy(0, torch.float16)
    swap.apply(copy, {"actor.0": {"bits": 4, "group": 32}})
    layers = swap.apply_lora(copy, paths, rank=8, adapters=3)
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(copy, mode=mode)
    obs = glad_obs(33, seed=1).cuda().half()
    task = torch.arange(33, device="cuda") % 4 - 1
    swap.select_lora(layers, task)
    for seed in (1, 2):
        master = policy(seed, torch.float32)
        run.sync_weights_from(master)
        for p in paths:
            mine, theirs = copy.get_submodule(p).base, master.get_submodule(p)
            assert torch.equal(mine.weight, theirs.weight.half()) and torch.equal(mine.bias, theirs.bias.half())
        lin = nn.Linear(224, 512).cuda().half()
        lin.weight.data.copy_(master.actor[0].weight)
        assert torch.equal(copy.actor[0].base.tiles, swap.W4Linear(lin, 32).tiles)
        with torch.no_grad():
            assert torch.equal(run.act(obs), copy.act_inference({"policy_obs": obs})[0])
    master = policy(3, torch.float32)
    for mod in swap.apply_lora(master, paths, rank=8, adapters=3).values():
        nn.init.normal_(mod.lora_b, std=0.1)
    with pytest.warns(UserWarning):
        run = InferenceRunner(copy, mode=mode)
    run.sync_weights_from(master)
    assert torch.equal(copy.actor[0].lora_b, master.actor[0].lora_b.half())
    assert torch.equal(copy.actor[2].base.weight, master.actor[2].base.weight.half())
    with torch.no_grad():
        first = run.act(obs).clone()
        assert torch.equal(first, copy.act_inference({"policy_obs": obs})[0])
        task.copy_(task.flip(0))                       # read at every call, a captured one too
        second = run.act(obs).clone()
        assert torch.equal(second, copy.act_inference({"policy_obs": obs})[0]) and not torch.equal(first, second)
    run.check_status()
    with pytest.warns(UserWarning):
        bare = InferenceRunner(policy(0, torch.float16), mode=mode)
    with pytest.raises(ValueError, match="adapters"):
        bare.sync_weights_from(master)


@gpu
@pytest.mark.parametrize("path", ["topk_scorer", "global_pool_selector", "critic_proprio_embedding", "query_projector",
                                  "actor_proprio_embedding"])
def test_adapters_over_the_encoder(path, golden_weights):
    """Layers that the fused forwards and the patched encoder read themselves: with adapters the policy runs op by op, and the adapters count, in
    the rollout and in the update."""
    from gpu_util import golden_model
    from rl_quant_b200 import InferenceRunner
    from rl_quant_b200.fused import FusedActor, FusedCritic, FusedUnsupported
    from rl_quant_b200.synthetic import glad_obs_pair
    m, _ = golden_model(golden_weights)
    po, co = (t.cuda().half() for t in glad_obs_pair(12, seed=3))
    heads = [(m.actor, po), (m.critic, co)]
    with torch.no_grad():
        before = [f(m._encode_terrain_orig(o)[0]) for f, o in heads]
    layers = swap.apply_lora(m, [path], rank=4)
    nn.init.normal_(layers[path].lora_b, std=0.5)
    adapted = [path != "critic_proprio_embedding", path != "actor_proprio_embedding"]      # the observation groups that it encodes
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(m, mode="eager", with_critic=True)
    assert [run._fused is None, run._fused_critic is None] == adapted
    with torch.no_grad():
        want = [f(m._encode_terrain_orig(o)[0]) for f, o in heads]
        assert [not torch.equal(a, b) for a, b in zip(want, before)] == adapted
        for got in ([run.act(po), run.evaluate(co)], [f(m._encode_terrain(o)[0]) for f, o in heads]):
            assert all(torch.equal(a, b) for a, b, on in zip(got, want, adapted) if on)
    make = FusedCritic if path == "critic_proprio_embedding" else FusedActor
    with pytest.raises(FusedUnsupported):
        make(m, need_mlp=False)
    # the update: a gradient for the adapters (the scorer has one in train mode only)
    m.train()
    m.map_cnn.eval()
    f, o = heads[path == "critic_proprio_embedding"]
    f(m._encode_terrain(o)[0]).float().square().sum().backward()
    assert layers[path].lora_a.grad is not None and layers[path].lora_b.grad.any()


@gpu
@pytest.mark.parametrize("mode", ["eager", "manual-graph", "max-autotune"])
def test_runner_follows_the_selection(mode):
    """Numbers, index tensors and none, selected between calls of one runner: each call is of the adapters selected then. New values in the
    same tensor need no new capture."""
    from rl_quant_b200 import InferenceRunner, build_glad
    from rl_quant_b200.synthetic import glad_obs_pair
    torch.manual_seed(0)
    m = build_glad().cuda().half().eval()
    layers = swap.apply_lora(m, ["actor.0", "critic.2"], rank=8, adapters=3)
    for mod in layers.values():
        nn.init.normal_(mod.lora_b, std=0.1)
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(m, mode=mode, with_critic=True)
    po, co = (t.cuda().half() for t in glad_obs_pair(10, seed=5))
    host = po.cpu().pin_memory()
    task = torch.tensor([0, 1, 2, -1, 0], device="cuda").repeat(2)
    seen = []
    for index in (0, 2, task, task.flip(0).contiguous(), task.int(), None, 2, task):
        swap.select_lora(layers, index)
        with torch.no_grad():
            want = m.act_inference({"policy_obs": po})[0], m.evaluate(co)
        got = run.act(po).clone(), run.evaluate(co).clone()
        out = run.act_host(host)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(out, want[0].float().cpu())
        seen.append(want[0].clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[2], seen[3]) and torch.equal(seen[1], seen[6])
    graphs = len(run._graphs)
    task.copy_(task.flip(0))
    assert torch.equal(run.act(po), seen[3]) and len(run._graphs) == graphs


@gpu
def test_adapters_over_the_encoder_take_float32_observations(golden_weights):
    """As the fused encoder does: the rows are rounded to the copy's type."""
    from gpu_util import golden_model
    from rl_quant_b200 import InferenceRunner
    from rl_quant_b200.synthetic import glad_obs_pair
    m, _ = golden_model(golden_weights)
    nn.init.normal_(swap.apply_lora(m, ["topk_scorer"], rank=4)["topk_scorer"].lora_b, std=0.5)
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(m, mode="manual-graph", normalize=False)
    po, co = (t.cuda() for t in glad_obs_pair(12, seed=3))
    assert torch.equal(run.act(po), run.act(po.half()))
    with torch.no_grad():
        for o in (po, co):
            assert all(torch.equal(a, b) for a, b in zip(m._encode_terrain(o), m._encode_terrain(o.half())))


@gpu
@pytest.mark.parametrize("paths", [["actor.4"], ["actor.0", "actor.6"], ["critic.2"]])
def test_adapters_over_the_quantised_policy(paths, golden_weights):
    """The int8 policy with adapters over QuantLinear layers of its MLP (or over the critic's): the fused encoder still runs, the MLP op by
    op, in the rollout and in the update; weights synchronised from a master are requantised below the adapters."""
    from gpu_util import golden_model
    from rl_quant_b200 import InferenceRunner, QuantLinear, build_glad
    from rl_quant_b200.synthetic import glad_obs_pair
    m, _ = golden_model(golden_weights)
    po, co = (t.cuda().half() for t in glad_obs_pair(20, seed=7))
    head, obs = (m.critic, co) if paths[0].startswith("critic") else (m.actor, po)
    with torch.no_grad():
        enc = m._encode_terrain(obs)[0].clone()
        before = head(enc)
    m.__dict__.pop("_glad_fused", None)
    layers = swap.apply_lora(m, paths, rank=8, adapters=2)
    for mod in layers.values():
        assert isinstance(mod.base, nn.Linear if head is m.critic else QuantLinear)
    task = torch.arange(20, device="cuda") % 3 - 1
    swap.select_lora(layers, task)
    for mode in ("eager", "manual-graph"):
        with pytest.warns(UserWarning, match="op by op"):
            run = InferenceRunner(m, mode=mode, with_critic=True)
        act = run.evaluate if head is m.critic else run.act
        with torch.no_grad():
            assert torch.equal(m._encode_terrain(obs)[0], enc)       # the same kernels, bit for bit
            if head is m.actor:
                assert torch.equal(act(obs), before)                 # new adapters change nothing
            for mod in layers.values():
                nn.init.normal_(mod.lora_b, std=0.2)
            got = act(obs).clone()
            assert torch.equal(got, head(enc) if head is m.actor else head(m._encode_terrain_orig(obs)[0]))
            swap.select_lora(layers, None)
            assert not torch.equal(act(obs), got) and (head is m.critic or torch.equal(act(obs), before))
            swap.select_lora(layers, task)
            for mod in layers.values():
                mod.lora_b.zero_()
    head(m._encode_terrain(obs)[0]).float().square().sum().backward()
    for mod in layers.values():
        assert mod.lora_b.grad.any() and mod.base.weight.grad is None
    master = build_glad(seed=1).cuda()
    run.sync_weights_from(master)
    for p, mod in layers.items():
        assert torch.equal(mod.base.weight, master.get_submodule(p).weight.half())
        if isinstance(mod.base, QuantLinear):
            w8 = mod.base.w8.clone()
            mod.base.requantize_()
            assert torch.equal(mod.base.w8, w8) and w8.any()


@gpu
@pytest.mark.parametrize("paths", [["actor.4", "critic.0"], ["topk_scorer", "actor.0"]])
def test_accelerated_policy_with_adapters(paths):
    """accelerate_runner over a policy with adapters: rollouts are of the adapters that the policy has selected then, and of its current
    weights after an update."""
    import types

    from rl_quant_b200 import accelerate_runner, build_glad
    from rl_quant_b200.synthetic import glad_obs_pair
    torch.manual_seed(0)
    policy = build_glad().cuda().eval()
    layers = swap.apply_lora(policy, paths, rank=8, adapters=3)
    for mod in layers.values():
        nn.init.normal_(mod.lora_b, std=0.3)
    obs = dict(zip(("policy_obs", "critic_obs"), (t.cuda() for t in glad_obs_pair(32, seed=6))))
    alg = types.SimpleNamespace(policy=policy, act=lambda o: None, update=lambda: {})
    with pytest.warns(UserWarning, match="op by op"):
        acc = accelerate_runner(types.SimpleNamespace(alg=alg, device="cuda", env=None), calib_obs=[obs], let_steps=5, mode="manual-graph",
                                rollout_training=False, verbose=False)
    inner = {p: acc.infer.get_submodule(p) for p in paths}
    assert all(isinstance(m, LoRALinear) for m in inner.values())
    seen = []
    task = torch.arange(32, device="cuda") % 4 - 1
    for index in (0, 2, task, None):
        if isinstance(index, torch.Tensor) and "topk_scorer" in paths:
            layers["actor.0"].select(index)               # the scorer's rows are those of a map
        else:
            swap.select_lora(layers, index)
        with torch.inference_mode():
            policy.update_distribution(policy.get_actor_obs(obs))
            mean, value = policy.action_mean.clone(), policy.evaluate(obs).clone()
            float_mean = policy.actor(acc._orig_ud.__self__._encode_terrain(policy.get_actor_obs(obs))[0])
        seen.append(mean)
        # the copy's int8 layers and 16-bit rows: a few percent, other adapters change more than that
        with torch.no_grad():
            float_value = acc._orig_eval(obs)
        assert float((mean - float_mean).norm() / float_mean.norm()) < 0.1
        assert float((value - float_value).norm() / float_value.norm()) < 0.1
        assert all(m.index is layers[p].index for p, m in inner.items())
    assert all(float((a - b).norm() / b.norm()) > 0.2 for a, b in zip(seen, seen[1:]))
    swap.select_lora(layers, 0)
    with torch.no_grad():
        for mod in layers.values():
            mod.lora_b.mul_(-1.0)
    alg.update()
    with torch.inference_mode():
        policy.update_distribution(policy.get_actor_obs(obs))
    assert not torch.equal(policy.action_mean, seen[0])
    for p, m in inner.items():
        assert torch.equal(m.lora_b, layers[p].lora_b.half())
    acc.detach()


def test_module_surgery():
    m = net(torch.float32, "cpu")
    m.eval()
    lin = m[0]
    with pytest.raises(AssertionError, match="not a linear"):
        swap.apply_lora(m, ["0", "1"])
    with pytest.raises(ValueError, match="rank"):
        swap.apply_lora(m, ["0"], rank=129)
    assert m[0] is lin and lin.weight.requires_grad       # all or none
    layers = swap.apply_lora(m, ["0"], rank=4, adapters=2, alpha=8)
    mod = layers["0"]
    assert isinstance(m[0], LoRALinear) and not m[0].training and mod.scale == 2.0
    assert mod.lora_a.shape == (2, 4, 96) and mod.lora_b.shape == (2, 128, 4) and not mod.lora_b.any()
    assert not lin.weight.requires_grad and {n for n, p in m.named_parameters() if p.requires_grad} == {
        "0.lora_a", "0.lora_b", "2.weight", "2.bias"}
    for bad in (2, -2):
        with pytest.raises(ValueError, match="adapter"):
            mod.select(bad)
    with pytest.raises(TypeError, match="int8"):
        mod(torch.zeros(3, 96, dtype=torch.int8))
    x = torch.randn(3, 96)
    assert torch.equal(mod.select(None)(x), lin(x))
    swap.restore_lora(m, layers)
    assert m[0] is lin and not lin.training


@pytest.mark.parametrize("other", [dict(rank=4), dict(adapters=2), dict(alpha=32.0)])
def test_sync_refuses_other_adapters(other):
    """A master's adapters of another rank, number or scale than the copy's: an error before anything is copied."""
    from rl_quant_b200 import InferenceRunner, build_glad
    common = dict(rank=8, adapters=3, alpha=16.0)
    copy, master = build_glad(0), build_glad(1)
    swap.apply_lora(copy, ["actor.0"], **common)
    swap.apply_lora(master, ["actor.0"], **{**common, **other})
    with pytest.warns(UserWarning, match="op by op"):
        run = InferenceRunner(copy)
    before = copy.actor[2].weight.clone()
    for _ in range(2):
        with pytest.raises(ValueError, match="actor.0: the source has"):
            run.sync_weights_from(master)
    assert torch.equal(copy.actor[2].weight, before)


def test_restore_below_adapters():
    """Plain layers put back for quantised ones come below the adapters that were put over those since."""
    m = net(torch.float32, "cpu").eval()
    weight = m[0].weight
    q = swap.apply(m, {"0": {"bits": 4, "group": 32}})
    layers = swap.apply_lora(m, ["0"], rank=4)
    swap.restore(m, q)
    assert m[0] is layers["0"] and type(m[0].base) is nn.Linear and m[0].base.weight is weight and not m[0].base.training
    swap.restore_lora(m, layers)
    assert type(m[0]) is nn.Linear and m[0].weight is weight


def test_layers_that_their_parent_computes_itself():
    """nn.MultiheadAttention and nn.TransformerEncoderLayer read weights of layers below instead of calling them: adapters over those would
    end in the next forward, so the swap refuses them, all or none."""
    m = nn.Sequential(nn.Linear(32, 32), nn.MultiheadAttention(32, 4), nn.TransformerEncoderLayer(32, 4, 64)).eval()
    x = torch.randn(5, 2, 32, generator=torch.Generator().manual_seed(0))

    def run():
        h = m[0](x)
        return m[2](m[1](h, h, h)[0])
    before = run().detach()
    for bad in ("1.out_proj", "2.linear1", "2.linear2", "2.self_attn.out_proj"):
        with pytest.raises(ValueError, match="reads the layer's weight"):
            swap.apply_lora(m, ["0", bad], rank=4)
    assert type(m[0]) is nn.Linear and m[0].weight.requires_grad and torch.equal(run(), before)


def test_refusals():
    x, a, b = torch.zeros(3, 8), torch.zeros(2, 4, 8), torch.zeros(2, 5, 4)
    i = torch.zeros(3, dtype=torch.int64)

    def call(x=x, a=a, b=b, index=i, **kw):
        return lora_linear(x, a, b, index, **kw)
    for bad, kind, what in (
            (dict(x=x.double()), TypeError, "x is"), (dict(a=a[0]), ValueError, "must be"), (dict(b=b[:1]), ValueError, "must be"),
            (dict(b=torch.zeros(2, 5, 3)), ValueError, "must be"), (dict(x=torch.zeros(3, 7)), ValueError, "inputs"),
            (dict(a=a.half()), TypeError, "expected x's"), (dict(index=None), ValueError, "need an index"),
            (dict(index=i.float()), TypeError, "index is"), (dict(index=i[:2]), ValueError, "does not match"),
            (dict(scale=torch.ones(3)), ValueError, "scale"), (dict(scale=torch.ones(2).half()), ValueError, "scale"),
            (dict(scale=torch.ones(2, requires_grad=True)), RuntimeError, "no gradient of scale"),
            (dict(base=torch.zeros(3, 4)), ValueError, "base"), (dict(base=torch.zeros(3, 5).half()), TypeError, "base"),
            (dict(a=torch.zeros(2, 200, 8), b=torch.zeros(2, 5, 200)), ValueError, "up to"),
            (dict(a=torch.zeros(2, 0, 8), b=torch.zeros(2, 5, 0)), ValueError, "up to"),
            (dict(a=torch.zeros(2, 4, 8, device="meta")), ValueError, "tensors on"),
            (dict(), RuntimeError, "CUDA")):
        with pytest.raises(kind, match=what):
            call(**bad)
    from rl_quant_b200 import _native as N
    lib = N.load()
    assert lib.glad_debug_lora_wait(2, 0) == lib.glad_debug_lora_wait(1, 2_000_000_001) == N.GLAD_ERR_INVALID_ARG
    big = torch.zeros(1, 8).expand(lora_mod.MAX_SIZE + 1, 8)
    with pytest.raises(ValueError, match="rows"):
        lora_linear(big, a[:1], b[:1])
    import torch.autograd.forward_ad as fwAD
    with fwAD.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(x=fwAD.make_dual(x, torch.ones_like(x)))
