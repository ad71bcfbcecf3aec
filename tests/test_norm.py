"""rms_norm / rms_norm_quant against the formula in 64 bits.

Tolerances, fixed before the first run: a row's sum of squares is at most 32 adds a thread and 10 levels of a tree, each
off by 2^-24 of the running sum of positive terms, and enters 1/rms by half; square root, quotient and two products add
2^-24 each. So y is off by at most F32 = 64 * 2^-24 relative before it is rounded (half a step, finfo.eps / 2). The
row sums of the backward pass have terms of both signs: 64 * 2^-24 of the sum of their magnitudes."""
import numpy as np
import pytest
import torch

from rl_quant_b200 import _native as N
from rl_quant_b200.norm import MAX_COLS, RMSNorm, rms_norm, rms_norm_quant

F32 = 64 * 2.0 ** -24
EPS = 1e-6
PAIRS = [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
         (torch.float16, torch.float32), (torch.bfloat16, torch.float32)]
gpu = pytest.mark.gpu


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):          # half the spacing of the subnormal numbers
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def rows(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def ref_norm(h, w, eps=EPS):
    h = h.double()
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * rstd * (1.0 if w is None else w.double()), rstd


def check_y(y, ref):
    tol = (half_step(y.dtype) * (1 + F32) + F32) * ref.abs() + tiny(y.dtype)
    assert ((y.double() - ref).abs() <= tol).all()


# widths: one column, a lone vector, off every vector width, one and two words a thread, the largest
SIZES = [(1, 1), (3, 8), (1, 2048), (2, 1000), (5, 1111), (1, 8192), (300, 264), (700, 1301), (600, 4096), (1, 32768),
         (2, 16391), (299, 32767), (310, 20000)]


@gpu
@pytest.mark.parametrize("x_t,r_t", PAIRS)
@pytest.mark.parametrize("shape", SIZES)
def test_forward(shape, x_t, r_t):
    x, r = rows(shape, x_t, 1), rows(shape, r_t, 2, 5.0)
    for w in (None, rows(shape[1:], x_t, 3), rows(shape[1:], torch.float32, 4)):
        y = rms_norm(x, w, eps=EPS)
        assert y.dtype == x_t and y.shape == x.shape
        check_y(y, ref_norm(x, w)[0])
    y, h = rms_norm(x, w, residual=r, eps=EPS)
    assert h.dtype == r_t and torch.equal(h, (x.float() + r.float()).to(r_t))
    check_y(y, ref_norm(h, w)[0])


def grads(h, w, dy, dh, x_t, r_t):
    """64-bit gradients and the magnitudes their roundings scale with."""
    C = h.shape[-1]
    h, dy = h.double(), dy.double()
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
    g = dy * (1.0 if w is None else w.double())
    d = rstd * (g - h * rstd ** 2 * (g * h).sum(-1, keepdim=True) / C)
    mag = rstd * (g.abs() + h.abs() * rstd ** 2 * (g * h).abs().sum(-1, keepdim=True) / C)
    if dh is not None:
        d, mag = d + dh.double(), mag + dh.double().abs()
    unit = h * rstd
    return d, mag, (dy * unit).sum(0), (dy * unit).abs().sum(0)


@gpu
@pytest.mark.parametrize("x_t,r_t", PAIRS)
@pytest.mark.parametrize("shape", SIZES + [(2500, 72), (1200, 512), (1, 32)])
@pytest.mark.parametrize("with_res", [False, True])
def test_backward(shape, x_t, r_t, with_res):
    if not with_res and r_t != x_t:
        pytest.skip("the residual's type without a residual")
    for w_t in {x_t, torch.float32}:
        x = rows(shape, x_t, 1).requires_grad_()
        w = (1 + 0.3 * rows(shape[1:], torch.float32, 3)).to(w_t).requires_grad_()
        r = rows(shape, r_t, 2, 5.0).requires_grad_() if with_res else None
        dy, dh = rows(shape, x_t, 5), rows(shape, r_t, 6) if with_res else None
        if with_res:
            y, h = rms_norm(x, w, residual=r, eps=EPS)
            dx, dw, dr = torch.autograd.grad((y, h), (x, w, r), (dy, dh))
        else:
            y, h = rms_norm(x, w, eps=EPS), x
            (dx, dw), dr = torch.autograd.grad(y, (x, w), dy), None
        check_y(y.detach(), ref_norm(h.detach(), w.detach())[0])
        d, mag, dw_ref, dw_mag = grads(h.detach(), w.detach(), dy, dh, x_t, r_t)
        for got, t in ((dx, x_t), (dr, r_t)):
            if got is not None:
                assert got.dtype == t
                tol = half_step(t) * d.abs() + 2 * F32 * mag + tiny(t)
                assert ((got.double() - d).abs() <= tol).all()
        assert dw.dtype == w_t
        tol = half_step(w_t) * dw_ref.abs() + (shape[0] + 64) * 2.0 ** -24 * dw_mag * (1 + half_step(w_t)) \
            + F32 * dw_mag + tiny(w_t)
        assert ((dw.double() - dw_ref).abs() <= tol).all()


@gpu
def test_gradient_against_differences():
    """Central differences of the scalar sum(dy * y + dh * h) along random directions, all in fp32: the step 2^-6 leaves a
    truncation error of order 2^-12 and a rounding error of order 2^-24 * 2^6 * sqrt(n), far below the 1% asked."""
    x, w, r = rows((6, 200), torch.float32, 1), 1 + 0.3 * rows((200,), torch.float32, 2), rows((6, 200), torch.float32, 3)
    dy, dh = rows((6, 200), torch.float32, 4), rows((6, 200), torch.float32, 5)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
    got = torch.autograd.grad((y, h), leaves, (dy, dh))

    def f(x, w, r):
        y, h = rms_norm(x, w, residual=r, eps=EPS)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    e = 2.0 ** -6
    for i in range(3):
        v = rows((x, w, r)[i].shape, torch.float32, 10 + i)
        up, dn = [x, w, r], [x, w, r]
        up[i], dn[i] = up[i] + e * v, dn[i] - e * v
        num = (f(*up) - f(*dn)) / (2 * e)
        ana = float((got[i].double() * v.double()).sum())
        assert abs(num - ana) <= 0.01 * float((got[i].double().abs() * v.double().abs()).sum() / 8 + abs(ana))


@gpu
def test_backward_parts():
    """One of the two outputs used alone, gradients asked for singly, no weight."""
    x, r = rows((40, 96), torch.bfloat16, 1).requires_grad_(), rows((40, 96), torch.bfloat16, 2).requires_grad_()
    w = rows((96,), torch.bfloat16, 3).requires_grad_()
    g = rows((40, 96), torch.bfloat16, 4)
    y, h = rms_norm(x, w, residual=r)
    full = torch.autograd.grad((y, h), (x, w, r), (g, torch.zeros_like(g)), retain_graph=True)
    only_y = torch.autograd.grad(y, (x, w, r), g, retain_graph=True)
    for a, b in zip(full, only_y):
        assert torch.equal(a, b)
    for i, leaf in enumerate((x, w, r)):
        assert torch.equal(torch.autograd.grad(y, leaf, g, retain_graph=True)[0], full[i])
    dx, dr = torch.autograd.grad(h, (x, r), g, retain_graph=True)
    assert torch.equal(dx, g) and torch.equal(dr, g)
    x2 = x.detach().float().requires_grad_()
    y2, h2 = rms_norm(x2, residual=r.detach().float())
    d, mag, _, _ = grads(h2.detach(), None, g.float(), None, torch.float32, torch.float32)
    (dx2,) = torch.autograd.grad(y2, x2, g.float())
    assert ((dx2.double() - d).abs() <= 2 * F32 * mag).all()
    # leaves accumulate: two uses of one weight
    w2 = w.detach().clone().requires_grad_()
    (rms_norm(x.detach(), w2) + rms_norm(r.detach(), w2)).backward(g)
    assert w2.grad.shape == (96,)


@gpu
def test_deterministic_and_empty():
    x, w = rows((3000, 1024), torch.bfloat16, 1).requires_grad_(), rows((1024,), torch.float32, 2).requires_grad_()
    g = rows((3000, 1024), torch.bfloat16, 3)
    a = torch.autograd.grad(rms_norm(x, w), (x, w), g)
    b = torch.autograd.grad(rms_norm(x, w), (x, w), g)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    e = torch.empty(0, 1024, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y, h = rms_norm(e, w, residual=e.detach())
    assert y.shape == h.shape == (0, 1024)
    dx, dw = torch.autograd.grad(y, (e, w), torch.empty_like(y))
    assert dx.shape == (0, 1024) and float(dw.abs().max()) == 0.0
    q, s = rms_norm_quant(e.detach(), w.detach())
    assert q.shape == (0, 1024) and s.shape == (0, 1)


@gpu
@pytest.mark.parametrize("x_t", [torch.float16, torch.float32])
def test_strides_and_alignment(x_t):
    """Rows inside a wider tensor, every start within a 16-byte line, transposed and 3-d inputs."""
    base = rows((64, 700), x_t, 1)
    w = rows((512,), torch.float32, 2)
    for at in (0, 1, 3, 8):
        x = base[:, at:at + 512]
        y, h = rms_norm(x, w[:512], residual=base[:, 150:662])
        assert torch.equal(h, (x.float() + base[:, 150:662].float()).to(x_t))
        check_y(y, ref_norm(h, w)[0])
        q, s = rms_norm_quant(x, w, group=64)
        q2, s2 = rms_norm_quant(x.contiguous(), w, group=64)
        # rows off 16 bytes are read one element at a time, so the two sums of squares run in other orders; each y is
        # within F32 of the exact value: scales within 2 F32 of one another, each code nearest to its own y / s
        assert ((s - s2).abs() <= 2 * F32 * s2).all()
        y, _ = ref_norm(x, w)
        for codes, scales in ((q, s), (q2, s2)):
            check_codes(codes, scales.double().repeat_interleave(64, 1), y, torch.int8)
    t = base.t()[:, :33]
    check_y(rms_norm(t), ref_norm(t, None)[0])
    b3 = base[:, :512].reshape(8, 8, 512).transpose(0, 1)
    check_y(rms_norm(b3, w), ref_norm(b3, w)[0])
    one = base[0, :512]
    check_y(rms_norm(one, w), ref_norm(one, w)[0])
    ws = torch.stack((w, w), dim=1)[:, 0]
    assert torch.equal(rms_norm(one, ws), rms_norm(one, w))
    xg = base[:, 1:513].detach().requires_grad_()
    dy = base[:, 100:612]
    (dx,) = torch.autograd.grad(rms_norm(xg, w), xg, dy)
    d, mag, _, _ = grads(xg.detach(), w, dy, None, x_t, x_t)
    assert ((dx.double() - d).abs() <= half_step(x_t) * d.abs() + 2 * F32 * mag + tiny(x_t)).all()


@gpu
def test_gradients_of_leaves_are_their_own():
    """x and a residual of its type have the same gradient: each leaf's is a tensor of its own, the same leaf in both
    places gets the sum, and one set of leaves serves two graphs that live at once."""
    x, r = rows((40, 96), torch.bfloat16, 1).requires_grad_(), rows((40, 96), torch.bfloat16, 2).requires_grad_()
    w, g = rows((96,), torch.bfloat16, 3).requires_grad_(), rows((40, 96), torch.bfloat16, 4)
    want = torch.autograd.grad(rms_norm(x, w, residual=r)[0], (x, w), g)
    y, h = rms_norm(x, w, residual=r)
    y2, _ = rms_norm(x, w, residual=r)
    y.backward(g)
    assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[0]) and torch.equal(w.grad, want[1])
    assert x.grad.data_ptr() != r.grad.data_ptr()
    x.grad.zero_()
    assert torch.equal(r.grad, want[0])
    r.grad = None
    y2.backward(g)
    assert torch.equal(x.grad, want[0]) and torch.equal(r.grad, want[0])
    y, h = rms_norm(x, w, residual=r)      # the sum alone: the gradient that arrives is passed on
    x.grad = r.grad = None
    h.backward(g)
    x.grad.zero_()
    assert torch.equal(r.grad, g) and bool(g.any())
    both = torch.autograd.grad(rms_norm(x, w, residual=x)[0], x, g)[0]
    one = torch.autograd.grad(rms_norm(x, w, residual=x.detach())[0], x, g)[0]
    assert torch.equal(both, one * 2)
    y, h = rms_norm(x, w, residual=r)
    with torch.no_grad():
        h.add_(1.0)                         # the backward pass reads the sum
    with pytest.raises(RuntimeError):
        y.backward(g)


@gpu
def test_broadcast_rows():
    """Rows that share memory: expanded inputs, and the expanded gradient that a mean over the rows sends back."""
    x, r, w = rows((1, 96), torch.float16, 1), rows((1, 96), torch.float16, 2), rows((96,), torch.float16, 3)
    xe, re = x.expand(40, 96), r.expand(40, 96)
    for a, b in ((rms_norm(xe, w), rms_norm(xe.contiguous(), w)),
                 (rms_norm(xe.unsqueeze(0), w)[0], rms_norm(xe.contiguous(), w)),
                 (rms_norm(xe, w, residual=re)[0], rms_norm(xe.contiguous(), w, residual=re.contiguous())[0]),
                 (rms_norm_quant(xe, w, residual=re)[0], rms_norm_quant(xe.contiguous(), w, residual=re.contiguous())[0])):
        assert torch.equal(a, b)
    leaf, wl = rows((40, 96), torch.float16, 4).requires_grad_(), w.clone().requires_grad_()
    dy = rows((96,), torch.float16, 5)
    for shape in ((40, 96), (4, 10, 96)):
        got = torch.autograd.grad(rms_norm(leaf.view(shape), wl), (leaf, wl), dy.expand(shape))
        want = torch.autograd.grad(rms_norm(leaf, wl), (leaf, wl), dy.expand(40, 96).contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    y, h = rms_norm(leaf, wl, residual=xe.contiguous())
    got = torch.autograd.grad((y, h), (leaf,), (dy.expand(40, 96), dy.expand(40, 96)), retain_graph=True)
    want = torch.autograd.grad((y, h), (leaf,), (dy.expand(40, 96).contiguous(), dy.expand(40, 96).contiguous()))
    assert torch.equal(got[0], want[0])


QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def check_codes(q, s_cols, y, out):
    """Each code is a nearest one to y / s: within half a step plus the fp32 error of y / s."""
    t = y / s_cols
    Q = QMAX[out]
    t = t.clamp(-Q, Q)
    d = (q.double() - t).abs()
    if out == torch.int8:
        assert (d <= 0.5 + 2 * F32 * Q).all()
    else:
        assert (d <= (2.0 ** -4 + 2 * F32) * t.abs() + 2.0 ** -10).all()


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("x_t,r_t", PAIRS)
@pytest.mark.parametrize("shape", SIZES)
def test_quant(shape, x_t, r_t, out):
    x, r, w = rows(shape, x_t, 1), rows(shape, r_t, 2, 5.0), rows(shape[1:], torch.float32, 3)
    R, C = shape
    for group in (0, 32, 64, 128):
        q, s, h = rms_norm_quant(x, w, residual=r, eps=EPS, out_dtype=out, group=group)
        assert q.dtype == out and torch.equal(h, (x.float() + r.float()).to(r_t))
        y, _ = ref_norm(h, w)
        width = group or C
        G = -(-C // width)
        assert s.shape == (R, G)
        pad = torch.zeros(R, G * width, dtype=torch.float64, device="cuda")
        pad[:, :C] = y.abs()
        ref = pad.view(R, G, width).amax(-1) / QMAX[out]
        ref = torch.where(ref > 0, ref, torch.ones_like(ref))
        assert ((s.double() - ref).abs() <= 2 * F32 * ref).all()
        check_codes(q, s.double().repeat_interleave(width, 1)[:, :C], y, out)
    given = torch.tensor(3.0 / QMAX[out], device="cuda")
    q, s = rms_norm_quant(x, w, eps=EPS, out_dtype=out, scale=given)
    assert s is given
    check_codes(q, given.double(), ref_norm(x, w)[0], out)


def as_code(t, out):
    """t (float32 or float64) to the nearest code, ties to even; NaN to 0 in int8."""
    Q = QMAX[out]
    t = t.clamp(-Q, Q)
    return t.round().nan_to_num(0.0).to(torch.int8) if out == torch.int8 else t.to(out)


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(200, 1024), (40, 8192), (65, 1001)])
def test_quant_codes_on_borders(shape, out):
    """bf16 values of few bits, so that y / s = h w Q / max|h w| often lies on a border between two codes. h w Q has at most
    24 bits and the quotient in 64 bits is exact there; elsewhere it is 2^-24 or more away, relatively. So every code
    is known."""
    g = torch.Generator().manual_seed(shape[1])
    x = (torch.randint(-127, 128, shape, generator=g) / 16).to(torch.bfloat16).cuda()
    r = torch.randint(-8, 9, shape, generator=g).to(torch.bfloat16).cuda()
    w = (torch.randint(1, 65, shape[1:], generator=g) / 32).to(torch.bfloat16).cuda()
    for group in (0, 32, 128):
        q, s, h = rms_norm_quant(x, w, residual=r, out_dtype=out, group=group)
        p = h.double() * w.double()
        width = group or shape[1]
        top = torch.stack([c.abs().amax(1) for c in p.split(width, dim=1)], dim=1)
        top = top.masked_fill(top == 0, 1.0).repeat_interleave(width, 1)[:, :shape[1]]
        assert torch.equal(q.float(), as_code(p * QMAX[out] / top, out).float())


def unit_rows(w, **kw):
    """rms_norm_quant of one row of ones without eps: the norm is 1 exactly, so y is the weight w."""
    w = torch.as_tensor(w, dtype=torch.float32)
    pad = torch.zeros(1 << max(w.numel() - 1, 1).bit_length())           # a mean of 1 needs no power of two, but this is one
    pad[:w.numel()] = w
    q, s = rms_norm_quant(torch.ones(1, pad.numel(), device="cuda"), pad.cuda(), eps=0.0, **kw)
    return q[0].cpu()[:w.numel()], s.cpu()


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_quant_scale_is_the_quotient(out):
    """s = max|y| / Q rounded once, for every significand of 17 bits (Qz y is exact then) and for sizes far from 1."""
    v = torch.arange(1 << 16, 1 << 17).float() * 2.0 ** -16
    for part in v.split(1024):
        w = torch.zeros(1024, 32)
        w[torch.arange(1024), torch.arange(1024) % 32] = part
        _, s = unit_rows(w.flatten(), group=32, out_dtype=out)
        assert np.array_equal(s[0].numpy(), part.numpy() / np.float32(QMAX[out]))
    for e in (-115, -100, -61, -60, -30, 60, 99, 101, 126):
        y = np.float32(2.0 ** e) * np.float32(1.25)
        assert float(unit_rows([0.0, y, 0.0], out_dtype=out)[1]) == float(y / np.float32(QMAX[out]))


def codes_near_borders(out):
    """(s, y) with y / s next to a border: a product with a reciprocal good to 2^-23 and one correction is off by at most
    2^-44.8 before it is rounded ((1.5 * 2^-23)^2), so it can round otherwise than
    the exact quotient only where that lies this close to the middle between two fp32 numbers, one of which is a border: a
    number M 2^i of b = 5 (e4m3) or 8 (int8) bits. In integers, 2 Y 2^k = S (M 2^(25 - b) +- 1) + c with |c| < 2^-44.8 2^49 < 19,
    so S is within 19 of a multiple of 2^(25 - b). All such S, and for each the y around every border's neighbours."""
    if out == torch.int8:
        ties, step = np.arange(0.5, 127.0, 1.0), 1 << 17
    else:
        codes = torch.arange(127, dtype=torch.uint8).view(out).double().numpy()
        ties, step = (codes[1:] + codes[:-1]) / 2, 1 << 20
    f = ties.astype(np.float32)
    assert (f == ties).all()
    middles = np.concatenate([(f.astype(np.float64) + np.nextafter(f, np.float32(t))) / 2 for t in (0.0, 1e9)] + [ties])
    for base in range(1 << 23, (1 << 24) + 1, step):
        for S in range(max(base - 19, 1 << 23), min(base + 20, 1 << 24)):
            y = (middles * S).astype(np.float32)                         # the product has at most 49 bits: exact in 64
            y = np.concatenate([y, np.nextafter(y, np.float32(0)), np.nextafter(y, np.float32(3e38))])
            yield np.float32(S * 2.0 ** -24), np.float32(2.0 ** -24) * np.concatenate([y, -y])


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_quant_given_scale_next_to_every_border(out):
    for s, y in codes_near_borders(out):
        q, _ = unit_rows(y, scale=torch.tensor(s, device="cuda"), out_dtype=out)
        assert torch.equal(q.view(torch.uint8), as_code(torch.from_numpy(y / s), out).view(torch.uint8)), float(s)


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_quant_given_scale_of_any_size(out):
    y = np.float32([0.0, -0.0, 1.0, -2.5, 1e-45, -1e-38, 3e38, -3.3e38, 1e30, 7e-30, np.inf, -np.inf, np.nan])
    with np.errstate(all="ignore"):
        for s in np.float32([2.0 ** 127, 1.5e38, 3e38, 2.0 ** 100, 1e25, 1e-30, 1e-38, 1e-45, 5e-40, 0.0, np.inf, np.nan, -1.0,
                             -1e-40, -2e38, 1.0]):
            q, _ = unit_rows(y, scale=torch.tensor(s, device="cuda"), out_dtype=out)
            want = as_code(torch.from_numpy(y / s), out)
            assert torch.equal(q.float().nan_to_num(1e3), want.float().nan_to_num(1e3)), float(s)


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(64, 512), (3, 4096), (40, 333), (2, 20000), (2, 20001), (9000, 288), (2500, 1001)])
def test_quant_rows_of_every_size(shape, out):
    """Rows and groups whose maximum leaves the range of fast quotients stand beside ordinary ones, zeros and NaN: each has its
    own scale and codes."""
    R, C = shape
    x = torch.ones(R, C, device="cuda")
    g = torch.Generator().manual_seed(C)
    w = torch.randn(C, generator=g)
    size = torch.tensor([1.0, 0.0, 1e-20, 1e25, 1e-36, 3e36, 1e-44])
    w *= size.repeat_interleave(32).repeat(-(-C // 224))[:C]
    w[C // 2] = float("nan")
    for group in (32, 64):
        q, s = rms_norm_quant(x, w.cuda(), eps=0.0, out_dtype=out, group=group)
        y = w.double()
        top = torch.stack([c.abs().amax() for c in y.split(group)])
        ref = top / QMAX[out]
        ref32 = ref.float()                                # what underflows to 0 has the scale 1
        ref = torch.where(ref32 == 0, torch.ones_like(ref), ref)
        nan = torch.isnan(ref)
        same = lambda a, b: torch.equal(a.float().nan_to_num(1e3), b.float().nan_to_num(1e3))  # noqa: E731
        assert same(q, q[:1].expand_as(q)) and same(s, s[:1].expand_as(s))
        wide = torch.ones(R, C + 3, device="cuda", dtype=torch.float16)[:, 3:]     # rows off every word, other types
        for x2, r2 in ((x, torch.zeros_like(x)), (wide, torch.zeros_like(x)), (wide, wide * 0)):
            q2, s2, _ = rms_norm_quant(x2, w.cuda(), residual=r2, eps=0.0, out_dtype=out, group=group)
            assert same(q2[0], q2[R - 1]) and same(s2, s2[:1].expand_as(s2))
            assert (s2[0] - s[0]).abs().nan_to_num(0.0).le(4 * F32 * s[0].nan_to_num(1.0) + 2.0 ** -148).all()
            assert torch.equal(torch.isnan(s2[0]), torch.isnan(s[0]))
        for r in {0, R - 1}:
            got = s[r].cpu().double()
            assert torch.equal(torch.isnan(got), nan)
            # the norm of ones is 1 to within F32; near the smallest number a rounding is half of 2^-149
            assert ((got - ref).abs() <= 2 * F32 * ref + 2.0 ** -149)[~nan].all()
            per = s[r].cpu().double().repeat_interleave(group)[:C]
            live = ~torch.isnan(per)
            check_codes(q[r].cpu()[live], per[live], y[live], out)
            assert not q[r].cpu()[~live].float().nan_to_num(0.0).any()


@gpu
def test_quant_zero_and_nonfinite_rows():
    x = rows((6, 256), torch.float32, 1)
    x[0] = 0
    x[1, :64] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    x[4] = 3e38                      # the sum of squares overflows: y is 0
    for out in QMAX:
        q, s = rms_norm_quant(x, out_dtype=out)
        assert float(s[0]) == 1.0 and not q[0].float().any()
        assert bool(torch.isnan(s[2])) and bool(torch.isnan(s[3]))
        assert float(s[4]) == 1.0 and not q[4].float().any()
        assert torch.isfinite(s[[1, 5]]).all() and float(q[5].float().abs().max()) == QMAX[out]
        q, s = rms_norm_quant(x, out_dtype=out, group=64)
        assert float(s[1, 0]) == 1.0 and not q[1, :64].float().any() and bool(torch.isnan(s[2]).all())
    tiny_rows = torch.full((2, 64), 1e-38, device="cuda")
    q, s = rms_norm_quant(tiny_rows, eps=1.0)          # a scale below the smallest normal number
    assert torch.isfinite(s).all() and (q.abs() >= 120).all()


@gpu
@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_quant_scale_that_rounds_to_zero(out):
    """A largest value below half the smallest subnormal times Q has a scale of zero: the scale is 1, all codes are 0."""
    x = torch.zeros(2, 64, device="cuda")
    x[:, 3] = 1.0
    w = torch.full((64,), 2.0 ** -149 * 5, device="cuda")       # y[:, 3] is about 8 * 5 * 2^-149
    for group in (0, 32):
        for wide in (x, torch.cat((x, x), 1)[:, 1:64]):
            q, s = rms_norm_quant(wide, w[:wide.shape[1]], out_dtype=out, group=group)
            assert torch.equal(s, torch.ones_like(s)) and not q.float().any()


@gpu
def test_streams_graph_and_64_bit_offsets():
    x, w = rows((50, 1000), torch.float16, 1), rows((1000,), torch.float16, 2)
    want = rms_norm(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rms_norm(x, w)
    s.synchronize()
    assert torch.equal(got, want)
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    dy = rows((50, 1000), torch.float16, 3)
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(rms_norm(xs, ws), (xs, ws), dy)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = rms_norm(xs, ws)
        dx, dw = torch.autograd.grad(y, (xs, ws), dy)
        q, sc, h = rms_norm_quant(xs.detach(), ws.detach(), residual=dy)
    with torch.no_grad():
        xs.copy_(rows((50, 1000), torch.float16, 9))
    g.replay()
    torch.cuda.synchronize()
    y = y.detach()
    assert torch.equal(y, rms_norm(xs.detach(), ws.detach()))
    x2, w2 = xs.detach().clone().requires_grad_(), ws.detach().clone().requires_grad_()
    dx2, dw2 = torch.autograd.grad(rms_norm(x2, w2), (x2, w2), dy)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    for a, b in zip((q, sc, h), rms_norm_quant(xs.detach(), ws.detach(), residual=dy)):
        assert torch.equal(a, b)
    # rows past 2^31 elements
    big = torch.zeros(70000, 32768, dtype=torch.bfloat16, device="cuda")
    big[-1] = rows((32768,), torch.bfloat16, 4)
    y = rms_norm(big)
    check_y(y[-1], ref_norm(big[-1], None)[0])
    q, s = rms_norm_quant(big, group=128)
    q1, s1 = rms_norm_quant(big[-1:].clone(), group=128)
    assert torch.equal(q[-1:], q1) and torch.equal(s[-1:], s1)


@gpu
def test_module():
    src = torch.nn.RMSNorm(320, eps=1e-5, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        src.weight.copy_(rows((320,), torch.bfloat16, 1))
    m = RMSNorm.from_torch(src)
    assert m.weight is src.weight
    x = rows((9, 320), torch.bfloat16, 2)
    check_y(m(x).detach(), ref_norm(x, src.weight.detach(), 1e-5)[0])
    with torch.no_grad():
        q, s = m.quant(x, out_dtype=torch.float8_e4m3fn, group=64)
    assert q.shape == x.shape and s.shape == (9, 5)


def default_eps_layer(t, device):
    src = torch.nn.RMSNorm(192, device=device, dtype=t)
    with torch.no_grad():
        src.weight.copy_(torch.randn(192, generator=torch.Generator().manual_seed(1)))
    x = (torch.randn(40, 192, generator=torch.Generator().manual_seed(2))
         * torch.logspace(-4, 1, 40)[:, None]).to(t).to(device)
    return src, x


def check_default_eps(y, src, x):
    """torch's own layer and y are each off the formula with float32's eps by F32 and one rounding, so by twice that from one
    another; with another type's eps rows of 1e-2 are off by more than 10%."""
    ref, _ = ref_norm(x, src.weight.detach(), torch.finfo(torch.float32).eps)
    check_y(src(x).detach(), ref)
    check_y(y, ref)


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32])
def test_default_eps_is_torchs(t):
    src, x = default_eps_layer(t, "cpu")
    m = RMSNorm.from_torch(src)
    check_default_eps(ref_norm(x, src.weight.detach(), m.eps)[0].to(t), src, x)


@gpu
@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16, torch.float32])
def test_swapped_layer_with_default_eps(t):
    from rl_quant_b200 import swap
    src, x = default_eps_layer(t, "cuda")
    model = torch.nn.Sequential(src)
    swap.apply_norm(model)
    assert isinstance(model[0], RMSNorm)
    check_default_eps(model(x).detach(), src, x)


def forward_mode(call, *inputs):
    """``call`` with one input after another as a dual tensor, with gradients enabled and not, and once by torch.func."""
    from torch.autograd import forward_ad
    for i in range(len(inputs)):
        for grad in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                args = list(inputs)
                args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                call(*args)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda a: call(a, *inputs[1:]), (inputs[0],), (torch.ones_like(inputs[0]),))


def test_forward_mode_is_refused():
    x, w, r = torch.ones(4, 64), torch.ones(64), torch.ones(4, 64)
    forward_mode(lambda x, w, r: rms_norm(x, w, residual=r), x, w, r)
    forward_mode(lambda x, w, r: rms_norm_quant(x, w, residual=r), x, w, r)
    forward_mode(lambda s: rms_norm_quant(x, w, scale=s), torch.ones(()))
    forward_mode(RMSNorm(64), x, r)


# -- refusals (no GPU) -----------------------------------------------------------------------------


def test_refusals():
    x = torch.zeros(4, 64)
    for bad, kw in ((TypeError, dict(x=x.to(torch.float64))), (TypeError, dict(x=x.to(torch.int8))),
                    (ValueError, dict(x=torch.zeros(4, 0))), (ValueError, dict(x=torch.zeros(1, MAX_COLS + 1))),
                    (ValueError, dict(x=torch.tensor(1.0))),
                    (ValueError, dict(x=x, weight=torch.zeros(63))), (ValueError, dict(x=x, weight=torch.zeros(4, 64))),
                    (TypeError, dict(x=x, weight=torch.zeros(64, dtype=torch.float16))),
                    (ValueError, dict(x=x, residual=torch.zeros(64))),
                    (ValueError, dict(x=x, residual=torch.zeros(1, 64))),
                    (TypeError, dict(x=x, residual=x.half())),
                    (TypeError, dict(x=x.half(), residual=x.bfloat16())),
                    (ValueError, dict(x=x, eps=-1.0)), (ValueError, dict(x=x, eps=float("nan"))),
                    (ValueError, dict(x=x, residual=x.to("meta"))), (RuntimeError, dict(x=x))):
        with pytest.raises(bad):
            rms_norm(**kw)
        with pytest.raises(bad):
            rms_norm_quant(**kw)
    with pytest.raises(TypeError):
        rms_norm_quant(x, out_dtype=torch.uint8)
    with pytest.raises(ValueError):
        rms_norm_quant(x, group=16)
    with pytest.raises(ValueError):
        rms_norm_quant(x, group=64, scale=torch.tensor(1.0))
    with pytest.raises(ValueError):
        rms_norm_quant(x, scale=torch.ones(2))
    with pytest.raises(ValueError):
        rms_norm_quant(x, scale=torch.ones(1, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_quant(x.clone().requires_grad_())
    with pytest.raises(ValueError):
        RMSNorm.from_torch(torch.nn.RMSNorm((4, 8), eps=1e-6))
    with pytest.raises(ValueError):
        RMSNorm.from_torch(torch.nn.RMSNorm(8, elementwise_affine=False))


def test_abi_refusals():
    lib = N.load()
    a = np.zeros(4096, np.float32).ctypes.data // 16 * 16 + 16          # an address that no call may reach

    def fwd(x=a, xt=N.DTYPE_F16, ld=64, r=None, rt=0, ldr=64, w=None, wt=0, rows=2, cols=64, eps=1e-6, y=a, h=None):
        return lib.glad_rms_norm_forward(x, xt, ld, r, rt, ldr, w, wt, rows, cols, eps, y, h, None, None)

    bad = N.GLAD_ERR_INVALID_ARG
    assert fwd(rows=0) == N.GLAD_OK
    for kw in (dict(x=None), dict(y=None), dict(xt=N.DTYPE_I8), dict(xt=77), dict(ld=63), dict(cols=0), dict(cols=32769),
               dict(rows=-1), dict(rows=1 << 31), dict(eps=-1.0), dict(eps=float("nan")), dict(x=a + 1), dict(y=a + 1),
               dict(w=a, wt=N.DTYPE_BF16), dict(w=a + 1, wt=N.DTYPE_F16), dict(r=a, rt=N.DTYPE_F16),
               dict(h=a), dict(r=a, rt=N.DTYPE_BF16, h=a), dict(r=a, rt=N.DTYPE_F16, h=a, ldr=8),
               dict(r=a, rt=N.DTYPE_F32, h=a + 2)):
        assert fwd(**kw) == bad, kw
        assert lib.glad_last_error()

    def qnt(qt=N.DTYPE_I8, group=0, given=None, q=a, s=a, rows=2):
        return lib.glad_rms_norm_quant(a, N.DTYPE_F16, 64, None, 0, 0, None, 0, rows, 64, 1e-6, qt, group, given, q, s,
                                       None, None)

    assert qnt(rows=0) == N.GLAD_OK
    for kw in (dict(qt=N.DTYPE_F16), dict(group=1), dict(group=256), dict(given=a, group=64), dict(s=None), dict(q=None),
               dict(s=a + 2), dict(given=a + 1)):
        assert qnt(**kw) == bad, kw

    def bwd(dy=a, ds=None, h=a, ht=N.DTYPE_F16, w=a, rstd=a, dx=a, dr=None, dw=None, ws=None, n=0, rows=2, ld=64):
        return lib.glad_rms_norm_backward(dy, N.DTYPE_F16, ld, ds, ht, 64, h, 64, w, N.DTYPE_F16, rstd, rows, 64, dx, dr,
                                          dw, ws, n, None)

    need = lib.glad_rms_norm_backward_workspace_size(2, 64)
    assert need >= 8 * 64 * 4 and lib.glad_rms_norm_backward_workspace_size(0, 64) == 0
    assert lib.glad_rms_norm_backward_workspace_size(1 << 30, 64) < 1 << 20
    for kw in (dict(dy=None), dict(h=None), dict(rstd=None), dict(dx=None), dict(ht=N.DTYPE_BF16), dict(dw=a, w=None),
               dict(ld=8), dict(dx=a + 1), dict(rows=-1)):
        assert bwd(**kw) == bad, kw
    assert bwd(dw=a, ws=None) == bwd(dw=a, ws=a, n=need - 1) == bwd(dw=a, ws=a + 8, n=need) == N.GLAD_ERR_WORKSPACE
