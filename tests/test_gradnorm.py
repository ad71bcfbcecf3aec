"""grad_norm / clip_grads / clip_grads_ / clip_grad_norm_ against the formula in 64 bits.

Tolerances: they allow a thread batches of up to 128 squares in four running sums (33 roundings
of 2^-24 each, and 2 to join them), the rest in 64 bits; the root halves that and its rounding to float32 adds one: NORM2 = 20 *
2^-24, and 37 * 2^-24 for the sum of magnitudes (test_bounds_of_the_present_batch has those of the batches that the kernel takes). The maximum is exact. The coefficient adds three roundings, the product one."""
import itertools
import math

import pytest
import torch

from rl_quant_b200 import gradnorm
from rl_quant_b200.gradnorm import clip_grad_norm_, clip_grads, clip_grads_, grad_norm

gpu = pytest.mark.gpu
U = 2.0 ** -24
ERR = {2.0: 20 * U, 1.0: 37 * U, math.inf: 0.0}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(t):
    return 0.0 if t == torch.float32 else torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(sizes, types, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    kinds = itertools.cycle(types)
    return [(torch.randn(s, generator=g) * scale).to(next(kinds)).cuda() for s in sizes]


def ref_norm(ts, p):
    flat = torch.cat([t.double().reshape(-1) for t in ts]) if ts else torch.zeros(0, dtype=torch.float64)
    if not flat.numel():
        return 0.0
    return float(torch.linalg.vector_norm(flat, p))


def check(ts, max_norm, p):
    before = [t.clone() for t in ts]
    n = ref_norm(ts, p)
    got = grad_norm(ts, p)
    assert got.dtype == torch.float32 and got.shape == ()
    assert abs(float(got) - n) <= ERR[p] * n
    out, norm = clip_grads(ts, max_norm, p)
    assert torch.equal(norm, got)
    assert all(torch.equal(a, b) for a, b in zip(ts, before))
    c = min(1.0, max_norm / (n + 1e-6))
    for t, o in zip(before, out):
        assert o.dtype == t.dtype and o.shape == t.shape
        ref = t.double() * c
        tol = (half_step(t.dtype) + (ERR[p] + 5 * U)) * (1 + half_step(t.dtype)) * ref.abs() + tiny(t.dtype)
        assert ((o.double() - ref).abs() <= tol).all()
        if c == 1.0:
            assert torch.equal(o, t)
    same = clip_grads_(ts, max_norm, p)
    assert torch.equal(same, got) and all(torch.equal(a, b) for a, b in zip(ts, out))


SIZES = [[1], [7], [0, 5, 0], [2048], [2049, 1, 4095], [3] * 129, [100_003], [1_000_001, 17, 262_144]]


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("sizes", SIZES)
def test_sizes(sizes, types, p):
    ts = make(sizes, types, 1)
    check(ts, 0.25, p)
    check(make(sizes, types, 2), 1e9, p)


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0])
@pytest.mark.parametrize("types", [[t] for t in TYPES] + [TYPES])
def test_bounds_of_the_present_batch(types, p):
    """A thread adds at most 32 values (16 of float32) in four running sums before they become 64-bit: 8 roundings of a sum's squares, 7 of
    its magnitudes, 2 to join the four, the root halves them and its rounding to float32 adds one: 6 * 2^-24, and 10 for the magnitudes; one
    more of each covers the 64-bit sums. Values whose squares round the same way are among them."""
    bound = {2.0: 7 * U, 1.0: 11 * U}[p]
    sets = [make(sizes, types, 11) for sizes in ([100_003], [2048, 33, 4095], [1_000_001, 17, 262_144])]
    same = [torch.full((70_001,), 1.0 + 2 ** -k, dtype=t, device="cuda") for t in types for k in (3, 6, 7)]
    for ts in sets + [same]:
        n = ref_norm(ts, p)
        assert abs(float(grad_norm(ts, p)) - n) <= bound * n


@gpu
def test_more_tensors_than_one_launch_takes():
    ts = make([1 + i % 37 for i in range(2500)], TYPES, 3)
    check(ts, 1.0, 2.0)


@gpu
def test_large():
    ts = make([40_000_003, 9], [torch.bfloat16], 4)
    check(ts, 3.0, 2.0)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 3])
def test_off_vector_boundaries(dtype, shift):
    """Views at element addresses; outputs at the same and at other offsets."""
    flat = make([50_000], [dtype], 5)[0]
    ts = [flat[shift:20_001], flat[20_001:20_004], flat[20_004:]]
    room = torch.full((50_010,), 7.0, dtype=dtype, device="cuda")
    for off in (shift, shift + 1, 8):
        room.fill_(7.0)
        at, outs = off, []
        for t in ts:
            outs.append(room[at:at + t.numel()])
            at += t.numel()
        got, norm = clip_grads(ts, 0.5, out=outs)
        want, norm2 = clip_grads([t.clone() for t in ts], 0.5)
        assert torch.equal(norm, norm2) or abs(float(norm) - float(norm2)) <= 2 * ERR[2.0] * float(norm)
        for a, b in zip(got, want):
            assert ((a.double() - b.double()).abs() <= (2 * ERR[2.0] + 2 * half_step(dtype) + 4 * U) * b.double().abs()
                    + 2 * tiny(dtype)).all()
        assert (room[:off] == 7.0).all() and (room[at:] == 7.0).all()


@gpu
def test_strides():
    g = torch.Generator().manual_seed(6)
    base = torch.randn(40, 60, generator=g).cuda()
    a, b = base.clone().t(), base.clone()[:, ::2]            # dense but transposed; with gaps
    c = torch.randn(2, 3, 4, 5, generator=g).cuda().to(memory_format=torch.channels_last)
    ts = [a, b, c]
    before = [t.clone() for t in ts]
    n = ref_norm(before, 2)
    out, norm = clip_grads(ts, 1.0)
    assert abs(float(norm) - n) <= ERR[2.0] * n
    clip_grads_(ts, 1.0)
    for t, o, w in zip(ts, out, before):
        assert torch.equal(t, o)
        assert torch.allclose(t.double(), w.double() * (1.0 / (n + 1e-6)), rtol=32 * U, atol=0)


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e25, 1e37])
def test_magnitudes(scale):
    """Squares outside fp32's range. A norm above float32's largest number (7.1e38 for 1e37) is inf as a float32."""
    ts = make([5000, 3], [torch.float32], 7, scale)
    n = ref_norm(ts, 2)
    if n > torch.finfo(torch.float32).max:
        assert float(grad_norm(ts)) == math.inf
    else:
        assert abs(float(grad_norm(ts)) - n) <= ERR[2.0] * n + tiny(torch.float32)
    n = ref_norm(ts, 1)
    if n < 3e38:
        assert abs(float(grad_norm(ts, 1)) - n) <= ERR[1.0] * n


@gpu
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_nan_and_inf(p):
    ts = make([3000, 10], [torch.float32], 8)
    ts[0][2999] = math.inf
    n = clip_grads_(ts, 1.0, p)
    assert float(n) == math.inf and float(ts[1].abs().max()) == 0.0 and math.isnan(float(ts[0][2999]))
    ts = make([3000, 10], [torch.float16], 8)
    ts[1][3] = math.nan
    n = clip_grads_(ts, 1.0, p)
    assert math.isnan(float(n)) and all(t.isnan().all() for t in ts)
    zeros = [torch.zeros(5000, device="cuda")]
    assert float(clip_grads_(zeros, 1.0, p)) == 0.0 and not zeros[0].any()


@gpu
def test_within_the_limit_is_left_alone():
    ts = make([1000], [torch.float32], 9)
    n = float(grad_norm(ts))
    before = ts[0].clone()
    clip_grads_(ts, n * 1.01)
    assert torch.equal(ts[0], before)
    clip_grads_(ts, 0.0)
    assert not ts[0].any()


@gpu
def test_parameters_as_torch():
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.ELU(), torch.nn.Linear(65, 7)).cuda()
    x = torch.randn(20, 33, device="cuda")

    def back():
        m.zero_grad(set_to_none=True)
        m(x).square().sum().backward()
    back()
    m[2].bias.grad = None
    want = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.5)
    ref = [p.grad for p in m.parameters()]
    back()
    m[2].bias.grad = None
    version = m[0].weight.grad._version
    got = clip_grad_norm_(m.parameters(), 0.5, error_if_nonfinite=True)
    assert m[0].weight.grad._version > version
    assert torch.allclose(got, want, rtol=40 * U)
    for p, r in zip(m.parameters(), ref):
        assert (p.grad is None) == (r is None)
        if r is not None:
            assert torch.allclose(p.grad, r, rtol=80 * U, atol=0)
    m[0].weight.grad[0, 0] = math.nan
    keep = m[0].weight.grad.clone()
    with pytest.raises(RuntimeError, match="not clipped"):
        clip_grad_norm_(m.parameters(), 0.5, error_if_nonfinite=True)
    assert torch.equal(keep[1:], m[0].weight.grad[1:])


@gpu
def test_graph_stream_and_repeats():
    ts = make([70_001, 3, 900], TYPES, 10)
    outs = [torch.empty_like(t) for t in ts]
    first, n0 = clip_grads(ts, 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again, n1 = clip_grads(ts, 0.5)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, n2 = clip_grads(ts, 0.5, out=outs)
    ts[0].mul_(3.0)
    graph.replay()
    want, n3 = clip_grads(ts, 0.5)
    assert torch.equal(n2, n3) and all(torch.equal(a, b) for a, b in zip(outs, want))


@gpu
def test_inference_mode():
    with torch.inference_mode():
        t = torch.ones(100, device="cuda")
        assert float(clip_grads_([t], 1.0)) == 10.0


def test_no_tensors():
    assert float(grad_norm([])) == 0.0 and float(clip_grads_([], 1.0)) == 0.0
    assert clip_grads([], 1.0)[0] == []
    p = torch.nn.Parameter(torch.ones(3))
    assert float(clip_grad_norm_(p, 1.0, error_if_nonfinite=True)) == 0.0


def test_refusals():
    t = torch.ones(4)
    for bad in (3.0, 0.5, -math.inf):
        with pytest.raises(ValueError, match="norm_type"):
            grad_norm([t], bad)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads_([t], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        clip_grads([t], math.nan)
    with pytest.raises(TypeError, match="float64"):
        grad_norm([t.double()])
    with pytest.raises(TypeError, match="dense"):
        grad_norm([t.to_sparse()])
    with pytest.raises(TypeError, match="tensors"):
        grad_norm([1.0])
    with pytest.raises(ValueError, match="tensors on"):
        grad_norm([t, torch.ones(3, device="meta")])
    with pytest.raises(ValueError, match="in out"):
        clip_grads([t], 1.0, out=[])
    with pytest.raises(RuntimeError, match="CUDA"):
        grad_norm([t])
    leaf = torch.ones(3, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        clip_grads([leaf], 1.0)
    with pytest.raises(RuntimeError, match="no gradient"):
        grad_norm([leaf])


@gpu
def test_shared_memory_is_refused():
    x = torch.ones(10, device="cuda")
    for ts in ([x, x], [x[:6], x[5:]]):
        with pytest.raises(ValueError, match="share memory"):
            clip_grads_(ts, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_grads_([torch.ones(1, device="cuda").expand(4)], 1.0)
    five = torch.ones(5, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        clip_grads([x[:5], five], 1.0, out=[five.clone(), x[4:9]])
    assert (x == 1).all()
    out, n = clip_grads([x[:5], x[5:]], 1.0, out=[x[:5], x[5:]])        # in place
    assert torch.allclose(x, torch.full_like(x, 10 ** -0.5), rtol=1e-6)
    with pytest.raises(ValueError, match="does not match"):
        clip_grads([x], 1.0, out=[x[:9]])
    with pytest.raises(ValueError, match="does not match"):
        clip_grads([x], 1.0, out=[torch.ones(10)])
    with pytest.raises(ValueError, match="strides"):
        clip_grads([torch.ones(3, 4, device="cuda")], 1.0, out=[torch.ones(4, 3, device="cuda").t()])


def test_the_library_finds_shared_memory():
    """The C entry's own check, on host addresses that nothing reads: it comes before any launch."""
    import ctypes

    from rl_quant_b200 import _native as N
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    lib = N.load()

    def call(src, dst, sizes):
        n = len(src)
        arr = lambda t, v: (t * n)(*v)  # noqa: E731
        return lib.glad_clip_grads(arr(ctypes.c_uint64, src), arr(ctypes.c_uint64, dst), arr(ctypes.c_int64, sizes),
                                   arr(ctypes.c_int32, [N.DTYPE_F32] * n), n, 2, 1.0, at + 2048, None, 0, None)
    for src, dst, sizes in (([at, at], [at, at], [4, 4]), ([at, at + 12], [at, at + 12], [4, 4]),
                            ([at, at + 64], [at + 128, at + 64], [40, 4]), ([at], [at + 8], [4])):
        assert call(src, dst, sizes) == N.GLAD_ERR_INVALID_ARG and b"share" in lib.glad_last_error()
    for src, dst, sizes in (([at, at + 16], [at, at + 16], [4, 4]), ([at, at], [at, at + 64], [0, 4])):
        assert call(src, dst, sizes) == N.GLAD_ERR_WORKSPACE
