"""GPU: the sequence operators (layer_norm, gru_scan, gated_mlp) against plain forms in 64 bits.

Tolerances count roundings: an output of type T is off by at most half a step, finfo(T).eps / 2 relative to its value -- and to the smallest
normal number below that one, where the steps stay as they are there (fp16: 2^-14 x 2^-11) --, every fp32 operation on the way by 2^-24 of its
result.  A sum of n values taken in any order is off by at most (its longest chain of additions) x 2^-24
x the sum of their absolute values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype, value):
    f = torch.finfo(dtype)
    return f.eps / 2 * value.abs().clamp_min(f.smallest_normal)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol):
    got, want = got.detach().double(), want.double()
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        t = tol.expand_as(want).reshape(-1)[i] if torch.is_tensor(tol) else tol
        raise AssertionError("%d of %d values off; first at %d: %r, wanted %r within %r" % (int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]),
                                                                                       float(want.reshape(-1)[i]), float(t)))


@pytest.fixture(scope="module")
def ops():
    from motif_amd import ops
    return ops


# ------------------------------------------------------------------------------------------------------------------ layer_norm
def ln_reference(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits, and the magnitudes that their tolerances are made of."""
    x, dy = x.double(), dy.double()
    d = x.shape[-1]
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    m = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
    n = (x - m) * r
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    # n: the chain of the two row sums (16 values in a lane, up to 10 levels and 16 partial sums above) and a few operations: 48 roundings of
    # values up to max |x| r; a relative error of r comes from the squares' sum (48 again, relative) and the root
    en = 48 * F32 * ((x.abs().amax(-1, keepdim=True) * r) + 2 * n.abs())
    ey = en * w.abs() + 4 * F32 * (n * w).abs() + 2 * F32 * b.abs()
    # dx: both means (48 roundings of mean |.|), n's error through the last term twice
    mg, mgn = g.abs().mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    edx = r * (52 * F32 * (g.abs() + mg + n.abs() * mgn) + en * mgn + n.abs() * (g.abs() * en).mean(-1, keepdim=True)) + 100 * F32 * dx.abs()
    return (n * w + b, dx, (dy * n).sum(rows), dy.sum(rows)), (ey, edx, en), (n, g)


def ln_check(ops, x, w, b, eps=1e-5, dy=None, seed=0):
    dy = torch.randn(x.shape, generator=gen(seed + 99), device="cuda").to(x.dtype) if dy is None else dy
    (y0, dx0, dw0, db0), (ey, edx, en), (n, g) = ln_reference(x, w, b, dy, eps)
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    it = iter(leaves)
    xl, wl, bl = next(it), next(it) if w is not None else None, next(it) if b is not None else None
    y = ops.layer_norm(xl, wl, bl, eps)
    assert y.dtype == x.dtype and y.shape == x.shape
    within(y, y0, half_step(x.dtype, y0) + ey)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps), y), "with and without gradients: the same bits"
    got = torch.autograd.grad(y, leaves, dy)
    within(got[0], dx0, half_step(x.dtype, dx0) + edx)
    rows = tuple(range(x.dim() - 1))
    count = x.numel() // x.shape[-1]
    chain = count / 256 + 80                              # rows of one lane, its workgroup's slots, the partial sums (an upper bound)
    if w is not None:
        t = (dy.double() * n).abs().sum(rows)
        within(got[1], dw0, half_step(w.dtype, dw0) + chain * F32 * t + (dy.double().abs() * en).sum(rows))
    if b is not None:
        within(got[-1], db0, half_step(b.dtype, db0) + chain * F32 * dy.double().abs().sum(rows))
    return y, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, d", [(1, 1), (3, 2), (5, 63), (17, 64), (1, 65), (33, 256), (7, 257), (6, 1000), (1030, 1001), (5, 1024), (3, 1028),
                                     (2, 4096), (4, 4097), (2, 16384), (1, 16383), (70000, 48), (2051, 520)])
def test_layer_norm_and_its_gradients(ops, dtype, rows, d):
    g = gen(rows + d)
    x = (torch.randn(rows, d, generator=g, device="cuda") * 1.5 + 0.3).to(dtype)
    w = (torch.randn(d, generator=g, device="cuda") * 0.2 + 1).to(dtype)
    b = (torch.randn(d, generator=g, device="cuda") * 0.2).to(dtype)
    ln_check(ops, x, w, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["columns", "odd columns", "every second row", "transposed", "four axes", "broadcast rows", "misaligned"])
def test_layer_norm_takes_strided_inputs(ops, dtype, kind):
    g = gen(5)
    base = (torch.randn(24, 1056, generator=g, device="cuda") + 0.1).to(dtype)
    x = {"columns": base[:, 32:544], "odd columns": base[:, 3:515], "every second row": base[::2, :512], "transposed": base[:, :24].t()[:, :20],
         "four axes": base.view(2, 3, 4, 1056).permute(1, 0, 2, 3)[..., :264], "broadcast rows": base[:1, :512].expand(9, 512),
         "misaligned": base.reshape(-1)[1:1 + 24 * 1000].view(24, 1000)}[kind]
    w = torch.randn(x.shape[-1], generator=g, device="cuda").to(dtype)
    dy = torch.randn(x.shape, generator=g, device="cuda").to(dtype)
    y, got = ln_check(ops, x, w, None, dy=dy)
    yc, gotc = ln_check(ops, x.clone(memory_format=torch.contiguous_format), w, None, dy=dy)
    assert torch.equal(y, yc) or kind in ("odd columns", "misaligned"), "another layout of the same rows changes no bits (but lanes' shares where alignment differs)"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_takes_fp32_parameters(ops, dtype):
    g = gen(6)
    x = torch.randn(37, 320, generator=g, device="cuda").to(dtype)
    w, b = torch.randn(320, generator=g, device="cuda"), torch.randn(320, generator=g, device="cuda")
    ln_check(ops, x, w, b)
    ln_check(ops, x, None, b)
    ln_check(ops, x, w, None)
    ln_check(ops, x, None, None)


def test_layer_norm_of_constant_rows_of_large_offsets_and_of_nothing(ops):
    x = torch.full((4, 96), 3.25, device="cuda")
    y = ops.layer_norm(x)
    assert torch.equal(y, torch.zeros_like(y))
    x = torch.randn(8, 512, generator=gen(1), device="cuda") + 1000.0      # the mean is 1000 times the spread: the squares are of differences
    ln_check(ops, x, None, None)
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert y.shape == (0, 64) and dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(dw))


def test_layer_norm_keeps_a_bad_row_to_itself(ops):
    x = torch.randn(40, 200, generator=gen(2), device="cuda")
    want = ops.layer_norm(x)
    bad = x.clone()
    bad[3, 7], bad[20, 0], bad[39, 199] = math.inf, math.nan, -math.inf
    got = ops.layer_norm(bad)
    rows = [i for i in range(40) if i not in (3, 20, 39)]
    assert torch.equal(got[rows], want[rows])
    assert all(torch.isnan(got[i]).any() for i in (3, 20, 39))


def test_layer_norm_gradient_against_differences(ops):
    g = gen(3)
    x, w, b = (torch.randn(s, generator=g, device="cuda") for s in ((6, 80), (80,), (80,)))
    dy = torch.randn(6, 80, generator=g, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    with torch.no_grad():
        for i, t in enumerate(leaves):
            way = torch.randn(t.shape, generator=g, device="cuda")
            h = 2.0 ** -7
            f = [(ops.layer_norm(*[v + s * h * way if j == i else v for j, v in enumerate(leaves)]).double() * dy.double()).sum() for s in (1, -1)]
            got, want = float((f[0] - f[1]) / (2 * h)), float((grads[i].double() * way.double()).sum())
            # the third derivative's share h^2 / 6 (order 1 x the sum's size), and 2 x 480 values rounded at 2^-24 over 2 h
            size = float((dy.double().abs()).sum()) * 8
            assert abs(got - want) <= size * (h * h / 6 * 8 + 64 * F32 / h), (got, want)


def test_layer_norm_gives_the_same_bits_every_time_on_any_stream_and_in_a_graph(ops):
    g = gen(4)
    x, w, b, dy = (torch.randn(s, generator=g, device="cuda") for s in ((3001, 192), (192,), (192,), (3001, 192)))
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = ops.layer_norm(*leaves)
        return (y,) + torch.autograd.grad(y, leaves, dy)
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [t.detach().clone() for t in step()]           # (no eager graph of these leaves lives into the capture)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for k in range(3):
        for t in held:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want)), k
    with torch.no_grad():
        x.copy_(x * 2)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))
