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
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()                                   # (y is detached: no eager graph of these leaves lives into the capture)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for k in range(3):
        for t in held:
            t.zero_()
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


# ------------------------------------------------------------------------------------------------------------------ gru_scan
def scan_reference(z, q, h0, dh, dlast):
    """One batch of whole sequences [B, T, D], row by row in 64 bits: h, last, dz, dq, dh0, and bounds of the errors that fp32 sums carry.
    mh_t is the same recurrence on absolute values: every product and sum on the way is at most that."""
    z, q, dh, dlast = z.double(), q.double(), dh.double(), dlast.double()
    B, T, D = z.shape
    s = torch.zeros(B, D, dtype=torch.float64, device=z.device) if h0 is None else h0.double()
    h, mh, m, first = [], [], s.abs(), s
    a = 1 - z
    for t in range(T):
        s = a[:, t] * s + z[:, t] * q[:, t]
        m = a[:, t].abs() * m + (z[:, t] * q[:, t]).abs()
        h.append(s)
        mh.append(m)
    dz, dq, c, mc = torch.zeros_like(z), torch.zeros_like(z), dlast, dlast.abs()
    mg, mb = torch.zeros_like(z), torch.zeros_like(z)
    for t in range(T - 1, -1, -1):
        g, mg[:, t] = c + dh[:, t], mc + dh[:, t].abs()
        before = h[t - 1] if t else first
        dz[:, t], dq[:, t] = g * (q[:, t] - before), g * z[:, t]
        mb[:, t] = mh[t - 1] if t else first.abs()
        c, mc = a[:, t] * g, a[:, t].abs() * mg[:, t]
    last = s
    return (torch.stack(h, 1) if T else q.clone(), last, dz, dq, c), (torch.stack(mh, 1) if T else q.clone(), m, mg, mb, mc)


# Roundings that one value collects relative to the magnitudes above: a row adds three (1 - z, the product, the sum), and what is older than
# the last n rows has shrunk by prod(1 - z); in the worst case, z = 0, every row adds 3.  A composition of runs replaces additions of rows by
# as many of runs.  chain(T) = 3 T + 64 is safe whatever z is.
def chain(T):
    return (3 * T + 64) * F32


def scan_check(ops, z, q, h0, cu=None, seed=0, grads=True):
    g = gen(seed + 7)
    S = (cu.numel() - 1) if cu is not None else z.shape[0]
    D = z.shape[-1]
    dh = torch.randn(z.shape, generator=g, device="cuda").to(z.dtype)
    dlast = torch.randn(S, D, generator=g, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (z, q, h0) if t is not None]
    hl = leaves[2] if h0 is not None else None
    h, last = ops.gru_scan(leaves[0], leaves[1], hl, cu_seqlens=cu)
    assert h.dtype == q.dtype and h.shape == q.shape and last.dtype == torch.float32 and last.shape == (S, D)
    with torch.no_grad():
        h2, last2 = ops.gru_scan(z, q, h0, cu_seqlens=cu)
    assert torch.equal(h, h2) and torch.equal(last, last2)
    got = torch.autograd.grad([h, last], leaves, [dh, dlast])
    spans = [(slice(i, i + 1), lo, hi) for i, (lo, hi) in enumerate(zip(cu.tolist(), cu.tolist()[1:]))] if cu is not None else [(slice(None), 0, z.shape[1])]
    cut = (lambda x, lo, hi: x[lo:hi].unsqueeze(0)) if cu is not None else (lambda x, lo, hi: x)
    for own, lo, hi in spans:
        (h0r, lr, dzr, dqr, dh0r), (mh, ml, mg, mb, mc) = scan_reference(cut(z, lo, hi), cut(q, lo, hi), None if h0 is None else h0[own], cut(dh, lo, hi), dlast[own])
        e = chain(hi - lo)
        if hi > lo:
            within(cut(h, lo, hi), h0r, half_step(q.dtype, h0r) + e * mh)
        within(last[own], lr, e * ml)
        if hi > lo:
            # dz = g (q - h_{t-1}): g's error, and h_{t-1} as it was written, half a step of its type off
            qb = cut(q, lo, hi).double().abs() + mb
            within(cut(got[0], lo, hi), dzr, half_step(q.dtype, dzr) * (1 + 2 ** -6) + 2 * e * mg * qb + mg * half_step(q.dtype, mb) * (1 + 2 ** -6))
            within(cut(got[1], lo, hi), dqr, half_step(q.dtype, dqr) + e * mg * cut(z, lo, hi).double().abs())
        if h0 is not None:
            within(got[2][own], dh0r, e * mc)
    if cu is not None:
        covered = torch.zeros(z.shape[0], dtype=torch.bool)
        for _, lo, hi in spans:
            covered[lo:hi] = True
        behind = (~covered).cuda()
        for t in (h, got[0], got[1]):
            assert torch.equal(t[behind], torch.zeros_like(t[behind])), "rows that no sequence covers"
    return h, last, got


def scan_inputs(shape, S, dtype, seed, shift=-2.0):
    g = gen(seed)
    z = torch.sigmoid(torch.randn(*shape, generator=g, device="cuda") * 1.5 + shift).to(dtype)
    q = torch.tanh(torch.randn(*shape, generator=g, device="cuda")).to(dtype)
    return z, q, torch.randn(S, shape[-1], generator=g, device="cuda") * 0.5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, T, D", [(1, 1, 1), (3, 1, 64), (2, 2, 7), (1, 16, 128), (1, 17, 128), (2, 127, 33), (1, 128, 64), (3, 129, 72), (1, 1000, 8), (1, 4099, 24),
                                     (1, 3000, 5), (5, 300, 520), (1, 40, 140000), (2, 7, 4096), (600, 20, 40)])
def test_gru_scan_and_its_gradients(ops, dtype, B, T, D):
    z, q, h0 = scan_inputs((B, T, D), B, dtype, B * 7 + T + D)
    scan_check(ops, z, q, h0)
    if T <= 200:
        scan_check(ops, z, q, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 24, 33, 64, 136, 1100])
@pytest.mark.parametrize("bounds, T", [([0, 5], 5), ([0, 0, 1, 1, 1, 40, 41, 300, 300], 310), ([3, 3, 10, 700], 700), ([0, 0, 0], 4), ([0, 0], 0),
                                       ([0, 1, 2, 3, 131, 259, 388, 1500, 1501, 3999], 4001)])
def test_gru_scan_of_packed_sequences(ops, dtype, D, bounds, T):
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    z, q, h0 = scan_inputs((T, D), len(bounds) - 1, dtype, T + D)
    covered = torch.zeros(T, dtype=torch.bool, device="cuda")
    for lo, hi in zip(bounds, bounds[1:]):
        covered[lo:hi] = True
    z[~covered], q[~covered] = math.nan, math.inf
    scan_check(ops, z, q, h0, cu)
    if D == 24:
        scan_check(ops, z, q, None, cu)


def test_gru_scan_packed_equals_the_sequences_alone(ops):
    bounds = [0, 300, 300, 301, 700, 1211]
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    z, q, h0 = scan_inputs((1211, 40), 5, torch.float32, 3)
    h, last = ops.gru_scan(z, q, h0, cu_seqlens=cu)
    for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if hi == lo:
            assert torch.equal(last[i], h0[i])
            continue
        alone, end = ops.gru_scan(z[None, lo:hi], q[None, lo:hi], h0[i:i + 1])
        m = 2 * chain(hi - lo)                            # both are within chain() of the exact state, |h| <= 1 + |h0|
        within(h[None, lo:hi], alone, m * (1 + h0[i].abs().double()))
        within(last[i:i + 1], end, m * (1 + h0[i].abs().double()))


def test_gru_scan_in_pieces_down_to_single_rows_continues_the_state(ops):
    z, q, h0 = scan_inputs((2, 50, 96), 2, torch.float32, 4)
    whole, last = ops.gru_scan(z, q, h0)
    state, rows = h0, []
    for lo, hi in [(0, 20), (20, 21), (21, 22), (22, 22), (22, 50)]:
        h, state = ops.gru_scan(z[:, lo:hi], q[:, lo:hi], state)
        rows.append(h)
    m = 2 * chain(50) * 3
    within(torch.cat(rows, 1), whole, m)
    within(state, last, m)
    one = ops.gru_update(z[:, 0].contiguous(), q[:, 0].contiguous(), h0)
    within(ops.gru_scan(z[:, :1], q[:, :1], h0)[1], one, 8 * F32 * 4)


@pytest.mark.parametrize("kind", ["columns", "odd columns", "time first", "every second row", "broadcast gate", "transposed"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gru_scan_takes_strided_inputs(ops, dtype, kind):
    z0, q0, _ = scan_inputs((4, 320, 160), 4, dtype, 9)
    pick = {"columns": lambda x: x[:, :, 32:96], "odd columns": lambda x: x[:, :, 3:67], "time first": lambda x: x.transpose(0, 1)[:150],
            "every second row": lambda x: x[:, ::2], "broadcast gate": lambda x: x[:1].expand(4, 320, 160), "transposed": lambda x: x.transpose(1, 2)}[kind]
    z, q = pick(z0), (q0 if kind == "broadcast gate" else pick(q0))
    h0 = torch.randn(z.shape[0], z.shape[2], generator=gen(1), device="cuda")
    scan_check(ops, z, q, h0)


def test_gru_scan_gates_at_their_ends_and_bad_values_stay_in_their_channel(ops):
    z, q, h0 = scan_inputs((1, 700, 64), 1, torch.float32, 5)
    z[:, ::3], z[:, 1::3] = 0.0, 1.0                      # keep all / take all
    scan_check(ops, z, q, h0)
    want, wl = ops.gru_scan(z * 0.5, q, h0)
    bad = q.clone()
    bad[0, 300, 5], bad[0, 10, 40] = math.inf, math.nan
    got, gl = ops.gru_scan(z * 0.5, bad, h0)
    keep = [c for c in range(64) if c not in (5, 40)]
    assert torch.equal(got[..., keep], want[..., keep]) and torch.equal(gl[:, keep], wl[:, keep])
    assert torch.equal(got[:, :300, 5], want[:, :300, 5]) and torch.equal(got[:, :10, 40], want[:, :10, 40])


def test_gru_scan_of_no_rows_and_no_sequences(ops):
    h0 = torch.randn(3, 8, device="cuda", requires_grad=True)
    z = torch.empty(3, 0, 8, device="cuda", requires_grad=True)
    h, last = ops.gru_scan(z, z.detach(), h0)
    assert h.shape == (3, 0, 8) and torch.equal(last, h0)
    dz, dh0 = torch.autograd.grad(last, (z, h0), torch.ones_like(last))
    assert dz.shape == z.shape and torch.equal(dh0, torch.ones_like(dh0))
    z = torch.empty(0, 5, 8, device="cuda")
    h, last = ops.gru_scan(z, z)
    assert h.shape == (0, 5, 8) and last.shape == (0, 8)


def test_gru_scan_gradient_against_differences(ops):
    g = gen(11)
    z, q, h0 = scan_inputs((2, 150, 16), 2, torch.float32, 6)
    leaves = [t.requires_grad_() for t in (z, q, h0)]
    dh, dl = torch.randn(2, 150, 16, generator=g, device="cuda"), torch.randn(2, 16, generator=g, device="cuda")
    grads = torch.autograd.grad(ops.gru_scan(*leaves), leaves, (dh, dl))
    with torch.no_grad():
        for i, t in enumerate(leaves):
            way = torch.randn(t.shape, generator=g, device="cuda")
            h = 2.0 ** -10
            f = []
            for s in (1, -1):
                a, b = ops.gru_scan(*[v + s * h * way if j == i else v for j, v in enumerate(leaves)])
                f.append(float((a.double() * dh.double()).sum() + (b.double() * dl.double()).sum()))
            got, want = (f[0] - f[1]) / (2 * h), float((grads[i].double() * way.double()).sum())
            # linear in q and h0; in z the cubic share is h^2 / 6 x (third differences of products of up to 150 gates, each |way| / 0.1)
            size = float(dh.double().abs().sum() + dl.double().abs().sum())
            assert abs(got - want) <= size * (chain(150) / h + h * h / 6 * 1000), (i, got, want)


def test_gru_scan_gives_the_same_bits_every_time_on_any_stream_and_in_a_graph(ops):
    cu = torch.tensor([0, 100, 100, 2500, 2990], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    for args, c in ((scan_inputs((3000, 72), 4, torch.float32, 8), cu), (scan_inputs((2, 1500, 96), 2, torch.bfloat16, 8), None)):
        z, q, h0 = leaves = [t.requires_grad_() for t in args]
        dh, dl = torch.ones_like(q.detach()), torch.ones_like(h0.detach())

        def step():
            h, last = ops.gru_scan(z, q, h0, cu_seqlens=c)
            return (h.detach(), last.detach()) + torch.autograd.grad((h, last), leaves, (dh, dl))
        want = [t.clone() for t in step()]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for k in range(3):
            for t in held:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), k
            assert all(torch.equal(a, b) for a, b in zip(step(), want)), k
            torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------------------------ gated_mlp
def gate_reference(g, act):
    s, rest = torch.sigmoid(g), torch.sigmoid(-g)          # 1 - s: not as a difference, which is 0 from g = 37 on
    if act == "sigmoid":
        return s, s * rest
    if act == "silu":
        return g * s, s * (1 + g * rest)
    phi = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def mlp_check(ops, x, wg, wu, bg, bu, act, seed=0):
    """Against 64 bits.  A product of n terms in fp32 is off by at most c(n) x the sum of the terms' absolute values: n / 32 accumulations of the
    matrix instruction with up to 32 roundings inside (n + 64 in all, counted fully: c(n) = (n + 64) x 2^-24).  fp32 data: three parts lose three
    products of at most 2^-23 each, and add six times the accumulations.  Every |.| below is of the exact values."""
    dt = x.dtype
    M, K, F = x.numel() // x.shape[-1], x.shape[-1], wg.shape[0]
    dh = torch.randn(x.shape[:-1] + (F,), generator=gen(seed + 5), device="cuda").to(dt)
    many = 6 if dt == torch.float32 else 1
    c = lambda n: (many * n + 64) * F32 + (3 * 2.0 ** -23 if many > 1 else 0)  # noqa: E731
    params = [x, wg, wu, bg, bu]
    leaves = [None if t is None else t.detach().requires_grad_() for t in params]
    h = ops.gated_mlp(*leaves, act=act)
    assert h.dtype == dt and h.shape == x.shape[:-1] + (F,)
    with torch.no_grad():
        assert torch.equal(ops.gated_mlp(*params, act=act), h)
    live = [t for t in leaves if t is not None]
    got = dict(zip([n for n, t in zip(("x", "wg", "wu", "bg", "bu"), leaves) if t is not None], torch.autograd.grad(h, live, dh)))
    X, WG, WU, DH = x.double().reshape(M, K), wg.double(), wu.double(), dh.double().reshape(M, F)
    G, U = X @ WG.t(), X @ WU.t()
    eG, eU = c(K) * (X.abs() @ WG.abs().t()), c(K) * (X.abs() @ WU.abs().t())
    if bg is not None:
        G, eG = G + bg.double(), eG + F32 * (G.abs() + bg.double().abs())
    if bu is not None:
        U, eU = U + bu.double(), eU + F32 * (U.abs() + bu.double().abs())
    v, dv = gate_reference(G, act)
    # the activations: |act'| <= 1.13, |act''| <= 1; v_exp_f32 and v_rcp_f32 on g to 2^-24 (|g| + 4) relative of the sigmoid; erff, expf a few places
    rel = (16 + 2 * G.abs()) * F32
    ev = 1.13 * eG + rel * v.abs() + (16 * F32 * G.abs() if act == "gelu" else 0)
    edv = eG + rel * (dv.abs() + 1)
    within(h.reshape(M, F), v * U, half_step(dt, v * U) + 1.001 * (ev * U.abs() + eU * v.abs() + ev * eU) + 2 * F32 * (v * U).abs())
    dG, dU = DH * U * dv, DH * v
    # rounded once to operands (fp32: kept to 2^-23 by their parts)
    step = (lambda t: half_step(dt, t)) if many == 1 else (lambda t: 2.0 ** -23 * t.abs())
    edG = DH.abs() * (eU * dv.abs() + edv * U.abs() + eU * edv) + 4 * F32 * dG.abs()
    edU = DH.abs() * ev + 4 * F32 * dU.abs()
    rG, rU = edG + 1.01 * step(dG.abs() + edG), edU + 1.01 * step(dU.abs() + edU)
    dx = dG @ WG + dU @ WU
    tx = rG @ WG.abs() + rU @ WU.abs() + c(2 * F) * (dG.abs() @ WG.abs() + dU.abs() @ WU.abs())
    within(got["x"].reshape(M, K), dx, half_step(dt, dx) + 1.01 * tx)
    for n, d, r in (("wg", dG, rG), ("wu", dU, rU)):
        w = d.t() @ X
        within(got[n], w, half_step(dt, w) + 1.01 * (r.t() @ X.abs() + c(M) * (d.abs().t() @ X.abs())))
    for n, d, e in (("bg", dG, edG), ("bu", dU, edU)):
        if n in got:
            within(got[n], d.sum(0), half_step(dt, d.sum(0)) + 1.01 * (e.sum(0) + (64 + M / 64) * F32 * d.abs().sum(0)))
    return h, got


def mlp_inputs(M, K, F, dtype, seed, bias):
    g = gen(seed)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)  # noqa: E731
    x, wg, wu = n(M, K), n(F, K, scale=K ** -0.5), n(F, K, scale=K ** -0.5)
    return x, wg, wu, n(F, scale=0.2) if bias else None, n(F, scale=0.2) if bias else None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K, F, act, bias", [(1, 1, 1, "silu", True), (1, 64, 64, "gelu", False), (3, 40, 17, "sigmoid", True), (16, 33, 100, "silu", False),
                                                (17, 128, 48, "gelu", True), (33, 100, 130, "silu", True), (64, 72, 31, "sigmoid", False), (65, 32, 64, "silu", True),
                                                (65, 31, 65, "gelu", True), (127, 64, 63, "silu", False), (128, 96, 128, "gelu", False), (129, 160, 129, "sigmoid", True),
                                                (300, 1000, 70, "silu", True), (1030, 48, 258, "gelu", True), (4100, 64, 40, "silu", False), (70, 520, 2050, "gelu", False)])
def test_gated_mlp_and_its_gradients(ops, dtype, M, K, F, act, bias):
    mlp_check(ops, *mlp_inputs(M, K, F, dtype, M + K + F, bias), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K, F, act, bias", [(65, 4, 8, "silu", True), (1, 8, 16, "gelu", True), (66, 16, 24, "sigmoid", False), (100, 20, 40, "gelu", True),
                                                (1000, 32, 64, "silu", True), (333, 36, 72, "silu", False), (1001, 60, 136, "gelu", True), (9001, 64, 248, "sigmoid", True),
                                                (9000, 64, 256, "gelu", False), (700, 64, 264, "silu", True), (5003, 28, 96, "silu", True), (130, 64, 2064, "gelu", True)])
def test_gated_mlp_of_narrow_layers(ops, dtype, M, K, F, act, bias):
    """K up to 64: weights in registers, the backward pass in one; columns of less than a wave's 32, rows that end within a workgroup's share."""
    mlp_check(ops, *mlp_inputs(M, K, F, dtype, M + K + F, bias), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["columns", "odd columns", "broadcast rows", "transposed", "one bias"])
def test_gated_mlp_of_narrow_layers_takes_strided_inputs(ops, dtype, kind):
    x, wg, wu, bg, bu = mlp_inputs(300, 48, 72, dtype, 3, True)
    base = torch.randn(300, 160, generator=gen(4), device="cuda").to(dtype)
    if kind == "columns":
        x = base[:, 32:80]
    elif kind == "odd columns":
        x = base[:, 3:51]
    elif kind == "broadcast rows":
        x = base[:1, :48].expand(300, 48)
    elif kind == "transposed":
        x = torch.randn(48, 300, generator=gen(5), device="cuda").to(dtype).t()
    else:
        bu = None
    mlp_check(ops, x, wg, wu, bg, bu, "gelu")


def test_gated_mlp_of_narrow_layers_keeps_bad_rows_to_themselves(ops):
    for dtype in DTYPES:
        x, wg, wu, bg, bu = mlp_inputs(300, 36, 72, dtype, 6, True)
        dh = torch.randn(300, 72, generator=gen(7), device="cuda").to(dtype)

        def step(x, dh):
            x = x.detach().requires_grad_()
            h = ops.gated_mlp(x, wg.detach().requires_grad_(), wu, bg, bu)
            return h.detach(), torch.autograd.grad(h, x, dh, retain_graph=True)[0]
        want = step(x, dh)
        bad, bad_dh = x.clone(), dh.clone()
        bad[3, 7], bad[299, 35], bad_dh[17, 70] = math.inf, math.nan, math.nan
        got = step(bad, bad_dh)
        rest = [i for i in range(300) if i not in (3, 299, 17)]
        assert all(torch.equal(a[rest], b[rest]) for a, b in zip(got, want))
        assert not torch.isfinite(got[0][3]).all() and torch.isnan(got[0][299]).all() and torch.isnan(got[1][17]).all()
        assert torch.equal(got[0][17], want[0][17])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K, F, act, bias", [(4200, 72, 264, "silu", True), (5000, 100, 300, "gelu", True), (1030, 1003, 517, "sigmoid", False), (1100, 1000, 770, "silu", True),
                                                (2050, 504, 1001, "gelu", True), (4097, 136, 1000, "sigmoid", True), (1500, 333, 1030, "silu", False), (300, 2056, 1224, "silu", True)])
def test_gated_mlp_in_tiles_with_edges(ops, dtype, M, K, F, act, bias):
    """Products that are too large for 64 rows to a workgroup, small enough for 128 x 128 tiles: ends inside a tile in every axis, operands as they lie and
    laid out."""
    mlp_check(ops, *mlp_inputs(M, K, F, dtype, M + K + F, bias), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K, F, act, bias", [(65, 1024, 1024, "silu", True), (200, 300, 333, "gelu", True), (1000, 136, 72, "sigmoid", True), (513, 72, 520, "silu", False),
                                                (129, 2048, 31, "gelu", True), (4000, 66, 9, "silu", True), (20, 1030, 47, "silu", True),
                                                (33, 1500, 100, "gelu", True), (128, 1111, 72, "sigmoid", False), (64, 1280, 33, "silu", True)])
def test_gated_mlp_of_small_products(ops, dtype, M, K, F, act, bias):
    """Workgroups of 64 rows beyond the first 64, the last ones part empty; long rows, whose steps fp32 requests one ahead."""
    mlp_check(ops, *mlp_inputs(M, K, F, dtype, M + K + F, bias), act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["columns", "odd columns", "transposed", "one bias"])
def test_gated_mlp_in_tiles_takes_strided_inputs(ops, dtype, kind):
    x, wg, wu, bg, bu = mlp_inputs(4200, 96, 264, dtype, 3, True)
    base = torch.randn(4200, 160, generator=gen(4), device="cuda").to(dtype)
    if kind == "columns":
        x = base[:, 32:128]
    elif kind == "odd columns":
        x = base[:, 3:99]
    elif kind == "transposed":
        x = torch.randn(96, 4200, generator=gen(5), device="cuda").to(dtype).t()
    else:
        bg = None
    mlp_check(ops, x, wg, wu, bg, bu, "silu")


def test_gated_mlp_in_tiles_keeps_bad_rows_to_themselves_and_spans_fp32s_magnitudes(ops):
    x, wg, wu, bg, bu = mlp_inputs(4200, 128, 264, torch.float32, 6, True)
    want = ops.gated_mlp(x, wg, wu, bg, bu)
    bad = x.clone()
    bad[3, 7], bad[4199, 127] = math.inf, math.nan
    got = ops.gated_mlp(bad, wg, wu, bg, bu)
    assert torch.equal(got[4:4199], want[4:4199]) and torch.equal(got[:3], want[:3])
    assert not torch.isfinite(got[3]).all() and torch.isnan(got[4199]).all()
    # the three parts carry 24 bits at any exponent: h is s U, whose relative error c(128) times the terms' sum does not depend on the scale
    x = x * torch.logspace(-20, 15, 4200, device="cuda")[:, None]
    u = ops.gated_mlp(x, torch.zeros_like(wg), wu, act="sigmoid")
    X, W = x.double(), wu.double()
    within(u, 0.5 * (X @ W.t()), 0.5 * 1.01 * ((6 * 128 + 64) * F32 + 3 * 2.0 ** -23) * (X.abs() @ W.abs().t()) + 4 * F32 * (X @ W.t()).abs())


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_mlp_in_large_tiles(ops, dtype):
    """Enough rows and columns for the 256 x 256 tiles in all three products, with edges in both axes."""
    mlp_check(ops, *mlp_inputs(4229, 4130, 2060, dtype, 1, True), "silu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("kind", ["columns", "odd columns", "every second row", "three axes", "transposed", "weights transposed", "one bias"])
def test_gated_mlp_takes_strided_inputs(ops, dtype, rows, kind):
    x, wg, wu, bg, bu = mlp_inputs(rows, 96, 72, dtype, 3, True)
    g = gen(4)
    base = torch.randn(2 * rows, 160, generator=g, device="cuda").to(dtype)
    if kind == "columns":
        x = base[:rows, 32:128]
    elif kind == "odd columns":
        x = base[:rows, 3:99]
    elif kind == "every second row":
        x = base[::2, :96]
    elif kind == "three axes":
        x = base[:rows].reshape(rows, 1, 160)[:, :, :96].expand(rows, 2, 96)
    elif kind == "transposed":
        x = torch.randn(96, rows, generator=g, device="cuda").to(dtype).t()
    elif kind == "weights transposed":
        wg = torch.randn(96, 72, generator=g, device="cuda").to(dtype).t()
    else:
        bg = None
    mlp_check(ops, x, wg, wu, bg, bu, "silu")


def test_gated_mlp_keeps_bad_rows_to_themselves_and_takes_none(ops):
    for rows in (40, 300):
        x, wg, wu, bg, bu = mlp_inputs(rows, 128, 96, torch.float32, 6, True)
        want = ops.gated_mlp(x, wg, wu, bg, bu)
        bad = x.clone()
        bad[3, 7], bad[20, 127] = math.inf, math.nan
        got = ops.gated_mlp(bad, wg, wu, bg, bu)
        rest = [i for i in range(rows) if i not in (3, 20)]
        assert torch.equal(got[rest], want[rest])
        assert not torch.isfinite(got[3]).all() and torch.isnan(got[20]).all()
    x = torch.empty(2, 0, 128, device="cuda", requires_grad=True)
    w = wg.detach().requires_grad_()
    h = ops.gated_mlp(x, w, wu)
    dx, dw = torch.autograd.grad(h, (x, w), torch.empty_like(h))
    assert h.shape == (2, 0, 96) and dx.shape == x.shape and torch.equal(dw, torch.zeros_like(dw))


def test_gated_mlp_of_fp32_spans_its_magnitudes(ops):
    """The three parts carry 24 bits at any exponent: rows of 1e-20 and of 1e+15 beside one another."""
    x, wg, wu, _, _ = mlp_inputs(200, 64, 64, torch.float32, 9, False)
    scale = torch.logspace(-20, 15, 200, device="cuda")[:, None]
    h = ops.gated_mlp(x * scale, wg, wu, act="sigmoid")
    X = (x * scale).double()
    G, U = X @ wg.double().t(), X @ wu.double().t()
    s = torch.sigmoid(G)
    size = X.abs() @ wu.double().abs().t()
    eG = (7 * 64 + 64) * F32 * (X.abs() @ wg.double().abs().t())
    # the sigmoid moves by its own derivative over G's error, and by its relative error where it is small (underflows: below 1e-38)
    lo, hi = torch.sigmoid(G - eG), torch.sigmoid(G + eG)
    within(h, s * U, 1.01 * ((hi - lo) * U.abs() + (16 + 2 * G.abs().clamp_max(100)) * F32 * (s * U).abs() + (7 * 64 + 64) * F32 * size * hi) + 1e-37 * U.abs() + 1e-38)


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K", [(16, 128), (100, 128), (16, 8), (100, 8)])
def test_gated_mlp_gates_far_from_zero(ops, dtype, act, M, K):
    """Gates of up to 1e30 (fp16: 6e4) through each kind of kernel: G is column 0 of x, U column 1.  The activations and their derivatives are 0, 1 or g
    there: to the type's rounding, and to 1e-30 where they underflow."""
    values = [0.0, 20.0, 60.0, 90.0, 200.0, 6e4] + ([] if dtype == torch.float16 else [1e10, 1e30])
    g = torch.tensor([s * v for v in values for s in (1, -1)], device="cuda")
    x = torch.zeros(M, K, device="cuda", dtype=dtype)
    x[:, 0] = g[torch.arange(M, device="cuda") % len(g)].to(dtype)
    x[:, 1] = 1
    wg, wu = torch.zeros(16, K, device="cuda", dtype=dtype), torch.zeros(16, K, device="cuda", dtype=dtype)
    wg[:, 0], wu[:, 1] = 1, 1
    x.requires_grad_()
    h = ops.gated_mlp(x, wg, wu, act=act)
    dx, = torch.autograd.grad(h, x, torch.full_like(h, 1 / 16))
    v, d = gate_reference(x[:, 0].detach().double(), act)
    within(h, v[:, None].expand(M, 16), half_step(dtype, v[:, None]) + 200 * F32 * v[:, None].abs() + 1e-30)
    # one rounding of dG and dU to operands, sums of 16 alike (exact), one of dx; dG is d / 16, dU v / 16
    tol = lambda t: 2.01 * half_step(dtype, t) + 16 * 2.01 * half_step(dtype, t / 16) + 200 * F32 * t.abs() + 1e-30  # noqa: E731
    within(dx[:, 0], d, tol(d))
    within(dx[:, 1], v, tol(v))


def test_gated_mlp_gradient_against_differences(ops):
    g = gen(13)
    params = [t.requires_grad_() for t in mlp_inputs(100, 48, 40, torch.float32, 12, True)]
    dh = torch.randn(100, 40, generator=g, device="cuda")
    grads = torch.autograd.grad(ops.gated_mlp(*params, act="gelu"), params, dh)
    with torch.no_grad():
        for i, t in enumerate(params):
            way = torch.randn(t.shape, generator=g, device="cuda") * (48 ** -0.5 if t.dim() == 2 and i else 1)
            h = 2.0 ** -6
            f = [float((ops.gated_mlp(*[v + s * h * way if j == i else v for j, v in enumerate(params)], act="gelu").double() * dh.double()).sum()) for s in (1, -1)]
            got, want = (f[0] - f[1]) / (2 * h), float((grads[i].double() * way.double()).sum())
            # third differences of act(g) u along a way of order 1 in g and u are of order 10; values of order 10 rounded at c(48)
            size = float(dh.abs().sum()) * 10
            assert abs(got - want) <= size * (h * h / 6 + (6 * 48 + 64) * F32 / h), (i, got, want)


def test_gated_mlp_gives_the_same_bits_every_time_on_any_stream_and_in_a_graph(ops):
    side = torch.cuda.Stream()
    for shape, dtype in (((500, 200, 136), torch.bfloat16), ((3000, 64, 96), torch.float32), ((9, 64, 96), torch.float16)):
        leaves = [t.requires_grad_() for t in mlp_inputs(*shape, dtype, 2, True)]
        dh = torch.ones(shape[0], shape[2], device="cuda", dtype=dtype)

        def step():
            h = ops.gated_mlp(*leaves)
            return (h.detach(),) + torch.autograd.grad(h, leaves, dh)
        want = [t.clone() for t in step()]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(other, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for k in range(3):
            for t in held:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(held, want)), k
            assert all(torch.equal(a, b) for a, b in zip(step(), want)), k
            torch.cuda.synchronize()


def test_gated_mlp_gradients_of_some_tensors_only(ops):
    for which in ("x", "wg", "wu", "bg", "bu"):
        tensors = dict(zip(("x", "wg", "wu", "bg", "bu"), mlp_inputs(130, 64, 72, torch.bfloat16, 8, True)))
        full = mlp_check(ops, *tensors.values(), "silu")[1]
        tensors[which].requires_grad_()
        h = ops.gated_mlp(*tensors.values())
        dh = torch.randn(130, 72, generator=gen(5), device="cuda").to(torch.bfloat16)
        assert torch.equal(torch.autograd.grad(h, tensors[which], dh)[0], full[which]), which


@pytest.mark.parametrize("D", [3, 64, 200])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gru_scan_bad_values_stay_in_their_packed_sequence(ops, dtype, D):
    bounds = [0, 400, 400, 410, 1500, 1501, 3000]
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    z, q, h0 = scan_inputs((3000, D), 6, dtype, 21)
    dh, dl = torch.randn(3000, D, generator=gen(2), device="cuda").to(dtype), torch.randn(6, D, generator=gen(3), device="cuda")

    def step(q, h0, dh, dl):
        leaves = [t.detach().requires_grad_() for t in (z, q, h0)]
        h, last = ops.gru_scan(*leaves, cu_seqlens=cu)
        return (h.detach(), last.detach()) + torch.autograd.grad((h, last), leaves, (dh, dl))
    want = step(q, h0, dh, dl)
    bad_q, bad_h0, bad_dh, bad_dl = q.clone(), h0.clone(), dh.clone(), dl.clone()
    bad_q[100], bad_q[2000] = math.inf, math.nan          # sequences 0 and 5
    bad_h0[3] = -math.inf
    bad_dh[1500], bad_dl[0] = math.inf, math.nan          # the single row between 3 and 5
    got = step(bad_q, bad_h0, bad_dh, bad_dl)
    for a, b in zip(got, want):
        if a.shape[0] == 3000:
            assert torch.equal(a[400:410], b[400:410])
        else:
            assert torch.equal(a[1:3], b[1:3])
    assert torch.equal(got[0][:100], want[0][:100]) and torch.equal(got[0][1500:2000], want[0][1500:2000])      # forward: what lies before them
    assert torch.equal(got[3][1501:], want[3][1501:])     # dq of the sequence behind the bad gradient: it reads neither q nor h


def test_gradients_of_gradients_are_refused(ops):
    x = torch.randn(5, 40, device="cuda", requires_grad=True)
    z = torch.rand(1, 5, 40, device="cuda", requires_grad=True)
    w = torch.randn(16, 40, device="cuda", requires_grad=True)
    for y, leaf in ((ops.layer_norm(x), x), (ops.gru_scan(z, z.detach())[0], z), (ops.gated_mlp(x, w, w), x)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), leaf, create_graph=True)


# ------------------------------------------------------------------------------------------------------------------ together
def block(ops, norm, mlp, out, x, h0, cu=None):
    """A recurrent block over the frames of a clip, its gates from the normalised frame: norm -> gated projections -> scan -> add, norm."""
    d = x.shape[-1]
    f = mlp(norm(x))
    h, last = ops.gru_scan(torch.sigmoid(f[..., :d]), torch.tanh(f[..., d:]), h0, cu_seqlens=cu)
    return out(x + h), last


def block_reference(norm, mlp, out, x, h0):
    d = x.shape[-1]

    def ln(m, v):
        return torch.nn.functional.layer_norm(v, (d,), m.weight.double(), m.bias.double(), m.eps)
    n = ln(norm, x.double())
    g, u = n @ mlp.gate.weight.double().t() + mlp.gate.bias.double(), n @ mlp.up.weight.double().t() + mlp.up.bias.double()
    f = torch.nn.functional.silu(g) * u
    z, q, s, h = torch.sigmoid(f[..., :d]), torch.tanh(f[..., d:]), h0.double(), []
    for t in range(x.shape[1]):
        s = (1 - z[:, t]) * s + z[:, t] * q[:, t]
        h.append(s)
    return ln(out, x.double() + torch.stack(h, 1)), s


def block_of(d, seed):
    from motif_amd.models.modules.layers import GatedMLP, LayerNorm
    torch.manual_seed(seed)
    parts = [LayerNorm(d), GatedMLP(d, 2 * d), LayerNorm(d)]
    with torch.no_grad():
        for p in (p for m in parts for p in m.parameters()):
            p.add_(0.1 * torch.randn_like(p))
    return [m.cuda() for m in parts]


def test_the_operators_together_as_a_recurrent_block_in_training(ops):
    parts = block_of(64, 1)
    x = torch.randn(3, 90, 64, generator=gen(1), device="cuda", requires_grad=True)
    h0 = torch.randn(3, 64, generator=gen(2), device="cuda", requires_grad=True)
    dy, dl = torch.randn(3, 90, 64, generator=gen(3), device="cuda"), torch.randn(3, 64, generator=gen(4), device="cuda")
    leaves = [x, h0] + [p for m in parts for p in m.parameters()]
    y, last = block(ops, *parts, x, h0)
    got = torch.autograd.grad((y, last), leaves, (dy, dl))
    yr, lr = block_reference(*parts, x, h0)
    want = torch.autograd.grad((yr, lr), leaves, (dy.double(), dl.double()))
    # five stages, each within a few hundred roundings of 2^-24 of values of order 1 (sums: of their terms' root sum of squares, at most 10 x the
    # result's scale here): 2^-24 x 500 x 10
    for a, b in zip((y, last) + got, (yr, lr) + want):
        within(a, b, 5000 * F32 * (1 + b.abs().max()))


def test_the_operators_together_stream_a_clip_and_replay_in_a_graph(ops):
    """Serving: a clip at once, frame by frame with the state carried along, and frame by frame as the replay of one captured frame."""
    for dtype, tol in ((torch.float32, 4000 * F32), (torch.bfloat16, 2.0 ** -4)):      # bf16: six roundings of 2^-8 on values up to 4
        parts = [m.to(dtype) for m in block_of(96, 2)]
        x = torch.randn(2, 12, 96, generator=gen(5), device="cuda").to(dtype)
        h0 = torch.zeros(2, 96, device="cuda")
        with torch.no_grad():
            whole, last = block(ops, *parts, x, h0)
            state, rows = h0, []
            for t in range(12):
                y, state = block(ops, *parts, x[:, t:t + 1], state)
                rows.append(y)
            within(torch.cat(rows, 1), whole, tol)
            within(state, last, tol)
            frame, held = x[:, :1].clone(), h0.clone()
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(graph, stream=side):
                out, new = block(ops, *parts, frame, held)
                held.copy_(new)
            for t in range(12):
                frame.copy_(x[:, t:t + 1])
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, rows[t]), (dtype, t)
                block(ops, *parts, x, h0)                 # eager work between the replays
            assert torch.equal(held, state)


def test_the_operators_together_on_packed_clips(ops):
    parts = block_of(64, 3)
    bounds = [0, 7, 7, 30, 31]
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    x = torch.randn(31, 64, generator=gen(6), device="cuda")
    h0 = torch.randn(4, 64, generator=gen(7), device="cuda")
    with torch.no_grad():
        y, last = block(ops, *parts, x, h0, cu)
        for i, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
            if hi > lo:
                yi, li = block(ops, *parts, x[None, lo:hi], h0[i:i + 1])
                within(y[None, lo:hi], yi, 2000 * F32)
                within(last[i:i + 1], li, 2000 * F32)
            else:
                assert torch.equal(last[i], h0[i])


def test_two_streams_and_two_captured_graphs_share_nothing(ops):
    """Workspaces belong to their call: two streams at once, and two graphs replayed in turn, give the bits of the calls alone."""
    leaves = [[t.requires_grad_() for t in mlp_inputs(700, 200, 72, torch.float32, s, True)] for s in (1, 2)]
    scans = [[t.requires_grad_() for t in scan_inputs((3000, 40), 3, torch.bfloat16, s)] for s in (1, 2)]
    cu = torch.tensor([0, 1000, 1001, 2900], dtype=torch.int32, device="cuda")

    def step(i):
        h = ops.gated_mlp(*leaves[i])
        s, last = ops.gru_scan(*scans[i], cu_seqlens=cu)
        n = ops.layer_norm(leaves[i][0])
        return [t.detach() for t in (h, s, last, n)] + list(torch.autograd.grad(h, leaves[i], torch.ones_like(h))) + \
            list(torch.autograd.grad((s, last), scans[i], (torch.ones_like(s), torch.ones_like(last)))) + list(torch.autograd.grad(n, leaves[i][0], h.detach()[:, :1].expand_as(n)))
    want = [[t.clone() for t in step(i)] for i in (0, 1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for k in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i])), i
    del got
    graphs, held = [], []
    for i, s in enumerate(streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            held.append(step(i))
        graphs.append(g)
    for k in range(3):
        for t in held[0] + held[1]:
            t.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(held[i], want[i])), (k, i)
        step(0)


def test_gru_scan_bounds_behind_the_rows_end_with_them(ops):
    z, q, h0 = scan_inputs((50, 24), 3, torch.float32, 31)
    got = ops.gru_scan(z, q, h0, cu_seqlens=torch.tensor([0, 20, 70, 90], dtype=torch.int32, device="cuda"))
    want = ops.gru_scan(z, q, h0, cu_seqlens=torch.tensor([0, 20, 50, 50], dtype=torch.int32, device="cuda"))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ------------------------------------------------------------------------------------------------------------------ unusual calls
def test_one_tensor_in_several_places_and_broadcast_parameters(ops):
    """x as both weights, the gate as its own candidate, a weight of one value for all columns, a row for all rows: gradients add up over the places."""
    a = torch.randn(70, 64, generator=gen(41), device="cuda").mul_(0.125).requires_grad_()
    g, = torch.autograd.grad(ops.gated_mlp(a, a, a).sum(), a)
    b = a.detach().double().requires_grad_()
    p = b @ b.t()
    want, = torch.autograd.grad((torch.nn.functional.silu(p) * p).sum(), b)
    # products of 64 terms below 2 in sum, three roundings on the way, sums of 2 x 70: within 2000 x 2^-24 of the largest gradient
    within(g, want, 2000 * F32 * want.abs().max())
    z = torch.rand(2, 50, 8, generator=gen(42), device="cuda").requires_grad_()
    h, last = ops.gru_scan(z, z)
    g, = torch.autograd.grad(h.sum() + last.sum(), z)
    d = z.detach().double().requires_grad_()
    s, total = torch.zeros(2, 8, device="cuda", dtype=torch.float64), 0
    for t in range(50):
        s = (1 - d[:, t]) * s + d[:, t] * d[:, t]
        total = total + s.sum()
    want, = torch.autograd.grad(total + s.sum(), d)
    within(g, want, 1000 * F32 * (1 + want.abs().max()))
    x, w = torch.randn(1, 64, generator=gen(43), device="cuda").requires_grad_(), torch.ones(1, device="cuda", requires_grad=True)
    got = torch.autograd.grad(ops.layer_norm(x.expand(5, 64), w.expand(64)).square().sum(), (x, w))
    x2, w2 = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    n = (x2 - x2.mean()) / (x2.var(unbiased=False) + 1e-5).sqrt()
    want = torch.autograd.grad((n.expand(5, 64) * w2).square().sum(), (x2, w2))
    # dx is a difference of terms of order 2 n / sigma (5 rows): absolute, to 100 roundings of their size
    within(got[0], want[0], 100 * F32 * 5 * 2 * float(n.detach().abs().max()) ** 2 * torch.ones_like(want[0]))
    within(got[1], want[1], 100 * F32 * want[1].abs())


def test_offsets_beyond_32_bits(ops):
    rows, d = 3 << 20, 1024                              # 3.2e9 values
    x = torch.zeros(rows, d, device="cuda", dtype=torch.bfloat16)
    x[-1] = torch.arange(d, device="cuda").bfloat16()
    with torch.no_grad():
        y = ops.layer_norm(x)
        assert torch.equal(y[-1], ops.layer_norm(x[-1:].clone())[0]) and not y[:-1].any()
        del y
        z = torch.full_like(x, 0.5)
        h, last = ops.gru_scan(z, x.fill_(1), cu_seqlens=torch.tensor([0, rows - 5, rows], dtype=torch.int32, device="cuda"))
        assert (h[rows - 6] == 1).all() and (h[rows - 5] == 0.5).all() and (last[1] == 1 - 2.0 ** -5).all()
        del h, z, x
        x = torch.randn(4 << 20, 64, generator=gen(44), device="cuda").bfloat16()
        wg, wu = (torch.randn(1024, 64, generator=gen(45 + i), device="cuda").mul_(0.125).bfloat16() for i in (0, 1))
        y = ops.gated_mlp(x, wg, wu)                     # narrow: 4.3e9 outputs
        assert torch.equal(y[-100:], ops.gated_mlp(x[-100:].clone(), wg, wu))
        del y, x
        x = torch.randn(2 << 20, 1032, generator=gen(47), device="cuda", dtype=torch.bfloat16)[:, :1024]
        wg, wu = (torch.randn(1040, 1024, generator=gen(48 + i), device="cuda").mul_(2.0 ** -5).bfloat16() for i in (0, 1))
        y = ops.gated_mlp(x, wg, wu)                     # tiles: 2.2e9 inputs and outputs
        p, q = (x[-100:].double() @ w.double().t() for w in (wg, wu))
        size = x[-100:].double().abs() @ wg.double().abs().t(), x[-100:].double().abs() @ wu.double().abs().t()
        v = torch.nn.functional.silu(p)
        c = (1024 + 64) * F32
        within(y[-100:], v * q, half_step(torch.bfloat16, v * q) + 1.01 * (1.13 * c * size[0] * q.abs() + c * size[1] * v.abs()) + (20 + 2 * p.abs()) * F32 * (v * q).abs())


# ------------------------------------------------------------------------------------------------------------------ infinities and ranges
def same_kind(got, want):
    """Infinite, with its sign, or NaN where the 64-bit result is; finite where it is."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    for kind in (torch.isnan, lambda t: t == math.inf, lambda t: t == -math.inf):
        bad = kind(got) != kind(want)
        assert not bad.any(), (int(bad.sum()), bad.numel(), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("M, K, F", [(40, 200, 600), (500, 64, 96), (2050, 200, 600)], ids=["few rows", "narrow", "tiles"])
def test_gated_mlp_of_fp32_infinities_come_out_as_they_would_in_fp32(ops, M, K, F):
    """Whatever the number of rows: an infinite value among finite ones, beside weights of many bits and of few (their lower parts are 0) and of none."""
    x, wg, wu, bg, bu = mlp_inputs(M, K, F, torch.float32, 31, True)
    for w in (wg, wu):
        w[::3] = w[::3].bfloat16().float()
        w[1::9] = torch.exp2(torch.floor(torch.log2(w[1::9].abs()))) * w[1::9].sign()
    wu[2, 7] = wg[4, 7] = 0.0
    x[3, 7], x[M - 1, K - 1], x[17, 0], x[17, 1] = math.inf, -math.inf, math.inf, -math.inf
    dh = torch.randn(M, F, generator=gen(32), device="cuda")
    dh[5, 11], dh[M - 2, F - 1] = math.inf, -math.inf
    for act in ("silu", "gelu", "sigmoid"):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        h = ops.gated_mlp(*leaves, bg, bu, act=act)
        X, WG, WU, DH = (t.double().cpu() for t in (x, wg, wu, dh))
        G, U = X @ WG.t() + bg.double().cpu(), X @ WU.t() + bu.double().cpu()
        v, dv = gate_reference(G, act)
        same_kind(h, v * U)
        assert torch.isfinite(h[:3]).all() and torch.isinf(h[3]).any()
        # backward from what the activations give for finite gates; infinite ones have derivatives of inf - inf and 0 x inf
        finite = torch.isfinite(G).all(1) & torch.isfinite(U).all(1)
        rows = finite.nonzero()[:, 0]
        dx, = torch.autograd.grad(h, leaves[:1], dh)
        dG, dU = (DH * U * dv)[rows], (DH * v)[rows]
        same_kind(dx[rows.cuda()], dG @ WG + dU @ WU)
        assert not torch.isfinite(dx[5]).all()


def mlp_ranges_check(ops, x, wg, wu, dh, act):
    """mlp_check's bounds of dx, dWg and dWu for fp16 gradients of any size.  dG and dU are rounded once: by 2^-11 of their value, and of no less than
    2^-14 where their largest value P lies in 2^-4 .. 65504, of no less than 2^-28 P elsewhere (a power of two takes P to 2^14 and more)."""
    M, K, F = x.shape[0], x.shape[1], wg.shape[0]
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = ops.gated_mlp(*leaves, act=act)
    got = torch.autograd.grad(h, leaves, dh)
    X, WG, WU, DH = (t.double() for t in (x, wg, wu, dh))
    G, U = X @ WG.t(), X @ WU.t()
    c = lambda n: (n + 64) * F32  # noqa: E731
    eG, eU = c(K) * (X.abs() @ WG.abs().t()), c(K) * (X.abs() @ WU.abs().t())
    v, dv = gate_reference(G, act)
    rel = (16 + 2 * G.abs()) * F32
    ev = 1.13 * eG + rel * v.abs() + (16 * F32 * G.abs() if act == "gelu" else 0)
    edv = eG + rel * (dv.abs() + 1)
    dG, dU = DH * U * dv, DH * v
    edG = DH.abs() * (eU * dv.abs() + edv * U.abs() + eU * edv) + 4 * F32 * dG.abs()
    edU = DH.abs() * ev + 4 * F32 * dU.abs()
    peak = max(float(dG.abs().max()), float(dU.abs().max()))
    least = 2.0 ** -14 if 2.0 ** -4 <= peak <= 65504 else 2.0 ** -28 * peak
    step = lambda t: 2.0 ** -11 * t.clamp_min(least)  # noqa: E731
    rG, rU = edG + 1.01 * step(dG.abs() + edG), edU + 1.01 * step(dU.abs() + edU)
    want = [dG @ WG + dU @ WU, dG.t() @ X, dU.t() @ X]
    tol = [rG @ WG.abs() + rU @ WU.abs() + c(2 * F) * (dG.abs() @ WG.abs() + dU.abs() @ WU.abs())]
    tol += [r.t() @ X.abs() + c(M) * (d.abs().t() @ X.abs()) for d, r in ((dG, rG), (dU, rU))]
    sizes = []
    for a, w, t in zip(got, want, tol):
        t = half_step(torch.float16, w) + 1.01 * t
        inside, outside = w.abs() + t < 65504, w.abs() - t > 65520
        within(torch.where(inside, a.double(), 0), torch.where(inside, w, 0), t)
        assert torch.equal(a[outside].double(), torch.sign(w[outside]) * math.inf), "gradients that do not fit are infinite"
        sizes.append(float(inside.double().mean()))
    return peak, sizes


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("M, K, F", [(40, 200, 600), (2050, 200, 600), (1500, 333, 1030), (700, 64, 96), (1000, 20, 256)])
def test_gated_mlp_of_fp16_gradients_of_any_size(ops, M, K, F, act):
    """The products dh U and dh act(G) pass fp16's range, or lie below its normal numbers, where the gradients made of them do not: in tiles, in the
    narrow layers' one pass."""
    g = gen(M + K + F)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).half()  # noqa: E731
    # (x, weights, dh): G and U of about 1 to 30; peaks beyond 65504 with finite dx, with finite dW; far below 2^-4
    for x, w, dh, finite in ((2.0 ** 11, 2.0 ** -6, 8192.0, 0), (2.0 ** -9, 2.0 ** 14, 8192.0, 1), (1.0, 1.0, 2.0 ** -17, 0), (1.0, 1.0, 2.0 ** -11, 1)):
        peak, sizes = mlp_ranges_check(ops, n(M, K, scale=x), n(F, K, scale=w * K ** -0.5), n(F, K, scale=w * K ** -0.5), n(M, F, scale=dh), act)
        assert (peak > 65504) == (dh > 1) and sizes[finite] > 0.99, (peak, sizes)
    # one gradient far above the others: they keep what fp16 numbers beside it keep
    dh = n(M, F, scale=2.0 ** -6)
    dh[3, 5] = 60000.0
    mlp_ranges_check(ops, n(M, K, scale=4.0), n(F, K, scale=4 * K ** -0.5), n(F, K, scale=K ** -0.5), dh, act)


def test_gated_mlp_of_fp16_bad_gradients_stay_in_their_rows(ops):
    """An infinite or NaN gradient is no measure of the others, and biases are summed from what was not rounded."""
    for M, K, F in ((300, 136, 200), (300, 36, 72)):
        x, wg, wu, bg, bu = mlp_inputs(M, K, F, torch.float16, 6, True)
        dh = torch.randn(M, F, generator=gen(7), device="cuda").half()

        def step(dh):
            leaves = [t.detach().requires_grad_() for t in (x, bg, bu)]
            return torch.autograd.grad(ops.gated_mlp(leaves[0], wg, wu, *leaves[1:]), leaves, dh)
        want = step(dh)
        bad = dh.clone()
        bad[3, 7], bad[299, 35] = math.inf, math.nan
        got = step(bad)
        rest = [i for i in range(300) if i not in (3, 299)]
        assert torch.equal(got[0][rest], want[0][rest]) and not torch.isfinite(got[0][3]).all() and torch.isnan(got[0][299]).all()
        keep = [f for f in range(F) if f not in (7, 35)]
        assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got[1:], want[1:]))


def test_gated_mlp_of_fp16_gradients_of_any_size_in_a_graph(ops):
    """The same captured step serves gradients of every size: what they need is found on the device."""
    for M, K, F in ((300, 136, 200), (300, 36, 72)):
        leaves = [t.requires_grad_() for t in mlp_inputs(M, K, F, torch.float16, 8, True)]
        dh = torch.randn(M, F, generator=gen(9), device="cuda").half()

        def step():
            h = ops.gated_mlp(*leaves)
            return (h.detach(),) + torch.autograd.grad(h, leaves, dh)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
        for scale in (1.0, 2.0 ** -18, 20000.0, 1.0, 2.0 ** -10):
            with torch.no_grad():
                dh.copy_(torch.randn(M, F, generator=gen(10), device="cuda") * scale)
            for t in held:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(held, step())), scale
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, T, D", [(512, 300, 16), (511, 300, 16), (512, 130, 64), (4097, 16, 8), (70000, 1, 3), (20000, 20, 3), (20000, 20, 8), (700, 33, 1000), (520, 18, 1020),
                                     (3000, 7, 257), (257, 100, 1024), (1000, 70, 200)])
def test_gru_scan_of_many_batches(ops, dtype, B, T, D):
    """Many sequences of few channels: time slots, or lanes of several batches in one wave; runs that end within a batch's last lanes."""
    z, q, h0 = scan_inputs((B, T, D), B, dtype, B + T + D)
    scan_check(ops, z, q, h0)
    # as a slice of a larger tensor, time first: batch strides that differ from one another's
    big, _, _ = scan_inputs((T, B, D + 5), B, dtype, 3)
    scan_check(ops, big[..., 3:3 + D].transpose(0, 1), q, None)


def test_gru_scan_of_very_many_packed_sequences_and_of_bounds_before_the_first_row(ops):
    """More sequences than a grid holds workgroups, nearly all of them empty; and bounds below 0, which count as 0."""
    S, T, D = 17 << 20, 40, 2
    cu = torch.zeros(S + 1, dtype=torch.int32, device="cuda")
    cu[5:], cu[S // 2:], cu[S:] = 7, 30, 38
    z, q, _ = scan_inputs((T, D), 1, torch.float32, 51)
    h0 = torch.randn(S, D, generator=gen(52), device="cuda")
    with torch.no_grad():
        h, last = ops.gru_scan(z, q, h0, cu_seqlens=cu)
        rows = [4, S // 2 - 1, S - 1]                    # 0 .. 6, 7 .. 29, 30 .. 37
        want, end = ops.gru_scan(z, q, h0[rows].contiguous(), cu_seqlens=torch.tensor([0, 7, 30, 38], dtype=torch.int32, device="cuda"))
        assert torch.equal(h, want) and torch.equal(last[rows], end)
        keep = torch.ones(S, dtype=torch.bool, device="cuda")
        keep[rows] = False
        assert torch.equal(last[keep], h0[keep])
        del keep, last
        h0 = h0[:4].contiguous()
        got = ops.gru_scan(z, q, h0, cu_seqlens=torch.tensor([-9, -3, 12, 12, 40], dtype=torch.int32, device="cuda"))
        want = ops.gru_scan(z, q, h0, cu_seqlens=torch.tensor([0, 0, 12, 12, 40], dtype=torch.int32, device="cuda"))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------------------------ every tile of every type
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M, K, F, act, bias", [(8190, 2040, 5624, "silu", False), (1100, 2040, 4088, "gelu", True), (1100, 2041, 4085, "sigmoid", True)])
def test_gated_mlp_weights_gradients_in_large_tiles(ops, dtype, M, K, F, act, bias):
    """The 256 x 256 tiles of the weights' gradients in every type: ends inside a tile on every axis, operands as they lie and laid out, whole and cut along the
    reduction (8190: 352 tiles, 96 behind the last whole round of the chip)."""
    from motif_amd import _lib
    x, wg, wu, bg, bu = mlp_inputs(M, K, F, dtype, 61, bias)
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    tile = [_lib.load().motif_gated_mlp_tile(x.data_ptr(), K, wg.data_ptr(), wu.data_ptr(), M, K, F, code, product) for product in range(4)]
    assert tile[3] == 256 and (M < 8190 or tile == [256] * 4), tile
    mlp_check(ops, x, wg, wu, bg, bu, act)


def one_hot_rows(rows, cols, place, value):
    t = torch.zeros(rows, cols, device="cuda")
    t[torch.arange(rows, device="cuda"), place] = value
    return t


# A product of two 24-bit values as six of the nine products of their 8-bit parts: with p1 < 2^-7 and p2 < 2^-15 of a value's leading power of two (truncation), the
# three that are left out are below 2 x 2^-22 + 2^-30 of the product of both powers, that is, of the product; the six are exact (16 bits) and added with up to
# two roundings' worth each (2 x 2^-24, whether the matrix cores round or truncate).  Any one of the six left out instead misses by up to 2^-14 or 2^-15.
SIX = 2.0 ** -21 + 2.0 ** -30 + 12 * F32


@pytest.mark.parametrize("M, K, F, tile", [(2050, 200, 600, 128), (1030, 1003, 517, 128), (4229, 4130, 2060, 256), (8190, 600, 5624, 256)])
def test_gated_mlp_of_fp32_in_tiles_holds_all_of_a_products_bits(ops, M, K, F, tile):
    """Sums of one product each (the others are 0), so that what is off is a product's own error: every part of every product has to be there, forward, in dx and in
    the weights' gradients."""
    from motif_amd import _lib
    g = gen(62)
    size = lambda *s: (torch.rand(*s, generator=g, device="cuda") + 1) * torch.exp2(torch.randint(-3, 4, s, generator=g, device="cuda").float())  # noqa: E731
    sign = lambda *s: torch.randint(0, 2, s, generator=g, device="cuda").float() * 2 - 1  # noqa: E731
    place = torch.randint(0, K, (M,), generator=g, device="cuda")
    value = size(M) * sign(M)
    x, w = one_hot_rows(M, K, place, value), size(F, K)
    for product in range(4):
        assert _lib.load().motif_gated_mlp_tile(x.data_ptr(), K, w.data_ptr(), w.data_ptr(), M, K, F, 0, product) in ((tile, 128) if product else (tile,))
    V, W = value.double(), w.double()
    exact = V[:, None] * W.t()[place]
    zero, one = torch.zeros_like(w), torch.ones(F, device="cuda")
    # h = U / 2 (sigmoid(0) is 1 / 2), and h = silu(G) of gates of 64 and more, where it is G (1 - exp(-64)), times u = 1 (8 roundings of the activation)
    within(ops.gated_mlp(x, zero, w, act="sigmoid"), exact / 2, SIX * exact.abs() / 2)
    within(ops.gated_mlp(x.abs() * 4096, w, zero, None, one, act="silu"), 4096 * exact.abs(), (SIX + 8 * F32) * 4096 * exact.abs())
    # backward with one gradient to a row and to a column: dU = dh / 2, dG = dh U / 4 (act sigmoid at 0), every entry of dx = dU Wu, of dWu and dWg one product
    n = min(M, F)
    column = torch.randperm(F, generator=g, device="cuda")[:n]
    dvalue = size(n) * sign(n)
    dh = torch.zeros(M, F, device="cuda")
    dh[torch.arange(n, device="cuda"), column] = dvalue
    dense, wg, wu = size(M, K) * sign(M, K), zero.clone().requires_grad_(), w.clone().requires_grad_()
    xl = dense.clone().requires_grad_()
    bias = torch.full((F,), 1.5, device="cuda")            # (U for dG: x is dense here, and x wu would be a sum)
    D, X = dvalue.double(), dense.double()
    h = ops.gated_mlp(xl, wg, wu, None, None, act="sigmoid")
    dx, dwu = torch.autograd.grad(h, (xl, wu), dh)
    want = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    want[:n] = D[:, None] / 2 * W[column]
    within(dx, want, SIX * want.abs())
    want = torch.zeros(F, K, dtype=torch.float64, device="cuda")
    want[column] = D[:, None] / 2 * X[:n]
    within(dwu, want, SIX * want.abs())
    dwg, = torch.autograd.grad(ops.gated_mlp(dense, wg, zero, None, bias, act="sigmoid"), (wg,), dh)
    want[column] = D[:, None] * 0.375 * X[:n]             # dh x 1.5 x 1 / 4: a rounding or two
    within(dwg, want, (SIX + 4 * F32) * want.abs())


@pytest.mark.parametrize("M, K", [(64, 128), (2100, 200), (3000, 32)], ids=["few rows", "tiles", "narrow"])
def test_gated_mlp_of_fp32_gelu_keeps_its_digits_on_the_negative_side(ops, M, K):
    """gelu(g) and its derivative relative to their own size down to g = -12.  E = exp(-g^2 / 2): the square, its product with log2 e and that constant are rounded, 2.4 x 2^-24 of
    an exponent of g^2 / 2, and E itself to 2 x 2^-24.  The fit is off by 6.2e-8 (1.1 x 2^-24), its eight steps, reciprocal and products by 16 x 2^-24 more."""
    F = 600 if M == 2100 else 64
    g = -torch.rand(M, generator=gen(71), device="cuda") * 12
    x = torch.zeros(M, K, device="cuda")
    x[:, 0] = g
    wg, zero = torch.zeros(F, K, device="cuda"), torch.zeros(F, K, device="cuda")
    wg[:, 0] = 1
    one = torch.ones(F, device="cuda")
    x.requires_grad_()
    h = ops.gated_mlp(x, wg, zero, None, one, act="gelu")
    dh = torch.zeros(M, F, device="cuda")
    dh[:, 5] = 1
    dx, = torch.autograd.grad(h, x, dh)
    G = g.double()
    phi, pdf = torch.special.erfc(-G / math.sqrt(2)) / 2, torch.exp(-0.5 * G * G) / math.sqrt(2 * math.pi)
    rel = (1.2 * G * G + 2 + 18) * F32
    within(h, (G * phi)[:, None].expand(M, F), (rel * (G * phi).abs())[:, None])
    six = (2.0 ** -21 if M == 2100 else 0) + 8 * F32       # dx: one product with 1
    within(dx[:, 0], phi + G * pdf, (rel + six) * (phi + (G * pdf).abs()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [3, 24, 300, 512, 1000, 4097])
def test_layer_norm_bits_do_not_depend_on_strides_and_alignment(ops, dtype, D):
    """Which lane holds which column follows from D alone: the same rows give the same bits, output and all gradients, wherever they lie."""
    rows = 37
    g = gen(D)
    base = torch.randn(2 * rows, D + 64, generator=g, device="cuda").to(dtype)
    w, b = torch.randn(D, generator=g, device="cuda").to(dtype), torch.randn(D, generator=g, device="cuda").to(dtype)
    dbase = torch.randn(2 * rows, D + 64, generator=g, device="cuda").to(dtype)
    flat = torch.randn(rows * D + 1, generator=g, device="cuda").to(dtype)
    layouts = {"columns": lambda t: t[:rows, 32:32 + D], "odd columns": lambda t: t[:rows, 3:3 + D], "every second row": lambda t: t[::2, :D], "last columns": lambda t: t[rows:, 64:],
               "misaligned": lambda t: flat[1:].view(rows, D), "transposed": lambda t: t[:rows, :D].t().contiguous().t(), "one row for all": lambda t: t[:1, 5:5 + D].expand(rows, D)}

    def step(x, dy, w, b):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.layer_norm(*leaves)
        return (y.detach(),) + torch.autograd.grad(y, leaves, dy)
    for name, view in layouts.items():
        x, dy = view(base), view(dbase)
        want = step(x.clone(memory_format=torch.contiguous_format), dy.clone(memory_format=torch.contiguous_format), w, b)
        odd = torch.cat([w[:1], w, b])                   # parameters at odd addresses
        for got in (step(x, dy, w, b), step(x, dy, odd[1:1 + D], odd[1 + D:])):
            for part, p, q in zip(("y", "dx", "dw", "db"), got, want):
                assert torch.equal(p, q), (name, part)
