"""linear_act against the formulas in 64 bits, forward and backward."""

import math

import pytest
import torch

from maskrcnn_amd.ops import linear_act

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu"]
U = 2.0 ** -24


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / \
            math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def inputs(m, k, n, dtype, device, seed=0, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)

    def make(*shape, scale=1.0):
        return torch.randn(*shape, generator=g).mul(scale).to(device, dtype)
    return (make(m, k), make(n, k, scale=1 / math.sqrt(max(k, 1))),
            make(n) if bias else None, make(m, n) if residual else None,
            make(m, n))


def check(x, w, b, r, dy, act):
    """Values and gradients within what fp32 sums and the roundings allow.

    A sum of K products in fp32 in any order, truncated or rounded, is off
    by at most 2 U (K + 8) of the sum of magnitudes. act has a slope below
    1.13 and the slope one below 0.8 (jumps of ReLU's are allowed where z is
    within its error of 0); erf, exp and the products around them take 8 U.
    In 16 bits the derivative is kept in steps of 2^-15.
    """
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    leaves = [t.detach().requires_grad_() if t is not None else None
              for t in (x, w, b, r)]
    y = linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3])
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), leaves)
             if t is not None]
    got = dict(zip(names, torch.autograd.grad(
        y, [t for t in leaves if t is not None], dy)))
    with torch.no_grad():
        assert torch.equal(linear_act(x, w, b, act, r), y)
        assert y.dtype == dtype and y.is_contiguous()
        n, k = w.shape
        m = dy.numel() // n
        X, W, D = (t.double().reshape(s) for t, s in
                   ((x, (m, k)), (w, (n, k)), (dy, (m, n))))
        B = b.double() if b is not None else torch.zeros(n, device=x.device)
        z = X @ W.t() + B
        a, slope = act64(z, act)
        ez = 2 * U * (k + 8) * (X.abs() @ W.t().abs() + B.abs())
        want = a if r is None else a + r.double().reshape(-1, n)
        lim = half * want.abs() + 1.13 * ez + 8 * U * z.abs() + \
            2 * U * (a.abs() + (want - a).abs()) + tiny
        compare("y", y.reshape(-1, n), want, lim)
        if act == "none":
            es = torch.zeros_like(z)
        elif act == "relu":
            es = (z.abs() <= ez).double()
        else:
            es = 0.8 * ez + 8 * U * (1 + z.abs()) + tiny
            if dtype != torch.float32:
                es = es + 2.0 ** -16
        dz = D * slope
        edb = D.abs() * es + U * dz.abs()
        edz = edb + half * dz.abs() + tiny
        compare("db", got.get("db"), dz.sum(0), half * dz.sum(0).abs() +
                edb.sum(0) + U * (m + 200) * dz.abs().sum(0) + tiny)
        dx, dw = dz @ W, dz.t() @ X
        compare("dx", got["dx"].reshape(m, k), dx, half * dx.abs() +
                edz @ W.abs() + 2 * U * (n + 8) * (dz.abs() @ W.abs()) + tiny)
        compare("dw", got["dw"], dw, half * dw.abs() + edz.t() @ X.abs() +
                2 * U * (m + 40) * (dz.abs().t() @ X.abs()) + tiny)
        if r is not None:
            assert torch.equal(got["dr"].reshape(-1, n), dy.reshape(-1, n))


def compare(name, got, want, lim):
    if got is None:
        return
    assert got.shape == want.shape, name
    off = (got.double() - want).abs()
    assert bool((off <= lim).all()), (
        name, float((off / lim.clamp(min=1e-300)).max()),
        (off > lim).nonzero()[:4].tolist())


# m, k, n: single rows and columns, sizes about the tiles' edges, k about a
# step's and a packet's, sizes that split the k axis and that do not.
SHAPES = [(1, 1, 1), (1, 8, 8), (2, 3, 5), (1, 1024, 81), (7, 64, 64),
          (16, 63, 17), (17, 65, 16), (63, 128, 65), (64, 72, 128),
          (65, 120, 129), (100, 1024, 81), (127, 257, 120), (128, 64, 256),
          (130, 1000, 136), (200, 1024, 324), (257, 40, 255), (300, 512, 250),
          (33, 5000, 40), (5, 2, 700), (700, 7, 3)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(device, dtype, shape):
    act = ACTS[sum(shape) % 4]
    check(*inputs(*shape, dtype, device, seed=sum(shape)), act)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, True), (False, False),
                                           (True, False), (False, True)])
def test_epilogue(device, dtype, act, bias, residual):
    for n in (72, 75):
        check(*inputs(50, 96, n, dtype, device, 3, bias, residual), act)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [
    (400, 12544, 1024), (1000, 2048, 1024), (3999, 1024, 1030),
    (8191, 264, 513), (5000, 520, 2048), (2048, 2056, 4096),
    (20000, 136, 300)])
def test_large(dtype, shape):
    check(*inputs(*shape, dtype, "cuda", 1), "gelu")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_strides(device, dtype):
    m, k, n = 37, 80, 56
    x, w, b, r, dy = inputs(m, k, n, dtype, device)
    want = linear_act(x, w, b, "silu", r)
    for at, ld in ((0, 96), (1, 97), (8, 96), (3, 120)):
        held = {}
        for name, t in (("x", x), ("w", w), ("r", r), ("dy", dy)):
            # Behind the rows lies what must never count.
            base = torch.full((t.shape[0], ld), float("nan"), dtype=dtype,
                              device=device)
            held[name] = base[:, at:at + t.shape[1]]
            held[name].copy_(t)
        if device == "cuda":      # the library on the CPU goes by strides
            assert torch.equal(want, linear_act(held["x"], held["w"], b,
                                                "silu", held["r"]))
        check(held["x"], held["w"], b, held["r"], held["dy"], "silu")
    check(x.t().contiguous().t(), w.t().contiguous().t(), b, r, dy, "gelu")
    check(x[:1].expand(m, k), w, b, r, dy[:1].expand(m, n), "relu")
    check(x, w, torch.stack([b, b], 1)[:, 0], r[:1].expand(m, n), dy, "none")
    check(x[::2], w[::2], b[::2], r[::2, ::2], dy[::2, ::2], "relu")


@pytest.mark.parametrize("device", DEVICES)
def test_leading_dimensions(device):
    x, w, b, r, dy = inputs(24, 40, 48, torch.bfloat16, device)
    check(x.view(2, 3, 4, 40), w, b, r.view(2, 3, 4, 48),
          dy.view(2, 3, 4, 48), "gelu")
    check(x.view(4, 6, 40).transpose(0, 1), w, b, r.view(6, 4, 48),
          dy.view(6, 4, 48), "gelu")
    y = linear_act(x[0], w, b)
    assert y.shape == (48,) and torch.equal(y, linear_act(x[:1], w, b)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_sum_or_compute(device):
    x, w, b, r, dy = inputs(4, 16, 8, torch.bfloat16, device)
    check(x[:0], w, b, r[:0], dy[:0], "gelu")
    check(x[:, :0], w[:, :0], b, r, dy, "gelu")
    check(x[:0, :0], w[:, :0], b, r[:0], dy[:0], "relu")
    y = linear_act(x.view(2, 2, 16)[..., :0], w[:, :0], b)
    assert torch.equal(y, b.expand(2, 2, 8))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite_stays_where_it_is(device, dtype):
    x, w, b, _, _ = inputs(70, 72, 80, dtype, device)
    x[3, 71] = float("inf")
    x[69, 0] = float("nan")
    w[79, 5] = float("nan")
    for act in ACTS:
        y = linear_act(x, w, b, act)
        bad = torch.zeros(70, 80, dtype=torch.bool, device=device)
        bad[69], bad[:, 79] = True, True
        assert y[bad].isnan().all()
        bad[3] = True
        assert y[~bad].isfinite().all()
        assert not y[3, :79].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ACTS)
def test_gradient_by_differences(device, act):
    x, w, b, r, dy = inputs(5, 12, 9, torch.float32, device, 2)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    grads = torch.autograd.grad(linear_act(leaves[0], leaves[1], leaves[2],
                                           act, leaves[3]), leaves, dy)

    def loss(args):
        a, c, e, f = args
        z = a @ c.t() + e
        return float(((act64(z, act)[0] + f) * dy.double()).sum())
    h = 1e-5
    for i, g in enumerate(grads):
        for at in range(0, g.numel(), 5):
            side = []
            for s in (h, -h):
                args = [t.double().clone() for t in (x, w, b, r)]
                args[i].view(-1)[at] += s
                side.append(loss(args))
            # h^2 / 6 of third derivatives below 100, 1e-13 / h of
            # cancellation, fp32's 1e-5 of values up to 10 (no z of this
            # seed lies within h of ReLU's corner).
            assert abs((side[0] - side[1]) / (2 * h) -
                       float(g.view(-1)[at])) < 2e-4


@pytest.mark.parametrize("device", DEVICES)
def test_only_what_is_asked_for(device):
    x, w, b, r, dy = inputs(20, 24, 32, torch.bfloat16, device)
    full = [t.detach().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(linear_act(full[0], full[1], full[2], "gelu",
                                          full[3]), full, dy)
    for i in range(4):
        args = [t.detach().requires_grad_(i == j)
                for j, t in enumerate((x, w, b, r))]
        y = linear_act(args[0], args[1], args[2], "gelu", args[3])
        got, = torch.autograd.grad(y, [args[i]], dy)
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, b, r, _ = inputs(4, 16, 8, torch.bfloat16, device)
    for args in ((x, w[:, :8]), (x, w[0]), (x, w.float()),
                 (x, w, b[:4]), (x, w, b.float()), (x, w, b[None]),
                 (x, w[:0]), (x, w, b, "none", r[:2]),
                 (x, w, b, "none", r.float()), (x, w, b, "none", r[:1])):
        with pytest.raises(RuntimeError):
            linear_act(*args)
    with pytest.raises(ValueError):
        linear_act(x, w, b, "tanh")


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, w, b, r, _ = inputs(4, 16, 8, torch.bfloat16, "cuda")
    for args in ((x.double(), w.double()), (x, w.cpu()), (x, w, b.cpu()),
                 (x, w, b, "none", r.cpu())):
        with pytest.raises(RuntimeError):
            linear_act(*args)
    far = torch.empty_strided((2, 16), (1 << 23, 1), dtype=x.dtype,
                              device="cuda")
    with pytest.raises(RuntimeError, match="far apart"):
        linear_act(far, w)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """More than 2^32 bytes and 2^31 values in x and in y; dW over them."""
    m, k, n = 140_000, 16_384, 8
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda")
    w[:, ::64] = torch.arange(1, n + 1, device="cuda")[:, None]
    rows = torch.tensor([0, 255, 65_535, 65_536, 131_071, 131_072, m - 1],
                        device="cuda")
    x[rows, 64] = 1.0
    y = linear_act(x, w)
    want = torch.zeros(m, n, device="cuda")
    want[rows] = torch.arange(1, n + 1, device="cuda").float()
    assert torch.equal(y.float(), want)
    wl = w.detach().requires_grad_()
    dw, = torch.autograd.grad(linear_act(x, wl), wl,
                              torch.ones_like(y))
    assert float(dw[:, 64].float().min()) == len(rows) == \
        float(dw.float().sum(1).max())
    del x, dw
    out = linear_act(torch.ones(m, 8, dtype=w.dtype, device="cuda"),
                     torch.ones(16_384, 8, dtype=w.dtype, device="cuda"))
    assert bool((out[-1] == 8).all()) and bool((out[::997] == 8).all())


@pytest.mark.gpu
def test_same_results_every_time():
    args = inputs(400, 4096, 512, torch.bfloat16, "cuda")
    x, w, b, r, dy = args

    def run():
        leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = linear_act(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
        return (y, *torch.autograd.grad(y, leaves, dy))
    one, two = run(), run()
    assert all(torch.equal(a, c) for a, c in zip(one, two))


@pytest.mark.gpu
def test_other_stream_and_graphs():
    """Two captured graphs with workspaces of their own, replayed in turn."""
    x, w, b, r, dy = inputs(300, 2000, 250, torch.bfloat16, "cuda")
    want = linear_act(x, w, b, "gelu", r)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = linear_act(x, w, b, "gelu", r)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for act in ("gelu", "relu"):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(linear_act(x, w, b, act, r))
    for seed in range(3):
        x.copy_(inputs(300, 2000, 250, torch.bfloat16, "cuda", seed + 9)[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for act, out in zip(("gelu", "relu"), outs):
            assert torch.equal(out, linear_act(x, w, b, act, r))


@pytest.mark.gpu
def test_captured_backward():
    """Forward and backward in one graph, on leaves of its own."""
    args = inputs(300, 500, 250, torch.bfloat16, "cuda")
    dy = args[4]
    leaves = [t.detach().clone().requires_grad_() for t in args[:4]]

    def step(x, w, b, r, dy):
        y = linear_act(x, w, b, "silu", r)
        return (y.detach(), *torch.autograd.grad(y, (x, w, b, r), dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves, dy)
    for seed in range(3):
        new = inputs(300, 500, 250, torch.bfloat16, "cuda", seed + 5)
        with torch.no_grad():
            for leaf, t in zip(leaves, new):
                leaf.copy_(t)
        dy.copy_(new[4])
        graph.replay()
        torch.cuda.synchronize()
        want = step(*[t.requires_grad_() for t in new[:4]], new[4])
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_no_second_gradient(device):
    x, w, b, r, dy = inputs(4, 16, 8, torch.float32, device)
    x.requires_grad_()
    y = linear_act(x, w, b, "gelu", r)
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(y, x, dy, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_negative_views(device):
    """An imaginary part of a conjugate is a view that negates lazily."""
    x, w, b, r, dy = inputs(6, 16, 8, torch.float32, device)
    held = []
    for t in (x, w, b, r, dy):
        c = torch.complex(torch.zeros_like(t), -t).conj()
        assert c.imag.is_neg()
        held.append(c.imag)
    check(*held, "gelu")


@pytest.mark.gpu
def test_far_rows_where_they_do_not_matter():
    """One row has no distance, and a gradient's strides are not the
    caller's."""
    x, w, b, r, dy = inputs(2, 16, 8, torch.bfloat16, "cuda")
    far = torch.empty_strided((2, 16), (1 << 23, 1), dtype=x.dtype,
                              device="cuda")
    far.copy_(x)
    assert torch.equal(linear_act(far[:1], w, b), linear_act(x[:1], w, b))
    assert torch.equal(linear_act(x, far[1:], b[:1]),
                       linear_act(x, x[1:], b[:1]))
    wide = far.as_strided((2, 8), far.stride())
    wide.copy_(dy)
    check(x, w, b, r, wide, "none")
    check(x, w, b, r, wide, "silu")


@pytest.mark.gpu
def test_captured_backward_of_a_held_leaf():
    """An earlier graph of a leaf, on another stream, is refused."""
    x, w, b, r, dy = inputs(40, 64, 32, torch.bfloat16, "cuda")
    for i in range(4):
        leaves = [t.detach().clone().requires_grad_(i == j)
                  for j, t in enumerate((x, w, b, r))]
        leaves.insert(3, "gelu")
        i += i == 3
        held = linear_act(*leaves)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="free that graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y = linear_act(*leaves)
                torch.autograd.grad(y, leaves[i], dy)
        want, = torch.autograd.grad(held, leaves[i], dy)
        del held, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = linear_act(*leaves)
            got, = torch.autograd.grad(y, leaves[i], dy)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_whole_numbers_are_refused(device):
    x = torch.ones(2, 8, dtype=torch.int32, device=device)
    with pytest.raises(RuntimeError):
        linear_act(x, x)


@pytest.mark.parametrize("device", DEVICES)
def test_bias_may_change_before_the_backward(device):
    """It has no part in any gradient, so no version of it is kept."""
    x, w, b, r, dy = inputs(4, 16, 8, torch.float32, device)
    b.requires_grad_()
    y = linear_act(x, w, b)
    with torch.no_grad():
        b.add_(1.0)
    db, = torch.autograd.grad(y, b, dy)
    assert torch.allclose(db, dy.sum(0), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,bits,least", [(torch.bfloat16, 8, -61),
                                              (torch.float16, 9, -38)])
@pytest.mark.parametrize("act,lowest", [("gelu", -8.0), ("silu", -30.0)])
def test_small_derivatives(device, dtype, bits, least, act, lowest):
    """With one weight of 1 the gradient of x is the kept derivative times dy.

    It is off by dz's rounding, by half of what the derivative is kept to
    (steps of 2^-15, or `bits` bits of itself below 2^(bits - 15), or half the
    smallest step), and by 2^-12 of itself for the functions: 16-bit GELU's
    integral is off by 1% of itself at -8, which is 1/64 of its derivative,
    and less above; fp32's exponentials by 1e-5 at most.
    """
    z = torch.linspace(lowest, 8.0, 2049).to(dtype).double()
    dy = 1.0 if dtype == torch.bfloat16 else 1024.0
    x = z.to(device, dtype)[:, None].requires_grad_()
    one = torch.ones(1, 1, dtype=dtype, device=device)
    dx, = torch.autograd.grad(linear_act(x, one, None, act), x,
                              torch.full_like(x, dy))
    _, slope = act64(z, act)
    kept = torch.where(slope.abs() < 2.0 ** (bits - 15),
                       slope.abs() * 2.0 ** -(bits + 1) + 2.0 ** least,
                       2.0 ** -16)
    info = torch.finfo(dtype)
    lim = dy * (kept + slope.abs() * (info.eps / 2 * 1.01 + 2.0 ** -12)) + \
        info.smallest_normal * info.eps / 2
    off = (dx[:, 0].double().cpu() - dy * slope).abs()
    assert (off <= lim).all(), z[off > lim]
    big = slope.abs() * dy > info.smallest_normal
    assert (dx[:, 0].cpu() != 0)[big].all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(device, grad):
    """A result without a tangent would count as a derivative of zero."""
    args = inputs(4, 16, 8, torch.float32, device)[:4]
    with torch.autograd.forward_ad.dual_level():
        for i in range(4):
            given = [t.clone().requires_grad_(grad and i != j)
                     for j, t in enumerate(args)]
            given[i] = torch.autograd.forward_ad.make_dual(
                given[i], torch.ones_like(given[i]))
            x, w, b, r = given
            with pytest.raises(NotImplementedError):
                linear_act(x, w, b, "gelu", r)
    assert linear_act(*args[:3]).isfinite().all()


@pytest.mark.gpu
def test_as_many_rows_as_are_taken():
    """2^30 rows: 64-wide tiles would be 2^32 threads, which no launch has.
    In fp32 the larger tile's would be as many, and the call is refused."""
    m = 1 << 30
    x = torch.ones(m, 1, dtype=torch.bfloat16, device="cuda")
    x[::1000] = 3.0
    w = torch.full((1, 1), 2.0, dtype=torch.bfloat16, device="cuda")
    y = linear_act(x, w)
    for part in (slice(0, 5000), slice(m // 2 - 2500, m // 2 + 2500),
                 slice(m - 5000, m)):
        assert torch.equal(y[part], 2 * x[part])
    assert int((y > 2).sum()) == -(-m // 1000)
    del x, y
    x = torch.ones(m, 1, device="cuda")
    with pytest.raises(RuntimeError, match="too large"):
        linear_act(x, w.float())
    y = linear_act(x[:m - 64], w.float())
    assert bool((y[-1000:] == 2).all()) and float(y.min()) == 2
    del x, y
    torch.cuda.empty_cache()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act,lowest", [("gelu", -8.0), ("silu", -80.0)])
def test_fp32_functions(device, act, lowest):
    """Values and derivatives in fp32 with one weight of 1, relative to
    themselves: 16 units for the exponential (2), erfc (8), quotients, sums
    and products, and z^2 more where the exponents' arguments z^2 / 2 and
    (z / sqrt 2)^2 are rounded, twice each. Near the derivative's zero, within
    the terms that cancel there. (64-bit erfc: ndtr's small values cancel, to
    1e-17 where they are 6e-16.)"""
    z = torch.linspace(lowest, 8.0, 4097).double()
    z = z.float().double()
    x = z.to(device, torch.float32)[:, None].requires_grad_()
    y = linear_act(x, torch.ones(1, 1, device=device), None, act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    s = torch.sigmoid(z)
    if act == "gelu":
        s = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        more = z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    else:
        more = s * z * (1 - s)
    want, slope = z * s, s + more
    rel = (16 + (2 * z * z if act == "gelu" else 0)) * U
    tiny = torch.finfo(torch.float32).smallest_normal
    off = (y[:, 0].detach().double().cpu() - want).abs()
    assert (off <= rel * want.abs() + tiny).all(), z[off > rel * want.abs()]
    terms = torch.where(z > -3, s + more.abs(), slope.abs())
    off = (dx[:, 0].double().cpu() - slope).abs()
    assert (off <= rel * terms + tiny).all(), z[off > rel * terms]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("shape", [
    (1, 2, 1055), (4, 2, 2095), (16, 1, 2), (48, 735, 4), (64, 64, 64),
    (65, 130, 129), (200, 72, 257), (700, 264, 513), (5, 9, 6000),
    (6000, 9, 5)])
def test_gradients_take_dz_whole(device, dtype, act, shape):
    """dz is no 16-bit number on its way into the products: dx and dW are off
    by their own rounding, by what the derivative is kept to (2^-16) and by
    fp32's sums, as in check(); in fp16 by 2^-25 of the second part's own
    smallest step. (Its rounding would add 2^-9 or 2^-12 of each term, many
    times the result's where the terms cancel.)"""
    m, k, n = shape
    x, w, b, _, dy = inputs(m, k, n, dtype, device, seed=sum(shape))
    x, w = (t.requires_grad_() for t in (x, w))
    dx, dw = torch.autograd.grad(linear_act(x, w, b, act), (x, w), dy)
    X, W, B, D = (t.detach().double() for t in (x, w, b, dy))
    z = X @ W.t() + B
    _, slope = act64(z, act)
    dz = D * slope
    info = torch.finfo(dtype)
    half = info.eps / 2 * (1 + 2.0 ** -6)
    tiny = info.smallest_normal * info.eps
    es = 1.6 * U * (k + 8) * (X.abs() @ W.t().abs() + B.abs()) + \
        8 * U * (1 + z.abs()) + 2.0 ** -16
    edz = D.abs() * es + (U + half ** 2) * dz.abs() + tiny / 2
    want = dz @ W
    compare("dx", dx, want, half * want.abs() + edz @ W.abs() +
            2 * U * (2 * n + 8) * (dz.abs() @ W.abs()) + tiny)
    want = dz.t() @ X
    compare("dw", dw, want, half * want.abs() + edz.t() @ X.abs() +
            2 * U * (2 * m + 40) * (dz.abs().t() @ X.abs()) + tiny)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_not_finite_gradients_stay_where_they_are(device, dtype):
    x, w, b, _, dy = inputs(70, 72, 80, dtype, device)
    dy[3, 5] = float("inf")
    dy[9, 7] = float("nan")
    x, w = (t.requires_grad_() for t in (x, w))
    for act in ACTS[2:]:
        dx, dw = torch.autograd.grad(linear_act(x, w, b, act), (x, w), dy)
        assert dx[3].isinf().all() and dx[9].isnan().all()
        assert dw[5].isinf().all() and dw[7].isnan().all()
        dx[3] = dx[9] = dw[5] = dw[7] = 0
        assert dx.isfinite().all() and dw.isfinite().all()


@pytest.mark.gpu
def test_second_part_past_32_bits():
    """dz of more than 2^32 bytes lies in front of its second part. In dx and
    in dW a derivative of 1.118 meets minus the bf16 number nearest to it,
    and what is left is the second part."""
    m, n, near = 140_000, 16_384, 1.1171875
    x = torch.zeros(m, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(n, 8, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    x[:, :2] = 1.0
    x[m - 1, 0] = 8.0                   # derivative 1 in the last row
    w[:, 0] = 1.203125
    w[n - 2, 0] = 8.0                   # and in the last column but one
    w[n - 1, 7] = w[n - 2, 7] = 1.0
    rows = torch.tensor([0, 131_072], device="cuda")
    dy[rows, n - 1] = 1.0
    dy[rows, n - 2] = -near
    dy[m - 1, n - 1] = -2 * near
    _, slope = act64(w[n - 1, 0].double(), "gelu")
    left = float(slope) - near
    assert 2.0 ** -11 < left < 2.0 ** -8
    x, w = (t.requires_grad_() for t in (x, w))
    dx, dw = torch.autograd.grad(linear_act(x, w, None, "gelu"), (x, w), dy)
    # The derivatives of 1 are off by 8 U, the other is kept to 2^-16.
    lim = 2.0 ** -16 + 2.0 ** -20 + 2.0 ** -8 * left
    assert ((dx[rows, 7].double() - left).abs() <= lim).all()
    assert abs(float(dw[n - 1, 1]) - 2 * left) <= 2 * lim
    assert int(dx[:, 7].count_nonzero()) == 3
    assert int(dw[:, 1].count_nonzero()) == 2
    del dy, dx, dw
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_captured_backward_of_a_held_leaf_behind_a_cast():
    """fp32 weights, cast and flattened as the box head does it."""
    x, _, b, r, dy = inputs(40, 64, 32, torch.bfloat16, "cuda")
    w = torch.randn(32, 16, 2, 2, device="cuda", requires_grad=True)

    def layer():
        return linear_act(x, w.reshape(32, -1).to(x.dtype), b, "relu", r)
    held = layer()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="free that graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            y = layer()
            torch.autograd.grad(y, w, dy)
    want, = torch.autograd.grad(held, w, dy)
    del held, y
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer()
        got, = torch.autograd.grad(y, w, dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
