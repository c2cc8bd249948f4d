"""layer_norm against the formulas in 64 bits, forward and backward."""

import pytest
import torch

from maskrcnn_amd.ops import LayerNorm, layer_norm

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24          # half a step of fp32


def exact(x, w, b, dy, eps):
    x, dy = x.double(), dy.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) \
        if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + eps)
    xh = (x - mu) * r
    d = dy * w
    dx = r * (d - d.mean(-1, keepdim=True) -
              xh * (d * xh).mean(-1, keepdim=True))
    return {"y": xh * w + b, "dx": dx, "dw": (dy * xh).flatten(0, -2).sum(0),
            "db": dy.flatten(0, -2).sum(0), "xh": xh, "r": r, "d": d, "w": w,
            "b": b}


def bounds(e, x, dy, dtype, wdtype):
    """What fp32 arithmetic and one rounding at the end may be off by.

    A sum over a row goes through at most 32 values in one lane, 20 strides
    of the widest kernel's 1024 lanes and 6 + 16 exchanges: 60 additions, so
    a mean is off by 60 U of the mean magnitude, xh by r times that and by
    (60 / 2 + 4) U of itself. A weight's sum takes rows / 1024 + 32 + 128 +
    8 additions. Two units of slack cover the products' own roundings.
    """
    half, whalf = torch.finfo(dtype).eps / 2, torch.finfo(wdtype).eps / 2
    rows = x.numel() // x.shape[-1]
    exh = U * (62 * e["r"] * x.double().abs().mean(-1, keepdim=True) +
               36 * e["xh"].abs())
    md = e["d"].abs().mean(-1, keepdim=True)
    mdx = (e["d"] * e["xh"]).abs().mean(-1, keepdim=True)
    s2 = (e["d"] * e["xh"]).mean(-1, keepdim=True).abs()
    edx = e["r"] * (
        U * 64 * (md + e["xh"].abs() * mdx) +
        U * 40 * (e["d"].abs() + md + e["xh"].abs() * mdx) +
        exh * s2 + e["xh"].abs() *
        (e["d"].abs() * exh).mean(-1, keepdim=True))
    # r itself is off by its share of the row's differences.
    edx = edx + e["dx"].abs() * (36 * U + 62 * U * e["r"] *
                                 x.double().abs().mean(-1, keepdim=True))
    adds = rows / 1024 + 170
    ady = dy.double().abs()
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return {
        "y": half * e["y"].abs() + exh * e["w"].abs() + 4 * U *
        ((e["xh"] * e["w"]).abs() + e["b"].abs()) + tiny,
        "dx": half * e["dx"].abs() * 1.01 + edx + tiny,
        "dw": whalf * e["dw"].abs() + (
            ady * exh + U * adds * (ady * e["xh"].abs())
        ).flatten(0, -2).sum(0) + tiny,
        "db": whalf * e["db"].abs() + U * adds * ady.flatten(0, -2).sum(0) +
        tiny}


def close(got, want, bound, name):
    off = (got.double() - want).abs()
    assert got.shape == want.shape, name
    assert bool((off <= bound).all()), (
        name, float((off / bound.clamp(min=1e-300)).max()))


def run(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None
              for t in (x, w, b)]
    y = layer_norm(*leaves, eps=eps)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    return {"y": y.detach(), **dict(zip(
        [n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None],
        grads))}


def check(x, w, b, dy, eps=1e-5):
    e = exact(x, w, b, dy, eps)
    lim = bounds(e, x, dy, x.dtype, w.dtype if w is not None else x.dtype)
    got = run(x, w, b, dy, eps)
    for name, t in got.items():
        close(t, e[name], lim[name], name)
    with torch.no_grad():
        assert torch.equal(layer_norm(x, w, b, eps=eps), got["y"])


def inputs(rows, width, dtype, wdtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, width, generator=g) * 2 + 0.5
    dy = torch.randn(rows, width, generator=g)
    w = 1 + 0.3 * torch.randn(width, generator=g)
    b = 0.3 * torch.randn(width, generator=g)
    return [t.to(device, k) for t, k in
            ((x, dtype), (w, wdtype), (b, wdtype), (dy, dtype))]


# Widths on both sides of each team's limit, odd and even, with 1 value and
# with 16 bytes an access, up to the kernels that keep no row in registers.
WIDTHS = [1, 2, 3, 8, 9, 16, 31, 64, 65, 100, 127, 128, 256, 257, 264, 511,
          512, 520, 777, 1024, 1032, 2048, 2056, 2500, 4096, 4104, 8192, 8200,
          12544, 16384, 16392, 20000]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype,wdtype", [
    (torch.float32, torch.float32), (torch.bfloat16, torch.float32),
    (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32),
    (torch.float16, torch.float16)])
def test_widths(device, dtype, wdtype):
    for width in WIDTHS:
        check(*inputs(5, width, dtype, wdtype, device, seed=width))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows", [1, 2, 3, 31, 33, 400, 1025, 9000])
@pytest.mark.parametrize("width", [7, 256])
def test_rows(device, rows, width):
    check(*inputs(rows, width, torch.bfloat16, torch.float32, device, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width", [(131072, 256), (70000, 24),
                                        (2050, 16392)])
def test_many_rows(rows, width):
    check(*inputs(rows, width, torch.bfloat16, torch.float32, "cuda"))


@pytest.mark.parametrize("device", DEVICES)
def test_offsets_and_scales(device):
    """A mean far from 0, a constant row, a tiny and a huge row."""
    x, w, b, dy = inputs(6, 300, torch.float32, torch.float32, device)
    x[0] += 1000.0
    x[1] = 3.25
    x[2] *= 1e-6
    x[3] *= 1e15
    x[4] = 0.0
    check(x, w, b, dy)


@pytest.mark.parametrize("device", DEVICES)
def test_optional_parameters(device):
    x, w, b, dy = inputs(9, 48, torch.bfloat16, torch.float32, device)
    check(x, None, None, dy)
    check(x, w, None, dy)
    check(x, None, b, dy)


@pytest.mark.parametrize("device", DEVICES)
def test_strides_and_shapes(device):
    x, w, b, dy = inputs(12, 64, torch.bfloat16, torch.float32, device)
    wide = torch.zeros(12, 200, dtype=x.dtype, device=device)
    for at in (0, 1, 8):
        part = wide[:, at:at + 64]
        part.copy_(x)
        check(part, w, b, dy)
        check(x, w, b, part)
    check(x.t().contiguous().t(), w, b, dy)
    check(x[:1].expand(12, 64), w, b, dy)
    check(x, w, b, dy[:1].expand(12, 64))
    check(x.view(3, 4, 64), w, b, dy.view(3, 4, 64))
    check(x.view(3, 4, 64).transpose(0, 1), w, b, dy.view(4, 3, 64))
    check(x[::2], w, b, dy[::2])
    ww = torch.stack([w, w], 1)[:, 0]
    check(x, ww, b, dy)


@pytest.mark.parametrize("device", DEVICES)
def test_no_rows(device):
    x, w, b, _ = inputs(1, 16, torch.float32, torch.float32, device)
    got = run(x[:0], w, b, x[:0])
    assert got["y"].shape == (0, 16) and got["dx"].shape == (0, 16)
    assert not got["dw"].any() and not got["db"].any()


@pytest.mark.parametrize("device", DEVICES)
def test_one_vector(device):
    x, w, b, _ = inputs(1, 16, torch.float32, torch.float32, device)
    assert torch.equal(layer_norm(x[0], w, b), layer_norm(x, w, b)[0])


@pytest.mark.parametrize("device", DEVICES)
def test_not_finite_stays_in_its_row(device):
    x, w, b, dy = inputs(4, 40, torch.float32, torch.float32, device)
    x[1, 3] = float("nan")
    x[2, 5] = float("inf")
    y = layer_norm(x, w, b)
    assert y[1].isnan().all() and y[2].isnan().all()
    assert y[0].isfinite().all() and y[3].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_by_differences(device):
    """The formula's gradient against differences of the 64-bit forward."""
    x, w, b, dy = inputs(3, 10, torch.float32, torch.float32, device)
    got = run(x, w, b, dy)
    h = 1e-5
    for name, t in (("dx", x), ("dw", w), ("db", b)):
        for i in range(0, t.numel(), 3):
            side = []
            for s in (h, -h):
                args = [a.double().clone() for a in (x, w, b)]
                args[("dx", "dw", "db").index(name)].view(-1)[i] += s
                side.append(float((exact(*args, dy, 1e-5)["y"] *
                                   dy.double()).sum()))
            # Differences: h^2 / 6 of a third derivative below 1e3, and
            # 1e-14 of cancellation over 2 h; fp32 adds 1e-5 of values to 30.
            assert abs((side[0] - side[1]) / (2 * h) -
                       float(got[name].view(-1)[i])) < 1e-4


def test_module():
    m = LayerNorm(12)
    x = torch.randn(4, 12)
    assert torch.equal(m(x), layer_norm(x, m.weight, m.bias, 1e-5))
    assert set(m.state_dict()) == {"weight", "bias"}


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x, w, b, _ = inputs(2, 8, torch.float32, torch.float32, device)
    with pytest.raises(RuntimeError):
        layer_norm(x, w[:4], b)
    with pytest.raises(RuntimeError):
        layer_norm(x, w, b[None])
    with pytest.raises(RuntimeError):
        layer_norm(x[:, :0], w[:0], b[:0])


@pytest.mark.gpu
def test_refusals_of_types_and_devices():
    x, w, b, _ = inputs(2, 8, torch.float32, torch.float32, "cuda")
    for args in ((x.double(), w, b), (x, w.half(), b.half()),
                 (x, w.cpu(), b), (x.bfloat16(), w, b.bfloat16())):
        with pytest.raises(RuntimeError):
            layer_norm(*args)


@pytest.mark.gpu
def test_same_gradients_every_time():
    x, w, b, dy = inputs(5000, 256, torch.bfloat16, torch.float32, "cuda")
    one, two = run(x, w, b, dy), run(x, w, b, dy)
    assert all(torch.equal(one[k], two[k]) for k in one)


@pytest.mark.gpu
def test_other_stream_and_graph():
    x, w, b, dy = inputs(200, 256, torch.bfloat16, torch.float32, "cuda")
    want = run(x, w, b, dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, w, b, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(want[k], got[k]) for k in want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer_norm(x, w, b)
    for seed in range(3):
        new = inputs(200, 256, torch.bfloat16, torch.float32, "cuda", seed)[0]
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, layer_norm(new, w, b))


@pytest.mark.gpu
def test_captured_backward():
    """Forward and backward in one graph, on leaves of its own."""
    x, w, b, dy = inputs(200, 264, torch.bfloat16, torch.float32, "cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)]

    def step():
        y = layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        new = inputs(200, 264, torch.bfloat16, torch.float32, "cuda", seed)
        with torch.no_grad():
            leaves[0].copy_(new[0])
        dy.copy_(new[3])
        graph.replay()
        torch.cuda.synchronize()
        want = run(new[0], w, b, new[3])
        for t, name in zip(out, ("y", "dx", "dw", "db")):
            assert torch.equal(t, want[name])


@pytest.mark.parametrize("device", DEVICES)
def test_no_second_gradient(device):
    x, w, b, dy = inputs(4, 16, torch.float32, torch.float32, device)
    x.requires_grad_()
    y = layer_norm(x, w, b)
    with pytest.raises(RuntimeError):
        d, = torch.autograd.grad(y, x, dy, create_graph=True)
        d.sum().backward()


@pytest.mark.parametrize("device", DEVICES)
def test_whole_numbers_are_refused(device):
    with pytest.raises(RuntimeError):
        layer_norm(torch.ones(2, 8, dtype=torch.int32, device=device))


@pytest.mark.parametrize("device", DEVICES)
def test_negative_views(device):
    x, w, b, dy = inputs(6, 16, torch.float32, torch.float32, device)

    def neg(t):
        held = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert held.is_neg()
        return held
    want, got = run(x, w, b, dy), run(neg(x), neg(w), neg(b), neg(dy))
    assert all(torch.equal(want[k], got[k]) for k in want)


@pytest.mark.gpu
def test_more_rows_than_one_launch_has():
    rows = (1 << 28) + 37
    x = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda")
    x[::5, 0] = 4.0
    y = layer_norm(x)
    for part in (slice(0, 100), slice((1 << 28) - 50, rows)):
        assert torch.equal(y[part], layer_norm(x[part].clone()))
    assert int((y[:, 0] > 0.5).sum()) == -(-rows // 5)


@pytest.mark.gpu
def test_captured_backward_of_a_held_leaf():
    """An earlier graph of a leaf, on another stream, is refused."""
    x, w, b, dy = inputs(40, 64, torch.bfloat16, torch.float32, "cuda")
    for i in range(3):
        leaves = [t.detach().clone().requires_grad_(i == j)
                  for j, t in enumerate((x, w, b))]
        held = layer_norm(*leaves)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="free that graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                y = layer_norm(*leaves)
                torch.autograd.grad(y, leaves[i], dy)
        want, = torch.autograd.grad(held, leaves[i], dy)
        del held, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer_norm(*leaves)
            got, = torch.autograd.grad(y, leaves[i], dy)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


@pytest.mark.parametrize("device", DEVICES)
def test_bias_may_change_before_the_backward(device):
    """It has no part in any gradient, so no version of it is kept."""
    x, w, b, dy = inputs(4, 16, torch.float32, torch.float32, device)
    b.requires_grad_()
    y = layer_norm(x, w, b)
    with torch.no_grad():
        b.add_(1.0)
    db, = torch.autograd.grad(y, b, dy)
    assert torch.allclose(db, dy.sum(0), rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(device, grad):
    """A result without a tangent would count as a derivative of zero."""
    args = inputs(4, 16, torch.float32, torch.float32, device)[:3]
    with torch.autograd.forward_ad.dual_level():
        for i in range(3):
            given = [t.clone().requires_grad_(grad and i != j)
                     for j, t in enumerate(args)]
            given[i] = torch.autograd.forward_ad.make_dual(
                given[i], torch.ones_like(given[i]))
            with pytest.raises(NotImplementedError):
                layer_norm(*given)
    assert layer_norm(*args).isfinite().all()


@pytest.mark.gpu
def test_more_wide_rows_than_one_launch_has():
    """Rows of 1024 threads each: 2^22 of them are 2^32."""
    rows, width = (1 << 22) + 3, 16400
    row = torch.zeros(width, dtype=torch.bfloat16, device="cuda")
    row[::5] = 4.0
    want = layer_norm(row)
    y = layer_norm(row.expand(rows, width))
    for part in (slice(0, 3), slice((1 << 21) - 2, (1 << 21) + 2),
                 slice(rows - 5, rows)):
        assert torch.equal(y[part], want.expand_as(y[part]))
    del y
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_gradient_of_many_wide_rows():
    """The backward's launch splits by rows as the forward's does: rows on
    either side of the border, in a view of the same memory."""
    rows, width = (1 << 21) + 2, 16400
    row = torch.zeros(width, dtype=torch.bfloat16, device="cuda")
    row[::5] = 4.0
    dy = torch.zeros_like(row)
    dy[7] = 1.0

    def grad(x, d):
        x = x.detach().requires_grad_()
        y = layer_norm(x)
        return torch.autograd.grad(y, x, d)[0]
    want = grad(row[None], dy[None])
    got = grad(row.expand(rows, width), dy.expand(rows, width))
    for part in (slice(0, 3), slice(rows - 5, rows)):
        assert torch.equal(got[part], want.expand_as(got[part]))
    del got
    torch.cuda.empty_cache()
