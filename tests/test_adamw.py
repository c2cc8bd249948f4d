"""adamw_step, grad_norm and the packed 8-bit states against 64 bits."""

import math

import numpy as np
import pytest
import torch

from maskrcnn_amd.ops import (
    adamw_step, grad_norm, pack_state8, unpack_state8,
)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
BLOCK = 256


def tensors(sizes, dtype, device, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(s, generator=g).mul(0.05).to(device, dtype)
         for s in sizes]
    gr = [torch.randn(s, generator=g).mul(scale).to(device, dtype)
          for s in sizes]
    m = [torch.randn(s, generator=g).mul(scale / 2).to(device)
         for s in sizes]
    v = [torch.randn(s, generator=g).mul(scale).square().to(device)
         for s in sizes]
    return p, gr, m, v


HYPER = dict(step=7, lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def exact(p, g, m, v, clip, step, lr, betas, eps, weight_decay):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    u = lr / (1 - betas[0] ** step) * m / (
        torch.sqrt(v / (1 - betas[1] ** step)) + eps)
    return p * (1 - lr * weight_decay) - u, m, v, u


def bound_p(p, u, m, g, betas, dtype):
    """p: one rounding to its type, then fp32's: two on the decay and the
    difference, 8 on the update, whose numerator may cancel (three roundings
    of its own terms)."""
    terms = betas[0] * m.double().abs() + (1 - betas[0]) * g.double().abs()
    new = (betas[0] * m.double() + (1 - betas[0]) * g.double()).abs()
    part = u.abs() * terms / new.clamp(min=1e-300)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (half * 1.01 + 3 * U) * p.abs() + 3 * U * u.abs() + \
        8 * U * u.abs() + 4 * U * part + tiny


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [
    [1], [3], [4], [255, 256, 257], [1023, 1, 4097, 4096, 5],
    [(17, 3), (8, 4, 3, 3), (), (0,), (64,)], [70000]])
def test_step_32(device, dtype, sizes):
    p, g, m, v = tensors(sizes, dtype, device)
    was = [[t.clone() for t in k] for k in (p, m, v)]
    adamw_step(p, g, m, v, **HYPER)
    for i in range(len(p)):
        ep, em, ev, u = exact(was[0][i], g[i], was[1][i], was[2][i], 1.0,
                              **HYPER)
        off = (p[i].double() - ep).abs()
        assert (off <= bound_p(ep, u, was[1][i], g[i], HYPER["betas"],
                               dtype)).all()
        # Two products, a sum, and the constants' own rounding.
        em_abs = 0.9 * was[1][i].double().abs() + 0.1 * g[i].double().abs()
        assert ((m[i].double() - em).abs() <= 4 * U * em_abs).all()
        assert ((v[i].double() - ev).abs() <= 5 * U * ev).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(device, bits):
    """More tensors than a launch takes, of two types, one of them empty."""
    sizes = [(i * 37) % 700 + (i % 7 == 0) * 4096 for i in range(200)]
    p, g, m, v = tensors(sizes, torch.float32, device)
    for i in range(0, 200, 3):
        p[i], g[i] = p[i].bfloat16(), g[i].bfloat16()
    if bits == 8:
        packed = [pack_state8(t, True) for t in m], \
            [pack_state8(t, False) for t in v]
        (m, ms), (v, vs) = (map(list, zip(*k)) for k in packed)
        scales = dict(exp_avg_scales=ms, exp_avg_sq_scales=vs)
    else:
        scales = {}
    one = [[t.clone() for t in k] for k in (p, g, m, v)]
    two = {k: [t.clone() for t in v] for k, v in scales.items()}
    adamw_step(p, g, m, v, **scales, **HYPER)
    for i in range(200):      # the same, one tensor a call
        adamw_step(*[k[i:i + 1] for k in one],
                   **{k: t[i:i + 1] for k, t in two.items()}, **HYPER)
        for a, b in zip((p, m, v), (one[0], one[2], one[3])):
            assert torch.equal(a[i], b[i])
        for k in scales:
            assert torch.equal(scales[k][i], two[k][i])


@pytest.mark.parametrize("device", DEVICES)
def test_norm(device):
    g = torch.Generator().manual_seed(3)
    sizes = [1, 5, 4096, 4097, 100003, 0, 33] + [7] * 300
    t = [torch.randn(n, generator=g).to(device, TYPES[i % 3])
         for i, n in enumerate(sizes)]
    want = math.sqrt(sum(float(x.double().square().sum()) for x in t))
    assert abs(float(grad_norm(t)) - want) <= 1.01 * U * want
    assert float(grad_norm([t[0][:0]])) == 0.0
    assert abs(float(grad_norm([t[4].view(-1)[::2]])) - math.sqrt(float(
        t[4][::2].double().square().sum()))) <= 1.01 * U * want
    t[3][7] = float("inf")
    assert float(grad_norm(t)) == math.inf
    t[2][7] = float("nan")
    assert math.isnan(float(grad_norm(t)))
    # Squares past fp32's range.
    big = torch.full((10,), 1e30, device=device)
    assert abs(float(grad_norm([big])) / (1e30 * math.sqrt(10)) - 1) < 1e-6


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1e-4, 1.0])
def test_clipped_step(device, scale):
    p, g, m, v = tensors([300, 5000], torch.float32, device, scale=scale)
    was = [[t.clone() for t in k] for k in (p, g, m, v)]
    norm = grad_norm(g)
    adamw_step(p, g, m, v, grad_norm=norm, max_grad_norm=5.0, **HYPER)
    n = math.sqrt(sum(float(t.double().square().sum()) for t in g))
    clip = min(1.0, 5.0 / (n + 1e-6))
    assert (clip < 1) == (scale == 1.0)
    for i in range(2):
        assert torch.equal(g[i], was[1][i])
        ep, em, ev, u = exact(was[0][i], g[i], was[2][i], was[3][i], clip,
                              **HYPER)
        lim = bound_p(ep, u, was[2][i], g[i] * clip, HYPER["betas"],
                      torch.float32)
        # The factor: 3 roundings in itself, once on g.
        assert ((p[i].double() - ep).abs() <= 2 * lim).all()
        em_abs = 0.9 * was[2][i].double().abs() + \
            0.1 * g[i].double().abs() * clip
        assert ((m[i].double() - em).abs() <= 8 * U * em_abs).all()
        assert ((v[i].double() - ev).abs() <= 13 * U * ev).all()


# ------------------------------------------------------------ 8-bit states

def grid(x, signed):
    """x in 64 bits rounded to the code's values, to nearest even."""
    low = 14 if signed else 30
    n = x.numel()
    b = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    b[:n] = x.double().reshape(-1).cpu()
    b = b.view(-1, BLOCK)
    _, e = torch.frexp(b.abs().amax(1, keepdim=True))
    unit = torch.ldexp(torch.ones_like(b[:, :1]), (e - 1).clamp(min=40 - 127))
    r = b.abs() / unit
    _, k = torch.frexp(r)
    k = (k - 1).clamp(min=-low) - 3
    q = torch.ldexp(torch.round(torch.ldexp(r, -k)), k).clamp(max=1.875)
    if not signed:
        q = torch.where((r > 0) & (q == 0), 2.0 ** -(low + 3), q)
    return (torch.sign(b) * q * unit).view(-1)[:n].view(x.shape).to(x.device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("n", [0, 1, 2, 255, 256, 257, 513, 70001])
def test_pack(device, signed, n):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * torch.exp(
        6 * torch.randn(n, generator=g))
    x = (x if signed else x.square()).to(device)
    codes, scales = pack_state8(x, signed)
    assert codes.shape == x.shape and scales.numel() == -(-n // BLOCK)
    got = unpack_state8(codes, scales, signed)
    assert torch.equal(got.double(), grid(x, signed))
    assert torch.equal(
        unpack_state8(codes, scales, signed, torch.bfloat16).float(), got)
    # What is held packs to itself.
    again, s = pack_state8(got, signed)
    assert torch.equal(unpack_state8(again, s, signed), got)
    # Half a step of 3 bits where the ratio is a normal one, both codes.
    top = torch.zeros(-(-n // BLOCK) * BLOCK)
    top[:n] = x.abs().cpu()
    top = top.view(-1, BLOCK).amax(1).repeat_interleave(BLOCK)[:n].to(device)
    near = x.abs() >= top * (2.0 ** -13 if signed else 2.0 ** -29)
    assert ((got - x).abs() <= x.abs() * 2.0 ** -4)[near].all()


@pytest.mark.parametrize("device", DEVICES)
def test_every_code(device):
    for signed in (True, False):
        codes = torch.arange(256, dtype=torch.uint8, device=device)
        for e in (40, 127, 200, 254):
            scales = torch.full((1,), e, dtype=torch.uint8, device=device)
            got = unpack_state8(codes, scales, signed).double().cpu()
            c = torch.arange(256)
            mag = (c & 127) if signed else c
            low = 14 if signed else 30
            ex, man = mag >> 3, (mag & 7).double()
            want = torch.where(ex > 0, (1 + man / 8) *
                               2.0 ** (ex - 1 - low).double(),
                               man / 8 * 2.0 ** -low)
            want = want * 2.0 ** (e - 127)
            if signed:
                want = torch.where(c > 127, -want, want)
            fits = want.abs() < 3.4e38
            assert torch.equal(got[fits], want[fits])


@pytest.mark.parametrize("device", DEVICES)
def test_pack_edges(device):
    x = torch.zeros(1024, device=device)
    codes, scales = pack_state8(x, False)
    assert not codes.any()
    assert not unpack_state8(codes, torch.zeros_like(scales), False).any()
    x[0], x[1] = 1.0, 1e-38          # far below the block's largest
    x[300] = float("inf")
    x[600] = float("nan")
    x[768:] = 1e-42                  # subnormal
    big = torch.tensor([3e38, 1e38, 2.0 ** 127, 2.0 ** 126], device=device)
    for signed in (True, False):
        y = unpack_state8(*pack_state8(big, signed), signed)
        assert ((y - big).abs() <= big * 2.0 ** -4).all()
    for signed in (True, False):
        y = unpack_state8(*pack_state8(x, signed), signed)
        assert y[0] == 1.0 and (y[1] > 0) == (not signed)
        assert y[256:768].isnan().all()
        assert y[2:256].abs().sum() == 0
        assert (y[768:] > 0).all() == (not signed)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [255], [256, 257, 3], [1025, 4097],
                                   [(16, 9, 3), (0,), (70001,)]])
def test_step_8(device, dtype, sizes):
    p, g, m, v = tensors(sizes, dtype, device)
    (m, ms), (v, vs) = (map(list, zip(*[pack_state8(t, k == 0) for t in s]))
                        for k, s in enumerate((m, v)))
    was_p = [t.clone() for t in p]
    m0 = [unpack_state8(a, b, True) for a, b in zip(m, ms)]
    v0 = [unpack_state8(a, b, False) for a, b in zip(v, vs)]
    adamw_step(p, g, m, v, exp_avg_scales=ms, exp_avg_sq_scales=vs, **HYPER)
    for i in range(len(p)):
        ep, em, ev, u = exact(was_p[i], g[i], m0[i], v0[i], 1.0, **HYPER)
        # The update goes by the states before they are rounded to 8 bits.
        assert ((p[i].double() - ep).abs() <= bound_p(
            ep, u, m0[i], g[i], HYPER["betas"], dtype)).all()
        if not p[i].numel():
            continue
        # fp32's error first (as in 32 bits), then half a step of the code:
        # where that error crosses a border, a whole step.
        for got, want, signed, err in (
                (unpack_state8(m[i], ms[i], True), em, True, 4 * U * (
                    0.9 * m0[i].double().abs() +
                    0.1 * g[i].double().abs())),
                (unpack_state8(v[i], vs[i], False), ev, False, 5 * U * ev)):
            off = (got.double() - grid(want, signed)).abs()
            far = off > 0
            assert far.float().mean() <= 0.02 + 1 / want.numel()
            step = grid(want, signed).abs().double() / 8 * 1.01
            assert (off <= step + err)[far].all()


@pytest.mark.parametrize("device", DEVICES)
def test_zero_state_begins(device):
    """Zeros in codes and scales are a state of zeros."""
    p, g, _, _ = tensors([300], torch.float32, device)
    q = [p[0].clone()]
    z32 = [torch.zeros(300, device=device) for _ in range(2)]
    z8 = [torch.zeros(300, dtype=torch.uint8, device=device)
          for _ in range(2)]
    s8 = [torch.zeros(2, dtype=torch.uint8, device=device) for _ in range(2)]
    hyper = dict(HYPER, step=1)
    adamw_step(p, g, z32[:1], z32[1:], **hyper)
    adamw_step(q, g, z8[:1], z8[1:], exp_avg_scales=s8[:1],
               exp_avg_sq_scales=s8[1:], **hyper)
    assert torch.equal(p[0], q[0])


@pytest.mark.parametrize("device", DEVICES)
def test_not_finite_gradient_shows(device):
    p, g, m, v = tensors([600], torch.float32, device)
    (mc, ms), (vc, vs) = pack_state8(m[0], True), pack_state8(v[0], False)
    g[0][300] = float("nan")
    adamw_step(p, g, [mc], [vc], exp_avg_scales=[ms], exp_avg_sq_scales=[vs],
               **HYPER)
    assert p[0].isnan().sum() == 1
    for y in (unpack_state8(mc, ms, True), unpack_state8(vc, vs, False)):
        assert y[256:512].isnan().all() and y[:256].isfinite().all() \
            and y[512:].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_strides(device):
    """channels_last parameters, gradients in another layout, odd starts."""
    p, g, m, v = tensors([(8, 6, 3, 3)], torch.float32, device)
    ref = [[t.clone() for t in k] for k in (p, g, m, v)]
    adamw_step(*ref, **HYPER)
    cl = torch.channels_last
    q, mm, vv = (k[0].to(memory_format=cl) for k in (p, m, v))
    adamw_step([q], g, [mm], [vv], **HYPER)     # gradient contiguous
    assert q.is_contiguous(memory_format=cl)
    for a, b in zip((q, mm, vv), (ref[0], ref[2], ref[3])):
        assert torch.equal(a, b[0])
    for start in (1, 2, 3, 4):
        base = [torch.zeros(450, device=device) for _ in range(4)]
        part = []
        for t, k in zip(base, (p, g, m, v)):
            part.append(t[start:start + 432])
            part[-1].copy_(k[0].view(-1))
        adamw_step(*[[t] for t in part], **HYPER)
        assert torch.equal(part[0], ref[0][0].view(-1))
        for t in base:
            assert not t[:start].any() and not t[start + 432:].any()


@pytest.mark.parametrize("device", DEVICES)
def test_neighbours_stay(device):
    """Codes and scales around a tensor's own are left as they were."""
    p, g, m, v = tensors([301], torch.bfloat16, device)
    codes = [torch.full((320,), 77, dtype=torch.uint8, device=device)
             for _ in range(2)]
    scales = [torch.full((8,), 99, dtype=torch.uint8, device=device)
              for _ in range(2)]
    part, sc = [c[3:304] for c in codes], [s[2:4] for s in scales]
    for t, s, x, signed in zip(part, sc, (m[0], v[0]), (True, False)):
        a, b = pack_state8(x, signed)
        t.copy_(a)
        s.copy_(b)
    adamw_step(p, g, part[:1], part[1:], exp_avg_scales=sc[:1],
               exp_avg_sq_scales=sc[1:], **HYPER)
    for c in codes:
        assert (c[:3] == 77).all() and (c[304:] == 77).all()
    for s in scales:
        assert (s[:2] == 99).all() and (s[4:] == 99).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_gives_the_cpu_states(bits, dtype):
    sizes = [1, 300, 4096, 10000]
    a = tensors(sizes, dtype, "cpu")
    norm = grad_norm(a[1])
    scales = {}
    if bits == 8:
        (m, ms), (v, vs) = (
            map(list, zip(*[pack_state8(t, k == 0) for t in s]))
            for k, s in enumerate(a[2:]))
        a = (a[0], a[1], m, v)
        scales = dict(exp_avg_scales=ms, exp_avg_sq_scales=vs)
    b = [[t.cuda() for t in k] for k in a]
    bs = {k: [t.cuda() for t in s] for k, s in scales.items()}
    for step in (1, 2, 50):
        h = dict(HYPER, step=step, max_grad_norm=0.5)
        adamw_step(*a, **scales, grad_norm=norm, **h)
        adamw_step(*b, **bs, grad_norm=norm.cuda(), **h)
        for x, y in zip((*a[2:], *scales.values()), (*b[2:], *bs.values())):
            for s, t in zip(x, y):
                assert torch.equal(s, t.cpu())
        for s, t in zip(a[0], b[0]):
            # The update is below 100 lr; 4 units in its last place between
            # the two, a rounding of p each, the same again from a step
            # before it.
            half = torch.finfo(dtype).eps / 2
            off = (s.double() - t.cpu().double()).abs()
            assert (off <= 3 * (2 * half * s.double().abs() +
                                100 * HYPER["lr"] * 8 * U)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    p, g, m, v = tensors([8, 8], torch.float32, device)
    bad = [
        (p, g[:1], m, v, {}),
        (p, [g[0], g[1].bfloat16()], m, v, {}),
        (p, g, [m[0], m[1].bfloat16()], v, {}),
        (p, g, m, [v[0], v[1][:4]], {}),
        (p, [g[0], g[1][:4]], m, v, {}),
        ([t.double() for t in p], [t.double() for t in g], m, v, {}),
        (p, g, m, v, dict(exp_avg_scales=[m[0], m[1]])),
    ]
    for *args, more in bad:
        with pytest.raises(RuntimeError):
            adamw_step(*args, **more, **HYPER)
    for more in (dict(step=0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -1)),
                 dict(grad_norm=grad_norm(g))):
        with pytest.raises(ValueError):
            adamw_step(p, g, m, v, **{**HYPER, **more})
    with pytest.raises(RuntimeError):
        grad_norm([])
    with pytest.raises(RuntimeError):
        pack_state8(torch.zeros(4, dtype=torch.bfloat16, device=device), True)
    with pytest.raises(RuntimeError):
        unpack_state8(torch.zeros(4, dtype=torch.uint8, device=device),
                      torch.zeros(2, dtype=torch.uint8, device=device), True)
    adamw_step([], [], [], [], **HYPER)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    p, g, m, v = tensors([8, 8], torch.float32, "cuda")
    before = [t.clone() for t in p]
    for args in (([p[0], p[0]], g, m, v), (p, g, [m[0], m[0]], v),
                 (p, g, m, [v[0], m[0]]), ([p[0][:4], p[0][2:6]],
                                           [g[0][:4]] * 2,
                                           [t[:4] for t in m],
                                           [t[:4] for t in v]),
                 (p, [g[0], g[1].cpu()], m, v),
                 ([t[::2] for t in p], [t[::2] for t in g],
                  [t[::2] for t in m], [t[::2] for t in v])):
        with pytest.raises(RuntimeError):
            adamw_step(*args, **HYPER)
    both = torch.zeros(12, device="cuda")
    with pytest.raises(RuntimeError, match="shares memory"):
        adamw_step([both[:8]], [both[4:]], m[:1], v[:1], **HYPER)
    with pytest.raises(RuntimeError):
        adamw_step(p, g, m, v, grad_norm=torch.ones(()), max_grad_norm=1.0,
                   **HYPER)
    with pytest.raises(RuntimeError):
        grad_norm([g[0], g[1].cpu()])
    assert all(torch.equal(a, b) for a, b in zip(p, before))


@pytest.mark.gpu
def test_capture_is_refused_and_norm_replays():
    p, g, m, v = tensors([5000, 77], torch.float32, "cuda")
    graph = torch.cuda.CUDAGraph()
    grad_norm(g)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            adamw_step(p, g, m, v, **HYPER)
        out = grad_norm(g)
    for k in range(3):
        g[0].mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, grad_norm(g))


@pytest.mark.gpu
def test_other_stream():
    p, g, m, v = tensors([5000, 77], torch.float32, "cuda")
    a = [[t.clone() for t in k] for k in (p, g, m, v)]
    adamw_step(*a, grad_norm=grad_norm(a[1]), max_grad_norm=0.1, **HYPER)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        adamw_step(p, g, m, v, grad_norm=grad_norm(g), max_grad_norm=0.1,
                   **HYPER)
    s.synchronize()
    assert all(torch.equal(x, y) for k, j in zip((p, m, v), (a[0], a[2], a[3]))
               for x, y in zip(k, j))


@pytest.mark.parametrize("device", DEVICES)
def test_autograd_sees_the_change(device):
    """A graph that saved a parameter does not take its new values."""
    p, g, m, v = tensors([8], torch.float32, device)
    w = p[0].requires_grad_()
    x = torch.ones(8, device=device, requires_grad=True)
    y = (w * x).sum()
    adamw_step([w], g, m, v, **HYPER)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    with torch.inference_mode():
        q = [t.detach().clone() for t in (w, g[0], m[0], v[0])]
        adamw_step(*[[t] for t in q], **HYPER)


@pytest.mark.parametrize("device", DEVICES)
def test_shared_gradient(device):
    """One tensor may be the gradient of two parameters."""
    p, g, m, v = tensors([300, 300], torch.float32, device)
    one = [[t.clone() for t in k] for k in (p, m, v)]
    adamw_step(p, [g[0], g[0]], m, v, **HYPER)
    for i in range(2):
        adamw_step([one[0][i]], [g[0]], [one[1][i]], [one[2][i]], **HYPER)
        assert torch.equal(p[i], one[0][i])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.3, 0.2), (0.0, 0.0),
                                   (0.5, 0.5), (0.2, 0.99)])
def test_betas(device, betas):
    """Small ones as well, and states that tower over what comes."""
    p, g, m, v = tensors([5000], torch.float32, device)
    m[0][:2000] *= 1e6
    v[0][:2000] *= 1e9
    for _ in range(2):
        old = [t[0].clone() for t in (m, v)]
        adamw_step(p, g, m, v, **dict(HYPER, betas=betas))
        assert p[0].isfinite().all()
        # As in test_step_32, with these betas: two roundings of terms, a
        # sum's and the constants'.
        for got, was, new, beta in ((m[0], old[0], g[0].double(), betas[0]),
                                    (v[0], old[1], g[0].double().square(),
                                     betas[1])):
            a, b = beta * was.double(), (1 - beta) * new
            off = (got.double() - (a + b)).abs()
            assert (off <= 5 * U * (a.abs() + b.abs()) + 1e-40).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.3, 0.2)])
def test_overflown_state(device, betas):
    """It stays one and leaves its parameter to the decay alone."""
    p, g, m, v = tensors([300], torch.float32, device)
    v[0][7] = float("inf")
    for _ in range(2):
        was = float(p[0][7])
        adamw_step(p, g, m, v, **dict(HYPER, betas=betas))
        assert v[0][7].isinf() and v[0].isinf().sum() == 1
        assert abs(float(p[0][7]) - was * (1 - 1e-4)) <= 2 * U * abs(was)
        assert p[0].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_codes_are_the_unrounded_states(device):
    """Sums that fp32 rounds to the middle between two codes: (1 + g) / 2 with
    g = 1.125 + k 2^-23 lies k/2 units above or below it."""
    n, u = 512, 2.0 ** -23
    m = torch.ones(n, device=device)
    g = torch.full((n,), 1.125, device=device)
    g[0::4] += u
    g[1::4] -= u
    g[2::4] += 3 * u
    mc, ms = pack_state8(m, True)
    vc, vs = pack_state8(m, False)
    adamw_step([m.clone()], [g], [mc], [vc], exp_avg_scales=[ms],
               exp_avg_sq_scales=[vs], step=1, lr=0.1, betas=(0.5, 0.5))
    got = unpack_state8(mc, ms, True)
    # The middle itself goes to the even code.
    for at, want in enumerate((1.125, 1.0, 1.125, 1.0)):
        assert (got[at::4] == want).all(), at
    square = g * g
    want = (1.0 + square.double()) / 2
    assert torch.equal(unpack_state8(vc, vs, False), grid(want, False))


# ------------------------------------------ 8-bit states rounded at random

def eight(m, v):
    """(codes of m, codes of v, the scales as adamw_step takes them)"""
    (m, ms), (v, vs) = (map(list, zip(*[pack_state8(t, k == 0) for t in s]))
                        for k, s in enumerate((m, v)))
    return m, v, dict(exp_avg_scales=ms, exp_avg_sq_scales=vs)


def held(m, v, scales, i=0):
    return (unpack_state8(m[i], scales["exp_avg_scales"][i], True),
            unpack_state8(v[i], scales["exp_avg_sq_scales"][i], False))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.3, 0.2)])
def test_seeded_codes_have_the_states_mean(device, dtype, betas):
    """Over 400 seeds: each code lies next to the unrounded state, and their
    mean is the state to six deviations (each at most half a distance of two
    codes), value by value and over all values."""
    n, seeds = 600, 400
    p, g, m, v = tensors([n], dtype, device)
    spread = torch.exp(3 * torch.randn(
        n, generator=torch.Generator().manual_seed(1))).to(device)
    m[0], v[0] = m[0] * spread, v[0] * spread
    m, v, scales = eight(m, v)
    hyper = dict(HYPER, betas=betas)
    _, em, ev, _ = exact(p[0], g[0], *held(m, v, scales), 1.0, **hyper)
    total = [0.0, 0.0]
    for seed in range(seeds):
        a = [[t.clone() for t in k] for k in (p, m, v)]
        s = {k: [t.clone() for t in x] for k, x in scales.items()}
        adamw_step(a[0], g, a[1], a[2], **s, seed=seed, **hyper)
        if seed == 0:       # the update goes by the unrounded states
            one = [[t.clone() for t in k] for k in (p, m, v)]
            adamw_step(one[0], g, one[1], one[2], **hyper, **{
                k: [t.clone() for t in x] for k, x in scales.items()})
            assert torch.equal(one[0][0], a[0][0])
        got = held(a[1], a[2], s)
        for k, (x, want) in enumerate(zip(got, (em, ev))):
            # The code's distance: an eighth of the power of two below; for
            # the smallest, of the block's exponent or the next.
            low = 14 if k == 0 else 30
            _, e = torch.frexp(want.abs())
            top = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64,
                              device=device)
            top[:n] = want.abs()
            _, unit = torch.frexp(top.view(-1, BLOCK).amax(1))
            unit = unit.repeat_interleave(BLOCK)[:n]
            dist = 2.0 ** torch.maximum(e - 4, unit - low - 3).double()
            err = 5 * U * (want.abs() + g[0].double().abs() ** (k + 1))
            assert ((x.double() - want).abs() <= dist + err).all()
            total[k] = total[k] + (x.double() - want) / dist
    for t in total:
        t = t / seeds
        assert (t.abs() <= 6 * 0.5 / seeds ** 0.5).all()
        assert abs(t.mean()) <= 6 * 0.5 / (seeds * n) ** 0.5


@pytest.mark.parametrize("device", DEVICES)
def test_seeded_calls_repeat(device):
    p, g, m, v = tensors([700, 700, 300], torch.float32, device)
    for k in (p, g, m, v):
        k[1].copy_(k[0])
    m, v, scales = eight(m, v)

    def step(seed, only=slice(None), **more):
        a = [[t.clone() for t in k[only]] for k in (p, g, m, v)]
        s = {k: [t.clone() for t in x[only]] for k, x in scales.items()}
        adamw_step(*a, **s, seed=seed, **{**HYPER, **more})
        return a[2] + a[3]
    one = step(5)
    assert all(torch.equal(a, b) for a, b in zip(one, step(5)))
    assert all(torch.equal(a, b) for a, b in zip(one, step(np.int64(5))))
    # Other seeds, steps and tensors have bits of their own.
    for other in (step(6), step(5 + (1 << 40)), step(-5), step(5, step=8)):
        assert not torch.equal(one[0], other[0])
        assert not torch.equal(one[3], other[3])
    assert not torch.equal(one[0], one[1])
    alone = step(5, slice(0, 1))
    assert torch.equal(one[0], alone[0]) and torch.equal(one[3], alone[1])
    # fp32 states take no seed into account.
    a, b = (tensors([300], torch.float32, device) for _ in range(2))
    adamw_step(*a, **HYPER)
    adamw_step(*b, seed=1, **HYPER)
    assert all(torch.equal(x[0], y[0]) for x, y in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 255, 257, 600])
def test_seeded_edges(device, n):
    """Zeros stay zeros, a v above zero never gets the code of zero, the
    largest finite states stay finite, and NaN stays in its block."""
    z = torch.zeros(n, device=device)
    for seed in range(20):
        m, v, scales = eight([z], [z])
        adamw_step([z.clone()], [z], m, v, **scales, seed=seed, **HYPER)
        assert not m[0].any() and not v[0].any()
        x = z + 1e-30
        x[0] = 1.0
        m, v, scales = eight([z + 3.3e38], [x])
        adamw_step([z.clone()], [z], m, v, **scales, seed=seed,
                   **dict(HYPER, betas=(0.9999999, 0.9999999)))
        mm, vv = held(m, v, scales)
        assert mm.isfinite().all() and (mm >= 1.875 * 2.0 ** 127).all()
        assert (vv > 0).all() and 0.875 <= vv[0] <= 1.125
    g = z.clone()
    g[-1] = float("nan")
    m, v, scales = eight([z + 1], [z + 1])
    adamw_step([z.clone()], [g], m, v, **scales, seed=3, **HYPER)
    for y in held(m, v, scales):
        last = (n - 1) // BLOCK * BLOCK
        assert y[last:].isnan().all() and y[:last].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
def test_seeded_largest_value_grows(device):
    """A block whose values lie at the exponent's last code, 1.875, and whose
    steps are far below the distance to the next one, 2."""
    n = 4096
    z = torch.zeros(n, device=device)
    m, v, scales = eight([z], [z + 1.875])
    for step in range(1, 401):
        adamw_step([z.clone()], [z + 4.0 ** 0.5], m, v, **scales, seed=0,
                   step=step, lr=0.0, betas=(0.9, 0.999))
    want = 4.0 - (4.0 - 1.875) * 0.999 ** 400
    # Variance: 400 steps of at most (1 - beta2) (4 - v) D, D at most 1/4.
    dev = (400 * 0.001 * 2.125 * 0.25 / n) ** 0.5
    assert abs(float(held(m, v, scales)[1].double().mean()) - want) <= 6 * dev


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_gpu_gives_the_cpu_seeded_states(dtype):
    sizes = [1, 300, 4096, 10000, 0, 7]
    p, g, m, v = tensors(sizes, dtype, "cpu")
    m[2] *= torch.exp(6 * torch.randn(          # small codes as well
        4096, generator=torch.Generator().manual_seed(1)))
    m, v, scales = eight(m, v)
    a = (p, g, m, v)
    b = [[t.cuda() for t in k] for k in a]
    bs = {k: [t.cuda() for t in s] for k, s in scales.items()}
    for step in (1, 2, 50, (1 << 33) + 5):
        h = dict(HYPER, step=step, seed=(1 << 50) + 3)
        adamw_step(*a, **scales, **h)
        adamw_step(*b, **bs, **h)
        for x, y in zip((*a[2:], *scales.values()), (*b[2:], *bs.values())):
            for s, t in zip(x, y):
                assert torch.equal(s, t.cpu())


@pytest.mark.gpu
def test_seeded_places_past_32_bits():
    n = (1 << 32) + 600
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.full_like(p, 0.3)
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda")
            for _ in range(2))
    s = [torch.zeros(-(-n // BLOCK), dtype=torch.uint8, device="cuda")
         for _ in range(2)]
    adamw_step([p], [g], [m], [v], exp_avg_scales=s[:1],
               exp_avg_sq_scales=s[1:], seed=0, step=1, lr=0.5)
    for t in (m, v):
        first, last = t[:600], t[-600:]
        assert len(first.unique()) == 2 and len(last.unique()) == 2
        assert not torch.equal(first, last)
    assert (p[-600:] == p[0]).all() and p[0] < 0


@pytest.mark.gpu
def test_pack_more_than_one_launch_has():
    n = (1 << 34) + 300
    x = torch.zeros(n, device="cuda")
    at = torch.tensor([0, (1 << 33) - 1, 1 << 33, (1 << 34) + 1, n - 1],
                      device="cuda")
    x[at] = torch.tensor([1.0, 2.0, 3.0, 4.0, 5.0], device="cuda")
    codes, scales = pack_state8(x, True)
    assert int(codes.count_nonzero()) == 5
    for i, want in zip(at.tolist(), (1.0, 2.0, 3.0, 4.0, 5.0)):
        part = slice(i // BLOCK * BLOCK, min(i // BLOCK * BLOCK + BLOCK, n))
        got = unpack_state8(codes[part], scales[i // BLOCK:i // BLOCK + 1],
                            True)
        assert float(got[i % BLOCK]) == want
    del x, codes, scales
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_norm_in_a_tensor_to_write_is_refused():
    """Workgroups read it at any time, before and after it would change."""
    p, g, m, v = tensors([300, 8], torch.float32, "cuda")
    before = [t.clone() for k in (p, m, v) for t in k]
    for t in (p[0], m[1], v[0]):
        with pytest.raises(RuntimeError, match="shares memory"):
            adamw_step(p, g, m, v, grad_norm=t[3].abs_(), max_grad_norm=1.0,
                       **HYPER)
    for a, b in zip((t for k in (p, m, v) for t in k), before):
        assert torch.equal(a.abs(), b.abs())
    # A gradient is only read.
    g[0][0] = 2.0
    adamw_step(p, g, m, v, grad_norm=g[0][0], max_grad_norm=1.0, **HYPER)


@pytest.mark.parametrize("device", DEVICES)
def test_norm_has_a_gradient(device):
    """t / |g| for each tensor: three roundings, one of them to its type. And
    a gradient of it, and none where none is wanted."""
    g = torch.Generator().manual_seed(2)
    t = [torch.randn(n, generator=g).to(device, d)
         for n, d in ((5, torch.float32), (300, torch.bfloat16),
                      (0, torch.float32), (7, torch.float16))]
    assert not grad_norm(t).requires_grad
    for x in t[1:]:
        x.requires_grad_()
    with torch.no_grad():
        assert not grad_norm(t).requires_grad
    norm = grad_norm(t)
    got = torch.autograd.grad(norm * 3.0, t[1:], retain_graph=True)
    n = float(norm.detach())
    for x, d in zip(t[1:], got):
        want = 3.0 * x.detach().double() / n
        half = torch.finfo(x.dtype).eps / 2
        assert d.dtype == x.dtype and d.shape == x.shape
        assert ((d.double() - want).abs() <= (half * 1.01 + 4 * U) *
                want.abs() + torch.finfo(x.dtype).smallest_normal).all()
    x = torch.tensor([3.0, 4.0], device=device, requires_grad=True)
    d, = torch.autograd.grad(grad_norm([x]), x, create_graph=True)
    dd, = torch.autograd.grad(d[0], x)
    # d/dx of x0 / |x| is (1 - x0^2 / n^2) / n and -x0 x1 / n^3.
    want = torch.tensor([0.128, -0.096], device=device)
    assert ((dd - want).abs() <= 16 * U).all()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(),
                                                   torch.ones_like(x))
        if device == "cuda":
            with pytest.raises(NotImplementedError):
                grad_norm([dual])
