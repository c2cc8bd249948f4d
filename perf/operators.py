"""Cases and plain forms of the training and head operators.

Three operators: a matrix product with bias, activation and residual in
its epilogue (``linear_act``), a layer norm (``layer_norm``) and an AdamW
step over many tensors with states in 32 or 8 bits (``adamw_step`` with
``grad_norm``). ``run`` computes them from elementary torch operations
where ``own`` is false, and through ``maskrcnn_amd.ops`` where it is true.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16,
          "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
LN_EPS = 1e-5
# AdamW's settings: the clip norm is the training configuration's.
LR, BETA1, BETA2, EPS, DECAY = 1e-4, 0.9, 0.999, 1e-8, 1e-2
MAX_NORM = 5.0
BLOCK = 256            # values that share one scale in an 8-bit state


# ------------------------------------------------------------------ cases

def listed():
    return [
        # Class scores of one image's detections: a small product with an
        # odd width, where the call's latency counts.
        {"name": "logits 100x1024x81", "op": "linear", "m": 100, "k": 1024,
         "n": 81, "act": "none", "residual": False, "train": False,
         "dtype": "bf16"},
        # The box head's first layer over one image's proposals.
        {"name": "fc1 1000x12544x1024", "op": "linear", "m": 1000,
         "k": 12544, "n": 1024, "act": "relu", "residual": False,
         "train": False, "dtype": "bf16"},
        # The same layer over a served batch of 32 images.
        {"name": "fc1 32000x12544x1024", "op": "linear", "m": 32000,
         "k": 12544, "n": 1024, "act": "relu", "residual": False,
         "train": False, "dtype": "bf16"},
        # The same layer in a training step of two images, 200 RoIs each.
        {"name": "fc1 train 400x12544x1024", "op": "linear", "m": 400,
         "k": 12544, "n": 1024, "act": "relu", "residual": False,
         "train": True, "dtype": "bf16"},
        # A residual layer over two images' training proposals, a row short.
        {"name": "residual train 3999x1024", "op": "linear", "m": 3999,
         "k": 1024, "n": 1024, "act": "gelu", "residual": True,
         "train": True, "dtype": "fp16"},
        # The box deltas' layer trained in 32 bits.
        {"name": "deltas train fp32", "op": "linear", "m": 200, "k": 1024,
         "n": 324, "act": "none", "residual": False, "train": True,
         "dtype": "fp32"},
        # The box head's norm in a training step.
        {"name": "norm train 400x1024", "op": "norm", "rows": 400,
         "width": 1024, "train": True, "dtype": "bf16", "wdtype": "fp32"},
        # The finest pyramid level of two images, a norm over channels.
        {"name": "norm train 131072x256", "op": "norm", "rows": 131072,
         "width": 256, "train": True, "dtype": "bf16", "wdtype": "fp32"},
        # Whole pooled tiles of one image's proposals, forward alone.
        {"name": "norm 1000x12544 fp32", "op": "norm", "rows": 1000,
         "width": 12544, "train": False, "dtype": "fp32",
         "wdtype": "fp32"},
        # Fine-tuning of the last two layers alone: few small tensors.
        {"name": "adamw last layers", "op": "adamw", "tensors": 4,
         "largest": 331776, "layers": "last", "bits": 32, "dtype": "fp32"},
        # A step over the whole detector with the 101-layer backbone.
        {"name": "adamw resnet101", "op": "adamw", "tensors": 250,
         "largest": 12845056, "layers": "all", "bits": 32,
         "dtype": "fp32"},
        # The same with both states in 8 bits.
        {"name": "adamw8 resnet101", "op": "adamw", "tensors": 250,
         "largest": 12845056, "layers": "all", "bits": 8, "dtype": "fp32"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(
        rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "norm", "adamw"])
    if kind == "linear":
        m, k, n = _log(rng, 1, 32000), _log(rng, 1, 12544), _log(rng, 1, 4096)
        small = m * k * n * 16 < 32000 * 12544 * 1024
        train = small and rng.random() < 0.5
        dtype = rng.choice(["bf16", "fp16", "fp32"] if small
                           else ["bf16", "fp16"])
        # In 32 bits relu's slope flips where two orders of one sum lie on
        # either side of 0, so its gradient is drawn in 16 bits alone.
        return {"op": "linear", "m": m, "k": k, "n": n,
                "act": rng.choice(["none", "gelu", "silu"] +
                                  ["relu"] * (not train or dtype != "fp32")),
                "residual": rng.random() < 0.5, "train": train,
                "dtype": dtype}
    if kind == "norm":
        width = _log(rng, 1, 16384)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        return {"op": "norm", "width": width,
                "rows": _log(rng, 1, min(262144, (1 << 25) // width)),
                "train": rng.random() < 0.6, "dtype": dtype,
                "wdtype": rng.choice([dtype, "fp32"])}
    tensors, largest = _log(rng, 1, 250), _log(rng, 1, 1 << 22)
    return {"op": "adamw", "tensors": tensors, "largest": largest,
            "layers": "drawn", "split": rng.randrange(1 << 20),
            "bits": rng.choice([8, 32]),
            "dtype": rng.choice(["fp32", "bf16"])}


def _sizes(case):
    """(sizes of the decayed tensors, sizes of the others)."""
    if case["layers"] == "drawn":
        g = torch.Generator().manual_seed(case["split"])
        u = torch.rand(case["tensors"], generator=g, dtype=torch.float64)
        sizes = (case["largest"] ** u).long().clamp(min=1).tolist()
        return sizes[::2], sizes[1::2]
    last = [(81, 1024), (324, 1024)]
    if case["layers"] == "last":
        convs = last
    else:
        convs, width = [(64, 3 * 49)], 64
        for blocks, planes in ((3, 64), (4, 128), (23, 256), (3, 512)):
            convs.append((planes * 4, width))
            for _ in range(blocks):
                convs += [(planes, width), (planes, planes * 9),
                          (planes * 4, planes)]
                width = planes * 4
        convs += [(256, c) for c in (256, 512, 1024, 2048)]
        convs += [(256, 256 * 9)] * 4                        # pyramid
        convs += [(512, 256 * 9), (6, 512), (12, 512)]       # proposals
        convs += [(1024, 12544), (1024, 1024)] + last        # box head
        convs += [(256, 256 * 9)] * 4 + [(256, 1024), (81, 256)]  # masks
    return [a * b for a, b in convs], [a for a, _ in convs]


def work(case):
    if case["op"] == "linear":
        m, k, n, b = case["m"], case["k"], case["n"], BYTES[case["dtype"]]
        once = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if not case["train"]:
            return {"bytes": once * b, "flops": 2.0 * m * n * k}
        back = m * n + m * k + n * k + n + (m * n if case["residual"] else 0)
        return {"bytes": (once + back) * b, "flops": 6.0 * m * n * k}
    if case["op"] == "norm":
        r, c, b, w = (case["rows"], case["width"], BYTES[case["dtype"]],
                      BYTES[case["wdtype"]])
        if not case["train"]:
            return {"bytes": 2 * r * c * b + 2 * c * w, "flops": 8.0 * r * c}
        return {"bytes": 4 * r * c * b + 4 * c * w, "flops": 20.0 * r * c}
    count = sum(sum(s) for s in _sizes(case))
    each = 3 * BYTES[case["dtype"]] + (16 if case["bits"] == 32 else 8)
    return {"bytes": count * each, "flops": 20.0 * count}


# ----------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda",
                           dtype=dtype).mul_(scale)

    if case["op"] == "linear":
        m, k, n, t = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
        s = {"case": case, "x": normal(m, k, dtype=t),
             "w": normal(n, k, dtype=t, scale=math.sqrt(2.0 / k)),
             "b": normal(n, dtype=t, scale=0.1),
             "r": normal(m, n, dtype=t) if case["residual"] else None}
        if case["train"]:
            s["dy"] = normal(m, n, dtype=t, scale=0.1)
            for name in ("x", "w", "b", "r"):
                if s[name] is not None:
                    s[name].requires_grad_()
        return s
    if case["op"] == "norm":
        r, c = case["rows"], case["width"]
        t, tw = DTYPES[case["dtype"]], DTYPES[case["wdtype"]]
        s = {"case": case, "x": normal(r, c, dtype=t, scale=2.0).add_(0.5),
             "w": normal(c, dtype=tw, scale=0.2).add_(1.0),
             "b": normal(c, dtype=tw, scale=0.2)}
        if case["train"]:
            s["dy"] = normal(r, c, dtype=t, scale=0.1)
            for name in ("x", "w", "b"):
                s[name].requires_grad_()
        return s
    t = DTYPES[case["dtype"]]
    groups = []
    # Gradients whose norm is about 8: early steps, which the norm clips.
    rms = 8.0 / math.sqrt(sum(sum(sizes) for sizes in _sizes(case)))
    for sizes, decay in zip(_sizes(case), (DECAY, 0.0)):
        if not sizes:
            continue
        # One buffer a group, each tensor a view that begins at a block.
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK) * BLOCK
        live = torch.zeros(total, device="cuda")
        for a, n in zip(starts, sizes):
            live[a:a + n] = 1.0
        group = {"decay": decay,
                 "p": normal(total, dtype=torch.float32,
                             scale=0.05).mul_(live).to(t),
                 "g": normal(total, dtype=torch.float32,
                             scale=rms).mul_(live).to(t)}
        m = normal(total, dtype=torch.float32, scale=0.3 * rms).mul_(live)
        v = normal(total, dtype=torch.float32, scale=0.6 * rms) \
            .square_().mul_(live)
        if case["bits"] == 8:
            group["m"], group["ms"] = _pack(m, True)
            group["v"], group["vs"] = _pack(v, False)
        else:
            group["m"], group["v"] = m, v
        for key in ("p", "g", "m", "v"):
            group[key + "_list"] = [group[key][a:a + n]
                                    for a, n in zip(starts, sizes)]
        if case["bits"] == 8:
            for key in ("ms", "vs"):
                group[key + "_list"] = [
                    group[key][a // BLOCK:a // BLOCK + -(-n // BLOCK)]
                    for a, n in zip(starts, sizes)]
        groups.append(group)
    return {"case": case, "groups": groups, "step": 100}


# ------------------------------------------------------------ plain forms

def _act(z, act):
    """The activation and its derivative."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * \
            (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    return z, torch.ones_like(z)


def _linear(s, wide):
    case, t = s["case"], s["x"].dtype
    x, w, b = s["x"].to(wide), s["w"].to(wide), s["b"].to(wide)
    z = x @ w.t() + b
    y, slope = _act(z, case["act"])
    if s["r"] is not None:
        y = y + s["r"].to(wide)
    if not case["train"]:
        return {"y": y.to(t)}
    dy = s["dy"].to(wide)
    dz = dy * slope
    out = {"y": y.to(t), "dx": (dz @ w).to(t), "dw": (dz.t() @ x).to(t),
           "db": dz.sum(0).to(t)}
    if s["r"] is not None:
        out["dr"] = dy.to(t)
    return out


def _norm(s, wide):
    x, w, b = s["x"].to(wide), s["w"].to(wide), s["b"].to(wide)
    xc = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(xc.square().mean(1, keepdim=True) + LN_EPS)
    xh = xc * rstd
    out = {"y": (xh * w + b).to(s["x"].dtype)}
    if s["case"]["train"]:
        dy = s["dy"].to(wide)
        d = dy * w
        dx = rstd * (d - d.mean(1, keepdim=True) -
                     xh * (d * xh).mean(1, keepdim=True))
        out.update(dx=dx.to(s["x"].dtype), dw=(dy * xh).sum(0).to(s["w"].dtype),
                   db=dy.sum(0).to(s["b"].dtype))
    return out


def _pack(x, signed):
    """fp32 values -> (8-bit codes, the blocks' exponents).

    A block of 256 shares the power of two 2^(E-127) that its largest
    magnitude has. A code is the ratio to it with 3 bits of mantissa: sign
    and 4 bits of exponent for the first moment, 5 bits of exponent for the
    second, whose values above zero never get the code of zero.
    """
    low, top = (14, 127) if signed else (30, 255)
    bits = x.abs().view(torch.int32)
    e = (bits.view(-1, BLOCK).amax(1) >> 23).clamp(min=40)
    one = torch.ldexp(torch.ones_like(e, dtype=torch.float32), 127 - e)
    r = (x.abs().view(-1, BLOCK) * one[:, None]).view(-1)
    rb = r.view(torch.int32)
    normal = ((rb + 0x7FFFF + ((rb >> 20) & 1)) >> 20) - ((126 - low) << 3)
    small = torch.round(r * 2.0 ** (low + 3)).to(torch.int32)
    code = torch.where(r >= 2.0 ** -low, normal.clamp(max=top), small)
    if signed:
        code = code | ((x.view(torch.int32) < 0).to(torch.int32) << 7)
    else:
        code = torch.where((x > 0) & (code == 0), 1, code)
    return code.to(torch.uint8), e.to(torch.uint8)


def _unpack(codes, scales, signed):
    """The values that the codes stand for, in 32 bits."""
    low = 14 if signed else 30
    c = codes.to(torch.int32)
    mag = c & 127 if signed else c
    normal = ((mag + ((126 - low) << 3)) << 20).view(torch.float32)
    r = torch.where(mag >= 8, normal, mag * 2.0 ** -(low + 3))
    if signed:
        r = torch.where(c > 127, -r, r)
    one = torch.ldexp(torch.ones_like(scales, dtype=torch.float32),
                      scales.to(torch.int32) - 127)
    return (r.view(-1, BLOCK) * one[:, None]).view(-1)


def _adamw(s):
    s["step"] += 1
    t = s["step"]
    total = sum(grp["g"].double().square().sum() for grp in s["groups"])
    norm = torch.sqrt(total).float()
    scale = (torch.full_like(norm, MAX_NORM) / (norm + 1e-6)).clamp(max=1.0)
    out = {"norm": norm}
    rate = LR / (1.0 - BETA1 ** t)
    inv = 1.0 / math.sqrt(1.0 - BETA2 ** t)
    for i, grp in enumerate(s["groups"]):
        g = grp["g"].float() * scale
        if s["case"]["bits"] == 8:
            m = _unpack(grp["m"], grp["ms"], True)
            v = _unpack(grp["v"], grp["vs"], False)
        else:
            m, v = grp["m"], grp["v"]
        m = m * BETA1 + g * (1.0 - BETA1)
        v = v * BETA2 + (g * g) * (1.0 - BETA2)
        step = m / (torch.sqrt(v) * inv + EPS)
        p = grp["p"].float() * (1.0 - LR * grp["decay"]) - step * rate
        grp["p"].copy_(p)
        out["p%d" % i] = grp["p"]
        if s["case"]["bits"] == 8:
            for key, x, signed in (("m", m, True), ("v", v, False)):
                codes, scales = _pack(x, signed)
                grp[key].copy_(codes)
                grp[key + "s"].copy_(scales)
                out[key + str(i)] = _unpack(
                    codes, scales, signed).to(torch.bfloat16)
        else:
            grp["m"].copy_(m)
            grp["v"].copy_(v)
            out["m%d" % i], out["v%d" % i] = grp["m"], grp["v"]
    return out


# ------------------------------------------------------- the framework's

def _own_linear(s):
    from maskrcnn_amd.ops import linear_act
    case = s["case"]
    y = linear_act(s["x"], s["w"], s["b"], activation=case["act"],
                   residual=s["r"])
    if not case["train"]:
        return {"y": y}
    names = [n for n in ("x", "w", "b", "r") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y.detach(),
            **{"d" + n: g for n, g in zip(names, grads)}}


def _own_norm(s):
    from maskrcnn_amd.ops import layer_norm
    y = layer_norm(s["x"], s["w"], s["b"], eps=LN_EPS)
    if not s["case"]["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def _own_adamw(s):
    from maskrcnn_amd.ops import adamw_step, grad_norm, unpack_state8
    s["step"] += 1
    eight = s["case"]["bits"] == 8
    norm = grad_norm([g for grp in s["groups"] for g in grp["g_list"]])
    out = {"norm": norm}
    for i, grp in enumerate(s["groups"]):
        adamw_step(grp["p_list"], grp["g_list"], grp["m_list"],
                   grp["v_list"],
                   exp_avg_scales=grp["ms_list"] if eight else None,
                   exp_avg_sq_scales=grp["vs_list"] if eight else None,
                   step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                   weight_decay=grp["decay"], grad_norm=norm,
                   max_grad_norm=MAX_NORM)
        out["p%d" % i] = grp["p"]
        for key, signed in (("m", True), ("v", False)):
            out[key + str(i)] = grp[key] if not eight else unpack_state8(
                grp[key], grp[key + "s"], signed=signed,
                dtype=torch.bfloat16)
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "norm": _own_norm,
                "adamw": _own_adamw}[op](state)
    with torch.no_grad():
        if op == "linear":
            return _linear(state, torch.float32)
        return _norm(state, torch.float32) if op == "norm" \
            else _adamw(state)


# ------------------------------------------------------------- in 64 bits

def _exact_linear(s):
    x, w, b = (s[k].detach().double() for k in ("x", "w", "b"))
    act = s["case"]["act"]
    z = torch.addmm(b, x, w.t())
    phi = torch.special.ndtr(z) if act == "gelu" else None
    y = {"none": lambda: z, "relu": lambda: torch.relu(z),
         "gelu": lambda: z * phi,
         "silu": lambda: z * torch.sigmoid(z)}[act]()
    if s["r"] is not None:
        y = y + s["r"].detach().double()
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].double()
    if act == "relu":
        dz = torch.where(z > 0, dy, torch.zeros_like(dy))
    elif act == "gelu":
        dz = dy * (phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
    elif act == "silu":
        sig = torch.sigmoid(z)
        dz = dy * (sig + z * sig * (1 - sig))
    else:
        dz = dy
    out = {"y": y, "dx": torch.mm(dz, w), "dw": torch.mm(dz.t(), x),
           "db": dz.sum(0)}
    if s["r"] is not None:
        out["dr"] = dy
    return out


def _exact_norm(s):
    x, w, b = (s[k].detach().double() for k in ("x", "w", "b"))
    var, mean = torch.var_mean(x, 1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + LN_EPS)
    xh = (x - mean) / sd
    out = {"y": torch.addcmul(b, xh, w)}
    if s["case"]["train"]:
        dy, c = s["dy"].double(), x.shape[1]
        d = dy * w
        out["dx"] = (c * d - d.sum(1, keepdim=True) -
                     xh * (d * xh).sum(1, keepdim=True)) / (c * sd)
        out["dw"], out["db"] = (dy * xh).sum(0), dy.sum(0)
    return out


def _grid(x, signed):
    """Values in 64 bits rounded to what an 8-bit state can hold."""
    low = 14 if signed else 30
    b = x.view(-1, BLOCK)
    _, e = torch.frexp(b.abs().amax(1, keepdim=True))
    unit = torch.ldexp(torch.ones_like(b[:, :1]), (e - 1).clamp(min=-87))
    r = b.abs() / unit
    _, k = torch.frexp(r)
    k = (k - 1).clamp(min=-low) - 3
    one = torch.ones_like(r)
    q = torch.round(torch.ldexp(r, -k)) * torch.ldexp(one, k)
    q = q.clamp(max=1.875)
    if not signed:
        q = torch.where((r > 0) & (q == 0), one * 2.0 ** -(low + 3), q)
    return (torch.sign(b) * q * unit).view(-1)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] != "adamw":
            return (_exact_linear if case["op"] == "linear"
                    else _exact_norm)(s)
        t = s["step"] + 1
        eight = case["bits"] == 8
        flat = torch.cat([grp["g"].double() for grp in s["groups"]])
        norm = torch.linalg.vector_norm(flat)
        out = {"norm": norm}
        scale = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
        for i, grp in enumerate(s["groups"]):
            g = grp["g"].double() * scale
            m, v = grp["m"], grp["v"]
            if eight:
                m, v = _unpack(m, grp["ms"], True), \
                    _unpack(v, grp["vs"], False)
            m = torch.lerp(g, m.double(), BETA1)
            v = torch.lerp(g * g, v.double(), BETA2)
            mh, vh = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
            p = grp["p"].double()
            out["p%d" % i] = p - LR * grp["decay"] * p - \
                LR * mh / (vh.sqrt() + EPS)
            out["m%d" % i] = _grid(m, True) if eight else m
            out["v%d" % i] = _grid(v, False) if eight else v
        return out
