"""The AdamW optimizer, the layer-normed box head, and the two in training."""

import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from maskrcnn_amd.engine.optim import AdamW
from maskrcnn_amd.engine.trainer import Trainer, build_optimizer
from maskrcnn_amd.model import MaskRCNN
from maskrcnn_amd.model.heads import FPNClassifierHead
from maskrcnn_amd.ops import unpack_state8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(device, seed=0):
    torch.manual_seed(seed)
    return nn.Sequential(nn.Linear(37, 64), nn.ReLU(),
                         nn.Linear(64, 5)).to(device)


def backward(model, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(16, 37, generator=g).to(next(model.parameters()).device)
    model.zero_grad(set_to_none=True)
    (model(x).square().sum() * 10).backward()


@pytest.mark.parametrize("device", DEVICES)
def test_steps_as_torchs(device):
    """Four steps, clipped, with decayed and other parameters, beside
    torch's AdamW and clip_grad_norm_ in 64 bits."""
    a, b = make(device), make(device).double()
    kw = dict(lr=1e-2, betas=(0.8, 0.95), eps=1e-6)

    def groups(m):
        return [{"params": [m[0].weight, m[2].weight], "weight_decay": 0.1},
                {"params": [m[0].bias, m[2].bias], "weight_decay": 0.0}]
    oa = AdamW(groups(a), max_grad_norm=1.5, **kw)
    ob = torch.optim.AdamW(groups(b), **kw)
    for seed in range(4):
        backward(a, seed)
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad = p.grad.double()
        before = [p.grad.clone() for p in a.parameters()]
        norm = torch.nn.utils.clip_grad_norm_(b.parameters(), 1.5)
        oa.step()
        ob.step()
        assert abs(float(oa.grad_norm) / float(norm) - 1) < 1e-6
        assert all(torch.equal(p.grad, g)
                   for p, g in zip(a.parameters(), before))
    for p, q in zip(a.parameters(), b.parameters()):
        # Values to 0.5, four updates of 0.01 each in fp32 (a few units of
        # the last place, more where the first moment cancels).
        assert (p.double() - q).abs().max() < 4e-7
    for p, q in zip(a.parameters(), b.parameters()):
        for k in ("exp_avg", "exp_avg_sq"):
            want = ob.state[q][k]
            assert (oa.state[p][k].double() - want).abs().max() <= \
                1e-6 * want.abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_and_copy(device, bits):
    a = make(device)
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    for seed in range(3):
        backward(a, seed)
        opt.step()
    saved = copy.deepcopy(opt.state_dict())
    b = copy.deepcopy(a)
    other = AdamW(b.parameters(), lr=5.0, state_bits=bits, max_grad_norm=1.0)
    other.load_state_dict(saved)
    for p, q in zip(a.parameters(), b.parameters()):
        for k, v in opt.state[p].items():
            w = other.state[q][k]
            assert w == v if k == "step" else (
                w.dtype == v.dtype and torch.equal(w, v) and
                w.data_ptr() != v.data_ptr())
    backward(a, 9)
    backward(b, 9)
    opt.step()
    other.step()
    assert all(torch.equal(p, q)
               for p, q in zip(a.parameters(), b.parameters()))
    twin = copy.deepcopy(other)
    assert (twin.state_bits, twin.max_grad_norm) == (bits, 1.0)
    with pytest.raises(ValueError, match="bits"):
        AdamW(b.parameters(), state_bits=40 - bits).load_state_dict(saved)
    sgd = torch.optim.SGD(b.parameters(), lr=0.1, momentum=0.9)
    sgd.step()
    with pytest.raises(ValueError):
        other.load_state_dict(sgd.state_dict())


@pytest.mark.parametrize("device", DEVICES)
def test_8_bit_state_in_another_layout(device):
    """Blocks lie in memory order: a state saved from a contiguous weight
    goes into a channels_last one by value."""
    torch.manual_seed(0)
    p = nn.Parameter(torch.randn(24, 20, 3, 3, device=device))
    opt = AdamW([p], state_bits=8)
    p.grad = torch.randn_like(p)
    opt.step()
    q = nn.Parameter(p.detach().to(memory_format=torch.channels_last))
    other = AdamW([q], state_bits=8)
    other.load_state_dict(opt.state_dict())
    for name, signed in (("exp_avg", True), ("exp_avg_sq", False)):
        one, two = (unpack_state8(o.state[t][name], o.state[t][f"{name}_scale"
                                  if name == "exp_avg" else
                                  "exp_avg_sq_scale"], signed)
                    for o, t in ((opt, p), (other, q)))
        # Blocks of other values: what was the smallest kept may round.
        top = one.abs().max()
        near = one.abs() > top * 2.0 ** -10
        assert torch.equal(one[near], two[near])
        assert ((one - two).abs() <= top * 2.0 ** -13).all()
    q.grad = p.grad.to(memory_format=torch.channels_last)
    other.step()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_missed_steps_and_empty(device, bits):
    """A parameter without gradients keeps its step number and value."""
    a, b = (nn.Parameter(torch.ones(300, device=device)) for _ in range(2))
    none = nn.Parameter(torch.ones(0, device=device))
    opt = AdamW([a, b, none], lr=0.1, state_bits=bits, max_grad_norm=10.0)
    opt.step()
    assert opt.grad_norm is None
    a.grad = torch.full_like(a, 0.01)
    none.grad = torch.ones_like(none)
    opt.step()
    assert (b == 1).all() and not opt.state[b]
    b.grad = torch.full_like(b, 0.01)
    opt.step()
    assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1
    # The first step of any constant gradient is lr (and the decay).
    want = 1 - 0.1 * 0.01 - 0.1
    assert (b - want).abs().max() < 1e-5


def test_refusals():
    p = [nn.Parameter(torch.ones(3))]
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)),
               dict(eps=-1.0), dict(weight_decay=-1.0),
               dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            AdamW(p, **kw)


# ---------------------------------------------------------------- the head

class HeadConfig:
    POOL_SIZE = 7
    FPN_CLASSIF_FC_LAYERS_SIZE = 64
    NUM_CLASSES = 5
    TRAIN_BN = False
    IMAGE_SHAPE = [128, 128, 3]
    CLASSIF_HEAD_NORM = "layer"


def head_by_torch(head, x):
    w1, w2 = (m.weight.flatten(1) for m in (head.mrcnn_class_conv1,
                                            head.mrcnn_class_conv2))
    h = F.relu(F.linear(x.flatten(1), w1, head.mrcnn_class_conv1.bias))
    h = F.layer_norm(h, (64,), head.mrcnn_class_ln1.weight,
                     head.mrcnn_class_ln1.bias, 1e-5)
    h = F.relu(F.linear(h, w2, head.mrcnn_class_conv2.bias)) + h
    h = F.layer_norm(h, (64,), head.mrcnn_class_ln2.weight,
                     head.mrcnn_class_ln2.bias, 1e-5)
    return (F.linear(h, head.mrcnn_class_logits.weight,
                     head.mrcnn_class_logits.bias),
            F.linear(h, head.mrcnn_bbox_fc.weight, head.mrcnn_bbox_fc.bias))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_and_its_gradients(device, dtype):
    """The chain of dense layers and norms beside torch's in 64 bits."""
    torch.manual_seed(0)
    head = FPNClassifierHead(HeadConfig(), in_channels=16).to(device)
    with torch.no_grad():
        for m in (head.mrcnn_class_ln1, head.mrcnn_class_ln2):
            m.weight.uniform_(0.5, 1.5)
            m.bias.uniform_(-0.5, 0.5)
    x = torch.randn(30, 16, 7, 7, device=device, dtype=dtype,
                    requires_grad=True)
    ref = copy.deepcopy(head).double()
    xd = x.detach().double().requires_grad_()
    g1, g2 = (torch.randn(30, n, device=device, dtype=dtype) for n in (5, 20))
    outs = head._dense_layers(x)
    assert all(o.dtype == dtype for o in outs)
    params = [p for p in head.parameters()]
    grads = torch.autograd.grad(outs, [x, *params], (g1, g2))
    douts = head_by_torch(ref, xd)
    dgrads = torch.autograd.grad(douts, [xd, *ref.parameters()],
                                 (g1.double(), g2.double()))
    # Seven roundings to the type on the way to an output and as many back,
    # of relative size eps / 2 each, through layers of gain about 1; values
    # of a tensor are compared in the 2-norm, where they add in quadrature
    # at worst times the 14; in fp32 64 more from the sums.
    tol = torch.finfo(dtype).eps / 2 * (14 if dtype == torch.bfloat16 else 64)
    if dtype == torch.bfloat16:
        # A ReLU whose argument lies within its error of 0 (3 roundings, of
        # values about 1) may go the other way: that share of the gradient's
        # square.
        tol = (tol ** 2 + 6 * torch.finfo(dtype).eps / 2) ** 0.5
    for got, want in zip((*outs, *grads), (*douts, *dgrads)):
        assert (got.double() - want).norm() <= tol * want.norm()


@pytest.mark.gpu
def test_head_under_autocast_and_graph():
    torch.manual_seed(0)
    head = FPNClassifierHead(HeadConfig(), in_channels=16).cuda().eval()
    x = torch.randn(30, 16, 7, 7, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad(), torch.autocast("cuda", torch.bfloat16):
        want = head._dense_layers(x)
        assert want[0].dtype == torch.bfloat16
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = head._dense_layers(x)
        for k in range(3):
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            want = head._dense_layers(x)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_head_refuses_another_norm():
    class Other(HeadConfig):
        CLASSIF_HEAD_NORM = "group"
    with pytest.raises(ValueError):
        FPNClassifierHead(Other(), in_channels=16)


# ------------------------------------------------------------- in training

def test_build_optimizer(shapes_config, tmp_path):
    class Cfg(type(shapes_config)):
        CLASSIF_HEAD_NORM = "layer"
        OPTIMIZER = "adamw8"
    cfg = Cfg()
    m = MaskRCNN("training", cfg, model_dir=str(tmp_path))
    opt = build_optimizer(m.model, cfg, 1e-3)
    assert isinstance(opt, AdamW) and opt.state_bits == 8
    assert opt.max_grad_norm == cfg.GRADIENT_CLIP_NORM
    plain = {id(p) for p in opt.param_groups[1]["params"]}
    head = m.model.classifier_head
    for ln in (head.mrcnn_class_ln1, head.mrcnn_class_ln2):
        assert id(ln.weight) in plain and id(ln.bias) in plain
    cfg.OPTIMIZER = "lion"
    with pytest.raises(ValueError):
        build_optimizer(m.model, cfg, 1e-3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["adamw", "adamw8"])
def test_training_resumes(device, kind, shapes_config, shapes_dataset,
                          tmp_path):
    """A step of training through the new head, saved and resumed; another
    optimizer's state is left alone."""
    class Cfg(type(shapes_config)):
        CLASSIF_HEAD_NORM = "layer"
        OPTIMIZER = kind
    cfg = Cfg()
    m = MaskRCNN("training", cfg, model_dir=str(tmp_path))
    assert m.device.type == device or device == "cpu"
    head = m.model.classifier_head
    before = {n: p.detach().clone() for n, p in head.named_parameters()}
    tr = Trainer(m, shapes_dataset)
    tr.fit(1e-3, epochs=1, layers="heads", steps_per_epoch=2)
    for n, p in head.named_parameters():
        assert p.isfinite().all() and not torch.equal(p, before[n]), n
    m2 = MaskRCNN("training", cfg, model_dir=str(tmp_path))
    m2.load_weights(m2.find_last(), by_name=True)
    tr2 = Trainer(m2, shapes_dataset)
    tr2.fit(1e-3, epochs=2, layers="heads", steps_per_epoch=1)
    assert tr2._resumed_opt

    class Sgd(Cfg):
        OPTIMIZER = "sgd"
    m3 = MaskRCNN("training", Sgd(), model_dir=str(tmp_path))
    m3.load_weights(m3.find_last(), by_name=True)
    tr3 = Trainer(m3, shapes_dataset)
    tr3.fit(1e-3, epochs=m3.epoch + 1, layers="heads", steps_per_epoch=1)
    assert not tr3._resumed_opt


def test_layer_head_detects_and_exports(shapes_config, tmp_path):
    import numpy as np
    from maskrcnn_amd.serving.savedmodel import (
        export_saved_model, load_saved_model,
    )

    class Cfg(type(shapes_config)):
        CLASSIF_HEAD_NORM = "layer"
    m = MaskRCNN("inference", Cfg(), model_dir=str(tmp_path))
    r = m.detect([(np.random.rand(128, 128, 3) * 255).astype(np.uint8)])[0]
    assert r["rois"].shape[1] == 4
    path = export_saved_model(m.model, m.config, str(tmp_path / "export"))
    state, config, _ = load_saved_model(path)
    assert config["CLASSIF_HEAD_NORM"] == "layer"
    assert "classifier_head.mrcnn_class_ln1.weight" in state


def test_keras_map_without_the_heads_batch_norms():
    from maskrcnn_amd.utils.keras_import import keras_weight_map
    full, less = keras_weight_map(), keras_weight_map("resnet101", "layer")
    gone = set(full) - set(less)
    assert gone and all(k.startswith(("mrcnn_class_bn1/", "mrcnn_class_bn2/"))
                        for k in gone)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("beta2", [0.99, 0.999])
@pytest.mark.parametrize("then", [1.0, 0.1, 0.0])
@pytest.mark.parametrize("normal", [True, False])
def test_8_bit_states_follow_over_many_steps(device, beta2, then, normal):
    """3000 steps beside fp32 states, on normal or constant gradients, from
    the middle on `then` times as large.

    v in 8 bits has v's mean. A step that moves it by d between codes D apart
    adds at most |d| D to its variance, with d = (1 - beta2)(g^2 - v) and D at
    most v / 8; the older variance falls by beta2^2. The mean over the values
    is held to six of its deviations.
    """
    n, steps = 2048, 3000
    g = torch.Generator().manual_seed(0)
    bank = torch.randn(500, n, generator=g) if normal else torch.ones(500, n)
    bank = bank.to(device)
    p, q = (nn.Parameter(torch.zeros(n, device=device)) for _ in range(2))
    kw = dict(lr=1e-3, betas=(0.9, beta2), weight_decay=0.0)
    wide, narrow = AdamW([p], **kw), AdamW([q], state_bits=8, **kw)
    var = torch.zeros(n, dtype=torch.float64, device=device)
    moved = [0.0, 0.0]
    for t in range(steps):
        p.grad = q.grad = bank[t % 500] * (1.0 if t < steps // 2 else then)
        if t >= steps - 300:
            was = p.detach().clone(), q.detach().clone()
        if t:
            v = wide.state[p]["exp_avg_sq"].double()
            var = beta2 ** 2 * var + (1 - beta2) / 8 * (
                p.grad.double().square() * v + v * v + var)
        wide.step()
        narrow.step()
        if t >= steps - 300:
            for i, (a, b) in enumerate(zip((p, q), was)):
                moved[i] += float((a.detach() - b).double().square().mean())
    s = narrow.state[q]
    want = wide.state[p]["exp_avg_sq"].double().mean()
    got = unpack_state8(s["exp_avg_sq"], s["exp_avg_sq_scale"],
                        False).double().mean()
    assert abs(got - want) <= 6 * (var.mean() / n).sqrt()
    # Updates: 1 / v of a spread of a quarter to a half has a mean 1.07 to
    # 1.33 times that of none, m's own rounding adds a fifth to its square.
    if then:
        assert 0.95 <= (moved[1] / moved[0]) ** 0.5 <= 1.35


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_state_changes_nothing(device, bits):
    """States of other shapes, one that would broadcast among them, scales
    that are missing or too few, and a state of fewer parameters."""
    def fresh():
        torch.manual_seed(0)
        ps = [nn.Parameter(torch.randn(n, device=device)) for n in (300, 91)]
        opt = AdamW(ps, lr=1e-2, state_bits=bits)
        for p in ps:
            p.grad = torch.ones_like(p)
        opt.step()
        return ps, opt

    def saved(**more):
        state = copy.deepcopy(fresh()[1].state_dict())
        state["param_groups"][0]["lr"] = 5.0
        state["state"][1].update(more)
        return state
    dtype = torch.float32 if bits == 32 else torch.uint8
    bad = [saved(**{name: torch.ones(n, dtype=dtype)})
           for name in ("exp_avg", "exp_avg_sq") for n in (1, 81, (91, 1))]
    bad.append(saved(exp_avg_sq=torch.ones(91, dtype=torch.bfloat16)))
    if bits == 8:
        bad += [saved(exp_avg_scale=torch.ones(2, dtype=dtype)),
                saved(exp_avg_sq_scale=torch.ones(1)),
                saved(exp_avg=torch.ones(182, dtype=dtype)[::2])]
    for name in ("step", "exp_avg_sq") + (("exp_avg_scale",) * (bits == 8)):
        bad.append(saved())
        del bad[-1]["state"][1][name]
    bad.append(saved())
    bad[-1]["param_groups"][0]["params"] = [0]
    want, same = fresh()
    same.step()
    for state in bad:
        ps, opt = fresh()
        with pytest.raises(ValueError):
            opt.load_state_dict(state)
        opt.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, want))
        for p, q in zip(ps, want):
            assert all(torch.equal(torch.as_tensor(v),
                                   torch.as_tensor(same.state[q][k]))
                       for k, v in opt.state[p].items())
    ps, opt = fresh()
    opt.load_state_dict(saved())
    opt.step()


def test_configurations_without_the_new_fields(shapes_config):
    """A class of the caller's own: the batch-normed head and SGD."""
    class Old:
        POOL_SIZE, FPN_CLASSIF_FC_LAYERS_SIZE, NUM_CLASSES = 7, 64, 5
        TRAIN_BN, IMAGE_SHAPE = False, [128, 128, 3]
        WEIGHT_DECAY, LEARNING_MOMENTUM = 1e-4, 0.9
    head = FPNClassifierHead(Old(), in_channels=16)
    assert not head.layer_norm and hasattr(head, "mrcnn_class_bn1")
    opt = build_optimizer(head, Old(), 1e-3)
    assert isinstance(opt, torch.optim.SGD)
