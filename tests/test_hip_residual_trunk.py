"""Layer norm, the linear layer and Muon together, as a model and its trainer use them: models.fields.ResidualLayer / IndirectLight(residual=True)
and fneus.optim.FlatMuon against the same network and the same optimiser in float64, the stage-2 / 3 trainers with optimizer="muon".

Tolerances.  Gradients of the five-layer trunk in fp32: each layer adds about sqrt(512) 2^-24 = 1.3e-6 of its scale, ten products deep: 1e-4 of a
tensor's largest value is the bound (a ReLU whose pre-activation lies within that of 0 would break it: the inputs are smooth activations).
A Muon step in the float64 reference starts from the kernels' own gradients, so that the optimiser alone is compared: 1e-5 of the update
(test_hip_muon.py), Adam 1e-5."""
import os
import sys

import pytest
import torch
import torch.nn as nn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "factored-neus_amd"))
sys.path.insert(0, os.path.join(ROOT, "tests"))


def trunk(width=64, n_in=39, n_out=36, act="silu", seed=0):
    from models.fields import ActLinear, ResidualLayer
    torch.manual_seed(seed)
    net = nn.Sequential(ActLinear(n_in, width, act), *(ResidualLayer(width, act) for _ in range(3)), ActLinear(width, n_out))
    with torch.no_grad():
        for m in net:
            if hasattr(m, "norm_weight"):
                m.norm_weight.add_(0.2 * torch.randn(width))
                m.norm_bias.add_(0.2 * torch.randn(width))
    return net


@pytest.mark.gpu
@pytest.mark.parametrize("width,rows", [(64, 5), (64, 300), (512, 512), (256, 4096)])
def test_trunk_against_float64(width, rows):
    net = trunk(width)
    ref = trunk(width).double()                       # (on the CPU the modules run torch's own operators)
    g = torch.Generator().manual_seed(3)
    x, cot = torch.randn(rows, 39, generator=g), torch.randn(rows, 36, generator=g)
    xr = x.double().requires_grad_(True)
    yr = ref(xr)
    (yr * cot.double()).sum().backward()
    net = net.cuda()
    xg = x.cuda().requires_grad_(True)
    y = net(xg)
    (y * cot.cuda()).sum().backward()
    for got, want, name in [(y, yr, "y"), (xg.grad, xr.grad, "dx")] + [(p.grad, q.grad, n) for (n, p), q in zip(net.named_parameters(), ref.parameters())]:
        err = float((got.detach().double().cpu() - want.detach()).abs().max()) / float(want.detach().abs().max())
        assert err <= 1e-4, (name, err)


@pytest.mark.gpu
def test_trunk_shapes_frozen_and_partial_gradients():
    from fneus import autograd
    net = trunk().cuda()
    x = torch.randn(4, 3, 39, device="cuda")
    y = net(x)
    assert y.shape == (4, 3, 36) and torch.equal(y.reshape(12, 36), net(x.reshape(12, 39)))
    assert net(x[:0]).shape == (0, 3, 36)
    net(x[:0]).sum().backward()
    assert all(float(p.grad.abs().max()) == 0.0 for n, p in net.named_parameters() if "norm" not in n)
    for p in net.parameters():
        p.requires_grad_(False)
        p.grad = None
    assert not net(x).requires_grad
    xg = x.clone().requires_grad_(True)
    net(xg).sum().backward()
    full = xg.grad.clone()
    assert all(p.grad is None for p in net.parameters())
    net[2].weight.requires_grad_(True)
    xg.grad = None
    net(xg).sum().backward()
    assert torch.equal(xg.grad, full) and net[2].weight.grad is not None and net[2].bias.grad is None
    with pytest.raises(ValueError):
        autograd.linear(x, torch.randn(5, 39, device="cuda"), residual=torch.randn(5, device="cuda"))
    w, b = torch.ones(39, device="cuda"), torch.zeros(39, device="cuda", requires_grad=True)
    for args in ((None, None), (w, None), (None, b), (w.requires_grad_(True), b)):
        xg = x.clone().requires_grad_(True)
        autograd.layer_norm(xg, *args).square().sum().backward()
        xr = x.detach().clone().requires_grad_(True)
        nn.functional.layer_norm(xr, (39,), *[None if a is None else a.detach() for a in args]).square().sum().backward()
        assert float((xg.grad - xr.grad).abs().max()) <= 2e-5
    # gradients of gradients are refused, not wrong
    xg = x.clone().requires_grad_(True)
    (gx,) = torch.autograd.grad(autograd.layer_norm(xg, w).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_trunk_sixteen_bits(t):
    """16-bit modules: forward and gradients within a few roundings (a half step each, 12 in a row, doubled) of float64 at the same weights"""
    net = trunk(128).to(t)
    ref = trunk(128).to(t).double()
    x, cot = torch.randn(200, 39).to(t), torch.randn(200, 36).to(t)
    yr = ref(x.double())
    (yr * cot.double()).sum().backward()
    net = net.cuda()
    y = net(x.cuda())
    (y * cot.cuda()).sum().backward()
    lim = 24 * torch.finfo(t).eps / 2
    for got, want, name in [(y, yr, "y")] + [(p.grad, q.grad, n) for (n, p), q in zip(net.named_parameters(), ref.parameters())]:
        err = float((got.detach().double().cpu() - want.detach()).norm() / want.detach().norm())
        assert err <= lim, (name, err)


def muon64(p, g, m, lr, mu=0.95):
    from test_hip_muon import ns64
    m = mu * m + (1 - mu) * g
    return p - lr * 0.2 * max(p.shape) ** 0.5 * ns64((1 - mu) * g + mu * m), m


@pytest.mark.gpu
def test_flat_muon_steps_against_float64():
    from fneus.optim import FlatMuon
    net = trunk().cuda()
    opt = FlatMuon(net.parameters(), lr=3e-3)
    names = {p: n for n, p in net.named_parameters()}
    assert [names[p] for p in opt.matrices] == ["0.weight", "1.weight", "2.weight", "3.weight", "4.weight"]
    for p in net.parameters():
        p.grad = torch.zeros_like(p)
    x, cot = torch.randn(80, 39, device="cuda"), torch.randn(80, 36, device="cuda")
    mom = {p: torch.zeros_like(p, dtype=torch.float64) for p in opt.matrices}
    adam = {p: (torch.zeros_like(p, dtype=torch.float64), torch.zeros_like(p, dtype=torch.float64)) for p in net.parameters() if p not in mom}
    for step in range(1, 4):
        lr = 3e-3 / step
        opt.set_lr(lr)
        (net(x) * cot).sum().backward()
        before = {p: (p.detach().double().clone(), p.grad.double().clone()) for p in net.parameters()}
        opt.step()
        for p, (old, g) in before.items():
            assert float(p.grad.abs().max()) == 0.0                          # cleared by the kernels
            if p in mom:
                want, m = muon64(old.cpu(), g.cpu(), mom[p].cpu(), lr)
                mom[p] = m.cuda()
                want = want.cuda()
            else:
                m, v = adam[p]
                m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
                adam[p] = (m, v)
                want = old - lr * (m / (1 - 0.9 ** step)) / ((v / (1 - 0.999 ** step)).sqrt() + 1e-8)
            moved, err = float((want - old).norm()), float((p.detach().double() - want).norm())
            assert err <= 2e-5 * moved + 2.0 ** -23 * float(want.norm()), (names[p], step, err, moved)


@pytest.mark.gpu
def test_flat_muon_state_dict_and_graph():
    """a run that is saved, loaded into a fresh optimiser and continued equals the run that went on; a captured step equals the eager one"""
    import io
    from fneus.optim import FlatMuon
    x, cot = torch.randn(80, 39, device="cuda"), torch.randn(80, 36, device="cuda")

    def make():
        net = trunk().cuda()
        for p in net.parameters():
            p.grad = torch.zeros_like(p)
        return net, FlatMuon(net.parameters(), lr=2e-3)

    def step(net, opt):
        (net(x) * cot).sum().backward()
        opt.step()

    a, oa = make()
    for _ in range(2):
        step(a, oa)
    buf = io.BytesIO()
    torch.save({"net": a.state_dict(), "opt": oa.state_dict()}, buf)
    buf.seek(0)
    ck = torch.load(buf, map_location="cuda")
    b, ob = make()
    b.load_state_dict(ck["net"])
    ob.load_state_dict(ck["opt"])
    for _ in range(2):
        step(a, oa), step(b, ob)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    with pytest.raises(ValueError):
        ob.load_state_dict({"state": {0: {"exp_avg": torch.zeros(64, 39)}}, "param_groups": ck["opt"]["param_groups"]})
    # capture on b, eager on a
    import gc
    gc.collect()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b, ob)
    torch.cuda.current_stream().wait_stream(side)
    step(a, oa)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, ob)
    for k in range(3):
        oa.set_lr(1e-3 / (k + 1)), ob.set_lr(1e-3 / (k + 1))
        x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        step(a, oa)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters())), k


@pytest.mark.gpu
def test_flat_muon_skips_and_follows():
    """a parameter without a gradient is left alone; re-attached gradients and an assigned learning rate are followed"""
    from fneus.optim import FlatMuon
    p, q, r = (nn.Parameter(torch.randn(40, 50, device="cuda")) for _ in range(3))
    opt = FlatMuon([p, q, r], lr=1e-2)
    opt.step()                                                        # no gradient at all: nothing to do
    p.grad, q.grad = torch.randn_like(p), torch.randn_like(q)
    keep = r.detach().clone()
    old = p.detach().clone()
    opt.step()
    assert torch.equal(r, keep) and not torch.equal(p, old)
    opt.param_groups[0]["lr"] = 0.0
    p.grad = torch.randn_like(p)                                      # another buffer
    old = p.detach().clone()
    opt.step()
    assert torch.equal(p, old) and float(p.grad.abs().max()) == 0.0


def test_flat_muon_refusals_cpu():
    from fneus.optim import FlatMuon
    p = nn.Parameter(torch.randn(40, 50))
    for bad in (dict(momentum=1.0), dict(steps=0), dict(eps=0.0), dict(adjust="other"), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            FlatMuon([p], **bad)
    with pytest.raises(NotImplementedError):
        FlatMuon([{"params": [p]}, {"params": [nn.Parameter(torch.randn(3))]}])
    opt = FlatMuon([p, nn.Parameter(torch.randn(3)), nn.Parameter(torch.randn(50, 4))])
    assert opt.matrices == [p] and len(opt.adam.param_groups[0]["params"]) == 2
    p.grad = torch.randn_like(p)
    with pytest.raises(ValueError):
        opt.step()                                                    # no CPU fallback
    with pytest.raises(NotImplementedError):
        opt.step(lambda: None)
    opt.add_param_group({"params": [nn.Parameter(torch.randn(40, 40))]})
    with pytest.raises(NotImplementedError):
        opt.step()


def test_indirect_light_residual_cpu():
    from models.fields import IndirectLight, _mlp_spec
    net = IndirectLight(residual=True)
    assert _mlp_spec(net.indi) is None and _mlp_spec(IndirectLight().indi) is not None
    out = net(torch.randn(6, 3))
    assert out.shape == (6, 24, 7)
    out.sum().backward()
    assert all(p.grad is not None for p in net.parameters())
    assert sorted({k.rsplit(".", 1)[0] for k in net.state_dict()}) == ["indi.0", "indi.1", "indi.2", "indi.3", "indi.4"]


def test_conf_selects_muon_and_residual():
    from fneus import hocon
    text = open(os.path.join(ROOT, "factored-neus_amd", "confs", "wmask.conf")).read()
    conf = hocon.parse_string(text.replace("train {", "train {\n    optimizer = muon", 1).replace("model {", "model {\n    indirect_light { residual = True }", 1))
    assert conf["train"].get_string("optimizer", "adam") == "muon" and dict(conf["model"]["indirect_light"]) == {"residual": True}
    conf = hocon.parse_string(text)
    assert conf["train"].get_string("optimizer", "adam") == "adam" and "indirect_light" not in conf["model"]


@pytest.mark.gpu
@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("stage", [2, 3])
def test_stage_trainers_with_muon_and_residual_trunk(stage, use_graph):
    from fneus import synth
    from fneus.trainer import WMASK_MODEL
    from fneus.trainer2 import LVIS_RENDERER, Stage2Trainer
    from fneus.trainer3 import Stage3Trainer
    dev = torch.device("cuda:0")
    conf = dict(WMASK_MODEL, indirect_light=dict(residual=True))
    small = dict(n_samples=16, n_importance=16, n_outside=0, up_sample_steps=4, perturb=1.0)
    if stage == 2:
        tr = Stage2Trainer(dev, model_conf=dict(conf, lvis_renderer=dict(LVIS_RENDERER, **small)), seed=5, use_graph=use_graph, optimizer="muon")
    else:
        tr = Stage3Trainer(dev, model_conf=dict(conf, neus_renderer=small), seed=5, use_graph=use_graph, optimizer="muon")
    data = torch.from_numpy(synth.ray_batch(32, seed=5, n_miss=2)).to(dev)
    before = [p.detach().clone() for p in tr.params]
    for _ in range(5):
        out = tr.train_step(data)
        assert out is not None and bool(torch.isfinite(out["loss"]))
    assert tr.graph_error is None
    moved = [not torch.equal(p, q) for p, q in zip(tr.params, before)]
    assert len(tr.optimizer.matrices) > 0 and sum(moved) >= 0.9 * len(moved)
    assert all(bool(torch.isfinite(p).all()) for p in tr.params)
    sd = tr.optimizer_state_dict()
    tr.load_optimizer_state_dict(sd)
    tr.set_lr(1e-4)
    assert tr.get_lr() == 1e-4
    assert tr.train_step(data) is not None
    with pytest.raises(ValueError):
        (Stage2Trainer if stage == 2 else Stage3Trainer)(dev, optimizer="sgd")


def _stepped_adam_state(opt, value):
    """what FlatAdam's step leaves for its parameters, without a GPU"""
    for p in opt.adam.param_groups[0]["params"]:
        opt.adam.state[p] = {"step": torch.tensor(float(value)), "exp_avg": torch.full_like(p, value), "exp_avg_sq": torch.full_like(p, value)}


def test_flat_muon_load_replaces_adam_state_cpu():
    """a loaded state takes the place of all that the optimiser had: what it does not hold (a fresh optimiser's, a parameter that had no
    gradient) starts anew, for Adam's parameters too"""
    from fneus.optim import FlatMuon
    make = lambda: FlatMuon([nn.Parameter(torch.zeros(40, 50)), nn.Parameter(torch.zeros(3)), nn.Parameter(torch.zeros(5))])  # noqa: E731
    a = make()
    w, b, c = a.param_groups[0]["params"]
    _stepped_adam_state(a, 100.0)
    a.state[w] = {"momentum_buffer": torch.ones(40, 50)}
    a.adam._segs = object()
    a.load_state_dict(make().state_dict())                            # an empty state
    assert len(a.state.get(w, {})) == len(a.adam.state.get(b, {})) == len(a.adam.state.get(c, {})) == 0 and a.adam._segs is None
    assert not a.state_dict()["state"]
    partial = make()
    _stepped_adam_state(partial, 7.0)
    del partial.adam.state[partial.param_groups[0]["params"][2]]      # one of the two has no state
    sd = partial.state_dict()
    _stepped_adam_state(a, 100.0)
    a.load_state_dict(sd)
    assert float(a.adam.state[b]["step"]) == 7.0 and float(a.adam.state[b]["exp_avg"][0]) == 7.0 and len(a.adam.state.get(c, {})) == 0
    assert sorted(a.state_dict()["state"]) == [1]


def test_flat_muon_table_follows_what_it_was_built_from_cpu(monkeypatch):
    """the table of jobs is built anew where something it holds has changed at the same addresses: adjust, a matrix's shape, a gradient's layout"""
    from fneus import ops
    from fneus.optim import FlatMuon
    built = []
    monkeypatch.setattr(ops, "muon_jobs", lambda ps, gs, ms, adjust: built.append((adjust, [tuple(p.shape) for p in ps], [g.stride() for g in gs])))
    monkeypatch.setattr(ops, "muon_launch", lambda *a: None)
    p = nn.Parameter(torch.zeros(40, 40))
    p.grad = torch.ones(40, 40)
    opt = FlatMuon([p], lr=1e-2)
    opt.step(), opt.step()
    assert len(built) == 1
    opt.param_groups[0]["adjust"] = "original"
    opt.step(), opt.step()
    assert len(built) == 2 and built[-1][0] == "original"
    p.grad.t_()                                                       # the same memory, transposed
    opt.step()
    assert len(built) == 3 and built[-1][2] == [(1, 40)]
    with torch.no_grad():
        p.grad = None
        m = opt.state[p]["momentum_buffer"]
        g = torch.ones(1600)
        p.grad = g.view(40, 40)
        opt.step()
        p.grad = None
        p.data, opt.state[p]["momentum_buffer"] = p.data.view(50, 32), m.view(50, 32)
        p.grad = g.view(50, 32)
    opt.step()
    assert built[-1][1] == [(50, 32)]


@pytest.mark.gpu
def test_flat_muon_adjust_between_steps():
    """the factor on the learning rate, assigned between steps, is the one the next step takes"""
    from fneus.optim import FlatMuon
    p = nn.Parameter(torch.zeros(64, 100, device="cuda"))
    grad = torch.randn(64, 100, device="cuda")
    moved = []
    opt = FlatMuon([p], lr=1e-2, adjust=1.0, momentum=0.0)
    p.grad = torch.zeros_like(p)
    for adjust in (1.0, 3.0):
        opt.param_groups[0]["adjust"] = adjust
        with torch.no_grad():
            p.zero_(), p.grad.copy_(grad)
        opt.step()
        moved.append(p.detach().double().clone())
    # the same orthogonalised gradient, times lr adjust: one fp32 product and one difference from 0 each (2^-24 both), lr adjust itself 2^-24
    assert float((moved[1] - 3.0 * moved[0]).abs().max()) <= 4 * 2.0 ** -24 * float(moved[1].abs().max())


def test_flat_muon_refuses_its_first_step_in_a_capture_cpu(monkeypatch):
    """buffers cleared, or a learning rate written, inside a captured step would be so again in every replay: the state has to be there before"""
    from fneus import ops, optim
    from fneus.optim import FlatMuon
    launched = []
    monkeypatch.setattr(ops, "muon_jobs", lambda *a: None)
    monkeypatch.setattr(ops, "muon_launch", lambda *a: launched.append(a))
    capturing = [True]
    monkeypatch.setattr(optim, "_capturing", lambda device: capturing[0])
    p, v = nn.Parameter(torch.zeros(40, 40)), nn.Parameter(torch.zeros(5))
    p.grad, v.grad = torch.ones(40, 40), torch.ones(5)
    opt = FlatMuon([p], lr=1e-2)
    with pytest.raises(RuntimeError, match="eager step"):
        opt.step()
    assert not launched and not opt.state[p]
    capturing[0] = False
    opt.step()
    capturing[0] = True
    opt.step()
    p.grad = torch.ones(40, 40)                                       # (another gradient: host work alone)
    opt.step()
    assert len(launched) == 3
    opt.param_groups[0]["lr"] = 0.5                                   # (would be written by the captured step, in every replay)
    with pytest.raises(RuntimeError, match="set_lr"):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-2
    opt.load_state_dict(FlatMuon([nn.Parameter(torch.zeros(40, 40))], lr=1e-2).state_dict())
    with pytest.raises(RuntimeError, match="eager step"):
        opt.step()
    both = FlatMuon([p, v], lr=1e-2)                                  # Adam's parameters alone are stale
    both.state[p]["momentum_buffer"], both._lr_dev, both._lr_host = torch.zeros(40, 40), torch.zeros(()), 1e-2
    with pytest.raises(RuntimeError, match="eager step"):
        both.step()


@pytest.mark.gpu
def test_flat_muon_refuses_its_first_step_in_a_capture():
    from fneus.optim import FlatMuon
    p = nn.Parameter(torch.randn(40, 50, device="cuda"))
    p.grad = torch.randn_like(p)
    old = p.detach().clone()
    opt = FlatMuon([p], lr=1e-2)
    graph, other = torch.cuda.CUDAGraph(), torch.zeros(8, device="cuda")
    with torch.cuda.graph(graph):
        other.add_(1.0)
        with pytest.raises(RuntimeError, match="eager step"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert float(other[0]) == 1.0 and torch.equal(p, old) and not opt.state[p]
    opt.step()
    assert not torch.equal(p, old)


@pytest.mark.gpu
def test_optimizers_launch_on_the_device_of_their_parameters(monkeypatch):
    """another device is current when step() is called: the launch is made with the parameters' device current, on that device's stream (here the
    runtime is made to say that device 1 is current until somebody selects device 0)"""
    from fneus.optim import FlatAdam, FlatMuon
    p = nn.Parameter(torch.randn(7, device="cuda:0"))
    p.grad = torch.ones_like(p)
    entered = []

    class select(torch.cuda.device):
        def __enter__(self):
            entered.append(self.idx)
            return super().__enter__()

    for opt in (FlatAdam([p], lr=1e-2), FlatMuon([p], lr=1e-2)):
        start = p.detach().clone()
        p.grad.fill_(1.0)
        del entered[:]
        with monkeypatch.context() as m:
            m.setattr(torch.cuda, "current_device", lambda: entered[-1] if entered else 1)
            m.setattr(torch.cuda, "device", select)
            opt.step()
        assert entered and set(entered) == {0}
        assert float((p.detach() - start).abs().min()) > 0.0
