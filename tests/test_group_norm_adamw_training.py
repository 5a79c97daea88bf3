"""Group norm and AdamW where they are used: models, engines, the trainer."""

import glob
import os

import pytest
import torch

from eventgrad_amd.config import DataConfig, OptimConfig, RunConfig, preset
from eventgrad_amd.models import BatchNorm2d, GroupNorm2d, build_model
from eventgrad_amd.ops import functional as O
from eventgrad_amd.parallel import AdamW, FlatParamSpace
from eventgrad_amd.parallel.engine import SerialEngine, _build_adamw

import optim_workers as W
from util_dist import run_world


def adamw(bits=32, **kw):
    return OptimConfig(lr=2e-3, optimizer="adamw", weight_decay=0.01,
                       state_bits=bits, **kw)


def serial_cfg(tmp_path=None, device="cpu", model="mlp", epochs=1, bits=8,
               **kw):
    mnist = model in ("mlp", "cnn2")
    return RunConfig(
        mode="serial", model=model, epochs=epochs, device=device,
        optim=adamw(bits), eval_at_end=False, final_consensus=False,
        data=DataConfig(dataset="synthetic-mnist" if mnist else "synthetic",
                        batch_size=16, synthetic_train_samples=64,
                        synthetic_test_samples=16),
        checkpoint_path=(os.path.join(tmp_path, "ck.pt") if tmp_path
                         else None), **kw)


# ---------------------------------------------------------------- settings

def test_flags_reach_the_config():
    from eventgrad_amd.train.cli import build_parser, config_from_args
    args = build_parser().parse_args(
        ["--preset", "dcifar10-event", "--optimizer", "adamw",
         "--state-bits", "8", "--weight-decay", "0.05", "--norm", "group",
         "--norm-groups", "16"])
    cfg = config_from_args(args)
    assert (cfg.optim.optimizer, cfg.optim.state_bits) == ("adamw", 8)
    assert cfg.optim.weight_decay == 0.05
    assert (cfg.norm, cfg.norm_groups) == ("group", 16)
    assert RunConfig.from_json(cfg.to_json()) == cfg
    # and without them a preset is what it was
    cfg = config_from_args(build_parser().parse_args(
        ["--preset", "dcifar10-event"]))
    assert cfg == preset("dcifar10-event")
    assert (cfg.optim.optimizer, cfg.norm) == ("sgd", "batch")


def test_engine_takes_its_optimizer():
    space = FlatParamSpace(build_model("cnn2"), torch.device("cpu"))
    cfg = RunConfig(optim=OptimConfig())
    assert _build_adamw(space, cfg) is None
    cfg.optim = adamw(8, beta2=0.95, decay_1d=False)
    opt = _build_adamw(space, cfg)
    assert isinstance(opt, AdamW) and opt.state_bits == 8
    assert opt.betas == (0.9, 0.95) and not opt.decay_1d
    cfg.optim.optimizer = "adam"
    with pytest.raises(ValueError):
        _build_adamw(space, cfg)


def test_engine_step_follows_lr_and_gives_norms():
    space = FlatParamSpace(build_model("cnn2"), torch.device("cpu"),
                           momentum=False)
    cfg = RunConfig(mode="serial", optim=adamw())
    eng = SerialEngine(space, cfg, 0, 1, torch.device("cpu"))
    space.grad.normal_()
    eng.step()
    norms = [float(p.square().sum()) for p in
             (space.seg(space.param, i) for i in range(space.sz))]
    assert torch.allclose(eng._last_norms_sq, torch.tensor(norms), rtol=1e-5)
    before = space.param.clone()
    cfg.optim.lr = 0.0
    eng.step()
    assert eng.opt.lr == 0.0
    assert torch.equal(space.param, before)


def test_models_take_the_norm():
    for norm, kind in (("batch", BatchNorm2d), ("group", GroupNorm2d)):
        m = build_model("resnet20", norm=norm)
        assert sum(isinstance(k, kind) for k in m.modules()) == 21


# ---------------------------------------------------------------- CPU runs

@pytest.mark.parametrize("mode,model,norm,bits", [
    ("event", "cnn2", "batch", 8), ("spevent", "cnn2", "batch", 32),
    ("decent", "resnet20", "group", 8), ("cent", "cnn2", "batch", 8)])
def test_two_ranks_twice(tmp_path, mode, model, norm, bits):
    """Two ranks end with one model, and a second run is the first to the
    bit, events and all."""
    run_world(W.adamw_twice_worker, 2, str(tmp_path), mode, model, norm, bits)
    outs = [torch.load(f, weights_only=False)["runs"]
            for f in sorted(glob.glob(os.path.join(tmp_path, "adamw_r*.pt")))]
    assert len(outs) == 2
    for runs in outs:
        (p1, e1, s1), (p2, e2, s2) = runs
        assert torch.isfinite(p1).all()
        assert torch.equal(p1, p2) and e1 == e2
        assert s1 == s2 > 0
    assert torch.allclose(outs[0][0][0], outs[1][0][0], atol=1e-6)


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_resumes(tmp_path, device, bits):
    """One epoch, a checkpoint and one more are two epochs: to the bit on the
    CPU; on the GPU the weight gradients' atomics leave the order open."""
    from eventgrad_amd.train.trainer import Trainer
    straight = Trainer(serial_cfg(device=device, epochs=2, bits=bits))
    straight.train()
    Trainer(serial_cfg(tmp_path, device, epochs=1, bits=bits)).train()
    tr = Trainer(serial_cfg(tmp_path, device, epochs=2, bits=bits,
                            resume=True))
    assert tr.engine.opt.steps == 4
    tr.train()
    assert tr.engine.opt.steps == 8
    if device == "cpu":
        assert torch.equal(tr.space.param, straight.space.param)
        assert all(torch.equal(a, b) for a, b in zip(
            tr.engine.opt.moments(), straight.engine.opt.moments()))
    else:
        assert torch.isfinite(tr.space.param).all()


def test_checkpoint_of_the_other_optimizer_is_refused(tmp_path):
    from eventgrad_amd.train.trainer import Trainer
    Trainer(serial_cfg(tmp_path)).train()
    for change in (dict(optimizer="sgd"), dict(state_bits=32)):
        cfg = serial_cfg(tmp_path, resume=True, epochs=2)
        for k, v in change.items():
            setattr(cfg.optim, k, v)
        with pytest.raises(ValueError):
            Trainer(cfg)


# ---------------------------------------------------------------- GPU runs

@pytest.mark.gpu
@pytest.mark.parametrize("name", ["resnet20", "resnet18q"])
def test_gpu_direct_gradients_equal_autograds(name):
    """The gradients that the kernels add into the flat space against those
    of a model without one. Group norm's forward does not depend on the order
    of anything, so the whole pass is the same but for the fp32 atomics of
    the weight gradients."""
    dev = torch.device("cuda")
    models = []
    for _ in range(2):
        torch.manual_seed(5)
        models.append(build_model(name, norm="group").to(dev).train())
    alone, flat = models
    space = FlatParamSpace(flat, dev)
    torch.manual_seed(6)
    x = torch.randn(16, 3, 32, 32, device=dev)
    y = torch.randint(0, 10, (16,), device=dev)
    space.zero_grad()
    losses = []
    for m in models:
        loss = O.nll_of_logits(m(x), y)
        loss.backward()
        losses.append(loss.detach())
    torch.cuda.synchronize()
    assert torch.equal(*losses)
    for (k, p), q in zip(alone.named_parameters(), flat.parameters()):
        err = (p.grad - q.grad).norm() / (p.grad.norm() + 1e-12)
        assert float(err) < 1e-4, (k, float(err))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_gpu_training_step_captured(bits):
    """The trainer's step: forward and backward in a graph, AdamW behind it,
    with eager work between. Every replay's loss is the eager pass's."""
    from eventgrad_amd.train.graphstep import FwdBwdGraph
    dev = torch.device("cuda")
    torch.manual_seed(0)
    model = build_model("resnet20", norm="group").to(dev).train()
    space = FlatParamSpace(model, dev, momentum=False)
    eng = SerialEngine(space, RunConfig(mode="serial", optim=adamw(bits)),
                       0, 1, dev)
    graph = FwdBwdGraph(model, space, (8, 3, 32, 32), dev)
    g = torch.Generator().manual_seed(1)
    for t in range(4):
        x = torch.randn(8, 3, 32, 32, generator=g).to(dev)
        y = torch.randint(0, 10, (8,), generator=g).to(dev)
        _, loss = graph.step(x, y)
        got, grads = float(loss.detach()), space.grad.clone()
        assert graph._graph is not False
        space.zero_grad()
        want = O.nll_of_logits(model(x), y)
        want.backward()
        torch.cuda.synchronize()
        assert got == float(want.detach())
        err = (grads - space.grad).norm() / space.grad.norm()
        assert float(err) < 1e-4
        before = space.param.clone()
        eng.step()
        assert torch.isfinite(space.param).all()
        assert not torch.equal(space.param, before)
    assert eng.opt.steps == 4


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["event", "spevent"])
def test_gpu_gossip_with_adamw(mode):
    """The gossip engine on the GPU, both neighbours this rank itself."""
    from eventgrad_amd.config import TriggerConfig
    from eventgrad_amd.parallel.engine import (GossipEngine,
                                               SparseGossipEngine)
    from test_gpu_engine import LoopbackTransport
    dev = torch.device("cuda")
    torch.manual_seed(0)
    model = build_model("resnet20", norm="group").to(dev).train()
    space = FlatParamSpace(model, dev, momentum=False)
    cfg = RunConfig(mode=mode, optim=adamw(8),
                    trigger=TriggerConfig(adaptive=True, horizon=1.05,
                                          initial_comm_passes=3))
    cfg.topk_percent = 10.0
    kind = SparseGossipEngine if mode == "spevent" else GossipEngine
    eng = kind(space, cfg, rank=0, world=2, device=dev)
    eng.transport = LoopbackTransport()
    x = torch.randn(8, 3, 32, 32, device=dev)
    y = torch.randint(0, 10, (8,), device=dev)
    for p in range(1, 9):
        eng.begin_pass(p)
        space.zero_grad()
        O.nll_of_logits(model(x), y).backward()
        eng.after_backward()
        eng.step()
        norms = torch.stack([space.seg(space.param, i).square().sum()
                             for i in range(space.sz)])
        assert torch.allclose(eng._last_norms_sq, norms, rtol=1e-5)
    assert torch.isfinite(space.param).all()
    assert eng.num_events >= 2 * space.sz * 2


@pytest.mark.gpu
def test_gpu_trainer_runs():
    from eventgrad_amd.train.trainer import Trainer
    tr = Trainer(serial_cfg(device="cuda", model="resnet20", epochs=2,
                            norm="group"))
    m = tr.train()
    assert tr.engine.opt.steps == 8 == m.total_passes
    assert torch.isfinite(tr.space.param).all()
    tr.evaluate()


def test_checkpoint_of_another_norm_is_refused(tmp_path):
    """The parameters have the same names and shapes under every norm, so
    that nothing but the norm itself tells them apart. A refused file leaves
    the model as it was."""
    from eventgrad_amd.train.checkpoint import load_checkpoint, save_checkpoint
    from eventgrad_amd.train.trainer import Trainer

    def trainer(norm, groups=8, bits=32):
        return Trainer(serial_cfg(tmp_path, model="resnet20", norm=norm,
                                  norm_groups=groups, bits=bits))

    def load(tr, path):
        return load_checkpoint(path, tr.space, tr.engine, tr.device,
                               model=tr.model)

    kinds = {"batch": trainer("batch"), "group8": trainer("group"),
             "group4": trainer("group", 4)}
    for k, tr in kinds.items():
        tr.space.param.normal_()
        tr.engine.opt.exp_avg.normal_()
        save_checkpoint(str(tmp_path / k), tr.cfg, 1, 4, tr.space, tr.engine,
                        model=tr.model)
    for k, tr in kinds.items():
        for other in kinds:
            before = tr.space.param.clone(), tr.engine.opt.exp_avg.clone()
            if other == k:
                assert load(tr, str(tmp_path / k))["pass_num"] == 4
                continue
            with pytest.raises(ValueError, match="norm"):
                load(tr, str(tmp_path / other))
            assert torch.equal(tr.space.param, before[0])
            assert torch.equal(tr.engine.opt.exp_avg, before[1])
    # a file from before there was a choice holds a batch-norm model
    old = torch.load(tmp_path / "batch", weights_only=False)
    del old["config"]["norm"], old["config"]["norm_groups"]
    torch.save(old, tmp_path / "old")
    load(kinds["batch"], str(tmp_path / "old"))
    with pytest.raises(ValueError, match="norm"):
        load(kinds["group8"], str(tmp_path / "old"))
    # and a model whose buffers are not the file's is another one
    del old["buffers"]["bn.running_mean"]
    torch.save(old, tmp_path / "less")
    with pytest.raises(ValueError, match="bn.running_mean"):
        load(kinds["batch"], str(tmp_path / "less"))


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("decay_1d", [True, False])
def test_engine_step_follows_weight_decay(device, decay_1d):
    """As SGD's step does: with gradients of zero a step is the decay alone,
    the one that the settings hold when it is taken."""
    dev = torch.device(device)
    space = FlatParamSpace(build_model("cnn2").to(dev), dev, momentum=False)
    cfg = RunConfig(mode="serial", optim=adamw(decay_1d=decay_1d))
    eng = SerialEngine(space, cfg, 0, 1, dev)
    for wd in (0.01, 0.5, 0.0):
        cfg.optim.weight_decay = wd
        before = space.param.clone()
        eng.step()
        assert eng.opt.weight_decay == wd
        for i, shape in enumerate(space.shapes):
            d = wd if decay_1d or len(shape) > 1 else 0.0
            got, was = (space.seg(t, i) for t in (space.param, before))
            # 1 - lr wd and the product round, or lr wd and the fused sum
            assert torch.allclose(got, was * (1 - cfg.optim.lr * d),
                                  rtol=2.0 ** -22, atol=0)
    with pytest.raises(ValueError):
        eng.opt.weight_decay = -1.0


def test_preflight_runs_what_the_flags_ask_for(monkeypatch):
    """bench.py's smoke run of every mode, up to its first engine."""
    import types
    import bench
    seen = {}

    class Built(Exception):
        pass

    def model(name, **kw):
        seen["norm"] = kw.get("norm", "batch")
        return build_model("cnn2")

    def engine(space, cfg, *rest):
        seen["optim"], seen["space"] = cfg.optim, space
        raise Built

    monkeypatch.setattr(bench, "build_model", model)
    monkeypatch.setattr(bench, "build_engine", engine)
    for norm, optimizer, bits, lr in (("group", "adamw", 8, 1e-3),
                                      ("batch", "sgd", 32, 1e-2)):
        args = types.SimpleNamespace(norm=norm, optimizer=optimizer,
                                     state_bits=bits)
        with pytest.raises(Built):
            bench.preflight(0, 1, torch.device("cpu"), args)
        assert seen["norm"] == norm
        assert (seen["optim"].optimizer, seen["optim"].state_bits,
                seen["optim"].lr) == (optimizer, bits, lr)
        assert (seen["space"].momentum is None) == (optimizer == "adamw")


@pytest.mark.parametrize("device", [
    "cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_holds_all_of_the_state(tmp_path, device, bits):
    """What a resumed run starts with is what the saved one ended with, to the
    bit, and one more step on the same gradients is the same step."""
    from eventgrad_amd.train.trainer import Trainer
    first = Trainer(serial_cfg(tmp_path, device, epochs=1, bits=bits))
    first.train()
    second = Trainer(serial_cfg(tmp_path, device, epochs=2, bits=bits,
                                resume=True))
    assert (second.pass_num, second.start_epoch) == (first.pass_num, 2)

    def same():
        a, b = first.engine.opt, second.engine.opt
        assert torch.equal(first.space.param, second.space.param)
        assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
        assert all(torch.equal(getattr(a, k), getattr(b, k)) for k in
                   ("_step", "_powers", "_coef", "_decay", "codes",
                    "exponents"))
        assert a.seed == b.seed

    same()
    first.space.grad.normal_()
    second.space.grad.copy_(first.space.grad)
    for tr in (first, second):
        tr.engine.step()
    same()
