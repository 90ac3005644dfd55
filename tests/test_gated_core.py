"""The gated core in the nets, the actor loop and the learner."""

import copy

import numpy as np
import pytest
import torch

from pytorch_r2d2_dpg_amd.actor import ActorWorker, VectorActorWorker
from pytorch_r2d2_dpg_amd.checkpoint import load_checkpoint, save_checkpoint
from pytorch_r2d2_dpg_amd.config import Config
from pytorch_r2d2_dpg_amd.envs import make_env
from pytorch_r2d2_dpg_amd.learner import Learner
from pytorch_r2d2_dpg_amd.models import ActorNet, GatedCore, make_models
from pytorch_r2d2_dpg_amd.replay.buffer import SequenceReplay


def small_cfg(**model):
    cfg = Config()
    cfg.env.name = "pendulum"
    cfg.env.time_limit = 50
    cfg.model.hidden_size = 16
    cfg.model.trunk_sizes = (16,)
    cfg.model.core = "gated"
    cfg.replay.seq_len = 12
    cfg.replay.burn_in = 4
    cfg.replay.overlap = 6
    cfg.replay.n_step = 3
    cfg.replay.capacity = 128
    cfg.replay.min_fill = 4
    cfg.learner.batch_size = 8
    for k, v in model.items():
        setattr(cfg.model, k, v)
    return cfg


def test_steps_match_sequence():
    torch.manual_seed(0)
    core = GatedCore(5, 8).double()
    x = torch.randn(9, 3, 5).double()
    seq, (h1, h2) = core(x)
    st, ys = None, []
    for t in range(9):
        y, st = core.step(x[t], st)
        ys.append(y)
    assert torch.allclose(torch.stack(ys), seq, atol=1e-12)
    assert torch.allclose(st[0], h1, atol=1e-12) and torch.allclose(st[1], h2, atol=1e-12)
    tail, _ = core(x[4:], core(x[:4])[1])  # burn-in, then the rest
    assert torch.allclose(tail, seq[4:], atol=1e-12)


def test_gradients_against_differences():
    torch.manual_seed(1)
    core = GatedCore(3, 4).double()
    x = torch.randn(4, 2, 3, dtype=torch.double, requires_grad=True)
    h = torch.randn(2, 2, 4, dtype=torch.double, requires_grad=True)

    def flat(x, h):
        y, (h1, h2) = core(x, (h[0], h[1]))
        return y, h1, h2
    assert torch.autograd.gradcheck(flat, (x, h))


def test_state_stays_wide_and_unknown_core_is_refused():
    core = GatedCore(5, 8).bfloat16()
    assert core.zero_state(3)[0].dtype == torch.float32
    y, (h1, h2) = core(torch.randn(2, 3, 5).bfloat16())
    assert y.dtype == torch.bfloat16 and h1.dtype == h2.dtype == torch.float32
    with pytest.raises(ValueError, match="unknown model.core"):
        ActorNet((3,), 1, hidden_size=8, trunk_sizes=(8,), core="gru")


def test_actor_learner_and_checkpoint(tmp_path):
    cfg = small_cfg()
    worker = ActorWorker(cfg, actor_id=0, sigma=0.3)
    rep = SequenceReplay(cfg.replay.capacity, cfg.replay.seq_len + cfg.replay.n_step,
                         worker.spec.obs_shape, worker.spec.action_dim, cfg.model.hidden_size,
                         per_alpha=cfg.replay.per_alpha, seed=0)
    while len(rep) < cfg.replay.min_fill:
        rep.add(worker.rollout(60))
    lrn = Learner(cfg, worker.spec, device="cpu", replay=rep)
    before = [p.clone() for p in list(lrn.actor.parameters()) + list(lrn.critic.parameters())]
    stats = lrn.train_step(rep.sample(cfg.learner.batch_size))
    assert np.isfinite(stats.critic_loss) and np.isfinite(stats.actor_loss)
    after = list(lrn.actor.parameters()) + list(lrn.critic.parameters())
    assert all(not torch.equal(a, b) for a, b in zip(before, after))
    sd = lrn.actor_state_for_sync()
    worker.load_weights(sd["actor"], sd["critic"])
    path = save_checkpoint(lrn, str(tmp_path))
    other = Learner(cfg, worker.spec, device="cpu", replay=rep)
    load_checkpoint(other, path)
    for a, b in zip(other.actor.parameters(), lrn.actor.parameters()):
        assert torch.equal(a, b)
    assert VectorActorWorker(cfg, num_envs=3).rollout(40) is not None


# ------------------------------------------------------------------------ GPU
def batch_of(cfg, spec, B, seed, idx=None):
    L = cfg.replay.seq_len + cfg.replay.n_step
    g = torch.Generator().manual_seed(seed)
    return {
        "obs": torch.randn(B, L, *spec.obs_shape, generator=g).cuda(),
        "action": torch.randn(B, L, spec.action_dim, generator=g).clamp_(-1, 1).cuda(),
        "reward": torch.rand(B, L, generator=g).cuda(),
        "done": torch.zeros(B, L).cuda(),
        "state": (torch.randn(B, 4, cfg.model.hidden_size, generator=g) * 0.1).cuda(),
        "weight": torch.ones(B).cuda(),
        "idx": idx,
    }


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T, B, I, H", [(1, 64, 40, 128), (37, 5, 23, 72), (90, 3, 8, 33)])
def test_core_against_64_bits(T, B, I, H, dtype):
    torch.manual_seed(2)
    core = GatedCore(I, H).to("cuda", dtype)
    x = torch.randn(T, B, I, device="cuda").to(dtype).requires_grad_(True)
    h = [torch.randn(B, H, device="cuda").requires_grad_(True) for _ in range(2)]
    wide = copy.deepcopy(core).double().cpu()
    xw = x.detach().double().cpu().requires_grad_(True)
    hw = [t.detach().double().cpu().requires_grad_(True) for t in h]
    dy = torch.randn(T, B, H)
    got, want = [], []
    for c, a, s, out in ((core, x, h, got), (wide, xw, hw, want)):
        y, (h1, h2) = c(a, tuple(s))
        ins = [a, *s, *c.parameters()]
        out += [y, h1, h2] + list(torch.autograd.grad(
            [y, h1, h2], ins, [dy.to(y.device, y.dtype), s[0].detach(), s[1].detach()]))
    # On the longest path twelve results are rounded to the type forward and as
    # many backward, each by half a step of its norm at most; the norms in between
    # set every sum back to its own scale.
    bound = 24 * torch.finfo(dtype).eps / 2 + 1e-5
    for i, (g, w) in enumerate(zip(got, want)):
        off = (g.detach().double().cpu() - w).norm() / w.norm()
        assert off < bound, (i, float(off))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_learner_step_gpu(dtype, monkeypatch):
    spec = make_env("humanoid-run").spec
    results = []
    for sequential in (False, True):
        if sequential:
            monkeypatch.setenv("R2D2_NO_OVERLAP", "1")
        cfg = small_cfg(dtype=dtype, hidden_size=96, trunk_sizes=(96,))
        torch.manual_seed(4)
        lrn = Learner(cfg, spec, device="cuda")
        for s in range(2):
            stats = lrn.train_step(batch_of(cfg, spec, 24, s))
            assert np.isfinite(stats.critic_loss) and np.isfinite(stats.actor_loss)
        # a gradient reaches every parameter (a step of 1e-4 does not move a bf16 one)
        for p in list(lrn.actor.parameters()) + list(lrn.critic.parameters()):
            assert p.grad.isfinite().all() and p.grad.any()
        results.append([p.detach().clone() for p in
                        list(lrn.actor.parameters()) + list(lrn.critic.parameters())])
    for a, b in zip(*results):  # the side stream changes no result
        assert torch.allclose(a.float(), b.float(), atol=2e-3, rtol=1e-2)


@pytest.mark.gpu
def test_learner_graph_replays_match_eager():
    spec = make_env("humanoid-run").spec
    cfg = small_cfg(dtype="bf16", hidden_size=64, trunk_sizes=(64,))
    idx = torch.arange(16).cuda()
    torch.manual_seed(5)
    graphed = Learner(cfg, spec, device="cuda")
    graphed.capture_graph(batch_of(cfg, spec, 16, 0, idx))
    for s in range(3):
        # an eager learner from the graphed one's weights and moments, one step on
        eager = Learner(cfg, spec, device="cuda")
        for name in ("actor", "critic", "target_actor", "target_critic"):
            getattr(eager, name).load_state_dict(getattr(graphed, name).state_dict())
        for name in ("opt_actor", "opt_critic"):
            state = copy.deepcopy(getattr(graphed, name).state_dict())
            getattr(eager, name).load_state_dict(state)
        batch = batch_of(cfg, spec, 16, 1 + s, idx)
        a, b = graphed.train_step(batch), eager.train_step(batch)
        torch.cuda.synchronize()
        assert abs(a.critic_loss - b.critic_loss) <= 1e-3 * abs(b.critic_loss) + 1e-6
        assert abs(a.actor_loss - b.actor_loss) <= 1e-3 * abs(b.actor_loss) + 1e-6
        for p, q in zip(graphed.critic.parameters(), eager.critic.parameters()):
            assert torch.allclose(p.float(), q.float(), atol=2e-3, rtol=1e-2)


# ------------------------------------------------ the state on its way to the learner
@pytest.mark.parametrize("core, stored", [("gated", torch.float32), ("lstm", torch.bfloat16)])
def test_replay_keeps_the_state_as_wide_as_the_core(core, stored):
    """The gated core's state stays in 32 bits in a bf16 run's shard too; the LSTM's is
    bf16 in its learner and may be stored so."""
    from pytorch_r2d2_dpg_amd.orchestrator import run_training
    cfg = small_cfg(dtype="bf16", core=core)
    cfg.actor.num_actors = 1
    lrn = run_training(cfg, device="cpu", max_steps=1)
    rep = lrn.replay
    assert rep.state.dtype == stored and rep.action.dtype == torch.bfloat16
    state = rep.state[:len(rep)].float()
    assert torch.equal(state, state.bfloat16().float()) == (stored == torch.bfloat16)
    assert rep.sample(4)["state"].dtype == stored


def test_bench_keeps_the_state_as_wide_as_the_core(monkeypatch, capsys):
    import sys

    import bench
    shards = []
    make = bench.GpuSequenceReplay
    monkeypatch.setattr(bench, "GpuSequenceReplay", lambda **kw: shards.append(make(**kw)) or shards[-1])
    for core, stored in (("gated", torch.float32), ("lstm", torch.bfloat16)):
        monkeypatch.setattr(sys, "argv", [
            "bench.py", "--device", "cpu", "--core", core, "--hidden", "16", "--batch", "4", "--seq-len", "8",
            "--burn-in", "2", "--replay-capacity", "16", "--steps", "1", "--warmup", "0"])
        assert bench.main() in (0, None)
        assert shards[-1].state.dtype == stored
    assert capsys.readouterr().out.count('"metric"') == 2
