"""Normalised heads, the scaled embedding with a gradient by token and AdamW with moments in 8 bits, as jobs use them: through models,
engine, checkpoints and flags, on CPU ranks and together in whole steps on a GPU."""
import math
import os

import pytest
import torch

from dist_utils import run_workers
from test_dist_cpu import PIPE_1x2, PIPE_2x1, tiny_cfg
from zorse_b200.config.training_config import parse_pipeline_dict
from zorse_b200.engine.zero import AdamConfig
from zorse_b200.models import registry
from zorse_b200.trainer import Trainer, TrainerOptions

OVERRIDES = {"qk_norm": True, "embed_scale": 3.0, "embed_by_token": True}
ONE = [{"gpu_ranks": [0], "num_microbatches_per_rank": [4], "layer_partition": [0, 2], "zero_config": [[0]]}]


def _one_rank(reduce="float32", compute="float32", model="tiny_llama", seq=32, pipe=ONE, **kw):
    return parse_pipeline_dict(tiny_cfg(pipe, seq=seq, model_name=model, reduce_dtype=reduce, autocast_dtype=compute, **kw))


def _state(tr):
    return [t.clone() for st in tr.stages for u in st.engine.units for t in u.state_tensors().values()]


def _adamw_oracle(cfg, overrides, lr, decay):
    from zorse_b200.utils.oracle import OracleTrainer

    orc = OracleTrainer(cfg, model_overrides=overrides)
    orc.opt = torch.optim.AdamW(orc.flats, lr=lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=decay)
    return orc


@pytest.mark.parametrize("model,more", [("tiny_llama", {}), ("deepspeedmistral_toy", {}), ("toygpt", {"heads": 4})])
@pytest.mark.parametrize("schedule,recompute", [("1f1b", False), ("zero2", True)])
def test_gradients_match_autograd(model, more, schedule, recompute):
    """The explicit backward passes against autograd through the same model (RoPE and grouped heads, a window, learned positions)."""
    from zorse_b200.utils.oracle import OracleTrainer

    cfg = _one_rank(model=model)
    ov = {"layers": 2, **OVERRIDES, **more}
    tr = Trainer(cfg, TrainerOptions(schedule=schedule, ops="ref", activation_recompute=recompute, model_overrides=ov, lr=0.0))
    assert any("qnorm_w" in dict(u.layer.layout()[0]) for u in tr.stages[0].engine.units)
    batch = tr.synthetic_batch()
    loss, grads = OracleTrainer(cfg, model_overrides=ov).grads(batch)
    assert tr.train_step_from_host(batch) == pytest.approx(loss, rel=1e-5)
    for u, want in zip(tr.stages[0].engine.units, grads):
        got = u.m[:want.numel()] / 0.1             # lr = 0: the first moment after one step is a tenth of the gradient
        assert (got - want).abs().max() <= 2e-4 * want.abs().max() + 1e-8


@pytest.mark.parametrize("how", [dict(defer_wgrad=True), dict(defer_tail_wgrad=2)])
def test_held_back_weight_gradients_change_nothing(how):
    """Schedules that hold weight gradients back leave those of the head norms and the embedding where they are."""
    states = []
    for more in ({}, how):
        tr = Trainer(_one_rank(), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2, **OVERRIDES}, optimizer="adamw", **more))
        batch = tr.synthetic_batch()
        for _ in range(2):
            tr.train_step_from_host(batch)
        states.append(_state(tr))
    for a, b in zip(*states):
        torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("in_backward", [False, True])
def test_adamw_follows_torch(in_backward):
    cfg = _one_rank()
    ov = {"layers": 2, **OVERRIDES}
    tr = Trainer(cfg, TrainerOptions(schedule="1f1b", ops="ref", model_overrides=ov, optimizer="adamw", weight_decay=0.1,
                                     optimizer_in_backward=in_backward))
    orc = _adamw_oracle(cfg, ov, 1e-3, 0.1)
    batch = tr.synthetic_batch()
    for _ in range(3):
        assert tr.train_step_from_host(batch) == pytest.approx(orc.step(batch), abs=2e-4)
    for u, f in zip(tr.stages[0].engine.units, orc.flats):
        assert (u.master[:f.numel()] - f.detach()).abs().max() < 5e-4
    assert tr.counters()[0].adam_steps == 3 * len(tr.stages[0].engine.units)


def test_one_launch_for_all_units_and_the_same_bits_as_one_by_one(monkeypatch):
    """The step behind the backward pass gets the stage's units as one list; the optimizer inside it gets them one by one."""
    cfg = _one_rank()
    states, sizes = [], []
    for in_backward in (False, True):
        tr = Trainer(cfg, TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}, optimizer="adamw",
                                         moment_bits=8, optimizer_in_backward=in_backward))
        step, calls = tr.ops.adamw_step, []
        monkeypatch.setattr(tr.ops, "adamw_step", lambda p, *a, **k: calls.append(len(p)) or step(p, *a, **k), raising=False)
        for _ in range(2):
            tr.train_step_from_host(tr.synthetic_batch())
        monkeypatch.undo()
        states.append(_state(tr))
        sizes.append(calls)
    units = len(tr.stages[0].engine.units)
    assert sizes == [[units] * 2, [1] * (2 * units)]
    assert all(torch.equal(a, b) for a, b in zip(*states))


def test_moments_in_8_bits_take_two_bytes_a_parameter_and_train():
    cfg = _one_rank()
    losses = []
    for bits in (32, 8):
        tr = Trainer(cfg, TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}, optimizer="adamw", moment_bits=bits))
        batch = tr.synthetic_batch()
        losses.append([tr.train_step_from_host(batch) for _ in range(6)])
    u = tr.stages[0].engine.units[1]
    assert u.m is None and u.v is None
    assert sum(t.numel() * t.element_size() for t in u.moments) <= 2 * u.shard_n + 4 * (u.shard_n // 256 + 1)
    # the first step has nothing rounded behind it, so the first two losses are the same
    assert losses[0][:2] == pytest.approx(losses[1][:2], abs=1e-5)


def _save(rank, world, cfg, ckdir, opts):
    from zorse_b200.ckpt.writer import save_checkpoint

    tr = Trainer(parse_pipeline_dict(cfg), TrainerOptions(backend="gloo", schedule="layer_major", **opts))
    batch = tr.synthetic_batch()
    for _ in range(3):
        tr.train_step_from_host(batch)
    save_checkpoint(tr, ckdir, 3)
    loss = [tr.global_loss(tr.train_step_from_host(batch)) for _ in range(2)]
    return loss, _state(tr)


def _resume(rank, world, cfg, ckdir, opts):
    from zorse_b200.ckpt.reader import load_checkpoint

    tr = Trainer(parse_pipeline_dict(cfg), TrainerOptions(backend="gloo", schedule="layer_major", **opts))
    load_checkpoint(tr, os.path.join(ckdir, "step_3"))
    batch = tr.synthetic_batch()
    loss = [tr.global_loss(tr.train_step_from_host(batch)) for _ in range(2)]
    return loss, _state(tr)


def test_checkpoints_of_8_bit_moments_resume_with_the_same_bits(tmp_path):
    """Two ranks that share each unit: the job that goes on and the one resumed under the same plan end in the same state, moments
    included; under another plan, and with moments in 32 bits, it goes on too."""
    opts = dict(optimizer="adamw", moment_bits=8, weight_decay=0.01, model_overrides=OVERRIDES)
    ck = str(tmp_path / "ck")
    a = run_workers(2, _save, tiny_cfg(PIPE_1x2), ck, opts)
    b = run_workers(2, _resume, tiny_cfg(PIPE_1x2), ck, opts)
    for (la, sa), (lb, sb) in zip(a, b):
        assert la == lb and all(torch.equal(x, y) for x, y in zip(sa, sb))
    c = run_workers(2, _resume, tiny_cfg(PIPE_2x1), ck, opts)
    assert c[0][0][0] == pytest.approx(a[0][0][0], abs=1e-4)
    d = run_workers(2, _resume, tiny_cfg(PIPE_1x2), ck, {**opts, "moment_bits": 32})
    assert d[0][0][0] == pytest.approx(a[0][0][0], abs=1e-5)


def _tp_losses(rank, world, cfg):
    tr = Trainer(parse_pipeline_dict(cfg), TrainerOptions(backend="gloo", schedule="1f1b", optimizer="adamw", weight_decay=0.1,
                                                          model_overrides=OVERRIDES))
    batch = tr.synthetic_batch()
    losses = [tr.global_loss(tr.train_step_from_host(batch)) for _ in range(3)]
    whole = {u.gid: u.full_master()[:u.layer.layout()[1]].clone() for st in tr.stages for u in st.engine.units}
    return losses, whole, tr.tp_index


def test_tensor_parallel_slices_share_the_head_weights():
    """The weights of the head norms are whole on every slice, their gradients summed over the lane."""
    cfg = tiny_cfg([dict(ONE[0], layer_partition=[0, 4])], tensor_parallel_size=2)
    got = run_workers(2, _tp_losses, cfg)
    orc = _adamw_oracle(parse_pipeline_dict(tiny_cfg([dict(ONE[0], layer_partition=[0, 4])])), OVERRIDES, 1e-3, 0.1)
    g = torch.Generator().manual_seed(7919)
    batch = {k: torch.randint(0, 512, (4, 2, 32), generator=g) for k in ("inputs", "targets")}
    want = [orc.step(batch) for _ in range(3)]
    spec = registry.get_spec("tiny_llama", vocab=512, **OVERRIDES)
    for losses, _, _ in got:
        assert losses == pytest.approx(want, abs=2e-4)
    for gid in range(1, 5):
        whole = torch.zeros_like(orc.flats[gid].detach())
        for _, params, t in got:
            registry.make_block(spec, 2, t).store_into_whole(params[gid], whole)
        assert (whole - orc.flats[gid].detach()).abs().max() < 5e-4


def test_refusals():
    for wrong in (dict(moment_bits=8), dict(moment_bits=16, decoupled=True)):
        with pytest.raises(ValueError):
            AdamConfig(**wrong)
    cfg = _one_rank()
    with pytest.raises(ValueError):
        Trainer(cfg, TrainerOptions(ops="ref", optimizer="sgd"))
    with pytest.raises(ValueError):
        Trainer(cfg, TrainerOptions(ops="ref", moment_bits=8))
    vit = registry.get_spec("deepspeedvit_default", embed_by_token=True)
    with pytest.raises(ValueError):
        registry.make_embedding(vit, 0)
    with pytest.raises(RuntimeError, match="tensor-parallel"):
        run_workers(2, _tp_8_bits, tiny_cfg([dict(ONE[0], layer_partition=[0, 4])], tensor_parallel_size=2))


def _tp_8_bits(rank, world, cfg):
    Trainer(parse_pipeline_dict(cfg), TrainerOptions(backend="gloo", optimizer="adamw", moment_bits=8))


def test_fused_collectives_are_refused_with_adamw():
    """The fused reduce-scatter kernel steps with Adam itself; the engine says so before it builds such a unit."""
    from types import SimpleNamespace

    from zorse_b200.engine.zero import EngineConfig, StageEngine

    group = SimpleNamespace(size=2, ranks=(0, 1), index_of=lambda r: 0)
    one = SimpleNamespace(size=1, ranks=(0,), index_of=lambda r: 0)
    with pytest.raises(ValueError, match="AdamW"):
        StageEngine([], [], device=SimpleNamespace(type="cuda"), cfg=EngineConfig(collectives="fused", adam=AdamConfig(decoupled=True)),
                    ops=None, shard=group, replicate=one, rank=0, streams=object())


def test_flags_reach_the_job(tmp_path):
    import json

    from zorse_b200.cli.train import model_overrides
    from zorse_b200.config.flags import parse_args_zorse

    f = tmp_path / "c.json"
    f.write_text(json.dumps(tiny_cfg(ONE)))
    base = ["--config_file", str(f)]
    a = parse_args_zorse(base)
    assert (a.optimizer, a.weight_decay, a.moment_bits, model_overrides(a)) == ("adam", 0.0, 32, {})
    a = parse_args_zorse(base + ["--optimizer", "adamw", "--weight_decay", "0.1", "--moment_bits", "8", "--qk_norm", "--embed_scale", "3",
                                 "--embed_by_token"])
    assert (a.optimizer, a.weight_decay, a.moment_bits, model_overrides(a)) == ("adamw", 0.1, 8, OVERRIDES)


def test_models_without_the_options_keep_their_layout():
    for name in ("tiny_llama", "toygpt", "deepspeedmistral_toy"):
        a, b = registry.get_spec(name), registry.get_spec(name, qk_norm=True)
        plain, normed = registry.make_block(a), registry.make_block(b)
        assert "qnorm_w" not in plain.layout()[0]
        assert normed.num_params() == plain.num_params() + 2 * a.head_dim


# ---------------------------------------------------------------------------------------------------------------- on the GPU
def _gpu_cfg(model="tiny_llama", reduce="float32", layers=2, seq=256):
    d = tiny_cfg([dict(ONE[0], layer_partition=[0, layers])], seq=seq, vocab=2048, model_name=model, reduce_dtype=reduce,
                 autocast_dtype="bfloat16")
    return parse_pipeline_dict(d)


@pytest.mark.gpu
@pytest.mark.parametrize("model,more", [("tiny_llama", {}), ("deepspeedmistral_toy", {}), ("opt_125m", {})])
@pytest.mark.parametrize("schedule,recompute", [("1f1b", False), ("zero2", True)])
def test_step_on_the_gpu_matches_the_oracle(model, more, schedule, recompute):
    """All of them in one training step: loss and gradients against autograd in fp32, as the other models are held to."""
    from test_train_gpu import _oracle_from

    cfg = _gpu_cfg(model)
    ov = {"layers": 2, "qk_norm": True, "embed_scale": 4.0, "embed_by_token": True, **more}
    tr = Trainer(cfg, TrainerOptions(schedule=schedule, ops="sm100", activation_recompute=recompute, model_overrides=ov, lr=0.0,
                                     optimizer="adamw"))
    batch = tr.synthetic_batch()
    loss, grads = _oracle_from(tr, cfg, ov).grads(dict(batch))
    got = tr.train_step_from_host(batch)
    tr.check_kernels()
    assert abs(got - loss) < 0.03 * max(1.0, abs(loss))
    for u, want in zip(tr.stages[0].engine.units, grads):
        g = (u.m[:want.numel()] / (1 - 0.9)).float().cpu()
        cos = torch.nn.functional.cosine_similarity(g.flatten(), want.flatten(), dim=0).item()
        err = (g - want).abs().max().item() / (want.abs().max().item() + 1e-6)
        assert cos > 0.99 and err < 0.08, f"unit {u.gid} ({u.layer.kind}): rel err {err:.4f}, cosine {cos:.5f}"


@pytest.mark.gpu
@pytest.mark.parametrize("reduce", ["float32", "bfloat16"])
@pytest.mark.parametrize("in_backward,offload", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("bits", [32, 8])
def test_jobs_on_the_gpu_have_the_same_bits_twice(reduce, in_backward, offload, bits):
    """Whole steps, with the optimizer behind or inside the backward pass and with parked parameters, end in the same bits on a
    second run; with 8 bits every moment is one that the codes hold."""
    ends = []
    for _ in range(2):
        tr = Trainer(_gpu_cfg(reduce=reduce), TrainerOptions(schedule="1f1b", ops="sm100", model_overrides={"layers": 2, **OVERRIDES},
                                                             optimizer="adamw", weight_decay=0.1, moment_bits=bits,
                                                             optimizer_in_backward=in_backward, offload_model_params=offload))
        batch = tr.synthetic_batch()
        losses = [tr.train_step_from_host(batch) for _ in range(4)]
        tr.synchronize()
        ends.append((losses, _state(tr)))
    assert ends[0][0] == ends[1][0] and all(math.isfinite(x) for x in ends[0][0])
    assert all(torch.equal(a, b) for a, b in zip(ends[0][1], ends[1][1]))
    if bits == 8:
        for k in range(0, len(ends[0][1]), 3):
            for t in ends[0][1][k + 1:k + 3]:
                assert torch.equal(t.bfloat16().float(), t)


@pytest.mark.gpu
def test_optimizer_inside_and_behind_the_backward_pass_give_the_same_bits():
    ends = []
    for in_backward in (False, True):
        tr = Trainer(_gpu_cfg(), TrainerOptions(schedule="1f1b", ops="sm100", model_overrides={"layers": 2, **OVERRIDES},
                                                optimizer="adamw", moment_bits=8, optimizer_in_backward=in_backward))
        batch = tr.synthetic_batch()
        for _ in range(3):
            tr.train_step_from_host(batch)
        tr.synchronize()
        ends.append(_state(tr))
    assert all(torch.equal(a, b) for a, b in zip(*ends))


@pytest.mark.gpu
def test_native_calls_and_wrappers_give_the_same_bits():
    """The op layer's native calls against the wrappers that take what those decline."""
    from zorse_b200.ops import ref
    from zorse_b200.ops.api import get_ops
    from zorse_b200.ops.moments import encode

    ops = get_ops("sm100")
    k = ops.k
    g = torch.Generator().manual_seed(1)

    def bf(*shape):
        return torch.randn(*shape, generator=g).bfloat16().cuda()

    T, nq, nk, d, S = 96, 4, 2, 64, 48
    qkv, wq, wk, cs, dy = bf(T, (nq + 2 * nk) * d), bf(d), bf(d), ref.rope_table(S, d, 1e4).cuda(), bf(T, (nq + 2 * nk) * d)
    a, b = ops._qk_norm_rope_fwd(qkv, wq, wk, cs, S, nq, nk, d, 1e-5, True), k.qk_norm_rope_fwd(qkv, wq, wk, cs, S, nq, nk, d, 1e-5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    out = []
    for fn in (ops._qk_norm_rope_bwd, k.qk_norm_rope_bwd):
        gq, gk, dx = torch.ones(d, device="cuda"), torch.ones(d, device="cuda"), dy.clone()
        assert fn(dx, qkv, wq, wk, a[1], cs, S, nq, nk, d, gq, gk) is not None
        out.append((dx, gq, gk))
    assert all(torch.equal(x, y) for x, y in zip(*out))
    ids, table, pos, dout = torch.randint(0, 50, (T,), generator=g).cuda(), bf(50, 64), bf(S, 64), bf(T, 64)
    assert torch.equal(ops._embedding_scaled(ids, table, pos, S, 0, 2.0), k.embedding_scaled(ids, table, pos, S, 0, 2.0))
    out = []
    for fn in (ops._embedding_by_token, k.embedding_by_token):
        gt, gp = torch.ones(50, 64, device="cuda"), torch.ones(S, 64, device="cuda")
        fn(ids, dout, gt, gp, S, 0, 2.0)
        out.append((gt, gp))
    assert all(torch.equal(x, y) for x, y in zip(*out)) and (out[0][0] != 1).any()
    hyper = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.1, grad_scale=0.5)
    for bits in (32, 8):
        out = []
        for native in (True, False):
            g.manual_seed(3)
            p, gr = [torch.randn(n, generator=g).cuda() for n in (700, 33)], [torch.randn(n, generator=g).cuda() for n in (700, 33)]
            mom = [(torch.zeros_like(x), torch.zeros_like(x)) if bits == 32 else
                   type(encode(x, x.abs()))(*(t.cuda() for t in encode(x, x.abs()))) for x in p]
            p16, seeds = [torch.empty(700, dtype=torch.bfloat16, device="cuda"), None], [5, 6] if bits == 8 else None
            if native:
                assert ops._adamw_step(p, mom, gr, p16, seeds, [3, 9], 1e-3, 0.9, 0.999, 1e-8, 0.1, 0.5)
            else:
                k.adamw_step(p, mom, gr, p16, step=[3, 9], seeds=seeds, **hyper)
            out.append([*p, p16[0], *(t for m in mom for t in m)])
        assert all(torch.equal(x, y) for x, y in zip(*out))


@pytest.mark.gpu
def test_native_calls_decline_what_is_wrong():
    """What the native calls do not take goes to the wrappers, which refuse it in words."""
    from zorse_b200.ops.api import get_ops

    ops = get_ops("sm100")
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(x, w, w[:32], None, 4, 2, 1, 64, 1e-5)
    with pytest.raises(ValueError):
        ops.qk_norm_rope_fwd(x, w, w, None, 4, 3, 1, 64, 1e-5)
    with pytest.raises(ValueError):
        ops.embedding_bwd(torch.zeros(3, dtype=torch.long, device="cuda"), x, torch.zeros(5, 256, device="cuda"), by_token=True)
    p = torch.zeros(64, device="cuda")
    z = (p.clone(), p.clone())
    kw = dict(lr=1.0, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)
    with pytest.raises(ValueError, match="twice"):
        ops.adamw_step([p, p], [z, (p.clone(), p.clone())], [p.clone(), p.clone()], [None, None], step=1, **kw)
    with pytest.raises(ValueError):
        ops.adamw_step([p], [z], [p.clone()], [None], step=0, **kw)
