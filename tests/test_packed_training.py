"""Jobs on packed batches and with Muon: against the same documents one by one, against the formulas of the step, and what is refused."""
import json
import math
import os

import pytest
import torch

from dist_utils import run_workers
from test_dist_cpu import PIPE_2x1, tiny_cfg
from zorse_b200.config.training_config import parse_pipeline_dict
from zorse_b200.engine.zero import AdamConfig, EngineConfig, StageEngine
from zorse_b200.models import registry
from zorse_b200.ops import muon
from zorse_b200.ops.api import get_ops
from zorse_b200.parallel.groups import Group
from zorse_b200.trainer import Trainer, TrainerOptions
from zorse_b200.utils.data import pack_documents, random_documents

SMALL = {"hidden": 256, "ffn": 344}
ONE = [{"gpu_ranks": [0], "num_microbatches_per_rank": [4], "layer_partition": [0, 2], "zero_config": [[0]]}]
WHOLE = tiny_cfg([dict(ONE[0], layer_partition=[0, 4])])


def _cfg(model="tiny_llama", seq=32, **kw):
    return parse_pipeline_dict(tiny_cfg(ONE, seq=seq, model_name=model, **kw))


def test_pack_documents():
    docs = [torch.arange(1, 6), torch.arange(10, 13), torch.arange(20, 29), torch.arange(30, 31)]
    b = pack_documents(docs, 2, 2, 5)
    assert b["inputs"].view(2, 10).tolist() == [[1, 2, 3, 4, 5, 10, 11, 12, 20, 21], [22, 23, 24, 25, 26, 27, 28, 30, 0, 0]]
    assert b["targets"].view(2, 10).tolist() == [[2, 3, 4, 5, -100, 11, 12, -100, 21, -100], [23, 24, 25, 26, 27, 28, -100, -100, -100, -100]]
    assert b["offsets"].tolist() == [[0, 5, 8, 10], [0, 7, 8, 8]] and b["offsets"].dtype == torch.int32
    r = random_documents(3, 2, 50, 40, 7, torch.Generator().manual_seed(1))
    assert (r["offsets"][:, -1] == 100).all() and (r["offsets"].diff(dim=1) <= 50).all() and r["offsets"].shape[1] > 8
    assert pack_documents([], 1, 1, 4)["offsets"].tolist() == [[0]]


def _one_by_one(cfg, overrides, batch, params=None):
    """Loss and gradients by autograd through the model, each document by itself: the packed path is not used.  params: the layers' (as
    a GPU job draws them), None: as drawn on the CPU."""
    from zorse_b200.utils.oracle import OracleTrainer

    orc = OracleTrainer(cfg, model_overrides=overrides)
    if params is not None:
        with torch.no_grad():
            for flat, p in zip(orc.flats, params):
                flat.copy_(p[:flat.numel()])
    M, T = cfg.num_microbatches, cfg.microbatch_size * cfg.sequence_length
    total = 0.0
    for g in range(M):
        bounds = batch["offsets"][g].tolist()
        for lo, hi in zip(bounds, bounds[1:]):
            if lo == hi:
                continue
            x, y = (batch[k][g].reshape(-1)[lo:hi] for k in ("inputs", "targets"))
            ctx = {"B": 1, "S": hi - lo, "loss_scale": 1.0, "targets": y}
            for ly, flat in zip(orc.layers, orc.flats):
                ly.bind(flat, None)
                x = ly.forward(x, ctx, orc.ops, None)
            total = total + x.float().sum() / (M * T)
    total.backward()
    return float(total.detach()), [f.grad for f in orc.flats]


MODELS = [("tiny_llama", {}), ("deepspeedmistral_toy", {"window": 9}), ("toygpt", {}), ("tiny_llama", {"qk_norm": True, "embed_scale": 2.0})]


@pytest.mark.parametrize("model,more", MODELS)
@pytest.mark.parametrize("schedule,recompute", [("1f1b", False), ("zero2", True)])
def test_a_packed_batch_is_its_documents_one_by_one(model, more, schedule, recompute):
    cfg, ov = _cfg(model), {"layers": 2, **more}
    tr = Trainer(cfg, TrainerOptions(schedule=schedule, ops="ref", activation_recompute=recompute, model_overrides=ov, lr=0.0, documents=11))
    batch = tr.synthetic_batch()
    assert batch["offsets"].shape[1] > 4
    batch["targets"][1].view(-1)[50:] = -100           # the last tokens of this microbatch belong to nobody
    batch["offsets"][1].clamp_(max=50)
    loss, grads = _one_by_one(cfg, ov, batch)
    assert tr.train_step_from_host(batch) == pytest.approx(loss, rel=1e-5)
    for u, want in zip(tr.stages[0].engine.units, grads):
        got = u.m[:want.numel()] / 0.1             # lr = 0: the first moment after one step is a tenth of the gradient
        assert (got - want).abs().max() <= 2e-4 * want.abs().max() + 1e-8
    plain = {k: batch[k] for k in ("inputs", "targets")}
    assert tr.train_step_from_host(plain) != pytest.approx(loss, rel=1e-4)      # the packing goes with its batch


def _stages(rank, world, cfg):
    tr = Trainer(parse_pipeline_dict(cfg), TrainerOptions(backend="gloo", schedule="1f1b", documents=9, optimizer="adamw", model_overrides=SMALL))
    batch = tr.synthetic_batch()
    return [tr.global_loss(tr.train_step_from_host(batch)) for _ in range(2)]


def test_every_stage_of_a_pipeline_attends_by_document():
    tr = Trainer(parse_pipeline_dict(WHOLE), TrainerOptions(schedule="1f1b", ops="ref", documents=9, optimizer="adamw", model_overrides=SMALL))
    batch = tr.synthetic_batch()
    two = run_workers(2, _stages, tiny_cfg(PIPE_2x1))
    assert two[0] == pytest.approx([tr.train_step_from_host(batch) for _ in range(2)], abs=1e-5)


def test_refused_batches():
    tr = Trainer(_cfg(), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}, documents=9))
    batch = tr.synthetic_batch()
    o = batch["offsets"]
    for wrong in (o.long(), o[:2], o[0], o[:, :0], o + 1, o.flip(1), torch.cat([o, torch.full((4, 1), 65, dtype=torch.int32)], 1)):
        with pytest.raises(ValueError):
            tr.pack({**batch, "offsets": wrong})
    gpt = Trainer(_cfg("toygpt", seq=24), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2, "max_positions": 16}))
    with pytest.raises(ValueError, match="learned positions"):
        gpt.pack({"offsets": torch.tensor([[0, 30, 48]] * 4, dtype=torch.int32)})
    bert = Trainer(_cfg("tiny_llama"), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2, "pool": "first"}))
    with pytest.raises(ValueError, match="every position"):
        bert.pack(batch)
    assert tr.pack({"inputs": batch["inputs"]}) is None


def test_replays_take_the_packing():
    from zorse_b200.utils.replay import replay_check

    tr = Trainer(_cfg(), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}, documents=9))
    batch = tr.synthetic_batch()
    inputs, targets, _ = tr.to_device(batch)
    rep = replay_check(tr, inputs, targets, packed=tr.pack(batch))
    one = Trainer(_cfg(), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}, documents=9))
    want = float(one.train_step(inputs, targets, one.pack(batch)))
    assert rep["identical"] and rep["loss"] == (want, want)
    plain = Trainer(_cfg(), TrainerOptions(schedule="1f1b", ops="ref", model_overrides={"layers": 2}))
    assert float(plain.train_step(inputs, targets)) != want
    with pytest.raises(ValueError, match="documents"):
        Trainer(_cfg(), TrainerOptions(schedule="1f1b", ops="ref", documents=-3))


# ------------------------------------------------------------------------------------------------------------------ Muon
def _engine(device="cpu", **kw):
    spec = registry.get_spec("tiny_llama", vocab=512, layers=2, kv_heads=2, **SMALL)
    layers = [registry.make_embedding(spec, 32), registry.make_block(spec), registry.make_block(spec), registry.make_head(spec)]
    gpu = device == "cuda"
    cfg = EngineConfig(compute_dtype=torch.bfloat16 if gpu else torch.float32, adam=AdamConfig(decoupled=True, muon=True, weight_decay=0.1), **kw)
    one = Group(ranks=(0,), pg=None)
    return StageEngine(layers, [0, 1, 2, 3], device=torch.device("cuda", 0) if gpu else torch.device("cpu"), cfg=cfg,
                       ops=get_ops("sm100" if gpu else "ref"), shard=one, replicate=one, rank=0)


def _steps(engine, n=2):
    for k in range(n):
        for i, u in enumerate(engine.units):
            u.grad_views()
            u.grad.copy_(torch.randn(u.n, generator=torch.Generator().manual_seed(10 * k + i)) * 1e-2)
            u.reduce_grads()
        engine.optimizer_step()
        engine.finish_step()
    if engine.device.type == "cuda":
        torch.cuda.synchronize()
    return [{k: t.detach().float().cpu().clone() for k, t in u.state_tensors().items()} for u in engine.units]


def _expected(engine, n=2):
    """The state after n steps by the formulas, in 64 bits."""
    out = []
    for i, u in enumerate(engine.units):
        p = u.master.double().cpu()
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        is_matrix = torch.zeros(p.numel(), dtype=torch.bool)
        for o, r, c in u.layer.matrices():
            is_matrix[o:o + r * c] = True
        for k in range(n):
            g = (torch.randn(u.n, generator=torch.Generator().manual_seed(10 * k + i)) * 1e-2).to(u.cfg.reduce_dtype).double()
            old_m = m.clone()
            m = torch.where(is_matrix, 0.95 * m + g, 0.9 * m + 0.1 * g)
            v = torch.where(is_matrix, 0.0, 0.999 * v + 0.001 * g * g)
            step = 1e-3 * (m / (1 - 0.9 ** (k + 1))) / ((v / (1 - 0.999 ** (k + 1))).sqrt() + 1e-8)
            for o, r, c in u.layer.matrices():
                new = (0.95 * old_m + g)[o:o + r * c].view(r, c)
                x = muon.orthogonalize(g[o:o + r * c].view(r, c) + 0.95 * new)
                step[o:o + r * c] = 1e-3 * 0.2 * math.sqrt(max(r, c)) * x.reshape(-1)
            p = p * (1 - 1e-4) - step
        out.append({"master": p, "m": m, "v": v})
    return out


def test_the_matrices_of_a_block_cover_its_weights():
    for name, more in (("tiny_llama", {"kv_heads": 2}), ("toygpt", {}), ("llama2_7b", {}), ("opt_125m", {})):
        spec = registry.get_spec(name, **more)
        block = registry.make_block(spec)
        lay = block.layout()[0]
        covered = sorted((o, o + r * c) for o, r, c in block.matrices())
        want = sorted((o, o + math.prod(sh)) for n, (o, sh) in lay.items() if len(sh) == 2)
        merged = []
        for a, b in covered:
            if merged and merged[-1][1] == a and (a, b) not in want:
                merged[-1] = (merged[-1][0], b)
            else:
                merged.append((a, b))
        assert merged == want
        d, h = spec.head_dim, spec.hidden
        assert [(r, c) for _, r, c in block.matrices()][:4] == [(spec.heads * d, h), (spec.n_kv * d, h), (spec.n_kv * d, h), (h, spec.heads * d)]
    assert registry.make_embedding(spec, 8).matrices() == [] and registry.make_head(spec).matrices() == []


@pytest.mark.parametrize("in_backward,offload", [(False, False), (True, False), (True, True), (False, True)])
def test_muon_in_the_engine_cpu(in_backward, offload):
    engine = _engine(optimizer_in_backward=in_backward, offload_params=offload)
    expected = _expected(_engine())
    for u, got, want in zip(engine.units, _steps(engine), expected):
        for k in ("master", "m", "v"):
            assert torch.allclose(got[k].double(), want[k], rtol=1e-4, atol=2e-6), (u.layer.kind, k)
        assert u.v.numel() == u.n - sum(-(-r * c // 64) * 64 for _, r, c in u.layer.matrices())


def test_one_list_for_all_matrices(monkeypatch):
    engine = _engine()
    step, calls = engine.ops.muon_step, []
    monkeypatch.setattr(engine.ops, "muon_step", lambda p, *a, **k: calls.append([tuple(x.shape) for x in p]) or step(p, *a, **k), raising=False)
    _steps(engine, 1)
    assert calls == [[(256, 256), (64, 256), (64, 256), (256, 256), (344, 256), (344, 256), (256, 344)] * 2]


def _resume(rank, world, cfg, ckdir, optimizer="muon", **kw):
    from zorse_b200.ckpt.reader import load_checkpoint

    tr = Trainer(parse_pipeline_dict(cfg), TrainerOptions(schedule="layer_major", optimizer=optimizer, documents=13, model_overrides=SMALL,
                                                          **(kw or {"backend": "gloo"})))
    load_checkpoint(tr, os.path.join(ckdir, "step_2"))
    return tr.global_loss(tr.train_step_from_host(tr.synthetic_batch()))


def test_checkpoints_with_muon(tmp_path):
    """Under another split into stages too; another optimizer is refused by name, and the recovery command carries this one."""
    from zorse_b200.ckpt.reader import CheckpointError, flags_of, read_meta
    from zorse_b200.ckpt.writer import save_checkpoint

    ck = str(tmp_path / "ck")
    tr = Trainer(parse_pipeline_dict(WHOLE), TrainerOptions(schedule="layer_major", ops="ref", optimizer="muon", documents=13, model_overrides=SMALL))
    batch = tr.synthetic_batch()
    for _ in range(2):
        tr.train_step_from_host(batch)
    save_checkpoint(tr, ck, 2)
    want = tr.train_step_from_host(batch)
    assert _resume(0, 1, WHOLE, ck, ops="ref") == want
    assert run_workers(2, _resume, tiny_cfg(PIPE_2x1), ck)[0] == pytest.approx(want, abs=1e-4)
    with pytest.raises(CheckpointError, match="optimizer"):
        _resume(0, 1, WHOLE, ck, "adamw", ops="ref")
    assert flags_of(read_meta(os.path.join(ck, "step_2"))) == ["--optimizer", "muon"]


def test_refused_jobs(tmp_path):
    two, one = Group(ranks=(0, 1), pg=None), Group(ranks=(0,), pg=None)
    cfg = EngineConfig(compute_dtype=torch.float32, adam=AdamConfig(decoupled=True, muon=True))
    block = registry.make_block(registry.get_spec("tiny_llama", **SMALL))
    for groups in (dict(shard=two, replicate=one), dict(shard=one, replicate=one, tp_group=two)):
        with pytest.raises(ValueError, match="whole matrices"):
            StageEngine([block], [0], device=torch.device("cpu"), cfg=cfg, ops=get_ops("ref"), rank=0, **groups)
    for wrong in (dict(muon=True), dict(muon=True, decoupled=True, moment_bits=8)):
        with pytest.raises(ValueError):
            AdamConfig(**wrong)
    with pytest.raises(ValueError):
        Trainer(_cfg(), TrainerOptions(ops="ref", optimizer="muon", moment_bits=8))
    from zorse_b200.config.flags import parse_args_zorse

    f = tmp_path / "c.json"
    f.write_text(json.dumps(tiny_cfg(ONE)))
    a = parse_args_zorse(["--config_file", str(f), "--optimizer", "muon", "--documents", "300"])
    assert a.optimizer == "muon" and a.documents == 300 and parse_args_zorse(["--config_file", str(f)]).documents == 0


# ------------------------------------------------------------------------------------------------------------------ on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("in_backward,offload", [(False, False), (True, True)])
def test_muon_in_the_engine(in_backward, offload):
    """Matrices step within the products' error (tests/test_muon.py) of the formulas; everything else as AdamW does."""
    expected = _expected(_engine("cuda"))
    engine = _engine("cuda", optimizer_in_backward=in_backward, offload_params=offload)
    for u, got, want in zip(engine.units, _steps(engine), expected):
        assert torch.allclose(got["m"].double(), want["m"], rtol=1e-5, atol=1e-8) and torch.allclose(got["v"].double(), want["v"], rtol=1e-5, atol=1e-10)
        # 2 steps of 1e-3 times root mean square 0.2, one in a hundred off at most
        assert (got["master"].double() - want["master"]).norm() <= 1e-2 * 2 * 1e-3 * 0.2 * math.sqrt(u.n) + 1e-6 * want["master"].norm()
        copy = u.p_shard if u.p_shard is not None else u.host_p
        assert torch.equal(copy.float().cpu(), got["master"].bfloat16().float())


@pytest.mark.gpu
@pytest.mark.parametrize("model,more", MODELS)
def test_a_packed_job_on_the_gpu(model, more):
    """Loss and gradients of a packed batch through the kernels against the documents one by one in fp32, then steps with Muon."""
    heads = {"heads": 4, "hidden": 256} if model == "toygpt" else {}
    d = tiny_cfg(ONE, seq=128, vocab=512, model_name=model, reduce_dtype="float32", autocast_dtype="bfloat16")
    cfg, ov = parse_pipeline_dict(d), {"layers": 2, **heads, **more}
    tr = Trainer(cfg, TrainerOptions(schedule="1f1b", model_overrides=ov, lr=0.0, documents=40))
    batch = tr.synthetic_batch()
    loss, grads = _one_by_one(parse_pipeline_dict({**d, "autocast_dtype": "float32"}), ov, {k: t.clone() for k, t in batch.items()},
                              [u.p_shard.float().cpu() for u in tr.stages[0].engine.units])
    assert tr.train_step_from_host(batch) == pytest.approx(loss, rel=2e-3)
    for u, want in zip(tr.stages[0].engine.units, grads):
        got = u.m[:want.numel()].cpu() / 0.1
        # activations and their gradients are rounded to bf16 (2^-8) some ten times a block on the way through two blocks and back
        assert (got - want).norm() <= 40 * 2.0 ** -8 / 4 * want.norm(), u.layer.kind
    tr.check_kernels()
    tr = Trainer(cfg, TrainerOptions(schedule="1f1b", model_overrides=ov, optimizer="muon", lr=1e-3, weight_decay=0.1, documents=40))
    losses = [tr.train_step_from_host(batch) for _ in range(3)]
    assert all(math.isfinite(x) for x in losses) and len(set(losses)) == 3
    tr.check_kernels()
