"""Checkpoints of a model that is not the job's: refused at every tensor-parallel width, by name."""
import json
import os

import pytest
import torch

from dist_utils import run_workers
from test_dist_cpu import tiny_cfg
from zorse_b200.ckpt.reader import CheckpointError, load_checkpoint
from zorse_b200.ckpt.writer import save_checkpoint
from zorse_b200.config.training_config import parse_pipeline_dict
from zorse_b200.trainer import Trainer, TrainerOptions

ONE = [{"gpu_ranks": [0], "num_microbatches_per_rank": [4], "layer_partition": [0, 4], "zero_config": [[0]]}]
CFG = tiny_cfg(ONE)
TP2 = tiny_cfg(ONE, tensor_parallel_size=2)


def _job(**options):
    return Trainer(parse_pipeline_dict(CFG), TrainerOptions(ops="ref", **options))


def _save(directory, **options):
    tr = _job(**options)
    tr.train_step_from_host(tr.synthetic_batch())
    return save_checkpoint(tr, str(directory), 1), [u.full_master() for st in tr.stages for u in st.engine.units]


def _without_record(ck):
    """As checkpoints were before they held the model: sizes alone have to tell."""
    path = os.path.join(ck, "meta.json")
    with open(path) as f:
        meta = json.load(f)
    for key in ("model", "optimizer", "weight_decay", "moment_bits"):
        meta.pop(key, None)
    with open(path, "w") as f:
        json.dump(meta, f)


def _load_tp(rank, world, ck, options):
    tr = Trainer(parse_pipeline_dict(TP2), TrainerOptions(backend="gloo", **options))
    try:
        load_checkpoint(tr, ck)
    except CheckpointError as e:
        return str(e)
    lay = tr.stages[0].engine.units[1].layer.layout()[0]
    o, shape = lay["norm2_w"]
    return tr.stages[0].engine.units[1].full_master()[o:o + shape[0]].clone()


@pytest.mark.parametrize("saved,job", [(True, False), (False, True)])
def test_another_layout_is_refused_at_every_width(tmp_path, saved, job):
    ck, _ = _save(tmp_path, model_overrides={"qk_norm": saved})
    _without_record(ck)
    with pytest.raises(CheckpointError, match="elements saved"):
        load_checkpoint(_job(model_overrides={"qk_norm": job}), ck)
    for message in run_workers(2, _load_tp, ck, {"model_overrides": {"qk_norm": job}}):
        assert isinstance(message, str) and "elements saved" in message


def test_the_same_model_loads_at_another_width_without_a_record(tmp_path):
    ck, masters = _save(tmp_path, model_overrides={"qk_norm": True})
    _without_record(ck)
    tr = _job(model_overrides={"qk_norm": True})
    o, shape = tr.stages[0].engine.units[1].layer.layout()[0]["norm2_w"]
    for got in run_workers(2, _load_tp, ck, {"model_overrides": {"qk_norm": True}}):
        assert torch.equal(got, masters[1][o:o + shape[0]])


def test_a_slice_that_is_not_there_is_named(tmp_path):
    ck, _ = _save(tmp_path)
    path = os.path.join(ck, "meta.json")
    with open(path) as f:
        meta = json.load(f)
    meta["tensor_parallel_size"] = 2           # slice 0 only, and of another size
    with open(path, "w") as f:
        json.dump(meta, f)
    with pytest.raises(CheckpointError, match="unit 1"):
        load_checkpoint(_job(), ck)


@pytest.mark.parametrize("saved,job,name", [
    ({"embed_scale": 3.0}, {}, "embed_scale"), ({}, {"embed_scale": 3.0}, "embed_scale"), ({"embed_scale": 3.0}, {"embed_scale": 2.0}, "embed_scale"),
    ({"qk_norm": True}, {}, "qk_norm"), ({"window": 16}, {}, "window"), ({}, {"rope_theta": 500000.0}, "rope_theta")])
def test_another_model_is_refused_by_name(tmp_path, saved, job, name):
    ck, _ = _save(tmp_path, model_overrides=saved)
    with pytest.raises(CheckpointError, match=name):
        load_checkpoint(_job(model_overrides=job), ck)
    load_checkpoint(_job(model_overrides=saved), ck)


@pytest.mark.parametrize("job", [{}, {"embed_scale": 2.0}])
def test_another_model_is_refused_at_another_width(tmp_path, job):
    ck, _ = _save(tmp_path, model_overrides={"embed_scale": 3.0})
    for message in run_workers(2, _load_tp, ck, {"model_overrides": job}):
        assert isinstance(message, str) and "embed_scale" in message


def test_another_optimizer_is_refused_and_other_bits_are_not(tmp_path):
    ck, _ = _save(tmp_path, optimizer="adamw", moment_bits=8, weight_decay=0.1)
    with pytest.raises(CheckpointError, match="optimizer"):
        load_checkpoint(_job(), ck)
    for bits in (8, 32):
        assert load_checkpoint(_job(optimizer="adamw", moment_bits=bits), ck) == 1
    with open(os.path.join(ck, "meta.json")) as f:
        meta = json.load(f)
    assert (meta["optimizer"], meta["moment_bits"], meta["weight_decay"]) == ("adamw", 8, 0.1)


def test_what_changes_no_result_may_change(tmp_path):
    ck, _ = _save(tmp_path)
    assert load_checkpoint(_job(model_overrides={"embed_by_token": True, "init_std": 0.5}), ck) == 1


def test_a_checkpoint_without_the_record_loads(tmp_path):
    ck, masters = _save(tmp_path, model_overrides={"embed_scale": 3.0}, optimizer="adamw")
    _without_record(ck)
    tr = _job()
    assert load_checkpoint(tr, ck) == 1
    assert all(torch.equal(u.full_master(), m) for u, m in zip(tr.stages[0].engine.units, masters))


def test_the_recovery_command_has_the_flags(tmp_path):
    from zorse_b200.ckpt.reader import flags_of, read_meta
    from zorse_b200.cli.train import model_overrides
    from zorse_b200.config.flags import parse_args_zorse

    config = tmp_path / "c.json"
    config.write_text(json.dumps(CFG))
    for ov, options in (({}, {}), ({"qk_norm": True, "embed_scale": 22.627417, "embed_by_token": True},
                                   dict(optimizer="adamw", weight_decay=0.05, moment_bits=8))):
        ck, _ = _save(tmp_path / str(len(ov)), model_overrides=ov, **options)
        flags = flags_of(read_meta(ck))
        assert bool(flags) == bool(ov)
        a = parse_args_zorse(["--config_file", str(config), *flags])
        assert model_overrides(a) == ov
        assert (a.optimizer, a.weight_decay, a.moment_bits) == tuple({**dict(optimizer="adam", weight_decay=0.0, moment_bits=32), **options}.values())
        load_checkpoint(_job(model_overrides=model_overrides(a), optimizer=a.optimizer, moment_bits=a.moment_bits), ck)
