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
