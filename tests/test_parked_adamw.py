"""AdamW behind the backward pass with parked parameters: the engine's units step one by one, with the same result as resident ones."""
import pytest
import torch

from zorse_b200.engine.zero import AdamConfig, EngineConfig, StageEngine
from zorse_b200.models import registry
from zorse_b200.ops.api import get_ops
from zorse_b200.parallel.groups import Group


def _engine(device, offload, bits, decoupled=True):
    spec = registry.get_spec("tiny_llama", vocab=512, layers=2)
    layers = [registry.make_embedding(spec, 32)] + [registry.make_block(spec) for _ in range(2)]
    on_gpu = device == "cuda"
    cfg = EngineConfig(compute_dtype=torch.bfloat16 if on_gpu else torch.float32, offload_params=offload,
                       adam=AdamConfig(decoupled=decoupled, moment_bits=bits, weight_decay=0.1))
    one = Group(ranks=(0,), pg=None)
    return StageEngine(layers, [0, 1, 2], device=torch.device("cuda", 0) if on_gpu else torch.device("cpu"), cfg=cfg,
                       ops=get_ops("sm100" if on_gpu else "ref"), shard=one, replicate=one, rank=0)


def _steps(engine, n=2):
    for k in range(n):
        for i, u in enumerate(engine.units):
            u.grad_views()
            u.grad.copy_(torch.randn(u.n, generator=torch.Generator().manual_seed(10 * k + i)))
            u.reduce_grads()
        engine.optimizer_step()
        engine.finish_step()
    if engine.device.type == "cuda":
        torch.cuda.synchronize()
    return [t.detach().float().cpu().clone() for u in engine.units for t in u.state_tensors().values()]


def _same(device, bits, decoupled=True):
    here, parked = _engine(device, False, bits, decoupled), _engine(device, True, bits, decoupled)
    for a, b in zip(_steps(here), _steps(parked)):
        assert torch.equal(a, b)
    for a, b in zip(here.units, parked.units):
        assert a.step_count == b.step_count == 2 and b.master is None
        assert torch.equal(a.p_shard.float().cpu(), b.host_p.float())


@pytest.mark.parametrize("bits,decoupled", [(32, True), (8, True), (32, False)])
def test_parked_parameters_step_as_resident_ones_cpu(bits, decoupled):
    _same("cpu", bits, decoupled)


@pytest.mark.gpu
@pytest.mark.parametrize("bits,decoupled", [(32, True), (8, True), (32, False)])
def test_parked_parameters_step_as_resident_ones(bits, decoupled):
    _same("cuda", bits, decoupled)
