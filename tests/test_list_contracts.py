"""What the list passes and FlatAdamW promise around the arithmetic, as far as it can be checked without a GPU: which
tensors they take for what."""

import types
import weakref

import pytest
import torch

from yafsdp_amd import optim
from yafsdp_amd._common import FSDPMeshInfo
from yafsdp_amd._layout import RaggedShard
from yafsdp_amd._tensor import RaggedShardDTensor, RaggedShardSpec
from torch.distributed.tensor._dtensor_spec import TensorMeta

from ext_subclasses import Int8Master
from list_subclasses import OwnStorage, PairTensor


def _sharded(local, kind="", owner=None):
    meta = TensorMeta(torch.Size((2, 3)), (3, 1), torch.float32)
    placement = RaggedShard(local_numel=6, global_offset=0, shard_numels=(6,))
    spec = RaggedShardSpec(FSDPMeshInfo(1, 0), (placement,), meta, None if owner is None else weakref.ref(owner), kind)
    return RaggedShardDTensor(local, spec, requires_grad=False)


# ---- tensor subclasses -----------------------------------------------------------------------------------------
def test_what_a_list_takes_a_tensor_for():
    plain = torch.arange(6.0)
    for t in (plain, torch.nn.Parameter(plain), None, 3.0):
        assert optim._resolve(t) is t
    assert optim._resolve(_sharded(plain)) is plain
    # the group's own fragment of a tensor-subclass parameter: the first inner tensor, whatever else the subclass holds
    owner = torch.nn.Module()
    assert optim._resolve(_sharded(PairTensor(plain, plain + 1), "param", owner)) is plain
    # made from it by an op: only where one inner tensor holds all values
    assert optim._resolve(_sharded(Int8Master(plain))) is plain
    with pytest.raises(TypeError, match="PairTensor keeps its values"):
        optim._resolve(_sharded(PairTensor(plain, plain + 1)))
    own = plain.as_subclass(OwnStorage)
    assert optim._resolve(own) is own  # its elements are its own memory, whatever its attributes are


@pytest.mark.parametrize("make", [lambda: PairTensor(torch.ones(4), torch.ones(4), "cuda"), lambda: Int8Master(torch.ones(4))])
def test_wrappers_from_elsewhere_are_refused(make):
    """Not read as their first inner tensor: half of a value, or a value in another scale."""
    for call in (lambda ts: optim.list_grad_norm(ts), lambda ts: optim.list_clip_coef(ts, 1.0),
                 lambda ts: optim.list_clip_grad_norm_(ts, 1.0), lambda ts: optim.list_adamw_step(ts, ts, ts, ts, step=1)):
        with pytest.raises(TypeError, match="keeps its values in other tensors"):
            call([make()])


def _plain_units(params, grads, steps):
    """What FlatAdamW keeps of parameters outside any group."""
    units = []
    for p, g, s in zip(params, grads, steps):
        p.grad = g
        units.append(types.SimpleNamespace(group=None, params=[p], steps=[s], device=p.device,
                                           exp_avg=torch.zeros(p.numel()), exp_avg_sq=torch.zeros(p.numel())))
    return units


HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, decoupled=True)


def test_flat_adamw_refuses_a_wrapper_from_elsewhere():
    opt = object.__new__(optim.FlatAdamW)
    p, g = (PairTensor(torch.ones(4), torch.ones(4), "cuda") for _ in range(2))
    units = _plain_units([p], [g], [0])
    with pytest.raises(TypeError, match="keeps its values in other tensors"):
        opt._step_plain(units, HYPER, None, False)
