"""What the list passes and FlatAdamW promise around the arithmetic, as far as it can be checked without a GPU: which
tensors they take for what, which memory a call may share, what a
refused step leaves, where a gradient scale may lie, in which order parameters are stepped."""

import types
import weakref

import numpy as np
import pytest
import torch

from yafsdp_amd import _native, optim
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


# ---- the workspace ---------------------------------------------------------------------------------------------
OVERLAP = -9
AT = 0x100000  # of the workspace; every call below is refused before anything reads its addresses


def _norm(rows, clip, out=0x20000):
    fn = _native.lib.yafsdp_list_clip if clip else _native.lib.yafsdp_list_norm
    buf = np.array([(*r, 0) for r in rows], dtype=_native._LIST_ENTRY).tobytes()
    return fn(buf, len(rows), 2, 1.0, AT, _native.lib.yafsdp_list_workspace_bytes(len(rows)) + 0x1000, out, None)


def _scale(rows, coef=0x20000):
    buf = np.array([(*r, 0) for r in rows], dtype=_native._LIST_ENTRY).tobytes()
    return _native.lib.yafsdp_list_scale(buf, len(rows), coef, AT,
                                         _native.lib.yafsdp_list_workspace_bytes(len(rows)) + 0x1000, None)


def _adamw(rows, out=0, scale=None):
    buf = np.array(rows, dtype=_native._ADAMW_ENTRY).tobytes()
    return _native.lib.yafsdp_list_adamw(buf, len(rows), 1, out, 1e-3, 0.9, 0.95, 1e-8, 0.1, 1, scale, 1, AT,
                                         _native.lib.yafsdp_list_adamw_workspace_bytes(len(rows)) + 0x1000, None)


@pytest.mark.parametrize("count", [1, 400])  # partial sums only; with a list behind them
def test_memory_inside_the_workspace_is_refused(count):
    """Partial sums and staged lists are written there: a result, a coefficient or a tensor of the list would be
    overwritten, or read half before and half after."""
    used = _native.lib.yafsdp_list_workspace_bytes(count)
    rows = [(0x1000000 + 0x100 * i, 4, 1) for i in range(count)]
    for at in (AT - 4, AT, AT + 8, AT + used - 4):
        assert _norm(rows, True, out=at) == OVERLAP and _norm(rows, False, out=at) == OVERLAP, hex(at)
    for at in (AT, AT + 64, AT + used - 4):
        assert _scale(rows, coef=at) == OVERLAP
    for at, n in ((AT - 14, 8), (AT, 8), (AT + used - 2, 1), (AT - 0x1000, 0x100000)):
        inside = [*rows[1:], (at, n, 1)]
        assert [_norm(inside, True), _norm(inside, False), _scale(inside)] == [OVERLAP] * 3, hex(at)
    assert "workspace" in _native.error_string(OVERLAP)


def test_memory_inside_the_workspace_of_adamw_is_refused():
    used = _native.lib.yafsdp_list_adamw_workspace_bytes(100)
    rows = [tuple(0x1000000 * k + 0x100 * i for k in range(1, 6)) + (8,) for i in range(100)]
    for at in (AT, AT + used - 4):
        assert _adamw(rows, scale=at) == OVERLAP
        for k in range(5):  # the gradients too, which are only read
            assert _adamw(rows[1:] + [(*rows[0][:k], at, *rows[0][k + 1:])], out=2) == OVERLAP, k


# ---- step counts -----------------------------------------------------------------------------------------------
def test_a_refused_step_leaves_the_counts(monkeypatch):
    """Counts advance with the launch that steps their parameters: a list at a time, or one at a time where memory is
    shared."""
    opt = object.__new__(optim.FlatAdamW)
    steps = [3, 3, 0, 7]
    params = [torch.ones(4) for _ in steps]

    def refuse(*args, step, **kwargs):
        if step == bad:
            raise TypeError("refused")
        return shared is None

    def refuse_one(p, *args, **kwargs):
        if p.data_ptr() == params[shared].data_ptr():
            raise TypeError("refused")

    monkeypatch.setattr(_native, "list_adamw", refuse)
    monkeypatch.setattr(_native, "adamw_step", refuse_one)
    for bad, shared, after in ((4, None, [3, 3, 0, 7]), (1, None, [4, 4, 0, 7]), (8, None, [4, 4, 1, 7]),
                               (None, 0, [3, 3, 0, 7]), (None, 1, [4, 3, 0, 7]), (None, 3, [4, 4, 1, 7])):
        units = _plain_units(params, [torch.ones(4) for _ in params], steps)
        with pytest.raises(TypeError, match="refused"):
            opt._step_plain(units, HYPER, None, False)
        assert [u.steps[0] for u in units] == after, (bad, shared)
    bad = shared = None
    units = _plain_units(params, [torch.ones(4), None, torch.ones(4), torch.ones(4)], steps)
    opt._step_plain(units, HYPER, None, False)
    assert [u.steps[0] for u in units] == [4, 3, 1, 8]


# ---- a gradient scale in memory that the step writes -------------------------------------------------------------
def _shares(a, b):
    lo, hi = a.data_ptr(), a.data_ptr() + 4 * a.numel()
    return lo < b.data_ptr() + 4 * b.numel() and b.data_ptr() < hi


def _stand_ins(monkeypatch, calls):
    """The two native calls on CPU tensors with p -= scale * g as the step: the scale is read when a launch runs, and a
    list is refused where what it writes shares memory."""

    def one(p, g, m, v, out16=None, *, grad_scale, zero_grad, **kwargs):
        p.sub_(grad_scale.clone() * g)
        if zero_grad:
            g.zero_()

    def many(ps, gs, ms, vs, outs, resolve, *, grad_scale, zero_grad, **kwargs):
        written = [*ps, *ms, *vs, *(gs if zero_grad else ())]
        pairs = [(a, b) for i, a in enumerate(written) for b in written[:i]] + [(a, grad_scale) for a in written]
        calls.append(not any(_shares(a, b) for a, b in pairs))
        if calls[-1]:
            for p, g, m, v in zip(ps, gs, ms, vs):
                one(p, g, m, v, grad_scale=grad_scale, zero_grad=zero_grad)
        return calls[-1]

    monkeypatch.setattr(_native, "list_adamw", many)
    monkeypatch.setattr(_native, "adamw_step", one)


@pytest.mark.parametrize("where", ["gradient", "parameter", "elsewhere"])
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("steps", [[0, 0, 0], [1, 0, 0], [0, 1, 2]])
@torch.no_grad()
def test_a_scale_inside_what_the_step_writes(monkeypatch, where, shared, steps):
    """Every parameter is stepped with the value from before the step."""
    calls = []
    _stand_ins(monkeypatch, calls)
    base = torch.arange(12.0) + 1
    params = [base[:4], base[4:8], base[6:10] if shared else base[8:]]
    grads = [torch.full((4,), 0.5) for _ in params]
    scale = {"gradient": grads[0][1:2], "parameter": params[0][2:3], "elsewhere": torch.tensor([0.5])}[where]
    want, value = base.clone(), float(scale)
    for p, g in zip(params, grads):
        want[p.storage_offset():p.storage_offset() + 4] -= value * 0.5
    opt = object.__new__(optim.FlatAdamW)
    after = opt._step_plain(_plain_units(params, grads, steps), HYPER, scale, True)
    assert torch.equal(base, want)
    assert all(not g.any() for g in grads) and float(after) == value
    assert (after is scale) == (where == "elsewhere")
    if where == "elsewhere" and not shared:
        assert calls == [True] * len(set(steps))


def test_a_scale_without_memory_of_its_own_is_refused():
    """Its address is 0, which the library takes for "no scale"."""
    scale = PairTensor(torch.full((1,), 0.5), torch.full((1,), 0.5), "cuda")
    four = [[torch.zeros(2)] for _ in range(4)]
    with pytest.raises(TypeError, match="grad_scale must hold its value"):
        optim.list_adamw_step(*four, step=1, grad_scale=scale)
    with pytest.raises(TypeError, match="coef must hold its value"):
        optim.list_scale_grads_(four[0], scale)


# ---- order -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("steps", [[0, 0, 0, 0], [1, 0, 1, 0], [2, 1, 0, 3]])
@pytest.mark.parametrize("what", ["nothing", "parameters", "gradients", "gradients that are read"])
@torch.no_grad()
def test_memory_shared_across_step_counts_keeps_the_lists_order(monkeypatch, steps, what):
    """Parameters (or zero-filled gradients) that share memory are stepped in the list's order whatever their counts;
    others go in one pass per count."""
    _stand_ins(monkeypatch, [])
    order, many = [], _native.list_adamw
    base = torch.arange(16.0)
    params = [base[k:k + 5] if what == "parameters" else base[4 * k:4 * k + 4] for k in range(4)]
    shared = torch.ones(4)
    grads = [shared if what.startswith("gradients") else torch.ones(p.numel()) for p in params]
    at = [p.data_ptr() for p in params]

    def watch(ps, *args, **kwargs):
        taken = many(ps, *args, **kwargs)
        order.extend([at.index(p.data_ptr()) for p in ps] if taken else ())
        return taken

    def watch_one(p, *args, **kwargs):
        order.append(at.index(p.data_ptr()))

    monkeypatch.setattr(_native, "list_adamw", watch)
    monkeypatch.setattr(_native, "adamw_step", watch_one)
    units = _plain_units(params, grads, steps)
    object.__new__(optim.FlatAdamW)._step_plain(units, HYPER, torch.tensor([0.5]), what != "gradients that are read")
    if what in ("parameters", "gradients"):
        assert order == [0, 1, 2, 3]
    else:
        assert order == sorted(range(4), key=lambda k: (steps.index(steps[k]), k))
    assert [u.steps[0] for u in units] == [s + 1 for s in steps]


@pytest.mark.parametrize("helper", [True, False])
def test_any_shared(helper, monkeypatch):
    if helper:
        tl = pytest.importorskip("yafsdp_amd._tensorlist")
        assert tl.any_shared([torch.zeros(2), torch.zeros(8)[::2]]) is None  # handed back: not dense, not plain
        assert tl.any_shared([Int8Master(torch.zeros(2))]) is None and tl.any_shared(iter([])) is None
    else:
        monkeypatch.setattr(_native, "_tensorlist", None)
    base = torch.zeros(100)
    far, half = torch.zeros(5), torch.zeros(6, dtype=torch.bfloat16)
    cut = lambda *spans: [base[a:b] for a, b in spans]
    for tensors, shared in ((cut((50, 60), (0, 10), (10, 50)), False), (cut((50, 60), (0, 10), (9, 50)), True),
                            (cut((0, 100), (30, 40)), True), ([base, base], True), ([], False), ([far, half, base], False),
                            ([half, half[5:]], True), ([half[:5], half[5:]], False), (cut((3, 3), (0, 10), (3, 3)), False),
                            ([base.view(10, 10).t(), torch.nn.Parameter(base[99:])], True)):
        assert _native.any_shared(tensors) is shared
    assert not _native.any_shared([PairTensor(far, far, "cuda"), Int8Master(far)])  # no memory of their own
