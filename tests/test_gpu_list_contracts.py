"""What the list passes and FlatAdamW promise around the arithmetic, on the GPU: which tensors they take for what,
what a refused step leaves, where a gradient scale may lie."""

import pytest
import torch
import torch.nn as nn

from ext_subclasses import Int8Master
from helpers import assert_bits_equal, loc
from list_subclasses import OwnStorage, PairTensor

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32 = torch.float32
HP = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


# ---- tensor subclasses -----------------------------------------------------------------------------------------
def test_wrappers_from_elsewhere_are_refused_and_left_alone():
    from yafsdp_amd.optim import FlatAdamW, list_adamw_step, list_clip_grad_norm_, list_scale_grads_

    gen = torch.Generator(device=DEV).manual_seed(1)
    halves = [torch.randn(100, device=DEV, generator=gen) for _ in range(4)]
    before = [t.clone() for t in halves]
    p, g = nn.Parameter(PairTensor(*halves[:2])), PairTensor(*halves[2:])
    p.grad = g
    plain = nn.Parameter(torch.ones(7, device=DEV))
    plain.grad = torch.ones(7, device=DEV)
    m, v = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    opt = FlatAdamW([plain, p], **HP)
    for call in (lambda: list_clip_grad_norm_([plain.grad, g], 1e-3),
                 lambda: list_scale_grads_([g], torch.full((1,), 0.5, device=DEV)),
                 lambda: list_adamw_step([p], [g], [m], [v], step=1), lambda: opt.step()):
        with pytest.raises(TypeError, match="PairTensor keeps its values in other tensors"):
            call()
    for t, b in zip(halves, before):
        assert_bits_equal(t, b, "a refused call writes nothing")
    assert_bits_equal(plain, torch.ones(7), "nor any other tensor of its list")


def test_subclass_with_elements_of_its_own():
    from yafsdp_amd.optim import FlatAdamW, list_clip_grad_norm_

    gen = torch.Generator(device=DEV).manual_seed(2)
    base, grad = (torch.randn(300, device=DEV, generator=gen) for _ in range(2))
    out = []
    for cls in (OwnStorage, torch.Tensor):
        p = base.clone().as_subclass(cls).requires_grad_()
        p.grad = grad.clone().as_subclass(cls)
        norm = list_clip_grad_norm_([p.grad], 0.5)
        FlatAdamW([p], **HP).step()
        out.append([x.as_subclass(torch.Tensor).detach() for x in (norm, p.grad, p)])
    for a, b in zip(*out):
        assert_bits_equal(a, b, "subclass and plain tensor")


def test_fragments_of_sharded_subclass_parameters():
    """Parameters, gradients and states of a group whose parameters are a tensor subclass: the fragments' values."""
    from yafsdp_amd import FSDPMeshInfo, MixedPrecisionPolicy
    from yafsdp_amd._param_group import YaFSDPParamGroup, init_shared_state
    from yafsdp_amd.optim import list_adamw_step, list_clip_grad_norm_

    gen = torch.Generator().manual_seed(3)
    values = [torch.randn(s, generator=gen) * 0.08 for s in ((33, 7), (5, 13), (1000,))]
    policy = MixedPrecisionPolicy(param_dtype=torch.bfloat16, all_gather_dtype_to_param_cls={torch.int8: Int8Master})
    group = YaFSDPParamGroup([nn.Parameter(Int8Master(v.to(DEV))) for v in values], FSDPMeshInfo(2, 1), DEV, policy, 8)
    init_shared_state([group], DEV)
    fps = [fp for fp in group._all_gather_dtype_to_fsdp_params[torch.int8] if fp.sharded_numel]
    assert fps
    for fp in fps:
        fp.sharded_param_grad._local_tensor.copy_(torch.randn(fp.sharded_numel, generator=gen))
    params, grads = [fp.sharded_param for fp in fps], [fp.sharded_param_grad for fp in fps]
    plain = [[fp._sharded_param_data.clone() for fp in fps], [g._local_tensor.clone() for g in grads]]
    states = [[torch.zeros_like(p.detach()) for p in params] for _ in range(2)]
    assert isinstance(states[0][0]._local_tensor, Int8Master)
    plain += [[torch.zeros_like(p) for p in plain[0]] for _ in range(2)]
    norms = [list_clip_grad_norm_(g, 0.5) for g in (grads, plain[1])]
    assert_bits_equal(norms[0], norms[1], "norm")
    list_adamw_step(params, grads, *states, step=1, **HP)
    list_adamw_step(*plain, step=1, **HP)
    for k, fp in enumerate(fps):
        got = (fp._sharded_param_data, grads[k]._local_tensor, *(s[k]._local_tensor._data for s in states))
        for a, b in zip(got, (x[k] for x in plain)):
            assert_bits_equal(a, b, f"fragment {k}")


# ---- FlatAdamW -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sharded", [False, True])
def test_a_step_that_is_refused_can_be_made_again(sharded):
    """Bits and counts of a run in which every step is first refused are those of a run without refusals."""
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd.optim import FlatAdamW

    runs = []
    for refused in (False, True):
        gen = torch.Generator(device=DEV).manual_seed(5)
        model = nn.Module()
        for i, n in enumerate((100, 7, 2049)):
            model.register_parameter(f"p{i}", nn.Parameter(torch.randn(n, device=DEV, generator=gen)))
        if sharded:
            fully_shard(model, mesh=(1, 0), mp_policy=MixedPrecisionPolicy(param_dtype=torch.bfloat16))
        params = list(model.parameters())
        opt = FlatAdamW(params, **HP)
        for it in range(3):
            for p in params[it == 1:]:
                fresh = torch.randn(p.numel(), device=DEV, generator=gen)
                if sharded:
                    p.grad = p._yafsdp_param().sharded_param_grad
                    p.grad._local_tensor.copy_(fresh)
                else:
                    p.grad = fresh
            if it == 1:
                params[0].grad = None
            if refused:
                before = [loc(p).detach().clone() for p in params]
                with pytest.raises(TypeError, match="grad_scale"):
                    opt.step(grad_scale=torch.ones(1, device=DEV, dtype=torch.float64))
                with pytest.raises(RuntimeError, match="grad_scale"):
                    opt.step(grad_scale=torch.ones(1))
                for p, b in zip(params, before):
                    assert_bits_equal(loc(p).detach(), b, "a refused step writes nothing")
            opt.step()
        runs.append([loc(p).detach() for p in params])
        assert [int(s["step"]) for s in opt.state_dict()["state"].values()] == [2, 3, 3]
    for a, b in zip(*runs):
        assert_bits_equal(a, b, "with and without refused steps")


def _net(gen):
    model = nn.Module()
    model.inner = nn.Module()
    for module, name, n in ((model.inner, "a", 300), (model.inner, "b", 77), (model, "c", 100), (model, "d", 513)):
        module.register_parameter(name, nn.Parameter(torch.randn(n, device=DEV, generator=gen)))
    return model


@pytest.mark.parametrize("where", ["c", "inner.b"])
@pytest.mark.parametrize("kind", ["gradient", "parameter"])
@pytest.mark.parametrize("late", [False, True])
def test_a_scale_inside_what_the_step_writes(where, kind, late):
    """Sharded and plain parameters are all stepped with the value from before the step; with ``late``, one plain
    parameter's count is behind, so that it is stepped by a launch of its own."""
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd.optim import FlatAdamW

    runs = []
    for apart in (True, False):
        gen = torch.Generator(device=DEV).manual_seed(6)
        model = _net(gen)
        fully_shard(model.inner, mesh=(1, 0), mp_policy=MixedPrecisionPolicy(param_dtype=torch.bfloat16))
        named = dict(model.named_parameters())
        opt = FlatAdamW(named.values(), **HP)
        for it in range(2):
            for name, p in named.items():
                fresh = torch.randn(loc(p).numel(), device=DEV, generator=gen)
                if "inner" in name:
                    p.grad = p._yafsdp_param().sharded_param_grad
                    p.grad._local_tensor.copy_(fresh)
                else:
                    p.grad = None if late and it == 0 and name == "d" else fresh
            p = named[where]
            scale = loc(p.grad if kind == "gradient" else p)[5:6]
            with torch.no_grad():
                scale.fill_(0.375)
            opt.step(grad_scale=scale.clone() if apart else scale, zero_grad=True)
            assert all(p.grad is None or not loc(p.grad).any() for p in named.values())
        runs.append([loc(p).clone() for p in named.values()])
    for name, a, b in zip(named, *runs):
        assert_bits_equal(a, b, f"{name}: scale apart and in the {kind} of {where}")


@pytest.mark.parametrize("make", [
    lambda: PairTensor(*(torch.full((1,), 0.5, device=DEV) for _ in range(2))),
    lambda: torch._efficientzerotensor(1, device=DEV),
    lambda: torch.full((1,), 0.5j, device=DEV, dtype=torch.complex64).conj().imag,
])
def test_a_scale_without_a_value_in_memory_is_refused(make):
    """A wrapper and a zero without storage (address 0, "no scale" to the library); a lazily negated view (the other sign
    in memory)."""
    from yafsdp_amd import _native
    from yafsdp_amd.optim import FlatAdamW, list_adamw_step, list_scale_grads_

    p, g, m, v = (torch.ones(10, device=DEV) for _ in range(4))
    param = nn.Parameter(p)
    param.grad = g
    opt = FlatAdamW([param], **HP)
    for call in (lambda c: list_adamw_step([p], [g], [m], [v], step=1, grad_scale=c), lambda c: opt.step(grad_scale=c),
                 lambda c: list_scale_grads_([g], c), lambda c: _native.flat_scale(g, c),
                 lambda c: _native.adamw_step(p, g, m, v, None, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8,
                                              weight_decay=0.0, step=1, grad_scale=c)):
        with pytest.raises(TypeError, match="must hold its value in memory"):
            call(make())
    for t in (p, g, m, v):
        assert_bits_equal(t, torch.ones(10), "a refused call writes nothing")


# ---- an older error of the thread --------------------------------------------------------------------------------
@pytest.mark.parametrize("count", [3, 400])  # in the kernel arguments, through a staging slot
def test_an_error_of_an_earlier_call_is_not_the_launches(count):
    """A HIP error that another call of the thread left behind: the list calls report their own launches' status, run to
    their end and leave it for whoever asks.  More calls than staging slots, none of which may be given up early."""
    from yafsdp_amd import _native
    from yafsdp_amd.optim import list_clip_coef

    lib = _native.lib
    lists = [[torch.full((5 + k,), float(k + 1), device=DEV) for _ in range(count)] for k in range(40)]
    want = [torch.stack(list_clip_coef(ts, 1.0)) for ts in lists]
    entries = [_native.TensorList(ts) for ts in lists]
    nbytes = lib.yafsdp_list_workspace_bytes(count)
    workspaces = [torch.empty(nbytes, dtype=torch.uint8, device=DEV) for _ in lists]
    got = torch.zeros(len(lists), 2, device=DEV)
    torch.cuda.synchronize()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.hipPeekAtLastError() == 0
    older = lib.hipSetDevice(1 << 20)
    assert older != 0 and lib.hipPeekAtLastError() == older
    codes = [lib.yafsdp_list_norm(e.entries, e.count, 2, 1.0, w.data_ptr(), nbytes, got[k].data_ptr(), stream)
             for k, (e, w) in enumerate(zip(entries, workspaces))]
    left = lib.hipGetLastError()
    torch.cuda.synchronize()
    assert codes == [0] * len(lists) and left == older
    assert_bits_equal(got, torch.stack(want), "norms and coefficients")


# ---- order -----------------------------------------------------------------------------------------------------
def test_shared_memory_across_step_counts():
    """Three parameters on one storage, the middle one a step behind: stepped in the list's order, as one launch per
    parameter steps them."""
    from oracle import cref
    from yafsdp_amd.optim import FlatAdamW

    chp = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
    gen = torch.Generator().manual_seed(8)
    want = torch.randn(100, generator=gen)
    base = want.to(DEV)
    cuts = [slice(0, 60), slice(40, 90), slice(72, 100)]
    params = [nn.Parameter(base[c]) for c in cuts]
    state = [[torch.zeros(c.stop - c.start) for c in cuts] for _ in range(2)]
    opt, counts = FlatAdamW(params, **HP), [0, 0, 0]
    for it in range(3):
        for k, (p, c) in enumerate(zip(params, cuts)):
            g = torch.randn(c.stop - c.start, generator=gen)
            p.grad = None if (it, k) == (0, 1) else g.to(DEV)
            if p.grad is not None:
                counts[k] += 1
                part = want[c].clone()
                cref.adamw_step(part, g, state[0][k], state[1][k], None, step=counts[k], **chp)
                want[c] = part
        opt.step()
        assert_bits_equal(base, want, f"after step {it}")


# ---- one norm over the ranks -------------------------------------------------------------------------------------
def test_norm_of_fragments_and_replicated_gradients_joined_over_ranks():
    """Two logical ranks of a model with sharded and replicated parameters: the squares of the fragments' norms are summed
    over the ranks, those of the replicated gradients counted once; every rank clips by the coefficient of the whole
    gradient.  Each of the six roundings to binary32 on the way is off by at most 2^-24 of the norm."""
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd._tensor import RaggedShardDTensor
    from yafsdp_amd.optim import list_grad_norm, list_scale_grads_

    max_norm, squares, ranks, whole = 0.5, [], [], None
    for rank in range(2):
        gen = torch.Generator(device=DEV).manual_seed(9)
        model = _net(gen)
        full = {k: torch.randn(p.shape, device=DEV, generator=gen) for k, p in model.named_parameters()}
        whole = torch.cat([g.view(-1) for g in full.values()]).double()
        fully_shard(model.inner, mesh=(2, rank), mp_policy=MixedPrecisionPolicy(param_dtype=torch.bfloat16))
        for name, p in model.named_parameters():
            if isinstance(p, RaggedShardDTensor):
                p.grad = p._yafsdp_param().sharded_param_grad
                at = p.placements[0]
                p.grad._local_tensor.copy_(full[name][at.global_offset:at.global_offset + at.local_numel])
            else:
                p.grad = full[name]
        grads = [p.grad for p in model.parameters()]
        sharded = [g for g in grads if isinstance(g, RaggedShardDTensor)]
        plain = [g for g in grads if not isinstance(g, RaggedShardDTensor)]
        squares.append(list_grad_norm(sharded).double().square())
        ranks.append((grads, list_grad_norm(plain).double().square()))
    before = [[loc(g).clone() for g in grads] for grads, _ in ranks]
    coefs = []
    for grads, replicated in ranks:
        total_norm = (sum(squares) + replicated).sqrt().float()
        coefs.append((max_norm / (total_norm + 1e-6)).clamp(max=1.0))
        assert abs(total_norm.item() - whole.norm().item()) <= 6 * 2.0 ** -24 * whole.norm().item()
        list_scale_grads_(grads, coefs[-1])
    assert_bits_equal(coefs[0], coefs[1], "one coefficient on all ranks")
    assert coefs[0].item() < 1.0
    for (grads, _), olds in zip(ranks, before):
        for g, old in zip(grads, olds):
            assert_bits_equal(loc(g), old * coefs[0], "clipped fragment")
