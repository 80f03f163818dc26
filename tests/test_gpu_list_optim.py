"""Norm, clipping and AdamW over lists of separate tensors on the GPU, against plain 64-bit implementations and the C
oracle.

Tolerances: a 1- or 2-norm is a binary64 sum of n non-negative terms (each addition off by at most 2^-53 of the sum, so
n * 2^-53 in all, and the square root halves it) rounded once to binary32 (2^-24).  The largest magnitude is exact.
Coefficient, clipped gradients and the AdamW step are compared bit for bit."""

import copy
import math
import threading

import numpy as np
import pytest
import torch
import torch.nn as nn

from oracle import cref

from helpers import DTYPES, assert_bits_equal, mixed_values

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
INF = float("inf")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HP = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
CHP = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)

# around a 16-byte vector, a 128-byte line, a 4-KiB tile (1024 / 2048 elements) and two of AdamW's 256-element tiles
EDGES = [1, 0, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 511, 512, 513, 1023, 1024, 1025, 2047, 2048,
         2049, 4095, 4097, 6001]


def _cut(numels, dtype, gap, gen, std=0.02, first=0):
    """A buffer on the CPU and where its tensors start; ``gap`` elements between them."""
    starts, at = [], first
    for n in numels:
        starts.append(at)
        at += n + gap
    buf = (torch.randn(at + 9, generator=gen) * std).to(dtype)
    return buf, starts


def _views(buf, starts, numels):
    return [buf[s:s + n] for s, n in zip(starts, numels)]


def _norm64(tensors, p):
    flat = [t.detach().cpu().double().reshape(-1) for t in tensors if t is not None and t.numel()]
    if not flat:
        return 0.0
    if p == INF:
        return max(float(x.abs().max()) for x in flat)
    return math.fsum(float(x.abs().pow(p).sum()) for x in flat) ** (1.0 / p)


def _assert_norm(got, tensors, p):
    want = _norm64(tensors, p)
    n = sum(t.numel() for t in tensors if t is not None)
    tol = 0.0 if p == INF else want * (2.0 ** -24 * (1 + 2.0 ** -20) + n * 2.0 ** -53)
    assert abs(float(got) - want) <= tol, (float(got), want, tol)


def _coef32(norm, max_norm):
    """min(max_norm / (norm + 1e-6), 1), every operation rounded to binary32."""
    c = np.float32(max_norm) / (np.float32(norm) + np.float32(1e-6))
    return float(min(c, np.float32(1.0)))


# --------------------------------------------------------------------------------------------------- norm ----
@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap,first", [(1, 0), (0, 3), (5, 1)])
def test_norm_at_tile_edges(p, dtype, gap, first):
    from yafsdp_amd.optim import list_clip_coef, list_grad_norm

    gen = torch.Generator().manual_seed(1)
    buf, starts = _cut(EDGES, dtype, gap, gen, first=first)
    dev = buf.to(DEV)
    views = _views(dev, starts, EDGES)
    _assert_norm(list_grad_norm(views, p), _views(buf, starts, EDGES), p)
    for i in range(0, len(views), 5):  # one at a time
        if views[i].numel():
            norm, coef = list_clip_coef([views[i]], 1e-3, p)
            _assert_norm(norm, [views[i]], p)
            assert float(coef) == _coef32(norm.item(), 1e-3)
    assert_bits_equal(dev, buf, "the norm writes nothing")


@pytest.mark.parametrize("p", [1, 2, "inf"])
def test_norm_of_mixed_dtypes_none_and_empty(p):
    from yafsdp_amd.optim import list_clip_coef, list_grad_norm

    gen = torch.Generator().manual_seed(2)
    ts = [(torch.randn(n, generator=gen) * 0.1).to(DTYPES[i % 3]).to(DEV) for i, n in enumerate(EDGES * 2)]
    ts[4] = None
    _assert_norm(list_grad_norm(ts, p), ts, float(p))
    _assert_norm(list_grad_norm(iter(ts), p), ts, float(p))  # any iterable
    for empty in ([torch.zeros(0, device=DEV)], [None, torch.zeros(0, 5, device=DEV, dtype=BF16)]):
        norm, coef = list_clip_coef(empty, 0.5, p)
        assert norm.item() == 0.0 and coef.item() == 1.0
    assert norm.shape == coef.shape == () and norm.dtype == coef.dtype == F32 and norm.device == ts[0].device


@pytest.mark.parametrize("count,low,high", [(320, 1, 40), (321, 1, 40), (1000, 1, 3000), (700, 4096, 4096), (3000, 1, 9)])
def test_norm_of_more_ranges_than_one_launch_holds(count, low, high):
    from yafsdp_amd.optim import list_grad_norm

    rng = np.random.default_rng(count)
    numels = [int(x) for x in rng.integers(low, high + 1, count)]
    gen = torch.Generator().manual_seed(3)
    buf, starts = _cut(numels, BF16, 1, gen)
    views = _views(buf.to(DEV), starts, numels)
    for p in (1.0, 2.0, INF):
        _assert_norm(list_grad_norm(views, p), _views(buf, starts, numels), p)


@pytest.mark.parametrize("dtype,value", [(F32, 3e38), (F32, 1e-30), (F32, 1.4e-45), (BF16, 3e38), (BF16, 1e-38), (F16, 65504.0),
                                         (F16, 6e-8)])
def test_norm_where_squares_leave_binary32(dtype, value):
    """The 2-norm of four equal numbers is twice one of them: exact in binary64, whatever binary32 squares would do."""
    from yafsdp_amd.optim import list_grad_norm

    x = torch.tensor([value, -value, 0.0, value, value], dtype=dtype)
    one = float(x[0].double())
    assert float(list_grad_norm([x.to(DEV)], INF)) == one
    for p, factor in ((2.0, 2.0), (1.0, 4.0)):
        got, want = float(list_grad_norm([x.to(DEV)], p)), factor * one
        want = float(np.float32(want)) if want <= 3.4028235e38 else INF
        assert got == want, (p, got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("where", [0, 3000, 6000])
def test_norm_of_infinities_and_nan(dtype, p, where):
    from yafsdp_amd.optim import list_clip_coef

    x = torch.full((6001,), 0.5, dtype=dtype)
    other = torch.ones(77, dtype=F32, device=DEV)
    for bad in (INF, -INF):
        x[where] = bad
        norm, coef = list_clip_coef([other, x.to(DEV)], 1.0, p)
        assert norm.item() == INF and coef.item() == 0.0
    x[where] = float("nan")
    x[(where + 1) % 6001] = INF
    norm, coef = list_clip_coef([x.to(DEV), other], 1.0, p)
    assert math.isnan(norm.item()) and math.isnan(coef.item())


def test_norm_counts_shared_memory_twice_and_takes_any_dense_layout():
    from yafsdp_amd.optim import list_grad_norm

    x = torch.randn(300, 41, device=DEV)
    _assert_norm(list_grad_norm([x, x.view(-1)[100:5000], x]), [x, x.view(-1)[100:5000], x], 2.0)
    y = torch.randn(7, 5, 3, 11, device=DEV).to(memory_format=torch.channels_last)
    assert not y.is_contiguous()
    _assert_norm(list_grad_norm([x.t(), y]), [x, y], 2.0)
    with pytest.raises(NotImplementedError, match="dense"):
        list_grad_norm([x[:, :40]])
    with pytest.raises(TypeError, match="unsupported dtype"):
        list_grad_norm([x.double()])
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        list_grad_norm([x, x.cpu()])
    with pytest.raises(NotImplementedError, match="infinity-norm"):
        list_grad_norm([x], 3)


def test_norm_is_reproducible():
    from yafsdp_amd.optim import list_clip_coef

    ts = [torch.randn(n, device=DEV) for n in (100003, 5, 70001, 1)]
    first = list_clip_coef(ts, 1.0)
    for _ in range(5):
        again = list_clip_coef(ts, 1.0)
        assert_bits_equal(torch.stack(again), torch.stack(first), "same call, same bits")


# --------------------------------------------------------------------------------------------------- clip ----
def _clipped(buf, starts, numels, coef):
    want = buf.clone()
    for s, n in zip(starts, numels):
        part = want[s:s + n].clone()
        cref.flat_scale(part, coef)
        want[s:s + n] = part
    return want


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap,first", [(1, 0), (0, 3), (5, 1)])
def test_clip_bits_and_untouched_neighbours(p, dtype, gap, first):
    from yafsdp_amd.optim import list_clip_grad_norm_

    gen = torch.Generator().manual_seed(4)
    buf, starts = _cut(EDGES, dtype, gap, gen, first=first)
    dev = buf.to(DEV)
    views = _views(dev, starts, EDGES)
    max_norm = 0.37 * _norm64(views, p)
    norm = list_clip_grad_norm_(views, max_norm, p)
    _assert_norm(norm, _views(buf, starts, EDGES), p)
    assert_bits_equal(dev, _clipped(buf, starts, EDGES, _coef32(norm.item(), max_norm)), "clipped buffer")
    # within the bound: not a bit moves
    before = dev.clone()
    norm = list_clip_grad_norm_(views, 1e9, p)
    assert_bits_equal(dev, before, "nothing to clip")


def test_clip_of_many_tensors_of_every_dtype():
    from yafsdp_amd.optim import list_clip_grad_norm_

    rng = np.random.default_rng(7)
    numels = [int(x) for x in rng.integers(0, 3000, 900)]
    gen = torch.Generator().manual_seed(5)
    cpu = [(torch.randn(n, generator=gen) * 0.1).to(DTYPES[i % 3]) for i, n in enumerate(numels)]
    dev = [t.to(DEV) for t in cpu]
    dev[17], cpu[17] = None, None
    norm = list_clip_grad_norm_(dev, 1.0)
    _assert_norm(norm, cpu, 2.0)
    coef = _coef32(norm.item(), 1.0)
    for i, (a, b) in enumerate(zip(dev, cpu)):
        if b is not None:
            cref.flat_scale(b, coef)
            assert_bits_equal(a, b, f"tensor {i}")


@pytest.mark.parametrize("order", ["ascending", "descending"])
def test_clip_of_neighbours_of_other_dtypes(order):
    """Tensors of all dtypes back to back in one allocation: several of them inside one 16-byte vector, tiles of
    different waves in one cache line."""
    from yafsdp_amd.optim import list_clip_grad_norm_

    gen = torch.Generator().manual_seed(14)
    sizes = [1, 2, 3, 1, 5, 1, 1, 2, 9, 700, 1, 4096, 33, 2, 1, 6000] * 12
    raw = torch.zeros(200_000 * 4, dtype=torch.uint8)
    cpu, spans, at = [], [], 4
    for i, n in enumerate(sizes):
        dtype = DTYPES[i % 3]
        size = 4 if dtype == F32 else 2
        at = -(-at // size) * size
        t = raw[at:at + n * size].view(dtype)
        t.copy_(torch.randn(n, generator=gen))
        cpu.append(t)
        spans.append((at, n, size, dtype))
        at += n * size
    dev_raw = raw.to(DEV)
    dev = [dev_raw[a:a + n * size].view(dtype) for a, n, size, dtype in spans]
    if order == "descending":
        dev.reverse()
    norm = list_clip_grad_norm_(dev, 2.0)
    _assert_norm(norm, cpu, 2.0)
    for t in cpu:
        part = t.clone()
        cref.flat_scale(part, _coef32(norm.item(), 2.0))
        t.copy_(part)
    assert torch.equal(dev_raw.cpu(), raw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_clip_of_special_values(dtype):
    """Subnormals, signed zeros, ties: x * c in binary32, rounded once."""
    from yafsdp_amd.optim import list_scale_grads_

    x = mixed_values(torch.Generator().manual_seed(6), 5000, dtype)
    for c in (0.3, 0.5, 0.0, -0.7, 1e-30, 3e38, INF, float("nan"), 1.0):
        dev, want = x.to(DEV), x.clone()
        coef = torch.tensor([c], dtype=F32)
        list_scale_grads_([dev[:1234], None, dev[1234:]], coef.to(DEV))
        cref.flat_scale(want, float(coef))
        assert_bits_equal(dev, want, f"scale by {c}")


def test_scale_with_a_coefficient_from_elsewhere():
    """Norms of two lists joined outside (as those of several ranks are), the lists scaled by the common coefficient:
    the bits of clipping them as one list.  Long lists, sharded ones and refusals included."""
    from yafsdp_amd.optim import list_clip_coef, list_clip_grad_norm_, list_scale_grads_

    gen = torch.Generator().manual_seed(16)
    cpu = [torch.randn(n, generator=gen).to(DTYPES[i % 3]) for i, n in enumerate([5, 3000, 77, 1] + [9] * 400)]
    a, b = [t.to(DEV) for t in cpu], [t.to(DEV) for t in cpu]
    norm, coef = list_clip_coef(a, 1.0)
    parts = [list_clip_coef(a[:7], 1.0)[0], list_clip_coef(a[7:], 1.0)[0]]
    joined = torch.stack(parts).double().pow(2).sum().sqrt().float()
    assert abs(joined.item() - norm.item()) <= 2 * 2.0 ** -24 * norm.item()
    version = a[0]._version
    list_scale_grads_(a[:7], coef)
    list_scale_grads_(a[7:], coef)
    assert a[0]._version == version + 1
    list_clip_grad_norm_(b, 1.0)
    for x, y in zip(a, b):
        assert_bits_equal(x, y, "scaled in two lists, clipped as one")
    before = a[1].clone()
    with pytest.raises(RuntimeError, match="share memory"):
        list_scale_grads_([a[1], a[1][5:]], coef)
    with pytest.raises(TypeError, match="coef"):
        list_scale_grads_(a, coef.double())
    with pytest.raises(RuntimeError, match="coef must live on the GPU"):
        list_scale_grads_(a, torch.ones(1))
    assert_bits_equal(a[1], before, "a refused call writes nothing")


def test_scalars_that_share_memory_with_the_list():
    """Refused where the call writes them; right beside the list, or in a gradient that is only read, they are taken."""
    from yafsdp_amd.optim import list_adamw_step, list_scale_grads_

    x = torch.full((101,), 0.5, device=DEV)
    before = x.clone()
    for k in (0, 50, 99):
        with pytest.raises(RuntimeError, match="share memory"):
            list_scale_grads_([x[:100]], x[k])
    p, m, v = (torch.ones(100, device=DEV) for _ in range(3))
    with pytest.raises(RuntimeError, match="share memory"):
        list_adamw_step([p], [x[:100]], [m], [v], step=1, grad_scale=x[0], zero_grad=True)
    with pytest.raises(RuntimeError, match="share memory"):
        list_adamw_step([p], [x[:100]], [m], [v], step=1, grad_scale=p[99])
    assert_bits_equal(x, before, "a refused call writes nothing")
    assert_bits_equal(p, torch.ones_like(p), "a refused call writes nothing")
    list_scale_grads_([x[:100]], x[100])
    assert_bits_equal(x, torch.cat([before[:100] * 0.5, before[100:]]), "scaled by its neighbour")
    q, a, b = p.clone(), m.clone(), v.clone()
    list_adamw_step([p], [x[:100]], [m], [v], step=1, grad_scale=x[3])
    list_adamw_step([q], [x[:100]], [a], [b], step=1, grad_scale=x[3].clone())
    for got, want in ((p, q), (m, a), (v, b)):
        assert_bits_equal(got, want, "a factor inside a gradient that is only read")


def test_clip_of_nonfinite_gradients_follows_torch():
    from yafsdp_amd.optim import list_clip_grad_norm_

    for bad in (INF, float("nan")):
        ts = [torch.tensor([1.0, bad, -2.0], device=DEV), torch.ones(5, device=DEV, dtype=BF16)]
        params = [nn.Parameter(torch.zeros_like(t)) for t in ts]
        for q, t in zip(params, ts):
            q.grad = t.clone()
        want = torch.nn.utils.clip_grad_norm_(params, 1.0, foreach=False)
        got = list_clip_grad_norm_(ts, 1.0)
        assert_bits_equal(got, want.float(), "norm")
        for q, t in zip(params, ts):
            assert_bits_equal(t, q.grad, f"gradients with {bad}")


def test_clip_against_torch_on_one_dtype():
    from yafsdp_amd.optim import list_clip_grad_norm_

    ts = [torch.randn(n, device=DEV) for n in (1000, 3, 70000, 129)]
    for p in (1.0, 2.0, INF):
        params = [nn.Parameter(torch.zeros_like(t)) for t in ts]
        for q, t in zip(params, ts):
            q.grad = t.clone()
        want = torch.nn.utils.clip_grad_norm_(params, 0.5, norm_type=p)
        mine = [t.clone() for t in ts]
        got = list_clip_grad_norm_(mine, 0.5, p)
        # torch adds in binary32: 64 roundings of 2^-24 in a row allow for partial sums of 50 terms and a tree above them
        assert abs(got.item() - want.item()) <= 64 * 2.0 ** -24 * want.item()
        for q, t in zip(params, mine):
            torch.testing.assert_close(t, q.grad, rtol=70 * 2.0 ** -24, atol=0)


def test_clip_refuses_shared_memory_and_counts_versions():
    from yafsdp_amd.optim import list_clip_coef, list_clip_grad_norm_

    x = torch.randn(100, device=DEV)
    before = x.clone()
    for ts in ([x, x], [x[:50], x[49:]]):
        with pytest.raises(RuntimeError, match="share memory"):
            list_clip_grad_norm_(ts, 1e-3)
    assert_bits_equal(x, before, "a refused call writes nothing")
    v = x._version
    list_clip_coef([x], 1e-3)
    assert x._version == v
    list_clip_grad_norm_([x[:50], x[50:]], 1e-3)
    assert x._version > v
    with pytest.raises(NotImplementedError):
        list_clip_grad_norm_([x], 1.0, 0.5)


# -------------------------------------------------------------------------------------------------- AdamW ----
def _adam_case(numels, gdtype, odtype, gap, first, seed, specials=False):
    gen = torch.Generator().manual_seed(seed)
    cpu = {}
    for name, dtype, std in (("p", F32, 0.02), ("g", gdtype, 1e-2), ("m", F32, 1e-2), ("v", F32, 1e-2),
                             ("o", odtype, 1.0)):
        if dtype is None:
            continue
        buf, starts = _cut(numels, dtype, gap, gen, std, first)
        cpu[name] = buf.abs() if name == "v" else buf
    if specials:
        cpu["g"][:60] = mixed_values(gen, 60, gdtype)
    return cpu, starts


def _oracle_step(cpu, starts, numels, odtype, zero, skip=(), **hp):
    for i, (s, n) in enumerate(zip(starts, numels)):
        if i in skip or n == 0:
            continue
        p, m, v = (cpu[k][s:s + n].clone() for k in "pmv")
        g = cpu["g"][s:s + n].float().clone()
        o = None if odtype is None else torch.zeros(n, dtype=odtype)
        cref.adamw_step(p, g, m, v, o, zero_grad=zero, **hp)
        for k, x in (("p", p), ("m", m), ("v", v)):
            cpu[k][s:s + n] = x
        if o is not None:
            cpu["o"][s:s + n] = o
        if zero:
            cpu["g"][s:s + n] = 0


@pytest.mark.parametrize("gdtype", DTYPES)
@pytest.mark.parametrize("odtype", [None, BF16, F16])
@pytest.mark.parametrize("gap,first,zero,decoupled,scale", [
    (0, 0, False, True, None), (1, 3, True, True, 0.37), (4, 0, False, False, 0.5), (3, 1, True, False, None)])
def test_adamw_bits(gdtype, odtype, gap, first, zero, decoupled, scale):
    from yafsdp_amd.optim import list_adamw_step

    cpu, starts = _adam_case(EDGES, gdtype, odtype, gap, first, 8, specials=True)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, EDGES) for k, b in dev.items()}
    for step in (1, 7):
        list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists.get("o"), step=step,
                        decoupled_weight_decay=decoupled, zero_grad=zero,
                        grad_scale=None if scale is None else torch.tensor(scale, device=DEV), **HP)
        _oracle_step(cpu, starts, EDGES, odtype, zero, step=step, decoupled=decoupled, grad_scale=scale, **CHP)
        for k in cpu:
            assert_bits_equal(dev[k], cpu[k], f"buffer {k} after step {step}")


@pytest.mark.parametrize("gdtype,odtype", [(F32, None), (BF16, F16), (F16, BF16)])
def test_adamw_of_arrays_at_different_offsets(gdtype, odtype):
    """Nothing but the element size aligns the arrays with each other."""
    from yafsdp_amd.optim import list_adamw_step

    numels, first = [1, 5, 700, 4099, 64], {"p": 1, "g": 3, "m": 2, "v": 7, "o": 5}
    cpu, starts = {}, {}
    for k in ("p", "g", "m", "v") + (("o",) if odtype is not None else ()):
        case, at = _adam_case(numels, gdtype, odtype, first[k], first[k], 12)
        cpu[k], starts[k] = case[k], at
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(dev[k], starts[k], numels) for k in dev}
    list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists.get("o"), step=2, zero_grad=True, **HP)
    for i, n in enumerate(numels):
        part = {k: cpu[k][starts[k][i]:starts[k][i] + n] for k in cpu}
        fresh = {k: x.clone() for k, x in part.items()}
        cref.adamw_step(fresh["p"], part["g"].float(), fresh["m"], fresh["v"], fresh.get("o"), step=2, **CHP)
        for k, x in fresh.items():
            part[k].copy_(x)
        part["g"].zero_()
    for k in cpu:
        assert_bits_equal(dev[k], cpu[k], k)


@pytest.mark.parametrize("beta1,wd", [(0.3, 0.1), (0.9, 0.0), (0.0, 0.1)])
def test_adamw_other_hyperparameters(beta1, wd):
    from yafsdp_amd.optim import list_adamw_step

    numels = [1000, 3, 513]
    cpu, starts = _adam_case(numels, BF16, None, 2, 0, 9)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, numels) for k, b in dev.items()}
    list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], step=3, lr=1e-3, betas=(beta1, 0.95), eps=1e-8,
                    weight_decay=wd)
    _oracle_step(cpu, starts, numels, None, False, step=3, **{**CHP, "beta1": beta1, "weight_decay": wd})
    for k in cpu:
        assert_bits_equal(dev[k], cpu[k], k)


def test_adamw_against_the_formula_in_64_bits():
    """The textbook update in binary64.  m: two roundings and that of 1 - beta1, each at most 2^-24 of |m| + |g - m|.
    v: four of 2^-24 (two products, the sum, the scalars).  The quotient u = (lr / bc1) m / (sqrt(v) / sqrt(bc2) + eps)
    carries those of m and (halved) of v, and at most eight of its own; p then two more of its own size."""
    from yafsdp_amd.optim import list_adamw_step

    numels, h = [5000, 1, 700], 2.0 ** -24
    cpu, starts = _adam_case(numels, BF16, None, 1, 0, 10)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, numels) for k, b in dev.items()}
    list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], step=5, **HP)
    for s, n in zip(starts, numels):
        p, g, m, v = (cpu[k][s:s + n].double() for k in "pgmv")
        m1 = 0.9 * m + 0.1 * g
        v1 = 0.95 * v + 0.05 * g * g
        u = 1e-3 / (1 - 0.9 ** 5) * m1 / ((v1 / (1 - 0.95 ** 5)).sqrt() + 1e-8)
        p1 = p - 1e-3 * 0.1 * p - u
        m_tol = 4 * h * (m1.abs() + g.abs() + m.abs())
        got = {k: dev[k][s:s + n].cpu().double() for k in "pmv"}
        assert ((got["m"] - m1).abs() <= m_tol).all()
        assert ((got["v"] - v1).abs() <= 5 * h * v1).all()
        u_tol = u.abs() * 16 * h + (u / m1.where(m1 != 0, torch.ones_like(m1))).abs() * m_tol
        assert ((got["p"] - p1).abs() <= u_tol + 3 * h * (p.abs() + u.abs())).all()


def test_adamw_of_more_ranges_than_one_launch_holds_and_missing_gradients():
    from yafsdp_amd.optim import list_adamw_step

    rng = np.random.default_rng(11)
    numels = [int(x) for x in rng.integers(0, 1500, 500)]
    cpu, starts = _adam_case(numels, F16, BF16, 1, 0, 11)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, numels) for k, b in dev.items()}
    skip = {0, 100, 101, 499}
    grads = [None if i in skip else g for i, g in enumerate(lists["g"])]
    list_adamw_step(lists["p"], grads, lists["m"], lists["v"], lists["o"], step=2, **HP)
    _oracle_step(cpu, starts, numels, BF16, False, skip, step=2, **CHP)
    for k in cpu:
        assert_bits_equal(dev[k], cpu[k], k)


def test_adamw_refusals_on_the_gpu_and_versions():
    from yafsdp_amd.optim import list_adamw_step

    def fresh():
        return [[torch.randn(n, device=DEV).abs() for n in (40, 7)] for _ in range(4)]

    p, g, m, v = fresh()
    versions = [t._version for t in p + g + m + v]
    list_adamw_step(p, [g[0], None], m, v, step=1)
    moved = [t._version != x for t, x in zip(p + g + m + v, versions)]
    assert moved == [True, False, False, False, True, False, True, False]
    before = [t.clone() for t in p + g + m + v]
    bad = torch.zeros(40, device=DEV)
    for k, wrong, error in ((0, bad.bfloat16(), TypeError), (1, bad.double(), TypeError), (2, bad[:39], ValueError),
                            (3, torch.zeros(80, device=DEV)[::2], NotImplementedError), (1, bad.cpu(), RuntimeError)):
        lists = [list(x) for x in (p, g, m, v)]
        lists[k][0] = wrong
        with pytest.raises(error):
            list_adamw_step(*lists, step=1)
    with pytest.raises(TypeError, match="share a dtype"):
        list_adamw_step(p, [g[0], g[1].bfloat16()], m, v, step=1)
    with pytest.raises(TypeError, match="one dtype for all"):
        list_adamw_step(p, g, m, v, [bad, bad], step=1)
    with pytest.raises(RuntimeError, match="share memory"):
        list_adamw_step(p, g, m, [m[0], v[1]], step=1)
    for scale, error in ((torch.ones(1), RuntimeError), (torch.ones(1, device=DEV).double(), TypeError)):
        with pytest.raises(error, match="grad_scale"):
            list_adamw_step(p, g, m, v, step=1, grad_scale=scale)
    for t, b in zip(p + g + m + v, before):
        assert_bits_equal(t, b, "a refused call writes nothing")
    list_adamw_step(p, [g[0], g[0][:7]], m, v, step=2)  # gradients that are only read may share memory


# --------------------------------------------------------------------------- streams, threads, graphs, sizes ----
def test_two_streams_at_once():
    from yafsdp_amd.optim import list_clip_grad_norm_

    sets, wants = [], []
    for k in range(2):
        gen = torch.Generator().manual_seed(20 + k)
        cpu = [torch.randn(n, generator=gen) for n in (200003, 999, 64)]
        sets.append([t.to(DEV) for t in cpu])
        wants.append(cpu)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    norms = []
    for _ in range(3):
        for ts, s in zip(sets, streams):
            with torch.cuda.stream(s):
                norms.append(list_clip_grad_norm_(ts, 1.0))
    torch.cuda.synchronize()
    for k, cpu in enumerate(wants):
        for r in range(3):
            norm = norms[2 * r + k].item()
            _assert_norm(norm, cpu, 2.0)
            for t in cpu:
                cref.flat_scale(t, _coef32(norm, 1.0))
        for a, b in zip(sets[k], cpu):
            assert_bits_equal(a, b, f"stream {k}")


def test_two_threads_at_once():
    from yafsdp_amd.optim import list_clip_coef

    ts = [[torch.randn(5000 + 7 * k, device=DEV) * (k + 1) for _ in range(400)] for k in range(2)]
    want = [torch.stack(list_clip_coef(t, 1.0)).cpu() for t in ts]
    got = [[], []]

    def work(k):
        torch.cuda.set_device(0)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k].append(torch.stack(list_clip_coef(ts[k], 1.0)).cpu())

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for k in range(2):
        assert len(got[k]) == 20
        for x in got[k]:
            assert_bits_equal(x, want[k], f"thread {k}")


def test_more_long_lists_in_flight_than_staging_slots():
    """Sixty calls whose lists go through the workspace, queued on two streams behind other work: the later ones find
    every staging slot unread."""
    from yafsdp_amd.optim import list_adamw_step, list_clip_coef

    numels = [int(x) for x in np.random.default_rng(60).integers(1, 400, 350)]
    gen = torch.Generator().manual_seed(60)
    sets = []
    for _ in range(30):
        cpu, starts = _adam_case(numels, BF16, None, 1, 0, int(torch.randint(1 << 30, (1,), generator=gen)))
        sets.append((cpu, {k: b.to(DEV) for k, b in cpu.items()}))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    out = []
    for s in streams:
        with torch.cuda.stream(s):
            torch.cuda._sleep(40_000_000)
    for i, (_, dev) in enumerate(sets):
        with torch.cuda.stream(streams[i % 2]):
            lists = {k: _views(b, starts, numels) for k, b in dev.items()}
            norm, coef = list_clip_coef(lists["g"], 1e-3)
            list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], step=2, grad_scale=coef, **HP)
            out.append((norm, coef))
    torch.cuda.synchronize()
    for (cpu, dev), (norm, coef) in zip(sets, out):
        _assert_norm(norm, _views(cpu["g"], starts, numels), 2.0)
        assert float(coef) == _coef32(norm.item(), 1e-3)
        _oracle_step(cpu, starts, numels, None, False, step=2, grad_scale=float(coef), **CHP)
        for k in "pmv":
            assert_bits_equal(dev[k], cpu[k], k)


def test_list_longer_than_a_staging_slot():
    """11,000 tensors of AdamW (528 KB of list) travel in kernel arguments; the norm of the same gradients (132 KB) fits."""
    from yafsdp_amd.optim import list_adamw_step, list_clip_coef

    numels = [1 + i % 3 for i in range(11_000)]
    cpu, starts = _adam_case(numels, BF16, None, 1, 0, 15)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, numels) for k, b in dev.items()}
    norm, coef = list_clip_coef(lists["g"], 0.1)
    list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], step=2, grad_scale=coef, **HP)
    _assert_norm(norm, _views(cpu["g"], starts, numels), 2.0)
    live = torch.zeros(cpu["p"].numel(), dtype=torch.bool)
    for s, n in zip(starts, numels):
        live[s:s + n] = True
    part = {k: cpu[k][live].float() for k in "pgmv"}  # elementwise: all tensors as one
    cref.adamw_step(part["p"], part["g"], part["m"], part["v"], None, step=2, grad_scale=float(coef), **CHP)
    for k in "pmv":
        cpu[k][live] = part[k]
        assert_bits_equal(dev[k], cpu[k], k)


def test_kernel_timing_hook_covers_list_launches():
    from yafsdp_amd import _native
    from yafsdp_amd.optim import list_grad_norm

    ts = [torch.randn(n, device=DEV) for n in (1_000_000, 77)]
    want = list_grad_norm(ts)
    start, stop = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    _native.time_next_launch(start, stop)
    got = list_grad_norm(ts)
    torch.cuda.synchronize()
    assert 0.0 < start.elapsed_time(stop) < 1000.0
    assert_bits_equal(got, want, "timed launch")


def test_captured_step_replays_with_new_gradients():
    """Clip in place, then norm -> AdamW with the coefficient, captured once: two graphs alternate, eager calls and
    synchronizations in between, every replay against the same calls made eagerly on copies."""
    from yafsdp_amd.optim import list_adamw_step, list_clip_coef, list_clip_grad_norm_

    numels = [700, 1, 4097, 0, 90000] + [33] * 400
    gen = torch.Generator().manual_seed(30)

    def make():
        buf, starts = _cut(numels, F32, 1, gen)
        return buf.to(DEV), starts

    def one(st):
        norm = list_clip_grad_norm_(st["g"], 3.0)
        _, coef = list_clip_coef(st["g"], 2.0, INF)
        list_adamw_step(st["p"], st["g"], st["m"], st["v"], step=4, grad_scale=coef, **HP)
        return norm, coef

    states, graphs, outs = [], [], []
    for _ in range(2):
        bufs = {k: make() for k in "pgmv"}
        bufs["v"][0].abs_()
        st = {k: _views(b, s, numels) for k, (b, s) in bufs.items()}
        st["bufs"] = {k: b for k, (b, _) in bufs.items()}
        states.append(st)
    warm = torch.cuda.Stream()
    with torch.cuda.stream(warm):
        saved = [{k: b.clone() for k, b in st["bufs"].items()} for st in states]
        for st in states:
            one(st)
    warm.synchronize()
    for st, old in zip(states, saved):
        for k, b in st["bufs"].items():
            b.copy_(old[k])
    torch.cuda.synchronize()
    for st in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(one(st))
        graphs.append(graph)
    for replay in range(4):
        for k, st in enumerate(states):
            st["bufs"]["g"].copy_(torch.randn(st["bufs"]["g"].shape, generator=gen) * (replay + 1))
            mirror = {x: b.clone() for x, b in st["bufs"].items()}
            starts = _cut(numels, F32, 1, torch.Generator())[1]
            eager = {x: _views(b, starts, numels) for x, b in mirror.items()}
            graphs[k].replay()
            want = one(eager)
            torch.cuda.synchronize()
            for a, b in zip(outs[k], want):
                assert_bits_equal(a, b, f"replay {replay} of graph {k}")
            for x in "pgmv":
                assert_bits_equal(st["bufs"][x], mirror[x], f"buffer {x}, replay {replay} of graph {k}")


def test_more_than_2_to_the_31_elements():
    """One tensor whose byte and element offsets pass 32 bits, and one behind it."""
    from yafsdp_amd.optim import list_clip_grad_norm_, list_grad_norm

    n = (1 << 31) + 4099
    big = torch.zeros(n, dtype=BF16, device=DEV)
    at = [0, 5, (1 << 30) - 1, 1 << 31, n - 1]
    for k, i in enumerate(at):
        big[i] = k + 1.0
    small = torch.full((3,), 2.0, device=DEV)
    assert float(list_grad_norm([big, small], 1.0)) == 15.0 + 6.0
    assert float(list_grad_norm([big, small], INF)) == 5.0
    norm = list_clip_grad_norm_([big, small], 0.5)
    _assert_norm(norm, [torch.arange(1.0, 6.0), torch.full((3,), 2.0)], 2.0)
    coef = _coef32(norm.item(), 0.5)
    want = torch.arange(1.0, 6.0).to(BF16)
    cref.flat_scale(want, coef)
    assert_bits_equal(torch.stack([big[i] for i in at]), want, "elements on both sides of 2^31")
    assert int((big != 0).sum()) == len(at)
    del big
    torch.cuda.empty_cache()


def test_adamw_of_more_tiles_than_one_launch_takes():
    """2^30 elements and a few: every element against the flat pass on a copy."""
    from yafsdp_amd import _native
    from yafsdp_amd.optim import list_adamw_step

    n = (1 << 30) + 1029
    gen = torch.Generator(device=DEV).manual_seed(70)
    p, g, m = (torch.randn(n, device=DEV, generator=gen).mul_(1e-2) for _ in range(3))
    v = torch.randn(n, device=DEV, generator=gen).mul_(1e-2).square_()
    want = [t.clone() for t in (p, m, v)]
    list_adamw_step([p], [g], [m], [v], step=3, **HP)
    _native.adamw_step(want[0], g, want[1], want[2], None, step=3, **CHP)
    for a, b in zip((p, m, v), want):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    del p, g, m, v, want, a, b
    torch.cuda.empty_cache()


def test_clip_of_more_tiles_than_one_launch_takes():
    """2^22 tiles of 4 KiB and two: 17 GB of bfloat16, non-zero on both sides of every border."""
    from yafsdp_amd.optim import list_clip_grad_norm_

    n = (1 << 33) + 4099
    big = torch.zeros(n, dtype=BF16, device=DEV)
    at = [0, (1 << 31) + 1, (1 << 32) - 1, 1 << 32, (1 << 33) - 1, 1 << 33, (1 << 33) + 2048, n - 1]
    for i in at:
        big[i] = 3.0
    norm = list_clip_grad_norm_([big], 1.0)
    assert norm.item() == float(np.float32(math.sqrt(9.0 * len(at))))
    want = torch.full((len(at),), 3.0, dtype=BF16)
    cref.flat_scale(want, _coef32(norm.item(), 1.0))
    assert_bits_equal(torch.stack([big[i] for i in at]), want, "elements on both sides of the borders")
    assert sum(int(torch.count_nonzero(c)) for c in big.split(1 << 30)) == len(at)
    del big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("count", [7, 400])
def test_without_the_native_list_helper(count, monkeypatch):
    """The Python checks build the same entries: same bits."""
    from yafsdp_amd import _native
    from yafsdp_amd.optim import list_adamw_step, list_clip_grad_norm_

    numels = [int(x) for x in np.random.default_rng(count).integers(0, 600, count)]
    cpu, starts = _adam_case(numels, BF16, F16, 1, 0, 13)
    results = []
    for helper in (True, False):
        if not helper:
            monkeypatch.setattr(_native, "_tensorlist", None)
        dev = {k: b.to(DEV) for k, b in cpu.items()}
        lists = {k: _views(b, starts, numels) for k, b in dev.items()}
        lists["g"][1] = None
        norm = list_clip_grad_norm_(lists["g"], 0.01)
        versions = [lists["p"][0]._version, dev["m"]._version]
        list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists["o"], step=2, **HP)
        assert lists["p"][0]._version > versions[0] and dev["m"]._version > versions[1]
        results.append([norm, *dev.values()])
    for a, b in zip(*results):
        assert_bits_equal(a, b, "with and without the helper")


# -------------------------------------------------------------------------------------------- used together ----
@pytest.mark.parametrize("gdtype", DTYPES)
def test_norm_coefficient_and_step_together(gdtype):
    """As they are used: the coefficient of one call goes into the step of the next, three steps, against the oracle."""
    from yafsdp_amd.optim import list_adamw_step, list_clip_coef

    numels = [4096, 1000, 77, 1] + [64] * 100
    cpu, starts = _adam_case(numels, gdtype, BF16, 1, 0, 40)
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    lists = {k: _views(b, starts, numels) for k, b in dev.items()}
    for step in range(1, 4):
        fresh = torch.randn(cpu["g"].shape, generator=torch.Generator().manual_seed(step)).to(gdtype)
        cpu["g"].copy_(fresh), dev["g"].copy_(fresh)
        norm, coef = list_clip_coef(lists["g"], 1.0)
        list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists["o"], step=step, grad_scale=coef, **HP)
        _assert_norm(norm, _views(cpu["g"], starts, numels), 2.0)
        assert float(coef) == _coef32(norm.item(), 1.0) < 1.0
        _oracle_step(cpu, starts, numels, BF16, False, step=step, grad_scale=float(coef), **CHP)
        for k in cpu:
            assert_bits_equal(dev[k], cpu[k], f"buffer {k} after step {step}")


class _Net(nn.Module):
    def __init__(self):
        super().__init__()
        self.inner = nn.Sequential(nn.Linear(64, 96), nn.GELU(), nn.Linear(96, 64))
        self.scale = nn.Parameter(torch.ones(64))
        self.bias = nn.Parameter(torch.zeros(64))
        self.unused = nn.Parameter(torch.zeros(5))

    def forward(self, x):
        return self.inner(x) * self.scale + self.bias


def test_model_with_sharded_and_plain_parameters():
    """A wrapped submodule next to plain parameters: one norm over both kinds, FlatAdamW steps both."""
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd.optim import FlatAdamW, list_clip_coef, list_clip_grad_norm_

    torch.manual_seed(50)
    model0 = _Net().to(DEV)
    x = torch.randn(16, 64, device=DEV)
    results = []
    for fused in (True, False):
        model = copy.deepcopy(model0)
        fully_shard(model.inner, mesh=(1, 0), mp_policy=MixedPrecisionPolicy(param_dtype=F32))
        params = list(model.parameters())
        opt = FlatAdamW(params, **HP)
        for _ in range(3):
            model(x).pow(2).mean().backward()
            grads = [p.grad for p in params]
            assert any(g is None for g in grads)
            locals_ = [g if g is None else getattr(g, "_local_tensor", g) for g in grads]
            if fused:
                norm, coef = list_clip_coef(grads, 0.05)
                _assert_norm(norm, locals_, 2.0)
                opt.step(grad_scale=coef)
            else:
                before = [None if g is None else g.clone() for g in locals_]
                _assert_norm(list_clip_grad_norm_(grads, 0.05), before, 2.0)
                opt.step()
            opt.zero_grad(set_to_none=True)
        results.append([getattr(p.detach(), "_local_tensor", p.detach()).clone() for p in params])
    for a, b in zip(*results):
        assert_bits_equal(a, b, "coefficient in the step == clipping before it")
    assert torch.equal(results[0][2], torch.zeros(5, device=DEV)) or any(
        torch.equal(t, torch.zeros(5, device=DEV)) for t in results[0])


def test_adamw_list_step_on_sharded_parameters():
    """list_adamw_step on a wrapped model's fragments: FlatAdamW's bits, and the next forward casts the new masters."""
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd.optim import FlatAdamW, list_adamw_step

    torch.manual_seed(53)
    model0 = _Net().inner.to(DEV)
    x = torch.randn(16, 64, device=DEV)
    outs = []
    for with_list in (True, False):
        model = copy.deepcopy(model0)
        fully_shard(model, mesh=(1, 0), mp_policy=MixedPrecisionPolicy(param_dtype=BF16, cast_forward_inputs=True))
        params = list(model.parameters())
        opt = FlatAdamW(params, **HP)
        state = [[torch.zeros_like(p._local_tensor.detach()) for p in params] for _ in range(2)]
        ys = []
        for step in range(1, 4):
            y = model(x)
            ys.append(y.detach().clone())
            y.float().pow(2).mean().backward()
            if with_list:
                list_adamw_step(params, [p.grad for p in params], *state, step=step, zero_grad=True, **HP)
            else:
                opt.step()
            opt.zero_grad(set_to_none=True)
        ys.append(model(x).detach().clone())
        outs.append(ys + [p._local_tensor.detach().clone() for p in params])
    for a, b in zip(*outs):
        assert_bits_equal(a, b, "list step == flat step")


def test_clipping_a_sharded_gradient_makes_its_fused_norm_stale():
    from yafsdp_amd import MixedPrecisionPolicy, fully_shard
    from yafsdp_amd.optim import disable_fused_grad_norm, enable_fused_grad_norm, grad_clip_coef, list_clip_grad_norm_

    torch.manual_seed(51)
    model = _Net().inner.to(DEV)
    fully_shard(model, mesh=(1, 0), mp_policy=MixedPrecisionPolicy(param_dtype=F32))
    x = torch.randn(16, 64, device=DEV)
    model(x).pow(2).mean().backward()
    model.zero_grad(set_to_none=True)
    enable_fused_grad_norm(model)
    try:
        model(x).pow(2).mean().backward()
        before = grad_clip_coef(model, 1.0)[0].item()
        list_clip_grad_norm_([p.grad for p in model.parameters()], 0.25 * before)
        after = grad_clip_coef(model, 1.0)[0].item()
    finally:
        disable_fused_grad_norm(model)
    # the clipped norm: its coefficient and each element off by 2^-24 or so
    assert abs(after - 0.25 * before) <= 8 * 2.0 ** -24 * before + 1e-6


def test_flat_adamw_steps_many_plain_parameters():
    """Same bits as one launch per parameter; per-parameter step counts; a state dict in between."""
    from yafsdp_amd.optim import FlatAdamW

    gen = torch.Generator().manual_seed(52)
    numels = [1, 5, 4096, 513, 64, 7] + [33] * 120
    params = [nn.Parameter(torch.randn(n, generator=gen).to(DEV)) for n in numels]
    mirror = [(p.detach().cpu().clone(), torch.zeros(n), torch.zeros(n)) for p, n in zip(params, numels)]
    steps = [0] * len(numels)
    opt = FlatAdamW(params, **HP)
    for it in range(4):
        scale = None if it % 2 else 0.5
        for i, p in enumerate(params):
            p.grad = None if (i + it) % 5 == 0 else torch.randn(numels[i], generator=gen).to(DEV)
        for i, p in enumerate(params):
            if p.grad is not None:
                steps[i] += 1
                cref.adamw_step(*(mirror[i][0], p.grad.cpu(), mirror[i][1], mirror[i][2], None), step=steps[i],
                                grad_scale=scale, **CHP)
        opt.step(grad_scale=None if scale is None else torch.tensor([scale], device=DEV), zero_grad=it == 3)
        if it == 1:
            state = copy.deepcopy(opt.state_dict())
            opt = FlatAdamW(params, **HP)
            opt.load_state_dict(state)
        for i, p in enumerate(params):
            assert_bits_equal(p, nn.Parameter(mirror[i][0]), f"parameter {i} after iteration {it}")
    assert all(p.grad is None or float(p.grad.abs().max()) == 0.0 for p in params)
    assert [int(opt.state_dict()["state"][i]["step"]) for i in range(len(params))] == steps


def test_flat_adamw_of_parameters_that_share_memory():
    """Two parameters on one storage are stepped one after the other, as separate launches step them."""
    from yafsdp_amd.optim import FlatAdamW

    base = torch.randn(100, device=DEV)
    want = base.cpu().clone()
    a, b = nn.Parameter(base[:60]), nn.Parameter(base[40:])
    opt = FlatAdamW([a, b], **HP)
    a.grad, b.grad = torch.randn(60, device=DEV), torch.randn(60, device=DEV)
    for part, g in ((want[:60], a.grad.cpu()), (want[40:], b.grad.cpu())):
        p = part.clone()
        cref.adamw_step(p, g, torch.zeros(60), torch.zeros(60), None, step=1, **CHP)
        part.copy_(p)
    opt.step()
    assert_bits_equal(base, want, "shared storage")
