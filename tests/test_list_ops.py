"""The list passes without a GPU: what the C entry points refuse before they touch the device, what the Python side
refuses, and the C++ pass over tensor lists against the Python checks it short-cuts."""

import numpy as np
import pytest
import torch

from yafsdp_amd import _native

tl = pytest.importorskip("yafsdp_amd._tensorlist")
OK, INVALID, DTYPE, MISALIGNED, TOO_LARGE, OVERLAP = 0, -1, -2, -3, -6, -9
F32, BF16, F16 = 0, 1, 2
WS = _native.lib.yafsdp_list_workspace_bytes(1)


def _entries(*rows):
    return np.array([(*r, 0) for r in rows], dtype=_native._LIST_ENTRY).tobytes(), len(rows)


def _adam(*rows):
    return np.array(list(rows), dtype=_native._ADAMW_ENTRY).tobytes(), len(rows)


def _norm(entries, norm=2, workspace=0x10000, ws_bytes=WS, out=0x20000, clip=False, n=None):
    buf, count = entries
    fn = _native.lib.yafsdp_list_clip if clip else _native.lib.yafsdp_list_norm
    return fn(buf, count if n is None else n, norm, 1.0, workspace, ws_bytes, out, None)


def _scale(entries, coef=0x20000, workspace=0x10000, ws_bytes=WS):
    return _native.lib.yafsdp_list_scale(*entries, coef, workspace, ws_bytes, None)


# every refused call names addresses that are never read: the checks come before the first launch
@pytest.mark.parametrize("clip", [False, True])
def test_norm_and_clip_refusals(clip):
    one = _entries((0x1000, 4, F32))
    assert _norm(one, norm=0, clip=clip) == INVALID and _norm(one, norm=4, clip=clip) == INVALID
    assert _norm(one, workspace=None, clip=clip) == INVALID
    assert _norm(one, ws_bytes=WS - 1, clip=clip) == INVALID
    assert _norm(one, out=None, clip=clip) == INVALID
    assert _norm(one, workspace=0x10008, clip=clip) == MISALIGNED
    assert _norm(one, out=0x20002, clip=clip) == MISALIGNED
    assert _norm(one, n=-1, clip=clip) == INVALID
    many = _entries(*[(0x100000 + 0x100 * i, 4, F32) for i in range(321)])
    assert _norm(many, clip=clip) == INVALID  # a longer list needs a larger workspace
    assert _norm((None, 1), clip=clip) == INVALID
    assert _norm(_entries((0x1000, 4, 3)), clip=clip) == DTYPE
    assert _norm(_entries((0x1000, 4, -1)), clip=clip) == DTYPE
    assert _norm(_entries((0x1000, -4, F32)), clip=clip) == INVALID
    assert _norm(_entries((0, 4, F32)), clip=clip) == INVALID
    assert _norm(_entries((0x1000, 4, F32), (0x2002, 4, F32)), clip=clip) == MISALIGNED
    assert _norm(_entries((0x2001, 4, BF16)), clip=clip) == MISALIGNED
    assert _norm(_entries((0x1000, 1 << 47, F32)), clip=clip) == TOO_LARGE
    assert _norm(_entries((1 << 48, 4, F32)), clip=clip) == INVALID  # no device address
    # 2^45 bytes in one tensor are more tiles than one launch counts
    assert _norm(_entries((0x1000, 1 << 44, BF16)), clip=clip) == TOO_LARGE


@pytest.mark.parametrize("call", ["clip", "scale"])
@pytest.mark.parametrize("rows", [
    [(0x1000, 64, F32), (0x1000, 64, F32)],                        # the same tensor twice
    [(0x1000, 64, F32), (0x10fc, 4, F32)],                         # the last element of one is the first of the other
    [(0x9000, 8, BF16), (0x1000, 4096, F32), (0x2000, 8, F16)],    # out of order, across dtypes
])
def test_writes_to_shared_memory_are_refused(call, rows):
    e = _entries(*rows)
    rc = _norm(e, clip=True) if call == "clip" else _scale(e)
    assert rc == OVERLAP
    assert "share memory" in _native.error_string(rc)


def test_scalars_inside_what_is_written_are_refused():
    """A coefficient that its own call rewrites would be read by some waves before and by others after."""
    one = _entries((0x9000, 64, BF16), (0x1000, 64, F32))  # up to 0x9080 and 0x1100
    for at in (0x1000, 0x10fc, 0x907c):
        assert _scale(one, coef=at) == OVERLAP
    for at in (0xffc, 0x10fc, 0x8ffc, 0x9000):  # two numbers, eight bytes
        assert _norm(one, out=at, clip=True) == OVERLAP
    row = (0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 8)
    for k in (0, 2, 3):
        assert _adamw(_adam(row), scale=row[k] + 28) == OVERLAP
    assert _adamw(_adam(row), scale=0x2000, flags=_native.ADAM_ZERO_GRAD) == OVERLAP
    assert _adamw(_adam(row), scale=0x500c, out=F16) == OVERLAP


def test_scale_refusals_and_empty_list():
    one = _entries((0x1000, 4, F32))
    assert _scale(one, coef=None) == INVALID and _scale(one, coef=0x20001) == MISALIGNED
    assert _scale(one, workspace=None) == INVALID and _scale(one, workspace=0x10008) == MISALIGNED
    assert _scale(one, ws_bytes=WS - 1) == INVALID
    assert _scale(_entries((0x1000, 4, 9))) == DTYPE
    assert _scale(_entries((0x1002, 4, F32))) == MISALIGNED
    assert _scale((None, 0)) == OK
    assert _scale(_entries((0, 0, F32), (0x1001, 0, BF16))) == OK  # empty tensors


def _adamw(entries, grad=F32, out=F32, step=1, scale=None, flags=1, n=None, workspace=None, ws_bytes=0):
    buf, count = entries
    return _native.lib.yafsdp_list_adamw(buf, count if n is None else n, grad, out, 1e-3, 0.9, 0.95, 1e-8, 0.1, step,
                                         scale, flags, workspace, ws_bytes, None)


def test_adamw_refusals():
    row = (0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 8)
    assert _adamw(_adam(row), step=0) == INVALID
    assert _adamw(_adam(row), n=-1) == INVALID
    assert _adamw((None, 1)) == INVALID
    assert _adamw(_adam(row), grad=5) == DTYPE and _adamw(_adam(row), out=-1) == DTYPE
    assert _adamw(_adam(row), scale=0x6001) == MISALIGNED
    assert _adamw(_adam((*row[:5], -1))) == INVALID
    assert _adamw(_adam((*row[:5], 1 << 47))) == TOO_LARGE
    for k in range(4):
        assert _adamw(_adam(tuple(0 if i == k else x for i, x in enumerate(row)))) == INVALID
        assert _adamw(_adam(tuple(x + 2 if i == k else x for i, x in enumerate(row)))) == MISALIGNED
    assert _adamw(_adam((*row[:4], 0, 8)), out=BF16) == INVALID
    assert _adamw(_adam((*row[:4], 0x5001, 8)), out=BF16) == MISALIGNED
    assert _adamw(_adam((0x1000, 0x2001, 0x3000, 0x4000, 0, 8)), grad=BF16) == MISALIGNED
    assert _adamw(_adam((0, 0, 0, 0, 0, 0))) == OK and _adamw((None, 0)) == OK
    many = _adam(*[tuple(x + 0x100000 * i for x in row[:5]) + (8,) for i in range(81)])
    need = _native.lib.yafsdp_list_adamw_workspace_bytes(81)
    assert _adamw(many) == INVALID and _adamw(many, workspace=0x10000, ws_bytes=need - 1) == INVALID
    assert _adamw(many, workspace=0x10008, ws_bytes=need) == MISALIGNED
    ZERO = _native.ADAM_ZERO_GRAD
    far = (0x11000, 0x12000, 0x13000, 0x14000, 0x15000, 8)
    assert _adamw(_adam(row, (0x1000, *far[1:]))) == OVERLAP              # the same parameter twice
    assert _adamw(_adam(row, (0x2010, *far[1:]))) == OVERLAP              # a parameter inside another's gradient
    assert _adamw(_adam(row, (*far[:2], 0x401c, *far[3:]))) == OVERLAP    # moments of two positions
    assert _adamw(_adam((0x1000, 0x1000, 0x3000, 0x4000, 0, 8))) == OVERLAP
    assert _adamw(_adam(row, (*far[:4], 0x5000, 8)), out=F16) == OVERLAP
    assert _adamw(_adam(row, (far[0], 0x2000, *far[2:])), flags=ZERO) == OVERLAP  # one gradient zero-filled twice


# ---- the Python side -------------------------------------------------------------------------------------------
def test_lists_that_are_refused():
    from yafsdp_amd import optim

    for fn in (lambda ts: optim.list_grad_norm(ts), lambda ts: optim.list_clip_coef(ts, 1.0),
               lambda ts: optim.list_clip_grad_norm_(ts, 1.0)):
        with pytest.raises(RuntimeError, match="must live on the GPU"):
            fn([torch.zeros(4)])
        with pytest.raises(ValueError, match="no tensors"):
            fn([])
        with pytest.raises(ValueError, match="no tensors"):
            fn([None, None])
        with pytest.raises(TypeError, match="list of tensors"):
            fn(torch.zeros(4))
        with pytest.raises(TypeError, match="must be a tensor"):
            fn([1.0])
        with pytest.raises(NotImplementedError, match="strided"):
            fn([torch.zeros(3).to_sparse()])
    with pytest.raises(ValueError, match="Invalid step"):
        optim.list_adamw_step([], [], [], [], step=0)
    for wrong in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                  dict(lr=float("nan"))):
        with pytest.raises(ValueError, match="Invalid"):
            optim.list_adamw_step([], [], [], [], step=1, **wrong)
    with pytest.raises(ValueError, match="no parameter"):
        optim.list_adamw_step([torch.zeros(2)], [None], [torch.zeros(2)], [torch.zeros(2)], step=1)
    with pytest.raises(ValueError, match="exp_avgs: expected 1"):
        optim.list_adamw_step([torch.zeros(2)], [None], [], [torch.zeros(2)], step=1)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        optim.list_adamw_step(*[[torch.zeros(2)] for _ in range(4)], step=1)


@pytest.mark.parametrize("norm_type", [0, 3, 0.5, -1, float("-inf"), float("nan"), "fro"])
def test_norm_types_that_are_refused(norm_type):
    with pytest.raises((NotImplementedError, ValueError)):
        _native.norm_code(norm_type)


def test_norm_types_that_are_taken():
    assert [_native.norm_code(x) for x in (1, 1.0, 2, 2.0, float("inf"), "inf")] == [1, 1, 2, 2, 3, 3]


# ---- the C++ pass ----------------------------------------------------------------------------------------------
def _rows(buf, dtype):
    return np.frombuffer(buf, dtype=dtype).tolist()


def test_list_entries_of_cpu_tensors():
    a = torch.randn(6, 4)
    ts = [a, None, a.t(), torch.zeros(0, dtype=torch.bfloat16), torch.nn.Parameter(torch.zeros(3, dtype=torch.float16)),
          a.bfloat16().view(2, 3, 4).permute(2, 0, 1)]
    buf, count, index = tl.list_entries(ts, False)
    assert (count, index) == (5, -1)
    assert _rows(buf, _native._LIST_ENTRY) == [
        (a.data_ptr(), 24, F32, 0), (a.data_ptr(), 24, F32, 0), (0, 0, BF16, 0), (ts[4].data_ptr(), 3, F16, 0),
        (ts[5].data_ptr(), 24, BF16, 0)]
    assert tl.list_entries(tuple(ts), False)[0] == buf


@pytest.mark.parametrize("bad", [
    torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int32), torch.zeros(8)[::2],
    torch.zeros(1).expand(4), torch.zeros(4, 4)[:, :2], 3.0, torch.zeros(3).to_sparse(),
    torch.zeros(4, dtype=torch.complex64),
])
def test_list_entries_hands_back_what_it_does_not_take(bad):
    assert tl.list_entries([torch.zeros(4), bad], False) is None
    assert tl.list_entries([torch.zeros(4), torch.zeros(4)], True) is None  # a CPU tensor where GPU tensors are wanted
    assert tl.list_entries([], False) is None and tl.list_entries("ab", False) is None


def test_dense_means_the_same_on_both_sides():
    a = torch.zeros(4, 6, 5)
    for t in (a, a.t() if a.dim() == 2 else a.permute(2, 0, 1), a[:, :, ::2], a[1:], a[:, 1:], a.view(-1)[3:7],
              torch.zeros(1).expand(3), torch.zeros(3, 1, 4).permute(2, 1, 0), torch.zeros(0, 3).t(), torch.zeros(())):
        assert _native._is_dense(t) == (tl.list_entries([t], False) is not None), (t.shape, t.stride())


def test_adamw_entries_of_cpu_tensors():
    n = [5, 0, 7]
    ps, ms, vs = ([torch.zeros(k) for k in n] for _ in range(3))
    gs = [torch.zeros(k, dtype=torch.bfloat16) for k in n]
    os_ = [torch.zeros(k, dtype=torch.float16) for k in n]
    buf, count, index, g, o = tl.adamw_entries(ps, gs, ms, vs, os_, False)
    assert (count, index, g, o) == (2, -1, BF16, F16)
    assert _rows(buf, _native._ADAMW_ENTRY) == [
        tuple(x[k].data_ptr() for x in (ps, gs, ms, vs, os_)) + (n[k],) for k in (0, 2)]
    buf, count, _, g, o = tl.adamw_entries(ps, [gs[0], None, None], ms, vs, None, False)
    assert (count, g, o) == (1, BF16, 0) and _rows(buf, _native._ADAMW_ENTRY)[0][4] == 0
    good = [ps, gs, ms, vs, os_]
    for k, bad in ((0, torch.zeros(5).bfloat16()), (2, torch.zeros(6)), (1, torch.zeros(5)), (3, torch.zeros(10)[::2]),
                   (4, torch.zeros(5)), (4, torch.zeros(5).bfloat16()), (0, None)):
        lists = [list(x) for x in good]
        lists[k][0] = bad
        assert tl.adamw_entries(*lists, False) is None, (k, bad)
    assert tl.adamw_entries(ps, gs, ms, vs[:2], None, False) is None


def test_whole_calls_hand_back_what_they_do_not_take():
    """Nothing is called for a list that is not on the GPU asked for (the addresses here are not code)."""
    a = [torch.zeros(3)]
    assert tl.list_norm(8, 8, a, 0, 0, 2, 1.0) is None and tl.list_norm(8, 8, [], 0, 0, 2, 1.0) is None
    assert tl.list_adamw(8, 8, a, a, a, a, None, 0, 0, 1e-3, 0.9, 0.9, 1e-8, 0.0, 1, 0, 0) is None


def test_bump_versions_matches_torch():
    base = torch.zeros(8)
    a, b = base[:4], torch.zeros(3)
    before = (base._version, b._version)
    tl.bump_versions([a, None, b])
    assert (base._version, b._version) == (before[0] + 1, before[1] + 1)  # a view shares its base's counter
    tl.bump_versions([a, b], [None, 1])
    assert (base._version, b._version) == (before[0] + 1, before[1] + 2)
    with torch.inference_mode():
        c = torch.zeros(2)
    tl.bump_versions([c])  # has none
    with pytest.raises(TypeError):
        tl.bump_versions([1])
    with pytest.raises(TypeError):
        tl.bump_versions([b], [])


def test_workspace_sizes():
    """Partial sums, and behind them (AdamW: alone) lists that the kernel arguments do not hold: 3 (12) words per entry in
    whole pieces of 960."""
    norm, adamw = _native.lib.yafsdp_list_workspace_bytes, _native.lib.yafsdp_list_adamw_workspace_bytes
    assert norm(0) == norm(320) == 1024 * 8
    for n in (321, 640, 641, 5000):
        assert norm(n) == norm(0) + -(-3 * n // 960) * 960 * 4
    assert adamw(0) == adamw(80) == 0
    for n in (81, 160, 161, 3000):
        assert adamw(n) == -(-12 * n // 960) * 960 * 4


def test_staging_slots_with_a_simulated_gpu():
    """Threads claim, fill and queue slots while another plays the GPU that reads them late and out of order between
    queues: what it reads is what was filled, and a claim fails only while every slot is unread."""
    import importlib.util
    import os
    import subprocess

    here = os.path.dirname(os.path.abspath(__file__))
    spec = importlib.util.spec_from_file_location("c_build", os.path.join(here, "c", "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    out = subprocess.run([mod.build_stage_slots_check()], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "ok" in out.stdout
