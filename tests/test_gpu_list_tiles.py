"""The list passes at the ends of their tiles: ranges that begin on a tile's boundary, a little behind it or a little
before the next one, and end on it, one element short of it or one beyond.

Coefficient, clipped elements and the AdamW step are compared bit for bit with the C oracle.  Norms: n terms are added in
binary64 (n * 2^-53 of the sum) and rounded to binary32 once (2^-24)."""

import math

import pytest
import torch

from oracle import cref

from helpers import DTYPES, assert_bits_equal

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def _ends(tile, heads, tiles=3):
    """(elements in front of the range in its first tile, its length) for ranges that end about the end of each of the
    first `tiles` tiles."""
    return [(h, k * tile - h + d) for h in heads for k in range(1, tiles + 1) for d in (-1, 0, 1) if k * tile - h + d > 0]


def _laid_out(cases, align, dtype, gen, std):
    """A buffer whose first element lies on every boundary used here, and each case's range: `align` elements after the
    boundary behind the range before it, so that no two ranges follow each other in memory."""
    starts, at = [], 0
    for head, n in cases:
        start = (-(-at // align) + 1) * align + head
        starts.append(start)
        at = start + n
    buf = (torch.randn(at + align, generator=gen) * std).to(dtype)
    return buf, [(s, s + n) for s, (_, n) in zip(starts, cases)]


@pytest.mark.parametrize("gdtype", DTYPES)
@pytest.mark.parametrize("odtype", [None, BF16, F16])
@pytest.mark.parametrize("zero", [False, True])
def test_adamw_at_the_ends_of_its_tiles(gdtype, odtype, zero):
    """Tiles of 256 elements from a 256-byte boundary of the parameters: whole ones, a last one of one element, a first one
    of one, two or three (which no quad holds)."""
    from yafsdp_amd.optim import list_adamw_step

    cases = _ends(256, (0, 1, 2, 3, 4, 61, 63)) + [(0, 1), (63, 1), (0, 4), (62, 5)]
    gen = torch.Generator().manual_seed(1)
    cpu = {}
    for name, dtype, std in (("p", F32, 0.02), ("g", gdtype, 1e-2), ("m", F32, 1e-2), ("v", F32, 1e-2), ("o", odtype, 1.0)):
        if dtype is not None:
            cpu[name], spans = _laid_out(cases, 64, dtype, gen, std)
    cpu["v"].abs_()
    dev = {k: b.to(DEV) for k, b in cpu.items()}
    assert dev["p"].data_ptr() % 256 == 0
    tails = {(lo % 64 + hi - lo - 1) % 256 + 1 for lo, hi in spans}
    assert {1, 255, 256} <= tails and {hi - lo for lo, hi in spans} >= {255, 256, 257}
    lists = {k: [b[lo:hi] for lo, hi in spans] for k, b in dev.items()}
    list_adamw_step(lists["p"], lists["g"], lists["m"], lists["v"], lists.get("o"), step=3, lr=1e-3, betas=(0.9, 0.95),
                    eps=1e-8, weight_decay=0.1, grad_scale=torch.tensor(0.37, device=DEV), zero_grad=zero)
    for lo, hi in spans:
        part = {k: b[lo:hi].clone() for k, b in cpu.items()}
        cref.adamw_step(part["p"], part["g"].float(), part["m"], part["v"], part.get("o"), lr=1e-3, beta1=0.9, beta2=0.95,
                        eps=1e-8, weight_decay=0.1, step=3, grad_scale=float(torch.tensor(0.37)))
        if zero:
            part["g"].zero_()
        for k, x in part.items():
            cpu[k][lo:hi] = x
    for k in cpu:
        assert_bits_equal(dev[k], cpu[k], f"buffer {k}, the elements between the ranges included")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, INF])
@pytest.mark.parametrize("tiles,count", [(2, 1), (3, 6)])  # 58 tiles, which one workgroup takes; 650
def test_norm_and_clip_at_the_ends_of_their_tiles(dtype, p, tiles, count):
    """Tiles of 4 KiB from a 128-byte line."""
    from yafsdp_amd.optim import list_clip_grad_norm_

    size = 4 if dtype == F32 else 2
    line = 128 // size
    heads = (0, 1, 16 // size - 1, 16 // size, line - 1)
    cases = (_ends(4096 // size, heads, tiles) + [(0, 255), (1, 256), (line - 1, 257)]) * count
    gen = torch.Generator().manual_seed(2)
    cpu, spans = _laid_out(cases, line, dtype, gen, 0.02)
    dev = cpu.to(DEV)
    assert dev.data_ptr() % 128 == 0
    parts = [cpu[lo:hi] for lo, hi in spans]
    flat = torch.cat([x.double() for x in parts])
    want = float(flat.abs().max()) if p == INF else math.fsum(flat.abs().pow(p).tolist()) ** (1.0 / p)
    norm = list_clip_grad_norm_([dev[lo:hi] for lo, hi in spans], 0.37 * want, p)
    tol = 0.0 if p == INF else want * (2.0 ** -24 * (1 + 2.0 ** -20) + flat.numel() * 2.0 ** -53)
    assert abs(norm.item() - want) <= tol
    coef = float(torch.tensor(0.37 * want, dtype=F32) / (torch.tensor(norm.item(), dtype=F32) + torch.tensor(1e-6, dtype=F32)))
    for x in parts:
        y = x.clone()
        cref.flat_scale(y, coef)
        x.copy_(y)
    assert_bits_equal(dev, cpu, "the ranges, and the elements between them")
