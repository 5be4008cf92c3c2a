"""The weight's and the bias's gradients of layer norm over few and many rows: exact where every sum is a
whole number below 2^24, and within the roundings that the kernels make."""
from __future__ import annotations

import pytest
import torch

from tests.ops_util import DTYPES, U

pytestmark = pytest.mark.gpu

NAN = float("nan")
UNITS = 256  # compute units of the card
CHUNK = 1 << 25  # elements that the reference takes at once


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _place(t, gap):
    """t with `gap` NaN between its rows and before the first."""
    if not gap:
        return t
    rows, d = t.shape
    buf = torch.full((rows * (d + gap) + gap,), NAN, dtype=t.dtype, device="cuda")
    out = buf[gap:].view(rows, d + gap)[:, :d]
    out.copy_(t)
    return out


def _columns(dy, x, mean, rstd):
    """sum of dy xhat, of dy, and of their magnitudes, in 64 bits."""
    d = x.shape[1]
    sums = torch.zeros(4, d, dtype=torch.float64, device="cuda")
    step = max(1, CHUNK // d)
    for a in range(0, x.shape[0], step):
        g = dy[a:a + step].double()
        h = (x[a:a + step].double() - mean[a:a + step, None].double()) * rstd[a:a + step, None].double()
        sums += torch.stack([(g * h).sum(0), g.sum(0), (g * h).abs().sum(0), g.abs().sum(0)])
    return sums


ROWS = [(1, 768), (33, 768), (4099, 33), (3000, 9), (20000, 768), (100_001, 100), (50_003, 1023), (5001, 2500), (9000, 4096),
        (3000, 8200), (700, 12289), (700, 20001), (2_100_000, 1030), (6_000_000, 64)]


@pytest.mark.parametrize("rows,d", ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sums_of_whole_numbers_are_exact(rows, d, dtype):
    """With mean 0 and rstd 1 and whole numbers of -2 to 2 every partial sum is one below 2^24 and f32
    adds them exactly, in any order: a row that is left out, read twice or taken from another place shows."""
    _need_gpu()
    from luminamoon_amd import ops

    if dtype != "bf16" and rows * d > 1 << 28:
        pytest.skip("one type at the largest sizes")
    print(f"[case] {rows}x{d} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows + d)
    limit = 2 if 4 * rows < 1 << 24 else 1
    assert limit * limit * rows < 1 << 24
    x, dy = (torch.randint(-limit, limit + 1, (rows, d), generator=g, device="cuda", dtype=torch.int8).to(DTYPES[dtype])
             for _ in range(2))
    gap = 3 if rows * d < 1 << 26 else 0
    mean, rstd = torch.zeros(rows, device="cuda"), torch.ones(rows, device="cuda")
    w = torch.ones(d, device="cuda")
    _, dw, db = ops.layer_norm_backward(_place(dy, gap), _place(x, gap), w, mean, rstd)
    want = _columns(dy, x, mean, rstd)
    assert torch.equal(dw.double(), want[0]), "weight"
    assert torch.equal(db.double(), want[1]), "bias"


def _steps(rows, d):
    """Additions, one after the other, that a column's sum goes through at most: a group's rows, the groups
    of a wave (pairs), the parts of a block, and 64 lanes over the blocks' partial sums."""
    units = 2 * UNITS
    if d > 16384:
        blocks = min(rows, units)
        return -(-rows // blocks) + -(-blocks // 64) + 6
    group = next(t for t, most in ((8, 64), (16, 128), (32, 256), (64, 1024), (128, 2048), (256, 4096), (512, 8192), (1024, 16384))
                 if d <= most)
    threads = max(512, group)
    groups = threads // group
    blocks = min(-(-rows // groups), units)
    if blocks <= 4:
        blocks = 1
    pairs = {8: 3, 16: 2, 32: 1}.get(group, 0)
    parts = threads // max(group, 64)
    return -(-rows // (blocks * groups)) + pairs + parts + -(-blocks // 64) + 6


@pytest.mark.parametrize("rows,d", [r for r in ROWS if r[0] < 200_000])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_sums_within_the_roundings_made(rows, d, dtype):
    """Each term carries a difference, a product and the sum's own rounding (3 u), each addition one u of
    what is added up: the bound is the number of additions in a row, not of rows."""
    _need_gpu()
    from luminamoon_amd import ops

    print(f"[case] {rows}x{d} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(rows * 3 + d)
    x = torch.randn(rows, d, generator=g, device="cuda").mul_(1.5).add_(0.3).to(DTYPES[dtype])
    dy = torch.randn(rows, d, generator=g, device="cuda").mul_(0.1).to(DTYPES[dtype])
    w = torch.randn(d, generator=g, device="cuda")
    _, mean, rstd = ops.layer_norm_forward(x, w)
    _, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    want = _columns(dy, x, mean, rstd)
    u = (_steps(rows, d) + 4) * U
    assert ((dw.double() - want[0]).abs() <= u * want[2]).all(), "weight"
    assert ((db.double() - want[1]).abs() <= u * want[3]).all(), "bias"
