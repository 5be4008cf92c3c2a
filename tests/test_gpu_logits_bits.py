"""Which results over rows of logits are equal to the bit: the same rows in another place, at another
stride, in another number. 16-bit rows are read on 4-byte words, so where a row begins half way into one
its sums are of other groups of logits, and their last bits may differ."""
from __future__ import annotations

import pytest
import torch

from tests.ops_util import DTYPES, ROUND, U, distill_grad_ref, entropy_tol, log_prob_tol, teacher_ref

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


def _inputs(rows, v, dtype, seed, k=9):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(rows, v, generator=g) * 2.0 - 1.0).to(DTYPES[dtype]).cuda()
    tokens = torch.randint(0, v, (rows,), generator=g).cuda()
    tt = torch.randint(0, v, (rows, k), generator=g).cuda()
    return z, tokens, tt, torch.randn(rows, k, generator=g).cuda()


def _view(z, offset, gap):
    """z's rows at an offset of so many logits and so many more between them, NaN there."""
    rows, v = z.shape
    buf = torch.full((offset + rows * (v + gap),), NAN, dtype=z.dtype, device="cuda")
    out = buf[offset:].view(rows, v + gap)[:, :v]
    out.copy_(z)
    return out


def _everything(z, tokens, tt, tl, top):
    """Every result of the operators over these rows, by name."""
    from luminamoon_amd import ops

    ones = torch.ones(z.shape[0], device="cuda")
    out = ops.token_log_probs_forward(z, tokens, top=top)
    loss, stats = ops.distill_loss_forward(z, tt, tl)
    one, grad = ops.distill_loss_and_grad(z, tt, tl)
    return dict(out._asdict(), log_probs_grad=ops.token_log_probs_backward(ones, ones, z, tokens, out.stats, out.entropy),
                loss=loss, loss_stats=stats, loss_grad=ops.distill_loss_backward(1.0, z, tt, tl, stats), one=one, grad=grad)


def _same(a, b, what):
    for name, t in a.items():
        assert torch.equal(t, b[name]), f"{what}: {name}"


SIZES = [(5, 1003), (6, 1004), (3, 33000), (1100, 257), (9, 50257), (2, 140001), (2, 9), (40, 20011)]


@pytest.mark.parametrize("rows,v", SIZES)
@pytest.mark.parametrize("offset,gap", [(0, 1), (1, 3), (3, 8), (2, 47), (0, 64)])
def test_f32_rows_anywhere(rows, v, offset, gap):
    """f32 rows give the packed rows' bits at any offset and stride."""
    _need_gpu()
    z, tokens, tt, tl = _inputs(rows, v, "f32", v)
    _same(_everything(z, tokens, tt, tl, 4), _everything(_view(z, offset, gap), tokens, tt, tl, 4), f"{rows}x{v}")


@pytest.mark.parametrize("rows,v", SIZES)
@pytest.mark.parametrize("offset,gap", [(0, 2), (2, 8), (4, 64), (6, 46)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_rows_that_begin_on_words_alike(rows, v, offset, gap, dtype):
    """16-bit rows give the packed rows' bits wherever each begins at the same half of a word."""
    _need_gpu()
    z, tokens, tt, tl = _inputs(rows, v, dtype, v)
    _same(_everything(z, tokens, tt, tl, 4), _everything(_view(z, offset, gap), tokens, tt, tl, 4), f"{rows}x{v} {dtype}")


def _close(a, b, z, tt, tl, v):
    """Results of equal rows within twice what either may be off by, for logits z of either."""
    zc, ttc, tlc = z.cpu(), tt.cpu(), tl.cpu()
    tol, row, d, p = log_prob_tol(zc, 1.0)
    q, lq, _ = teacher_ref(ttc, tlc, v, 1.0)
    step = ROUND[z.dtype][0]
    at = ttc.clamp(0, v - 1)
    # a sum of k terms q (log q - log p), each off by log p's tolerance and a few roundings of its own
    lp = torch.log_softmax(zc.double(), -1).gather(-1, at)
    q_rel = U * (64 + 8 * tlc.double().abs().amax(-1, keepdim=True))
    allow = {"log_probs": tol.amax(-1), "entropy": entropy_tol(row, d, p), "top_log_probs": tol.amax(-1, keepdim=True),
             "loss": (q * (tol.gather(-1, at) + q_rel * (2 + lq.abs() + lp.abs()))).sum(-1)}
    allow["one"] = allow["loss"]
    _, dense = distill_grad_ref(zc, ttc, tlc, 1.0, torch.ones(z.shape[0], dtype=torch.float64))
    allow["grad"] = (tol + 16 * U) * p + torch.zeros_like(p).scatter_add_(-1, at, q * q_rel) + 4 * U * dense
    for name, t in allow.items():
        x, y = a[name].double().cpu(), b[name].double().cpu()
        rounding = (step if name == "grad" else U) * (x.abs() + y.abs()) + (2 * ROUND[z.dtype][1] if name == "grad" else 0.0)
        assert ((x - y).abs() <= 2 * t + rounding + 1e-37).all(), name
    for name in ("stats", "loss_stats"):
        assert torch.equal(a[name][:, 0], b[name][:, 0]), name
        assert ((a[name] - b[name])[:, 1].cpu().double().abs() <= 2 * row).all(), name
    assert torch.equal(a["top_tokens"], b["top_tokens"])


@pytest.mark.parametrize("v", [257, 1003, 20011, 50257, 140001])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_equal_16_bit_rows_of_an_odd_vocabulary(v, dtype):
    """Equal rows with equal teachers, even and odd numbers of rows apart: an even number of rows of an
    odd vocabulary keeps the half of the word and so the bits; an odd one does not, and the results are
    within the tolerance of either. The alternatives and the largest logits are always the same."""
    _need_gpu()
    z, tokens, tt, tl = (t[torch.zeros(7, dtype=torch.int64, device="cuda")] for t in _inputs(1, v, dtype, v))
    every = _everything(z, tokens, tt, tl, 8)
    for r in range(2, 7):
        for name, t in every.items():
            assert torch.equal(t[r], t[r - 2]), (name, r)
    halves = [{name: t[half::2][:3] for name, t in every.items()} for half in (0, 1)]
    _close(halves[0], halves[1], z[:3], tt[:3], tl[:3], v)


@pytest.mark.parametrize("v", [12000, 32000, 70001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_same_rows_among_few_and_many(v, dtype):
    """The number of rows decides how a row is cut, and with it the last bits; alternatives and largest
    logits stay the same, the rest within the tolerance."""
    _need_gpu()
    z, tokens, tt, tl = _inputs(6, v, dtype, v)
    few = _everything(z, tokens, tt, tl, 8)
    index = torch.arange(2100, device="cuda") % 6
    many = _everything(z[index], tokens[index], tt[index], tl[index], 8)
    _close(few, {name: t[:6] for name, t in many.items()}, z, tt, tl, v)
