"""Faults that the operators once had: each test here failed before its fault was mended."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no ROCm GPU")


@pytest.mark.parametrize("how", ["plain", "int32 tokens", "transposed logits", "a slice of positions"])
def test_results_can_be_changed_in_place(how):
    """Log probabilities masked in place, as a loss over some positions does, whichever way the call
    takes; the entropy, saved for the backward pass, keeps its own storage and version."""
    _need_gpu()
    from luminamoon_amd import ops

    g = torch.Generator().manual_seed(0)
    z = torch.randn(3, 5, 40, generator=g).cuda()
    if how == "transposed logits":
        z = z.transpose(0, 1)
    elif how == "a slice of positions":
        z = z[:, :-1]
    tokens = torch.randint(0, 40, z.shape[:-1], generator=g).cuda()
    if how == "int32 tokens":
        tokens = tokens.int()
    mask = (torch.rand(z.shape[:-1], generator=g) < 0.5).float().cuda()
    z = z.detach().requires_grad_()
    scores = ops.token_log_probs(z, tokens)
    assert scores.log_probs._base is None and scores.entropy._base is None
    scores.log_probs.mul_(mask)
    (scores.log_probs - 0.1 * scores.entropy).sum().backward()
    got, z.grad = z.grad, None
    scores = ops.token_log_probs(z, tokens)
    (scores.log_probs * mask - 0.1 * scores.entropy).sum().backward()
    assert torch.equal(got, z.grad)


def _us(call, calls=10, rounds=5):
    """The smallest time of a call over a few rounds, back to back."""
    call()
    best = float("inf")
    for _ in range(rounds):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(calls):
            call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / calls)
    return best


@pytest.mark.parametrize("rows,v", [(1, 32000), (1024, 32000), (8192, 4000), (256, 131072), (4096, 12000), (2048, 1000), (2048, 500)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_alternatives_of_rows_with_an_offset(rows, v, dtype):
    """An offset common to a row's logits changes neither the alternatives nor what the search for them
    costs: its bound and the vectors' largest logits were cut to 16 bits of f32 once, which most of such
    a row reached (up to 12 times as long; three times is allowed). The logits lie on steps that every
    offset keeps."""
    _need_gpu()
    from luminamoon_amd import ops
    from tests.ops_util import DTYPES

    g = torch.Generator().manual_seed(v)
    step = 2.0 ** -10 if dtype == "f32" else 0.5
    base = ((torch.randn(min(rows, 64), v, generator=g) / step).round() * step).cuda()
    base = base[torch.arange(rows, device="cuda") % base.shape[0]]
    tokens = torch.zeros(rows, dtype=torch.int64, device="cuda")
    for top in (8, 20, 64, 128):
        here = {}
        for offset in (0.0, 500.0, -1000.0):
            z = (base + offset).to(DTYPES[dtype])
            print(f"[case] {rows}x{v} {dtype} top {top} offset {offset}", flush=True)
            out = ops.token_log_probs_forward(z, tokens, top=top)
            want = torch.sort(z[:64].double(), dim=-1, descending=True, stable=True).indices[:, :top]
            assert torch.equal(out.top_tokens[:64], want)
            here[offset] = _us(lambda: ops.token_log_probs_forward(z, tokens, top=top))
        print(f"[time] {rows}x{v} {dtype} top {top} {here}", flush=True)
        assert max(here.values()) < 3 * here[0.0], here


def _graph_us(call, calls=20, replays=5):
    """A call's time on the GPU alone: the smallest of a few replays of many in a graph."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    return min(_us(graph.replay, calls=1) for _ in range(replays)) / calls


@pytest.mark.parametrize("rows,d,one_row", [(32, 768, 8), (4, 16384, 1), (4, 8192, 1), (64, 256, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_gradient_of_x_alone_uses_more_than_one_block(rows, d, one_row, dtype):
    """With frozen weights no columns' sums are wanted, and rows spread over blocks; one block walked
    them all before. A block has as many rows as it takes at a time: all take as long as one such block,
    where a walk takes two to three times that (1.6 is allowed). The gradient is the same to the bit."""
    _need_gpu()
    from luminamoon_amd import ops
    from tests.ops_util import DTYPES

    g = torch.Generator().manual_seed(d)
    x, dy = (torch.randn(rows, d, generator=g).to(DTYPES[dtype]).cuda() for _ in range(2))
    w = torch.randn(d, generator=g).cuda()
    _, mean, rstd = ops.layer_norm_forward(x, w)
    dx = ops.layer_norm_backward(dy, x, w, mean, rstd, True, False, False)[0]
    assert torch.equal(dx, ops.layer_norm_backward(dy, x, w, mean, rstd)[0])
    many = _graph_us(lambda: ops.layer_norm_backward(dy, x, w, mean, rstd, True, False, False))
    few = [t[:one_row] for t in (dy, x, mean, rstd)]
    one = _graph_us(lambda: ops.layer_norm_backward(few[0], few[1], w, few[2], few[3], True, False, False))
    print(f"[time] {rows}x{d} {dtype} {many:.2f} us, {one_row} rows {one:.2f} us", flush=True)
    assert many < 1.6 * one
