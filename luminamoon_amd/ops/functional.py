"""The operators on ROCm tensors, without autograd: checks, output tensors, one C call each on the
device's current stream.

Matrices are read with any row stride and at any offset as long as a row's elements are contiguous and
the leading axes collapse to one; others are copied first. f32, bf16 and f16; sums and statistics are
f32.

Every function first offers its arguments to the C++ module that makes ordinary calls (`_plain`); what
that does not take is checked, copied and refused here.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional, Tuple

import torch

from ..optimizer.hip_backend import _current_stream_handle, _get_device
from .backend import DTYPE_CODES, LAYER_NORM, LOGITS, load_host, load_library, raise_status

MAX_TOP = 128       # LV_OPS_MAX_TOP
MAX_TEACHER = 1024  # LV_OPS_MAX_TEACHER


_host = None
_host_loaded = False


def _plain(name: str, x: torch.Tensor, *args):
    """What the C++ module returns for a call on plain arguments, or None. x: the call's main tensor."""
    global _host, _host_loaded
    if not _host_loaded:
        load_library()  # raises if the operators are not built
        _host, _host_loaded = load_host(), True
    if _host is None or not x.is_cuda:
        return None
    device = _get_device()
    out = getattr(_host, name)(*args, device, _current_stream_handle(device))
    if type(out) is int:
        raise_status(out)
    return out


class TokenLogProbs(NamedTuple):
    """What `token_log_probs_forward` returns; the last two are None without alternatives."""
    log_probs: torch.Tensor
    entropy: torch.Tensor
    stats: torch.Tensor
    top_log_probs: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _matrix(t: torch.Tensor, name: str) -> Tuple[torch.Tensor, int, int, int]:
    """(tensor, rows, width, row stride) of t seen as rows of its last axis."""
    if not t.is_cuda:
        raise RuntimeError(
            f"LuminaV (MI355X build) runs on ROCm device tensors only; {name} is on '{t.device}'. Move it to the GPU first."
        )
    if t.dtype not in DTYPE_CODES:
        raise ValueError(f"LuminaV: unsupported dtype {t.dtype} for {name}.")
    dim = t.dim()
    if dim == 0:
        raise ValueError(f"LuminaV: {name} must have at least one dimension.")
    width = t.shape[-1]
    if width == 0:
        raise ValueError(f"LuminaV: the last axis of {name} must not be empty.")
    if t.is_contiguous():
        return t, t.numel() // width, width, width
    if dim <= 2 and (t.stride(-1) == 1 or width == 1):
        return t, (t.shape[0] if dim == 2 else 1), width, (t.stride(0) if dim == 2 else width)
    if dim > 2 and t.stride(-1) == 1:
        try:
            flat = t.view(-1, width)
            return flat, flat.shape[0], width, flat.stride(0)
        except RuntimeError:
            pass
    t = t.contiguous()
    return t, t.numel() // width, width, width


def _like(t: torch.Tensor, name: str, shape: torch.Size, ref: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """t, contiguous, after checking it."""
    if t.device != ref.device:
        raise ValueError(f"LuminaV: {name} is on {t.device}, expected {ref.device}.")
    if t.dtype is not dtype:
        raise ValueError(f"LuminaV: {name} must have dtype {dtype}, got {t.dtype}.")
    if t.shape != shape:
        raise ValueError(f"Shape mismatch for {name}: expected {tuple(shape)}, got {tuple(t.shape)}.")
    return t if t.is_contiguous() else t.contiguous()


def _tokens(t: torch.Tensor, name: str, shape: torch.Size, ref: torch.Tensor) -> torch.Tensor:
    if t.dtype is torch.int32:
        t = t.to(torch.int64)
    return _like(t, name, shape, ref, torch.int64)


def _call(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) on the device's current stream."""
    index = device.index
    if _get_device() == index:
        rc = fn(*args, _current_stream_handle(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _current_stream_handle(index))
    if rc != 0:
        raise_status(rc)


# ------------------------------------------------------------------------------------- layer norm


def _column_dtype(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], width: int) -> torch.dtype:
    """The dtype of weight and bias, after checking them."""
    dtype = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dtype is not torch.float32 and t.dtype is not x.dtype:
            raise ValueError(f"LuminaV: {name} must be float32 or of x's dtype {x.dtype}, got {t.dtype}.")
        if dtype is not None and t.dtype is not dtype:
            raise ValueError(f"DType mismatch between weight ({dtype}) and bias ({t.dtype}).")
        dtype = t.dtype
        if t.device != x.device:
            raise ValueError(f"LuminaV: {name} is on {t.device}, expected {x.device}.")
        if t.dim() != 1 or t.shape[0] != width:
            raise ValueError(f"Shape mismatch for {name}: expected ({width},), got {tuple(t.shape)}.")
    return torch.float32 if dtype is None else dtype


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """y = (x - mean) rstd weight + bias over the last axis: (y, mean, rstd), the last two f32 of
    x's leading shape, rstd = (var + eps)^-1/2."""
    out = _plain("layer_norm_forward", x, x, weight, bias, eps)
    if out is not None:
        return out
    xm, rows, width, stride = _matrix(x, "x")
    wdtype = _column_dtype(x, weight, bias, width)
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, *x.shape[:-1]), dtype=torch.float32, device=x.device)
    mean, rstd = stats[0], stats[1]
    args = LAYER_NORM.pack(xm.data_ptr(), 0, y.data_ptr(), _ptr(weight), _ptr(bias), mean.data_ptr(), rstd.data_ptr(), 0, 0,
                           rows, width, stride, 0, width, eps, DTYPE_CODES[x.dtype], DTYPE_CODES[wdtype], 0)
    _call(load_library().lv_layer_norm_forward, x.device, args)
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                        rstd: torch.Tensor, need_x: bool = True, need_weight: bool = True, need_bias: bool = True,
                        dtype: Optional[torch.dtype] = None,
                        ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dweight, dbias) of `layer_norm_forward` from its mean and rstd; None where not wanted.
    dweight and dbias have the weight's dtype, or `dtype` (f32) without a weight."""
    out = _plain("layer_norm_backward", x, dy, x, weight, mean, rstd, need_x, need_weight, need_bias)
    if out is not None:
        return out
    xm, rows, width, stride = _matrix(x, "x")
    if dy.shape != x.shape:
        raise ValueError(f"Shape mismatch for dy: expected {tuple(x.shape)}, got {tuple(dy.shape)}.")
    if dy.device != x.device:
        raise ValueError(f"LuminaV: dy is on {dy.device}, expected {x.device}.")
    if dy.dtype is not x.dtype:
        raise ValueError(f"DType mismatch between x ({x.dtype}) and dy ({dy.dtype}).")
    dm, _, _, dy_stride = _matrix(dy, "dy")
    wdtype = _column_dtype(x, weight, None, width)
    if weight is None and dtype is not None:
        if dtype is not torch.float32 and dtype is not x.dtype:
            raise ValueError(f"LuminaV: dtype must be float32 or x's dtype {x.dtype}, got {dtype}.")
        wdtype = dtype
    elif weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    mean = _like(mean, "mean", x.shape[:-1], x, torch.float32)
    rstd = _like(rstd, "rstd", x.shape[:-1], x, torch.float32)
    device = x.device
    dx = torch.empty(x.shape, dtype=x.dtype, device=device) if need_x else None
    dw = torch.empty(width, dtype=wdtype, device=device) if need_weight else None
    db = torch.empty(width, dtype=wdtype, device=device) if need_bias else None
    lib = load_library()
    args = LAYER_NORM.pack(xm.data_ptr(), dm.data_ptr(), _ptr(dx), _ptr(weight), 0, mean.data_ptr(), rstd.data_ptr(),
                           _ptr(dw), _ptr(db), rows, width, stride, dy_stride, width, 0.0, DTYPE_CODES[x.dtype],
                           DTYPE_CODES[wdtype], 0)
    ws = None
    nbytes = 0
    if need_weight or need_bias:
        nbytes = lib.lv_layer_norm_workspace_bytes(args)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _call(lib.lv_layer_norm_backward, device, args, _ptr(ws), nbytes)
    return dx, dw, db


# ------------------------------------------------------------------------------------- logits


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(distill: bool, device: int, rows: int, vocab: int, count: int, code: int) -> int:
    """Workspace of a forward call: a function of its sizes (and of the device's)."""
    lib = load_library()
    args = LOGITS.pack(*(0,) * 13, rows, vocab, vocab, vocab, 1.0, 1.0, count, code, 0, 0)
    with torch.cuda.device(device):
        return (lib.lv_distill_workspace_bytes if distill else lib.lv_token_log_probs_workspace_bytes)(args)


def _workspace(distill: bool, logits: torch.Tensor, rows: int, vocab: int, count: int) -> Tuple[Optional[torch.Tensor], int]:
    n = _workspace_bytes(distill, logits.device.index, rows, vocab, count, DTYPE_CODES[logits.dtype])
    return (torch.empty(n, dtype=torch.uint8, device=logits.device) if n else None), n


def token_log_probs_forward(logits: torch.Tensor, tokens: torch.Tensor, temperature: float = 1.0,
                            top: int = 0) -> TokenLogProbs:
    """Of p = softmax(logits / temperature) over the last axis: the log probability of each position's
    token (0 for a token outside the vocabulary, such as -100), the entropy, the row statistics that
    the backward pass takes ([..., 2]: largest logit, log sum), and the `top` most likely tokens with
    their log probabilities, most likely first, the lowest index first among equals."""
    out = _plain("token_log_probs_forward", logits, logits, tokens, temperature, top)
    if out is not None:
        return TokenLogProbs(*out)
    z, rows, vocab, stride = _matrix(logits, "logits")
    lead = logits.shape[:-1]
    tokens = _tokens(tokens, "tokens", lead, logits)
    device = logits.device
    # apart: views of one tensor could not be changed in place once autograd returns them
    log_probs = torch.empty(lead, dtype=torch.float32, device=device)
    entropy = torch.empty(lead, dtype=torch.float32, device=device)
    stats = torch.empty((*lead, 2), dtype=torch.float32, device=device)
    top = int(top)
    values = index = None
    if 0 < top <= min(MAX_TOP, vocab):
        values = torch.empty((*lead, top), dtype=torch.float32, device=device)
        index = torch.empty((*lead, top), dtype=torch.int64, device=device)
        ws, nbytes = _workspace(False, logits, rows, vocab, top)
    elif top == 0:
        ws, nbytes = _workspace(False, logits, rows, vocab, 0)
    else:
        raise ValueError(f"LuminaV: top must be between 0 and {min(MAX_TOP, vocab)}, got {top}.")
    args = LOGITS.pack(z.data_ptr(), tokens.data_ptr(), 0, 0, 0, 0, 0, log_probs.data_ptr(), entropy.data_ptr(),
                       stats.data_ptr(), _ptr(values), _ptr(index), 0, rows, vocab, stride, 0, temperature, 1.0, top,
                       DTYPE_CODES[logits.dtype], 0, 0)
    _call(load_library().lv_token_log_probs_forward, device, args, _ptr(ws), nbytes)
    return TokenLogProbs(log_probs, entropy, stats, values, index)


def token_log_probs_backward(d_log_probs: Optional[torch.Tensor], d_entropy: Optional[torch.Tensor], logits: torch.Tensor,
                             tokens: torch.Tensor, stats: torch.Tensor, entropy: torch.Tensor,
                             temperature: float = 1.0) -> torch.Tensor:
    """The logits' gradient from those of the log probabilities and the entropy (f32; None: zero), with
    the statistics and the entropy that `token_log_probs_forward` returned."""
    out = _plain("token_log_probs_backward", logits, d_log_probs, d_entropy, logits, tokens, stats, entropy, temperature)
    if out is not None:
        return out
    z, rows, vocab, stride = _matrix(logits, "logits")
    lead = logits.shape[:-1]
    tokens = _tokens(tokens, "tokens", lead, logits)
    if d_log_probs is not None:
        d_log_probs = _like(d_log_probs, "d_log_probs", lead, logits, torch.float32)
    if d_entropy is not None:
        d_entropy = _like(d_entropy, "d_entropy", lead, logits, torch.float32)
    stats = _like(stats, "stats", torch.Size((*lead, 2)), logits, torch.float32)
    entropy = _like(entropy, "entropy", lead, logits, torch.float32)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    args = LOGITS.pack(z.data_ptr(), tokens.data_ptr(), 0, 0, 0, _ptr(d_log_probs), _ptr(d_entropy), 0, entropy.data_ptr(),
                       stats.data_ptr(), 0, 0, grad.data_ptr(), rows, vocab, stride, vocab, temperature, 1.0, 0,
                       DTYPE_CODES[logits.dtype], 0, 0)
    _call(load_library().lv_token_log_probs_backward, logits.device, args)
    return grad


def _teacher(logits: torch.Tensor, tokens: torch.Tensor, values: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, int]:
    lead = logits.shape[:-1]
    if tokens.dim() == 0:
        raise ValueError("Shape mismatch for teacher_tokens: expected the logits' leading shape and one more axis.")
    count = tokens.shape[-1]
    if not 1 <= count <= MAX_TEACHER:
        raise ValueError(f"LuminaV: a teacher gives 1 to {MAX_TEACHER} logits per row, got {count}.")
    shape = torch.Size((*lead, count))
    tokens = _tokens(tokens, "teacher_tokens", shape, logits)
    if values.dtype not in DTYPE_CODES:
        raise ValueError(f"LuminaV: unsupported dtype {values.dtype} for teacher_logits.")
    return tokens, _like(values, "teacher_logits", shape, logits, values.dtype), count


def _row_weight(weight, lead: torch.Size, ref: torch.Tensor) -> Tuple[float, Optional[torch.Tensor]]:
    if isinstance(weight, torch.Tensor):
        return 1.0, _like(weight, "weight", lead, ref, torch.float32)
    return float(weight), None


def distill_loss_forward(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_logits: torch.Tensor,
                         temperature: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Distillation from a teacher's k logits per position: with q = softmax(teacher_logits /
    temperature) over the entries whose token is in the vocabulary (others, such as -100, are padding)
    and p = softmax(logits / temperature) over all of it, temperature^2 KL(q || p) per position, and
    the row statistics that the backward pass takes. A position without a teacher has loss 0. The
    teacher's values may be log probabilities."""
    out = _plain("distill_loss_forward", logits, logits, teacher_tokens, teacher_logits, temperature)
    if out is not None:
        return out
    z, rows, vocab, stride = _matrix(logits, "logits")
    tokens, values, count = _teacher(logits, teacher_tokens, teacher_logits)
    lead = logits.shape[:-1]
    loss = torch.empty(lead, dtype=torch.float32, device=logits.device)
    stats = torch.empty((*lead, 2), dtype=torch.float32, device=logits.device)
    ws, nbytes = _workspace(True, logits, rows, vocab, count)
    args = LOGITS.pack(z.data_ptr(), 0, tokens.data_ptr(), values.data_ptr(), 0, 0, 0, loss.data_ptr(), 0, stats.data_ptr(),
                       0, 0, 0, rows, vocab, stride, 0, temperature, 1.0, count, DTYPE_CODES[logits.dtype],
                       DTYPE_CODES[values.dtype], 0)
    _call(load_library().lv_distill_forward, logits.device, args, _ptr(ws), nbytes)
    return loss, stats


def distill_loss_backward(weight, logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_logits: torch.Tensor,
                          stats: torch.Tensor, temperature: float = 1.0) -> torch.Tensor:
    """The logits' gradient of sum(weight * loss), weight a number or an f32 tensor with one value per
    position, from the statistics that `distill_loss_forward` returned."""
    out = _plain("distill_loss_backward", logits, weight, logits, teacher_tokens, teacher_logits, stats, temperature)
    if out is not None:
        return out
    z, rows, vocab, stride = _matrix(logits, "logits")
    tokens, values, count = _teacher(logits, teacher_tokens, teacher_logits)
    lead = logits.shape[:-1]
    scalar, per_row = _row_weight(weight, lead, logits)
    stats = _like(stats, "stats", torch.Size((*lead, 2)), logits, torch.float32)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    args = LOGITS.pack(z.data_ptr(), 0, tokens.data_ptr(), values.data_ptr(), _ptr(per_row), 0, 0, 0, 0, stats.data_ptr(),
                       0, 0, grad.data_ptr(), rows, vocab, stride, vocab, temperature, scalar, count,
                       DTYPE_CODES[logits.dtype], DTYPE_CODES[values.dtype], 0)
    _call(load_library().lv_distill_backward, logits.device, args)
    return grad


def distill_loss_and_grad(logits: torch.Tensor, teacher_tokens: torch.Tensor, teacher_logits: torch.Tensor,
                          temperature: float = 1.0, weight=1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss per position, the logits' gradient of sum(weight * loss)) in one call, for a training loop
    that knows its weights (a number or an f32 tensor with one value per position) beforehand."""
    out = _plain("distill_loss_and_grad", logits, logits, teacher_tokens, teacher_logits, temperature, weight)
    if out is not None:
        return out
    z, rows, vocab, stride = _matrix(logits, "logits")
    tokens, values, count = _teacher(logits, teacher_tokens, teacher_logits)
    lead = logits.shape[:-1]
    scalar, per_row = _row_weight(weight, lead, logits)
    loss = torch.empty(lead, dtype=torch.float32, device=logits.device)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    ws, nbytes = _workspace(True, logits, rows, vocab, count)
    args = LOGITS.pack(z.data_ptr(), 0, tokens.data_ptr(), values.data_ptr(), _ptr(per_row), 0, 0, loss.data_ptr(), 0, 0,
                       0, 0, grad.data_ptr(), rows, vocab, stride, vocab, temperature, scalar, count,
                       DTYPE_CODES[logits.dtype], DTYPE_CODES[values.dtype], 0)
    _call(load_library().lv_distill_loss_and_grad, logits.device, args, _ptr(ws), nbytes)
    return loss, grad
