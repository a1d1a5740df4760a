"""Class / vocabulary operators on the GPU: what a model of classes is trained with and answers through.

The framework prepares what a model trains on and runs the classifier's forward pass
(:class:`ser_amd.GpuEmotionClassifier`); these are the operators on the class side of such a model, from the eight
emotions of the fast profile to the tokens of a transcript decoder behind :func:`ser_amd.log_mel_spectrogram`:

* :func:`sample_tokens` -- one class per row of scores, with temperature, top-k, top-p and min-p, from given uniform
  numbers; also the log-probability that a decoder's confidence check adds up
* :func:`distillation_loss` (differentiable) and :func:`distillation_step` (loss and gradient in one call) -- a student
  against a teacher's top logits
* :func:`embed_tokens` (differentiable) and :func:`embedding_gradient` -- the lookup that turns tokens into a model's
  input, and the gradient of its table

They have no counterpart in the reference (its classifier is trained by sklearn, its transcript lane is a third-party
package).  All take torch tensors on one GPU -- float32, bfloat16 or float16 scores and tables, rows of any stride -- and
launch the kernels of ``libserhip.so`` (``include/serhip.h``) on torch's current stream of that GPU; nothing
synchronises, so every call can be captured into a graph (after any first call on that GPU, which sets up its engine;
a whole training step is best captured as :func:`distillation_step` and :func:`embedding_gradient`, without autograd).
There is no CPU path: a tensor elsewhere is a ``ValueError``.  Results do not depend on what else runs: equal calls give
equal bits.
"""

from __future__ import annotations

import functools
import math
import os

import torch
from torch.autograd import forward_ad

from . import _native
from .engine import _engines, get_engine

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_INT_MAX = (1 << 31) - 1
_MAX_CLASSES = 1 << 24
_MAX_TEACHER = 2048
_LEAST_TEMPERATURE = 1e-30


# the address of torch's current stream; the public way costs as much as a launch (2.7 us against 0.1)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


# ------------------------------------------------------------------------------------------- arguments
def _require(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _check_tensor(t, name: str, dtypes, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a torch tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors are on {device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has dtype {t.dtype}; supported: {', '.join(str(d) for d in dtypes)}")
    if t.layout != torch.strided:
        raise ValueError(f"{name} must be a dense tensor")


def _require_no_tangent(t, name: str) -> None:
    # (outside a dual level nothing has one: asked of the module, which takes a tenth of unpack_dual's 0.6 us)
    if getattr(forward_ad, "_current_level", 0) >= 0:
        _require(forward_ad.unpack_dual(t).tangent is None, f"{name} has a tangent: there is no forward-mode derivative")


def _engine_of(t, name: str):
    """The engine of the tensor's GPU: the last check of a call."""
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be on the GPU (it is on {t.device}); there is no CPU path")
    index = t.device.index
    return _engines.get((os.getpid(), index)) or get_engine(index)


def _rows(t):
    """``[..., n]`` -> ``[rows, n]`` with contiguous rows, without a copy where the strides allow it."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((math.prod(t.shape[:-1]), t.shape[-1]))
    return t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous()


def _stride(t) -> int:
    """Elements from one row to the next (one row's own stride may be anything)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _call(engine, function, *args) -> None:
    """One library call on torch's current stream of the engine's device."""
    index = engine.device_index
    if torch.cuda.current_device() == index:
        status = function(engine._ctx.handle, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(engine._ctx.handle, *args, _raw_stream(index))
    if status < 0:
        _native.check(status)


def _written(t) -> None:
    """Tells autograd that ``t`` holds something else now: a kernel wrote to its address."""
    if not t.is_inference():   # (these keep no version)
        torch.autograd.graph.increment_version(t)


def _workspace(nbytes: int, device):
    """Scratch of one call, from torch's stream-ordered allocator."""
    return torch.empty((max(int(nbytes), 1),), dtype=torch.uint8, device=device)


# -------------------------------------------------------------------------------------------- sampling
def _number(value, name: str, most: float) -> float:
    number = float(value)
    _require(0.0 <= number <= most, f"{name} must be in 0..{most:g}, got {value!r}")   # (NaN is not)
    return number


def _per_row(value, name: str, shape, device, whole: bool = False):
    """A setting's per-row tensor as the kernel takes it."""
    _require(value.device == device, f"{name} must be on {device}, the device of logits")
    _require(tuple(value.shape) == shape, f"{name} must be a number or have shape {shape}, got {tuple(value.shape)}")
    if not whole:
        _require(value.is_floating_point(), f"{name} must hold floating-point numbers")
        if value.dtype == torch.float64 and name == "temperature":   # what float32 would round to 0 is not greedy
            value = torch.where(value > 0, value.clamp(min=_LEAST_TEMPERATURE), value)
        return value.to(torch.float32).contiguous()
    _require(value.dtype in (torch.int8, torch.uint8, torch.int16, torch.int32, torch.int64), f"{name} must hold whole numbers")
    if value.dtype == torch.int64:
        value = value.clamp(-_INT_MAX, _INT_MAX)
    return value.to(torch.int32).contiguous()


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """``(tokens int64 [...], logprobs float32 [...])`` for scores ``logits [..., classes]`` and ``uniform [...]``
    (float32 in [0, 1), one number per row).

    The classes are ordered by (score descending, index ascending); the first ``top_k`` are kept (0: all), of these the
    shortest prefix whose probability at ``temperature`` reaches ``top_p`` of theirs (at least one), of these those
    at least ``min_p`` times as likely as the likeliest.  The token is the first kept class, in index order, whose
    cumulative probability exceeds ``uniform``.  ``temperature`` 0 takes the first largest score.  Every setting is a
    number, or a tensor ``[...]`` with one value per row (there, a value out of range switches the setting off, and a
    temperature out of range is greedy).  A temperature between 0 and 1e-30 does as 1e-30.

    Probabilities are held in 64 bits; a class that is less than 2^-45 times as likely as the likeliest (2^-38 at 2^24
    classes) may count as impossible.

    NaN and -inf scores are masked classes.  A row without any other gives token -1 and log-probability -inf.
    ``logprobs`` is ``log_softmax(logits)[token]`` of the scores as they are -- the number that a decoder's
    temperature fallback averages -- from a sum in 32 bits, and carries no gradient.
    """
    _check_tensor(logits, "logits", _DTYPES)
    _require(logits.dim() >= 1 and 1 <= logits.shape[-1] <= _MAX_CLASSES, "logits must be [..., classes] with 1 to 2^24 classes")
    device, shape = logits.device, tuple(logits.shape[:-1])
    _check_tensor(uniform, "uniform", (torch.float32,), device)
    _require(tuple(uniform.shape) == shape, f"uniform must have shape {shape}, got {tuple(uniform.shape)}")
    t, k, p, m = 1.0, 0, 1.0, 0.0
    t_rows = k_rows = p_rows = m_rows = None
    if isinstance(temperature, torch.Tensor):
        temperature = _per_row(temperature, "temperature", shape, device)   # (the name keeps it alive)
        t_rows = temperature.data_ptr()
    else:
        t = _number(temperature, "temperature", 3.0e38)
        if 0.0 < t < _LEAST_TEMPERATURE:   # (float32 would round some of them to 0, which is greedy)
            t = _LEAST_TEMPERATURE
    if isinstance(top_k, torch.Tensor):
        top_k = _per_row(top_k, "top_k", shape, device, whole=True)
        k_rows = top_k.data_ptr()
    else:
        k = -1 if isinstance(top_k, float) and not math.isfinite(top_k) else int(top_k)
        _require(k == top_k and k >= 0, f"top_k must be a whole number >= 0, got {top_k!r}")
        k = min(k, _INT_MAX)
    if isinstance(top_p, torch.Tensor):
        top_p = _per_row(top_p, "top_p", shape, device)
        p_rows = top_p.data_ptr()
    else:
        p = _number(top_p, "top_p", 1.0)
    if isinstance(min_p, torch.Tensor):
        min_p = _per_row(min_p, "min_p", shape, device)
        m_rows = min_p.data_ptr()
    else:
        m = _number(min_p, "min_p", 1.0)
    engine = _engine_of(logits, "logits")
    token = torch.empty(shape, dtype=torch.int64, device=device)
    logprob = torch.empty(shape, dtype=torch.float32, device=device)
    if token.numel():
        x, u = _rows(logits), uniform.contiguous()
        _call(engine, engine._lib.serhip_sample, x.data_ptr(), _DTYPES[x.dtype], x.shape[0], x.shape[1], _stride(x),
              u.data_ptr(), t, k, p, m, t_rows, k_rows, p_rows, m_rows, token.data_ptr(), logprob.data_ptr())
    return token, logprob


# ---------------------------------------------------------------------------------------- distillation
def _check_distill(logits, teacher_index, teacher_logits, temperature):
    """Checks in the caller's grad mode: (engine, temperature)."""
    _check_tensor(logits, "logits", _DTYPES)
    _require(logits.dim() >= 1 and 1 <= logits.shape[-1] <= _MAX_CLASSES, "logits must be [..., classes] with 1 to 2^24 classes")
    _check_tensor(teacher_index, "teacher_index", (torch.int64, torch.int32), logits.device)
    _check_tensor(teacher_logits, "teacher_logits", _DTYPES, logits.device)
    _require(teacher_index.dim() >= 1 and teacher_index.shape[:-1] == logits.shape[:-1]
             and 1 <= teacher_index.shape[-1] <= _MAX_TEACHER,
             f"teacher_index must be {tuple(logits.shape[:-1])} + (entries,) with 1 to {_MAX_TEACHER} entries, "
             f"got {tuple(teacher_index.shape)}")
    _require(teacher_logits.shape == teacher_index.shape,
             f"teacher_logits must have the shape of teacher_index {tuple(teacher_index.shape)}, got {tuple(teacher_logits.shape)}")
    _require(not (teacher_logits.requires_grad and torch.is_grad_enabled()),
             "no gradient flows to the teacher: pass teacher_logits.detach()")
    temperature = float(temperature)
    _require(1e-3 <= temperature <= 1e3, f"temperature must be in 1e-3..1e3, got {temperature!r}")
    return _engine_of(logits, "logits"), temperature


def _distill_head(x, index, teacher, temperature):
    """What every call begins with, for logits as rows and contiguous entries."""
    return (x.data_ptr(), _DTYPES[x.dtype], x.shape[0], x.shape[1], _stride(x), index.data_ptr(),
            int(index.dtype == torch.int64), teacher.data_ptr(), _DTYPES[teacher.dtype], index.shape[-1], temperature)


@functools.lru_cache(maxsize=256)
def _distill_workspace(rows: int, classes: int, dtype: int) -> int:
    return _native.check(_native.load_library().serhip_distill_workspace(rows, classes, dtype))


def _loss_and_stats(engine, shape, x, head):
    """The loss, and what begins with the statistics of its rows (8 bytes for each; the call's scratch lies behind them: one
    allocation takes 2 us)."""
    rows, device = x.shape[0], x.device
    loss = torch.empty(shape, dtype=torch.float32, device=device)
    scratch = _distill_workspace(rows, x.shape[1], head[1])
    behind = (8 * rows + 255) // 256 * 256
    stats = _workspace(behind + scratch, device)
    if rows:
        at = stats.data_ptr()
        _call(engine, engine._lib.serhip_distill_loss, *head, loss.data_ptr(), at, at + behind, scratch)
    return loss, stats


class _DistillationLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, teacher_index, teacher_logits, temperature, engine):
        x, index, teacher = _rows(logits), teacher_index.contiguous(), teacher_logits.contiguous()
        head = _distill_head(x, index, teacher, temperature)
        loss, stats = _loss_and_stats(engine, logits.shape[:-1], x, head)
        ctx.call = engine, logits.shape, head
        # autograd keeps, offloads and frees these, and raises an error in backward if one of them was changed; of logits
        # whose rows had to be copied, the copy
        ctx.save_for_backward(logits if x is logits or x.data_ptr() == logits.data_ptr() else x, index, teacher, stats)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        logits, index, teacher, stats = ctx.saved_tensors
        engine, shape, head = ctx.call
        x = _rows(logits)
        weight = grad_loss.contiguous()   # (float32, as the loss is)
        grad = torch.empty(shape, dtype=x.dtype, device=x.device)
        if x.shape[0]:   # the sizes and types of the forward call; addresses and stride of what autograd hands back
            _call(engine, engine._lib.serhip_distill_gradient, x.data_ptr(), *head[1:4], _stride(x), index.data_ptr(), head[6],
                  teacher.data_ptr(), *head[8:], stats.data_ptr(), weight.data_ptr(), grad.data_ptr(), head[3])
        return grad, None, None, None, None


def distillation_loss(logits, teacher_index, teacher_logits, *, temperature=1.0):
    """Loss ``[...]`` (float32) of a student's ``logits [..., classes]`` against a teacher's top logits: classes
    ``teacher_index [..., k]`` (int32 or int64) with logits or log-probabilities ``teacher_logits [..., k]``.

    With ``p`` the softmax of the row's ``k`` teacher entries and ``q`` the softmax of all student logits, both at
    ``temperature``: ``temperature**2 * sum(p * (log p - log q[index]))``.  Differentiable once, in backward mode, with respect
    to ``logits`` (its gradient has their dtype; the forward pass keeps two numbers per row).  An entry whose index is
    outside the classes (padding, -1) or whose logit is -inf does not count, a row without entries has loss 0 and
    gradient 0, a row whose incoming gradient is 0 gets a gradient of 0 whatever it holds.

    ``temperature`` is 1e-3 to 1e3.  Up to 8 a row's sums are held in 32 bits and the loss is off by some ``temperature**2 *
    1e-7``; above, where the loss may be a millionth of ``temperature**2``, in 64.
    """
    # checked out here: inside autograd's frame gradients are disabled
    engine, temperature = _check_distill(logits, teacher_index, teacher_logits, temperature)
    _require_no_tangent(logits, "logits")
    _require_no_tangent(teacher_logits, "teacher_logits")
    if torch.is_grad_enabled() and logits.requires_grad:
        return _DistillationLoss.apply(logits, teacher_index, teacher_logits, temperature, engine)
    x, index, teacher = _rows(logits), teacher_index.contiguous(), teacher_logits.contiguous()
    return _loss_and_stats(engine, logits.shape[:-1], x, _distill_head(x, index, teacher, temperature))[0]


def _check_out(out, shape, dtype, device, grad_mode: bool, name: str = "out") -> None:
    """`grad_mode`: whether the caller's gradients are enabled."""
    _check_tensor(out, name, (dtype,), device)
    _require(tuple(out.shape) == tuple(shape), f"{name} must have shape {tuple(shape)}, got {tuple(out.shape)}")
    _require(out.is_contiguous() or (out.dim() == 2 and out.stride(1) == 1 and out.stride(0) >= out.shape[1]),
             f"{name} must be contiguous, or have contiguous rows that do not overlap")
    _require(not (out.requires_grad and grad_mode), f"{name} must not require a gradient: detach it")


def _extent(t):
    """(first byte, byte behind the last one) of a tensor with any elements."""
    size = t.element_size()
    first = t.data_ptr()
    return first, first + size * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))


def _share_memory(a, b) -> bool:
    """Whether an element of ``a`` may share a byte with one of ``b``: whatever their storages, and not where they lie side by
    side in one (pieces of a flat buffer, columns of a wide matrix)."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _extent(a), _extent(b)
    if a1 <= b0 or b1 <= a0:
        return False
    if a.dim() == b.dim() == 2 and a.stride(1) == b.stride(1) == 1:   # columns of rows of one length
        pitch = a.stride(0) * a.element_size()
        a_row, b_row = a.shape[1] * a.element_size(), b.shape[1] * b.element_size()
        if pitch == b.stride(0) * b.element_size() and pitch >= max(a_row, b_row):
            to_b = (b0 - a0) % pitch
            return to_b < a_row or to_b + b_row > pitch
    return True


def distillation_step(logits, teacher_index, teacher_logits, *, temperature=1.0, row_weight=None, out=None):
    """``(loss float32 [...], gradient [..., classes])`` in one call, for a training loop without autograd.

    The loss is :func:`distillation_loss`'s; the gradient is ``row_weight`` (float32 ``[...]``, default ones: what the
    loop's reduction would send back to each row) times the gradient of each row's loss, in the dtype of ``logits``.
    ``out`` receives the gradient; it may be ``logits`` itself (detached, where gradients are enabled), which then holds
    the gradient instead of the scores.
    """
    grad_mode = torch.is_grad_enabled()
    with torch.no_grad():
        engine, temperature = _check_distill(logits, teacher_index, teacher_logits, temperature)
        x, index, teacher = _rows(logits), teacher_index.contiguous(), teacher_logits.contiguous()
        head = _distill_head(x, index, teacher, temperature)
        rows = tuple(logits.shape[:-1])
        if row_weight is not None:
            _check_tensor(row_weight, "row_weight", (torch.float32,), logits.device)
            _require(tuple(row_weight.shape) == rows, f"row_weight must have shape {rows}, got {tuple(row_weight.shape)}")
            row_weight = row_weight.contiguous()
        given = out is not None
        if not given:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        else:
            _check_out(out, logits.shape, logits.dtype, logits.device, grad_mode)
            for t, name in ((teacher_index, "teacher_index"), (teacher_logits, "teacher_logits"), (row_weight, "row_weight")):
                _require(t is None or not _share_memory(out, t), f"out must not share memory with {name}")
            _require(not _share_memory(out, logits) or (out.data_ptr() == x.data_ptr() and out.stride() == logits.stride()),
                     "out may be logits itself, but must not overlap them otherwise")
        loss = torch.empty(rows, dtype=torch.float32, device=logits.device)
        if x.shape[0]:
            stride = _stride(out) if out.dim() == 2 else x.shape[1]
            ws = _workspace(_distill_workspace(x.shape[0], x.shape[1], head[1]), logits.device)
            _call(engine, engine._lib.serhip_distill_step, *head, None if row_weight is None else row_weight.data_ptr(),
                  loss.data_ptr(), out.data_ptr(), stride, ws.data_ptr(), ws.numel())
            if given:
                _written(out)
    return loss, out


# ------------------------------------------------------------------------------------------- embedding
def _check_tokens(tokens, device) -> None:
    _check_tensor(tokens, "tokens", (torch.int64, torch.int32), device)


def _lookup(tokens, table, scale: float, out=None):
    engine = _engine_of(table, "table")
    shape = (*tokens.shape, table.shape[1])
    given = out is not None
    if not given:
        out = torch.empty(shape, dtype=table.dtype, device=table.device)
    if out.numel():
        w, tok = _rows(table), tokens.contiguous()
        stride = _stride(out) if out.dim() == 2 else out.shape[-1]
        _call(engine, engine._lib.serhip_embed, tok.data_ptr(), int(tok.dtype == torch.int64), tok.numel(), w.data_ptr(),
              _DTYPES[w.dtype], _stride(w), w.shape[0], w.shape[1], scale, out.data_ptr(), stride)
        if given:
            _written(out)
    return out


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.scale, ctx.classes = scale, table.shape[0]
        return _lookup(tokens, table, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, embedding_gradient(grad, tokens, ctx.classes, scale=ctx.scale), None


def embed_tokens(tokens, table, *, scale=1.0, out=None):
    """``scale * table[tokens]``: ``[*tokens.shape, width]``, the product taken in float32 and rounded to the dtype of
    ``table [classes, width]``.

    ``tokens`` is int32 or int64; a token outside the table (padding, -1) gives a row of zeros.  Differentiable once,
    in backward mode, with respect to ``table`` (:func:`embedding_gradient`).  ``out`` receives the rows where no gradient is wanted.
    """
    _check_tensor(table, "table", _DTYPES)
    _require(table.dim() == 2 and table.shape[0] >= 1, "table must be [classes, width] with at least one class")
    _check_tokens(tokens, table.device)
    _require_no_tangent(table, "table")
    scale = float(scale)
    wants_grad = torch.is_grad_enabled() and table.requires_grad
    if out is not None:
        _require(not wants_grad, "out= has no gradient: detach the table, or leave out= away")
        _check_out(out, (*tokens.shape, table.shape[1]), table.dtype, table.device, torch.is_grad_enabled())
        _require(not _share_memory(out, table) and not _share_memory(out, tokens), "out must not share memory with the inputs")
    if wants_grad:
        return _EmbedTokens.apply(tokens, table, scale)
    return _lookup(tokens, table, scale, out)


@functools.lru_cache(maxsize=256)
def _gradient_workspace(tokens: int, classes: int, width: int) -> int:
    return _native.check(_native.load_library().serhip_embed_gradient_workspace(tokens, classes, width))


def embedding_gradient(grad, tokens, classes, *, scale=1.0, dtype=None, out=None, accumulate=False):
    """Gradient ``[classes, width]`` of :func:`embed_tokens` with respect to its table, for ``grad [*tokens.shape,
    width]``: row ``v`` is ``scale`` times the sum of the rows of ``grad`` whose token is ``v``.

    Sums are held in float32, in an order that depends on the tokens alone; the result is rounded once, to ``dtype``
    (that of ``grad``, the default, or float32).  Tokens outside ``0..classes-1`` take no part.  ``out`` receives the
    result; with ``accumulate`` it is added to what ``out`` holds (a gradient of several batches, or of a table that is
    also the output projection), and rows no token names are not touched.
    """
    _check_tensor(grad, "grad", _DTYPES)
    _check_tokens(tokens, grad.device)
    _require(grad.dim() >= 1 and grad.shape[:-1] == tokens.shape,
             f"grad must be {tuple(tokens.shape)} + (width,), got {tuple(grad.shape)}")
    classes, scale, width = int(classes), float(scale), grad.shape[-1]
    _require(1 <= classes <= (1 << 31) - 2, f"classes must be at least 1, got {classes}")
    grad_mode = torch.is_grad_enabled()
    with torch.no_grad():
        given = out is not None
        if not given:
            _require(not accumulate, "accumulate=True needs out=")
            dtype = grad.dtype if dtype is None else dtype
            _require(dtype in (grad.dtype, torch.float32), f"dtype must be {grad.dtype} or torch.float32, got {dtype}")
            _engine_of(grad, "grad")
            out = torch.empty((classes, width), dtype=dtype, device=grad.device)
        else:
            dtype = out.dtype if dtype is None and isinstance(out, torch.Tensor) else dtype
            _require(dtype in (grad.dtype, torch.float32), f"out must be {grad.dtype} or torch.float32, got {dtype}")
            _check_out(out, (classes, width), dtype, grad.device, grad_mode)
            _require(not _share_memory(out, grad) and not _share_memory(out, tokens), "out must not share memory with the inputs")
        engine = _engine_of(grad, "grad")
        if width:
            g, tok = _rows(grad), tokens.contiguous()
            n = tok.numel()
            ws = _workspace(_gradient_workspace(n, classes, width), grad.device)
            _call(engine, engine._lib.serhip_embed_gradient, g.data_ptr(), _DTYPES[g.dtype], _stride(g), tok.data_ptr(),
                  int(tok.dtype == torch.int64), n, classes, width, scale, int(bool(accumulate)), out.data_ptr(),
                  _DTYPES[out.dtype], _stride(out), ws.data_ptr(), ws.numel())
            if given:
                _written(out)
    return out


__all__ = ["sample_tokens", "distillation_loss", "distillation_step", "embed_tokens", "embedding_gradient"]
