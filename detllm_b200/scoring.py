"""Token scores and distillation on logits in device memory.

Torch views of the ``det_*_device`` calls of ``include/detgpu.h``: log
probability of a given token, entropy and the most likely tokens of each row
of logits; the divergence of a student's rows from a teacher's top lists; and
the gradients of both.  Rows are ``logits[i]``, f32, f16 or bf16, any distance
apart; ``-inf`` masks an entry out, a negative token or id is ignored.

Each call runs on the current stream of the logits' device, does not
synchronise, and may be captured into a CUDA graph.  Its results are new
tensors (the gradient ``out`` where given).  Nothing is recorded by autograd:
a training step takes the gradient from the ``_step`` call, or from the
``_grad`` call in the backward of its own ``torch.autograd.Function``.  Writing
to ``out`` counts as a change in place.

What is wrong on the host side raises (``ValueError``, or :class:`DetError`
with the library's status); what only the device sees (a NaN, a token outside
the vocabulary) makes its row's results NaN, as ``include/detgpu.h`` lists.  A
``_step`` call whose kernel gave up a bounded wait, which is not expected, has
NaN in all of its results.  There is no CPU fallback.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import DetError, lib

__all__ = ["TokenScores", "DistillLoss", "token_scores", "token_scores_grad", "token_scores_step", "distill_loss",
           "distill_grad", "distill_step"]

_F32 = torch.float32
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_IDS = {torch.int32: 4, torch.int64: 8}
# the handle of a device's current stream (0.1 us, where a Stream object takes 2)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


class TokenScores(NamedTuple):
    """Per row: log probability (natural) of the given token and entropy, the
    sums the gradient needs, and with ``top`` the most likely tokens."""

    logprob: torch.Tensor  # [n] f32
    entropy: torch.Tensor  # [n] f32
    stats: torch.Tensor  # [n, 4] f32: maximum m, S = sum exp(x - m), sum exp(x - m)(x - m), log S
    top_ids: Optional[torch.Tensor] = None  # [n, top] int32
    top_logprobs: Optional[torch.Tensor] = None  # [n, top] f32


class DistillLoss(NamedTuple):
    loss: torch.Tensor  # [n] f32
    stats: torch.Tensor  # [n, 4] f32, of (x - m) / temperature


def _logits(x, what="logits"):
    if not x.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if x.dim() != 2 or x.dtype not in _DTYPES:
        raise ValueError(f"{what} must be [rows, vocabulary] of float32, float16 or bfloat16")
    n, vocab = x.shape
    if vocab > 1 and x.stride(1) != 1:
        raise ValueError(f"{what}: the entries of a row must be adjacent")
    return n, vocab, x.stride(0) if n > 1 else vocab


def _on(t, logits, what, shape, dtypes, rows=False):
    """The data pointer of `t`, checked; rows: only its rows need be dense."""
    if t.shape != shape or t.dtype not in dtypes or t.device != logits.device:
        raise ValueError(f"{what} must be {list(shape)} of {' or '.join(str(d)[6:] for d in dtypes)} on {logits.device}")
    if not (t.stride(-1) == 1 or t.shape[-1] <= 1 if rows else t.is_contiguous()):
        raise ValueError(f"{what} must be {'dense in each row' if rows else 'contiguous'}")
    return t.data_ptr()


def _vector(t, logits, what, n):
    return None if t is None else _on(t, logits, what, (n,), (_F32,))


def _grad_out(logits, out, n, vocab):
    if out is None:
        return logits.new_empty((n, vocab)), vocab
    _on(out, logits, "out", (n, vocab), (logits.dtype,), rows=True)
    return out, out.stride(0) if n > 1 else vocab


def _given(out, grad):
    # autograd is told that a caller's tensor was written to, so a backward
    # that needs its old values is refused
    if out is not None:
        torch.autograd.graph.increment_version(out)
    return grad


def _lists(ids, teacher, logits, n):
    if ids.dim() != 2 or teacher.dim() != 2:
        raise ValueError("teacher_ids and teacher_logits must be [rows, entries]")
    k = ids.shape[1]
    pi = _on(ids, logits, "teacher_ids", (n, k), _IDS, rows=True)
    pt = _on(teacher, logits, "teacher_logits", (n, k), _DTYPES, rows=True)
    li, lt = (t.stride(0) if n > 1 else k for t in (ids, teacher))
    if li != lt:
        raise ValueError("teacher_ids and teacher_logits must have the same distance between rows")
    return pi, _IDS[ids.dtype], pt, _DTYPES[teacher.dtype], k, li


def _call(name, logits, *args):
    # the library works on the calling thread's current device
    index = logits.device.index
    fn = getattr(lib(), name)
    if torch.cuda.current_device() == index:
        st = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            st = fn(*args, _stream(index))
    if st:
        raise DetError(st, name)


def _new(logits, *shape):
    return logits.new_empty(shape, dtype=_F32)


@functools.lru_cache(maxsize=256)
def _scores_size(dtype, n, vocab, top):
    return lib().det_scores_workspace(_DTYPES[dtype], n, vocab, top)


@functools.lru_cache(maxsize=256)
def _step_size(n, vocab, k):
    return lib().det_step_workspace(n, vocab, k)


def _workspace(logits, size):
    return logits.new_empty(size, dtype=torch.uint8), size


def token_scores(logits, tokens, top: int = 0) -> TokenScores:
    """Log probability of ``tokens[i]`` under row i, the row's entropy, and its
    ``top`` (at most 128) most likely tokens, most likely first and equal ones
    in the order of their ids."""
    n, vocab, ld = _logits(logits)
    tok = _on(tokens, logits, "tokens", (n,), _IDS)
    if not 0 <= top <= min(vocab, 128):
        raise ValueError("top must be in 0 .. 128 and at most the vocabulary")
    logprob, entropy, stats = _new(logits, n), _new(logits, n), _new(logits, n, 4)
    ids = lps = None
    if top:
        ids = logits.new_empty((n, top), dtype=torch.int32)
        lps = _new(logits, n, top)
    work, size = _workspace(logits, _scores_size(logits.dtype, n, vocab, top))
    _call("det_token_scores_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, tok,
          _IDS[tokens.dtype], top, logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(),
          ids.data_ptr() if top else None, lps.data_ptr() if top else None, None, work.data_ptr(), size)
    return TokenScores(logprob, entropy, stats, ids, lps)


def token_scores_grad(logits, tokens, stats, grad_logprob=None, grad_entropy=None, out=None) -> torch.Tensor:
    """d (sum grad_logprob * logprob + grad_entropy * entropy) / d logits, from
    the ``stats`` that :func:`token_scores` gave for the same logits.  ``out``
    may be the logits themselves."""
    n, vocab, ld = _logits(logits)
    tok = _on(tokens, logits, "tokens", (n,), _IDS)
    ps = _on(stats, logits, "stats", (n, 4), (_F32,))
    gl = _vector(grad_logprob, logits, "grad_logprob", n)
    ge = _vector(grad_entropy, logits, "grad_entropy", n)
    grad, grad_ld = _grad_out(logits, out, n, vocab)
    _call("det_token_scores_grad_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, tok,
          _IDS[tokens.dtype], ps, gl, ge, grad.data_ptr(), grad_ld)
    return _given(out, grad)


def token_scores_step(logits, tokens, grad_logprob=None, grad_entropy=None, out=None):
    """:func:`token_scores` (without alternatives) and its gradient in one call
    that reads the logits once: ``(TokenScores, gradient)``.  With
    ``grad_logprob`` = -1/n it is the step of the mean code length."""
    n, vocab, ld = _logits(logits)
    tok = _on(tokens, logits, "tokens", (n,), _IDS)
    gl = _vector(grad_logprob, logits, "grad_logprob", n)
    ge = _vector(grad_entropy, logits, "grad_entropy", n)
    grad, grad_ld = _grad_out(logits, out, n, vocab)
    logprob, entropy, stats = _new(logits, n), _new(logits, n), _new(logits, n, 4)
    work, size = _workspace(logits, _step_size(n, vocab, 1))
    _call("det_token_scores_step_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, tok,
          _IDS[tokens.dtype], gl, ge, logprob.data_ptr(), entropy.data_ptr(), stats.data_ptr(), grad.data_ptr(),
          grad_ld, None, work.data_ptr(), size)
    return TokenScores(logprob, entropy, stats), _given(out, grad)


def distill_loss(logits, teacher_ids, teacher_logits, temperature: float = 1.0) -> DistillLoss:
    """Divergence (natural) of each row's distribution from the teacher's,
    which is softmax(teacher_logits / temperature) over the row's list of at
    most 128 tokens; the student's is softmax(logits / temperature) over the
    whole vocabulary.  The lists may be :func:`token_scores`' alternatives."""
    n, vocab, ld = _logits(logits)
    lists = _lists(teacher_ids, teacher_logits, logits, n)
    loss, stats = _new(logits, n), _new(logits, n, 4)
    work, size = _workspace(logits, _scores_size(logits.dtype, n, vocab, 0))
    _call("det_distill_loss_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, *lists,
          temperature, loss.data_ptr(), stats.data_ptr(), None, work.data_ptr(), size)
    return DistillLoss(loss, stats)


def distill_grad(logits, teacher_ids, teacher_logits, stats, grad_loss, temperature: float = 1.0,
                 out=None) -> torch.Tensor:
    """d (sum grad_loss * loss) / d logits, from the ``stats`` that
    :func:`distill_loss` gave for the same logits and temperature.  ``out`` may
    be the logits themselves."""
    n, vocab, ld = _logits(logits)
    lists = _lists(teacher_ids, teacher_logits, logits, n)
    ps = _on(stats, logits, "stats", (n, 4), (_F32,))
    g = _vector(grad_loss, logits, "grad_loss", n)
    grad, grad_ld = _grad_out(logits, out, n, vocab)
    _call("det_distill_grad_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, *lists,
          temperature, ps, g, grad.data_ptr(), grad_ld)
    return _given(out, grad)


def distill_step(logits, teacher_ids, teacher_logits, grad_loss, temperature: float = 1.0, out=None):
    """:func:`distill_loss` and its gradient in one call that reads the logits
    once: ``(DistillLoss, gradient)``."""
    n, vocab, ld = _logits(logits)
    lists = _lists(teacher_ids, teacher_logits, logits, n)
    g = _vector(grad_loss, logits, "grad_loss", n)
    grad, grad_ld = _grad_out(logits, out, n, vocab)
    loss, stats = _new(logits, n), _new(logits, n, 4)
    work, size = _workspace(logits, _step_size(n, vocab, lists[4]))
    _call("det_distill_step_device", logits, logits.data_ptr(), _DTYPES[logits.dtype], n, vocab, ld, *lists,
          temperature, g, loss.data_ptr(), stats.data_ptr(), grad.data_ptr(), grad_ld, None, work.data_ptr(), size)
    return DistillLoss(loss, stats), _given(out, grad)
