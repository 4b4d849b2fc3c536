"""Operators on logits: what a classifier over label embeddings answers, and what a student learns from its answers.

* ``token_logprobs``: per row, the log probabilities of given tokens (labels), the entropy, the log of the partition sum
  and the top alternatives, differentiable - one pass over the logits;
* ``distill_top_logits``: the KL loss of a student's logits against a teacher's top logits (the lists ``token_logprobs``
  returns), differentiable in the student's;
* ``label_logits``: cosines of embeddings with label embeddings - the logits of ``CLIP.classify`` and
  ``oadp_amd.dp.TopLogitsDistillation``, which call the two above with CLIP's scale.

The arithmetic runs in hand-written gfx950 kernels behind the C ABI (``oake_token_logprobs``, ``oake_distill_top_logits``
and their backward passes, include/oake_hip.h, which states every special case); tensors must live on the GPU.  Calls use
the current stream of the logits' device, whichever device is current, and can be captured into a graph.  (A backward pass
is captured with leaves made for the capture, on its stream and with no other graph of theirs alive: torch accumulates a
leaf's gradient on the stream its first graph was built on, and a capture does not take that.)
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .. import _lib

MAX_TOP = 128    # alternatives token_logprobs lists at most
MAX_LIST = 1024  # given tokens per row / entries of a teacher's list

_DTYPES = {torch.float32: _lib.OAKE_F32, torch.float16: _lib.OAKE_F16, torch.bfloat16: _lib.OAKE_BF16}
_INDEX = {torch.int32: _lib.OAKE_I32, torch.int64: _lib.OAKE_I64}


class TokenLogprobs(NamedTuple):
    """Outputs of ``token_logprobs``, fp32 (indices int64), shaped after the logits' leading dimensions."""
    logprobs: torch.Tensor | None       # as ``targets``
    entropy: torch.Tensor               # [...]
    lse: torch.Tensor                   # [...]: log sum e^z
    top_logprobs: torch.Tensor | None   # [..., top]
    top_indices: torch.Tensor | None    # [..., top], -1 where there are fewer alternatives


def _check_no_tangent(**tensors: torch.Tensor | None) -> None:
    if getattr(forward_ad, '_current_level', 0) < 0:  # (no level of dual tensors has been entered)
        return
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name} has a forward-mode tangent, which these operators do not carry on')


def _check_scale(scale: float | torch.Tensor) -> float:
    _check_no_tangent(scale=scale)
    if isinstance(scale, torch.Tensor) and scale.requires_grad and torch.is_grad_enabled():
        raise ValueError('scale gets no gradient: detach() it, or multiply the logits by a learnt scale')
    return float(scale)


def _check_logits(logits: torch.Tensor, scale: float) -> None:
    _check_no_tangent(logits=logits)
    if logits.dtype not in _DTYPES:
        raise TypeError(f'unsupported logits dtype {logits.dtype}')
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f'expected logits [..., vocab >= 1], got {tuple(logits.shape)}')
    if not 0.0 < scale <= 1e38:
        raise ValueError(f'scale must be positive and at most 1e38, got {scale}')


def _check_same_device(logits: torch.Tensor, **others: torch.Tensor | None) -> None:
    for name, t in others.items():
        if t is not None and t.device != logits.device:
            raise ValueError(f'{name} is on {t.device}, the logits are on {logits.device}')
    if not logits.is_cuda:
        raise RuntimeError('oadp_amd.clip runs on the GPU only (no CPU fallback): move the logits to a HIP device')


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., n] -> [rows, n] with the elements of a row next to each other (a view where that is possible)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _mask_rows(mask: torch.Tensor | None, logits: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    """(mask, bytes between its rows): one row of vocab bytes for all (0), or one for each row of the logits."""
    if mask is None:
        return None, 0
    if mask.dtype != torch.bool:
        raise TypeError(f'mask must be bool, got {mask.dtype}')
    if mask.dim() < 1 or mask.dim() > logits.dim() or mask.shape[-1] != logits.shape[-1] or any(
            m not in (1, n) for m, n in zip(reversed(mask.shape), reversed(logits.shape))):
        raise ValueError(f'mask {tuple(mask.shape)} does not broadcast over logits {tuple(logits.shape)}')
    if mask.numel() == mask.shape[-1]:
        return mask.reshape(-1).contiguous(), 0
    mask = _as_rows(mask.expand(logits.shape))
    return mask, mask.stride(0)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, vocab: int, dtype: int, top: int) -> int:
    lib, n = _lib.load(), C.c_size_t(0)
    _lib.check(lib, None, lib.oake_logits_workspace(rows, vocab, dtype, top, C.byref(n)), 'oake_logits_workspace')
    return n.value


# the current stream of a device as the C entries take it (the public call builds a Stream object: 1.1 us against 0.1,
# where a whole call takes about 15)
_current_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(_lib.load(), name)


def _launch(x: torch.Tensor, name: str, *args) -> None:
    """``name``(..., stream) with x's device current and its current stream."""
    dev = x.get_device()
    if _current_device() == dev:
        rc = _entry(name)(*args, _current_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = _entry(name)(*args, _current_stream(dev))
    if rc:
        _lib.check(_lib.load(), None, rc, name)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _f32(g: torch.Tensor | None) -> torch.Tensor | None:
    if g is None or (g.dtype is torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


def _workspace(x: torch.Tensor, rows: int, vocab: int, dtype: int, top: int) -> tuple[torch.Tensor | None, int]:
    n = _workspace_bytes(rows, vocab, dtype, top)
    return (x.new_empty(n, dtype=torch.uint8), n) if n else (None, 0)


def _score(x, targets, mask, mask_stride, top, scale, stats):
    (rows, vocab), dtype, f32 = x.shape, _DTYPES[x.dtype], torch.float32
    logprobs = top_lp = top_ids = None
    n = index = 0
    if targets is not None:
        n, index = targets.shape[1], _INDEX[targets.dtype]
        logprobs = x.new_empty((rows, n), dtype=f32)
    entropy, lse = x.new_empty(rows, dtype=f32), x.new_empty(rows, dtype=f32)
    if top:
        top_lp, top_ids = x.new_empty((rows, top), dtype=f32), x.new_empty((rows, top), dtype=torch.int64)
    ws, nbytes = _workspace(x, rows, vocab, dtype, top)
    _launch(x, 'oake_token_logprobs', x.data_ptr(), dtype, rows, vocab, x.stride(0), scale, _ptr(mask), mask_stride,
            _ptr(targets), index, n, top, _ptr(logprobs), lse.data_ptr(), entropy.data_ptr(), _ptr(top_lp), _ptr(top_ids),
            _ptr(stats), _ptr(ws), nbytes)
    return logprobs, entropy, lse, top_lp, top_ids


# The backward passes run in torch's device thread, where the same Python takes two to four times as long as in the caller's:
# what does not depend on the gradients is put together by the forward pass (``ctx.more``), and the launch stands in place
# (300 x 65, loss and gradient: 97 us with helpers, 86 without; 45 in one thread either way).  Strides are the saved tensors'
# own: a hook that moves them elsewhere and back (torch.autograd.graph.save_on_cpu) may have packed their rows.  The
# gradient's are dense whatever the logits' are (for rows that overlap, empty_like by itself would have others).
_DENSE = torch.contiguous_format


class _TokenLogprobs(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, targets, mask, mask_stride, top, scale):
        stats = x.new_empty((x.shape[0], 4), dtype=torch.float32)
        out = _score(x, targets, mask, mask_stride, top, scale, stats)
        ctx.save_for_backward(x, targets, mask, out[4], stats)
        n, index = (0, 0) if targets is None else (targets.shape[1], _INDEX[targets.dtype])
        ctx.more = (_entry('oake_token_logprobs_backward'), x.get_device(), _DTYPES[x.dtype], *x.shape, scale, index, n,
                    top)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(out[4])
        return out

    @staticmethod
    def backward(ctx, g_logprobs, g_entropy, g_lse, g_top, _):
        if torch.is_grad_enabled():  # a graph of the gradient is asked for: there is none
            return once_differentiable(_TokenLogprobs.backward)(ctx, g_logprobs, g_entropy, g_lse, g_top, _)
        x, targets, mask, top_ids, stats = ctx.saved_tensors
        entry, dev, dtype, rows, vocab, scale, index, n, top = ctx.more
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return _TokenLogprobs.backward(ctx, g_logprobs, g_entropy, g_lse, g_top, _)
        if g_logprobs is None and g_entropy is None and g_lse is None and g_top is None:
            return (None,) * 6
        g_logprobs, g_entropy, g_lse, g_top = _f32(g_logprobs), _f32(g_entropy), _f32(g_lse), _f32(g_top)
        if x.stride(1) != 1:
            x = x.contiguous()
        mask_stride = 0
        if mask is not None and mask.dim() == 2:
            mask = mask if mask.stride(1) == 1 else mask.contiguous()
            mask_stride = mask.stride(0)
        grad = torch.empty_like(x, memory_format=_DENSE)
        rc = entry(x.data_ptr(), dtype, rows, vocab, x.stride(0), scale, _ptr(mask), mask_stride, _ptr(targets), index, n,
                   _ptr(top_ids), top, stats.data_ptr(), _ptr(g_logprobs), _ptr(g_lse), _ptr(g_entropy), _ptr(g_top),
                   grad.data_ptr(), vocab, _current_stream(dev))
        if rc:
            _lib.check(_lib.load(), None, rc, 'oake_token_logprobs_backward')
        return grad, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor | None = None, *, top: int = 0,
                   mask: torch.Tensor | None = None, scale: float = 1.0) -> TokenLogprobs:
    """Log probabilities of ``softmax(scale * logits)`` over the last dimension.

    ``logits`` [..., vocab]: fp32, fp16 or bf16, any strides.  ``targets``: int32 / int64 ids, one a row ([...]) or
    several ([..., n], n <= 1024); negative ids are padding (log probability 0, no gradient), an id >= vocab gives NaN.
    ``top`` (0 .. 128): alternatives, best first, equal logits by the lowest index; index -1 and log probability -inf
    where a row has fewer.  ``mask`` (bool, broadcastable, at least [vocab]): False = not allowed, whatever stands there
    (NaN and inf included) is without effect and its gradient is 0.  A row with nothing allowed: lse -inf, entropy 0,
    log probabilities -inf, gradient 0.

    Differentiable once, backward, in ``logits`` (not in ``scale``: multiply the logits by a learnt one) through logprobs,
    entropy, lse and top_logprobs (a log probability of -inf is a constant); a forward-mode tangent is refused."""
    scale, top = _check_scale(scale), int(top)
    _check_logits(logits, scale)
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f'top must be 0 .. {MAX_TOP}, got {top}')
    lead = logits.shape[:-1]
    ids = None
    if targets is not None:
        if targets.dtype not in _INDEX:
            raise TypeError(f'targets must be int32 or int64, got {targets.dtype}')
        if targets.shape != lead and targets.shape[:-1] != lead:
            raise ValueError(f'targets {tuple(targets.shape)} do not match logits {tuple(logits.shape)}')
        n = 1 if targets.dim() == len(lead) else targets.shape[-1]
        if n > MAX_LIST:
            raise ValueError(f'at most {MAX_LIST} targets per row, got {n}')
        ids = targets.reshape(-1, n).contiguous() if n else targets.new_empty((lead.numel(), 0))
    mask, mask_stride = _mask_rows(mask, logits)
    _check_same_device(logits, targets=targets, mask=mask)
    x = _as_rows(logits)
    if x.requires_grad and torch.is_grad_enabled():
        out = _TokenLogprobs.apply(x, ids, mask, mask_stride, top, scale)
    else:
        out = _score(x, ids, mask, mask_stride, top, scale, None)
    logprobs, entropy, lse, top_lp, top_ids = out
    if targets is not None and logprobs.shape != targets.shape:
        logprobs = logprobs.view(targets.shape)
    if len(lead) != 1:
        entropy, lse = entropy.view(lead), lse.view(lead)
        if top:
            top_lp, top_ids = top_lp.view(*lead, top), top_ids.view(*lead, top)
    return TokenLogprobs(logprobs, entropy, lse, top_lp, top_ids)


def _distill(x, ids, v, scale, tail):
    (rows, vocab), dtype = x.shape, _DTYPES[x.dtype]
    loss, stats = x.new_empty(rows, dtype=torch.float32), x.new_empty((rows, 8), dtype=torch.float32)
    ws, nbytes = _workspace(x, rows, vocab, dtype, 0)
    _launch(x, 'oake_distill_top_logits', x.data_ptr(), dtype, rows, vocab, x.stride(0), scale, ids.data_ptr(),
            _INDEX[ids.dtype], v.data_ptr(), ids.shape[1], tail, loss.data_ptr(), stats.data_ptr(), _ptr(ws), nbytes)
    return loss, stats


class _DistillTopLogits(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, ids, v, scale, tail):
        loss, stats = _distill(x, ids, v, scale, tail)
        ctx.save_for_backward(x, ids, v, stats)
        ctx.more = (_entry('oake_distill_top_logits_backward'), x.get_device(), _DTYPES[x.dtype], *x.shape, scale,
                    _INDEX[ids.dtype], ids.shape[1], tail)
        return loss

    @staticmethod
    def backward(ctx, g_loss):
        if torch.is_grad_enabled():
            return once_differentiable(_DistillTopLogits.backward)(ctx, g_loss)
        x, ids, v, stats = ctx.saved_tensors
        entry, dev, dtype, rows, vocab, scale, index, k, tail = ctx.more
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return _DistillTopLogits.backward(ctx, g_loss)
        if g_loss.dtype is not torch.float32 or not g_loss.is_contiguous():
            g_loss = _f32(g_loss)
        if x.stride(1) != 1:
            x = x.contiguous()
        grad = torch.empty_like(x, memory_format=_DENSE)
        rc = entry(x.data_ptr(), dtype, rows, vocab, x.stride(0), scale, ids.data_ptr(), index, v.data_ptr(), k, tail,
                   stats.data_ptr(), g_loss.data_ptr(), grad.data_ptr(), vocab, _current_stream(dev))
        if rc:
            _lib.check(_lib.load(), None, rc, 'oake_distill_top_logits_backward')
        return grad, None, None, None, None


def distill_top_logits(logits: torch.Tensor, top_indices: torch.Tensor, top_logprobs: torch.Tensor, *,
                       scale: float = 1.0, tail: bool = False) -> torch.Tensor:
    """KL(teacher || student) per row, [...] fp32: the student is ``softmax(scale * logits)``, the teacher a list of
    ``top_indices`` (int32 / int64) and ``top_logprobs`` ([..., k <= 1024] each), as ``token_logprobs(..., top=k)``
    returns them.  Entries with a negative index or log probability -inf are absent; a row without entries has loss 0
    and gradient 0; an index >= vocab makes its row NaN.

    ``tail=False``: the teacher's entries are renormalised to 1.  ``tail=True``: they are taken as they are, and all
    places outside the list are one more outcome with the teacher's remaining probability, which keeps the student
    from moving its mass out of (or into) the list; that outcome is left out where the student rules out all of those
    places (-inf), while a listed place that it gives probability 0 makes the loss +inf.

    Temperature T: ``scale = 1 / T`` here and for the teacher's call, and T^2 times the loss to keep the gradient's size.

    Differentiable once, backward, in ``logits``; the teacher and ``scale`` get no gradient, a forward-mode tangent is
    refused."""
    scale, tail = _check_scale(scale), bool(tail)
    _check_logits(logits, scale)
    if top_indices.dtype not in _INDEX:
        raise TypeError(f'top_indices must be int32 or int64, got {top_indices.dtype}')
    if top_logprobs.dtype not in _DTYPES:
        raise TypeError(f'unsupported top_logprobs dtype {top_logprobs.dtype}')
    lead = logits.shape[:-1]
    if top_indices.shape != top_logprobs.shape or top_indices.dim() != logits.dim() or top_indices.shape[:-1] != lead:
        raise ValueError(f'expected top_indices and top_logprobs {(*lead, "k")}, got {tuple(top_indices.shape)} and '
                         f'{tuple(top_logprobs.shape)}')
    k = top_indices.shape[-1]
    if k > MAX_LIST:
        raise ValueError(f'at most {MAX_LIST} entries per row, got {k}')
    if top_logprobs.requires_grad and torch.is_grad_enabled():
        raise ValueError('the teacher gets no gradient: detach() its top_logprobs')
    _check_no_tangent(top_logprobs=top_logprobs)
    _check_same_device(logits, top_indices=top_indices, top_logprobs=top_logprobs)
    x = _as_rows(logits)
    ids, v = top_indices, top_logprobs.detach() if top_logprobs.requires_grad else top_logprobs
    if len(lead) != 1:
        ids, v = ids.reshape(x.shape[0], k), v.reshape(x.shape[0], k)
    ids, v = ids.contiguous(), _f32(v)
    if x.requires_grad and torch.is_grad_enabled():
        loss = _DistillTopLogits.apply(x, ids, v, scale, tail)
    else:
        loss, _ = _distill(x, ids, v, scale, tail)
    return loss if len(lead) == 1 else loss.view(lead)


def label_logits(embeddings: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    """Cosines [..., labels] (fp32) of embeddings [..., dim] with label embeddings [labels, dim] (the ViLD prompt
    ensemble of ``oadp_amd.prompts.vild``); both are normalised here."""
    if labels.dim() != 2 or embeddings.shape[-1] != labels.shape[1]:
        raise ValueError(f'embeddings {tuple(embeddings.shape)} and labels {tuple(labels.shape)} do not match')
    with torch.autocast(embeddings.device.type, enabled=False):  # (a cosine of 16 bits times CLIP's scale is off by 0.2)
        return F.normalize(embeddings.float(), dim=-1) @ F.normalize(labels.float(), dim=-1).t()
