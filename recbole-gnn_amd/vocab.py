"""Operators over large item vocabularies, beside those of ``ops.py``: rows of a table by id with the table's gradient, losses on
whole rows of logits with theirs, and scores from an 8-bit item table.  Tables and logits are float32, bfloat16 or float16;
arithmetic is in 32 bits and an output is rounded once.  GPU tensors only; calls run on the current stream and never synchronize.

An id, target or list entry outside its range (-1 is the usual "none") reads nothing and adds to nothing: the library cannot raise
for values that live on the device.

Gradients are those of reverse mode, once: gradients of gradients and forward mode raise.  The calls that return a gradient, and those in
8 bits, take their inputs as constants.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


_current_device, _raw_stream = torch.cuda.current_device, torch._C._cuda_getCurrentRawStream


def _call(fn, t, *args):
    """``fn(*args, stream)`` on the current stream of ``t``'s device, which is made the current device where it is not."""
    index = t.get_device()
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc:
        check(rc)


def _rows(t, name):
    """A 2-D floating tensor of a supported type on the GPU, columns next to each other (copied if they are not)."""
    if not t.is_cuda:
        raise RuntimeError(f"{name} must live on the GPU (the HIP engine has no CPU path)")
    if t.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if t.is_contiguous():
        return t
    n, d = t.shape
    if d > 1 and t.stride(1) != 1 or n > 1 and t.stride(0) < d:
        t = t.contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _like(t, of, name, shape, dtype):
    """``t`` as a contiguous ``dtype`` tensor of that shape on ``of``'s device; other devices are refused, never copied from."""
    if t.get_device() != of.get_device():
        raise RuntimeError(f"{name} is on {t.device}, expected {of.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        if dtype == torch.int64 and (t.is_floating_point() or t.dtype == torch.bool):
            raise TypeError(f"{name} must hold whole numbers, got {t.dtype}")
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def _differentiated(t):
    """Whether a call on ``t`` goes through its autograd function: a gradient may be asked for, or forward mode is on, where a tensor with a
    tangent is refused there (the functions have no forward-mode formula) instead of losing it."""
    return t.requires_grad and torch.is_grad_enabled() or forward_ad._current_level >= 0


def _c_int(n, name):
    """A size that the C entry takes in 32 bits: ctypes would pass its lower half alone."""
    if n > 0x7fffffff:
        raise ValueError(f"{name} = {n} is beyond 2^31 - 1")
    return n


def _ptr(t):
    return t.data_ptr() if t is not None else None


@functools.lru_cache(maxsize=1024)
def _bytes(fn, *sizes):
    nbytes = _lib.c_i64()
    check(getattr(lib, fn)(*sizes, ctypes.byref(nbytes)))
    return nbytes.value


def _workspace(of, fn, *sizes):
    """A workspace of the call's own, on the current stream (the caching allocator hands it out in stream order); None if it needs none."""
    nbytes = _bytes(fn, *sizes)
    return of.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


# ---------------------------------------------------------------------------------------------------------------------
# table rows and their gradient
# ---------------------------------------------------------------------------------------------------------------------
def _embedding(table, ids, scale):
    n, d = ids.numel(), _c_int(table.shape[1], "columns of table")
    out = table.new_empty((*ids.shape, d), dtype=table.dtype)
    if n and d:
        _call(lib.rbg_embedding, table, table.data_ptr(), _ld(table), table.shape[0], d, _DTYPES[table.dtype], ids.data_ptr(), n, scale,
              out.data_ptr(), d)
    return out


def _padding(padding_idx, n_rows):
    if padding_idx is None:
        return -1
    if not -n_rows <= padding_idx < n_rows:
        raise ValueError(f"padding_idx = {padding_idx} is not a row of {n_rows}")
    return int(padding_idx) % n_rows


def embedding_grad(grad, ids, n_rows, scale=1.0, padding_idx=None, out_dtype=None):
    """The gradient of :func:`embedding`'s table: ``out[v] = scale * sum of grad[i] over ids[i] == v`` as a dense [n_rows, d] tensor of
    ``out_dtype`` (``grad``'s type, the default, or float32), zeros where no id refers to a row and in row ``padding_idx`` (counted from the end when negative).  The
    places are sorted by id and summed in ascending order in 32 bits: the same bits from run to run.  Not differentiable itself."""
    if not grad.is_cuda:
        raise RuntimeError("grad must live on the GPU (the HIP engine has no CPU path)")
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        raise ValueError(f"grad must be {(*ids.shape, 'd')}, got {tuple(grad.shape)}")
    d = _c_int(grad.shape[-1], "columns of grad")
    grad = _rows(grad.reshape(ids.numel(), d) if grad.dim() != 2 else grad, "grad")
    ids = _like(ids, grad, "ids", tuple(ids.shape), torch.int64)
    padding_idx = _padding(padding_idx, n_rows)
    out_dtype = out_dtype or grad.dtype
    if out_dtype not in (grad.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {grad.dtype} or float32, got {out_dtype}")
    out = grad.new_empty((n_rows, d), dtype=out_dtype)
    if n_rows and d:
        n = ids.numel()
        work = _workspace(grad, "rbg_embedding_grad_workspace", n, n_rows, d)
        _call(lib.rbg_embedding_grad, grad, grad.data_ptr(), _ld(grad), _DTYPES[grad.dtype], ids.data_ptr(), n, n_rows, d, float(scale),
              padding_idx, out.data_ptr(), _DTYPES[out_dtype], _ptr(work))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rest = table.shape[0], scale, padding_idx
        return _embedding(table, ids, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        n_rows, scale, padding_idx = ctx.rest
        return embedding_grad(grad, ctx.saved_tensors[0], n_rows, scale, padding_idx), None, None, None


def embedding(table, ids, scale=1.0, padding_idx=None):
    """``scale * table[ids]`` for ``ids`` of any shape -> [*ids.shape, d]; zeros where an id is outside [0, n_rows).  Differentiable in
    ``table`` (:func:`embedding_grad`); row ``padding_idx`` is looked up like any other and gets no gradient, as in
    ``nn.Embedding``.  The wide-type, scaled form of :func:`ops.gather_rows` (lightgcn.py:60-68,128)."""
    table = _rows(table, "table")
    ids = _like(ids, table, "ids", tuple(ids.shape), torch.int64)
    _padding(padding_idx, table.shape[0])
    if _differentiated(table):
        return _Embedding.apply(table, ids, float(scale), padding_idx)
    return _embedding(table, ids, float(scale))


# ---------------------------------------------------------------------------------------------------------------------
# distillation from a teacher's top list
# ---------------------------------------------------------------------------------------------------------------------
def _teacher(logits, idx, val):
    n = logits.shape[0]
    if idx.dim() != 2 or idx.shape[0] != n:
        raise ValueError(f"teacher_idx must be [{n}, k], got {tuple(idx.shape)}")
    _c_int(idx.shape[1], "k")
    return (_like(idx, logits, "teacher_idx", tuple(idx.shape), torch.int64),
            _like(val, logits, "teacher_val", tuple(idx.shape), torch.float32))


def _distill(logits, idx, val, temperature, row_weight, want_stats, want_grad):
    n, v = logits.shape
    loss = logits.new_empty(n, dtype=torch.float32)
    stats = logits.new_empty((n, 2), dtype=torch.float32) if want_stats else None
    grad = logits.new_empty((n, v), dtype=logits.dtype) if want_grad else None
    work = _workspace(logits, "rbg_distill_topk_workspace", n, v)
    _call(lib.rbg_distill_topk, logits, logits.data_ptr(), _ld(logits), _DTYPES[logits.dtype], n, v, idx.data_ptr(), val.data_ptr(),
          idx.shape[1], temperature, _ptr(row_weight), loss.data_ptr(), _ptr(stats), _ptr(grad), v, _ptr(work))
    return loss, stats, grad


class _DistillTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, idx, val, temperature):
        loss, stats, _ = _distill(logits, idx, val, temperature, None, True, False)
        ctx.save_for_backward(logits, idx, val, stats)
        ctx.temperature = temperature
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, idx, val, stats = ctx.saved_tensors
        n, v = logits.shape
        g = g.to(torch.float32).contiguous()
        grad = logits.new_empty((n, v), dtype=logits.dtype)
        _call(lib.rbg_distill_topk_backward, logits, logits.data_ptr(), _ld(logits), _DTYPES[logits.dtype], n, v, idx.data_ptr(),
              val.data_ptr(), idx.shape[1], ctx.temperature, stats.data_ptr(), g.data_ptr(), grad.data_ptr(), v)
        return grad, None, None, None


def distill_topk(logits, teacher_idx, teacher_val, temperature=1.0):
    """Per row of ``logits`` [n, V], the divergence of the student's softmax from a teacher's top list (``teacher_idx``,
    ``teacher_val`` [n, k], as :func:`ops.full_sort_topk` returns them; idx -1 = no entry), both at ``temperature`` T:
    ``T^2 sum_j p_j (log p_j - log q_j)`` with p the softmax over the row's entries and q over all V.  A row without entries, or with
    all its logits at -inf, has loss 0 and gradient 0.  Returns [n] float32; differentiable in ``logits`` (the teacher is constant).
    k <= 256."""
    logits = _rows(logits, "logits")
    idx, val = _teacher(logits, teacher_idx, teacher_val)
    if _differentiated(logits):
        return _DistillTopk.apply(logits, idx, val, float(temperature))
    return _distill(logits, idx, val, float(temperature), None, False, False)[0]


def distill_topk_grad(logits, teacher_idx, teacher_val, temperature=1.0, row_weight=None):
    """:func:`distill_topk` and its gradient in one call, without an autograd graph: ``(loss [n], d(sum_b row_weight[b] loss[b]) /
    d(logits) [n, V])``.  The rows are read once."""
    logits = _rows(logits.detach(), "logits")
    idx, val = _teacher(logits, teacher_idx, teacher_val)
    if row_weight is not None:
        row_weight = _like(row_weight, logits, "row_weight", (logits.shape[0],), torch.float32)
    loss, _, grad = _distill(logits, idx, val, float(temperature), row_weight, False, True)
    return loss, grad


# ---------------------------------------------------------------------------------------------------------------------
# preference loss on pairs of packed sequences
# ---------------------------------------------------------------------------------------------------------------------
class _TokenLogp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets):
        m, v = logits.shape
        logp = logits.new_empty(m, dtype=torch.float32)
        stats = logits.new_empty((m, 2), dtype=torch.float32)
        work = _workspace(logits, "rbg_token_logp_workspace", m, v)
        _call(lib.rbg_token_logp, logits, logits.data_ptr(), _ld(logits), _DTYPES[logits.dtype], m, v, targets.data_ptr(), logp.data_ptr(),
              stats.data_ptr(), _ptr(work))
        ctx.save_for_backward(logits, targets, stats)
        return logp

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, targets, stats = ctx.saved_tensors
        m, v = logits.shape
        g = g.to(torch.float32).contiguous()
        grad = logits.new_empty((m, v), dtype=logits.dtype)
        _call(lib.rbg_token_logp_backward, logits, logits.data_ptr(), _ld(logits), _DTYPES[logits.dtype], m, v, targets.data_ptr(),
              stats.data_ptr(), g.data_ptr(), grad.data_ptr(), v)
        return grad, None


def token_logp(logits, targets):
    """``log_softmax(logits)[m, targets[m]]`` -> [m] float32 without the [m, V] matrix; 0 for a row without a target in [0, V) (-1: a
    prompt's token) and for one whose logits are all -inf.  Differentiable in ``logits``."""
    logits = _rows(logits, "logits")
    targets = _like(targets, logits, "targets", (logits.shape[0],), torch.int64)
    return _TokenLogp.apply(logits, targets)


def _pairs(of, offsets, ref):
    if offsets.dim() != 1 or offsets.shape[0] % 2 != 1:
        raise ValueError(f"offsets must be [2 pairs + 1], got {tuple(offsets.shape)}")
    return (_like(offsets, of, "offsets", tuple(offsets.shape), torch.int64),
            _like(ref, of, "ref_logp", (offsets.shape[0] - 1,), torch.float32), offsets.shape[0] // 2)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logp, offsets, ref, pairs, beta, smoothing):
        loss = logp.new_empty(pairs, dtype=torch.float32)
        margin = logp.new_empty(pairs, dtype=torch.float32)
        _call(lib.rbg_preference_loss, logp, logp.data_ptr(), logp.shape[0], offsets.data_ptr(), pairs, ref.data_ptr(), beta, smoothing,
              loss.data_ptr(), margin.data_ptr())
        ctx.save_for_backward(margin, offsets)
        ctx.rest = logp.shape[0], pairs, beta, smoothing
        return loss, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, g_loss, g_margin):
        margin, offsets = ctx.saved_tensors
        m, pairs, beta, smoothing = ctx.rest
        g_loss, g_margin = (g.to(torch.float32).contiguous() if g is not None else None for g in (g_loss, g_margin))
        grad = margin.new_empty(m, dtype=torch.float32)
        _call(lib.rbg_preference_loss_backward, margin, margin.data_ptr(), m, offsets.data_ptr(), pairs, beta, smoothing, _ptr(g_loss),
              _ptr(g_margin), grad.data_ptr())
        return grad, None, None, None, None, None


def preference_loss(logp, offsets, ref_logp, beta=0.1, label_smoothing=0.0):
    """Preference loss on pairs of packed sequences from their tokens' log-probabilities ``logp`` [m] (:func:`token_logp`): sequence s is
    the tokens ``offsets[s] .. offsets[s + 1]`` (``offsets`` [2 pairs + 1] ascending), sequence 2 i the preferred one of pair i and
    2 i + 1 the other, ``ref_logp`` [2 pairs] the reference model's sums.  Returns ``(loss, margin)`` [pairs] float32:
    ``margin = beta ((L_2i - ref_2i) - (L_2i+1 - ref_2i+1))``, ``loss = -(1 - e) log sigmoid(margin) - e log sigmoid(-margin)`` with e =
    ``label_smoothing``.  BPR (lightgcn.py:93-100) is the case of one token each and no reference.  Differentiable in ``logp``."""
    if not logp.is_cuda:
        raise RuntimeError("logp must live on the GPU (the HIP engine has no CPU path)")
    if logp.dim() != 1 or logp.dtype != torch.float32:
        raise TypeError(f"logp must be [m] float32, got {tuple(logp.shape)} {logp.dtype}")
    offsets, ref, pairs = _pairs(logp, offsets, ref_logp)
    return _PreferenceLoss.apply(logp.contiguous(), offsets, ref, pairs, float(beta), float(label_smoothing))


def preference_grad(logits, targets, offsets, ref_logp, beta=0.1, label_smoothing=0.0, pair_weight=None):
    """:func:`preference_loss` of ``token_logp(logits, targets)`` and its gradient in one call, without an autograd graph: ``(loss,
    margin, d(sum_i pair_weight[i] loss[i]) / d(logits) [m, V])``.  Log-probabilities stay in 64 bits between the two."""
    logits = _rows(logits.detach(), "logits")
    m, v = logits.shape
    targets = _like(targets, logits, "targets", (m,), torch.int64)
    offsets, ref, pairs = _pairs(logits, offsets, ref_logp)
    if pair_weight is not None:
        pair_weight = _like(pair_weight, logits, "pair_weight", (pairs,), torch.float32)
    loss = logits.new_empty((2, pairs), dtype=torch.float32)
    grad = logits.new_empty((m, v), dtype=logits.dtype)
    work = _workspace(logits, "rbg_preference_grad_workspace", m, v)
    _call(lib.rbg_preference_grad, logits, logits.data_ptr(), _ld(logits), _DTYPES[logits.dtype], m, v, targets.data_ptr(),
          offsets.data_ptr(), pairs, ref.data_ptr(), float(beta), float(label_smoothing), _ptr(pair_weight), loss[0].data_ptr(),
          loss[1].data_ptr(), grad.data_ptr(), v, _ptr(work))
    return loss[0], loss[1], grad


# ---------------------------------------------------------------------------------------------------------------------
# scores from 8 bits
# ---------------------------------------------------------------------------------------------------------------------
def _quantize(x, pad):
    n, k = x.shape
    ldc = (k + pad - 1) // pad * pad
    codes = x.new_empty((n, ldc), dtype=torch.int8)
    scale = x.new_empty(n, dtype=torch.float32)
    if n:
        _call(lib.rbg_quantize_rows_i8, x, x.data_ptr(), _ld(x), _DTYPES[x.dtype], n, k, codes.data_ptr(), ldc, scale.data_ptr())
    return codes, scale


def quantize_rows(x):
    """``(codes [n, K] int8, scale [n] float32)`` of the rows of ``x``: ``scale = max|row| / 127``, ``codes = round(row / scale)`` in
    [-127, 127].  A zero row has scale 0; one that holds an infinity or NaN has scale NaN (and its scores are NaN).  The codes
    are a view of rows padded with zeros to a multiple of 64 bytes, the layout :func:`score_int8` reads without a copy.  No gradient
    flows through it."""
    x = _rows(x, "x")
    if x.shape[1] == 0:
        raise ValueError("rows must have at least one column")
    codes, scale = _quantize(x.detach(), 64)
    return codes[:, :x.shape[1]], scale


def _codes(codes, k):
    """Rows of codes that the kernels can read 16 bytes at a time; copied where they are not."""
    n = codes.shape[0]
    need = (k + 15) // 16 * 16
    if (k == 1 or codes.stride(1) == 1) and codes.data_ptr() % 16 == 0:
        ld = codes.stride(0) if n > 1 else need
        room = codes.untyped_storage().nbytes() - codes.storage_offset()
        if ld % 16 == 0 and need <= ld <= 1 << 23 and (n - 1) * ld + need <= room:
            return codes, ld
    padded = codes.new_zeros((n, need))
    padded[:, :k] = codes
    return padded, need


def score_int8(u, codes, scales, out_dtype=torch.float32):
    """Scores [B, n] of the rows ``u`` [B, K] (float32, bfloat16 or float16) against a table in 8 bits (``codes`` [n, K], ``scales`` [n], as
    :func:`quantize_rows` makes them once): ``u`` is quantized row by row in the call, the products are summed exactly in 32-bit integers,
    and ``out_dtype`` is rounded to once.  No gradient flows through it.  The 8-bit form of :func:`ops.score` (lightgcn.py:131).  K <= 131071."""
    u = _rows(u.detach(), "u")
    b, k = u.shape
    if codes.dim() != 2 or codes.dtype != torch.int8:
        raise TypeError(f"codes must be [n, K] int8, got {tuple(codes.shape)} {codes.dtype}")
    if codes.device != u.device:
        raise RuntimeError(f"codes is on {codes.device}, expected {u.device}")
    n = codes.shape[0]
    if k == 0 or codes.shape[1] != k:
        raise ValueError(f"u is [*, {k}] but codes is [*, {codes.shape[1]}]")
    if out_dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    scales = _like(scales, u, "scales", (n,), torch.float32)
    out = u.new_empty((b, n), dtype=out_dtype)
    if b and n:
        codes, ldi = _codes(codes, k)
        work = _workspace(u, "rbg_score_rows_i8_workspace", b, k)
        _call(lib.rbg_score_rows_i8, u, u.data_ptr(), _ld(u), _DTYPES[u.dtype], b, codes.data_ptr(), ldi, scales.data_ptr(), n, k,
              out.data_ptr(), n, _DTYPES[out_dtype], _ptr(work))
    return out
