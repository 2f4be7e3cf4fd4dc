"""Softmax class head over many classes (``csrc/hip/head.hip``) + torch CPU path.

Scores z = (x w^T + bias) / T of rows ``x`` [n, d] against classes ``w`` [V, d]. Rows are taken in pieces: at most
``PIECE_BYTES`` of exponentials (or scores, head_topk) live at a time, or 256 rows of them where those are more
(2, with gradients in float32 10, in head_topk 4 bytes per row and class).

* :func:`softmax_head_loss`: per-row softmax cross entropy with the gradients of x, w and bias. With
  ``base_class`` one more class has score 0 and no weights (index V): the multiclass linear model's convention
  (``J/optimizer/MulticlassLinearHoagOptimizer.java:82-149``), whose fused row pass
  (:func:`ytk_learn_amd.ops.blas.multiclass_row_loss`) covers up to 64 classes.
* :func:`distill_head_loss`: the target of a row is a teacher's list of top logits.
* :func:`head_topk`: the k best classes of every row and the log of the sum of exponentials: what a teacher writes
  down for :func:`distill_head_loss`, and a classifier's answer.

float32 or bfloat16 (x, w and bias alike); any strides. float32 products run as six bf16 plane products
(24-bit operands); all sums, softmax statistics and losses are 32 bits or more. On bf16 inputs the score
gradient D = p - q is rounded to bf16 once before the two gradient products, and a p below e^-27 of the largest in its group of 64
classes counts as 0 there. Everything runs on the
current stream of x's device without a host synchronisation, in a workspace of its own per call (torch's
allocator), so calls on several streams and captured graphs do not share memory. Results are
bitwise reproducible. Gradients are returned; nothing is recorded for autograd.

x of rows that take part and w are finite; a class is switched off by a bias of -inf or the type's lowest value, and at
least one class is on.
"""
from __future__ import annotations

import contextlib
from typing import NamedTuple, Optional

import torch

from ._ext import hip, ptr, stream

# bytes of exponentials (or scores, head_topk) that live at a time; rows beyond are taken in further pieces, of 256 rows at least
PIECE_BYTES = 2 << 30
FEW_ROWS = 128           # == kFewRows (head.hip)
MAX_LIST = 256           # entries of a teacher's list, and k of head_topk
MAX_DIM = 1 << 21         # classes, features
_TYPES = (torch.float32, torch.bfloat16)


class HeadLoss(NamedTuple):
    """``loss`` [n] fp32 (weighted), ``lse`` [n] fp32, and the gradients of ``loss.sum()`` in the inputs' type
    (None where they were not asked for)."""
    loss: torch.Tensor
    lse: torch.Tensor
    dx: Optional[torch.Tensor]
    dw: Optional[torch.Tensor]
    db: Optional[torch.Tensor]


def _check(x, w, bias, temperature, **rows):
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"class head: x [n, d] and w [V, d] expected, got {tuple(x.shape)} and {tuple(w.shape)}")
    if x.dtype not in _TYPES or w.dtype != x.dtype:
        raise TypeError(f"class head: x and w of one type, float32 or bfloat16, expected, got {x.dtype} and {w.dtype}")
    n, d = x.shape
    V = w.shape[0]
    if d < 1 or V < 1 or d > MAX_DIM or V > MAX_DIM or n >= 1 << 31:
        raise ValueError(f"class head: 1 to {MAX_DIM} features and classes expected, got d = {d}, V = {V}")
    if bias is not None and (tuple(bias.shape) != (V,) or bias.dtype != w.dtype):
        raise ValueError(f"class head: bias [{V}] of type {w.dtype} expected")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError("class head: a temperature from 1e-6 to 1e6 expected")
    for name, t in dict(w=w, bias=bias, **rows).items():
        if t is not None and t.device != x.device:
            raise ValueError(f"class head: {name} is on {t.device}, x on {x.device}")
    if x.device.type not in ("cuda", "cpu"):
        raise ValueError("class head: tensors on the GPU or the CPU expected")


def _aligned(t):
    """Whether the products can read the rows in place: whole, aligned 16-byte pieces."""
    return int(t.dtype == torch.bfloat16 and t.stride(1) == 1 and t.shape[1] % 8 == 0 and t.stride(0) % 8 == 0
               and t.stride(0) >= t.shape[1] and t.data_ptr() % 16 == 0 and t.stride(0) <= 1 << 21)


def _operands(x, w):
    """Tensors that repeat memory or run backwards are copied, and those of few float32 rows whose columns are not dense;
    every other stride is read as it is."""
    few = x.dtype == torch.float32 and x.shape[0] <= FEW_ROWS

    def one(t):
        if t.shape[1] == 1:  # one column may carry any stride, and contiguous() leaves it
            t = t.as_strided(t.shape, (t.stride(0), 1))
        odd = (t.stride(0) <= 0 and t.shape[0] > 1) or (t.stride(1) <= 0 and t.shape[1] > 1)
        return t.contiguous() if odd or (few and t.stride(1) != 1) else t

    return one(x), one(w)


def _params(x, w, k, idx64, ignore, base, mode, want_dx, want_dw, bias):
    return [x.shape[0], x.shape[1], w.shape[0], k, int(x.dtype == torch.float32), x.stride(0), x.stride(1), w.stride(0),
            w.stride(1), idx64, ignore, int(base), mode, int(want_dx), int(want_dw), int(bias is not None),
            PIECE_BYTES, _aligned(x), _aligned(w)]


def _on(dev):
    """The device of the tensors as the current one (launches go to the current device)."""
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _loss(x, w, idx, tl, tlse, bias, weight, temperature, ignore, base, mode, want_dx, want_dw):
    n, V, dev = x.shape[0], w.shape[0], x.device
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    if n == 0:
        return HeadLoss(loss, lse, torch.zeros_like(x) if want_dx else None,
                        torch.zeros(w.shape, dtype=w.dtype, device=dev) if want_dw else None,
                        torch.zeros(V, dtype=w.dtype, device=dev) if want_dw and bias is not None else None)
    x, w = _operands(x, w)
    idx = idx.contiguous()
    bias, weight, tl, tlse = (None if t is None else t.contiguous() for t in (bias, weight, tl, tlse))
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if want_dx else None
    dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if want_dw else None
    db = torch.empty(V, dtype=w.dtype, device=dev) if want_dw and bias is not None else None
    lp = _params(x, w, idx.shape[1], int(idx.dtype == torch.int64), ignore, base, mode, want_dx, want_dw, bias)
    h = hip()
    ws = torch.empty(max(h.head_loss_ws(lp), 1), dtype=torch.uint8, device=dev)
    with _on(dev):
        h.head_loss([ptr(t) for t in (x, w, bias, idx, tl, tlse, weight, ws, loss, lse, dx, dw, db)], lp,
                    float(temperature), stream(x))
    return HeadLoss(loss, lse, dx, dw, db)


def _check_rows(n, weight, **vectors):
    for name, t in dict(weight=weight, **vectors).items():
        if t is not None and (tuple(t.shape) != (n,) or t.dtype != torch.float32):
            raise ValueError(f"class head: {name} [{n}] of type float32 expected")


def softmax_head_loss(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      weight: Optional[torch.Tensor] = None, ignore_index: int = -100, base_class: bool = False,
                      want_dx: bool = True, want_dw: bool = True) -> HeadLoss:
    """loss_i = weight_i (lse_i - z_i,label_i) and the gradients of its sum.

    ``labels`` [n] int64 / int32. A row labelled ``ignore_index`` or weighted 0 has loss 0 and no part in any gradient,
    whatever its x holds; any other label outside [0, V) (with ``base_class`` [0, V]) gives loss NaN and no gradient.
    ``db`` comes with ``want_dw`` where there is a bias."""
    _check(x, w, bias, 1.0, labels=labels, weight=weight)
    n = x.shape[0]
    if tuple(labels.shape) != (n,) or labels.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"softmax_head_loss: labels [{n}] of type int64 or int32 expected")
    _check_rows(n, weight)
    if not x.is_cuda:
        return _cpu_loss(x, w, labels[:, None], None, None, bias, weight, 1.0, ignore_index, base_class, 0, want_dx, want_dw)
    return _loss(x, w, labels[:, None], None, None, bias, weight, 1.0, int(ignore_index), base_class, 0, want_dx, want_dw)


def distill_head_loss(x: torch.Tensor, w: torch.Tensor, top_idx: torch.Tensor, top_logits: torch.Tensor,
                      bias: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, top_lse: Optional[torch.Tensor] = None, want_dx: bool = True,
                      want_dw: bool = True) -> HeadLoss:
    """loss_i = weight_i T^2 sum_j q_ij (log q_ij - log p_i,idx_ij) with p = softmax((x w^T + bias) / T), and the
    gradients of its sum.

    ``top_idx`` [n, k] int64 / int32 classes, -1 (any negative) for no entry; ``top_logits`` [n, k] float32, the
    teacher's logits before the division by T. q is the softmax of the row's own entries / T, or with ``top_lse``
    [n] float32 (log of the sum over ALL the teacher's classes of e^(logit / T)) the teacher's probabilities, the rest
    left out. A class named twice counts twice. A row without entries has loss 0 and no gradient; a class >= V
    gives loss NaN, its entry no gradient. k is at most 256. ``lse`` is of the scores / T."""
    _check(x, w, bias, temperature, top_idx=top_idx, top_logits=top_logits, weight=weight, top_lse=top_lse)
    n = x.shape[0]
    if top_idx.dim() != 2 or top_idx.shape[0] != n or not 1 <= top_idx.shape[1] <= MAX_LIST:
        raise ValueError(f"distill_head_loss: top_idx [{n}, k] with k from 1 to {MAX_LIST} expected")
    if top_idx.dtype not in (torch.int64, torch.int32):
        raise TypeError("distill_head_loss: top_idx of type int64 or int32 expected")
    if top_logits.shape != top_idx.shape or top_logits.dtype != torch.float32:
        raise ValueError("distill_head_loss: top_logits of top_idx's shape, float32, expected")
    _check_rows(n, weight, top_lse=top_lse)
    mode = 1 if top_lse is None else 2
    if not x.is_cuda:
        return _cpu_loss(x, w, top_idx, top_logits, top_lse, bias, weight, temperature, -1, False, mode, want_dx, want_dw)
    return _loss(x, w, top_idx, top_logits, top_lse, bias, weight, temperature, -1, False, mode, want_dx, want_dw)


def head_topk(x: torch.Tensor, w: torch.Tensor, k: int, bias: Optional[torch.Tensor] = None, temperature: float = 1.0):
    """(values [n, k] fp32 descending, classes [n, k] int64, lse [n] fp32) of the scores (x w^T + bias) / T.

    Classes and order are those of the scores summed in 64 bits, equal scores to the lower class: k + 8 candidates are found
    in 32 bits and scored again, and so is every other class that the 32-bit scores' error leaves possible (rows whose best
    scores lie closer together than 32 bits tell apart take longer, up to a 64-bit score of every class). 1 <= k <= min(V, 256). A row that holds NaN scores has some classes
    in some order, and lse NaN."""
    _check(x, w, bias, temperature)
    n, V, dev = x.shape[0], w.shape[0], x.device
    if not 1 <= k <= min(V, MAX_LIST):
        raise ValueError(f"head_topk: k from 1 to {min(V, MAX_LIST)} expected, got {k}")
    if not x.is_cuda:
        return _cpu_topk(x, w, k, bias, temperature)
    values = torch.empty((n, k), dtype=torch.float32, device=dev)
    classes = torch.empty((n, k), dtype=torch.int64, device=dev)
    lse = torch.empty(n, dtype=torch.float32, device=dev)
    if n == 0:
        return values, classes, lse
    x, w = _operands(x, w)
    bias = None if bias is None else bias.contiguous()
    lp = _params(x, w, k, 1, -1, False, 0, False, False, bias)
    h = hip()
    ws = torch.empty(max(h.head_topk_ws(lp), 1), dtype=torch.uint8, device=dev)
    with _on(dev):
        h.head_topk([ptr(t) for t in (x, w, bias, ws, values, classes, lse)], lp, float(temperature), stream(x))
    return values, classes, lse


# ------------------------------------------------------------------ CPU path (64 bits, rounded once)
@torch.no_grad()
def _cpu_loss(x, w, idx, tl, tlse, bias, weight, T, ignore, base, mode, want_dx, want_dw):
    n, V = x.shape[0], w.shape[0]
    xd, wd, idx = x.double(), w.double(), idx.long()
    z = xd @ wd.t()
    if bias is not None:
        z = z + bias.double()
    z = z / T
    if base:
        z = torch.cat([z, torch.zeros((n, 1), dtype=z.dtype)], 1)
    lse = torch.logsumexp(z, 1)
    g = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    there = idx != ignore if mode == 0 else idx >= 0
    bad = there & ((idx < 0) | (idx >= z.shape[1]))
    if mode == 0:
        logq = torch.zeros(idx.shape, dtype=torch.float64)
    else:
        t = torch.where(there, tl.double() / T, torch.full(tl.shape, -float("inf"), dtype=torch.float64))
        norm = tlse.double() if mode == 2 else torch.logsumexp(t, 1)
        norm = torch.where(norm == -float("inf"), torch.zeros_like(norm), norm) if mode == 1 else norm
        logq = t - norm[:, None]
    q = torch.where(there & ~bad, logq.exp(), torch.zeros_like(logq))
    at = torch.where(there & ~bad, idx, torch.zeros_like(idx))
    term = torch.where(q != 0, q * (logq - z.gather(1, at) + lse[:, None]), torch.zeros_like(q))
    term = torch.where(bad, torch.full_like(term, float("nan")), term).sum(1)
    s = q.sum(1)
    live = (g != 0) & (s != 0)
    loss = torch.where((g != 0) & ((s != 0) | term.isnan()), g * T * T * term, torch.zeros_like(term))
    dx = dw = db = None
    if want_dx or want_dw:
        D = ((z - lse[:, None]).exp() * s[:, None]).scatter_add(1, at, -q) * (g * T)[:, None]
        D = torch.where(live[:, None], D, torch.zeros_like(D))[:, :V]
        xz = torch.where(live[:, None], xd, torch.zeros_like(xd))
        dx = (D @ wd).to(x.dtype) if want_dx else None
        if want_dw:
            dw = (D.t() @ xz).to(w.dtype)
            db = D.sum(0).to(w.dtype) if bias is not None else None
    return HeadLoss(loss.float(), lse.float(), dx, dw, db)


@torch.no_grad()
def _cpu_topk(x, w, k, bias, T):
    z = x.double() @ w.double().t()
    if bias is not None:
        z = z + bias.double()
    z = z / T
    values, classes = z.sort(dim=1, descending=True, stable=True)
    return values[:, :k].float(), classes[:, :k].contiguous(), torch.logsumexp(z, 1).float()
