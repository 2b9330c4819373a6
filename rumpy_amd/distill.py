"""Distillation from a teacher's top logits on the HIP path (csrc/distill.hip): the teacher's k largest logits of every row (``top_logits``), the
loss of a student's logits against them and its gradient (``distill_loss``; as a module: ``sr_tools.loss_functions.TopLogitsDistillLoss``).

Stands beside the softmax cross-entropy with one target per row (rumpy/regression/models/contrastive_learning/handlers.py:57): here a row's target
is the teacher's distribution over the columns it lists.  Rows are [V] logits - a query's similarities to the 8192 keys of a contrastive queue, or a
vocabulary of any size.  With u = z / T, q = softmax(u) and p the teacher's distribution:

    l = T^2 [ sum_i p_i (log p_i - log q_i)  +  p_t (log p_t - log q_t) ]

over the listed columns i and, when the teacher's ``tail`` is given, the unlisted columns together as one more outcome t.  No CPU path."""
import functools

import torch

from rumpy_amd import _lib as L
from .residual_norm import _FMT, _launch, _new_like, _once_differentiable, _p, _rows

MAX_TOP = 256
MAX_COLUMNS = 1 << 30


def _need_gpu(name, t):
    if not t.is_cuda:
        raise RuntimeError('rumpy_amd: %s runs on an MI355X through the HIP extension; there is no CPU path' % name)


def _check_logits(name, logits, temperature):
    if logits.dtype not in _FMT:
        raise RuntimeError('rumpy_amd: %s takes float32, bfloat16 or float16 logits, not %s' % (name, logits.dtype))
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_COLUMNS:
        raise ValueError('rumpy_amd: %s takes [..., V] logits with V >= 1, not %s' % (name, tuple(logits.shape)))
    t = float(temperature)
    if not 1e-30 < t < 1e30:
        raise ValueError('rumpy_amd: %s takes a temperature above zero, not %r' % (name, temperature))
    return t


@torch.no_grad()
def top_logits(logits, k, temperature=1.0):
    """The k <= 256 largest logits of every row of [..., V]: (values [..., k] in the logits' type, indices [..., k] int64, tail [...] float32).

    Descending, equal values by index, NaN first; tail = log sum exp(logit / temperature) over all other columns (-inf: there are none): what
    ``distill_loss`` at that temperature takes.  No gradient: the teacher's side."""
    t = _check_logits('top_logits', logits, temperature)
    v = logits.shape[-1]
    if not 1 <= int(k) <= min(v, MAX_TOP):
        raise ValueError('rumpy_amd: top_logits takes 1 <= k <= %d of rows of %d logits, not %r' % (MAX_TOP, v, k))
    _need_gpu('top_logits', logits)
    k, lead = int(k), tuple(logits.shape[:-1])
    values = torch.empty(lead + (k,), dtype=logits.dtype, device=logits.device)
    indices = torch.empty(lead + (k,), dtype=torch.int64, device=logits.device)
    tail = torch.empty(lead, dtype=torch.float32, device=logits.device)
    if logits.numel() == 0:
        return values, indices, tail
    z, ld = _rows(logits)
    rows = logits.numel() // v
    wb = _work_bytes(rows, v, k)
    work = torch.empty(wb, dtype=torch.uint8, device=logits.device) if wb else None
    _launch('rumpy_top_logits', L.TopLogitsArgs(logits=z.data_ptr(), values=values.data_ptr(), indices=indices.data_ptr(), tail=tail.data_ptr(), work=_p(work),
                                                rows=rows, ld=ld, V=v, k=k, fmt=_FMT[logits.dtype], inv_tau=1.0 / t), logits.device)
    return values, indices, tail


@functools.lru_cache(maxsize=512)
def _work_bytes(rows, v, k):
    return int(L.lib().rumpy_top_logits_work_bytes(rows, v, k))


@functools.lru_cache(maxsize=512)
def _partial_floats(rows, v):
    return int(L.lib().rumpy_distill_partial_floats(rows, v))


class _DistillFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, indices, tail, row_weight, temperature, reduction):
        dev, v = logits.device, logits.shape[-1]
        rows, k = logits.numel() // v, values.shape[-1]
        z, ld = _rows(logits)
        # state [rows, 8], the reduction's factor, the workspace of rows that are cut, the rows' losses
        pf = _partial_floats(rows, v)
        none = reduction == 'none'
        state = torch.empty(rows * 9 + 1 + pf, dtype=torch.float32, device=dev)
        loss = torch.empty(logits.shape[:-1] if none else (), dtype=torch.float32, device=dev)
        at = state.data_ptr()
        _launch('rumpy_distill_fwd', L.DistillArgs(
            logits=z.data_ptr(), top_values=values.data_ptr(), top_indices=indices.data_ptr(), tail=_p(tail), row_weight=_p(row_weight),
            row_loss=loss.data_ptr() if none else at + 4 * (8 * rows + 1 + pf), state=at, loss=None if none else loss.data_ptr(), factor=at + 32 * rows,
            partial=at + 32 * rows + 4 if pf else None, rows=rows, ld=ld, V=v, k=k, fmt=_FMT[z.dtype], value_fmt=_FMT[values.dtype],
            index64=1 if indices.dtype == torch.int64 else 0, mean=1 if reduction == 'mean' else 0, tau=temperature, inv_tau=1.0 / temperature), dev)
        ctx.reduction, ctx.temperature = reduction, temperature
        ctx.save_for_backward(logits, values, indices, tail, row_weight, state)
        return loss

    @staticmethod
    def backward(ctx, g):
        _once_differentiable('distill_loss')
        logits, values, indices, tail, row_weight, state = ctx.saved_tensors
        dev, v = logits.device, logits.shape[-1]
        rows, k = logits.numel() // v, values.shape[-1]
        z, ld = _rows(logits)
        g = g.contiguous()
        dl = _new_like(logits)
        if rows:
            # (`loss` only says that g is the gradient of one number; nothing but dlogits is written)
            _launch('rumpy_distill_bwd', L.DistillArgs(
                logits=z.data_ptr(), top_values=values.data_ptr(), top_indices=indices.data_ptr(), tail=_p(tail), row_weight=_p(row_weight),
                row_loss=g.data_ptr(), state=state.data_ptr(), loss=None if ctx.reduction == 'none' else g.data_ptr(), factor=state.data_ptr() + 32 * rows,
                partial=state.data_ptr(), gout=g.data_ptr(), dlogits=dl.data_ptr(), rows=rows, ld=ld, V=v, k=k, fmt=_FMT[z.dtype], value_fmt=_FMT[values.dtype],
                index64=1 if indices.dtype == torch.int64 else 0, mean=1 if ctx.reduction == 'mean' else 0, tau=ctx.temperature,
                inv_tau=1.0 / ctx.temperature), dev)
        return dl, None, None, None, None, None, None


def distill_loss(logits, top_values, top_indices, tail=None, temperature=1.0, row_weight=None, reduction='mean'):
    """The distillation loss of [..., V] student logits against a teacher's top logits of the same rows; gradient to ``logits``.

    top_values   [..., k <= 256] the teacher's logits (float32, bfloat16 or float16); top_indices [..., k] int64 or int32, their columns.
                 A negative index is an entry that is not used; a column listed twice takes both shares; an index >= V makes the row's loss and
                 gradient NaN.
    tail         [...] float32 or None: log sum exp(logit / temperature) of the teacher's other columns (``top_logits`` makes it).  None: the
                 teacher's distribution is renormalised over the listed columns.
    row_weight   [...] or None: weights of the rows; a row of weight 0 (padding) is not looked at and gets no gradient.
    reduction    'mean' = sum(weight * l) / sum(weight) (0 when the weights sum to 0), 'sum', or 'none' = weight * l per row.
    The loss is float32, times temperature^2 so that its gradient's size does not depend on the temperature.  A row whose entries are all unused
    or -inf contributes 0."""
    t = _check_logits('distill_loss', logits, temperature)
    if reduction not in ('mean', 'sum', 'none'):
        raise ValueError("rumpy_amd: distill_loss reduces by 'mean', 'sum' or 'none', not %r" % (reduction,))
    lead, dev = tuple(logits.shape[:-1]), logits.device
    if tuple(top_values.shape) != tuple(top_indices.shape) or tuple(top_values.shape[:-1]) != lead or top_values.dim() != logits.dim() \
            or not 1 <= top_values.shape[-1] <= MAX_TOP:
        raise ValueError('rumpy_amd: distill_loss takes top logits and indices %s with k <= %d, not %s and %s'
                         % (lead + ('k',), MAX_TOP, tuple(top_values.shape), tuple(top_indices.shape)))
    if top_values.dtype not in _FMT or top_indices.dtype not in (torch.int64, torch.int32):
        raise RuntimeError('rumpy_amd: distill_loss takes float32, bfloat16 or float16 top logits with int64 or int32 indices, not %s and %s'
                           % (top_values.dtype, top_indices.dtype))
    for name, s in (('tail', tail), ('row_weight', row_weight)):
        if s is not None and tuple(s.shape) != lead:
            raise ValueError('rumpy_amd: distill_loss takes %s %s, not %s' % (name, lead, tuple(s.shape)))
    for s in (top_values, top_indices, tail, row_weight):
        if s is not None and s.device != dev:
            raise ValueError('rumpy_amd: distill_loss takes its tensors on one device, %s, not %s' % (dev, s.device))
    _need_gpu('distill_loss', logits)
    as_f32 = lambda s: None if s is None else s.detach().to(torch.float32).contiguous()
    values = top_values.detach() if top_values.requires_grad else top_values
    return _DistillFn.apply(logits, values.contiguous(), top_indices.contiguous(), as_f32(tail), as_f32(row_weight), t, reduction)
