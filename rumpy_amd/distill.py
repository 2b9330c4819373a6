"""Distillation from a teacher's top logits on the HIP path (csrc/distill.hip, bound to torch by csrc/torch_bind.cpp): the teacher's k largest logits of every row (``top_logits``), the
loss of a student's logits against them and its gradient (``distill_loss``; as a module: ``sr_tools.loss_functions.TopLogitsDistillLoss``).

Stands beside the softmax cross-entropy with one target per row (rumpy/regression/models/contrastive_learning/handlers.py:57): here a row's target
is the teacher's distribution over the columns it lists.  Rows are [V] logits - a query's similarities to the 8192 keys of a contrastive queue, or a
vocabulary of any size.  With u = z / T, q = softmax(u) and p the teacher's distribution:

    l = T^2 [ sum_i p_i (log p_i - log q_i)  +  p_t (log p_t - log q_t) ]

over the listed columns i and, when the teacher's ``tail`` is given, the unlisted columns together as one more outcome t.  No CPU path."""
from rumpy_amd import _lib as L

MAX_TOP = 256


def top_logits(logits, k, temperature=1.0):
    """The k <= 256 largest logits of every row of [..., V]: (values [..., k] in the logits' type, indices [..., k] int64, tail [...] float32).

    Descending, equal values by index, NaN first; tail = log sum exp(logit / temperature) over all other columns (-inf: there are none): what
    ``distill_loss`` at that temperature takes.  No gradient: the teacher's side."""
    return (L.OPS or L.ops()).top_logits(logits, k, temperature)


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
    or -inf contributes 0.  A probability of the teacher's under 2^-126 of its row's
    largest counts as 0, also where the student gives the column none at all."""
    return (L.OPS or L.ops()).distill_loss(logits, top_values, top_indices, tail, temperature, row_weight, reduction)
