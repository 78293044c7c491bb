"""Distillation from a teacher's top logits on MI355X: the loss of a student's logits against the few entries that a
teacher kept of every position, and its gradient, in one pass over the logits.

With p the teacher's distribution over its k entries of a row, q = softmax(logits / temperature) of the student:

    loss = temperature² · (Σ p (log p - log q) + p_rest (log p_rest - log q_rest))

teacher_lse None: p = softmax(teacher_logits / temperature) over the entries, no rest.  teacher_lse [T], the logsumexp of
all the teacher's logits / temperature: p = exp(teacher_logits / temperature - teacher_lse), and the rest of the teacher's
mass, max(0, 1 - Σ p), is compared with the student's mass outside the entries.  (A rest below 2^-16, the rounding of Σ p,
is dropped where the student has no mass outside at all, as when the entries are the whole vocabulary.)

Entries with an index outside [0, V) (-1, say) or a teacher logit of -inf are padding.  A row without any other entry has
loss and gradient 0, whatever its logits hold; so has the gradient of a row of weight 0.  An index that comes twice counts
twice in p and once in q.  Logits of -inf have q = 0: a teacher entry there makes the loss infinite.  A row whose logits
are all -inf has gradient 0.  NaN logits make their row NaN.
"""
import _native


def topk_kl_rows(logits, teacher_idx, teacher_logits, weight=None, temperature=1.0, teacher_lse=None, out=None):
    """(loss [T] fp32, d(Σ weight · loss) / d logits [T, V]) in one call, for a training step that knows its rows' weights.
    logits [T, V] bf16, f16 or f32, contiguous columns; teacher_idx [T, k] int32 or int64, teacher_logits [T, k], k <=
    1024; weight [T] or None for 1.  The gradient goes to `out` (which may be the logits), else to a new tensor."""
    return _native.host4().topk_kl_rows(logits, teacher_idx, teacher_logits, weight, temperature, teacher_lse, out)


def topk_kl(logits, teacher_idx, teacher_logits, temperature=1.0, teacher_lse=None):
    """The loss of every row, [T] fp32, differentiable with respect to the logits (the statistics of the forward pass are
    kept, so that the backward pass reads the logits once).  The teacher's side has no gradient."""
    return _native.host4().topk_kl(logits, teacher_idx, teacher_logits, temperature, teacher_lse)
