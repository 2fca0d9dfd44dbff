"""Cross entropy with its gradient, and log probabilities of given tokens,
on the gfx950 HIP kernels (token_loss_kernels.hip).

``cross_entropy`` is the training loss over a vocabulary (the reference's
word-level model takes nn.CrossEntropyLoss, dl_trainer.py:213);
``token_log_probs`` scores given tokens and also gives each row's entropy
and its best alternatives, for evaluation, for decoding, and, since it is
differentiable, for training on log probabilities.

Both take logits of float32, bfloat16 or float16 with any number of leading
dimensions, read them once, and compute and answer in float32; gradients
have the logits' type. A target equal to ``ignore_index`` takes no part. Any
other target outside the classes is an IndexError on the CPU; on a GPU,
where finding it would take a synchronisation, nothing is read for it and
its value and its row of the gradient are NaN. A logit of -inf is a masked
class: probability 0, gradient 0. A row with a NaN, a +inf or nothing but
-inf gives NaN. Neither function has a second derivative; the module has.
"""
from __future__ import annotations

import collections

import torch
import torch.nn as nn
import torch.nn.functional as F

from .grad_clip import load_lm, seen_whole

TokenLogProbs = collections.namedtuple(
    'TokenLogProbs', ['log_probs', 'entropy', 'top_log_probs', 'top_ids'])

_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_MAX_TOP = 64


def cross_entropy(logits, targets, ignore_index=-100, reduction='mean',
                  scaled=False):
    """``-log p[target]`` of each row, ``'none'``, or their ``'mean'`` over
    the rows that are not ignored (NaN where none is left), or ``'sum'``.

    logits: (..., classes); targets: (...), int64 or int32. float32.

    On a GPU the forward pass of a mean or a sum also leaves the gradient,
    for a backward pass that begins at the loss itself. ``scaled`` says that
    it will not (the loss is multiplied first, for mixed precision or
    accumulation): the gradient is the same, but is then worked out in the
    backward pass alone, where it would be worked out a second time
    otherwise (8190 x 50001 bfloat16: 675 us, with ``scaled`` 468, and 303
    for a loss that is not multiplied)."""
    if reduction not in _REDUCTIONS:
        raise ValueError('unknown reduction %r' % (reduction,))
    if logits.is_cuda:
        return load_lm().cross_entropy(logits, targets, int(ignore_index),
                                       _REDUCTIONS[reduction], bool(scaled))
    _check(logits, targets)
    return cross_entropy_reference(logits, targets, ignore_index, reduction)


def token_log_probs(logits, targets, top_k=0, ignore_index=-100):
    """A ``TokenLogProbs``, all float32 but the ids (int64):

    ``log_probs``: log probability of each target (0 where ignored);
    ``entropy``: of each row, in nats, also of ignored ones;
    ``top_log_probs``, ``top_ids``: (..., top_k), best first, of equal
    values the lowest index first, for ``top_k`` up to 64.

    The first two are differentiable; the last two are not."""
    if logits.is_cuda:
        return TokenLogProbs(*load_lm().token_log_probs(
            logits, targets, int(top_k), int(ignore_index)))
    _check(logits, targets)
    if not 0 <= top_k <= min(_MAX_TOP, logits.size(-1)):
        raise ValueError('top_k must be between 0 and the number of classes, '
                         'at most %d: %d' % (_MAX_TOP, top_k))
    return token_log_probs_reference(logits, targets, top_k, ignore_index)


def _check(logits, targets):
    if logits.dim() < 1 or logits.size(-1) < 1:
        raise ValueError('logits need a last dimension of classes')
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError('targets must be int64 or int32, not %s'
                        % targets.dtype)
    if targets.device != logits.device:
        raise ValueError('targets must be on the logits\' device')
    if targets.shape != logits.shape[:-1]:
        raise ValueError('targets must have the logits\' shape without the '
                         'last dimension: %s for logits %s'
                         % (list(targets.shape), list(logits.shape)))


class MgxCrossEntropyLoss(nn.CrossEntropyLoss):
    """nn.CrossEntropyLoss on the HIP kernels for (N, classes) logits and
    class indices, with second and further derivatives; the loss is float32
    whatever the logits' type. Weights, label smoothing, class
    probabilities, other shapes, and calls that torch has to see as its own
    operations (torch.compile and tracing, torch.func, forward-mode
    differentiation) go to torch."""

    def _use_hip_path(self, x, y):
        return (x.is_cuda and x.dtype in _TYPES and x.dim() == 2
                and y.dim() == 1 and y.dtype in (torch.int64, torch.int32)
                and x.size(0) == y.size(0) and self.weight is None
                and self.reduction in _REDUCTIONS
                and self.label_smoothing == 0.0 and seen_whole(x, y))

    def forward(self, x, y):
        if not self._use_hip_path(x, y):
            return super().forward(x, y)
        return load_lm().cross_entropy(x, y, int(self.ignore_index),
                                       _REDUCTIONS[self.reduction], False,
                                       True)


# --------------------------------------------------------------------------
# Plain torch: the CPU tier, and what the kernels are tested against.
# --------------------------------------------------------------------------

def _wide(logits):
    return logits if logits.dtype == torch.float64 else logits.float()


def cross_entropy_reference(logits, targets, ignore_index=-100,
                            reduction='mean'):
    x = _wide(logits).reshape(-1, logits.size(-1))
    loss = F.cross_entropy(x, targets.reshape(-1).long(),
                           ignore_index=ignore_index, reduction=reduction)
    return loss.view(targets.shape) if reduction == 'none' else loss


def token_log_probs_reference(logits, targets, top_k=0, ignore_index=-100):
    log = F.log_softmax(_wide(logits), dim=-1)
    keep = targets != ignore_index
    at = torch.where(keep, targets, torch.zeros_like(targets)).long()
    if bool(((at < 0) | (at >= logits.size(-1))).any()):
        raise IndexError('a target is outside the classes')
    lp = torch.where(keep, log.gather(-1, at.unsqueeze(-1)).squeeze(-1),
                     torch.zeros((), dtype=log.dtype, device=log.device))
    ids = _best(logits.detach(), top_k)
    top = log.detach().gather(-1, ids)
    # a class of probability 0 adds nothing: 0 times the lowest value
    low = torch.finfo(log.dtype).min
    if log.requires_grad:
        entropy = -(log.exp() * log.clamp(min=low)).sum(-1)
    else:
        # in place: 700 x 10000 take 4 ms, and 11 with new memory each time
        entropy = -log.exp().mul_(log.clamp_(min=low)).sum(-1)
    return TokenLogProbs(lp, entropy, top, ids)


def _best(x, k):
    """Indices of the ``k`` largest values of each row, best first, of equal
    ones the lowest index first; a NaN is larger than any other. torch.topk
    finds them where no two of the best ``k + 1`` are equal. In the other
    rows as many of those equal to the last are taken as there is room for,
    from the left, and only what is left is sorted: 700 rows of 10000 and
    their best five take 5 ms on eight cores, where sorting them whole takes
    130."""
    v, ids = torch.topk(x, min(k + 1, x.size(-1)))
    ids = ids[..., :k].contiguous()
    same = ((v[..., 1:] == v[..., :-1]) | v[..., 1:].isnan()).any(-1)
    if k == 0 or not bool(same.any()):
        return ids
    y = x[same]
    last = v[same][:, k - 1:k]
    nan, no_last = y.isnan(), last.isnan()
    above = (y > last) | (nan & ~no_last)
    equal = (y == last) | (nan & no_last)
    room = k - above.sum(-1, keepdim=True)
    keep = above | (equal & (equal.cumsum(-1) <= room))
    at = keep.nonzero()[:, 1].view(-1, k)
    order = torch.sort(y.gather(1, at), dim=-1, descending=True,
                       stable=True)[1]
    ids[same] = at.gather(1, order)
    return ids
