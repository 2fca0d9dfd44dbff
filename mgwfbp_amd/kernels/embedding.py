"""Token embedding with scaling, and its gradient by sorted tokens, on the
gfx950 HIP kernels (embedding_kernels.hip).

``embedding`` looks rows of a table up by token and scales them;
``MgxEmbedding`` is nn.Embedding on it (the reference's word-level model,
models/lstm.py:17). torch's gradient on a GPU sorts through a library and
takes many launches; this one takes three at most for up to 16384 tokens,
adds each token's rows up in float32, in an order that the positions decide,
and rounds once, so a repeated call gives the same bits.

The weight is float32, bfloat16 or float16; its gradient is dense and of
its type. A token outside the table is an IndexError on the CPU; on a GPU,
where finding it would take a synchronisation, nothing is read for it, its
output is NaN and it has no gradient. The function has no second derivative;
the module has.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import settings
from .grad_clip import load_lm, seen_whole

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_TOKENS = (torch.int64, torch.int32)


def embedding(tokens, weight, scale=1.0, padding_idx=None):
    """``scale * weight[tokens]``: (..., dim) of the weight's type.

    tokens: (...), int64 or int32; weight: (rows, dim). ``padding_idx``, a
    row that gets no gradient, counts from the end where it is negative."""
    if padding_idx is not None:
        if not -weight.size(0) <= padding_idx < weight.size(0):
            raise ValueError('padding_idx must be a row of the weight: %r'
                             % (padding_idx,))
        padding_idx %= weight.size(0)
    if weight.is_cuda:
        return load_lm().embedding(tokens, weight, float(scale),
                                   -1 if padding_idx is None
                                   else padding_idx)
    if tokens.dtype not in _TOKENS:
        raise TypeError('tokens must be int64 or int32, not %s'
                        % tokens.dtype)
    if tokens.device != weight.device:
        raise ValueError('tokens must be on the weight\'s device')
    if weight.dim() != 2:
        raise ValueError('the embedding weight must be a matrix')
    return embedding_reference(tokens, weight, scale, padding_idx)


class MgxEmbedding(nn.Embedding):
    """nn.Embedding on the HIP kernels, with a factor on its output, and
    with second and further derivatives. The options that only torch has
    (max_norm, sparse gradients, scaling by frequency), other types, and
    calls that torch has to see as its own operations (torch.compile and
    tracing, torch.func, forward-mode differentiation) go to torch."""

    def __init__(self, *args, scale=1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = scale

    def _use_hip_path(self, x, w):
        return (settings.USE_HIP_KERNELS and w.is_cuda
                and x.device == w.device and seen_whole(x, w)
                and x.dtype in _TOKENS and w.dtype in _TYPES
                and self.max_norm is None
                and not self.sparse and not self.scale_grad_by_freq)

    def forward(self, x):
        w = self.weight
        if not self._use_hip_path(x, w):
            y = super().forward(x)
            return y if self.scale == 1.0 else y * self.scale
        pad = self.padding_idx
        return load_lm().embedding(x, w, float(self.scale),
                                   -1 if pad is None else pad, True)

    def extra_repr(self):
        s = super().extra_repr()
        return s if self.scale == 1.0 else '%s, scale=%r' % (s, self.scale)


# --------------------------------------------------------------------------
# Plain torch: the CPU tier, and what the kernels are tested against.
# --------------------------------------------------------------------------

def embedding_reference(tokens, weight, scale=1.0, padding_idx=None):
    y = F.embedding(tokens, weight, padding_idx=padding_idx)
    return y if scale == 1.0 else y * scale
