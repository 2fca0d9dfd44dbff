"""Global gradient norm over many tensors, and clipping by it.

``clip_grad_norm_`` does what ``torch.nn.utils.clip_grad_norm_`` does
(reference dist_trainer.py:89-94 clips the recurrent models with it), in
two kernel launches whatever the number and types of the gradients, and
without a host synchronisation. ``clip_grads`` gives new tensors,
``grad_norm`` the norm alone. The update that clips as it goes, which never
writes clipped gradients at all, is ``FusedSGD.step(max_norm=...)``.

On a GPU the gradients are float32, bfloat16 or float16 (mixed as they
like), on one device, and no two of them share memory. Squares are summed in
64 bits and in a fixed order, so a repeated call gives the same bits. A norm
that is infinite or NaN is not refused (that would take a synchronisation):
as with torch's function, gradients come out zero or NaN, and the returned
norm says so.
"""
from __future__ import annotations

import importlib

import torch
from torch.autograd import forward_ad
from torch.compiler import is_compiling

_ext = None
_DATA = (torch.Tensor, torch.nn.Parameter)
_tracing = torch._C._get_tracing_state
_transforms = torch._C._are_functorch_transforms_active
_modes = torch._C._len_torch_dispatch_stack


def load_lm():
    """The language-model kernels' extension; raises ExtensionMissing
    where it is not built."""
    global _ext
    if _ext is None:
        from . import ExtensionMissing
        try:
            _ext = importlib.import_module('mgwfbp_amd.kernels.mgx_lm_ext')
        except ImportError as e:
            raise ExtensionMissing(
                'mgx_lm_ext (language-model kernels) is not built. Build it '
                'in-tree: python setup.py build_ext --inplace (original '
                'error: %s)' % e)
    return _ext


def seen_whole(x, y):
    """Whether the tensors are data that a kernel can be given, with nothing
    beside it that looks at the operations: no compiler or tracer, no
    transform of torch.func, no forward-mode differentiation, no dispatch
    mode, no tensor of another class. What stands for one of torch's modules
    leaves those to torch's own operations."""
    return not (is_compiling() or _tracing() is not None or _transforms()
                or _modes() or forward_ad._current_level >= 0) and \
        type(x) in _DATA and type(y) in _DATA


def _limits(max_norm, eps):
    if not max_norm >= 0.0:
        raise ValueError('max_norm must not be negative: %r' % (max_norm,))
    if not eps >= 0.0:
        raise ValueError('eps must not be negative: %r' % (eps,))
    return float(max_norm), float(eps)


@torch.no_grad()
def grad_norm(grads):
    """L2 norm of all of ``grads`` taken together: a float32 scalar on
    their device (zero on the CPU where there are none)."""
    grads = list(grads)
    if not grads:
        return torch.zeros(())
    if not grads[0].is_cuda:
        return grad_norm_reference(grads)
    return load_lm().grad_norm(grads)


@torch.no_grad()
def clip_grads(grads, max_norm, eps=1e-6):
    """``(clipped, norm)``: new tensors, of the gradients' types, that hold
    ``grads`` times ``min(1, max_norm / (norm + eps))``. On a GPU they lie
    in one new buffer, which lives as long as any of them."""
    grads = list(grads)
    max_norm, eps = _limits(max_norm, eps)
    if not grads:
        return [], torch.zeros(())
    if not grads[0].is_cuda:
        return clip_grads_reference(grads, max_norm, eps)
    return load_lm().clip_grads(grads, max_norm, eps)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, eps=1e-6):
    """Scale the gradients of ``parameters`` in place so that their norm,
    taken together, is at most ``max_norm``; returns the norm from before,
    a float32 scalar on their device."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    max_norm, eps = _limits(max_norm, eps)
    if not grads:
        return torch.zeros(())
    if not grads[0].is_cuda:
        new, norm = clip_grads_reference(grads, max_norm, eps)
        for g, n in zip(grads, new):
            g.copy_(n)
        return norm
    return load_lm().clip_grads_(grads, max_norm, eps)


# --------------------------------------------------------------------------
# Plain torch: the CPU tier, and what the kernels are tested against.
# --------------------------------------------------------------------------

def grad_norm_reference(grads):
    return torch.stack([g.double().square().sum()
                        for g in grads]).sum().sqrt().float()


def clip_grads_reference(grads, max_norm, eps=1e-6):
    norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    factor = (max_norm / (norm + eps)).clamp(max=1.0)
    return [(g.double() * factor).to(g.dtype) for g in grads], norm.float()
