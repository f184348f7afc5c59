"""The global norm of the gradients, and their clipping by it (csrc/clip.hip).

Not part of the reference's loop (autolabel/trainer.py:39-49 steps its optimizers on unclipped gradients); here it stands between the backward
pass and the optimizer: ``TrainEngine(max_grad_norm=...)`` / ``Trainer(max_grad_norm=...)`` / ``scripts/train.py --max-grad-norm``, or by hand:

    norm = clip.clip_grad_norm_([p.grad for p in model.parameters() if p.grad is not None], 1.0)

One launch for the squares and one for the scaling per 120 tensors, whatever their sizes and types; the norm stays on the device.
"""
import array
import contextlib
import math

import torch

from . import hip as H

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _dense(t):
    """True when the elements of t fill one run of memory without holes or overlaps (in any order of its axes)."""
    if t.is_contiguous():
        return True
    order = sorted((d for d in range(t.dim()) if t.shape[d] > 1), key=t.stride)
    step = 1
    for d in order:
        if t.stride(d) != step:
            return False
        step *= t.shape[d]
    return True


# Unbound methods mapped over the lists: a list of 60 small gradients costs more on the host than on the device.
_T = torch.Tensor
_PLAIN = {torch.Tensor, torch.nn.Parameter}
_dtype, _requires_grad = _T.dtype.__get__, _T.requires_grad.__get__


def _check_tracked(name, grads, out, apply):
    """Some tensor requires a gradient: refuse what autograd would not see, and parameters handed over in place of their gradients."""
    if torch.is_grad_enabled():
        raise ValueError(f'{name}: a tensor requires a gradient, and autograd does not see what is done here: pass the parameters\' .grad, or call under torch.no_grad()')
    if apply and any(o is t and torch.is_tensor(t) and t.requires_grad and t.is_leaf for t, o in zip(grads, grads if out is None else out)):
        raise ValueError(f'{name}: a tensor requires a gradient: it is a parameter, not one\'s gradient (pass the parameters\' .grad)')


def _check(name, grads, out, loss_scale, found_inf, norm):
    """Say what is wrong with the arguments (the slow way: one is known to be)."""
    dev = getattr(grads[0], 'device', None)
    for i, t in enumerate(grads):
        if not torch.is_tensor(t) or t.layout != torch.strided or t.dtype not in TYPES:
            raise ValueError(f'{name}: tensor {i} must be a dense fp16, bf16 or fp32 tensor')
        if not _dense(t):
            raise ValueError(f'{name}: tensor {i} with shape {tuple(t.shape)} and strides {t.stride()} does not fill one run of memory')
        if t.device != dev:
            raise ValueError(f'{name}: tensors on different devices: {dev} and {t.device}')
    for i, (t, o) in enumerate(zip(grads, out or ())):
        if not torch.is_tensor(o) or o.dtype != t.dtype or o.shape != t.shape or o.device != dev or (o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous())):
            raise ValueError(f'{name}: output {i} must have the type, shape, strides and device of its tensor')
    for what, w, dt in (('loss_scale', loss_scale, torch.float32), ('found_inf', found_inf, torch.int32), ('norm', norm, torch.float32)):
        if w is not None and (not torch.is_tensor(w) or w.dtype != dt or w.numel() < 1 or w.device != dev):
            raise ValueError(f'{name}: {what} must be a device tensor of {dt} beside the gradients')
    if norm is not None and norm.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{name}: norm requires a gradient, and autograd does not see what is written into it')
    if dev.type != 'cuda':
        raise ValueError(f'{name}: autolabel_amd.clip has no CPU path: needs device tensors')


def _launch(name, grads, max_norm, apply, out, loss_scale, found_inf, norm):
    grads = [grads] if torch.is_tensor(grads) else list(grads)
    n = len(grads)
    if not n:
        raise ValueError(f'{name}: an empty list of tensors')
    if out is not None:
        out = [out] if torch.is_tensor(out) else list(out)
        if len(out) != n:
            raise ValueError(f'{name}: {n} tensors, {len(out)} outputs')
    every = grads if out is None else grads + out
    codes = None                 # the tensors' types, where the quick checks already tell
    plain = set(map(type, every)) <= _PLAIN
    if any(map(_requires_grad, every)) if plain else any(getattr(t, 'requires_grad', False) for t in every):
        _check_tracked(name, grads, out, apply)
    if plain and all(map(_T.is_contiguous, every)):
        device, types = set(map(_T.get_device, every)), set(map(_dtype, every))
        same = out is None or all(map(_T.is_same_size, out, grads))
        if len(device) == 1 and len(types) == 1 and min(device) >= 0 and types <= TYPES.keys() and same:
            codes = array.array('i', (TYPES[types.pop()],)) * n
    if codes is None or loss_scale is not None or found_inf is not None or norm is not None:
        _check(name, grads, out, loss_scale, found_inf, norm)
        codes = array.array('i', [TYPES[t.dtype] for t in grads])
    dev = grads[0].device
    with contextlib.nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev):
        given = norm is not None
        if not given:
            norm = torch.empty((), dtype=torch.float32, device=dev)
        ws = torch.empty(H.lib().aln_grad_clip_ws_bytes(n), dtype=torch.uint8, device=dev)
        g, o = array.array('Q', map(_T.data_ptr, grads)), None if out is None else array.array('Q', map(_T.data_ptr, out))
        sizes = array.array('q', map(_T.numel, grads))
        H.call('aln_grad_clip', n, g.buffer_info()[0], None if o is None else o.buffer_info()[0], sizes.buffer_info()[0], codes.buffer_info()[0], max_norm,
               int(apply), loss_scale.data_ptr() if loss_scale is not None else None, norm.data_ptr(),
               found_inf.data_ptr() if found_inf is not None else None, ws.data_ptr(), ws.numel(), H.raw_stream())
    # (a backward pass that saved what is written notices; inference tensors have no version)
    if apply:
        torch.autograd.graph.increment_version(grads if out is None else out)
    if found_inf is not None or given:
        torch.autograd.graph.increment_version([w for w in (norm, found_inf) if w is not None])
    return norm


def grad_norm(grads, loss_scale=None, found_inf=None, norm=None):
    """sqrt of the sum of all squares of the tensors ``grads``, over ``loss_scale`` -> fp32 scalar on the device (squares and sums in fp64;
    the same bits on every call).  ``found_inf`` (int32, device) is set to 1 when the norm is not finite.  ``norm``: an fp32 tensor on the device
    to write the norm into and return (one that a captured graph and eager calls share, say).  Not differentiable: while gradients are tracked,
    tensors that require one are refused."""
    return _launch('grad_norm', grads, 0.0, False, None, loss_scale, found_inf, norm)


def clip_grad_norm_(grads, max_norm, out=None, loss_scale=None, found_inf=None, norm=None):
    """Scale the tensors ``grads`` by min(1, max_norm / (norm + 1e-6)), in place or into ``out``, and return their ``grad_norm``.

    The tensors may differ in type (fp16, bf16, fp32) and size; no two may share memory.  Gradients that a loss scaler has multiplied keep
    its factor: ``loss_scale`` (fp32, device) only divides the norm.  A norm that is not finite scales nothing (``out`` is then a copy) and
    sets ``found_inf``: the caller skips that step.  ``norm`` as in ``grad_norm``.

    Unlike torch.nn.utils.clip_grad_norm_ this takes the gradients, not the parameters: a leaf that requires a gradient is never scaled in place.
    As for ``grad_norm``, tensors that require one are refused while gradients are tracked; what is written counts as modified in place."""
    max_norm = float(max_norm)
    if math.isnan(max_norm) or max_norm < 0:
        raise ValueError(f'clip_grad_norm_: max_norm = {max_norm}')
    return _launch('clip_grad_norm_', grads, max_norm, True, out, loss_scale, found_inf, norm)
