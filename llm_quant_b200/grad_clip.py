"""llm_quant_b200.grad_clip -- the norm of many gradients together, and their clipping.

    norm = sqrt(sum g^2) over all values of all tensors
    out  = g * min(1, max_norm / (norm + 1e-6))

as torch.nn.utils.clip_grad_norm_ has it, for the adapters that ``QLoRA`` and
``AdapterBank`` train: the step between their backward pass and the optimizer.
Squares are added in fp32 by neighbours and from there on in fp64, in one order
(equal calls give equal bits), over the whole range of the types; the factor is
fp32 and each product is rounded once.  Nothing is read back on the host.
"""

from __future__ import annotations

from typing import Iterable, Optional, Sequence

import torch

from . import _C


def _dense(t: torch.Tensor) -> bool:
    """Whether t's values lie side by side, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    dims = sorted(range(t.ndim), key=lambda d: t.stride(d), reverse=True)
    return t.permute(dims).is_contiguous()


class GradClipper:
    """Clips a set of gradients that stay where they are (float32, float16 or
    bfloat16, mixed, on one CUDA device, any number of them), in place or into
    ``out`` (tensors of the same shapes, dtypes and strides, such as parts of an
    optimizer's flat buffer).  Addresses are taken once, here, and the memory is
    kept alive: for gradients that are made anew at each step use
    ``clip_grad_norm_``.  Tensors must not overlap."""

    def __init__(self, grads: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]] = None):
        grads = list(grads)
        outs = grads if out is None else list(out)
        if not grads:
            raise ValueError("GradClipper: no tensors")
        if len(outs) != len(grads):
            raise ValueError(f"GradClipper: {len(outs)} tensors in out for {len(grads)}")
        _C.require_cuda(*grads, *outs, what="GradClipper")
        self.device = grads[0].device
        spans = []
        for i, (g, o) in enumerate(zip(grads, outs)):
            _C.require_float(g, "GradClipper")
            if g.device != self.device or o.device != self.device:
                raise ValueError(f"GradClipper: tensor {i} is not on {self.device}")
            if o is not g and (o.dtype != g.dtype or o.shape != g.shape
                               or g.numel() > 1 and any(n > 1 and a != b for n, a, b in zip(g.shape, o.stride(), g.stride()))):
                raise ValueError(f"GradClipper: out {i} must have the shape, dtype and strides of its gradient")
            if not _dense(g):
                raise ValueError(f"GradClipper: tensor {i}'s values must lie side by side (strides {list(g.stride())})")
            if g.numel():
                nbytes = g.numel() * g.element_size()
                spans.append((o.data_ptr(), o.data_ptr() + nbytes, i, True))
                if o.data_ptr() != g.data_ptr():
                    spans.append((g.data_ptr(), g.data_ptr() + nbytes, i, False))
        spans.sort()
        end = read_end = 0  # the furthest ends so far of what is written, and of what is read
        for lo, hi, i, written in spans:
            if lo < end or written and lo < read_end:
                raise ValueError(f"GradClipper: tensor {i} overlaps another one")
            if written:
                end = max(end, hi)
            else:
                read_end = max(read_end, hi)
        # views of one buffer share its version
        bases = {id(b): b for b in (o if o._base is None else o._base for o in outs)}
        # aliases of their own: a tensor given other memory later leaves these as they are
        self._clipper = _C.ext().Clipper([g.detach() for g in grads], None if out is None else [o.detach() for o in outs],
                                         [b.detach() for b in bases.values() if not b.is_inference()])

    def clip(self, max_norm: float) -> torch.Tensor:
        """Clip to ``max_norm`` and return the norm before it (float32 scalar on
        the device; inf or NaN where the gradients are not finite, and the
        gradients are then what the formula makes of them)."""
        max_norm = float(max_norm)
        if not max_norm >= 0:
            raise ValueError(f"GradClipper.clip: max_norm {max_norm} must not be negative")
        return self._clipper.clip(max_norm)


def clip_grad_norm_(parameters: Iterable[torch.Tensor] | torch.Tensor, max_norm: float) -> torch.Tensor:
    """Clip the gradients of ``parameters`` (those that have one) in place to
    ``max_norm`` together, and return their norm before it (float32 scalar on the
    device).  A parameter may come only once."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros(())
    return GradClipper(grads).clip(max_norm)
