"""The global norm of many gradients, and clipping by it, for training steps under the loss.

A small gamma or a long series makes single Soft-DTW gradients far larger than their neighbours'; a step that
clips the global norm keeps them from undoing the model. Both passes run in this library's kernels: two launches
for any number of tensors up to 960, none of them waiting for the host.
"""

import math
from typing import Iterable, Sequence

import torch

from . import _ext

_ext.load()


@torch.library.register_fake("torchsoftdtw_b200::global_norm")
def _global_norm_fake(tensors, norm_type):
    wide = any(t.dtype == torch.float64 for t in tensors)
    return tensors[0].new_empty((), dtype=torch.float64 if wide else torch.float32)


@torch.library.register_fake("torchsoftdtw_b200::clip_grads")
def _clip_grads_fake(grads, out, max_norm, norm_type):
    wide = any(t.dtype == torch.float64 for t in grads)
    return grads[0].new_empty((), dtype=torch.float64 if wide else torch.float32)


def global_norm(tensors: Sequence[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all entries of all tensors together.

    Args:
        tensors: CUDA tensors on one device, float16, bfloat16, float32 or float64 in any mix.
        norm_type: 2 (Euclidean) or ``inf`` (largest magnitude).

    Returns:
        A 0-dim float32 tensor (float64 if one of the tensors is), on the tensors' device; on the CPU, and zero,
        for no tensors. Equal inputs give equal bits on every call.
    """
    tensors = list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return torch.ops.torchsoftdtw_b200.global_norm(tensors, float(norm_type))


def clip_grads(
    grads: Sequence[torch.Tensor],
    max_norm: float,
    norm_type: float = 2.0,
    out: Sequence[torch.Tensor] | None = None,
) -> tuple[list[torch.Tensor], torch.Tensor]:
    """The gradients times ``min(1, max_norm / (norm + 1e-6))``, norm their :func:`global_norm`.

    Args:
        grads: the gradients, as for :func:`global_norm`.
        max_norm: the bound, not negative.
        norm_type: 2 or ``inf``.
        out: tensors of the gradients' shapes and dtypes that the result is written to; the gradients themselves
            clip in place (and where nothing exceeds the bound, nothing is written). No two of them, nor one of
            them and another gradient, may share an entry (slices of one buffer may lie between one another). Defaults to new tensors.

    Returns:
        (clipped, norm): the list of results and the norm before clipping, a 0-dim tensor. Nothing waits for the
        device. A NaN or infinite norm makes the results NaN (or zero where the norm is infinite), as the factor is.
    """
    grads = list(grads)
    if not math.isfinite(max_norm) and not max_norm > 0:
        raise ValueError(f"max_norm must be a number that is not negative, got {max_norm}")
    out = [torch.empty_like(g) for g in grads] if out is None else list(out)
    if not grads:
        if out:
            raise ValueError("out must hold one tensor for each gradient")
        return [], torch.tensor(0.0)
    norm = torch.ops.torchsoftdtw_b200.clip_grads(grads, out, float(max_norm), float(norm_type))
    return out, norm


def clip_grad_norm_(
    parameters: torch.Tensor | Iterable[torch.Tensor],
    max_norm: float,
    norm_type: float = 2.0,
    error_if_nonfinite: bool = False,
) -> torch.Tensor:
    """Clip the gradients of the parameters in place by their global norm, for a training loop
    between the backward pass and the optimizer's step.

    Args:
        parameters: a tensor or an iterable of tensors; those without a gradient are passed over.
        max_norm: the bound, not negative.
        norm_type: 2 or ``inf``.
        error_if_nonfinite: raise, before any gradient changes, if the norm is NaN or infinite. This waits for the
            device; without it nothing does.

    Returns:
        The norm before clipping, a 0-dim tensor.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    seen: dict[int, torch.Tensor] = {}
    for p in parameters:
        if p.grad is not None:
            seen.setdefault(id(p), p.grad)  # a shared parameter listed twice has one gradient
    grads = list(seen.values())
    if not grads:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = global_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the global norm of the gradients is not finite ({norm.item()}); nothing was clipped")
    return clip_grads(grads, max_norm, norm_type, out=grads)[1]
