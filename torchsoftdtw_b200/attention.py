"""Cross attention between two padded series, and the head norm with rotation that prepares its operands.

The operators of a model that trains under the loss. They take the loss's own pair contract: per-sample
``lengths_x`` / ``lengths_y`` and the Sakoe-Chiba ``bandwidth``, with features split into heads. All compute runs
in this library's CUDA kernels (``torchsoftdtw_b200::cross_attention``, ``norm_rotate`` and their backward ops, autograd included).
"""

import math

import torch

from . import _ext

_ext.load()


# ---- FakeTensor kernels for torch.compile ----


@torch.library.register_fake("torchsoftdtw_b200::cross_attention")
def _cross_attention_fake(q, k, v, lengths_x, lengths_y, bandwidth, scale):
    return q.new_empty(q.shape)


@torch.library.register_fake("torchsoftdtw_b200::attention")
def _attention_fake(q, k, v, lengths_x, lengths_y, bandwidth, scale):
    B, N, H, _ = q.shape
    lo = q.new_empty((0,) if q.dtype == torch.float32 else q.shape)
    return q.new_empty(q.shape), lo, q.new_empty((B, H, N), dtype=torch.float32)


@torch.library.register_fake("torchsoftdtw_b200::attention_backward")
def _attention_backward_fake(dout, q, k, v, out, out_lo, lse, lengths_x, lengths_y, bandwidth, scale):
    return q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)


@torch.library.register_fake("torchsoftdtw_b200::norm_rotate")
def _norm_rotate_fake(x, weight, lengths, positions, rotary_dim, base, interleaved, eps):
    return x.new_empty(x.shape)


@torch.library.register_fake("torchsoftdtw_b200::norm_rotate_backward")
def _norm_rotate_backward_fake(dy, x, weight, lengths, positions, rotary_dim, base, interleaved, eps, need_weight):
    dw = weight.new_empty(weight.shape) if need_weight and weight is not None else x.new_empty((0,))
    return x.new_empty(x.shape), dw


def cross_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    lengths_x: torch.Tensor | None = None,
    lengths_y: torch.Tensor | None = None,
    bandwidth: int = -1,
    scale: float | None = None,
) -> torch.Tensor:
    """Attention of one series' queries to the states of another series.

    Row i of sample b attends to the columns that the loss's dynamic program visits in row i: all of
    ``[0, lengths_y[b])`` without a band, else the Sakoe-Chiba interval around the diagonal joining ``(0, 0)`` to
    ``(lengths_x[b] - 1, lengths_y[b] - 1)``. Differentiable in q, k and v (once). One query row a sample (N = 1, a
    decoded token) up to long series run through the same call; with few rows the states are split over the GPU.

    The band lies between the two series *of the call*, as in the loss: a series of one row has no diagonal, and its row spans all
    states whatever the band. A row that is decoded alone out of a longer, banded series is therefore called without a band
    on the states of its interval, ``cross_attention(q[:, i:i + 1], k[:, lo:hi], v[:, lo:hi])``.

    Scores, softmax statistics and sums are held in 32 bits. 16-bit operands: the weights, and in the gradients dS (see the
    header of the C ABI), are rounded to the operands' type once for their product, so that results are off by up to 1.5 times
    their own rounding. float32: products of an 11-bit head and tail each, without tail times tail (2^-22 a product).

    Args:
        q: (B, N, Hq, d) queries, float16, bfloat16 or float32; any strides.
        k: (B, M, Hkv, d) keys. Hq is a multiple of Hkv: query head h reads head ``h // (Hq // Hkv)``.
        v: (B, M, Hkv, d) values, of k's shape. 1 <= d <= 128.
        lengths_x: (B,) actual lengths of the queries' series, int32 or int64. Defaults to N for all.
        lengths_y: (B,) actual lengths of the states' series. Defaults to M for all.
        bandwidth: Sakoe-Chiba bandwidth, as in :func:`soft_dtw`. -1 means no constraint.
        scale: factor of the scores. Defaults to ``1 / sqrt(d)``.

    Returns:
        out: (B, N, Hq, d), contiguous, in q's dtype. Rows at or past ``lengths_x`` (and all rows of a sample whose
        ``lengths_y`` is 0) are zero and have no gradient. Rows of q, k and v past the lengths are not used: they
        may hold anything, NaN included; a NaN or infinity inside the lengths may reach every row of its sample. A
        length outside [0, N] / [0, M] makes the sample's rows NaN (its gradients zero) and is reported by
        :func:`check_errors`.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() > 0 and q.shape[-1] > 0 else 1.0
    return torch.ops.torchsoftdtw_b200.cross_attention(q, k, v, lengths_x, lengths_y, bandwidth, scale)


def norm_rotate(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    lengths: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    rotary_dim: int | None = None,
    base: float = 10000.0,
    interleaved: bool = False,
    eps: float = 1e-6,
) -> torch.Tensor:
    """RMS norm of every head, then the rotation of its features by the row's position, in one pass.

    ``u = x / sqrt(mean(x^2) + eps)``, ``z = u * weight``; pair p of the first ``rotary_dim`` features of z is turned
    by ``position * base ** (-2 p / rotary_dim)``. For the queries and keys of :func:`cross_attention`, each with
    the positions of its own series; positions may be real numbers, so that ``i * (ly - 1) / (lx - 1)`` lays the
    two series along the loss's diagonal, and ``i / factor`` stretches a context.

    Args:
        x: (B, N, H, d) heads, float16, bfloat16 or float32; any strides. 1 <= d <= 256.
        weight: (d,) factors of the normed features, in x's dtype or float32. Defaults to ones.
        lengths: (B,) actual lengths, int32 or int64. Rows past them come out as zeros, are not read and have no
            gradient. Defaults to N for all.
        positions: (B, N) or (N,), float32, int32 or int64. Defaults to 0 .. N - 1. Not differentiable.
        rotary_dim: how many leading features turn, even. Defaults to all (d, or d - 1 when d is odd).
        base: base of the frequencies.
        interleaved: pairs are features (2p, 2p + 1); otherwise (p, p + rotary_dim / 2).
        eps: floor of the mean square.

    Returns:
        y: (B, N, H, d), contiguous, in x's dtype. Differentiable in x and weight (once). Norms, products and sums are held in
        32 bits, angles in 64; cos and sin of 16-bit x are the hardware's (off by 2^-21 at most).
    """
    if rotary_dim is None:
        rotary_dim = x.shape[-1] // 2 * 2 if x.dim() > 0 else 0
    return torch.ops.torchsoftdtw_b200.norm_rotate(x, weight, lengths, positions, rotary_dim, base, interleaved, eps)
