"""Plain implementations, in 64 bits, of the sequence-model operators, and bounds on what their kernels may be
off by. u is half a step of the operand type (torch.finfo(t).eps / 2), g(n) = n 2^-24 bounds the relative error of a
sum of n products formed and added in 32 bits. fp32 operands may be multiplied as three products of 11-bit parts,
which drops at most 2^-21 of a product."""

import math

import torch

F32 = 2.0**-24


def unit(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def cell_mask(B, N, M, lx, ly, bandwidth):
    """(B, N, M) bool on the CPU: the cells of the band inside the lengths, by the reference's predicate per cell
    (band.h:23-38)."""
    mask = torch.zeros(B, N, M, dtype=torch.bool)
    for b in range(B):
        nx, ny = int(lx[b]), int(ly[b])
        if nx <= 0 or ny <= 0:
            continue
        i, j = torch.arange(nx).view(-1, 1), torch.arange(ny).view(1, -1)
        K, L = min(nx, ny), max(nx, ny)
        k, l = (i, j) if nx <= ny else (j, i)
        ok = torch.ones(nx, ny, dtype=torch.bool)
        if bandwidth >= 0:
            ok = 2 * (l * (K - 1) - k * (L - 1)).abs() <= max(2 * bandwidth * (K - 1), L - 1)
        mask[b, :nx, :ny] = ok.expand(nx, ny)
    return mask


def zero_padding(t, lengths):
    """t in 64 bits with the rows past the lengths zero, whatever they hold."""
    keep = torch.arange(t.shape[1], device=t.device).view(1, -1, 1, 1) < lengths.to(t.device).view(-1, 1, 1, 1)
    return torch.where(keep, t.double(), 0.0)


def attention(q, k, v, lx, ly, bandwidth, scale, dout=None):
    """Returns ({name: value}, {name: elementwise bound}) of out and, with dout, dq, dk, dv."""
    dtype, u = q.dtype, unit(q.dtype)
    B, N, H, d = q.shape
    M, Hkv = k.shape[1], k.shape[2]
    rep = H // Hkv
    mask = cell_mask(B, N, M, lx, ly, bandwidth).to(q.device).view(B, 1, N, M)
    Q = zero_padding(q, lx).transpose(1, 2)
    K, V = (zero_padding(t, ly).transpose(1, 2).repeat_interleave(rep, 1) for t in (k, v))
    s = Q @ K.transpose(2, 3) * scale
    s_abs = Q.abs() @ K.abs().transpose(2, 3) * abs(scale)
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    P = torch.where(total > 0, e / total.masked_fill(total == 0, 1.0), 0.0)
    out = P @ V
    # A score is off by at most (2^-21 + g(d)) of the sum of its products' magnitudes, and by the rounding of its
    # own product with scale / ln 2 and of its difference to the maximum (|s| <= s_abs); exp2 adds 2^-22. A weight's
    # numerator and denominator each carry that.
    worst = s_abs.masked_fill(~mask, 0.0).amax(-1, keepdim=True)
    rel = 2 * ((2**-21 + (d + 8) * F32) * worst + 2**-22) + (M + 8) * F32
    # 16-bit operands: the weights are rounded to the operand type for the second product.
    w = u if dtype != torch.float32 else 2**-21
    spread = P @ V.abs()
    out_err = (rel + w) * spread
    # fp16 rounds what lies below 2^-14 by up to 2^-25 whatever its size. The forward keeps weights 2^6 larger than
    # relative to (at most) the row's largest, which the denominator, at least one, divides: 2^-31 a cell. The backward
    # keeps P 2^10 larger: 2^-35 a cell; and dS so much larger that the largest |do| of the head's rows is at least 8:
    # 2^-28 of that |do| a cell.
    half = float(dtype == torch.float16)
    cells = mask.double()
    out_err = out_err + half * 2.0**-31 * (cells @ V.abs())
    vals = {"out": out.transpose(1, 2)}
    errs = {"out": (out_err + u * (out.abs() + out_err)).transpose(1, 2)}
    if dout is None:
        return vals, errs
    G = zero_padding(dout, lx).transpose(1, 2)
    dP = G @ V.transpose(2, 3)
    delta = (P * dP).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    a = G.abs() @ V.abs().transpose(2, 3)
    # delta comes from the stored output (in two parts: u^2 of it is lost) and carries its error and g(d).
    delta_err = (G.abs() * (out_err + (u * u + (d + 8) * F32) * (out.abs() + out_err))).sum(-1, keepdim=True)
    dS_err = (rel + w) * dS.abs() + P * (1 + rel) * ((2**-21 + (d + 8) * F32) * a + delta_err)
    peak = G.square().sum(-1).amax(-1).sqrt().view(B, Hkv, rep).amax(-1).repeat_interleave(rep, 1).view(B, H, 1, 1)
    dS_err = dS_err + half * 2.0**-28 * peak * cells
    long = (2**-21 + (max(N * rep, M) + 8) * F32)  # sums over rows or states

    def per_state(x):
        return x.view(B, Hkv, rep, M, d).sum(2).transpose(1, 2)

    dv_err = ((rel + w) * P + half * 2.0**-35 * cells).transpose(2, 3) @ G.abs() + long * (P.transpose(2, 3) @ G.abs())
    dq_err = abs(scale) * ((dS_err + long * (dS.abs() + dS_err)) @ K.abs())
    dk_err = abs(scale) * ((dS_err + long * (dS.abs() + dS_err)).transpose(2, 3) @ Q.abs())
    vals.update(dq=(dS @ K * scale).transpose(1, 2), dk=per_state(dS.transpose(2, 3) @ Q * scale),
                dv=per_state(P.transpose(2, 3) @ G))
    for name, err in (("dq", dq_err.transpose(1, 2)), ("dk", per_state(dk_err)), ("dv", per_state(dv_err))):
        errs[name] = err + (u + F32) * (vals[name].abs() + err)
    return vals, errs


def norm_rotate(x, weight, lengths, positions, rotary, base, interleaved, eps, dy=None):
    """Returns ({name: value}, {name: elementwise bound}) of y and, with dy, dx and dweight."""
    u = unit(x.dtype)
    B, N, H, d = x.shape
    dev = x.device
    X = zero_padding(x, lengths)
    keep = (torch.arange(N, device=dev).view(1, -1) < lengths.to(dev).view(-1, 1)).view(B, N, 1, 1)
    w = torch.ones(d, dtype=torch.float64, device=dev) if weight is None else weight.detach().double()
    pos = (torch.arange(N, device=dev) if positions is None else positions).double().expand(B, N).view(B, N, 1)
    angle = torch.zeros(B, N, d, dtype=torch.float64, device=dev)
    partner = torch.arange(d, device=dev)
    sign = torch.zeros(d, dtype=torch.float64, device=dev)
    for p in range(rotary // 2):
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + rotary // 2)
        angle[..., a] = angle[..., b] = pos[..., 0] * base ** (-2.0 * p / rotary)
        partner[a], partner[b], sign[a], sign[b] = b, a, -1.0, 1.0
    c, s = angle.cos().unsqueeze(2), (angle.sin() * sign).unsqueeze(2)

    def turn(z, way=1.0):
        return z * c + way * z[..., partner] * s

    def size(z):  # |.| of what a turn adds up
        return z.abs() * c.abs() + z[..., partner].abs() * s.abs()

    r = (X.square().mean(-1, keepdim=True) + eps).rsqrt()
    U = X * r
    Z = U * w
    # The mean carries g(d) (halved by the root), the root 2^-22, each product 2^-24; cos and sin of an angle
    # known to 2^-24 of a half turn carry 2^-22 each.
    rel = (d + 16) * F32 + 2**-22
    y = torch.where(keep, turn(Z), 0.0)
    # An angle is a position times a frequency whose power and quotient by 2 pi are rounded to 64 bits, and so is the
    # product: three relative errors of 2^-53; the plain angle above carries two.
    # 16-bit results take cos and sin from __sincosf, off by at most 2^-21.19 (CUDA's bound on [-pi, pi]), of an angle
    # rounded thrice more.
    hw = 2.0**-20 if x.dtype != torch.float32 else 0.0
    turn_err = 2 * 2**-22 + hw + 5 * 2.0**-53 * angle.abs().unsqueeze(2)
    y_err = (rel + turn_err) * (Z.abs() + Z[..., partner].abs()) * keep
    vals, errs = {"y": y}, {"y": y_err + u * (y.abs() + y_err)}
    if dy is None:
        return vals, errs
    Gy = zero_padding(dy, lengths)
    G = turn(Gy, -1.0)
    g_abs = Gy.abs() + Gy[..., partner].abs()
    dw = (G * U).sum((0, 1, 2))
    GW = G * w
    m = (GW * U).mean(-1, keepdim=True)
    dx = r * (GW - U * m)
    rel = rel + turn_err
    m_abs = ((1 + turn_err) * g_abs * w.abs() * U.abs()).mean(-1, keepdim=True)
    m_err = ((4 * rel) * g_abs * w.abs() * U.abs()).mean(-1, keepdim=True)
    dx_err = r * (4 * rel * (g_abs * w.abs() + U.abs() * m_abs) + U.abs() * m_err)
    count = B * N * H
    dw_err = ((2 * rel + 2**-20 + math.sqrt(count) * F32) * g_abs * U.abs()).sum((0, 1, 2))
    wu = u if weight is None else unit(weight.dtype)
    vals.update(dx=torch.where(keep, dx, 0.0), dweight=dw)
    errs.update(dx=(dx_err + u * (dx.abs() + dx_err)) * keep, dweight=dw_err + wu * (dw.abs() + dw_err))
    return vals, errs


def check(name, got, want, err):
    """Every element within its bound (and every NaN of `got` reported)."""
    got = got.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    tiny = 2.0**-24 if got.numel() else 0.0  # fp16 results below its normal numbers round by 2^-25
    bad = ~((got - want).abs() <= err + tiny * (err > 0))
    if bad.any():
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} outside their bounds; first at {at}: "
                             f"{got[at].item()} against {want[at].item()} +- {err[at].item()}")
