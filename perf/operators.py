"""The cases that the sequence-model operators beside the Soft-DTW loss are measured on.

Three operators, as a model that aligns two series uses them around the loss:

* ``cross_attention``: the queries of one series attend to the states of another, of another length, inside
  per-sample lengths and (optionally) the Sakoe-Chiba band of the loss; its gradients; single query tokens;
* ``norm_rotate``: RMS norm of every head followed by the rotation of its features by the position; its
  gradients;
* ``clip_grads``: the global norm of many gradient tensors and their clipping by it.

``run`` computes each in elementary torch operations (32 bits, 64 for angles and long sums) while ``own`` is
false, and calls this repository's operators when it is true. ``exact`` restates the definitions in 64 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "float64": torch.float64}
SIZEOF = {"float32": 4, "float16": 2, "bfloat16": 2, "float64": 8}
EPS = 1e-6  # floor of the RMS norm, and of the norm that clipping divides by


# ---- cases ----------------------------------------------------------------------------------------------

def attend(name, B, N, M, Hq, Hkv, d, dtype, bandwidth=-1, ragged=0, train=False):
    """N queries and M states a sample; ragged: 0 for full lengths, else the seed that they are drawn from."""
    return {"name": name, "op": "attend", "B": B, "N": N, "M": M, "Hq": Hq, "Hkv": Hkv, "d": d, "dtype": dtype,
            "bandwidth": bandwidth, "ragged": ragged, "train": train}


def rotate(name, B, N, H, d, dtype, rotary=None, interleaved=False, positions="", ragged=0, train=False):
    """positions: "" for 0, 1, ... along the series, "token" for whole positions anywhere in a long context,
    "stretch" for real ones that spread the series over another series' length."""
    return {"name": name, "op": "rotate", "B": B, "N": N, "H": H, "d": d, "dtype": dtype,
            "rotary": d if rotary is None else rotary, "interleaved": interleaved, "positions": positions,
            "ragged": ragged, "train": train}


def clip(name, width, layers, dtype, norm="2", max_norm=1.0):
    """The parameters of `layers` blocks of model width `width`; dtype "mixed" takes the four types in turn."""
    return {"name": name, "op": "clip", "width": width, "layers": layers, "dtype": dtype, "norm": norm,
            "max_norm": max_norm}


def listed():
    return [
        # One decoded query a sample against a short encoded series: latency.
        attend("attend_token", 8, 1, 512, 8, 8, 64, "bfloat16"),
        # One decoded query a sample against long encoded series, shared key heads: the cache's bytes.
        attend("attend_token_long", 16, 1, 32771, 32, 8, 128, "bfloat16"),
        # The ragged banded workload of the loss as a training step of its aligner, in float32.
        attend("attend_train_ragged", 64, 256, 192, 4, 4, 32, "float32", bandwidth=32, ragged=1, train=True),
        # A long pair of series, forward only: inference of a whole series at once.
        attend("attend_long", 2, 4096, 4096, 16, 16, 128, "bfloat16"),
        # The training step at the headline length.
        attend("attend_train", 32, 512, 512, 8, 8, 64, "bfloat16", train=True),
        # Long series of other, odd lengths with the long workload's band and shared key heads, trained in fp16.
        attend("attend_train_long", 4, 4096, 3001, 8, 2, 128, "float16", bandwidth=256, ragged=2, train=True),
        # The queries of one decoded token a sample, far into a long context: latency.
        rotate("rotate_token", 8, 1, 8, 64, "bfloat16", positions="token"),
        # A batch at the headline length as trained in float32, padded, stretched over the other series.
        rotate("rotate_train", 32, 512, 8, 64, "float32", positions="stretch", ragged=3, train=True),
        # Long series at once, part of an odd count of heads' features rotated in neighbouring pairs.
        rotate("rotate_train_long", 8, 4097, 13, 96, "float16", rotary=64, interleaved=True, train=True),
        # A small aligner of a few layers: dozens of tensors of a few thousand numbers, latency.
        clip("clip_small", 64, 2, "float32"),
        # A wide model in bf16: far more than the caches hold.
        clip("clip_large", 2048, 5, "bfloat16"),
        # Parameters of several types in one call, bounded by their largest entry.
        clip("clip_mixed", 500, 3, "mixed", norm="inf", max_norm=0.05),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    largest = [work(c) for c in listed()]
    limits = {k: max(w[k] for w in largest) for k in ("bytes", "flops")}
    while True:
        op = rng.choice(["attend", "attend", "rotate", "clip"])
        if op == "attend":
            hkv, group = rng.choice([1, 2, 3, 8]), rng.choice([1, 1, 2, 4])
            tokens = rng.random() < 0.3
            case = attend("", _log_int(rng, 1, 64), rng.randint(1, 4) if tokens else _log_int(rng, 5, 4096),
                          _log_int(rng, 1, 32771 if tokens else 4096), hkv * group, hkv,
                          rng.choice([16, 32, 33, 64, 80, 96, 128]),
                          rng.choice(["float32", "float16", "bfloat16", "bfloat16"]),
                          rng.choice([-1, -1, 0, 8, 32, 256]), rng.choice([0, rng.randint(1, 1 << 20)]),
                          (not tokens) and rng.random() < 0.5)
            if case["B"] * case["Hq"] * case["N"] * case["M"] > 2 * 16 * 4096 * 4096:
                continue  # the plain form holds that many scores
            narrow = case["bandwidth"] >= 0 and case["bandwidth"] * min(case["N"], case["M"]) < 8 * max(case["N"], case["M"])
            if case["train"] and (narrow or case["M"] < 16):
                continue  # a single state a query has weight one, and gradients of zero
        elif op == "rotate":
            d = rng.choice([16, 33, 64, 96, 128, 200, 256])
            case = rotate("", _log_int(rng, 1, 64), _log_int(rng, 1, 4100), rng.randint(1, 32), d,
                          rng.choice(["float32", "float16", "bfloat16"]), rng.choice([d // 2 * 2, d // 4 * 2, 2]),
                          rng.random() < 0.5, rng.choice(["", "token", "stretch"]),
                          rng.choice([0, rng.randint(1, 1 << 20)]), rng.random() < 0.6)
        else:
            case = clip("", _log_int(rng, 16, 2048), rng.randint(1, 5),
                        rng.choice(["float32", "bfloat16", "float16", "mixed"]), rng.choice(["2", "2", "inf"]),
                        rng.choice([0.05, 1.0, 1e6]))
        del case["name"]
        w = work(case)
        if all(w[k] <= limits[k] for k in limits):
            return case


def _lengths(case):
    """(lengths of the queries' series, lengths of the states' series), as lists."""
    B, N, M = case["B"], case["N"], case.get("M", case["N"])
    if not case["ragged"]:
        return [N] * B, [M] * B
    rng = random.Random(case["ragged"])
    return ([rng.randint((N + 3) // 4, N) for _ in range(B)], [rng.randint((M + 3) // 4, M) for _ in range(B)])


def _shapes(case):
    w = case["width"]
    block = [(w,), (w, w), (w, w), (w, w), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    names = ["float32", "bfloat16", "float16", "float64"] if case["dtype"] == "mixed" else [case["dtype"]]
    shapes = [(w, 17), (3,)] + block * case["layers"] + [(29, w)]
    return [(s, names[i % len(names)]) for i, s in enumerate(shapes)]


# ---- what a pass cannot do without ------------------------------------------------------------------------

def _row_cells(nx, ny, bandwidth):
    """In-band cells of an (nx, ny) pair: sum over rows of their column intervals."""
    if nx == 0 or ny == 0:
        return 0
    K, L = min(nx, ny), max(nx, ny)
    if bandwidth < 0 or K <= 1:
        return nx * ny
    h = max(2 * bandwidth * (K - 1), L - 1) // 2
    i = torch.arange(nx, dtype=torch.int64)
    num, den = (i * (L - 1), K - 1) if nx <= ny else (i * (K - 1), L - 1)
    lo = (-((h - num) // den)).clamp_min(0)
    hi = ((num + h) // den).clamp_max(ny - 1)
    return int((hi - lo + 1).sum())


def work(case):
    if case["op"] == "attend":
        lx, ly = _lengths(case)
        Hq, Hkv, d, size = case["Hq"], case["Hkv"], case["d"], SIZEOF[case["dtype"]]
        cells = sum(_row_cells(x, y, case["bandwidth"]) for x, y in zip(lx, ly))
        rows_q, rows_k = sum(lx) * Hq, sum(ly) * Hkv
        all_q, all_k = case["B"] * case["N"] * Hq, case["B"] * case["M"] * Hkv
        elems = rows_q + 2 * rows_k + all_q
        flops = 4 * cells * Hq * d
        if case["train"]:
            elems += rows_q + all_q + 2 * all_k
            flops += 10 * cells * Hq * d
        return {"bytes": elems * d * size, "flops": flops}
    if case["op"] == "rotate":
        lx, _ = _lengths(case)
        d, size = case["d"], SIZEOF[case["dtype"]]
        read, written = sum(lx) * case["H"] * d, case["B"] * case["N"] * case["H"] * d
        if case["train"]:
            return {"bytes": (2 * read + 2 * written) * size + 8 * d, "flops": 20 * read}
        return {"bytes": (read + written) * size + 4 * d, "flops": 7 * read}
    counts = [(math.prod(s), SIZEOF[t]) for s, t in _shapes(case)]
    return {"bytes": sum(2 * n * b for n, b in counts), "flops": sum(3 * n for n, _ in counts)}


# ---- inputs -------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "clip":
        state["grads"] = [normal(*s, dtype=DTYPES[t], scale=0.02) for s, t in _shapes(case)]
        state["out"] = [torch.empty_like(t) for t in state["grads"]]
        return state
    t = DTYPES[case["dtype"]]
    B, N, d = case["B"], case["N"], case["d"]
    lx, ly = _lengths(case)
    ragged = bool(case["ragged"])
    state["lengths_x"] = torch.tensor(lx, device=dev) if ragged else None
    if case["op"] == "attend":
        M, Hq, Hkv = case["M"], case["Hq"], case["Hkv"]
        state["lengths_y"] = torch.tensor(ly, device=dev) if ragged else None
        state["q"] = normal(B, N, Hq, d, dtype=t, scale=1.5)
        state["k"] = normal(B, M, Hkv, d, dtype=t)
        state["v"] = normal(B, M, Hkv, d, dtype=t)
        if case["train"]:
            state["grad_out"] = normal(B, N, Hq, d, dtype=t)
            for name in ("q", "k", "v"):
                state[name].requires_grad_(True)
        return state
    state["x"] = normal(B, N, case["H"], d, dtype=t, scale=2.0)
    state["weight"] = 1.0 + normal(d, dtype=torch.float32, scale=0.1)
    state["positions"] = None
    if case["positions"] == "token":
        start = torch.randint(0, 100000, (B, 1), generator=g, device=dev)
        state["positions"] = start + torch.arange(N, device=dev)
    elif case["positions"] == "stretch":
        ratio = 0.25 + 2 * torch.rand(B, 1, generator=g, device=dev)
        state["positions"] = ratio * torch.arange(N, device=dev, dtype=torch.float32)
    if case["train"]:
        state["grad_out"] = normal(B, N, case["H"], d, dtype=t)
        state["x"].requires_grad_(True)
        state["weight"].requires_grad_(True)
    return state


# ---- one pass -------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    return (_run_own if own else _run_plain)(state, case)


def _run_own(state, case):
    import torchsoftdtw_b200 as T

    if case["op"] == "clip":
        clipped, norm = T.clip_grads(state["grads"], case["max_norm"], norm_type=float(case["norm"]), out=state["out"])
        return {"norm": norm, "grads": clipped}
    if case["op"] == "attend":
        q, k, v = state["q"], state["k"], state["v"]
        out = T.cross_attention(q, k, v, state["lengths_x"], state["lengths_y"], bandwidth=case["bandwidth"])
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), state["grad_out"])
        return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}
    x, w = state["x"], state["weight"]
    out = T.norm_rotate(x, w, state["lengths_x"], state["positions"], rotary_dim=case["rotary"],
                        interleaved=case["interleaved"], eps=EPS)
    if not case["train"]:
        return {"out": out}
    dx, dw = torch.autograd.grad(out, (x, w), state["grad_out"])
    return {"out": out.detach(), "dx": dx, "dweight": dw}


@torch.no_grad()
def _run_plain(state, case):
    if case["op"] == "clip":
        return _plain_clip(state, case)
    return _plain_attend(state, case) if case["op"] == "attend" else _plain_rotate(state, case)


def _plain_clip(state, case):
    grads = state["grads"]
    if case["norm"] == "inf":
        norm = torch.stack([t.abs().max().double() for t in grads]).max()
    else:
        wide = torch.float64 if any(t.dtype == torch.float64 for t in grads) else torch.float32
        norm = torch.stack([t.to(wide).square().sum(dtype=torch.float64) for t in grads]).sum().sqrt()
    coef = (case["max_norm"] / (norm + EPS)).clamp(max=1.0)
    out = []
    for t in grads:
        out.append(t * coef if t.dtype == torch.float64 else (t.float() * coef.float()).to(t.dtype))
    return {"norm": norm if any(t.dtype == torch.float64 for t in grads) else norm.float(), "grads": out}


def _plain_mask(state, case, dev):
    """(B, N, M) bool: the cells inside the lengths and the band; None where all are."""
    N, M, bw = case["N"], case["M"], case["bandwidth"]
    if state["lengths_x"] is None and bw < 0:
        return None
    nx = state["lengths_x"] if state["lengths_x"] is not None else torch.full((case["B"],), N, device=dev)
    ny = state["lengths_y"] if state["lengths_y"] is not None else torch.full((case["B"],), M, device=dev)
    nx, ny = nx.view(-1, 1, 1), ny.view(-1, 1, 1)
    i = torch.arange(N, device=dev).view(1, -1, 1)
    j = torch.arange(M, device=dev).view(1, 1, -1)
    mask = (i < nx) & (j < ny)
    if bw >= 0:
        # |i (ny - 1) - j (nx - 1)| is the distance from the diagonal times (shorter length - 1).
        short, long = torch.minimum(nx, ny) - 1, torch.maximum(nx, ny) - 1
        mask &= (2 * (i * (ny - 1) - j * (nx - 1)).abs() <= torch.maximum(2 * bw * short, long)) | (short <= 0)
    return mask


def _plain_attend(state, case):
    q, k, v = state["q"], state["k"], state["v"]
    B, N, Hq, d = q.shape
    M, Hkv = k.shape[1], k.shape[2]
    group, scale = Hq // Hkv, 1.0 / math.sqrt(d)
    t = q.dtype
    qf = q.float().view(B, N, Hkv, group, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, group * N, d)
    kf = k.float().transpose(1, 2)
    vf = v.float().transpose(1, 2)
    s = torch.matmul(qf, kf.transpose(2, 3)).mul_(scale).view(B, Hkv, group, N, M)
    mask = _plain_mask(state, case, q.device)
    if mask is not None:
        s = s.masked_fill_(~mask.view(B, 1, 1, N, M), -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0)).view(B, Hkv, group * N, M)
    o = torch.matmul(p, vf)

    def rows(x):
        return x.view(B, Hkv, group, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, d).to(t)

    if not case["train"]:
        return {"out": rows(o)}
    do = state["grad_out"].float().view(B, N, Hkv, group, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, group * N, d)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, vf.transpose(2, 3))
    ds = ds.sub_((do * o).sum(dim=-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, kf).mul_(scale)
    dk = torch.matmul(ds.transpose(2, 3), qf).mul_(scale)
    return {"out": rows(o), "dq": rows(dq), "dk": dk.transpose(1, 2).to(t), "dv": dv.transpose(1, 2).to(t)}


def _turn(x, cos, sin, interleaved):
    """The pairs of x's last dimension turned by the angles of cos and sin."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), dim=-1)


def _plain_rotate(state, case):
    x, w = state["x"], state["weight"]
    B, N, H, d = x.shape
    r = case["rotary"]
    pos = state["positions"] if state["positions"] is not None else torch.arange(N, device=x.device).expand(B, N)
    freq = 10000.0 ** (-torch.arange(0, r, 2, device=x.device, dtype=torch.float64) / r)
    angle = pos.double().view(B, N, 1, 1) * freq
    cos, sin = angle.cos().float(), angle.sin().float()
    keep = None
    if state["lengths_x"] is not None:
        keep = (torch.arange(N, device=x.device) < state["lengths_x"].view(B, 1)).view(B, N, 1, 1)
    xf = x.float()
    rstd = (xf.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    unit = xf * rstd
    y = unit * w
    y = torch.cat((_turn(y[..., :r], cos, sin, case["interleaved"]), y[..., r:]), dim=-1)
    if keep is not None:
        y = torch.where(keep, y, 0.0)
    if not case["train"]:
        return {"out": y.to(x.dtype)}
    g = state["grad_out"].float()
    if keep is not None:
        g = torch.where(keep, g, 0.0)
    g = torch.cat((_turn(g[..., :r], cos, -sin, case["interleaved"]), g[..., r:]), dim=-1)
    dw = (g * unit).sum(dim=(0, 1, 2), dtype=torch.float64).float()
    g = g * w
    dx = rstd * (g - unit * (g * unit).mean(dim=-1, keepdim=True))
    return {"out": y.to(x.dtype), "dx": dx.to(x.dtype), "dweight": dw}


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------

@torch.no_grad()
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        return _exact_clip(state, case)
    return _exact_attend(state, case) if case["op"] == "attend" else _exact_rotate(state, case)


def _exact_clip(state, case):
    order = 2 if case["norm"] == "2" else math.inf
    parts = torch.stack([torch.linalg.vector_norm(t.double(), order) for t in state["grads"]])
    norm = torch.linalg.vector_norm(parts, order)
    factor = min(1.0, case["max_norm"] / (float(norm) + EPS))
    return {"norm": norm, "grads": [t.double() * factor for t in state["grads"]]}


def _exact_attend(state, case):
    B, N, M, Hq, Hkv, d = (case[n] for n in ("B", "N", "M", "Hq", "Hkv", "d"))
    lx, ly = _lengths(case)
    bw = case["bandwidth"]
    dev = state["q"].device
    out = torch.zeros(B, N, Hq, d, dtype=torch.float64, device=dev)
    train = case["train"]
    dq = torch.zeros_like(out) if train else None
    dk = torch.zeros(B, M, Hkv, d, dtype=torch.float64, device=dev) if train else None
    dv = torch.zeros_like(dk) if train else None
    for b in range(B):
        nx, ny = lx[b], ly[b]
        if nx == 0 or ny == 0:
            continue
        allowed = None
        K, L = min(nx, ny), max(nx, ny)
        if bw >= 0 and K > 1:
            i, j = torch.arange(nx, device=dev)[:, None], torch.arange(ny, device=dev)[None, :]
            on_short, on_long = (i, j) if nx <= ny else (j, i)
            allowed = 2 * (on_long * (K - 1) - on_short * (L - 1)).abs() <= max(2 * bw * (K - 1), L - 1)
        for h in range(Hkv):
            kh, vh = state["k"][b, :ny, h].double(), state["v"][b, :ny, h].double()
            for hq in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                qh = state["q"][b, :nx, hq].double()
                score = qh @ kh.T / math.sqrt(d)
                if allowed is not None:
                    score = score.masked_fill(~allowed, -math.inf)
                prob = torch.softmax(score, dim=1)
                out[b, :nx, hq] = prob @ vh
                if train:
                    g = state["grad_out"][b, :nx, hq].double()
                    dp = g @ vh.T
                    dscore = prob * (dp - (prob * dp).sum(1, keepdim=True)) / math.sqrt(d)
                    dq[b, :nx, hq] = dscore @ kh
                    dk[b, :ny, h] += dscore.T @ qh
                    dv[b, :ny, h] += prob.T @ g
    return {"out": out, "dq": dq, "dk": dk, "dv": dv} if train else {"out": out}


def _exact_rotate(state, case):
    """The rotation as products of complex numbers; gradients a sample at a time."""
    B, N, H, d = (case[n] for n in ("B", "N", "H", "d"))
    r, half = case["rotary"], case["rotary"] // 2
    dev = state["x"].device
    lx, _ = _lengths(case)
    index = torch.arange(r, device=dev)
    first = index[0::2] if case["interleaved"] else index[:half]
    second = index[1::2] if case["interleaved"] else index[half:]
    w = state["weight"].double()
    freq = torch.exp(torch.arange(half, device=dev, dtype=torch.float64) * (-2.0 / r * math.log(10000.0)))
    out = torch.zeros(B, N, H, d, dtype=torch.float64, device=dev)
    dx, dw = torch.zeros_like(out), torch.zeros(d, dtype=torch.float64, device=dev)
    for b in range(B):
        n = lx[b]
        pos = torch.arange(n, device=dev) if state["positions"] is None else state["positions"][b, :n]
        angle = pos.double()[:, None, None] * freq
        spin = torch.polar(torch.ones_like(angle), angle)
        x = state["x"][b, :n].double()
        ms = x.square().sum(-1, keepdim=True) / d + EPS
        unit = x / ms.sqrt()
        y = unit * w
        z = torch.complex(y[..., first], y[..., second]) * spin
        y[..., first], y[..., second] = z.real, z.imag
        out[b, :n] = y
        if case["train"]:
            g = state["grad_out"][b, :n].double()
            z = torch.complex(g[..., first], g[..., second]) * spin.conj()
            g[..., first], g[..., second] = z.real, z.imag
            dw += (g * unit).sum((0, 1))
            g = g * w
            dx[b, :n] = g / ms.sqrt() - x * (g * x).sum(-1, keepdim=True) / (d * ms * ms.sqrt())
    return {"out": out, "dx": dx, "dweight": dw} if case["train"] else {"out": out}
