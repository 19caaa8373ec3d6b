"""The operators of a distillation step in 64 bits, with the error each kernel's roundings allow.

As in tests/packed_refs.py: ``u(dtype)`` is half a step of a type relative to the value, F32 that
of fp32, and sums of n terms one after the other are off by at most n F32 of their absolute sum.
"""

import torch

from tests.packed_refs import F32, u


def tiny(dtype):
    """Half a step below the smallest normal number (fp16), or all of it (flushed to zero)."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def embedding64(weight, ids, scale, ignore_index, dout):
    """(value, bound) of out and of dweight; NaN rows for ids outside the table."""
    dt, ids = weight.dtype, ids.long().flatten()
    w, d = weight.double(), dout.double().reshape(len(ids), -1)
    inside = (ids >= 0) & (ids < w.shape[0]) & (ids != ignore_index)
    out = scale * w[torch.where(inside, ids, 0)]
    fill = torch.where(ids == ignore_index, 0.0, float("nan")).double()
    out = torch.where(inside[:, None], out, fill[:, None])
    grad, size = torch.zeros_like(w), torch.zeros_like(w)
    grad.index_add_(0, ids[inside], d[inside])
    size.index_add_(0, ids[inside], d[inside].abs())
    count = torch.bincount(ids[inside], minlength=w.shape[0])[:, None]
    # the scale's own rounding and its product are two steps
    grad *= scale
    bound = abs(scale) * size * F32 * (count + 2) + u(dt) * grad.abs() + tiny(dt) * (count > 0)
    return (out, (2 * F32 + u(dt)) * out.abs() + tiny(dt)), (grad, bound)


def _turn(a, cos, sin, n, interleaved):
    """The rotation of the first 2n columns, and |a| + |b| of each pair in both its places."""
    part, rest = a[..., :2 * n], a[..., 2 * n:]
    x, y = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])

    def join(p, q):
        out = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
        return out

    size = x.abs() + y.abs()
    return (torch.cat((join(x * cos - y * sin, y * cos + x * sin), rest), -1),
            torch.cat((join(size, size), rest.abs()), -1))


def norm_rotary64(x, weight, positions, freqs, eps, amplitude, interleaved, dy):
    """{name: (value, bound)} of y, dx and dweight."""
    dt, n = x.dtype, freqs.shape[0]
    T, H, D = x.shape
    # a lane adds up to 16 squares (64-lane walks: D / 64 pairs), 6 steps join the lanes, and
    # up to 20 roundings act on a term on its way
    K = F32 * (48 + D / 32)
    x, w, dy = x.double(), weight.double(), dy.double()
    angle = positions.double()[:, None, None] * freqs.double()
    cos, sin = amplitude * angle.cos(), amplitude * angle.sin()
    # sine and cosine (rotary64 of packed_refs): 8 steps, and the fp64 product of a far position
    ea = 8 * F32 + float(angle.abs().max() if angle.numel() else 0) * 2.0 ** -51
    amp = torch.ones(D, dtype=torch.float64, device=x.device)
    amp[:2 * n] = abs(amplitude)

    rstd = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xhat = x * rstd
    y, size = _turn(xhat * w, cos, sin, n, interleaved)
    out = {"y": (y, amp * size * (K + ea) + u(dt) * y.abs() + tiny(dt))}
    dn, size = _turn(dy, cos, -sin, n, interleaved)
    edn = amp * size * ea
    g, eg = dn * w, (edn + K * dn.abs()) * w.abs()
    m, em = (g * xhat).mean(-1, keepdim=True), ((eg + K * g.abs()) * xhat.abs()).mean(-1, keepdim=True)
    dx = rstd * (g - xhat * m)
    edx = rstd * (eg + xhat.abs() * em + K * (g.abs() + (xhat * m).abs()))
    out["dx"] = (dx, edx + u(dt) * dx.abs() + tiny(dt))
    # a lane adds the tokens of its workgroup, then 512 lanes' rows and a card's partial rows
    N = T / 256 + 512 + 2048 / 64 + 8
    dw, edw = (dn * xhat).sum((0, 1)), ((edn + (K + N * F32) * dn.abs()) * xhat.abs()).sum((0, 1))
    out["dweight"] = (dw, edw + u(dt) * dw.abs() + tiny(dt))
    return out


def distill64(logits, target, teacher, ids, tau, soft, hard, ignore_index, dloss):
    """(value, bound) of the loss and of dlogits."""
    dt = logits.dtype
    rows, cols = logits.shape
    live = target != ignore_index
    n = int(live.sum())
    z, t, ids = logits.double(), teacher.double(), ids.long()
    inside, label = ids >= 0, torch.where(live, target, 0).clamp(0, cols - 1)[:, None]
    at = torch.where(inside, ids, 0)
    m = z.amax(1, keepdim=True)
    d = (z - m).abs()
    # sums over a row: a thread adds a 64th of it or less and 20 more steps join the parts. An
    # exponential's argument is off by 3 roundings of itself, and each is off by 2 steps more.
    N = cols / 64 + 32

    def softmax(c):
        q = torch.softmax(z * c, 1)
        es = F32 * (N + 4 + 3 * (q * d * c).sum(1, keepdim=True))  # of the sum, relative
        return q, torch.logsumexp(z * c, 1, keepdim=True) - m * c, es

    t = torch.where(inside, t / tau, -float("inf"))
    tm = torch.where(inside.any(1, keepdim=True), t.amax(1, keepdim=True), 0.0)
    tm = torch.where(tm.isinf(), 0.0, tm)
    some = (t > -float("inf")).any(1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, t, 0.0), 1), 0.0)
    td = torch.where(p > 0, (t - tm).abs(), 0.0)
    et = F32 * (ids.shape[1] + 16 + 3 * (p * td).sum(1, keepdim=True))
    elogp = F32 * 3 * td + et + 2 * F32 * (p * td).sum(1, keepdim=True)
    ep = p * (F32 * (3 * td + 4) + et)

    q, lq, eq = softmax(1.0 / tau)
    logq = (z - m).gather(1, at) / tau - lq
    elogq = F32 * (3 * d.gather(1, at) / tau + 3 * lq.abs()) + eq
    logp = torch.where(p > 0, torch.log(torch.where(p > 0, p, 1.0)), 0.0)
    logq = torch.where(p > 0, logq, 0.0)
    gap = logp - logq
    row = soft * tau ** 2 * (p * gap).sum(1)
    erow = abs(soft) * tau ** 2 * (ep * gap.abs() + p * (elogp + elogq)
                                   + F32 * (ids.shape[1] + 8) * (p * (logp.abs() + logq.abs()))).sum(1)
    h, lh, eh = softmax(1.0)
    if hard:
        each = lh[:, 0] - (z - m).gather(1, label)[:, 0]
        row = row + hard * each
        erow = erow + abs(hard) * (F32 * 3 * (lh[:, 0].abs() + d.gather(1, label)[:, 0]) + eh[:, 0])
    row, erow = torch.where(live, row, 0.0), torch.where(live, erow, 0.0)
    loss = row.sum() / n
    eloss = (erow.sum() + F32 * (rows / 1024 + 40) * row.abs().sum()) / n

    g = float(dloss) / n
    eexp = lambda c: F32 * (3 * d * c + 6)  # noqa: E731
    overlay = torch.zeros_like(z).scatter_add_(1, at, torch.where(inside, p, 0.0))
    eover = torch.zeros_like(z).scatter_add_(1, at, torch.where(inside, ep + F32 * 4 * p, 0.0))
    gs = g * soft * tau
    grad = gs * (q * some - overlay)
    egrad = abs(gs) * (q * some * (eexp(1.0 / tau) + eq) + eover + F32 * 4 * (q * some + overlay))
    if hard:
        one = torch.zeros_like(z).scatter_(1, label, 1.0)
        grad = grad + g * hard * (h - one)
        egrad = egrad + abs(g * hard) * (h * (eexp(1.0) + eh) + F32 * 6 * (h + one))
    egrad = egrad + F32 * 4 * grad.abs() + abs(g) * (abs(soft) * tau + abs(hard)) * 2.0 ** -126
    grad, egrad = (torch.where(live[:, None], v, 0.0) for v in (grad, egrad))
    return (loss, eloss + F32 * loss.abs()), (grad, egrad + u(dt) * grad.abs() + tiny(dt))
