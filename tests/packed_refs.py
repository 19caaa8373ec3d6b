"""The packed-batch operators in 64 bits, with the error each kernel's roundings allow.

``u(dtype)`` is half a step of a type relative to the value. A bound counts the roundings the
kernels document (operands of an MFMA product, outputs) against the sums of absolute values
they enter, plus ``f`` for fp32 arithmetic: products and sums in 32 bits are off by at most
the number of terms added one after the other times 2^-24 of their absolute sum.
"""

import torch


def u(dtype) -> float:
    return torch.finfo(dtype).eps / 2


F32 = 2.0 ** -24


def attention64(q, k, v, do, lengths, mfma):
    """[(value, bound)] of o, dq, dk, dv. ``mfma``: P and dS are rounded to the tensors' type
    before their products; the backward's delta is formed from the rounded o either way."""
    dt = q.dtype
    q, k, v, do = (t.double() for t in (q, k, v, do))
    T, H, D = q.shape
    group = H // k.shape[1]
    c = D ** -0.5
    out = [[torch.zeros_like(t), torch.zeros_like(t)] for t in (q, q, k, v)]
    ur = u(dt) if mfma else 0.0
    # below 2^-14 fp16 numbers lie 2^-24 apart, so a P or dS down there moves by up to 2^-25
    us = 2.0 ** -25 if mfma and dt == torch.float16 else 0.0
    a = 0
    for n in lengths:
        r = slice(a, a + n)
        a += n
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        f = F32 * (n + 2 * D + 32)
        for h in range(H):
            g = h // group
            Q, K, V, DO = q[r, h], k[r, g], v[r, g], do[r, h]
            s = (Q @ K.T * c).masked_fill(hidden, float("-inf"))
            p = torch.softmax(s, -1)
            # scores summed in fp32 shift p by their absolute error; exp2 and the row sum add more
            es = F32 * (D + 8) * (Q.abs() @ K.abs().T * c)
            es = es.masked_fill(hidden, 0.0)
            # fp32's (and bf16's) smallest normal number is 2^-126: a p below it may become zero,
            # an error of p itself, at most 2^-126
            ep = p * (es + (p * es).sum(-1, keepdim=True) + f) + torch.clamp(p, max=2.0 ** -126)
            o = p @ V
            seen = (~hidden).double()
            eo = (ur * p + us * seen + ep) @ V.abs() + f * (p @ V.abs()) + u(dt) * o.abs()
            delta = (DO * o).sum(-1, keepdim=True)
            edelta = (DO.abs() * (eo + f * o.abs())).sum(-1, keepdim=True)
            dp = DO @ V.T
            edp = f * (DO.abs() @ V.abs().T)
            ds = p * (dp - delta)
            eds = ep * (dp - delta).abs() + p * (edp + edelta) + (ur + f) * ds.abs() + us * seen
            dq, edq = c * (ds @ K), c * (eds @ K.abs() + f * (ds.abs() @ K.abs()))
            dk, edk = c * (ds.T @ Q), c * (eds.T @ Q.abs() + f * (ds.abs().T @ Q.abs()))
            dv, edv = p.T @ DO, (ur * p + us * seen + ep + f * p).T @ DO.abs()
            for i, (x, e, at) in enumerate(((o, eo, h), (dq, edq, h), (dk, edk, g), (dv, edv, g))):
                out[i][0][r, at] += x
                out[i][1][r, at] += e
    for i in (1, 2, 3):
        out[i][1] += u(dt) * out[i][0].abs()
    # below the smallest normal number a half step is absolute (fp16), or the number is zero
    for pair in out:
        pair[1] += (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)
    return [tuple(p) for p in out]


def rotary64(x, positions, freqs, amplitude, interleaved, inverse=False):
    """(value, bound) of the rotation (its transpose with ``inverse``)."""
    dt = x.dtype
    x = x.double()
    angle = positions.double()[:, None, None] * freqs.double()
    cos, sin = amplitude * angle.cos(), amplitude * angle.sin() * (-1 if inverse else 1)
    n = freqs.shape[0]
    part = x[..., :2 * n]
    x1, x2 = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n], part[..., n:])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    # the reduced angle (2^-24 of an eighth turn), sine and cosine (2 steps), amplitude, products
    # and sum, 8 steps in all; and the fp64 product of a far position, 2^-52 of the angle twice
    e = abs(amplitude) * (x1.abs() + x2.abs()) * (8 * F32 + angle.abs() * 2.0 ** -51)

    def join(a, b):
        return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)

    value = torch.cat((join(y1, y2), x[..., 2 * n:]), -1)
    bound = torch.cat((join(e, e), 0 * x[..., 2 * n:]), -1) + u(dt) * value.abs()
    bound[..., 2 * n:] = 0  # copied columns are exact
    if dt == torch.float16:
        bound[..., :2 * n] += 2.0 ** -25
    return value, bound


def block_norm64(x, h, w1, gate, w2, alpha, eps, ds, dy):
    """{name: (value, bound)} of s, y and the gradients. K bounds the fp32 arithmetic: a thread
    adds at most 32 terms in turn, a workgroup's 16 waves and 64 lanes add 22 more, and up to
    40 roundings act on a term on its way; column sums add their own rows' count."""
    dt = x.dtype
    rows, cols = x.shape
    K = F32 * (128 + cols / 1024 + rows / 512)
    x, h, w1, w2, ds, dy = (t.double() for t in (x, h, w1, w2, ds, dy))
    g = torch.ones((), dtype=torch.float64, device=x.device) if gate is None else gate.double()

    def mean(t):
        return t.mean(-1, keepdim=True)

    rh = (mean(h * h) + eps).rsqrt()
    hhat = h * rh
    n = hhat * w1
    s = x + alpha * g * n
    es = K * (x.abs() + (alpha * g * n).abs())
    rs = (mean(s * s) + eps).rsqrt()
    shat = s * rs
    eshat = es * rs + shat.abs() * (K + mean(es * s.abs()) * rs * rs)
    y = shat * w2
    out = {"s": (s, es), "y": (y, eshat * w2.abs() + K * y.abs())}
    dyw = dy * w2
    m1 = mean(dyw * shat)
    em1 = mean(dyw.abs() * (eshat + K * shat.abs()))
    e = ds + rs * (dyw - shat * m1)
    ee = (K * (ds.abs() + rs * (dyw.abs() + (shat * m1).abs()))
          + rs * (eshat * m1.abs() + shat.abs() * em1)
          + (rs * (dyw - shat * m1)).abs() * mean(es * s.abs()) * rs * rs)
    dn, edn = alpha * g * e, (alpha * g).abs() * (ee + K * e.abs())
    b, eb = dn * w1, edn * w1.abs()
    m2, em2 = mean(b * hhat), mean((eb + K * b.abs()) * hhat.abs())
    dh = rh * (b - hhat * m2)
    out["dx"] = (e, ee)
    out["dh"] = (dh, rh * (eb + hhat.abs() * em2 + K * (b.abs() + (hhat * m2).abs())))
    out["dpost_weight"] = ((dn * hhat).sum(0), ((edn + K * dn.abs()) * hhat.abs()).sum(0))
    if gate is not None:
        dg, edg = alpha * e * n, abs(alpha) * (ee + K * e.abs()) * n.abs()
        if gate.dim() == 1:
            dg, edg = dg.sum(0), edg.sum(0)
        elif gate.shape[1] == 1 and cols > 1:
            dg, edg = dg.sum(1, keepdim=True), edg.sum(1, keepdim=True)
        out["dgate"] = (dg, edg)
    out["dpre_weight"] = ((dy * shat).sum(0), (dy.abs() * (eshat + K * shat.abs())).sum(0))
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    return {k: (v, e + u(dt) * v.abs() + tiny) for k, (v, e) in out.items()}


def assert_within(name, got, value, bound):
    assert got.shape == value.shape, (name, tuple(got.shape), tuple(value.shape))
    over = (got.double() - value).abs() - bound
    bad = ~(over <= 0)
    if bool(bad.any()):
        i = int(torch.where(bad, over.nan_to_num(float("inf"), float("inf")), -1.0).argmax())
        raise AssertionError(
            f"{name}: {int(bad.sum())} of {got.numel()} beyond the bound, worst at flat {i}: got "
            f"{float(got.flatten()[i])}, want {float(value.flatten()[i])} +- "
            f"{float(bound.flatten()[i]):.3g}")
