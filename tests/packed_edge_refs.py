"""Causal attention of one packed batch in 64 bits for the cases at the edge of the kernels'
arithmetic, with the error that their roundings allow: tests/packed_refs.py's count, but for a
delta formed in fp32 (rows whose keys fit one tile) and for dS beyond fp16's range."""

import torch

from tests.packed_refs import F32, u


def takes_mfma(dtype, D):
    return dtype != torch.float32 and D in (64, 128)


def attention64(q, k, v, do, lengths, half_range=False):
    """({name: (value, bound)} of o, dq, dk, dv, lse, the largest |dS|). The MFMA kernels round P and
    dS to the tensors' type before their products. delta of a sequence's first rows, whose keys fit
    one tile, is sum p dp in fp32; the others' takes the stored o. ``half_range``: a row's or a key's
    dS of a tile, past 2^15, is rounded to fp16 as a multiple of the power of two that brings the
    largest below 2^15."""
    dt, mfma = q.dtype, takes_mfma(q.dtype, q.shape[2])
    tile = 64 if mfma else 32 if q.shape[2] <= 64 else 16
    q, k, v, do = (t.double() for t in (q, k, v, do))
    T, H, D = q.shape
    group, c = H // k.shape[1], D ** -0.5
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)]
           for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v), ("lse", q[..., 0].T))}
    ur = u(dt) if mfma else 0.0
    half = mfma and dt == torch.float16
    up = 2.0 ** -25 if half else 0.0  # half of fp16's smallest step
    most = 0.0
    a = 0
    for n in lengths:
        r = slice(a, a + n)
        a += n
        if n == 0:
            continue
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        seen = (~hidden).double()
        f = F32 * (n + 2 * D + 32)
        for h in range(H):
            g = h // group
            Q, K, V, DO = q[r, h], k[r, g], v[r, g], do[r, h]
            s = (Q @ K.T * c).masked_fill(hidden, float("-inf"))
            p = torch.softmax(s, -1)
            es = (F32 * (D + 8) * (Q.abs() @ K.abs().T * c)).masked_fill(hidden, 0.0)
            epsum = (p * es).sum(-1, keepdim=True)
            ep = p * (es + epsum + f) + torch.clamp(p, max=2.0 ** -126)
            o = p @ V
            eo = (ur * p + up * seen + ep) @ V.abs() + f * (p @ V.abs()) + u(dt) * o.abs()
            dp = DO @ V.T
            edp = f * (DO.abs() @ V.abs().T)
            delta = (p * dp).sum(-1, keepdim=True)
            edelta = (ep * dp.abs() + p * edp + f * p * dp.abs()).sum(-1, keepdim=True)
            stored = (DO.abs() * (eo + f * o.abs())).sum(-1, keepdim=True)
            edelta[tile:] = torch.maximum(edelta, stored)[tile:]
            ds = p * (dp - delta)
            big = float(ds.abs().max())
            most = max(most, big)
            # a tile's power of two is at most twice its largest over 2^15
            us = up * max(1.0, 2.0 * big / 2.0 ** 15) if half_range else up
            eds = ep * (dp - delta).abs() + p * (edp + edelta) + (ur + f) * ds.abs() + us * seen
            got = {"o": (o, eo, h),
                   "dq": (c * (ds @ K), c * (eds @ K.abs() + f * (ds.abs() @ K.abs())), h),
                   "dk": (c * (ds.T @ Q), c * (eds.T @ Q.abs() + f * (ds.abs().T @ Q.abs())), g),
                   "dv": (p.T @ DO, (ur * p + up * seen + ep + f * p).T @ DO.abs(), g)}
            for name, (x, e, at) in got.items():
                out[name][0][r, at] += x
                out[name][1][r, at] += e
            lse = torch.logsumexp(s, -1)
            out["lse"][0][h, r] = lse
            # the scores' error, the sum's, and two fp32 roundings of its logarithm and the result
            out["lse"][1][h, r] = epsum[:, 0] + f + 4 * F32 * lse.abs()
    for name in ("dq", "dk", "dv"):
        out[name][1] += u(dt) * out[name][0].abs()
    for name in ("o", "dq", "dk", "dv"):
        out[name][1] += 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
    return {n: tuple(x) for n, x in out.items()}, most
