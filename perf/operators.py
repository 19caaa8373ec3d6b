"""Performance cases of the packed-batch operators: attention over packed prompts, rotary
positions per token, and the norms around a block with its gate and residual scale.

A pass is a training step's use of one operator through its public functions, forward then
backward, or the forward alone as an evaluation or a generation step runs it. With ``own``
false the same results come from elementary torch operations in fp32 (angles in fp64).
``exact`` evaluates a case in fp64 from the operators' definitions, its gradients by
differentiating them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
EPS = 1e-6


# ------------------------------------------------------------------------------ cases
def _attn(H, KVH, D, seqs, total, longest, pad, dtype, passes="step", mix=0, **more):
    """``total`` tokens in ``seqs`` sequences, the longest of ``longest``, the others'
    lengths spread over their logarithm; ``pad`` rows behind the last sequence."""
    return dict(kind="attention", H=H, KVH=KVH, D=D, seqs=seqs, total=total, longest=longest,
                pad=pad, dtype=dtype, passes=passes, mix=mix, **more)


def _rotary(T, H, KVH, D, R, layout, scaling, far, dtype, passes="step", **more):
    """q and k of T tokens, R of the D columns of a head rotated, positions up to ``far``."""
    return dict(kind="rotary", T=T, H=H, KVH=KVH, D=D, R=R, layout=layout, scaling=scaling,
                far=far, dtype=dtype, passes=passes, **more)


def _norm(rows, cols, gate, alpha, dtype, passes="step", **more):
    """``gate``: "none", "channel" [cols], "row" [rows, 1] or "element" [rows, cols]."""
    return dict(kind="block_norm", rows=rows, cols=cols, gate=gate, alpha=alpha, dtype=dtype,
                passes=passes, **more)


def listed():
    return [
        # The smallest attention: a few short prompts of a small model checked in fp32.
        _attn(4, 1, 32, 3, 77, 33, 0, "float32", mix=1, name="attention_3x77_4x1x32_fp32"),
        # fp32 training of a small grouped-query model on one packed batch.
        _attn(8, 2, 64, 6, 1500, 700, 36, "float32", mix=2, name="attention_6x1500_8x2x64_fp32"),
        # Chat turns: many prompts of tens of tokens, Llama-3-8B heads.
        _attn(32, 8, 128, 160, 4096, 120, 0, "bfloat16", mix=3,
              name="attention_160x4096_32x8x128_bf16"),
        # Multi-head fp16 encoder-decoder heads of 64 columns, ragged lengths and padding.
        _attn(12, 12, 64, 9, 2901, 1111, 171, "float16", mix=4,
              name="attention_9x2901_12x12x64_fp16"),
        # The ordinary training batch of Llama-3-8B heads: documents packed to 8192 tokens.
        _attn(32, 8, 128, 11, 8192, 3001, 0, "bfloat16", mix=5,
              name="attention_11x8192_32x8x128_bf16"),
        # The largest: a long-context batch with one document of 16384 tokens.
        _attn(32, 8, 128, 7, 32768, 16384, 0, "bfloat16", mix=6,
              name="attention_7x32768_32x8x128_bf16"),
        # A generation step: one token of each of 32 requests, far into a scaled context.
        _rotary(32, 32, 8, 128, 128, "half", "bands", 131072, "bfloat16", passes="forward",
                name="rotary_32tok_bf16"),
        # Interleaved pairs over part of the head, an odd token count, base scaling.
        _rotary(5003, 16, 16, 96, 64, "interleaved", "base", 32768, "float16",
                name="rotary_5003tok_partial_fp16"),
        # A long packed batch of Llama-3-8B heads.
        _rotary(32768, 32, 8, 128, 128, "half", "none", 16384, "bfloat16",
                name="rotary_32768tok_bf16"),
        # The norms around a block of a small fp32 model, a learned gate per channel.
        _norm(64, 768, "channel", 1.0, "float32", name="block_norm_64x768_fp32"),
        # A gate per element (a modulated block) over an odd number of rows, odd width.
        _norm(4099, 1538, "element", 0.5, "bfloat16", name="block_norm_4099x1538_bf16"),
        # The norms around a block of a Llama-3-8B-sized layer over a large batch.
        _norm(16384, 4096, "channel", 0.7071, "bfloat16", name="block_norm_16384x4096_bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: sizes log-uniform, odd ones among them."""
    kind = rng.choice(["attention", "attention", "attention", "rotary", "rotary", "block_norm",
                       "block_norm"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    passes = rng.choice(["step", "step", "step", "forward"])
    if kind == "attention":
        kvh = rng.choice([1, 2, 4, 8])
        H = min(32, kvh * rng.choice([1, 2, 4, 8]))
        if dtype == "float32":
            kvh, H = min(kvh, 2), min(H, 8)
            D = rng.choice([16, 32, 64, 80, 128])
            total = _log(rng, 16, 2048)
        else:
            D = rng.choice([64, 64, 128, 128, 128, 96])
            total = _log(rng, 16, 16384 if D != 96 else 2048)
        longest = _log(rng, max(1, total // 32), total)
        seqs = -(-total // longest) + rng.randint(0, 24)
        seqs = 1 if longest == total else max(seqs, 2)
        return _attn(H, kvh, D, seqs, total, longest, rng.choice([0, 0, rng.randint(1, 200)]),
                     dtype, passes, mix=rng.randint(1, 10 ** 6))
    if kind == "rotary":
        kvh = rng.choice([1, 2, 4, 8])
        H = min(32, kvh * rng.choice([1, 2, 4, 8]))
        D = rng.choice([64, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, D // 2, D // 4])
        return _rotary(_log(rng, 1, 16384), H, kvh, D, R, rng.choice(["half", "interleaved"]),
                       rng.choice(["none", "linear", "base", "bands"]), _log(rng, 4096, 1 << 20),
                       dtype, passes)
    cols = _log(rng, 256, 8192)
    cols = cols if rng.random() < 0.25 else max(64, cols // 64 * 64)
    return _norm(_log(rng, 1, 16384 if cols <= 4096 else 8192), cols,
                 rng.choice(["none", "channel", "row", "element"]), rng.choice([1.0, 0.5, 0.7071]),
                 dtype, passes)


def _lengths(case):
    """The sequences' lengths: the longest first drawn into a place of its own, the others
    log-uniform and scaled to the total, an empty one where a batch of many has one."""
    total, n, longest = case["total"], case["seqs"], case["longest"]
    rng = random.Random(case["mix"])
    if n == 1:
        return [total]
    rest, cap = total - longest, longest
    weights = [math.exp(rng.uniform(0.0, 3.0)) for _ in range(n - 1)]
    scale = rest / sum(weights)
    lens = [min(cap, int(w * scale)) for w in weights]
    left = rest - sum(lens)
    for i in sorted(range(n - 1), key=lambda i: lens[i]):  # what rounding and the cap left
        add = min(cap - lens[i], left)
        lens[i] += add
        left -= add
    lens.insert(rng.randrange(n), longest)
    assert sum(lens) == total and min(lens) >= 0 and max(lens) == longest
    return lens


def _pairs(case):
    return sum(n * (n + 1) // 2 for n in _lengths(case))


def work(case):
    e, step = SIZE[case["dtype"]], case["passes"] == "step"
    if case["kind"] == "attention":
        T, H, KVH, D = case["total"] + case["pad"], case["H"], case["KVH"], case["D"]
        q, kv = T * H * D, T * KVH * D
        elements = 2 * q + 2 * kv + (2 * q + 2 * kv if step else 0)
        return {"bytes": e * elements, "flops": (14 if step else 4) * D * H * _pairs(case)}
    if case["kind"] == "rotary":
        n = case["T"] * (case["H"] + case["KVH"]) * case["D"]
        return {"bytes": e * n * (4 if step else 2), "flops": 3 * n * (2 if step else 1)}
    n = case["rows"] * case["cols"]
    g = {"none": 0, "channel": case["cols"], "row": case["rows"], "element": n}[case["gate"]]
    return {"bytes": e * (n * (8 if step else 4) + g * (2 if step else 1)),
            "flops": n * (40 if step else 12)}


# ----------------------------------------------------------------------------- inputs
def _generator(case, seed):
    text = repr(sorted((k, v) for k, v in case.items() if k != "name")) + f"|{seed}"
    return torch.Generator(device=DEVICE).manual_seed(random.Random(text).getrandbits(48))


def _inputs(case, seed):
    """The tensors a pass is given, from the case and the seed alone."""
    gen, dt = _generator(case, seed), DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dt)

    if case["kind"] == "attention":
        T, H, KVH, D = case["total"] + case["pad"], case["H"], case["KVH"], case["D"]
        bounds = [0]
        for n in _lengths(case):
            bounds.append(bounds[-1] + n)
        # q, k and v as one projection gives them: column ranges of the same rows
        qkv = normal(T, (H + 2 * KVH) * D)
        return dict(q=qkv[:, :H * D].view(T, H, D),
                    k=qkv[:, H * D:(H + KVH) * D].view(T, KVH, D),
                    v=qkv[:, (H + KVH) * D:].view(T, KVH, D), do=normal(T, H, D),
                    cu=torch.tensor(bounds, dtype=torch.int32, device=DEVICE))
    if case["kind"] == "rotary":
        T, H, KVH, D = case["T"], case["H"], case["KVH"], case["D"]
        positions = torch.randint(0, case["far"], (T,), generator=gen, device=DEVICE)
        if case["passes"] == "step":  # a packed batch: runs of consecutive positions
            run = torch.arange(T, device=DEVICE)
            positions = (positions[0] + run) % case["far"]
        return dict(q=normal(T, H, D), k=normal(T, KVH, D), dq=normal(T, H, D),
                    dk=normal(T, KVH, D), positions=positions.to(torch.int32))
    rows, cols = case["rows"], case["cols"]
    shape = {"none": None, "channel": (cols,), "row": (rows, 1), "element": (rows, cols)}
    shape = shape[case["gate"]]
    out = dict(x=normal(rows, cols), h=normal(rows, cols),
               w1=(1.0 + 0.1 * normal(cols).float()).to(dt),
               w2=(1.0 + 0.1 * normal(cols).float()).to(dt), dout=normal(2, rows, cols))
    out["gate"] = None if shape is None else (0.5 + 0.2 * normal(*shape).float()).to(dt)
    return out


THETA, FACTOR, TRAINED, LOW, HIGH = 500000.0, 8.0, 8192, 1.0, 4.0


def _frequencies(case):
    """Radians per position of each pair, fp64."""
    R = case["R"]
    i = torch.arange(0, R, 2, dtype=torch.float64, device=DEVICE)
    kind = case["scaling"]
    theta = THETA * FACTOR ** (R / (R - 2)) if kind == "base" else THETA
    f = theta ** (-i / R)
    if kind == "linear":
        f = f / FACTOR
    if kind == "bands":
        turns = TRAINED * f / (2 * math.pi)  # over the trained context
        keep = ((turns - LOW) / (HIGH - LOW)).clamp(0.0, 1.0)
        f = keep * f + (1.0 - keep) * f / FACTOR
    return f


SCALING = {
    "none": None,
    "linear": {"kind": "linear", "factor": FACTOR},
    "base": {"kind": "base", "factor": FACTOR},
    "bands": {"kind": "bands", "factor": FACTOR, "context": TRAINED, "low": LOW, "high": HIGH},
}


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "attention":
        state["bounds"] = state["cu"].tolist()  # the batch's own lengths, which its loader has
    if case["kind"] == "rotary":
        if own:
            from evograd_amd.pairs import rotary

            state["freqs"] = rotary.rotary_frequencies(case["R"], THETA, SCALING[case["scaling"]],
                                                       device=DEVICE)
        else:
            state["freqs"] = _frequencies(case)
    return state


# ------------------------------------------------------------------------- plain forms
def _plain_attention(st, step):
    q, k, v, do = st["q"], st["k"], st["v"], st["do"]
    T, H, D = q.shape
    KVH, dt = k.shape[1], q.dtype
    group, scale = H // KVH, D ** -0.5
    o = torch.zeros(T, H, D, dtype=torch.float32, device=q.device)
    grads = [torch.zeros(t.shape, dtype=torch.float32, device=q.device)
             for t in (q, k, v)] if step else None
    for a, b in zip(st["bounds"][:-1], st["bounds"][1:]):
        n = b - a
        if n == 0:
            continue
        masked = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
        # as many heads at a time as keep the scores near a gigabyte
        at_once = max(1, min(KVH, (1 << 28) // max(1, group * n * n)))
        for g0 in range(0, KVH, at_once):
            g1 = min(KVH, g0 + at_once)
            heads = slice(g0 * group, g1 * group)

            def split(t):
                return t[a:b, heads].float().transpose(0, 1).contiguous()

            def shared(t):
                return (t[a:b, g0:g1].float().transpose(0, 1)
                        .repeat_interleave(group, 0).contiguous())

            qs, ks, vs = split(q), shared(k), shared(v)
            s = torch.matmul(qs, ks.transpose(1, 2).contiguous()) * scale
            s.masked_fill_(masked, -math.inf)
            s -= s.amax(-1, keepdim=True)
            p = s.exp_()
            p /= p.sum(-1, keepdim=True)
            os = torch.matmul(p, vs)
            o[a:b, heads] = os.transpose(0, 1)
            if not step:
                continue
            dos = split(do)
            per_head = torch.matmul(p.transpose(1, 2).contiguous(), dos)
            grads[2][a:b, g0:g1] = per_head.view(g1 - g0, group, n, D).sum(1).transpose(0, 1)
            ds = torch.matmul(dos, vs.transpose(1, 2).contiguous())
            ds -= (dos * os).sum(-1, keepdim=True)
            ds *= p
            ds *= scale
            grads[0][a:b, heads] = torch.matmul(ds, ks).transpose(0, 1)
            per_head = torch.matmul(ds.transpose(1, 2).contiguous(), qs)
            grads[1][a:b, g0:g1] = per_head.view(g1 - g0, group, n, D).sum(1).transpose(0, 1)
    if not step:
        return o.to(dt)
    return (o.to(dt), *(g.to(dt) for g in grads))


def _plain_turn(x, cos, sin, layout, R):
    out = x.float().clone()
    if layout == "half":
        a, b = slice(0, R // 2), slice(R // 2, R)
    else:
        a, b = slice(0, R, 2), slice(1, R, 2)
    x1, x2 = x[..., a].float(), x[..., b].float()
    out[..., a] = x1 * cos - x2 * sin
    out[..., b] = x2 * cos + x1 * sin
    return out.to(x.dtype)


def _plain_rotary(st, step):
    case = st["case"]
    angle = st["positions"].double()[:, None, None] * st["freqs"]
    cos, sin = angle.cos().float(), angle.sin().float()
    turn = [(st["q"], sin), (st["k"], sin)]
    if step:
        turn += [(st["dq"], -sin), (st["dk"], -sin)]
    return tuple(_plain_turn(t, cos, sn, case["layout"], case["R"]) for t, sn in turn)


def _plain_block_norm(st, step):
    x, h, w1, w2 = (st[n].float() for n in ("x", "h", "w1", "w2"))
    gate, alpha, dt = st["gate"], st["case"]["alpha"], st["x"].dtype
    g = 1.0 if gate is None else gate.float()
    rh = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hhat = h * rh
    s = x + alpha * g * (hhat * w1)
    rs = (s.square().mean(-1, keepdim=True) + EPS).rsqrt()
    shat = s * rs
    out = torch.stack((s, shat * w2)).to(dt)
    if not step:
        return out
    ds, dy = st["dout"][0].float(), st["dout"][1].float()
    dyw = dy * w2
    dx = ds + rs * (dyw - shat * (dyw * shat).mean(-1, keepdim=True))
    dn = alpha * g * dx
    dnw = dn * w1
    dh = rh * (dnw - hhat * (dnw * hhat).mean(-1, keepdim=True))
    grads = [dx, dh, (dn * hhat).sum(0)]
    if gate is not None:
        dg = alpha * dx * (hhat * w1)
        grads.append({"channel": lambda: dg.sum(0), "row": lambda: dg.sum(1, keepdim=True),
                      "element": lambda: dg}[st["case"]["gate"]]())
    grads.append((dy * shat).sum(0))
    return (out, *(t.to(dt) for t in grads))


# ------------------------------------------------------------------- the library's calls
def _own_attention(st, step):
    from evograd_amd.pairs import packed_attention as pair

    o, saved = pair.packed_attention_forward_with_saved(st["q"], st["k"], st["v"], st["cu"])
    if not step:
        return o
    return (o, *pair.packed_attention_backward_from_saved(st["do"], saved))


def _own_rotary(st, step):
    from evograd_amd.pairs import rotary as pair

    interleaved = st["case"]["layout"] == "interleaved"
    (q, k), saved = pair.rotary_qk_forward_with_saved(st["q"], st["k"], st["positions"],
                                                      st["freqs"], interleaved=interleaved)
    if not step:
        return q, k
    return (q, k, *pair.rotary_qk_backward_from_saved((st["dq"], st["dk"]), saved,
                                                      interleaved=interleaved))


def _own_block_norm(st, step):
    from evograd_amd.pairs import block_norm as pair

    alpha = st["case"]["alpha"]
    out, saved = pair.block_norm_forward_with_saved(st["x"], st["h"], st["w1"], st["gate"],
                                                    st["w2"], scale=alpha, eps=EPS)
    if not step:
        return out
    grads = pair.block_norm_backward_from_saved(st["dout"], saved, scale=alpha)
    return (out, *(g for g in grads if g is not None))


_PLAIN = {"attention": _plain_attention, "rotary": _plain_rotary, "block_norm": _plain_block_norm}
_OWN = {"attention": _own_attention, "rotary": _own_rotary, "block_norm": _own_block_norm}


def run(state):
    case = state["case"]
    with torch.no_grad():
        return (_OWN if own else _PLAIN)[case["kind"]](state, case["passes"] == "step")


# ------------------------------------------------------------------------ in 64 bits
def _exact_attention(case, t):
    q, k, v, do = (t[n].double() for n in ("q", "k", "v", "do"))
    T, H, D = q.shape
    group = H // case["KVH"]
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in _lengths(case):
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        visible = torch.arange(n, device=q.device)
        visible = visible[:, None] >= visible[None, :]
        for h in range(H):
            leaves = [x.clone().requires_grad_(True)
                      for x in (q[rows, h], k[rows, h // group], v[rows, h // group])]
            with torch.enable_grad():
                scores = (leaves[0] / math.sqrt(D)) @ leaves[1].T
                out = torch.softmax(torch.where(visible, scores, -math.inf), -1) @ leaves[2]
            o[rows, h] = out.detach()
            if case["passes"] == "step":
                a, b, c = torch.autograd.grad(out, leaves, do[rows, h])
                dq[rows, h] = a
                dk[rows, h // group] += b
                dv[rows, h // group] += c
    return (o, dq, dk, dv) if case["passes"] == "step" else o


def _exact_rotary(case, t):
    R = case["R"]
    angle = torch.outer(t["positions"].double(), _frequencies(case))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]  # e^(i angle)
    out = []
    for name, z in (("q", turn), ("k", turn), ("dq", turn.conj()), ("dk", turn.conj())):
        x = t[name].double()
        part, rest = x[..., :R], x[..., R:]
        if case["layout"] == "half":
            c = torch.complex(part[..., :R // 2].contiguous(), part[..., R // 2:].contiguous()) * z
            part = torch.cat((c.real, c.imag), -1)
        else:
            c = torch.view_as_complex(part.reshape(*part.shape[:-1], R // 2, 2).contiguous()) * z
            part = torch.view_as_real(c.resolve_conj()).flatten(-2)
        out.append(torch.cat((part, rest), -1))
    return tuple(out if case["passes"] == "step" else out[:2])


def _exact_block_norm(case, t):
    names = ["x", "h", "w1"] + ([] if t["gate"] is None else ["gate"]) + ["w2"]
    leaf = {n: t[n].double().requires_grad_(True) for n in names}
    with torch.enable_grad():
        def norm(a, w):
            return a / torch.sqrt((a * a).mean(-1, keepdim=True) + EPS) * w

        branch = norm(leaf["h"], leaf["w1"])
        if "gate" in leaf:
            branch = leaf["gate"] * branch
        s = leaf["x"] + case["alpha"] * branch
        out = torch.stack((s, norm(s, leaf["w2"])))
    if case["passes"] != "step":
        return out.detach()
    grads = torch.autograd.grad(out, [leaf[n] for n in names], t["dout"].double())
    return (out.detach(), *grads)


def exact(case, seed):
    t = _inputs(case, seed)
    return {"attention": _exact_attention, "rotary": _exact_rotary,
            "block_norm": _exact_block_norm}[case["kind"]](case, t)
