"""Performance cases of the operators at the two ends and in the middle of a distillation step
over a packed batch: the embedding lookup and its gradient, the norms of queries and keys per
head with the rotation behind them, and the loss against a teacher's top logits.

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
THETA = 500000.0
IGNORE = -100


# ------------------------------------------------------------------------------ cases
def _embed(T, V, H, tokens, scale, dtype, passes="step", **more):
    """T tokens of a table [V, H]. ``tokens``: "flat" (uniform), "skewed" (frequencies that fall
    as one over the rank, as a text's do) or "padded" (skewed, a third of them one token and
    a tenth ignored)."""
    return dict(kind="embedding", T=T, V=V, H=H, tokens=tokens, scale=scale, dtype=dtype,
                passes=passes, **more)


def _norm_rotary(T, H, KVH, D, R, layout, far, dtype, passes="step", **more):
    """q and k of T tokens, R of the D columns of a head rotated, positions up to ``far``."""
    return dict(kind="norm_rotary", T=T, H=H, KVH=KVH, D=D, R=R, layout=layout, far=far,
                dtype=dtype, passes=passes, **more)


def _distill(rows, V, K, tau, soft, hard, cut, dtype, passes="step", **more):
    """K teacher logits a row; ``cut``: only a nucleus of them is kept, none in some rows."""
    return dict(kind="distillation", rows=rows, V=V, K=K, tau=tau, soft=soft, hard=hard, cut=cut,
                dtype=dtype, passes=passes, **more)


def listed():
    return [
        # A generation step: one token of each of 32 requests, a Llama-3-8B table.
        _embed(32, 128256, 4096, "flat", 1.0, "bfloat16", passes="forward",
               name="embedding_32tok_128256x4096_bf16"),
        # A small fp32 model's step, rows scaled by the root of their width.
        _embed(700, 5003, 768, "skewed", 768 ** 0.5, "float32",
               name="embedding_700tok_5003x768_fp32"),
        # Odd widths and a batch with padding: one token a third of the time, some ignored.
        _embed(8191, 50257, 1538, "padded", 1.0, "float16",
               name="embedding_8191tok_50257x1538_fp16"),
        # The large packed batch of a Llama-3-8B table.
        _embed(16384, 128256, 4096, "skewed", 1.0, "bfloat16",
               name="embedding_16384tok_128256x4096_bf16"),
        # A generation step: one token of each of 32 requests, far into the context.
        _norm_rotary(32, 32, 8, 128, 128, "half", 131072, "bfloat16", passes="forward",
                     name="norm_rotary_32tok_bf16"),
        # fp32 training of a small grouped-query model.
        _norm_rotary(1500, 8, 2, 64, 64, "half", 4096, "float32",
                     name="norm_rotary_1500tok_fp32"),
        # Interleaved pairs over part of the head, an odd token count.
        _norm_rotary(5003, 16, 16, 96, 64, "interleaved", 32768, "float16",
                     name="norm_rotary_5003tok_partial_fp16"),
        # A long packed batch of Llama-3-8B heads.
        _norm_rotary(32768, 32, 8, 128, 128, "half", 16384, "bfloat16",
                     name="norm_rotary_32768tok_bf16"),
        # A few rows of a wide vocabulary: a short answer's step.
        _distill(16, 128256, 32, 1.0, 1.0, 0.0, False, "bfloat16",
                 name="distillation_16x128256_k32_bf16"),
        # A small fp32 student, soft and hard labels at temperature 2.
        _distill(1000, 32000, 64, 2.0, 0.5, 0.5, False, "float32",
                 name="distillation_1000x32000_k64_fp32"),
        # An odd vocabulary, nucleus-cut teacher entries of an odd count.
        _distill(2047, 50257, 21, 1.5, 1.0, 0.0, True, "float16",
                 name="distillation_2047x50257_k21_fp16"),
        # The large batch over a Llama-3-8B vocabulary.
        _distill(8192, 128256, 64, 2.0, 0.7, 0.3, False, "bfloat16",
                 name="distillation_8192x128256_k64_bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case of the listed ranges: sizes log-uniform, odd ones among them."""
    kind = rng.choice(["embedding", "norm_rotary", "distillation"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    passes = rng.choice(["step", "step", "step", "forward"])
    if kind == "embedding":
        H = _log(rng, 64, 4096)
        H = H if rng.random() < 0.25 else H // 64 * 64
        V = _log(rng, 256, 131072 if dtype != "float32" else 65536)
        return _embed(_log(rng, 1, 16384), V, H, rng.choice(["flat", "skewed", "padded"]),
                      rng.choice([1.0, H ** 0.5]), dtype, passes)
    if kind == "norm_rotary":
        kvh = rng.choice([1, 2, 4, 8])
        H = min(32, kvh * rng.choice([1, 2, 4, 8]))
        D = rng.choice([64, 80, 96, 128, 128, 256])
        R = rng.choice([D, D, D // 2, D // 4])
        return _norm_rotary(_log(rng, 1, 16384 if D <= 128 else 8192), H, kvh, D, R,
                            rng.choice(["half", "interleaved"]), _log(rng, 4096, 1 << 20), dtype,
                            passes)
    V = _log(rng, 1000, 131072)
    rows = _log(rng, 1, min(8192, (1 << 30) // V if dtype != "float32" else (1 << 29) // V))
    return _distill(rows, V, _log(rng, 1, 256), rng.choice([1.0, 1.5, 2.0, 4.0]),
                    rng.choice([1.0, 0.5]), rng.choice([0.0, 0.5]), rng.choice([False, True]),
                    dtype, passes)


def _ids(case, seed):
    """The tokens of an embedding case, on the CPU."""
    T, V, how = case["T"], case["V"], case["tokens"]
    gen = torch.Generator().manual_seed(random.Random(f"{T} {V} {how} {seed}").getrandbits(48))
    u = torch.rand(T, generator=gen, dtype=torch.float64)
    if how == "flat":
        return (u * V).long().clamp_(max=V - 1)
    rank = torch.exp(u * math.log(V)).long().clamp_(max=V) - 1  # P(rank) ~ 1 / (rank + 1)
    ids = rank * 7919 % V  # frequent tokens all over the table
    if how == "padded":
        v = torch.rand(T, generator=gen, dtype=torch.float64)
        ids[v < 1 / 3] = V // 2
        ids[v > 0.9] = IGNORE
    return ids


def work(case):
    e, step = SIZE[case["dtype"]], case["passes"] == "step"
    if case["kind"] == "embedding":
        T, V, H = case["T"], case["V"], case["H"]
        ids = _ids(case, 0)
        rows, used = int((ids >= 0).sum()), int(torch.unique(ids[ids >= 0]).numel())
        moved = used * H + T * H + (rows * H + V * H if step else 0)
        return {"bytes": e * moved + 4 * T, "flops": T * H + (2 * rows * H if step else 0)}
    if case["kind"] == "norm_rotary":
        n = case["T"] * (case["H"] + case["KVH"]) * case["D"]
        return {"bytes": e * n * (4 if step else 2), "flops": n * (25 if step else 8)}
    n, nk = case["rows"] * case["V"], case["rows"] * case["K"]
    both = case["soft"] != 0.0 and case["hard"] != 0.0 and case["tau"] != 1.0
    return {"bytes": e * n * (2 if step else 1) + 8 * nk,
            "flops": n * ((6 if both else 4) + ((6 if both else 4) if step else 0))}


# ----------------------------------------------------------------------------- inputs
def _generator(case, seed):
    text = repr(sorted((k, v) for k, v in case.items() if k != "name")) + f"|{seed}"
    return torch.Generator(device=DEVICE).manual_seed(random.Random(text).getrandbits(48))


def _inputs(case, seed):
    """The tensors a pass is given, from the case and the seed alone."""
    gen, dt = _generator(case, seed), DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dt)

    if case["kind"] == "embedding":
        return dict(weight=normal(case["V"], case["H"]), dout=normal(case["T"], case["H"]),
                    ids=_ids(case, seed).to(DEVICE, torch.int32))
    if case["kind"] == "norm_rotary":
        T, H, KVH, D = case["T"], case["H"], case["KVH"], case["D"]
        positions = torch.randint(0, case["far"], (T,), generator=gen, device=DEVICE)
        if case["passes"] == "step":  # a packed batch: runs of consecutive positions
            positions = (positions[0] + torch.arange(T, device=DEVICE)) % case["far"]
        # q and k as one projection gives them: column ranges of the same rows, v behind them
        qkv = normal(T, (H + 2 * KVH) * D)
        return dict(q=qkv[:, :H * D].view(T, H, D),
                    k=qkv[:, H * D:(H + KVH) * D].view(T, KVH, D),
                    qw=(1.0 + 0.1 * normal(D).float()).to(dt),
                    kw=(1.0 + 0.1 * normal(D).float()).to(dt),
                    dq=normal(T, H, D), dk=normal(T, KVH, D),
                    positions=positions.to(torch.int32))
    rows, V, K = case["rows"], case["V"], case["K"]
    logits = normal(rows, V).mul_(2.0)
    # K different columns a row, in no order; the teacher's values fall from about 12
    ids = torch.randint(0, V - K + 1, (rows, K), generator=gen, device=DEVICE).sort(1).values
    ids += torch.arange(K, device=DEVICE)
    order = torch.rand(rows, K, generator=gen, device=DEVICE).argsort(1)
    ids = ids.gather(1, order)
    teacher = (torch.randn(rows, K, generator=gen, device=DEVICE) * 2.0 + 8.0)
    teacher = teacher.sort(1, descending=True).values
    near = 0.8 * teacher + torch.randn(rows, K, generator=gen, device=DEVICE)
    logits.scatter_(1, ids, near.to(dt))  # the student has learnt some of it
    if case["cut"]:
        kept = torch.randint(0, K + 1, (rows, 1), generator=gen, device=DEVICE)
        ids = torch.where(torch.arange(K, device=DEVICE) < kept, ids, -1)
    target = torch.randint(0, V, (rows,), generator=gen, device=DEVICE)
    prompt = torch.rand(rows, generator=gen, device=DEVICE) < 0.1  # rows of prompts: ignored
    prompt[0] = False
    # fp16 training scales its loss, so that gradients stay above the type's smallest numbers
    scale = 65536.0 if case["dtype"] == "float16" else 1.0
    return dict(logits=logits, target=torch.where(prompt, IGNORE, target),
                teacher=teacher.to(dt), ids=ids.to(torch.int32),
                dloss=torch.full((), scale, device=DEVICE))


def _frequencies(case):
    """Radians per position of each pair, fp64."""
    i = torch.arange(0, case["R"], 2, dtype=torch.float64, device=DEVICE)
    return THETA ** (-i / case["R"])


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["kind"] == "norm_rotary":
        state["freqs"] = _frequencies(case)
    return state


# ------------------------------------------------------------------------- plain forms
def _plain_embedding(st, step):
    weight, ids, scale = st["weight"], st["ids"].long(), st["case"]["scale"]
    kept = (ids != IGNORE)[:, None]
    at = ids.clamp(min=0)
    out = torch.where(kept, weight[at].float() * scale, 0.0).to(weight.dtype)
    if not step:
        return out
    grad = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device)
    grad.index_add_(0, at, torch.where(kept, st["dout"].float(), 0.0))
    return out, (grad * scale).to(weight.dtype)


def _turn(x, cos, sin, layout, R):
    out = x.clone()
    if layout == "half":
        a, b = slice(0, R // 2), slice(R // 2, R)
    else:
        a, b = slice(0, R, 2), slice(1, R, 2)
    out[..., a] = x[..., a] * cos - x[..., b] * sin
    out[..., b] = x[..., b] * cos + x[..., a] * sin
    return out


def _plain_norm_rotary(st, step):
    case, dt = st["case"], st["q"].dtype
    angle = st["positions"].double()[:, None, None] * st["freqs"]
    cos, sin = angle.cos().float(), angle.sin().float()
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((st["q"], st["qw"], st["dq"]), (st["k"], st["kw"], st["dk"])):
        x, w = x.float(), w.float()
        rstd = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        xhat = x * rstd
        outs.append(_turn(xhat * w, cos, sin, case["layout"], case["R"]).to(dt))
        if step:
            dn = _turn(dy.float(), cos, -sin, case["layout"], case["R"])
            wgrads.append((dn * xhat).sum((0, 1)).to(dt))
            dn *= w
            grads.append((rstd * (dn - xhat * (dn * xhat).mean(-1, keepdim=True))).to(dt))
    return (*outs, *grads, *wgrads)


def _plain_distillation(st, step):
    case = st["case"]
    tau, soft, hard = case["tau"], case["soft"], case["hard"]
    logits, target, dt = st["logits"], st["target"], st["logits"].dtype
    counted = target != IGNORE
    n = counted.sum().float()
    z = logits.float()
    top = z.amax(1, keepdim=True)
    # the teacher's distribution over its kept entries
    ids = st["ids"].long()
    kept = ids >= 0
    at = ids.clamp(min=0)
    t = torch.where(kept, st["teacher"].float() / tau, -math.inf)
    tmax = t.amax(1, keepdim=True)
    tmax = torch.where(tmax == -math.inf, 0.0, tmax)
    e = (t - tmax).exp()
    total = e.sum(1, keepdim=True)
    some = total > 0
    total = torch.where(some, total, 1.0)
    p = e / total
    q = ((z - top) / tau).exp()
    qsum = q.sum(1, keepdim=True)
    logq = (z.gather(1, at) - top) / tau - qsum.log()
    logp = t - tmax - total.log()
    loss = soft * tau * tau * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    if hard:
        h = (z - top).exp()
        hsum = h.sum(1, keepdim=True)
        label = target.clamp(min=0)[:, None]
        loss = loss + hard * (hsum.log() + top - z.gather(1, label))[:, 0]
    loss = torch.where(counted, loss, 0.0).sum() / n
    if not step:
        return loss
    del z
    g = torch.where(counted, st["dloss"] / n, 0.0)[:, None]
    q *= g * soft * tau * some / qsum
    q.scatter_add_(1, at, torch.where(kept, -g * soft * tau * p, 0.0))
    if hard:
        h *= g * hard / hsum
        q += h
        q.scatter_add_(1, label, -g * hard)
    return loss, q.to(dt)


# ------------------------------------------------------------------- the library's calls
def _own_embedding(st, step):
    from evograd_amd.pairs import embedding as pair

    scale = st["case"]["scale"]
    out, saved = pair.embedding_forward_with_saved(st["weight"], st["ids"], scale=scale,
                                                   ignore_index=IGNORE)
    if not step:
        return out
    return out, pair.embedding_backward_from_saved(st["dout"], saved, scale=scale,
                                                   ignore_index=IGNORE)


def _own_norm_rotary(st, step):
    from evograd_amd.pairs import norm_rotary as pair

    interleaved = st["case"]["layout"] == "interleaved"
    (q, k), saved = pair.norm_rotary_qk_forward_with_saved(
        st["q"], st["k"], st["qw"], st["kw"], st["positions"], st["freqs"], eps=EPS,
        interleaved=interleaved)
    if not step:
        return q, k
    return (q, k, *pair.norm_rotary_qk_backward_from_saved((st["dq"], st["dk"]), saved, eps=EPS,
                                                           interleaved=interleaved))


def _own_distillation(st, step):
    from evograd_amd.pairs import topk_distillation as pair

    case = st["case"]
    how = dict(temperature=case["tau"], soft_weight=case["soft"], hard_weight=case["hard"],
               ignore_index=IGNORE)
    loss, saved = pair.topk_distillation_forward_with_saved(st["logits"], st["target"],
                                                            st["teacher"], st["ids"], **how)
    if not step:
        return loss
    return loss, pair.topk_distillation_backward_from_saved(st["dloss"], saved, **how)


_PLAIN = {"embedding": _plain_embedding, "norm_rotary": _plain_norm_rotary,
          "distillation": _plain_distillation}
_OWN = {"embedding": _own_embedding, "norm_rotary": _own_norm_rotary,
        "distillation": _own_distillation}


def run(state):
    case = state["case"]
    with torch.no_grad():
        return (_OWN if own else _PLAIN)[case["kind"]](state, case["passes"] == "step")


# ------------------------------------------------------------------------ in 64 bits
def _exact_embedding(case, t):
    w = t["weight"].double().requires_grad_(True)
    live = torch.nonzero(t["ids"] != IGNORE)[:, 0]
    with torch.enable_grad():
        rows = case["scale"] * w[t["ids"][live].long()]
    out = torch.zeros(case["T"], case["H"], dtype=torch.float64, device=w.device)
    out[live] = rows.detach()
    if case["passes"] != "step":
        return out
    grad, = torch.autograd.grad(rows, w, t["dout"][live].double())
    return out, grad


def _exact_norm_rotary(case, t):
    R = case["R"]
    angle = torch.outer(t["positions"].double(), _frequencies(case))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]  # e^(i angle)
    outs, grads, wgrads = [], [], []
    for x, w, dy in (("q", "qw", "dq"), ("k", "kw", "dk")):
        leaves = [t[x].double().requires_grad_(True), t[w].double().requires_grad_(True)]
        with torch.enable_grad():
            n = leaves[0] / torch.sqrt((leaves[0] ** 2).mean(-1, keepdim=True) + EPS) * leaves[1]
            part, rest = n[..., :R], n[..., R:]
            if case["layout"] == "half":
                c = torch.complex(part[..., :R // 2], part[..., R // 2:]) * turn
                part = torch.cat((c.real, c.imag), -1)
            else:
                c = torch.complex(part[..., 0::2], part[..., 1::2]) * turn
                part = torch.stack((c.real, c.imag), -1).flatten(-2)
            y = torch.cat((part, rest), -1)
        outs.append(y.detach())
        if case["passes"] == "step":
            a, b = torch.autograd.grad(y, leaves, t[dy].double())
            grads.append(a)
            wgrads.append(b)
    return (*outs, *grads, *wgrads)


def _exact_distillation(case, t):
    tau, rows, V = case["tau"], case["rows"], case["V"]
    n = int((t["target"] != IGNORE).sum())
    step = case["passes"] == "step"
    loss = torch.zeros((), dtype=torch.float64, device=DEVICE)
    grad = torch.zeros(rows, V, dtype=torch.float64, device=DEVICE) if step else None
    at_once = max(1, (1 << 27) // V)
    for a in range(0, rows, at_once):
        r = slice(a, min(rows, a + at_once))
        z = t["logits"][r].double().requires_grad_(step)
        live, ids = t["target"][r] != IGNORE, t["ids"][r].long()
        some = (ids >= 0).any(1)
        teacher = t["teacher"][r].double() / tau
        # rows without entries get any distribution, their part is left out below
        teacher = torch.where((ids >= 0) | ~some[:, None], teacher, -math.inf)
        logp = torch.log_softmax(teacher, 1)
        with torch.set_grad_enabled(step):
            logq = torch.log_softmax(z / tau, 1).gather(1, ids.clamp(min=0))
            terms = logp.exp() * (torch.where(logp > -math.inf, logp, 0.0) - logq)
            part = case["soft"] * tau ** 2 * terms.sum(1) * some
            if case["hard"]:
                part = part + case["hard"] * torch.nn.functional.cross_entropy(
                    z, t["target"][r], reduction="none", ignore_index=IGNORE)
            part = (part * live).sum() / n
        loss += part.detach()
        if step:
            grad[r], = torch.autograd.grad(part, z, t["dloss"].double())
    return (loss, grad) if step else loss


def exact(case, seed):
    t = _inputs(case, seed)
    return {"embedding": _exact_embedding, "norm_rotary": _exact_norm_rotary,
            "distillation": _exact_distillation}[case["kind"]](case, t)
