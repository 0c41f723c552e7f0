"""What a policy-gradient step does around its loss, as timed cases: scores of given tokens (log-probs, entropy, the top
alternatives), their gradient, the norm of a model's gradients with clipping, and the clipped Nesterov update of a
model's tensors.

`run` computes each operator in elementary torch operations, or, with `own` set, through the framework's entry points.
Inputs are made on the GPU from the seed alone. `exact` restates each operator in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IDS = {"i32": torch.int32, "i64": torch.int64}
QWEN_VOCAB = 151936      # the vocabulary of configurations 2 to 5
GPT_VOCAB = 50257        # odd: its 16-bit rows start off 16 bytes
PAD = -100               # the id of an alternative of a row that is not scored


def listed() -> list[dict]:
    return [
        # One sequence's decode step: the drawn token's log-prob, the entropy and 20 alternatives, as a server reports them.
        dict(name="score_row", kind="score", dtype="bf16", S=1, T=1, V=QWEN_VOCAB, pad=0, k=20, temperature=1.0,
             shifted=False, banned=0.0, id_type="i32"),
        # One decode step of configuration 2's 64 rollouts, in the sampler's f32, part of the vocabulary forbidden.
        dict(name="score_rollouts", kind="score", dtype="f32", S=64, T=1, V=QWEN_VOCAB, pad=0, k=5, temperature=0.75,
             shifted=False, banned=0.25, id_type="i64"),
        # Whole rollouts scored afterwards: an odd vocabulary in padded rows, logits[:, :-1] against the next tokens.
        dict(name="score_odd", kind="score", dtype="f16", S=16, T=96, V=GPT_VOCAB, pad=47, k=8, temperature=1.0,
             shifted=True, banned=0.0, id_type="i32"),
        # The training step's eight sequences of 512 over the real vocabulary, log-probs and entropy alone: the largest.
        dict(name="score_batch", kind="score", dtype="bf16", S=8, T=512, V=QWEN_VOCAB, pad=0, k=0, temperature=1.0,
             shifted=False, banned=0.0, id_type="i32"),
        # Configuration 1's toy shape: launches and latency are the time.
        dict(name="grad_toy", kind="grad", dtype="f32", out="f32", S=8, T=128, V=1024, pad=0, temperature=1.0,
             shifted=False, banned=0.0, accumulate=False),
        # f32 gradients of bf16 logits over an odd vocabulary, logits[:, :-1] against the next tokens.
        dict(name="grad_odd", kind="grad", dtype="bf16", out="f32", S=16, T=128, V=GPT_VOCAB, pad=0, temperature=0.75,
             shifted=True, banned=0.0, accumulate=False),
        # The entropy bonus of the training step, added to the loss head's dlogits: the largest.
        dict(name="grad_batch", kind="grad", dtype="bf16", out="bf16", S=8, T=512, V=QWEN_VOCAB, pad=0, temperature=1.0,
             shifted=False, banned=0.0, accumulate=True),
        # The toy model's 26 gradient tensors, clipped into the optimizer's flat buffer: launches are the time.
        dict(name="clip_toy", kind="clip", hidden=64, ff=172, kv=64, layers=2, V=1024, grads="f32", norm="l2", clip=True),
        # Tensors of odd sizes in three types, some of them empty, by their largest magnitude.
        dict(name="clip_ragged", kind="clip", hidden=390, ff=1111, kv=77, layers=9, V=GPT_VOCAB, grads="mixed", norm="max",
             clip=True),
        # A 0.5B model's 290 bf16 gradient tensors into the flat f32 buffer: the largest.
        dict(name="clip_model", kind="clip", hidden=896, ff=4864, kv=128, layers=24, V=QWEN_VOCAB, grads="bf16", norm="l2",
             clip=True),
        # The toy model's whole optimizer step: norm, coefficient, update.
        dict(name="update_toy", kind="update", hidden=64, ff=172, kv=64, layers=2, V=1024, grads="f32", norm="l2",
             clip=True, shadow=False, mode="sutskever"),
        # The 0.5B model's: bf16 gradients where the backward pass left them, f32 weights and velocities, the next
        # forward's bf16 weights.
        dict(name="update_model", kind="update", hidden=896, ff=4864, kv=128, layers=24, V=QWEN_VOCAB, grads="bf16",
             norm="l2", clip=True, shadow=True, mode="sutskever"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _vocab(rng) -> int:
    return rng.choice([QWEN_VOCAB, GPT_VOCAB, _log_int(rng, 1000, 262144), 8 * _log_int(rng, 125, 32768)])


def draw(rng) -> dict:
    kind = rng.choice(["score", "score", "grad", "grad", "clip", "update"])
    if kind in ("score", "grad"):
        V = _vocab(rng)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        out = rng.choice([dtype, dtype, "f32"])
        accumulate = rng.random() < 0.4
        # Up to the largest listed rows: 1.2 GB read, or 3.7 GB read and written.
        per = V * (DTYPES[dtype].itemsize if kind == "score" else
                   DTYPES[dtype].itemsize + (2 if accumulate else 1) * DTYPES[out].itemsize)
        most = 4096 * QWEN_VOCAB * (2 if kind == "score" else 6) // per
        tokens = _log_int(rng, 1 if kind == "score" else 4, min(16384, most))
        S = _log_int(rng, 1, min(64, tokens))
        T = max(1, tokens // S)
        case = dict(kind=kind, dtype=dtype, S=S, T=T, V=V, pad=rng.choice([0, 0, rng.randint(1, 127)]),
                    temperature=rng.choice([1.0, 1.0, 0.75, 2.0]), shifted=T > 1 and rng.random() < 0.3,
                    banned=rng.choice([0.0, 0.0, 0.3, 0.9]))
        if kind == "score":
            # The plain form's sort keys take 8 bytes an element.
            k = rng.choice([0, _log_int(rng, 1, 64)]) if S * T * V <= 1 << 28 else 0
            return dict(case, k=k, id_type=rng.choice(["i32", "i64"]))
        return dict(case, out=out, accumulate=accumulate)
    hidden = _log_int(rng, 48, 832)
    case = dict(kind=kind, hidden=hidden, ff=_log_int(rng, 2 * hidden, 5 * hidden + 384), kv=max(8, hidden // 7),
                layers=_log_int(rng, 1, 24), V=_log_int(rng, 1000, QWEN_VOCAB),
                grads=rng.choice(["f32", "bf16", "bf16", "f16", "mixed"]), norm=rng.choice(["l2", "l2", "max"]),
                clip=rng.random() < 0.7)
    if kind == "update":
        case.update(shadow=rng.random() < 0.6, mode=rng.choice(["sutskever", "mlir"]))
    return case


# ---- inputs ---------------------------------------------------------------------------


def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 64 + salt)


def _logits(case: dict, g: torch.Generator) -> torch.Tensor:
    """[S, T, V] as a language model gives them: a normal bulk, a few tokens that stand out, forbidden ones at -inf."""
    S, T, V = case["S"], case["T"], case["V"]
    out = torch.zeros((S, T, V + case["pad"]), dtype=DTYPES[case["dtype"]], device=DEV)[..., :V]
    for s in range(S):
        x = torch.randn((T, V), generator=g, device=DEV).mul_(3.0)
        at = torch.randint(0, V, (T, 24), generator=g, device=DEV)
        x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=DEV) * 14)
        if case["banned"]:
            ban = torch.rand(V, generator=g, device=DEV) < case["banned"]
            ban[torch.randint(0, V, (1,), generator=g, device=DEV)] = False
            x.masked_fill_(ban, -math.inf)
        out[s] = x.to(out.dtype)
    return out


def _tokens(case: dict, x: torch.Tensor, g: torch.Generator) -> dict:
    """Tokens drawn from the rows that score them, and the mask of their sequences' lengths."""
    S, T, V = case["S"], case["T"], case["V"]
    rows, off = _layout(case)
    ids = torch.zeros((S, T), dtype=torch.int64, device=DEV)
    for s in range(S):
        e = torch.empty((rows, V), device=DEV).exponential_(generator=g)
        ids[s, off:] = (x[s, :rows].float() / case["temperature"] - e.log()).argmax(1)
    lengths = torch.randint(max(1, T // 4), T + 1, (S, 1), generator=g, device=DEV)
    return {"ids": ids, "mask": (torch.arange(T, device=DEV) < lengths).float()}


def _sizes(case: dict) -> list[int]:
    """A decoder's tensors: embedding, per layer its projections, biases and norms, the last norm."""
    h, ff, kv = case["hidden"], case["ff"], case["kv"]
    layer = [h * h, h, kv * h, kv, kv * h, kv, h * h, ff * h, ff * h, h * ff, h, h]
    if case["grads"] == "mixed":   # some parameters are frozen: they have no elements here
        layer[1] = layer[5] = 0
    return [case["V"] * h] + layer * case["layers"] + [h]


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed, 1)
    st = dict(case)
    if case["kind"] in ("score", "grad"):
        x = st["logits"] = _logits(case, g)
        st.update(_tokens(case, x, g))
        if case["kind"] == "grad":
            S, T = case["S"], case["T"]
            rows, off = _layout(case)
            # What scoring these rows has given: the maximum, the log of the sum, the entropy.
            stats = torch.zeros((3, S, T), device=DEV)
            for s in range(S):
                stats[:, s, off:] = torch.stack(_row_stats(x[s, :rows], case["temperature"])[:3])
            stats *= st["mask"]
            st["row_max"], st["log_sum"], st["entropy"] = stats
            # Advantages over a sequence's length, and the weight of the entropy; a scaled loss for half precision.
            lengths = st["mask"][:, off:].sum(1, keepdim=True).clamp(min=1)
            w = st["mask"] / (S * lengths) * (1024.0 if case["out"] == "f16" else 1.0)
            st["dlogp"] = -torch.randn((S, 1), generator=g, device=DEV) * w
            st["dentropy"] = -0.05 * w
            wide = torch.zeros((S, T, case["V"]), dtype=DTYPES[case["out"]], device=DEV)
            if case["accumulate"]:
                for s in range(S):
                    wide[s] = (torch.randn(wide.shape[1:], generator=g, device=DEV) * w[s].max() * 1e-3).to(wide.dtype)
            st["dlogits"] = wide
        return st
    sizes = _sizes(case)
    types = [DTYPES[case["grads"] if case["grads"] != "mixed" else ("f32", "bf16", "f16")[i % 3]] for i in range(len(sizes))]
    total = sum(sizes)
    st["grads"] = [(torch.randn(n, generator=g, device=DEV) * (1e-3 * (1 + i % 5))).to(t)
                   for i, (n, t) in enumerate(zip(sizes, types))]
    usual = 1e-3 * math.sqrt(11.0 * total) if case["norm"] == "l2" else 0.02
    st["max_norm"] = usual * (0.25 if case["clip"] else 4.0)
    if case["kind"] == "clip":
        st["flat"] = torch.zeros(total, device=DEV)
        st["out"] = list(st["flat"].split(sizes))
    else:
        st["p"] = torch.randn(total, generator=g, device=DEV) * 0.02
        st["v"] = torch.randn(total, generator=g, device=DEV) * 1e-3
        st["b"] = torch.zeros(total, dtype=torch.bfloat16, device=DEV) if case["shadow"] else None
        st["params"], st["velocities"] = list(st["p"].split(sizes)), list(st["v"].split(sizes))
        st["copies"] = list(st["b"].split(sizes)) if case["shadow"] else None
        st["lr"], st["mu"] = 0.01, 0.9
    return st


# ---- one pass -------------------------------------------------------------------------


def _layout(st: dict) -> tuple[int, int]:
    """(token-carrying rows, token of row 0)."""
    return (st["T"] - 1, 1) if st["shifted"] else (st["T"], 0)


def run(st: dict):
    if own:
        return _run_own(st)
    return {"score": _score, "grad": _grad, "clip": _clip, "update": _update}[st["kind"]](st)


def _run_own(st: dict):
    # A program that makes such calls again and again keeps the buffers of their results.
    from pcp_amd import scores, step
    kept = st.get("kept")
    if st["kind"] == "score":
        rows, off = _layout(st)
        o = scores.token_scores(st["logits"], st["ids"], st["mask"], k=st["k"], temperature=st["temperature"], rows=rows,
                                tok_offset=off, top_ids_dtype=IDS[st["id_type"]],
                                outputs=kept, sync=False)
        out = [o.logp, o.entropy, o.row_max, o.log_sum] + ([o.top_logp, o.top_ids] if st["k"] else [])
    elif st["kind"] == "grad":
        rows, off = _layout(st)
        o = st["dlogits"]
        scores.token_scores_bwd(st["logits"], st["ids"], st["row_max"], st["log_sum"], st["entropy"], dlogp=st["dlogp"],
                                dentropy=st["dentropy"], mask=st["mask"], temperature=st["temperature"], rows=rows,
                                tok_offset=off, dlogits=o, accumulate=st["accumulate"], sync=False)
        return o
    elif st["kind"] == "clip":
        o = step.clip_grads(st["grads"], st["max_norm"], norm_type=st["norm"], out=st["out"], outputs=kept, sync=False)
        out = o.norm, o.coef, st["flat"]
    else:
        o = step.grad_norm(st["grads"], st["max_norm"], norm_type=st["norm"], outputs=kept, sync=False)
        step.nesterov_update_many(st["params"], st["velocities"], st["grads"], st["copies"], coef=o.coef,
                                  learning_rate=st["lr"], momentum=st["mu"], mode=st["mode"], sync=False)
        out = [o.norm, st["p"], st["v"]] + ([st["b"]] if st["shadow"] else [])
    st["kept"] = o
    return out


def _row_stats(x, temperature):
    """Of rows [..., V]: the largest logit, the log of the sum of exp((x - max) / temperature), the entropy, and those
    differences."""
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = (x - m).div_(temperature)
    e = d.exp()
    total = e.sum(-1, dtype=torch.float64)
    log_sum = total.log()
    # (exp(-inf) times -inf counts as 0.)
    entropy = log_sum - e.mul_(d).nan_to_num_(nan=0.0).sum(-1, dtype=torch.float64) / total
    return m[..., 0], log_sum.float(), entropy.float(), d


def _score(st: dict):
    S, T, V, k = st["S"], st["T"], st["V"], st["k"]
    rows, off = _layout(st)
    x = st["logits"][:, :rows]
    live = st["mask"][:, off:] != 0
    m, log_sum, entropy, d = _row_stats(x, st["temperature"])
    logp = d.gather(2, st["ids"][:, off:, None])[..., 0].double() - log_sum.double()

    def token(v):
        o = torch.zeros((S, T), device=v.device)
        o[:, off:] = torch.where(live, v, 0.0).float()
        return o

    out = [token(logp), token(entropy), token(m), token(log_sum)]
    if k:
        # Keys that order as (logit, then the lower id first), so that equal logits leave no choice.
        b = (x.float() + 0.0).view(torch.int32).to(torch.int64)
        b = torch.where(b < 0, -(b & 0x7fffffff), b)
        key = (b << 32) + (V - 1 - torch.arange(V, device=x.device))
        at = V - 1 - (torch.topk(key, k, dim=2).values & 0xffffffff)
        lp = (d.gather(2, at).double() - log_sum.double()[..., None]).float()
        top_logp = torch.zeros((S, T, k), device=x.device)
        top_ids = torch.full((S, T, k), PAD, dtype=IDS[st["id_type"]], device=x.device)
        top_logp[:, off:] = torch.where(live[..., None], lp, 0.0)
        top_ids[:, off:] = torch.where(live[..., None], at, PAD).to(top_ids.dtype)
        if off:
            top_ids[:, :off] = 0   # tokens that no row scores stay as they were: zero
        out += [top_logp, top_ids]
    return out


def _grad(st: dict):
    rows, off = _layout(st)
    tau = st["temperature"]
    ids, live = st["ids"][:, off:, None], (st["mask"][:, off:] != 0)[..., None]
    gl, gh = (torch.where(live, st[n][:, off:, None], 0.0) for n in ("dlogp", "dentropy"))
    log_p = (st["logits"][:, :rows].float() - st["row_max"][:, off:, None]).div_(tau).sub_(st["log_sum"][:, off:, None])
    p = log_p.exp()
    # d/dz: dlogp (1[token] - p) - dentropy p (log p + entropy), over the temperature.
    dz = log_p.add_(st["entropy"][:, off:, None]).mul_(gh).add_(gl).mul_(p).nan_to_num_(nan=0.0).neg_()
    dz.scatter_add_(2, ids, gl.expand_as(ids).contiguous())
    dz = dz.div_(tau).masked_fill_(~live, 0.0)
    if st["accumulate"]:
        dz += st["dlogits"][:, :rows].float()
        st["dlogits"][:, :rows] = dz.to(st["dlogits"].dtype)
    else:
        st["dlogits"][:, :rows] = dz.to(st["dlogits"].dtype)
        st["dlogits"][:, rows:] = 0
    return st["dlogits"]


def _norm(st: dict):
    """The gradients in one f32 tensor, their norm and the coefficient that brings it down to max_norm."""
    flat = torch.cat([g.float() for g in st["grads"]])
    norm = flat.double().square_().sum().sqrt() if st["norm"] == "l2" else flat.abs().max().double()
    coef = torch.where(norm > st["max_norm"], st["max_norm"] / norm, 1.0)
    return flat, norm.float(), coef.float()


def _clip(st: dict):
    flat, norm, coef = _norm(st)
    torch.mul(flat, coef, out=st["flat"])
    return norm, coef, st["flat"]


def _update(st: dict):
    g, norm, coef = _norm(st)
    p, v, lr, mu = st["p"], st["v"], st["lr"], st["mu"]
    g.mul_(coef)
    if st["mode"] == "sutskever":
        v.mul_(mu).add_(g)
        p.sub_(g.add_(v * mu).mul_(lr))
    else:
        v.mul_(mu).add_(g.mul_(lr))
        p.sub_(v)
    if not st["shadow"]:
        return [norm, p, v]
    st["b"].copy_(p)
    return [norm, p, v, st["b"]]


# ---- what a pass cannot do without ----------------------------------------------------


def work(case: dict) -> dict:
    if case["kind"] in ("score", "grad"):
        V, size = case["V"], DTYPES[case["dtype"]].itemsize
        rows, _ = _layout(case)
        N = case["S"] * case["T"]
        # Sequences are live over 5/8 of their length on average (the whole of it where that is one token).
        live = case["S"] * rows * (0.625 if case["T"] > 1 else 1.0)
        if case["kind"] == "score":
            entry = 4 + IDS[case["id_type"]].itemsize
            return {"bytes": int(live * (V * size + 28 + case["k"] * entry)), "flops": int(live * 6 * V)}
        o = DTYPES[case["out"]].itemsize
        wide = live * V * (size + 2 * o) if case["accumulate"] else live * V * size + N * V * o
        return {"bytes": int(wide + live * 32), "flops": int(live * 8 * V)}
    sizes = _sizes(case)
    total = sum(sizes)
    each = {"f32": 4, "bf16": 2, "f16": 2}
    read = (total * each[case["grads"]] if case["grads"] != "mixed" else
            sum(n * (4 if i % 3 == 0 else 2) for i, n in enumerate(sizes)))
    if case["kind"] == "clip":
        return {"bytes": read + 4 * total, "flops": 3 * total}
    return {"bytes": read + total * (16 + (2 if case["shadow"] else 0)), "flops": 8 * total}


# ---- the operators' definitions in 64 bits --------------------------------------------


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"score": _exact_score, "grad": _exact_grad, "clip": _exact_clip, "update": _exact_update}[case["kind"]](st)


def _exact_score(st: dict):
    S, T, V, k, tau = st["S"], st["T"], st["V"], st["k"], st["temperature"]
    rows, off = _layout(st)
    out = [torch.zeros((S, T), dtype=torch.float64, device=DEV) for _ in range(4)]
    if k:
        top_logp = torch.zeros((S, T, k), dtype=torch.float64, device=DEV)
        top_ids = torch.zeros((S, T, k), dtype=IDS[st["id_type"]], device=DEV)
    step = max(1, (1 << 25) // V)
    for s in range(S):
        for t0 in range(0, rows, step):
            x = st["logits"][s, t0:min(t0 + step, rows)].double()
            to = slice(off + t0, off + t0 + len(x))
            on = st["mask"][s, to] != 0
            log_p = torch.log_softmax(x / tau, 1)
            plogp = torch.special.entr(log_p.exp())
            values = (log_p.gather(1, st["ids"][s, to, None])[:, 0], plogp.sum(1), x.amax(1),
                      torch.logsumexp(x / tau, 1) - x.amax(1) / tau)
            for o, v in zip(out, values):
                o[s, to] = torch.where(on, v, 0.0)
            if k:
                v, i = torch.sort(x, dim=1, descending=True, stable=True)
                top_logp[s, to] = torch.where(on[:, None], log_p.gather(1, i[:, :k]), 0.0)
                top_ids[s, to] = torch.where(on[:, None], i[:, :k], PAD).to(top_ids.dtype)
    return out + ([top_logp, top_ids] if k else [])


def _exact_grad(st: dict):
    """By differentiating the definitions."""
    S, T, V, tau = st["S"], st["T"], st["V"], st["temperature"]
    rows, off = _layout(st)
    if S * T * V > 1 << 30:
        return None
    out = st["dlogits"].double() if st["accumulate"] else torch.zeros((S, T, V), dtype=torch.float64, device=DEV)
    step = max(1, (1 << 24) // V)
    for s in range(S):
        for t0 in range(0, rows, step):
            n = min(step, rows - t0)
            to = slice(off + t0, off + t0 + n)
            x = st["logits"][s, t0:t0 + n].double().requires_grad_()
            log_p = torch.log_softmax(x / tau, 1)
            p = log_p.exp()
            entropy = -(p * log_p.masked_fill(p == 0, 0.0)).sum(1)
            logp = log_p.gather(1, st["ids"][s, to, None])[:, 0]
            on = st["mask"][s, to].double()
            value = (on * (st["dlogp"][s, to].double() * logp + st["dentropy"][s, to].double() * entropy)).sum()
            d, = torch.autograd.grad(value, x)
            out[s, t0:t0 + n] += d
    return out


def _exact_norm(st: dict):
    parts = [g.double() for g in st["grads"]]
    if st["norm"] == "l2":
        norm = math.sqrt(math.fsum(float((g * g).sum()) for g in parts))
    else:
        norm = max(float(g.abs().max()) for g in parts if g.numel())
    return torch.cat(parts), norm, min(1.0, st["max_norm"] / norm)


def _exact_clip(st: dict):
    flat, norm, coef = _exact_norm(st)
    return torch.tensor(norm, dtype=torch.float64), torch.tensor(coef, dtype=torch.float64), flat * coef


def _exact_update(st: dict):
    g, norm, coef = _exact_norm(st)
    g = g * coef
    p, v = st["p"].double(), st["v"].double()
    if st["mode"] == "sutskever":
        v = st["mu"] * v + g
        p = p - st["lr"] * (g + st["mu"] * v)
    else:
        v = st["mu"] * v + st["lr"] * g
        p = p - v
    return [torch.tensor(norm, dtype=torch.float64), p, v] + ([p] if st["shadow"] else [])
