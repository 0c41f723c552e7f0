"""Distillation from a teacher's top logits and verification of drafted tokens, as timed cases: the top logits of
rows (what a teacher hands on), the loss on them with its gradient, and the check of a draft model's tokens against
the target's probabilities.

`run` computes each operator in elementary torch operations, or, with `own` set, through the framework's entry points.
Inputs are made on the GPU from the seed alone. `exact` restates each operator in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
IDS = {"i32": torch.int32, "i64": torch.int64}
QWEN_VOCAB = 151936      # the vocabulary of configurations 2 to 5
GPT_VOCAB = 50257        # odd: its 16-bit rows start off 16 bytes
PAD = -100               # the id of an unused teacher entry and of a token past the verified ones
TAIL_FLOOR = 2.0 ** -24  # the least probability of the tokens outside a teacher's entries


def listed() -> list[dict]:
    return [
        # One row of a decode step: the target's top logits for the draft model that learns beside it.
        dict(name="top_row", kind="top", dtype="bf16", R=1, V=QWEN_VOCAB, k=64, temperature=1.0, ids="i32"),
        # An odd vocabulary in f32, rows off 16 bytes, a short list at a raised temperature.
        dict(name="top_odd", kind="top", dtype="f32", R=777, V=GPT_VOCAB, k=20, temperature=2.0, ids="i64"),
        # Long lists of half-precision rows, fewer rows than would fill the GPU row by row.
        dict(name="top_long", kind="top", dtype="f16", R=192, V=QWEN_VOCAB, k=256, temperature=1.0, ids="i32"),
        # A teacher's pass over eight sequences of 512: the largest.
        dict(name="top_batch", kind="top", dtype="bf16", R=4096, V=QWEN_VOCAB, k=64, temperature=1.0, ids="i32"),
        # Configuration 1's toy shape: launches and latency are the time; the teacher's entries renormalised.
        dict(name="distill_toy", kind="distill", dtype="f32", out="f32", S=8, T=128, V=1024, k=8, divergence="forward",
             tail=False, temperature=1.0, shifted=False, cut=False, ids="i64"),
        # A micro-batch: four short answers over the real vocabulary.
        dict(name="distill_micro", kind="distill", dtype="bf16", out="bf16", S=4, T=16, V=QWEN_VOCAB, k=64,
             divergence="forward", tail=True, temperature=1.0, shifted=False, cut=False, ids="i32"),
        # Reverse divergence on an odd vocabulary, logits[:, :-1] against the next tokens' mask, lists of all lengths.
        dict(name="distill_reverse", kind="distill", dtype="bf16", out="bf16", S=16, T=256, V=GPT_VOCAB, k=32,
             divergence="reverse", tail=True, temperature=2.0, shifted=True, cut=True, ids="i32"),
        # The ordinary training step: eight sequences of 512 over the real vocabulary, the largest.
        dict(name="distill_batch", kind="distill", dtype="bf16", out="bf16", S=8, T=512, V=QWEN_VOCAB, k=64,
             divergence="forward", tail=True, temperature=1.0, shifted=False, cut=False, ids="i32"),
        # One sequence with four drafted tokens: what a single rollout's decode step waits for.
        dict(name="verify_one", kind="verify", dtype="bf16", S=1, n=4, V=QWEN_VOCAB, temperature=1.0, draft="model",
             ragged=False),
        # Drafts looked up rather than sampled (no draft distribution), odd f32 rows, drafts of all lengths.
        dict(name="verify_lookup", kind="verify", dtype="f32", S=48, n=6, V=GPT_VOCAB, temperature=0.75, draft="lookup",
             ragged=True),
        # Greedy decoding of 16 rollouts: drafted tokens against the target's largest logits.
        dict(name="verify_greedy", kind="verify", dtype="f32", S=16, n=5, V=QWEN_VOCAB, temperature=0.0, draft="lookup",
             ragged=False),
        # Configuration 2's 64 rollouts with eight tokens each from a draft model: the largest.
        dict(name="verify_batch", kind="verify", dtype="bf16", S=64, n=8, V=QWEN_VOCAB, temperature=1.0, draft="model",
             ragged=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _vocab(rng) -> int:
    return rng.choice([QWEN_VOCAB, GPT_VOCAB, _log_int(rng, 1000, 262144), 8 * _log_int(rng, 125, 32768)])


def draw(rng) -> dict:
    kind = rng.choice(["top", "distill", "distill", "verify"])
    V = _vocab(rng)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    size = DTYPES[dtype].itemsize
    if kind == "top":
        # Up to the largest listed rows (1.2 GB).
        R = _log_int(rng, 1, min(8192, 4096 * QWEN_VOCAB * 2 // (V * size)))
        return dict(kind=kind, dtype=dtype, R=R, V=V, k=_log_int(rng, 1, 256), temperature=rng.choice([1.0, 0.75, 2.0]),
                    ids=rng.choice(["i32", "i64"]))
    if kind == "distill":
        out = rng.choice([dtype, dtype, "f32"])
        # Up to the largest listed rows, read and written (2.5 GB).
        tokens = _log_int(rng, 4, min(16384, 4096 * QWEN_VOCAB * 4 // (V * (size + DTYPES[out].itemsize))))
        S = _log_int(rng, 1, max(1, min(32, tokens // 2)))
        divergence = rng.choice(["forward", "forward", "reverse"])
        return dict(kind=kind, dtype=dtype, out=out, S=S, T=max(2, tokens // S), V=V, k=_log_int(rng, 1, 256),
                    divergence=divergence, tail=divergence == "reverse" or rng.random() < 0.6,
                    temperature=rng.choice([1.0, 1.0, 2.0]), shifted=rng.random() < 0.3, cut=rng.random() < 0.3,
                    ids=rng.choice(["i32", "i64"]))
    n = rng.randint(1, 12)
    # Up to the largest listed rows (0.33 GB).
    S = _log_int(rng, 1, max(1, min(256, 64 * 17 * QWEN_VOCAB * 2 // ((2 * n + 1) * V * size))))
    temperature = rng.choice([0.0, 0.75, 1.0, 1.0])
    return dict(kind=kind, dtype=dtype, S=S, n=n, V=V, temperature=temperature,
                draft="lookup" if temperature == 0.0 else rng.choice(["model", "model", "lookup"]),
                ragged=rng.random() < 0.4)


# ---- inputs ---------------------------------------------------------------------------


def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed * 64 + salt)


def _logits(shape, dtype: str, g: torch.Generator, scale: float = 3.0) -> torch.Tensor:
    """Rows as a language model gives them: a normal bulk and a few tokens that stand out."""
    *lead, V = shape
    rows = math.prod(lead)
    out = torch.empty((rows, V), dtype=DTYPES[dtype], device=DEV)
    step = max(1, (1 << 27) // V)
    for r0 in range(0, rows, step):
        x = torch.randn((min(step, rows - r0), V), generator=g, device=DEV).mul_(scale)
        at = torch.randint(0, V, (x.shape[0], 24), generator=g, device=DEV)
        x.scatter_add_(1, at, torch.rand(at.shape, generator=g, device=DEV) * 14)
        out[r0:r0 + step] = x.to(out.dtype)
    return out.view(shape)


def _near(x: torch.Tensor, by: float, g: torch.Generator) -> torch.Tensor:
    """Another model's logits for the same text."""
    rows = x.view(-1, x.shape[-1])
    out = torch.empty_like(rows)
    step = max(1, (1 << 27) // rows.shape[1])
    for r0 in range(0, rows.shape[0], step):
        c = rows[r0:r0 + step].float()
        out[r0:r0 + step] = (c + by * torch.randn(c.shape, generator=g, device=DEV)).to(out.dtype)
    return out.view(x.shape)


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed, 1)
    st = dict(case)
    if case["kind"] == "top":
        st["logits"] = _logits((case["R"], case["V"]), case["dtype"], g)
    elif case["kind"] == "distill":
        S, T, V, k = case["S"], case["T"], case["V"], min(case["k"], case["V"])
        st["logits"] = _logits((S, T, V), case["dtype"], g)
        # The teacher's entries of every row, as it hands them on: by falling logit, with its log-sum-exp.
        tids = torch.empty((S, T, k), dtype=IDS[case["ids"]], device=DEV)
        tval = torch.empty((S, T, k), dtype=torch.float32, device=DEV)
        tlse = torch.empty((S, T), dtype=torch.float32, device=DEV)
        for s in range(S):
            t = _near(st["logits"][s], 1.0, g).float()
            v, i = torch.topk(t, k, dim=1)
            tids[s], tval[s] = i.to(tids.dtype), v
            tlse[s] = torch.logsumexp(t.double() / case["temperature"], 1).float()
        if case["cut"]:   # lists that end early, some of them empty
            n = torch.randint(0, k + 1, (S, T, 1), generator=g, device=DEV)
            tids[torch.arange(k, device=DEV) >= n] = PAD
        lengths = torch.randint(max(1, T // 4), T + 1, (S, 1), generator=g, device=DEV)
        st.update(teacher_ids=tids, teacher_logits=tval, teacher_lse=tlse if case["tail"] else None,
                  mask=(torch.arange(T, device=DEV) < lengths).float())
    else:
        S, n, V = case["S"], case["n"], case["V"]
        st["target"] = _logits((S, n + 1, V), case["dtype"], g)
        near = _near(st["target"][:, :n].contiguous(), 0.7, g)
        st["draft"] = near if case["draft"] == "model" else None
        if case["temperature"] > 0:   # the drafted tokens come from the draft model's distribution
            ids = torch.empty((S, n), dtype=torch.int64, device=DEV)
            for s in range(S):
                e = torch.empty((n, V), device=DEV).exponential_(generator=g)
                ids[s] = (near[s].float() / case["temperature"] - e.log()).argmax(1)
        else:
            ids = near.float().argmax(2)
        st["draft_ids"] = ids
        st["uniforms"] = torch.rand((S, n + 1), generator=g, device=DEV)
        st["draft_lens"] = (torch.randint(0, n + 1, (S,), generator=g, device=DEV).to(torch.int32)
                            if case["ragged"] else None)
    return st


# ---- one pass -------------------------------------------------------------------------


def _layout(st: dict) -> tuple[int, int]:
    """(token-carrying rows, token of row 0)."""
    return (st["T"] - 1, 1) if st["shifted"] else (st["T"], 0)


def run(st: dict):
    if own:
        return _run_own(st)
    return {"top": _top, "distill": _distill, "verify": _verify}[st["kind"]](st)


def _run_own(st: dict):
    # A program that makes such calls again and again keeps the buffers of their results.
    from pcp_amd import distill, step
    kept = st.get("kept")
    if st["kind"] == "top":
        o = distill.top_logits(st["logits"], st["k"], temperature=st["temperature"], ids_dtype=IDS[st["ids"]],
                               outputs=kept, sync=False)
        out = o.values, o.ids, o.lse
    elif st["kind"] == "distill":
        rows, off = _layout(st)
        o = distill.distill_fwd_bwd(st["logits"], st["teacher_ids"], st["teacher_logits"], st["teacher_lse"],
                                    st["mask"], divergence=st["divergence"], temperature=st["temperature"], rows=rows,
                                    tok_offset=off, dlogits_dtype=DTYPES[st["out"]], outputs=kept, sync=False)
        out = o.loss, o.token_loss, o.dlogits
    else:
        o = step.verify_drafts(st["target"], st["draft_ids"], st["draft"], temperature=st["temperature"],
                               uniforms=st["uniforms"], draft_lens=st["draft_lens"], outputs=kept, sync=False)
        out = o.tokens, o.accepted, o.logp
    st["kept"] = o
    return out


def _top(st: dict):
    x = st["logits"].float()
    R, V = x.shape
    # Keys that order as (logit, then the lower id first), so that equal logits leave no choice.
    b = (x + 0.0).view(torch.int32).to(torch.int64)
    b = torch.where(b < 0, -(b & 0x7fffffff), b)
    key = (b << 32) + (V - 1 - torch.arange(V, device=x.device))
    ids = V - 1 - (torch.topk(key, st["k"], dim=1).values & 0xffffffff)
    z = x / st["temperature"]
    m = z.amax(1, keepdim=True)
    lse = m[:, 0].double() + (z - m).exp().sum(1, dtype=torch.float64).log()
    return x.gather(1, ids), ids.to(IDS[st["ids"]]), lse.float()


def _distill(st: dict):
    S, T, V, tau = st["S"], st["T"], st["V"], st["temperature"]
    rows, off = _layout(st)
    mask = st["mask"]
    w = torch.zeros((S, T), device=mask.device)
    w[:, :rows] = mask[:, off:off + rows]
    ids = st["teacher_ids"].long()
    has = ids >= 0
    at = torch.where(has, ids, ids[..., :1].clamp(min=0))          # an unused entry repeats the first one's id
    w = w * has.any(2)
    # The student: exp(z/tau - max) of every token, its sum, and the sum outside the teacher's entries.
    z = st["logits"].float() / tau
    zi = z.gather(2, at).double()
    m = z.amax(2, keepdim=True)
    e = (z - m).exp_()
    total = e.sum(2, keepdim=True, dtype=torch.float64)
    outside = e.scatter(2, at, 0.0).sum(2, keepdim=True, dtype=torch.float64)
    log_total = m.double() + total.log()
    log_q = zi - log_total
    q = torch.where(has, log_q.exp(), 0.0)
    # The teacher: probabilities of its entries, and of all other tokens together.
    t = torch.where(has, st["teacher_logits"].double() / tau, -math.inf)
    lse = (torch.logsumexp(t, 2) if st["teacher_lse"] is None else st["teacher_lse"].double())[..., None]
    log_p = t - lse
    p = log_p.exp()

    def term(a, log_ratio):
        return torch.where(a > 0, a * log_ratio, 0.0)

    if st["teacher_lse"] is not None:
        has_tail = outside > 0
        p_t = torch.where(has_tail, (1 - p.sum(2, keepdim=True)).clamp(min=TAIL_FLOOR), 0.0)
        q_t = outside / total
        log_pt, log_qt = p_t.log(), q_t.log()
    if st["divergence"] == "forward":
        l = term(p, log_p - log_q).sum(2)
        big_p = p.sum(2, keepdim=True)
        scale = big_p
        if st["teacher_lse"] is not None:
            l = l + term(p_t, log_pt - log_qt)[..., 0]
            big_p = big_p + p_t
            scale = big_p - torch.where(has_tail, p_t / q_t, 0.0)
        grad = q * big_p - p
    else:
        f = torch.where(q > 0, log_q - log_p, 0.0)
        f_t = torch.where(has_tail, log_qt - log_pt, 0.0)
        l = (q * f).sum(2) + (q_t * f_t)[..., 0]
        scale = f_t - l[..., None]
        grad = q * (f - l[..., None])
    token = torch.where(w > 0, w * l, 0.0)
    length = mask[:, off:off + rows].double().sum(1, keepdim=True).clamp(min=1)
    loss = (token / length).sum() / S
    c = (w / (S * length * tau))[..., None]
    dz = e.mul_((c * scale / total).float())
    # An unused entry writes the first one's gradient again.
    dz.scatter_(2, at, torch.where(has, c * grad, c * grad[..., :1]).float())
    dz.masked_fill_((w == 0)[..., None], 0.0)
    tok = torch.zeros((S, T), device=mask.device)
    tok[:, off:off + rows] = token[:, :rows].float()
    return loss.float(), tok, dz.to(DTYPES[st["out"]])


def _verify(st: dict):
    S, n, V, T = st["S"], st["n"], st["V"], st["temperature"]
    x, d, dev = st["target"], st["draft_ids"], st["target"].device
    lens = st["draft_lens"].long() if st["draft_lens"] is not None else torch.full((S,), n, device=dev)
    drafted = torch.arange(n, device=dev) < lens[:, None]
    seq = torch.arange(S, device=dev)
    if T < 1e-6:
        best = (x == x.amax(2, keepdim=True)).to(torch.uint8).argmax(2)      # [S, n + 1], the first of equals
        accepted = ((best[:, :n] == d) & drafted).long().cumprod(1).sum(1)
        last = best[seq, accepted]
        logp = torch.zeros((S, n + 1), device=dev)
    else:
        z = x.double() / T
        log_p = z - torch.logsumexp(z, 2, keepdim=True)                      # [S, n + 1, V]
        lp_d = log_p[:, :n].gather(2, d[..., None])[..., 0]
        u = st["uniforms"].double()
        if st["draft"] is not None:
            y = st["draft"].double() / T
            log_q = y - torch.logsumexp(y, 2, keepdim=True)
            q_d = log_q.gather(2, d[..., None])[..., 0].exp()
        else:
            q_d = torch.ones((S, n), dtype=torch.float64, device=dev)
        accepted = ((u[:, :n] * q_d < lp_d.exp()) & drafted).long().cumprod(1).sum(1)
        # The token after the accepted ones: from max(p - q, 0) where a draft was refused, else from p.
        p = log_p[seq, accepted].exp()
        j = accepted.clamp(max=max(n - 1, 0))
        q = log_q[seq, j].exp() if st["draft"] is not None else torch.nn.functional.one_hot(d[seq, j], V).double()
        r = torch.where((accepted < lens)[:, None], (p - q).clamp(min=0), p)
        cdf = r.cumsum(1)
        last = (cdf <= u[:, n:] * cdf[:, -1:]).sum(1)
        logp = torch.zeros((S, n + 1), device=dev)
        logp[:, :n] = lp_d.float()
        logp[seq, accepted] = log_p[seq, accepted, last].float()
        logp = torch.where(torch.arange(n + 1, device=dev) <= accepted[:, None], logp, 0.0)
    tokens = torch.full((S, n + 1), PAD, dtype=torch.int64, device=dev)
    tokens[:, :n] = torch.where(torch.arange(n, device=dev) < accepted[:, None], d, PAD)
    tokens[seq, accepted] = last
    return tokens, accepted.to(torch.int32), logp


# ---- what a pass cannot do without ----------------------------------------------------


def work(case: dict) -> dict:
    size, V = DTYPES[case["dtype"]].itemsize, case["V"]
    if case["kind"] == "top":
        R, k = case["R"], case["k"]
        return {"bytes": R * (V * size + k * (4 + IDS[case["ids"]].itemsize) + 4), "flops": 3 * R * V}
    if case["kind"] == "distill":
        N, k = case["S"] * case["T"], case["k"]
        # Sequences are live over 5/8 of their length on average; the gradient is written everywhere.
        live = 0.625 * N
        return {"bytes": int(live * (V * size + k * (4 + IDS[case["ids"]].itemsize) + 4)
                             + N * (V * DTYPES[case["out"]].itemsize + 8)), "flops": int(live * 5 * V)}
    S, n = case["S"], case["n"]
    drafted = S * n // (2 if case["ragged"] else 1)
    rows = S + drafted + (drafted if case["draft"] == "model" else 0)
    return {"bytes": rows * V * size + S * (n + 1) * 24, "flops": rows * V * (1 if case["temperature"] == 0 else 3)}


# ---- the operators' definitions in 64 bits --------------------------------------------


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    return {"top": _exact_top, "distill": _exact_distill, "verify": _exact_verify}[case["kind"]](st)


def _exact_top(st: dict):
    R, V, k = st["R"], st["V"], st["k"]
    values = torch.empty((R, k), dtype=torch.float64, device=DEV)
    ids = torch.empty((R, k), dtype=IDS[st["ids"]], device=DEV)
    lse = torch.empty(R, dtype=torch.float64, device=DEV)
    step = max(1, (1 << 25) // V)
    for r0 in range(0, R, step):
        x = st["logits"][r0:r0 + step].double()
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        values[r0:r0 + step], ids[r0:r0 + step] = v[:, :k], i[:, :k].to(ids.dtype)
        lse[r0:r0 + step] = torch.logsumexp(x / st["temperature"], 1)
    return values, ids, lse


def _row_divergence(z, ids, t, lse, forward: bool):
    """One number a row from its scaled student logits z, in categories: the teacher's entries, and the rest."""
    has = ids >= 0
    inside = torch.zeros(z.shape, dtype=torch.bool, device=z.device)
    r = torch.arange(len(z), device=z.device)[:, None].expand_as(ids)
    inside[r[has], ids[has]] = True
    lse_q = torch.logsumexp(z, 1)
    log_q = z.gather(1, ids.clamp(min=0)) - lse_q[:, None]
    if lse is None:
        lse = torch.logsumexp(t.masked_fill(~has, -math.inf), 1)
        tail = None
    else:
        tail = (1 - (t - lse[:, None]).exp().masked_fill(~has, 0.0).sum(1)).clamp(min=TAIL_FLOOR)
    log_p = t - lse[:, None]
    if forward:
        per = log_p.exp() * (log_p - log_q)
    else:
        per = log_q.exp() * (log_q - log_p)
    out = per.masked_fill(~has, 0.0).sum(1)
    if tail is not None:
        log_rest = torch.logsumexp(z.masked_fill(inside, -math.inf), 1) - lse_q
        out = out + (tail * (tail.log() - log_rest) if forward else log_rest.exp() * (log_rest - tail.log()))
    return out


def _exact_distill(st: dict):
    S, T, V, tau = st["S"], st["T"], st["V"], st["temperature"]
    rows, off = _layout(st)
    dz = torch.zeros((S * T, V), dtype=torch.float64, device=DEV)
    tok = torch.zeros((S, T), dtype=torch.float64, device=DEV)
    loss = torch.zeros((), dtype=torch.float64, device=DEV)
    mask = st["mask"].double()
    step = max(1, (1 << 24) // V)
    for s in range(S):
        length = max(float(mask[s, off:off + rows].sum()), 1.0)
        for t0 in range(0, rows, step):
            t1 = min(t0 + step, rows)
            w = mask[s, off + t0:off + t1]
            on = ((w > 0) & (st["teacher_ids"][s, t0:t1] >= 0).any(1)).nonzero()[:, 0]
            if len(on) == 0:
                continue
            at = on + t0
            x = st["logits"][s, at].double().requires_grad_()
            lse = None if st["teacher_lse"] is None else st["teacher_lse"][s, at].double()
            l = w[on] * _row_divergence(x / tau, st["teacher_ids"][s, at].long(), st["teacher_logits"][s, at].double() / tau,
                                        lse, st["divergence"] == "forward")
            part = l.sum() / (length * S)
            dz[s * T + at], = torch.autograd.grad(part, x)
            tok[s, at + off] = l.detach()
            loss += part.detach()
    return loss, tok, dz.view(S, T, V)


def _exact_verify(st: dict):
    """Sequence by sequence on the host, as one would verify by hand."""
    S, n, T = st["S"], st["n"], st["temperature"]
    x = st["target"].float().cpu().numpy()
    y = st["draft"].float().cpu().numpy() if st["draft"] is not None else None
    d, u = st["draft_ids"].cpu().numpy(), st["uniforms"].cpu().numpy().astype(np.float64)
    lens = st["draft_lens"].cpu().numpy() if st["draft_lens"] is not None else np.full(S, n)
    tokens = np.full((S, n + 1), PAD, np.int64)
    accepted = np.zeros(S, np.int32)
    logp = np.zeros((S, n + 1))

    def softmax(row):
        a = row.astype(np.float64) / T
        a = np.exp(a - a.max())
        return a / a.sum()

    for s in range(S):
        i = 0
        while True:
            drafted = i < lens[s]
            if T < 1e-6:
                best = int(np.argmax(x[s, i]))
                if drafted and d[s, i] == best:
                    tokens[s, i] = best
                    i += 1
                    continue
                tokens[s, i] = best
                break
            p = softmax(x[s, i])
            if drafted:
                q = softmax(y[s, i]) if y is not None else np.zeros_like(p)
                if y is None:
                    q[d[s, i]] = 1.0
                if u[s, i] * q[d[s, i]] < p[d[s, i]]:
                    tokens[s, i], logp[s, i] = d[s, i], np.log(p[d[s, i]])
                    i += 1
                    continue
                r = np.maximum(p - q, 0.0)
            else:
                r = p
            c = np.cumsum(r)
            tokens[s, i] = np.searchsorted(c, u[s, n] * c[-1], side="right")
            logp[s, i] = np.log(p[tokens[s, i]])
            break
        accepted[s] = i
    return (torch.from_numpy(tokens).to(DEV), torch.from_numpy(accepted).to(DEV), torch.from_numpy(logp).to(DEV))
