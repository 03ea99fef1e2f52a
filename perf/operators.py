"""The measured operators of the answering path: a paged key/value cache, the attention that reads it, and the draw of the next token.

``kv_append`` writes the keys and values of new tokens into the pages of a cache, ``kv_copy_pages`` copies pages through all layers (several
completions of one prompt fork its last page; compaction moves pages together), ``paged_attention`` attends from one new token of each
sequence over its pages, ``sample_tokens`` draws the next token by temperature, top-k, top-p and min-p from one given uniform number a row.

Head counts, head sizes and vocabularies are those of the architecture presets; lengths run from one token to 131072.  A layer's pages are
``[pages, 2, kv heads, page size, head size]`` (index 1: keys, values); e4m3 pages come with fp32 scales ``[pages, 2, kv heads, page size]``.
"""
from __future__ import annotations

import math

import torch

own = False

VOCABS = (32768, 128256, 151936)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def listed():
    return [
        # One decode step of one layer: 64 sequences get the keys and values of one token each.  Latency is all of it.
        dict(name="append_token", op="append", B=64, T=1, lo=1, hi=1, before=900, Hkv=8, D=128, P=16, type="bf16"),
        # The prompts of a batch, ragged, padded to the longest: what the prompt pass of one layer stores.
        dict(name="append_prompts", op="append", B=8, T=4096, lo=1000, hi=4096, before=0, Hkv=8, D=128, P=64, type="bf16"),
        # Eight completions of one prompt part ways: its last, partly filled page is copied seven times in every layer of a small model.
        dict(name="pages_fork", op="pages", L=28, n=7, spare=20, Hkv=8, D=128, P=16, type="bf16"),
        # Compaction after most sequences of a batch ended: 128 pages of 64 tokens move in each of 36 layers.
        dict(name="pages_compact", op="pages", L=36, n=128, spare=40, Hkv=8, D=128, P=64, type="bf16"),
        # One short chat turn on a small model: latency only.
        dict(name="attend_short", op="attend", B=1, Hq=16, Hkv=8, D=128, P=16, lo=300, hi=300, type="bf16", window=0, softcap=0.0, sinks=False),
        # A ragged batch of answers in progress.
        dict(name="attend_batch", op="attend", B=64, Hq=32, Hkv=8, D=128, P=16, lo=100, hi=4096, type="bf16", window=0, softcap=0.0, sinks=False),
        # Two sequences of the longest context: the length has to be split over the whole GPU.
        dict(name="attend_long", op="attend", B=2, Hq=64, Hkv=8, D=128, P=64, lo=100001, hi=131072, type="bf16", window=0, softcap=0.0, sinks=False),
        # A large batch over an 8-bit cache, eight query heads to each key/value head.
        dict(name="attend_e4m3", op="attend", B=128, Hq=32, Hkv=4, D=128, P=64, lo=2000, hi=16384, type="e4m3", window=0, softcap=0.0, sinks=False),
        # A sliding-window layer with sink logits and capped scores, heads of 64, fp16.
        dict(name="attend_window", op="attend", B=32, Hq=64, Hkv=8, D=64, P=32, lo=40, hi=8000, type="fp16", window=128, softcap=30.0, sinks=True),
        # One chat token under the usual settings.
        dict(name="sample_chat", op="sample", B=1, V=151936, type="fp32", filters="all"),
        # A group of rollouts at temperature 1 without filters, bf16 logits as the LM-head product leaves them.
        dict(name="sample_rollouts", op="sample", B=64, V=128256, type="bf16", filters="none"),
        # A large batch whose rows ask for different things: greedy rows, top-k rows, top-p rows, min-p rows.
        dict(name="sample_mixed", op="sample", B=256, V=151936, type="fp32", filters="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "pages", "attend", "attend", "attend", "sample", "sample"])
    heads = [(16, 8), (32, 8), (40, 8), (64, 8), (32, 4), (64, 4), (28, 4), (14, 2), (12, 2), (8, 8)]
    if op == "append":
        if rng.random() < 0.4:
            T = lo = hi = 1
            B, before = _log_int(rng, 1, 512), _log_int(rng, 1, 1000)
        else:
            B, T = rng.randint(1, 8), _log_int(rng, 2, 4096)
            hi, lo, before = T, rng.randint(1, T), rng.choice([0, 0, rng.randint(1, 200)])
        return dict(op="append", B=B, T=T, lo=lo, hi=hi, before=before, Hkv=rng.choice([1, 2, 4, 8]), D=rng.choice([64, 128, 128, 256]) if T < 2000 else 128,
                    P=rng.choice([16, 32, 64, 128]), type=rng.choice(["bf16", "bf16", "fp16"]))
    if op == "pages":
        P = rng.choice([16, 32, 64])
        return dict(op="pages", L=rng.randint(1, 36), n=_log_int(rng, 1, 128 * 64 // P // 2), spare=rng.randint(0, 60), Hkv=rng.choice([2, 4, 8]), D=rng.choice([64, 128]), P=P,
                    type=rng.choice(["bf16", "fp16"]))
    if op == "attend":
        Hq, Hkv = rng.choice(heads)
        D, type_ = rng.choice([64, 128, 128, 128, 256]), rng.choice(["bf16", "bf16", "fp16", "e4m3"])
        B = _log_int(rng, 1, 128)
        room = 2 * 131072 * 8 * 128 * 2 // (B * Hkv * D * BYTES[type_]) // 2     # half the largest listed case's bytes
        hi = _log_int(rng, 1, max(1, min(131072, room)))
        lo = rng.choice([hi, max(1, hi // 2), 1, max(1, hi // 10)])
        return dict(op="attend", B=B, Hq=Hq, Hkv=Hkv, D=D, P=rng.choice([16, 32, 64, 128]), lo=lo, hi=hi, type=type_, window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]),
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), sinks=rng.random() < 0.25)
    B = _log_int(rng, 1, 256)
    V = rng.choice([rng.choice(VOCABS), _log_int(rng, 300, 151936)])
    return dict(op="sample", B=B, V=V, type=rng.choice(["fp32", "fp32", "bf16", "fp16"]), filters=rng.choice(["all", "mixed", "mixed", "none", "top_p", "top_k", "min_p"]))


def _spread(case):
    """Lengths (or counts) of the rows: spread evenly over [lo, hi], the longest among them, the same for every seed but for their order."""
    lo, hi, B = case["lo"], case["hi"], case["B"]
    return [hi if b == 0 else lo + int((hi - lo) * ((b * 0.6180339887498949) % 1.0)) for b in range(B)]


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _shuffled_pages(g, B, per_row, pages):
    return torch.randperm(pages, generator=g, device="cuda")[:B * per_row].view(B, per_row).to(torch.int32)


def _normal(g, shape, dtype, scale=1.0):
    """Normal numbers of ``dtype``, made a part at a time so that no fp32 copy of a large cache exists."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    step = 1 << 27
    for a in range(0, flat.numel(), step):
        n = min(step, flat.numel() - a)
        flat[a:a + n] = torch.randn(n, generator=g, device="cuda").mul_(scale).to(dtype)
    return out


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "append":
        B, T, Hkv, D, P, dt = case["B"], case["T"], case["Hkv"], case["D"], case["P"], TYPES[case["type"]]
        per_row = (case["before"] + T + P - 1) // P
        pages = B * per_row + 3
        count = torch.tensor(_spread(case), device="cuda", dtype=torch.int32)[torch.randperm(B, generator=g, device="cuda")]
        qkv = _normal(g, (B, T, 6 * Hkv, D), dt)                        # packed projections: four query heads to a key head, then keys, then values
        return dict(op="append", kv=_normal(g, (pages, 2, Hkv, P, D), dt), k=qkv[:, :, 4 * Hkv:5 * Hkv], v=qkv[:, :, 5 * Hkv:], table=_shuffled_pages(g, B, per_row, pages),
                    start=torch.full((B,), case["before"], device="cuda", dtype=torch.int32), count=count, P=P)
    if case["op"] == "pages":
        pages = 2 * case["n"] + case["spare"]
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        return dict(op="pages", kv=_normal(g, (case["L"], pages, 2, case["Hkv"], case["P"], case["D"]), TYPES[case["type"]]), src=order[:case["n"]].contiguous(),
                    dst=order[case["n"]:2 * case["n"]].contiguous())
    if case["op"] == "attend":
        B, Hq, Hkv, D, P = case["B"], case["Hq"], case["Hkv"], case["D"], case["P"]
        per_row = (case["hi"] + P - 1) // P
        pages = B * per_row + 2
        lengths = torch.tensor(_spread(case), device="cuda", dtype=torch.int32)[torch.randperm(B, generator=g, device="cuda")]
        qt = torch.bfloat16 if case["type"] == "e4m3" else TYPES[case["type"]]
        q = _normal(g, (B, Hq + 2 * Hkv, D), qt, 2.0)[:, :Hq]           # the query part of packed projections
        scales = None
        if case["type"] == "e4m3":                                      # what a quantising append leaves: the largest value of a token and head at 448
            kv = torch.empty((pages, 2, Hkv, P, D), dtype=torch.float8_e4m3fn, device="cuda")
            scales = torch.empty((pages, 2, Hkv, P), device="cuda")
            for a in range(0, pages, 256):
                x = torch.randn((min(256, pages - a), 2, Hkv, P, D), generator=g, device="cuda")
                s = x.abs().amax(-1) / 448.0
                kv[a:a + 256] = (x / s[..., None]).to(torch.float8_e4m3fn)
                scales[a:a + 256] = s
        else:
            kv = _normal(g, (pages, 2, Hkv, P, D), TYPES[case["type"]])
        sinks = torch.randn(Hq, generator=g, device="cuda") if case["sinks"] else None
        return dict(op="attend", q=q, kv=kv, scales=scales, table=_shuffled_pages(g, B, per_row, pages), lengths=lengths, sinks=sinks, window=case["window"],
                    softcap=case["softcap"])
    B, V = case["B"], case["V"]
    logits = torch.randn((B, V), generator=g, device="cuda").mul_(2.5)
    peaks = torch.randint(0, V, (B, 8), generator=g, device="cuda")     # a few tokens that the model favours, more or less sure of itself
    logits.scatter_add_(1, peaks, torch.rand((B, 8), generator=g, device="cuda") * 14.0)
    logits = logits.to(TYPES[case["type"]])
    ones = torch.ones(B, device="cuda")
    temperature, top_k, top_p, min_p = ones.clone(), torch.zeros(B, dtype=torch.int32, device="cuda"), ones.clone(), torch.zeros(B, device="cuda")
    row = torch.arange(B, device="cuda")
    f = case["filters"]
    if f == "all":
        temperature, top_k, top_p, min_p = temperature * 0.7, top_k + 20, top_p * 0.8, min_p + 0.01
    elif f == "top_p":
        top_p = 0.5 + 0.49 * torch.rand(B, generator=g, device="cuda")
    elif f == "top_k":
        temperature, top_k = temperature * 0.9, torch.randint(1, max(2, min(V, 2000)), (B,), generator=g, device="cuda").to(torch.int32)
    elif f == "min_p":
        temperature, min_p = temperature * 1.3, 0.001 + 0.1 * torch.rand(B, generator=g, device="cuda")
    elif f == "mixed":
        temperature = torch.where(row % 5 == 0, 0.0, 0.4 + torch.rand(B, generator=g, device="cuda"))
        top_k = torch.where(row % 5 == 1, 40, torch.where(row % 5 == 4, 1000, 0)).to(torch.int32)
        top_p = torch.where((row % 5 == 2) | (row % 5 == 4), 0.9, 1.0)
        min_p = torch.where(row % 5 == 3, 0.05, 0.0)
    return dict(op="sample", logits=logits, u=torch.rand(B, generator=g, device="cuda"), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


# ---------------------------------------------------------------------------------------------- plain forms
def _plain_append(s):
    kv, k, v, P = s["kv"], s["k"], s["v"], s["P"]
    B, T = k.shape[:2]
    # a padded place writes its row's last token once more (the same values to the same place)
    t = torch.minimum(torch.arange(T, device=k.device)[None], s["count"][:, None].long() - 1)
    pos = s["start"][:, None].long() + t
    page, off = s["table"].long().gather(1, pos // P), pos % P
    rows = torch.arange(B, device=k.device)[:, None]
    kv[page, 0, :, off] = k[rows, t].to(kv.dtype)
    kv[page, 1, :, off] = v[rows, t].to(kv.dtype)
    return kv


def _plain_pages(s):
    s["kv"][:, s["dst"].long()] = s["kv"][:, s["src"].long()]
    return s["kv"]


def _plain_attend(s):
    q, kv, table, n = s["q"], s["kv"], s["table"].long(), s["lengths"].long()
    B, Hq, D = q.shape
    Hkv = kv.shape[2]
    x = kv[table].float()                                               # [B, pages of a row, 2, Hkv, P, D]
    if s["scales"] is not None:
        x = x * s["scales"][table][..., None]
    x = x.permute(0, 2, 3, 1, 4, 5).reshape(B, 2, Hkv, -1, D)
    j = torch.arange(x.shape[3], device=q.device)
    ok = j < n[:, None]
    if s["window"]:
        ok = ok & (j >= n[:, None] - s["window"])
    sc = (q.float().reshape(B, Hkv, Hq // Hkv, D) @ x[:, 0].transpose(-1, -2)) * (1.0 / math.sqrt(D))
    if s["softcap"]:
        sc = torch.tanh(sc / s["softcap"]) * s["softcap"]
    sc = sc.masked_fill(~ok[:, None, None], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - m)
    den = e.sum(-1, keepdim=True)
    lse = (m + torch.log(den))
    if s["sinks"] is not None:
        den = den + torch.exp(s["sinks"].float().reshape(1, Hkv, -1, 1) - m)
    v = torch.where(ok[:, None, :, None], x[:, 1], 0.0)
    return (e @ v / den).reshape(B, Hq, D).to(q.dtype), lse.reshape(B, Hq)


def _plain_sample(s):
    lf = s["logits"].double()
    B, V = lf.shape
    T = s["temperature"].double()[:, None]
    greedy = T <= 0
    l, idx = torch.sort(lf, dim=1, descending=True, stable=True)        # equal logits keep the order of their indices
    x = (l - l[:, :1]) / torch.where(greedy, 1.0, T)
    rank = torch.arange(V, device=lf.device)[None]
    k = s["top_k"].long()[:, None]
    keep = (rank < torch.where(k > 0, k, V)) & ((s["min_p"][:, None] <= 0) | (x >= torch.log(s["min_p"].double().clamp_min(1e-300))[:, None]))
    w = torch.where(keep, torch.exp(x), 0.0)
    before = torch.cumsum(w, 1) - w
    p = s["top_p"].double()[:, None]
    keep = keep & ((p >= 1) | (before < p * w.sum(1, keepdim=True)))
    keep = torch.where(greedy, rank == 0, keep)
    w = torch.zeros_like(lf).scatter_(1, idx, torch.where(keep, torch.exp(x), 0.0))
    c = torch.cumsum(w, 1)
    tok = (c > s["u"].double()[:, None] * c[:, -1:]).to(torch.int8).argmax(1)
    lp = lf.gather(1, tok[:, None])[:, 0] - torch.logsumexp(lf, 1)
    return tok.to(torch.int32), lp.float()


def run(state):
    op = state["op"]
    if own:
        from surogate_b200 import ops

        if op == "append":
            ops.kv_append(state["kv"], state["k"], state["v"], state["table"], state["start"], count=state["count"])
            return state["kv"]
        if op == "pages":
            ops.kv_copy_pages(state["kv"], state["src"], state["dst"])
            return state["kv"]
        if op == "attend":
            return ops.paged_attention(state["q"], state["kv"], state["table"], state["lengths"], window=state["window"], softcap=state["softcap"], sinks=state["sinks"],
                                       scales=state["scales"], return_lse=True)
        return ops.sample_tokens(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    return {"append": _plain_append, "pages": _plain_pages, "attend": _plain_attend, "sample": _plain_sample}[op](state)


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "append":
        n = sum(_spread(case))
        return {"bytes": 2 * n * 2 * case["Hkv"] * case["D"] * size, "flops": 0}
    if case["op"] == "pages":
        return {"bytes": 2 * case["L"] * case["n"] * 2 * case["Hkv"] * case["P"] * case["D"] * size, "flops": 0}
    if case["op"] == "attend":
        n = sum(min(x, case["window"]) if case["window"] else x for x in _spread(case))
        row = 2 * case["Hkv"] * (case["D"] * size + (4 if case["type"] == "e4m3" else 0))
        return {"bytes": n * row + case["B"] * case["Hq"] * (4 * case["D"] + 4), "flops": 4 * n * case["Hq"] * case["D"]}
    # a subtraction, a division and an exponential for each weight and for each term of the log-sum
    return {"bytes": case["B"] * (case["V"] * size + 28), "flops": 6 * case["B"] * case["V"]}


# ---------------------------------------------------------------------------------------------- the same from the definitions, in 64 bits
def _exact_attend(s):
    q, kv, table = s["q"].double(), s["kv"], s["table"].long()
    B, Hq, D = q.shape
    Hkv, P = kv.shape[2], kv.shape[3]
    out, lse = torch.zeros((B, Hq, D), dtype=torch.float64, device="cuda"), torch.full((B, Hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["lengths"].tolist()):
        a = max(0, n - s["window"]) if s["window"] else 0
        pages = table[b, a // P:(n + P - 1) // P]
        skip = a - a // P * P
        for h in range(Hkv):
            part = kv[pages, :, h].double()                             # [pages, 2, P, D]
            if s["scales"] is not None:
                part = part * s["scales"][pages, :, h].double().unsqueeze(-1)
            kk = part[:, 0].reshape(-1, D)[skip:skip + n - a]
            vv = part[:, 1].reshape(-1, D)[skip:skip + n - a]
            for i in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                t = kk.mv(q[b, i]) / math.sqrt(D)
                if s["softcap"]:
                    t = s["softcap"] * torch.tanh(t / s["softcap"])
                lse[b, i] = torch.logsumexp(t, 0)
                total = lse[b, i] if s["sinks"] is None else torch.logaddexp(lse[b, i], s["sinks"][i].double())
                out[b, i] = vv.t().mv(torch.exp(t - total))
    return out, lse


def _exact_sample(s):
    import numpy as np

    rows = s["logits"].double().cpu().numpy()
    B, V = rows.shape
    par = [s[n].double().cpu().numpy() for n in ("u", "temperature", "top_k", "top_p", "min_p")]
    tok, lp = np.zeros(B, np.int32), np.zeros(B)
    for b in range(B):
        r = rows[b]
        u, T, k, p, mp = (float(a[b]) for a in par)
        best = int(r.argmax())
        top = r[best]
        if T <= 0:
            tok[b] = best
        else:
            weight = np.exp((r - top) / T)
            allowed = np.flatnonzero(weight >= mp) if mp > 0 else np.arange(V)
            order = allowed[np.lexsort((allowed, -r[allowed]))]
            if k > 0:
                order = order[:int(k)]
            if p < 1:
                through = np.cumsum(weight[order])
                order = order[:1 + int(np.searchsorted(through, p * through[-1], side="left"))]
            order = np.sort(order)
            through = np.cumsum(weight[order])
            tok[b] = order[min(len(order) - 1, int(np.searchsorted(through, u * through[-1], side="right")))]
        lp[b] = r[tok[b]] - top - math.log(float(np.exp(r - top).sum()))
    return torch.from_numpy(tok), torch.from_numpy(lp)


def exact(case, seed):
    if case["op"] in ("append", "pages"):
        return None                                                     # copies: nothing is computed
    if case["op"] == "attend":
        return _exact_attend(prepare(case, seed)) if case["B"] * case["Hq"] <= 6000 else None
    return _exact_sample(prepare(case, seed))
