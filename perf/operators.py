"""The operators of a step that samples many continuations of one prompt with drafted tokens, as cases that can be timed and compared.

    attend    attention of the step's rows over a paged cache in which groups of requests share the pages of a long prefix: one call
              of ops.attention_shared, as a layer of the model makes it, with the plan that all layers of a step share
    verify    the drafted tokens against the target's logits: one call of ops.verify_drafts

The plain forms are elementary torch operations in 32 bits on padded batches; `exact` goes through the requests one by one in 64 bits."""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda:0"


# ------------------------------------------------------------------------------------------ cases
def _attend(name, groups, per_group, rows, prefix, tail, heads=32, kv_heads=8, dim=128, page=16, dtype="bfloat16", ragged=True, lens=1):
    """`groups` prefixes of up to `prefix` tokens, each shared by `per_group` requests that hold up to `tail` tokens of their own and
    bring up to `rows` rows; ragged: the numbers vary below these bounds (made from `lens`)."""
    c = dict(op="attend", groups=groups, per_group=per_group, rows=rows, prefix=prefix, tail=tail, heads=heads, kv_heads=kv_heads, dim=dim,
             page=page, dtype=dtype, ragged=ragged, lens=lens)
    return dict(c, name=name) if name else c


def _verify(name, requests, drafts, vocab, logits="float32", draft_probs="none", greedy=0, temperature=0.8, ragged=True, lens=1):
    """`requests` requests with up to `drafts` drafted tokens; every `greedy`-th one (0: none) at temperature 0; draft_probs: "none" (a
    draft that was looked up), or the element type of the distributions the drafts were drawn from."""
    c = dict(op="verify", requests=requests, drafts=drafts, vocab=vocab, logits=logits, draft_probs=draft_probs, greedy=greedy,
             temperature=temperature, ragged=ragged, lens=lens)
    return dict(c, name=name) if name else c


def listed():
    return [
        # two answers to one short question on an idle engine: launches and latency count
        _attend("attend_two", 1, 2, 1, 509, 24, dim=64),
        # eight samples of one 2,048-token prompt, the engine's headline batch, plain decoding
        _attend("attend_samples_8", 1, 8, 1, 2048, 128, dim=64),
        # the same with four drafted tokens a request
        _attend("attend_drafts_8", 1, 8, 5, 2048, 128, dim=64, ragged=False),
        # many users of one long system prompt at the 8B layer sizes, plain decoding: own tokens and prefix weigh alike
        _attend("attend_users_64", 1, 64, 1, 8192, 512),
        # four documents, a dozen questions each, with drafts; three query heads a kv head, pages of 32, odd lengths
        _attend("attend_documents", 4, 12, 6, 5003, 301, heads=24, page=32),
        # the largest: 96 samples with three drafted tokens behind a 24k-token context
        _attend("attend_context_96", 1, 96, 4, 24571, 1024, ragged=False),
        # the 32-bit engine, some samples with drafts
        _attend("attend_32bit", 1, 12, 3, 1777, 200, dim=64, dtype="float32"),
        # one answer with drafts found in its own text
        _verify("verify_one", 1, 3, 32000),
        # the headline batch, drafts found in the text, no distribution of their own
        _verify("verify_lookup_8", 8, 4, 128256),
        # a draft model's distributions beside the target's, some requests greedy
        _verify("verify_model_24", 24, 5, 128256, draft_probs="float32", greedy=4),
        # a large batch, 16-bit logits and distributions, a vocabulary of odd size
        _verify("verify_batch_96", 96, 7, 50021, logits="bfloat16", draft_probs="bfloat16", greedy=5, temperature=1.0),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n + 1 if n == 3072 else n


MOST = 0.9      # a drawn case's work, as a part of the largest listed one's


def draw(rng):
    while True:
        if rng.random() < 0.6:
            heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (24, 8, 128), (8, 8, 64), (28, 4, 128)])
            dtype = "float32" if rng.random() < 0.2 else "bfloat16"
            groups = rng.choice([1, 1, 1, 2, 3, 5])
            c = _attend(None, groups, _log_int(rng, 1, 128 // groups), rng.randint(1, 8), _log_int(rng, 100, 24000),
                        _log_int(rng, 9, 1024), heads, kv_heads, dim, rng.choice([16, 16, 32, 64]), dtype, rng.random() < 0.7,
                        rng.randrange(1 << 20))
        else:
            kind = rng.choice(["float32", "float32", "bfloat16"])
            c = _verify(None, _log_int(rng, 1, 128), rng.randint(1, 8), _log_int(rng, 20000, 130000), kind,
                        rng.choice(["none", "none", "float32", "bfloat16"]), rng.choice([0, 0, 3]), round(rng.uniform(0.3, 1.4), 2),
                        rng.random() < 0.7, rng.randrange(1 << 20))
        w, top = work(c), [work(x) for x in listed() if x["op"] == c["op"]]
        most = MOST / 4 if c.get("dtype") == "float32" else MOST      # a 32-bit pass takes longer at the same work
        if w["bytes"] <= most * max(t["bytes"] for t in top) and w["flops"] <= most * max(t["flops"] for t in top):
            return c


# ------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """Of an attend case: the groups' shared tokens (the whole pages of their prefixes), and every request's tokens in the cache and
    rows (requests of a group one after the other)."""
    r = random.Random(case["lens"])
    prefixes, ctx, rows = [], [], []
    for _ in range(case["groups"]):
        s = r.randint(case["prefix"] * 3 // 4, case["prefix"]) if case["ragged"] and case["groups"] > 1 else case["prefix"]
        prefixes.append(s // case["page"] * case["page"])
        for _ in range(case["per_group"]):
            n = r.randint(1, case["rows"]) if case["ragged"] else case["rows"]
            held = r.randint(0, case["tail"]) if case["ragged"] else case["tail"] - r.randint(0, min(15, case["tail"] // 2))
            ctx.append(s + held)       # (the prompt's last, part-filled page is among what a request holds)
            rows.append(n)
    return prefixes, ctx, rows


def _draft_lens(case):
    r = random.Random(case["lens"])
    return [r.randint(0, case["drafts"]) if case["ragged"] and case["requests"] > 1 else case["drafts"] for _ in range(case["requests"])]


def _size(name):
    return 4 if name == "float32" else 2


def work(case):
    if case["op"] == "attend":
        prefixes, ctx, rows = _lengths(case)
        per = case["per_group"]
        kept = sum(prefixes) + sum(c + n - prefixes[i // per] for i, (c, n) in enumerate(zip(ctx, rows)))
        seen = sum(n * c + n * (n + 1) // 2 for c, n in zip(ctx, rows))
        e, dim = _size(case["dtype"]), case["dim"]
        return {"bytes": kept * 2 * case["kv_heads"] * dim * e + 2 * sum(rows) * case["heads"] * dim * e,
                "flops": 4 * case["heads"] * dim * seen}
    lens, V = _draft_lens(case), case["vocab"]
    n = sum(x + 1 for x in lens)
    q = 0 if case["draft_probs"] == "none" else _size(case["draft_probs"]) * V * sum(x > 0 for x in lens)
    return {"bytes": n * V * _size(case["logits"]) + q + 4 * V * case["requests"], "flops": 3 * n * V}


# ------------------------------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return (_prepare_attend if case["op"] == "attend" else _prepare_verify)(case, seed, gen)


def _prepare_attend(case, seed, gen):
    prefixes, ctx, rows = _lengths(case)
    per, ps, Hq, Hkv, D = case["per_group"], case["page"], case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    R, T = len(ctx), sum(rows)
    # block tables: the pages of a prefix are the same ones in its group, the rest are a request's own
    counts = [-(-(c + n) // ps) for c, n in zip(ctx, rows)]
    shared = [s // ps for s in prefixes]
    total = sum(shared) + sum(k - shared[i // per] for i, k in enumerate(counts))
    ids = list(range(total))
    random.Random(seed).shuffle(ids)
    at, table = 0, torch.full((R, max(counts)), -1, dtype=torch.int32)
    for g, n in enumerate(shared):
        common = ids[at:at + n]
        at += n
        for i in range(g * per, (g + 1) * per):
            mine = ids[at:at + counts[i] - n]
            at += counts[i] - n
            table[i, :counts[i]] = torch.tensor(common + mine, dtype=torch.int32)
    q = torch.randn(T, Hq * D, generator=gen, device=DEV).to(dtype)
    k = torch.empty(total, Hkv, ps, D, dtype=dtype, device=DEV).normal_(generator=gen)
    v = torch.empty(total, Hkv, ps, D, dtype=dtype, device=DEV).normal_(generator=gen)
    s = dict(case=case, q=q * (1.5 if D == 64 else 1.2), k=k, v=v, table=table.to(DEV), scale=D ** -0.5)
    if own:
        from hipinfer_b200.kernels import ops

        s["plan"] = ops.SharedPlan(rows, ctx, [(g * per, per, n) for g, n in enumerate(prefixes)], Hq, Hkv, D, ps, dtype, DEV)
        return s
    start = [sum(rows[:i]) for i in range(R)]
    most = max(rows)
    at = torch.tensor([[a + min(j, n - 1) for j in range(most)] for a, n in zip(start, rows)])
    s.update(rows=at.to(DEV), valid=torch.tensor([[j < n for j in range(most)] for n in rows]).to(DEV), ctx=torch.tensor(ctx).to(DEV),
             prefix=torch.tensor(prefixes).to(DEV), most_prefix=max(1, max(shared)),
             most_own=max(c + n - prefixes[i // per] for i, (c, n) in enumerate(zip(ctx, rows))))
    return s


def _prepare_verify(case, seed, gen):
    lens, R, K, V = _draft_lens(case), case["requests"], case["drafts"], case["vocab"]
    T = sum(n + 1 for n in lens)
    # a target with a few likely tokens among many unlikely ones, and a draft that mostly agrees with it
    logits = torch.randn(T, V, generator=gen, device=DEV).mul_(1.5)
    likely = torch.randint(V // 8, (T, 1), generator=gen, device=DEV) + torch.arange(8, device=DEV) * (V // 8)
    logits.scatter_(1, likely, torch.rand(T, 8, generator=gen, device=DEV) * 8 + 8)
    logits = logits.to(getattr(torch, case["logits"]))
    start = [sum(n + 1 for n in lens[:i]) for i in range(R)]
    rows = torch.tensor([[a + min(j, n) for j in range(K)] for a, n in zip(start, lens)]).to(DEV)
    temperature = torch.full((R,), case["temperature"])
    if case["greedy"]:
        temperature[::case["greedy"]] = 0.0
    temperature = temperature.to(DEV)
    hot = torch.where(temperature > 0, temperature, torch.full_like(temperature, 0.1))
    probs = torch.randn(R, K, V, generator=gen, device=DEV).mul_(0.4).add_(logits[rows].float())
    probs = torch.softmax(probs.div_(hot[:, None, None]), -1)
    race = torch.empty(R, K, V, device=DEV).exponential_(generator=gen)
    drafts = (probs / race).argmax(-1).to(torch.int32)
    del race
    s = dict(case=case, logits=logits, start=torch.tensor(start, dtype=torch.int32).to(DEV), drafts=drafts, temperature=temperature,
             n_drafts=torch.tensor(lens, dtype=torch.int32).to(DEV), uniform=torch.rand(R, K, generator=gen, device=DEV),
             noise=torch.empty(R, V, device=DEV).exponential_(generator=gen),
             probs=None if case["draft_probs"] == "none" else probs.to(getattr(torch, case["draft_probs"])))
    return s


# ------------------------------------------------------------------------------------------ a pass
def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from hipinfer_b200.kernels import ops

        if op == "attend":
            return ops.attention_shared(s["q"], s["k"], s["v"], s["table"], s["plan"], scale=s["scale"])
        return ops.verify_drafts(s["logits"], s["start"], s["n_drafts"], s["drafts"], s["temperature"], s["uniform"], s["noise"], s["probs"])
    return (_plain_attend if op == "attend" else _plain_verify)(s)


def _plain_attend(s):
    c = s["case"]
    Ng, per, ps, Hq, Hkv, D = c["groups"], c["per_group"], c["page"], c["heads"], c["kv_heads"], c["dim"]
    G, R, n = Hq // Hkv, Ng * per, s["rows"].shape[1]
    q = s["q"][s["rows"]].float().view(R, n, Hkv, G, D).permute(0, 2, 1, 3, 4) * s["scale"]      # [R, Hkv, n, G, D]
    # the prefixes, once a group
    first = s["table"][::per, :s["most_prefix"]].long().clamp_min(0)
    pages = lambda x: x[first].float().permute(0, 2, 1, 3, 4).reshape(Ng, Hkv, -1, D)            # noqa: E731
    qg = q.reshape(Ng, per, Hkv, n * G, D).permute(0, 2, 1, 3, 4).reshape(Ng, Hkv, per * n * G, D)
    sp = qg @ pages(s["k"]).transpose(-1, -2)
    sp = sp.masked_fill(torch.arange(sp.shape[-1], device=DEV) >= s["prefix"][:, None, None, None], -math.inf)
    # the requests' own keys, padded to the longest
    begin = s["prefix"].repeat_interleave(per)
    pos = begin[:, None] + torch.arange(s["most_own"], device=DEV)
    page = s["table"].long().gather(1, (pos // ps).clamp_max(s["table"].shape[1] - 1)).clamp_min(0)
    mine = lambda x: x[page, :, pos % ps].float().transpose(1, 2)                                 # noqa: E731  [R, Hkv, S, D]
    so = (q.reshape(R, Hkv, n * G, D) @ mine(s["k"]).transpose(-1, -2)).view(R, Hkv, n, G, -1)
    at = s["ctx"][:, None] + torch.arange(n, device=DEV)
    so = so.masked_fill((pos[:, None, :] > at[:, :, None])[:, None, :, None, :], -math.inf).view(R, Hkv, n * G, -1)
    # joined
    back = lambda x: x.view(Ng, Hkv, per, n * G, -1).transpose(1, 2).reshape(R, Hkv, n * G, -1)   # noqa: E731
    m = torch.maximum(back(sp.amax(-1, keepdim=True)), so.amax(-1, keepdim=True))
    group = m.view(Ng, per, Hkv, n * G, 1).transpose(1, 2).reshape(Ng, Hkv, per * n * G, 1)
    ep, eo = (sp - group).exp(), (so - m).exp()
    total = back(ep.sum(-1, keepdim=True)) + eo.sum(-1, keepdim=True)
    o = (back(ep @ pages(s["v"])) + eo @ mine(s["v"])) / total
    o = o.view(R, Hkv, n, G, D).transpose(1, 2).reshape(R, n, Hq * D)
    return o[s["valid"]].to(s["q"].dtype)


def _plain_verify(s):
    R, K = s["drafts"].shape
    n, V = s["n_drafts"].long(), s["logits"].shape[1]
    steps = torch.arange(K + 1, device=DEV)
    rows = s["start"].long()[:, None] + torch.minimum(steps, n[:, None])
    x = s["logits"][rows].float()                                                # [R, K + 1, V]
    t = s["temperature"][:, None, None]
    x = x / torch.where(t > 0, t, torch.ones_like(t))
    m = x.amax(-1, keepdim=True)
    index = torch.arange(V, device=DEV)
    best = torch.where(x == m, index, V).amin(-1)                                # the lowest of the largest
    z = (x - m).exp()
    total = z.sum(-1, keepdim=True)
    p = torch.where(t > 0, z / total, (index == best[:, :, None]).float())
    d = s["drafts"].long()[:, :, None]
    pd = p[:, :K].gather(-1, d)[..., 0]
    qd = torch.ones_like(pd) if s["probs"] is None else s["probs"].gather(-1, d)[..., 0].float()
    ok = (s["uniform"] * qd < pd) & (steps[:K] < n[:, None])
    taken = ok.long().cumprod(-1).sum(-1)                                        # accepted drafts
    each = torch.arange(R, device=DEV)
    last = p[each, taken]
    i = taken.clamp_max(K - 1)
    away = (index == d[each, i]).float() if s["probs"] is None else s["probs"][each, i].float()
    rest = (last - away).clamp_min(0)
    rest = torch.where((taken < n)[:, None] & (rest.amax(-1, keepdim=True) > 0), rest, last)
    score = torch.where(rest > 0, rest / s["noise"], -1.0)
    final = torch.where(score == score.amax(-1, keepdim=True), index, V).amin(-1)
    tokens = torch.where(steps < taken[:, None], torch.nn.functional.pad(s["drafts"], (0, 1)).long(), final[:, None])
    gone = steps > taken[:, None]
    logp = (x - m).gather(-1, tokens[:, :, None])[..., 0] - total[..., 0].log()
    return tokens.masked_fill(gone, -1).to(torch.int32), (taken + 1).to(torch.int32), logp.masked_fill(gone, 0.0)


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return (_exact_attend if case["op"] == "attend" else _exact_verify)(case, s)


def _exact_attend(case, s):
    _, ctx, rows = _lengths(case)
    Hq, Hkv, D, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out, row = [], 0
    for i, (held, n) in enumerate(zip(ctx, rows)):
        ids = s["table"][i, :-(-(held + n) // ps)].long()
        keys, values = (torch.cat(list(x[ids]), 1)[:, :held + n].double() for x in (s["k"], s["v"]))          # [Hkv, L, D]
        q = s["q"][row:row + n].double().view(n, Hkv, Hq // Hkv, D)
        hidden = torch.arange(held + n, device=DEV)[None] > held + torch.arange(n, device=DEV)[:, None]
        score = torch.einsum("nhgd,hld->hgnl", q, keys) * s["scale"]
        weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        out.append(torch.einsum("hgnl,hld->nhgd", weight, values).reshape(n, Hq * D))
        row += n
    return torch.cat(out)


def _exact_verify(case, s):
    R, K = s["drafts"].shape
    logp = torch.zeros(R, K + 1, dtype=torch.float64, device=DEV)
    start, lens, temps, u = (s[x].tolist() for x in ("start", "n_drafts", "temperature", "uniform"))
    drafts = s["drafts"].tolist()
    for r in range(R):
        t = temps[r]
        for i in range(lens[r] + 1):
            lp = torch.log_softmax(s["logits"][start[r] + i].double() / (t or 1.0), 0)
            p = lp.exp() if t else torch.zeros_like(lp).index_fill_(0, torch.nonzero(lp == lp.max())[0], 1.0)
            w = p
            if i < lens[r]:
                d = drafts[r][i]
                q = torch.zeros_like(p).index_fill_(0, torch.tensor([d], device=DEV), 1.0) if s["probs"] is None else s["probs"][r, i].double()
                if u[r][i] * float(q[d]) < float(p[d]):
                    logp[r, i] = lp[d]
                    continue
                w = (p - q).clamp_min(0)
                w = w if float(w.max()) > 0 else p
            logp[r, i] = lp[int((w / s["noise"][r].double()).argmax())]
            break
    return None, None, logp
