"""The operators of a cache in 8 bits with a scale for each block of 16 places and head, as cases that can be timed and compared.

    attend    attention of a step's rows over the paged 8-bit cache: one call of ops.attention_cache8, as a layer of the model makes it
    store     a step's keys and values stored into the 8-bit cache, and the pages they lie on read back as numbers: one call each of
              ops.store_cache8 and ops.expand_cache8
    copy      pages copied in all layers and planes of a cache group, as a fork inside a page needs it: one call of ops.copy_pages

The plain forms are elementary torch operations in 32 bits on padded batches; `exact` goes through the requests or rows in 64 bits."""
from __future__ import annotations

import math
import random

import torch

own = False
DEV = "cuda:0"
BLOCK = 16                                     # places of a page that share a scale
MOST = {"int8": 127.0, "float8_e4m3fn": 448.0}
LEAST = 1e-30                                  # below it a block's largest number counts as this


# ------------------------------------------------------------------------------------------ cases
def _attend(name, requests, held, rows=1, portions=0, heads=32, kv_heads=8, dim=128, page=16, window=0, cache="int8", dtype="bfloat16",
            ragged=True, lens=1):
    """`requests` requests that hold up to `held` tokens; the first `portions` of them bring up to `rows` rows, the others one; ragged: the
    numbers vary below these bounds (made from `lens`)."""
    c = dict(op="attend", requests=requests, held=held, rows=rows, portions=portions, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
             window=window, cache=cache, dtype=dtype, ragged=ragged, lens=lens)
    return dict(c, name=name) if name else c


def _store(name, requests, held, rows=1, kv_heads=8, dim=128, page=16, cache="int8", dtype="bfloat16", ragged=True, lens=1):
    """`requests` requests that hold up to `held` tokens bring up to `rows` rows each."""
    c = dict(op="store", requests=requests, held=held, rows=rows, kv_heads=kv_heads, dim=dim, page=page, cache=cache, dtype=dtype,
             ragged=ragged, lens=lens)
    return dict(c, name=name) if name else c


def _copy(name, pages, pool, layers, kv_heads=8, dim=128, page=16, cache="int8"):
    """`pages` of the `pool` pages of a cache of `layers` layers; cache: int8 (codes and scales) or bfloat16."""
    c = dict(op="copy", pages=pages, pool=pool, layers=layers, kv_heads=kv_heads, dim=dim, page=page, cache=cache)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one request on an idle engine: launches and latency count
        _attend("attend_one", 1, 700, dim=64, ragged=False),
        # the engine's headline batch behind 2,048-token prompts, plain decoding
        _attend("attend_batch_8", 8, 2176, dim=64),
        # many users with long contexts at the 8B layer sizes: the cache's bytes count
        _attend("attend_users_64", 64, 8192),
        # e4m3 codes, seven query heads a kv head, pages of 32, odd lengths
        _attend("attend_fp8", 24, 5003, heads=28, kv_heads=4, page=32, cache="float8_e4m3fn"),
        # drafted tokens beside each request's newest
        _attend("attend_drafts_16", 16, 3001, rows=5, portions=16, dim=64),
        # a mixed step: portions of two prompts, one of them behind tokens it holds already, beside single tokens
        _attend("attend_mixed", 6, 2500, rows=1500, portions=2),
        # the 32-bit engine
        _attend("attend_32bit", 12, 1777, rows=3, portions=5, dim=64, dtype="float32"),
        # a decode step of a large batch
        _store("store_step_64", 64, 8192),
        # a step of prompt portions that fills max_prefill rows
        _store("store_prompts", 5, 700, rows=1600),
        # the 32-bit engine with e4m3 codes, odd lengths
        _store("store_32bit_fp8", 9, 301, rows=77, kv_heads=4, dim=64, page=32, cache="float8_e4m3fn", dtype="float32"),
        # forks of one prompt inside a page: one page each, 16 layers in 16 bits
        _copy("copy_forks", 8, 512, 16, dim=64, cache="bfloat16"),
        # a cache whose live pages are moved together, 32 layers in 8 bits
        _copy("copy_many", 500, 1100, 32),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "attend", "store", "store", "copy"])
        cache = rng.choice(["int8", "int8", "float8_e4m3fn"])
        dtype = "float32" if rng.random() < 0.2 else "bfloat16"
        lens = rng.randrange(1 << 20)
        if op == "attend":
            heads, kv_heads, dim = rng.choice([(32, 8, 64), (32, 8, 128), (24, 8, 128), (8, 8, 64), (28, 4, 128)])
            R, held = _log_int(rng, 1, 96), _log_int(rng, 40, 24000)
            kind, rows, portions = rng.random(), 1, 0
            if kind < 0.25:
                rows, portions = rng.randint(2, 9), rng.randint(1, R)
            elif kind < 0.5:
                R = min(R, 8)
                rows, portions = _log_int(rng, 20, 2000), rng.randint(1, min(R, 4))
            window = rng.choice([0, 0, 0, _log_int(rng, 30, 4000)])
            c = _attend(None, R, held, rows, portions, heads, kv_heads, dim, rng.choice([16, 16, 32, 64]), window, cache, dtype,
                        rng.random() < 0.7, lens)
        elif op == "store":
            kv_heads, dim = rng.choice([(8, 64), (8, 128), (4, 128), (2, 128)])
            R = _log_int(rng, 1, 128)
            rows = 1 if rng.random() < 0.4 else _log_int(rng, 2, 1600)
            c = _store(None, R, _log_int(rng, 9, 8000), rows, kv_heads, dim, rng.choice([16, 16, 32, 64]), cache, dtype, rng.random() < 0.7,
                       lens)
        else:
            kv_heads, dim = rng.choice([(8, 64), (8, 128), (4, 128)])
            n = _log_int(rng, 1, 500)
            c = _copy(None, n, 2 * n + rng.randint(9, 99), rng.choice([1, 16, 28, 32]), kv_heads, dim, rng.choice([16, 16, 32]),
                      rng.choice(["int8", "bfloat16"]))
        w, top = work(c), [work(x) for x in listed() if x["op"] == c["op"]]
        most = 0.25 if c.get("dtype") == "float32" else 0.9          # (a 32-bit pass takes longer at the same work)
        if w["bytes"] <= most * max(t["bytes"] for t in top) and w["flops"] <= most * max(t["flops"] for t in top):
            return c


# ------------------------------------------------------------------------------------------ sizes
def _lengths(case):
    """Every request's tokens in the cache and its rows in this step."""
    r = random.Random(case["lens"])
    held, rows = [], []
    for i in range(case["requests"]):
        most = case["rows"] if i < case.get("portions", case["requests"]) else 1
        rows.append(r.randint((most + 1) // 2, most) if case["ragged"] else most)
        # (the first portion of a step of portions begins a prompt)
        held.append(0 if i == 0 and most > 16 else r.randint(case["held"] // 2, case["held"]) if case["ragged"] else case["held"])
    return held, rows


def _size(name):
    return {"float32": 4, "bfloat16": 2}.get(name, 1)


def work(case):
    if case["op"] == "copy":
        page = 2 * case["kv_heads"] * (case["page"] * case["dim"] * _size(case["cache"]) + (4 * case["page"] // BLOCK if case["cache"] == "int8" else 0))
        return {"bytes": 2 * case["pages"] * case["layers"] * page, "flops": 0}
    held, rows = _lengths(case)
    e, D, Hkv = _size(case["dtype"]), case["dim"], case["kv_heads"]
    if case["op"] == "store":
        n = sum(rows) * Hkv
        back = sum(_touched(h, m, case["page"]) for h, m in zip(held, rows)) * case["page"] * Hkv      # places that are read back
        return {"bytes": 2 * (n * D * (e + 1) + back * D * (1 + e) + 4 * back // BLOCK), "flops": 4 * n * D}
    w = case["window"] or 1 << 60
    kept = sum(min(h, w - 1) + n for h, n in zip(held, rows))
    seen = sum(min(p + 1, w) for h, n in zip(held, rows) for p in range(h, h + n))
    return {"bytes": kept * Hkv * (2 * D + 8 / BLOCK) + 2 * sum(rows) * case["heads"] * D * e, "flops": 4 * case["heads"] * D * seen}


def _touched(held, rows, page):
    return (held + rows - 1) // page - held // page + 1


# ------------------------------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"attend": _prepare_attend, "store": _prepare_store, "copy": _prepare_copy}[case["op"]](case, seed, gen)


def _tables(case, seed, held, rows):
    """Pages handed out in no order: the requests' block tables (int32 on the host, -1 behind their ends) and how many pages there are."""
    counts = [-(-(h + n) // case["page"]) for h, n in zip(held, rows)]
    ids = list(range(sum(counts) + 3))
    random.Random(seed).shuffle(ids)
    table, at = torch.full((len(counts), max(counts)), -1, dtype=torch.int32), 0
    for r, n in enumerate(counts):
        table[r, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    return table, len(ids)


def _cache(case, pages, gen):
    """Keys' and values' codes and scales of a layer: what normal numbers leave, heads of unlike size, blocks of unlike largest numbers."""
    Hkv, ps, D, blocks = case["kv_heads"], case["page"], case["dim"], -(-case["page"] // BLOCK)
    out = []
    for _ in range(2):
        codes = torch.empty(pages, Hkv, ps, D, dtype=torch.bfloat16, device=DEV).normal_(generator=gen)
        codes = codes.mul_(30.0 if case["cache"] == "int8" else 100.0)
        codes = codes.round_().clamp_(-127, 127).to(torch.int8) if case["cache"] == "int8" else codes.clamp_(-448, 448).to(torch.float8_e4m3fn)
        size = 0.5 + torch.rand(Hkv, 1, generator=gen, device=DEV)
        scales = (0.8 + 0.5 * torch.rand(pages, Hkv, blocks, generator=gen, device=DEV)) * size / (30.0 if case["cache"] == "int8" else 100.0)
        out.append((codes, scales))
    return out


def _prepare_attend(case, seed, gen):
    held, rows = _lengths(case)
    table, pages = _tables(case, seed, held, rows)
    if case["window"]:                                          # pages that no row sees any more have been given back
        for r, h in enumerate(held):
            table[r, :max(0, h - case["window"] + 1) // case["page"]] = -1
    T, Hq, D = sum(rows), case["heads"], case["dim"]
    q = torch.randn(T, Hq * D, generator=gen, device=DEV).mul_(1.2).to(getattr(torch, case["dtype"]))
    (k, ks), (v, vs) = _cache(case, pages, gen)
    s = dict(case=case, q=q, scale=D ** -0.5)
    if own:
        from hipinfer_b200.engine.batch import StepEntry, build_step_batch
        from hipinfer_b200.kernels import ops

        ps = case["page"]
        rows_of = [[row[:-(-(h + n) // ps)].tolist()] for row, h, n in zip(table, held, rows)]
        slots = [[[t[0][p // ps] * ps + p % ps for p in range(h, h + n)]] for t, h, n in zip(rows_of, held, rows)]
        s["batch"] = build_step_batch([StepEntry(r, [0] * n) for r, n in enumerate(rows)], held, list(range(len(rows))), rows_of, slots, 1, DEV)
        s["cache"] = ops.Cache8(k, v, ks, vs)
        return s
    start, most = [sum(rows[:i]) for i in range(len(rows))], max(rows)
    s.update(k=k, v=v, ks=ks, vs=vs, table=table.to(DEV), held=torch.tensor(held).to(DEV), rows=most,
             row=torch.tensor([[a + min(j, n - 1) for j in range(most)] for a, n in zip(start, rows)]).to(DEV),
             valid=torch.tensor([[j < n for j in range(most)] for n in rows]).to(DEV))
    return s


def _prepare_store(case, seed, gen):
    held, rows = _lengths(case)
    table, pages = _tables(case, seed, held, rows)
    ps, T, W = case["page"], sum(rows), case["kv_heads"] * case["dim"]
    slots, touched, local = [], [], []
    for r, (h, n) in enumerate(zip(held, rows)):
        for p in range(h // ps, (h + n - 1) // ps + 1):
            touched.append(int(table[r, p]))
        first = len(touched) - 1 - ((h + n - 1) // ps - h // ps)
        for p in range(h, h + n):
            slots.append(int(table[r, p // ps]) * ps + p % ps)
            local.append(first + p // ps - h // ps)
    # heads of unlike size, now and then a token that stands out
    x = [torch.randn(T, W, generator=gen, device=DEV) * (0.3 + torch.rand(W // case["dim"], generator=gen, device=DEV).repeat_interleave(case["dim"])) for _ in range(2)]
    x[0].mul_(torch.where(torch.rand(T, 1, generator=gen, device=DEV) < 0.05, 4.0, 1.0))
    k, v = (y.to(getattr(torch, case["dtype"])) for y in x)
    (kc, ks), (vc, vs) = _cache(case, pages, gen)
    s = dict(case=case, k=k, v=v, slots=torch.tensor(slots, dtype=torch.int32).to(DEV), pages=torch.tensor(touched, dtype=torch.int32).to(DEV))
    if own:
        from hipinfer_b200.kernels import ops

        s["cache"] = ops.Cache8(kc, vc, ks, vs)
    else:
        s.update(kc=kc, ks=ks, vc=vc, vs=vs, local=torch.tensor(local).to(DEV))
    return s


def _prepare_copy(case, seed, gen):
    shape = (case["layers"], case["pool"], case["kv_heads"], case["page"])
    planes = []
    for _ in range(2):
        if case["cache"] == "int8":
            planes.append(torch.randint(-127, 128, shape + (case["dim"],), dtype=torch.int8, generator=gen, device=DEV))
            planes.append(torch.rand(shape[:3] + (-(-case["page"] // BLOCK),), generator=gen, device=DEV))
        else:
            planes.append(torch.empty(shape + (case["dim"],), dtype=torch.bfloat16, device=DEV).normal_(generator=gen))
    ids = list(range(case["pool"]))
    random.Random(seed).shuffle(ids)
    return dict(case=case, planes=planes, src=ids[:case["pages"]], dst=ids[case["pages"]:2 * case["pages"]])


# ------------------------------------------------------------------------------------------ a pass
def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from hipinfer_b200.kernels import ops

        if op == "attend":
            return ops.attention_cache8(s["q"], s["cache"], s["batch"], 0, s["case"]["heads"], window=s["case"]["window"], scale=s["scale"])
        if op == "store":
            ops.store_cache8(s["k"], s["v"], s["slots"], s["cache"])
            k, v = ops.expand_cache8(s["cache"], s["pages"], s["k"].dtype)
            return k, v, s["cache"].k_scale, s["cache"].v_scale
        ops.copy_pages(s["planes"], s["src"], s["dst"])
        return s["planes"]
    return {"attend": _plain_attend, "store": _plain_store, "copy": _plain_copy}[op](s)


def _plain_attend(s):
    c = s["case"]
    ps, Hq, Hkv, D, n = c["page"], c["heads"], c["kv_heads"], c["dim"], s["rows"]
    R, P = s["table"].shape
    page = s["table"].long().clamp_min(0)

    def values(codes, scales):                                                    # [R, Hkv, keys, D]
        x = codes.view(torch.uint8)[page].view(codes.dtype).float() * scales[page].repeat_interleave(BLOCK, -1)[..., :ps, None]
        return x.transpose(1, 2).reshape(R, Hkv, P * ps, D)

    q = s["q"][s["row"]].float().view(R, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, -1, D) * s["scale"]
    score = (q @ values(s["k"], s["ks"]).transpose(-1, -2)).view(R, Hkv, n, Hq // Hkv, P * ps)
    at = (s["held"][:, None] + torch.arange(n, device=DEV))[:, :, None]
    pos = torch.arange(P * ps, device=DEV)
    sees = (pos <= at) & (s["table"] >= 0).repeat_interleave(ps, 1)[:, None]
    if c["window"]:
        sees &= pos > at - c["window"]
    score = score.masked_fill_(~sees[:, None, :, None], -math.inf)
    w = (score - score.amax(-1, keepdim=True)).exp_()
    o = (w.view(R, Hkv, -1, P * ps) @ values(s["v"], s["vs"])).view(R, Hkv, n, Hq // Hkv, D) / w.sum(-1, keepdim=True)
    return o.permute(0, 2, 1, 3, 4).reshape(R, n, Hq * D)[s["valid"]].to(s["q"].dtype)


def _rounded(x, cache):
    return x.round().to(torch.int8) if cache == "int8" else x.to(torch.float8_e4m3fn)


def _plain_store(s):
    c = s["case"]
    ps, Hkv, D, M, cache = c["page"], c["kv_heads"], c["dim"], MOST[c["cache"]], c["cache"]
    blocks, pages = -(-ps // BLOCK), s["pages"].long()
    place = s["slots"].long() % ps
    block = s["local"] * blocks + place // BLOCK                                   # of the touched pages' blocks
    back = []
    for rows, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x = rows.float().view(-1, Hkv, D)
        most = torch.where(x.isfinite(), x, torch.zeros_like(x)).abs().amax(-1)    # [T, Hkv]
        n = len(pages) * blocks
        new = torch.zeros(n, Hkv, device=DEV).index_reduce_(0, block, most, "amax")
        new = new.clamp_min(LEAST) / torch.full_like(new, M)
        there = torch.zeros(n, 1, dtype=torch.bool, device=DEV).index_fill_(0, block, True)
        # (rows that are no block's first place mark a block of their own, behind the others)
        fresh = torch.zeros(n + 1, 1, dtype=torch.bool, device=DEV).index_fill_(0, torch.where(place % BLOCK == 0, block, n), True)[:n]
        old = scales[pages].transpose(1, 2).reshape(n, Hkv)
        now = torch.where(there, torch.where(fresh, new, torch.maximum(old, new)), old)
        factor = torch.where(fresh, torch.ones_like(now), old / now)
        each = lambda y: y.view(len(pages), blocks, Hkv).transpose(1, 2)           # noqa: E731
        wide = lambda y: each(y).repeat_interleave(BLOCK, -1)[..., :ps, None]      # noqa: E731
        page = _rounded(codes.view(torch.uint8)[pages].view(codes.dtype).float() * wide(factor), cache)
        y = (x * (1.0 / now[block])[..., None]).clamp(-M, M)
        page.view(torch.uint8)[s["local"], :, place] = _rounded(torch.where(y.isnan(), torch.zeros_like(y), y), cache).view(torch.uint8)
        codes.view(torch.uint8)[pages] = page.view(torch.uint8)
        scales[pages] = each(now)
        back.append((page.float() * wide(now)).to(rows.dtype))
    return back[0], back[1], s["ks"], s["vs"]


def _plain_copy(s):
    src, dst = torch.tensor(s["src"]).to(DEV), torch.tensor(s["dst"]).to(DEV)
    for plane in s["planes"]:
        plane[:, dst] = plane[:, src]
    return s["planes"]


# ------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attend": _exact_attend, "store": _exact_store, "copy": _exact_copy}[case["op"]](case, s)


def _exact_attend(case, s):
    held, rows = _lengths(case)
    Hq, Hkv, D, ps, w = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    out, row = [], 0
    for i, (h, n) in enumerate(zip(held, rows)):
        lo = max(0, h - w + 1) // ps if w else 0                                   # the first page that is still there
        ids = s["table"][i, lo:-(-(h + n) // ps)].long()
        keys, values = (torch.cat([x[j].float().double() * y[j].double().repeat_interleave(BLOCK, -1)[:, :ps, None] for j in ids.tolist()], 1)[:, :h + n - lo * ps]
                        for x, y in ((s["k"], s["ks"]), (s["v"], s["vs"])))        # [Hkv, keys, D]
        q = s["q"][row:row + n].double().view(n, Hkv, Hq // Hkv, D)
        pos, at = torch.arange(lo * ps, h + n, device=DEV)[None], torch.arange(h, h + n, device=DEV)[:, None]
        hidden = (pos > at) | (pos <= at - w) if w else pos > at
        for a in range(0, n, 256):                                                 # (rows by the hundred: scores in 64 bits are large)
            score = torch.einsum("nhgd,hld->hgnl", q[a:a + 256], keys) * s["scale"]
            weight = torch.softmax(score.masked_fill(hidden[a:a + 256], -math.inf), -1)
            out.append(torch.einsum("hgnl,hld->nhgd", weight, values).reshape(-1, Hq * D))
        row += n
    return torch.cat(out)


def _nearest(x, cache):
    """x in 64 bits to the nearest code, ties to the even one."""
    if cache == "int8":
        return x.round()
    step = torch.exp2(torch.frexp(x.abs().clamp_min(2.0 ** -6))[1].double() - 4)   # e4m3: three bits behind the first, 2^-9 the least
    return (x / step).round() * step


def _exact_store(case, s):
    _, rows = _lengths(case)
    ps, Hkv, D, M, cache = case["page"], case["kv_heads"], case["dim"], MOST[case["cache"]], case["cache"]
    slots = s["slots"].tolist()
    out = []
    for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        x, scales = x.double().view(-1, Hkv, D), scales.double()
        places = {p: codes[p].float().double() for p in s["pages"].tolist()}
        row = 0
        for n in rows:
            while n:
                page, place = divmod(slots[row], ps)
                b = place // BLOCK
                m = min(n, (b + 1) * BLOCK - place, ps - place)                    # rows of this block
                part = x[row:row + m]
                new = part.abs().amax((0, 2)).clamp_min(LEAST) / M
                old = scales[page, :, b].clone()
                now = new if place % BLOCK == 0 else torch.maximum(old, new)
                if place % BLOCK:
                    block = places[page][:, b * BLOCK:(b + 1) * BLOCK]
                    block.copy_(torch.where((now > old)[:, None, None], _nearest(block * (old / now)[:, None, None], cache), block))
                places[page][:, place:place + m] = _nearest((part / now[None, :, None]).clamp(-M, M), cache).transpose(0, 1)
                scales[page, :, b] = now
                row, n = row + m, n - m
        wide = scales.repeat_interleave(BLOCK, -1)[..., :ps, None]
        out += [torch.stack([places[p] * wide[p] for p in s["pages"].tolist()]), scales]
    return out[0], out[2], out[1], out[3]


def _exact_copy(case, s):
    for plane in s["planes"]:
        for layer in plane:
            for a, b in zip(s["src"], s["dst"]):
                layer[b] = layer[a]
    return [plane.double() if plane.is_floating_point() else None for plane in s["planes"]]
