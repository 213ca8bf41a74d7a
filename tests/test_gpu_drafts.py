"""Attention over shared prefixes and the verification of drafted tokens, against plain implementations in 64 bits."""
import math
import random

import pytest
import torch

from hipinfer_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 2.0 ** -24
BF16, F32 = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------------------------------- attention
def tables(q, c, groups, page_size, seed, extra=3):
    """Block tables whose shared positions name the same pages where whole pages are shared (a shared part of a page: the group's first table is
    the one that is read there), and the number of pages."""
    rng = random.Random(seed)
    counts = [-(-(n + m) // page_size) for n, m in zip(q, c)]
    ids = list(range(sum(counts) + extra))
    rng.shuffle(ids)
    t = torch.full((len(q), max(counts + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(counts):
        t[r, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
        at += n
    for first, n, shared in groups:
        for r in range(first + 1, first + n):
            k = shared // page_size
            t[r, :k] = t[first, :k]
    return t.to(DEV), len(ids)


def oracle(q, k, v, table, qs, cs, groups, Hq, Hkv, D, ps, scale):
    """(out, sum of p |v|, the largest sum of |q k| scale, the most keys) in 64 bits, row by row of requests; a key that a row does not see takes no part."""
    outs, mags, most, keys_most, row = [], [], 0.0, 1, 0
    via = {r: (f, s) for f, n, s in groups for r in range(f, f + n) if sum(x > 0 for x in qs[f:f + n]) > 1}
    G = Hq // Hkv
    for r, (n, held) in enumerate(zip(qs, cs)):
        first, shared = via.get(r, (r, 0))
        pos = torch.arange(held + n, device=DEV)
        page = torch.where(pos < shared, table[first].long()[pos // ps], table[r].long()[pos // ps])
        K, V = (x[page, :, pos % ps].double() for x in (k, v))                      # [L, Hkv, D]
        for i in range(n):
            L = held + i + 1
            x = q[row].double().view(Hkv, G, D)
            s = torch.einsum("hgd,lhd->hgl", x, K[:L]) * scale
            most = max(most, float((torch.einsum("hgd,lhd->hgl", x.abs(), K[:L].abs().nan_to_num(0, 0, 0)) * abs(scale)).max()))
            p = torch.softmax(s, -1)
            outs.append(torch.einsum("hgl,lhd->hgd", p, V[:L]).reshape(-1))
            mags.append(torch.einsum("hgl,lhd->hgd", p, V[:L].abs()).reshape(-1))
            keys_most = max(keys_most, L)
            row += 1
    return (torch.stack(outs), torch.stack(mags), most, keys_most) if outs else (torch.zeros(0, Hq * D, device=DEV).double(),) * 2 + (0.0, 1)


def bound(dtype, out, mag, most, keys, D):
    """The score of a key is off by at most (D + 4) roundings of its sum of |q k|, twice (numerator and denominator); sums over the keys and the parts
    are off by a rounding each; bfloat16 rounds the probabilities (a relative 2^-9, in numerator and quotient) and the result."""
    b = EPS * (2 * (D + 4) * most + keys + 32) * mag
    return b + (2.0 ** -8 * mag + 2.0 ** -8 * out.abs() if dtype == BF16 else EPS * out.abs())


def case(q, c, groups, Hq, Hkv, D, ps, dtype, seed=0, scale=None, spread=1.0, stride=0, poison=True):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    table, pages = tables(q, c, groups, ps, seed)
    T = sum(q)
    x = torch.randn(T, Hq * D + stride, generator=gen, device=DEV).mul_(spread).to(dtype)[:, :Hq * D]
    k, v = (torch.randn(pages, Hkv, ps, D, generator=gen, device=DEV).to(dtype) for _ in range(2))
    if poison:      # what no row sees: pages of nobody, places behind a request's end, and a group's other tables where the first is read
        seen = torch.zeros(pages, ps, dtype=torch.bool, device=DEV)
        via = {r: (f, s) for f, n, s in groups for r in range(f, f + n) if sum(y > 0 for y in q[f:f + n]) > 1}
        for r, (n, held) in enumerate(zip(q, c)):
            if n:
                first, shared = via.get(r, (r, 0))
                pos = torch.arange(held + n, device=DEV)
                seen[torch.where(pos < shared, table[first].long()[pos // ps], table[r].long()[pos // ps]), pos % ps] = True
        k.masked_fill_(~seen[:, None, :, None], math.nan)
        v.masked_fill_(~seen[:, None, :, None], math.inf)
    scale = D ** -0.5 if scale is None else scale
    return x, k, v, table, scale


def run_case(q, c, groups, Hq, Hkv, D, ps, dtype, **kw):
    x, k, v, table, scale = case(q, c, groups, Hq, Hkv, D, ps, dtype, **kw)
    plan = ops.SharedPlan(q, c, groups, Hq, Hkv, D, ps, dtype, DEV)
    got = ops.attention_shared(x, k, v, table, plan, scale=scale)
    ops.check_device_status()
    out, mag, most, keys = oracle(x, k, v, table, q, c, groups, Hq, Hkv, D, ps, scale)
    assert got.shape == out.shape and got.dtype == dtype
    bad = (got.double() - out).abs() > bound(dtype, out, mag, most, keys, D)
    assert not bad.any() and torch.isfinite(got).all(), (int(bad.sum()), float((got.double() - out).abs().max()))
    torch.cuda.synchronize()
    ops.check_device_status()
    return got


LENGTHS = [
    ("one token", [1], [0], []),
    ("two tokens of two", [1, 1], [0, 1], [(0, 2, 0)]),
    ("a shared page and nothing else", [1, 1, 1], [16, 16, 16], [(0, 3, 16)]),
    ("odd lengths", [1, 3, 2, 5], [333, 300, 401, 299], [(0, 4, 297)]),
    ("a tile's border", [2, 2], [128, 129], [(0, 2, 128)]),
    ("behind a tile's border", [1, 2], [257, 256], [(0, 2, 255)]),
    ("one shared token", [1, 1], [200, 9], [(0, 2, 1)]),
    ("two groups and a loner", [1, 4, 1, 2, 3], [700, 650, 40, 500, 513], [(0, 2, 640), (3, 2, 496)]),
    ("one brings nothing", [2, 0, 3], [150, 140, 145], [(0, 3, 130)]),
    ("long portions", [17, 40, 1], [90, 64, 300], [(0, 3, 64)]),
    ("portions without a cache", [16, 17, 33], [0, 0, 0], []),
    ("many", [1 + r % 3 for r in range(70)], [260 + 7 * r for r in range(70)], [(0, 70, 256)]),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(32, 8, 64, 16), (8, 2, 128, 16), (6, 2, 128, 32), (4, 4, 64, 8), (16, 1, 64, 64), (7, 1, 128, 16)])
@pytest.mark.parametrize("name,q,c,groups", LENGTHS, ids=[x[0] for x in LENGTHS])
def test_attention_shared(name, q, c, groups, Hq, Hkv, D, ps, dtype):
    run_case(q, c, groups, Hq, Hkv, D, ps, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(4, 2, 48, 16), (2, 2, 256, 4), (5, 1, 33, 7), (3, 3, 80, 1), (66, 1, 64, 16), (130, 1, 128, 16), (2, 1, 1, 3), (9, 1, 64, 128),
                                         (9, 1, 128, 256)])
def test_attention_shared_of_other_sizes(Hq, Hkv, D, ps, dtype):
    run_case([2, 1, 4, 20], [150, 171, 140, 133], [(0, 3, 131)], Hq, Hkv, D, ps, dtype)


def test_attention_shared_over_a_long_context():
    run_case([1, 2, 1], [20000, 20111, 20003], [(0, 3, 19999)], 8, 2, 128, 16, BF16)
    run_case([4] * 24, [9000 + 50 * r for r in range(24)], [(0, 24, 8999)], 8, 2, 64, 16, BF16)
    run_case([3] * 5, [9000 + 50 * r for r in range(5)], [(0, 5, 8999)], 4, 2, 64, 16, F32)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_far_apart(dtype):
    """Maxima that grow from tile to tile, and rows of one likely key: queries of a large spread."""
    for spread in (8.0, 40.0):
        x, k, v, table, scale = case([1, 3, 2], [500, 777, 640], [(0, 3, 450)], 8, 2, 128, 16, dtype, seed=3, spread=spread)
        plan = ops.SharedPlan([1, 3, 2], [500, 777, 640], [(0, 3, 450)], 8, 2, 128, 16, dtype, DEV)
        out, mag, most, keys = oracle(x, k, v, table, [1, 3, 2], [500, 777, 640], [(0, 3, 450)], 8, 2, 128, 16, scale)
        got = ops.attention_shared(x, k, v, table, plan)
        assert ((got.double() - out).abs() <= bound(dtype, out, mag, most, keys, 128)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_a_row_that_must_not_see_a_later_one(D, dtype):
    """The keys and values of a drafted token that overflowed stay out of the rows before it, and are in those from it on."""
    q, c, groups = [4, 3, 1], [130, 140, 133], [(0, 3, 128)]
    x, k, v, table, scale = case(q, c, groups, 8, 2, D, 16, dtype)
    plan = ops.SharedPlan(q, c, groups, 8, 2, D, 16, dtype, DEV)
    clean = ops.attention_shared(x, k, v, table, plan)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        pos = c[0] + 2
        k2[int(table[0, pos // 16]), :, pos % 16] = bad
        v2[int(table[0, pos // 16]), :, pos % 16] = bad
        got = ops.attention_shared(x, k2, v2, table, plan)
        keep = torch.tensor([0, 1, 4, 5, 6, 7], device=DEV)
        assert torch.equal(got[keep], clean[keep])
        assert not torch.isfinite(got[2:4]).all(-1).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_q_with_a_stride_and_out_given(dtype):
    q, c, groups = [2, 1, 1], [100, 90, 95], [(0, 3, 80)]
    x, k, v, table, scale = case(q, c, groups, 8, 2, 64, 16, dtype, stride=24)
    plan = ops.SharedPlan(q, c, groups, 8, 2, 64, 16, dtype, DEV)
    want = ops.attention_shared(x.contiguous(), k, v, table, plan)
    out = torch.full_like(want, math.nan)
    assert ops.attention_shared(x, k, v, table, plan, out=out) is out and torch.equal(out, want)
    odd = torch.cat([torch.zeros(4, 3, dtype=dtype, device=DEV), x], 1)[:, 3:]          # rows that start anywhere
    got = ops.attention_shared(odd, k, v, table, plan)
    ref, mag, most, keys = oracle(x, k, v, table, q, c, groups, 8, 2, 64, 16, scale)
    assert ((got.double() - ref).abs() <= bound(dtype, ref, mag, most, keys, 64)).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_the_same_bits_again_and_on_another_stream(dtype):
    q, c, groups = [2] * 20, [1200 + r for r in range(20)], [(0, 20, 1111)]
    x, k, v, table, scale = case(q, c, groups, 8, 2, 128, 16, dtype)
    plan = ops.SharedPlan(q, c, groups, 8, 2, 128, 16, dtype, DEV)
    want = ops.attention_shared(x, k, v, table, plan)
    for _ in range(5):
        assert torch.equal(ops.attention_shared(x, k, v, table, plan), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.attention_shared(x, k, v, table, plan)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_call_can_be_captured():
    q, c, groups = [3] * 6, [300 + r for r in range(6)], [(0, 6, 280)]
    x, k, v, table, scale = case(q, c, groups, 8, 2, 64, 16, BF16)
    plan = ops.SharedPlan(q, c, groups, 8, 2, 64, 16, BF16, DEV)
    want = ops.attention_shared(x, k, v, table, plan)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.attention_shared(x, k, v, table, plan)
    y = x.flip(0)
    x.copy_(y)
    graph.replay()
    assert torch.equal(got, ops.attention_shared(x, k, v, table, plan)) and not torch.equal(got, want)


# ---------------------------------------------------------------------------------------------- verification
def decide(logits, start, n, drafts, t, u, noise, probs):
    """One request in 64 bits: tokens, log probabilities, and how near its nearest decision was to the other answer."""
    tokens, logps, margin = [], [], math.inf
    for i in range(n + 1):
        x = logits[start + i].double()
        V = x.numel()
        top = math.nan if bool(x.isnan().any()) else float(x.max())
        best = int(x.isnan().nonzero()[0]) if math.isnan(top) else int((x == top).nonzero()[0])
        point = t == 0 or not math.isfinite(top)
        lp = torch.log_softmax(x / (t or 1.0), 0) if math.isfinite(top) else torch.zeros_like(x)
        p = lp.exp() if not point else torch.zeros(V, dtype=torch.float64)
        if point:
            p[best] = 1.0
        w = p
        if i < n:
            d = int(drafts[i])
            q = torch.zeros(V, dtype=torch.float64) if probs is None else probs[i].double()
            inside = 0 <= d < V
            if probs is None and inside:
                q[d] = 1.0
            pd, qd = (float(p[d]), float(q[d])) if inside else (0.0, 0.0)
            if inside and float(u[i]) * qd > 0:
                margin = min(margin, abs(math.log(max(pd, 1e-300) / (float(u[i]) * qd))))
            if float(u[i]) * qd < pd:
                tokens.append(d)
                logps.append(float(lp[d]))
                continue
            w = (p - q).clamp_min(0)
            if not float(w.max()) > 0:
                w = p
        s = torch.where(w > 0, w / noise.double(), torch.full_like(w, -1.0))
        order = torch.sort(s, descending=True, stable=True)
        if not point:
            if V > 1 and float(order.values[1]) > 0 and float(order.values[0]) != float(order.values[1]):
                margin = min(margin, math.log(float(order.values[0]) / float(order.values[1])))
            # what a difference of nearly equal numbers loses
            margin = min(margin, margin * float(w[order.indices[0]] / p[order.indices[0]]))
        token = best if point else int((s == s.max()).nonzero()[0])
        tokens.append(token)
        logps.append(float(lp[token]))
        return tokens, logps, margin


def check_verify(logits, start, lens, drafts, t, u, noise, probs=None, allow=0.02):
    got = ops.verify_drafts(logits, *(torch.tensor(x, dtype=torch.int32, device=DEV) for x in (start, lens)), drafts, t, u, noise, probs)
    tokens, counts, logps = (x.cpu() for x in got)
    host = [x.float().cpu() if x is not None else None for x in (logits, t, u, noise, probs)]
    near = 0
    for r, n in enumerate(lens):
        want, lp, margin = decide(host[0], start[r], n, drafts[r].tolist(), float(host[1][r]), host[2][r], host[3][r], None if probs is None else host[4][r])
        if margin < 1e-4:        # rounding may decide
            near += 1
            continue
        assert tokens[r].tolist() == want + [-1] * (drafts.shape[1] + 1 - len(want)), r
        assert int(counts[r]) == len(want)
        # x is exact; its difference from the largest, over t, is rounded four times; the sum's relative error is that of its exponents and of V additions
        for i, y in enumerate(lp):
            big = float(host[0][start[r] + i].nan_to_num(0, 0, 0).abs().max()) / (float(host[1][r]) or 1.0)
            assert abs(float(logps[r, i]) - y) <= EPS * (16 * big + 8 * abs(y) + 64), (r, i)
        assert (logps[r, len(lp):] == 0).all()
    assert near <= allow * len(lens)
    return tokens, counts


def make_verify(R, K, V, dtype=F32, probs=None, seed=0, ragged=True, greedy=3, pad=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)
    lens = [rng.randint(0, K) if ragged else K for _ in range(R)]
    start, at = [], 0
    for n in lens:
        start.append(at)
        at += n + 1
    logits = (torch.randn(at, V + pad, generator=gen, device=DEV) * 3).to(dtype)[:, :V]
    t = torch.rand(R, generator=gen, device=DEV) + 0.5
    if greedy:
        t[::greedy] = 0.0
    rows = torch.tensor([[a + min(j, n) for j in range(max(K, 1))] for a, n in zip(start, lens)], device=DEV)
    soft = torch.softmax((logits[rows].float() + torch.randn(R, max(K, 1), V, generator=gen, device=DEV) * 0.5) / (t + 0.05)[:, None, None], -1)
    drafts = (soft / torch.empty_like(soft).exponential_(generator=gen)).argmax(-1).to(torch.int32)[:, :K].contiguous()
    u = torch.rand(R, K, generator=gen, device=DEV)
    noise = torch.empty(R, V + pad, device=DEV).exponential_(generator=gen)[:, :V]
    return logits, start, lens, drafts, t, u, noise, None if probs is None else soft[:, :K].to(probs).contiguous()


@pytest.mark.parametrize("R,K,V", [(1, 0, 1), (1, 1, 2), (3, 2, 7), (40, 4, 100), (33, 7, 1025), (5, 63, 257), (9, 3, 8191), (7, 2, 32000), (2, 5, 128256), (300, 1, 33)])
@pytest.mark.parametrize("dtype,probs", [(F32, None), (F32, F32), (BF16, BF16), (BF16, None), (F32, BF16)])
def test_verify_drafts(R, K, V, dtype, probs):
    check_verify(*make_verify(R, K, V, dtype, probs, seed=R + K + V), allow=0.1)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad", [1, 3, 5])
def test_rows_that_start_anywhere(pad, dtype):
    """Rows of a wider tensor, of an odd number of elements."""
    check_verify(*make_verify(12, 3, 1000, dtype, dtype, seed=pad, pad=pad))
    logits, start, lens, drafts, t, u, noise, probs = make_verify(12, 3, 999, dtype, dtype, seed=pad)
    wide = torch.empty(12, 5, 999 + pad, dtype=dtype, device=DEV)
    wide[:, :3, :999] = probs
    check_verify(logits, start, lens, drafts, t, u, noise, wide[:, :3, :999])


def fixed(x, n=0, t=1.0, drafts=(), u=(), noise=None, probs=None):
    logits = torch.tensor(x, dtype=F32, device=DEV)
    V, K = logits.shape[1], len(drafts)
    return [y[0].tolist() for y in ops.verify_drafts(
        logits, torch.zeros(1, dtype=torch.int32, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV),
        torch.tensor([drafts], dtype=torch.int32, device=DEV).view(1, K), torch.tensor([t], dtype=F32, device=DEV), torch.tensor([u], dtype=F32, device=DEV).view(1, K),
        torch.ones(1, V, device=DEV) if noise is None else torch.tensor([noise], dtype=F32, device=DEV),
        None if probs is None else torch.tensor([probs], dtype=F32, device=DEV))]


def test_ties_go_to_the_lowest_index():
    assert fixed([[0.0, 5.0, 5.0, 1.0]], t=0.0)[0] == [1]
    assert fixed([[-0.0, 0.0, -1.0]], t=0.0)[0] == [0]
    assert fixed([[2.0, 2.0, 2.0]], t=1.0)[0] == [0]
    x = torch.zeros(1, 70001)
    x[0, 40000] = x[0, 69999] = 1.0
    assert fixed(x.tolist(), t=0.0)[0] == [40000]
    assert fixed(x.tolist(), t=1.0, noise=[0.5 if v in (40000, 69999) else 3.0 for v in range(70001)])[0] == [40000]


def test_rows_without_a_finite_largest_logit():
    inf, nan = math.inf, math.nan
    for t in (0.0, 0.7):
        assert fixed([[-inf, -inf, -inf]], t=t) == [[0], 1, [0.0]]
        assert fixed([[1.0, inf, inf]], t=t) == [[1], 1, [0.0]]
        assert fixed([[1.0, inf, nan, nan]], t=t) == [[2], 1, [0.0]]
        # a draft is accepted where it is that token, else refused
        assert fixed([[1.0, inf, 2.0], [-inf, -inf, 3.0]], n=1, t=t, drafts=[1], u=[0.999])[:2] == [[1, 2], 2]
        assert fixed([[1.0, inf, 2.0], [-inf, -inf, 3.0]], n=1, t=t, drafts=[0], u=[0.0])[:2] == [[1, -1], 1]
    assert fixed([[-inf, 4.0, -inf]], t=0.5) == [[1], 1, [0.0]]          # one possible token: log 1


def test_a_refused_draft_is_not_drawn_again():
    # its probability is the largest and the noise favours it
    assert fixed([[3.0, 1.0, 0.0], [0.0, 0.0, 0.0]], n=1, drafts=[0], u=[0.95], noise=[1e-6, 1.0, 1.0])[0] == [1, -1]
    assert fixed([[3.0, 1.0, 0.0], [0.0, 0.0, 0.0]], n=1, drafts=[0], u=[0.5], noise=[1.0, 1.0, 1e-6])[0] == [0, 2]
    # p and q the same, refused by the random number alone (a token p does not hold): the residual is empty and p stands in
    p = torch.softmax(torch.tensor([2.0, 1.0, -200.0]), 0)
    assert fixed([[2.0, 1.0, -200.0], [0.0, 0.0, 0.0]], n=1, drafts=[2], u=[0.5], probs=[[1.0, 1.0, 1.0]])[0] == [0, -1]
    assert fixed([[2.0, 1.0, 0.0], [0.0, 0.0, 0.0]], n=1, drafts=[1], u=[0.9], noise=[1.0, 1e-3, 1.0], probs=[[0.1, 0.6, 0.3]])[0] == [0, -1]
    assert float(p[2]) == 0


def test_numbers_out_of_range():
    assert fixed([[3.0, 1.0], [1.0, 2.0]], n=1, t=0.0, drafts=[5], u=[0.0])[0] == [0, -1]                 # no such token: refused
    assert fixed([[3.0, 1.0], [1.0, 2.0]], n=1, t=0.0, drafts=[-1], u=[0.0], probs=[[0.5, 0.5]])[0] == [0, -1]
    assert fixed([[3.0, 1.0], [1.0, 2.0]], n=9, t=0.0, drafts=[0], u=[0.0])[:2] == [[0, 1], 2]            # more drafts than there are: K
    assert fixed([[3.0, 1.0]], n=-3, t=0.0, drafts=[0], u=[0.0])[:2] == [[0, -1], 1]
    logits = torch.tensor([[3.0, 1.0]], device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)                                      # noqa: E731
    tokens, counts, logps = ops.verify_drafts(logits, i32(1, -1, 0), i32(0, 0, 1), i32(0, 0, 0).view(3, 1), torch.zeros(3, device=DEV), torch.zeros(3, 1, device=DEV),
                                              torch.ones(3, 2, device=DEV))
    assert tokens.tolist() == [[-1, -1], [-1, -1], [0, -1]] and counts.tolist() == [0, 0, 1] and logps[:2].eq(0).all()


def test_noise_at_its_ends():
    assert fixed([[0.0, 0.0, 0.0]], noise=[1.0, 0.0, 0.0])[0] == [1]
    assert fixed([[0.0, 0.0, 0.0]], noise=[math.inf, math.inf, 1.0])[0] == [2]
    assert fixed([[0.0, 0.0, -math.inf]], noise=[math.inf, math.inf, 1.0])[0] == [0]
    assert fixed([[0.0, 0.0, 0.0]], noise=[math.nan, 5.0, 9.0])[0] == [1]


@pytest.mark.parametrize("lookup", [False, True])
def test_what_is_produced_is_distributed_as_the_target(lookup):
    """First tokens of many requests with the same target and draft distributions: each token's share is within five standard deviations."""
    R, V = 60000, 6
    gen = torch.Generator(device=DEV).manual_seed(11)
    x = torch.tensor([1.0, 0.0, -1.0, 2.0, 0.5, -0.5], device=DEV)
    q = torch.softmax(torch.tensor([0.0, 1.0, 0.0, 1.0, -1.0, 0.5], device=DEV), 0)
    logits = x.repeat(2 * R, 1)
    drafts = torch.full((R, 1), 1, dtype=torch.int32, device=DEV) if lookup else torch.multinomial(q, R, replacement=True, generator=gen).to(torch.int32).view(R, 1)
    tokens, counts, _ = ops.verify_drafts(logits, torch.arange(0, 2 * R, 2, dtype=torch.int32, device=DEV), torch.ones(R, dtype=torch.int32, device=DEV), drafts,
                                          torch.full((R,), 0.8, device=DEV), torch.rand(R, 1, generator=gen, device=DEV),
                                          torch.empty(R, V, device=DEV).exponential_(generator=gen), None if lookup else q.repeat(R, 1, 1))
    p = torch.softmax(x.double() / 0.8, 0)
    for i in (0, 1):
        of = tokens[:, i] >= 0
        n = int(of.sum())
        share = torch.bincount(tokens[of, i].long(), minlength=V).double() / n
        assert (share - p).abs().le(5 * (p * (1 - p) / n).sqrt()).all(), (i, share, p)
    rate = float(p[1]) if lookup else float(torch.minimum(p, q.double()).sum())
    assert abs(float((counts - 1).double().mean()) - rate) <= 5 * math.sqrt(rate * (1 - rate) / R)


def test_verification_again_on_another_stream_and_captured():
    a = make_verify(6, 3, 5003, F32, F32, seed=4)
    args = [a[0]] + [torch.tensor(x, dtype=torch.int32, device=DEV) for x in a[1:3]] + list(a[3:])
    want = ops.verify_drafts(*args)
    for _ in range(4):
        assert all(torch.equal(x, y) for x, y in zip(ops.verify_drafts(*args), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.verify_drafts(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.verify_drafts(*args)
    graph.replay()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q,c,groups", [([1, 2], [200, 210], [(0, 2, 192)]), ([20, 40], [200, 210], [(0, 2, 192)])], ids=["few rows", "many rows"])
def test_a_score_that_is_not_finite_makes_its_rows_nan(q, c, groups, dtype):
    """At every place of a tile's steps, in the prefix, a request's own keys and the step's: NaN and +inf scores are NaN rows, -inf ones weigh nothing."""
    Hq, Hkv, D, ps = 8, 2, 64, 16
    x, k, v, table, scale = case(q, c, groups, Hq, Hkv, D, ps, dtype, poison=False)
    plan = ops.SharedPlan(q, c, groups, Hq, Hkv, D, ps, dtype, DEV)
    first = torch.tensor([[i] for n in q for i in range(n)], device=DEV)
    held = torch.tensor([[c[r]] for r, n in enumerate(q) for _ in range(n)], device=DEV)
    own = torch.tensor([[r == 1] for r, n in enumerate(q) for _ in range(n)], device=DEV)
    sign = x.view(-1, Hq, D)[:, :, 0]
    for pos in list(range(64, 192, 3)) + list(range(128, 192)) + [192, 200, 209, 210]:
        r = 1 if pos >= 192 else 0            # (the prefix is read through the first request's table)
        sees = (held + first >= pos) & (own if r == 1 else torch.ones_like(own))
        for bad in (math.nan, math.inf):
            k2 = k.clone()
            k2[int(table[r, pos // ps]), :, pos % ps, 0] = bad
            got = ops.attention_shared(x, k2, v, table, plan).view(-1, Hq, D)
            hit = sees & (torch.ones_like(sign, dtype=torch.bool) if math.isnan(bad) else sign > 0)
            assert got[hit].isnan().all() and torch.isfinite(got[~hit]).all(), (pos, bad)
    ops.check_device_status()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales(dtype):
    """A scale of 0 is the mean of the values; one that is negative or no number is refused."""
    x, k, v, table, _ = case([1, 3], [130, 140], [(0, 2, 128)], 4, 2, 64, 16, dtype)
    plan = ops.SharedPlan([1, 3], [130, 140], [(0, 2, 128)], 4, 2, 64, 16, dtype, DEV)
    out, mag, most, keys = oracle(x, k, v, table, [1, 3], [130, 140], [(0, 2, 128)], 4, 2, 64, 16, 0.0)
    got = ops.attention_shared(x, k, v, table, plan, scale=0.0)
    assert ((got.double() - out).abs() <= bound(dtype, out, mag, most, keys, 64)).all()
    for bad in (-0.1, math.nan, math.inf):
        with pytest.raises(ops.KernelError, match="scale"):
            ops.attention_shared(x, k, v, table, plan, scale=bad)


@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 64), (BF16, 80)])
def test_a_cache_of_more_than_32_bits_of_elements(dtype, D):
    """Pages at the far end of a cache of more than 2^31 elements give the bits that the same pages give in a small one."""
    q, c, groups, Hkv, ps = [2, 1, 18], [150, 171, 133], [(0, 2, 128)], 2, 16
    x, k, v, table, scale = case(q, c, groups, 4, Hkv, D, ps, dtype, poison=False)
    plan = ops.SharedPlan(q, c, groups, 4, Hkv, D, ps, dtype, DEV)
    want = ops.attention_shared(x, k, v, table, plan)
    pages = k.shape[0]
    total = 2 ** 31 // (Hkv * ps * D) + 2 * pages
    if torch.cuda.mem_get_info()[0] < 3 * total * Hkv * ps * D * x.element_size():
        pytest.skip("not enough free memory")
    far = []
    for small in (k, v):
        big = torch.empty(total, Hkv, ps, D, dtype=dtype, device=DEV)
        big[total - pages:] = small
        far.append(big)
    assert far[0].numel() > 2 ** 31
    got = ops.attention_shared(x, *far, torch.where(table < 0, table, table + (total - pages)), plan)
    assert torch.equal(got, want)
    ops.check_device_status()
    del far, big
    torch.cuda.empty_cache()
