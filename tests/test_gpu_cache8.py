"""A paged cache in 8 bits on the GPU: storing (bit for bit), reading back, attention against 64 bits, copying pages.

Tolerances of the attention, on |result - exact| against the largest number V of the row's values (a result is an average of values, weights of
sum 1). float32 rows: scores are sums of D products in 32 bits, off by at most D 2^-24 of their sum of absolute values, A; a weight by A D 2^-24 +
some 2^-22 of itself (its exponential), a sum of n of them by n 2^-24: together below V (2 A D 2^-24 + 2^-20) for the lengths here. bfloat16 rows:
the result's rounding, 2^-8 of itself, and weights (or keys and values) of 16 bits on the way: 2^-8 of V each at most, for keys times A, and errors
of many keys average; in all V 2^-8 (2 + A) as a bound that no row passes."""
import numpy as np
import pytest
import torch

import plain_cache8 as plain
from hipinfer_b200.engine.batch import StepEntry, build_step_batch
from hipinfer_b200.kernels import cache8, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CODES = [torch.int8, torch.float8_e4m3fn]
ids = lambda t: str(t).replace("torch.", "")


def filled(pages, heads, ps, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        codes = (torch.randn(pages, heads, ps, D, generator=g) * 40).clamp(-127, 127)
        codes = codes.round().to(torch.int8) if dtype == torch.int8 else codes.to(dtype)
        out.append((codes, torch.rand(pages, heads, ops.cache8_blocks(ps), generator=g) * 0.04 + 0.01))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def on_gpu(cache):
    return ops.Cache8(*(t.to(DEV) for t in cache))


def same(a, b):
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


# ------------------------------------------------------------------------------------------ storing
def runs(kind, ps, pages):
    """Places of a call's rows."""
    if kind == "one":
        return [2 * ps + ps - 1]
    if kind == "decode":                                                          # single tokens, some at a block's first place
        return [p * ps + (5 * p + 3) % ps for p in range(pages - 1)] + [(pages - 1) * ps]
    if kind == "portion":                                                         # from inside a block over pages in no order
        order = [3, 0, 4, 1][: pages - 1]
        return [order[i // ps] * ps + i % ps for i in range(7 % ps, len(order) * ps - 2)]
    if kind == "gaps":                                                            # rows that are not stored, and places outside of the cache
        return [ps, -1, ps + 1, ps + 2, pages * ps, 3 * ps + 1, -5, 0, 1]
    return [ps + 1, ps + 1, ps + 2, ps + 1] + [2 * ps] * 40                        # "again": one place several times, the last one counts


@pytest.mark.parametrize("kind", ["one", "decode", "portion", "gaps", "again"])
@pytest.mark.parametrize("heads, ps, D", [(8, 16, 64), (2, 16, 128), (3, 32, 128), (1, 64, 64), (5, 8, 96), (2, 24, 33), (4, 4, 256), (1, 1, 8)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_stored_codes_and_scales_are_those_of_the_formula(kind, heads, ps, D, codes, dtype):
    pages = 6
    cache, slots = filled(pages, heads, ps, D, codes), runs(kind, ps, pages)
    g = torch.Generator().manual_seed(len(slots))
    k, v = (torch.randn(len(slots), heads * D, generator=g).mul_(torch.rand(len(slots), 1, generator=g) * 4).to(dtype) for _ in range(2))
    got = on_gpu(cache)
    wide = torch.cat([torch.zeros(len(slots), 5), k.float(), v.float()], 1).to(dtype).to(DEV)        # (parts of wider rows, not aligned)
    ops.store_cache8(wide[:, 5:5 + heads * D], wide[:, 5 + heads * D:], torch.tensor(slots, dtype=torch.int32, device=DEV), got)
    for rows, c, s, gc, gs in ((k, cache[0], cache[2], got.k, got.k_scale), (v, cache[1], cache[3], got.v, got.v_scale)):
        wc, ws = plain.store(rows, slots, c, s)
        assert same(gs, ws) and same(gc, wc)
    again = on_gpu(cache)
    ops.store_cache8(k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV), again)
    assert all(same(a, b) for a, b in zip(again.tensors, got.tensors))


@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_numbers_that_are_not_finite_and_very_small_and_large_ones(codes, dtype):
    ps, D = 16, 64
    rows = torch.zeros(6, D)
    rows[0] = torch.linspace(-3, 3, D)
    rows[0, 3], rows[0, 4], rows[0, 5] = float("inf"), float("-inf"), float("nan")
    rows[1, 0] = 1e-38                         # a block of numbers below the least scale
    rows[3] = torch.finfo(dtype).max
    rows[4, ::2] = float("nan")                # nothing finite but zeros
    rows[5] = float("inf")
    rows = rows.to(dtype)
    slots = [0, ps, 2 * ps, 3 * ps, 4 * ps, 5 * ps]
    cache = filled(7, 1, ps, D, codes)
    got = on_gpu(cache)
    ops.store_cache8(rows.to(DEV), rows.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV), got)
    wc, ws = plain.store(rows, slots, cache[0], cache[2])
    assert same(got.k, wc) and same(got.k_scale, ws)
    assert torch.isfinite(got.k_scale).all() and (got.k_scale > 0).all()
    assert torch.equal(got.k[0, 0, 0, 3:6].float().cpu(), torch.tensor([float(plain.MOST[codes]), -float(plain.MOST[codes]), 0.0]))


@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_a_request_s_tokens_one_by_one_and_in_portions_stay_within_their_error(codes):
    """Every place is off by at most half a step of its code for its own rounding and for each time that its block's scale grew after it."""
    ps, D, T = 32, 64, 77
    g = torch.Generator().manual_seed(5)
    rows = (torch.randn(T, 2 * D, generator=g) * torch.rand(T, 1, generator=g).exp()).to(DEV)
    slots = torch.arange(T, dtype=torch.int32, device=DEV) + 2 * ps
    for cuts in ([1] * T, [40, 1, 1, 20, 15], [T]):
        cache, at, grew = ops.new_cache8(7, 2, ps, D, codes, DEV), 0, torch.zeros(T, 2)
        for n in cuts:
            before = cache.k_scale.clone()
            ops.store_cache8(rows[at:at + n], rows[at:at + n], slots[at:at + n], cache)
            up = (cache.k_scale > before)[2:].cpu().transpose(1, 2).reshape(-1, 2).repeat_interleave(16, 0)[:T]
            grew[:at] += up[:at]
            at += n
        got, _ = ops.expand_cache8(cache, torch.arange(2, 5, dtype=torch.int32, device=DEV), torch.float32)
        got = got.transpose(1, 2).reshape(-1, 2 * D)[:T].cpu()
        scale = cache.k_scale[2:5].cpu().transpose(1, 2).reshape(-1, 2).repeat_interleave(16, 0)[:T].repeat_interleave(D, 1)
        half = scale / 2 if codes == torch.int8 else torch.maximum(got.abs() / 15, scale * 2.0 ** -10)      # (e4m3: 2^-4 of the number or of its step's)
        assert ((got - rows.cpu()).abs() <= half * 1.001 * (1 + grew.repeat_interleave(D, 1))).all()


@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("heads, ps, D", [(8, 16, 64), (2, 32, 128), (3, 24, 40), (1, 4, 7)])
def test_pages_come_back_as_numbers(codes, dtype, heads, ps, D):
    cache = filled(5, heads, ps, D, codes, 3)
    pages = [4, 0, 4, -1, 5, 2]
    k, v = ops.expand_cache8(on_gpu(cache), torch.tensor(pages, dtype=torch.int32, device=DEV), dtype)
    for got, c, s in ((k, cache[0], cache[2]), (v, cache[1], cache[3])):
        want = torch.from_numpy(plain.values(c)) * s.repeat_interleave(16, -1)[:, :, :ps, None]
        want = torch.stack([want[p] if 0 <= p < 5 else torch.zeros_like(want[0]) for p in pages]).to(dtype)
        assert same(got, want)


# ------------------------------------------------------------------------------------------ attention
def step(held, rows, ps, window=0, spare=2, seed=0):
    """A batch whose requests hold `held` tokens and bring `rows` rows, with pages in no order."""
    counts = [-(-(h + n) // ps) for h, n in zip(held, rows)]
    order = np.random.default_rng(seed).permutation(sum(counts) + spare)
    tables, at = [], 0
    for h, c in zip(held, counts):
        t = order[at:at + c].tolist()
        gone = max(0, h - window + 1) // ps if window else 0
        tables.append([[-1] * gone + t[gone:]])
        at += c
    slots = [[[0] * n] for n in rows]
    batch = build_step_batch([StepEntry(i, [0] * n) for i, n in enumerate(rows)], held, list(range(len(rows))), tables, slots, 1, DEV)
    return batch, [t[0] for t in tables], sum(counts) + spare


def check(q, cache, batch, tables, heads, window=0, scale=None):
    got = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, heads, window=window, scale=scale)
    D = cache[0].shape[3]
    scale = D ** -0.5 if scale is None else scale
    want = plain.attend(q, cache, tables, batch.row_request.tolist(), batch.positions.tolist(), heads, window, scale)
    V = float(np.abs(plain.numbers(cache[1], cache[3])).max())
    A = float(q.float().abs().max()) * D ** 0.5 * abs(scale) * float(np.abs(plain.numbers(cache[0], cache[2])).std()) * 3
    tol = V * (2 * A * D * 2.0 ** -24 + 2.0 ** -20) if q.dtype == torch.float32 else V * 2.0 ** -8 * (2 + A)
    assert got.dtype == q.dtype and np.abs(got.double().cpu().numpy() - want).max() <= tol
    return got


STEPS = {
    "first token": ([0], [1]),
    "one": ([15], [1]),
    "long": ([5000], [1]),
    "decode": ([0, 1, 15, 16, 31, 300, 777, 64, 1023], [1] * 9),
    "drafts": ([3, 100, 517], [5, 1, 4]),
    "portion": ([0, 40], [70, 33]),
    "mixed": ([37, 0, 250, 9], [65, 17, 1, 3]),
}


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("heads, kv_heads, ps, D", [(32, 8, 16, 64), (8, 2, 16, 128), (7, 1, 32, 128), (4, 4, 64, 64), (6, 2, 8, 64), (24, 1, 16, 64),
                                                    (2, 1, 24, 80), (4, 2, 16, 256), (40, 1, 16, 128), (3, 1, 5, 3)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_attention(name, heads, kv_heads, ps, D, codes, dtype):
    held, rows = STEPS[name]
    batch, tables, pages = step(held, rows, ps)
    q = torch.randn(sum(rows), heads * D, generator=torch.Generator().manual_seed(1)).to(dtype)
    check(q, filled(pages, kv_heads, ps, D, codes), batch, tables, heads)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 1000])
@pytest.mark.parametrize("name", ["decode", "drafts", "mixed"])
@pytest.mark.parametrize("heads, kv_heads, ps, D", [(8, 2, 16, 64), (4, 1, 32, 128), (4, 2, 8, 40)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_a_window_and_pages_that_are_gone(window, name, heads, kv_heads, ps, D, dtype):
    held, rows = STEPS[name]
    batch, tables, pages = step(held, rows, ps, window)
    q = torch.randn(sum(rows), heads * D, generator=torch.Generator().manual_seed(2)).to(dtype)
    check(q, filled(pages, kv_heads, ps, D, torch.int8), batch, tables, heads, window, 0.2)


@pytest.mark.parametrize("D, ps", [(64, 16), (128, 16), (40, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_rows_that_see_nothing_are_zero_and_places_behind_them_do_not_count(D, ps, dtype):
    """Pages that are not there, and NaN codes and scales at places that no row sees."""
    held, rows = [40, 100, 7], [1, 1, 1]
    batch, tables, pages = step(held, rows, ps)
    batch.block_tables[0][0] = -1
    batch.block_tables[0][1, :2] = torch.tensor([pages + 3, -7])
    tables = [row.tolist() for row in batch.block_tables[0].cpu()]
    cache = filled(pages, 2, ps, D, torch.float8_e4m3fn)
    used = {(t[j // ps], j % ps) for t, h in zip(tables, held) for j in range(h + 1)}
    blocks = {(p, i // 16) for p, i in used}
    for p in range(pages):
        for i in range(ps):
            if (p, i) not in used:
                cache[0].view(torch.uint8)[p, :, i] = 0x7f
                cache[1].view(torch.uint8)[p, :, i] = 0xff
            if (p, i // 16) not in blocks:
                cache[2][p, :, i // 16] = float("nan")
                cache[3][p, :, i // 16] = float("inf")
    q = torch.randn(3, 4 * D, generator=torch.Generator().manual_seed(3)).to(dtype)
    got = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 4)
    keep = tuple(torch.nan_to_num(t.float(), 0, 0, 0).to(t.dtype) for t in cache)
    want = check(q, keep, batch, tables, 4)
    assert same(got, want) and not got[0].any() and torch.isfinite(got.float()).all()


@pytest.mark.parametrize("D", [64, 128, 72])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_rows_with_infinities_and_nan_are_nan_and_stay_alone(D, dtype):
    batch, tables, pages = step([200, 200, 200, 200], [1, 1, 1, 1], 16)
    q = torch.randn(4, 4 * D, generator=torch.Generator().manual_seed(4)).to(dtype)
    cache = filled(pages, 1, 16, D, torch.int8)
    want = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 4)
    q[1, 5], q[2, D + 1] = float("nan"), float("inf")
    got = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 4)
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert torch.equal(got.view(4, 4, D).isnan().all(-1).cpu(), bad) and same(got.view(4, 4, D)[~bad.to(DEV)], want.view(4, 4, D)[~bad.to(DEV)])


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4, 1e30])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_sizes_of_queries_and_values_far_from_one(size, dtype):
    """Scores that are the same numbers whatever the queries' and keys' sizes; values in blocks of very unlike sizes."""
    D, ps = 64, 16
    batch, tables, pages = step([300, 31], [1, 3], ps)
    q = (torch.randn(4, 8 * D, generator=torch.Generator().manual_seed(6)) * size).to(dtype)
    k, v, ks, vs = filled(pages, 2, ps, D, torch.int8)
    ks /= size
    check(q, (k, v, ks, vs), batch, tables, 8)
    check(q, (k, v, ks, vs * size), batch, tables, 8)
    vs[::3] *= 1e-6
    check(q, (k, v, ks, vs), batch, tables, 8)


def test_rows_of_wider_ones_an_output_of_one_s_own_and_another_stream():
    held, rows, D = [33, 500], [1, 1], 64
    batch, tables, pages = step(held, rows, 16)
    cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
    wide = torch.randn(2, 3 + 4 * D + 9, device=DEV).to(torch.bfloat16)
    q = wide[:, 3:3 + 4 * D]
    want = ops.attention_cache8(q.contiguous(), cache, batch, 0, 4)
    out = torch.full((2, 4 * D), 7.0, dtype=torch.bfloat16, device=DEV)
    assert ops.attention_cache8(q, cache, batch, 0, 4, out=out) is out and same(out, want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = ops.attention_cache8(q, cache, batch, 0, 4)
    torch.cuda.current_stream().wait_stream(stream)
    assert same(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_a_captured_step_follows_its_positions_and_tables(dtype):
    """Store and attention of a decode step in a CUDA graph: new rows, places and positions are written over the old ones."""
    D, ps, heads, kv = 64, 16, 8, 2
    held = [20, 45, 100]
    batch, tables, pages = step([511] * 3, [1] * 3, ps)          # (launches for the longest positions)
    start = filled(pages, kv, ps, D, torch.int8)
    cache = on_gpu(start)
    q = torch.zeros(3, heads * D, dtype=dtype, device=DEV)
    k, v = (torch.zeros(3, kv * D, dtype=dtype, device=DEV) for _ in range(2))

    def both():
        ops.store_cache8(k, v, batch.slot_maps[0], cache)
        return ops.attention_cache8(q, cache, batch, 0, heads)

    both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for t, s in zip(cache.tensors, start):
        t.view(torch.uint8).copy_(s.view(torch.uint8)) if t.dtype != torch.float32 else t.copy_(s)
    now = [t.clone() for t in start]
    for i in range(20):
        g = torch.Generator().manual_seed(i)
        new = [torch.randn(3, w, generator=g).to(dtype) for w in (heads * D, kv * D, kv * D)]
        slots = [t[h // ps] * ps + h % ps for t, h in zip(tables, held)]
        for dst, src in zip((q, k, v, batch.positions, batch.slot_maps[0]), new + [torch.tensor(held), torch.tensor(slots)]):
            dst.copy_(src)
        graph.replay()
        for j in range(2):
            now[j], now[2 + j] = plain.store(new[1 + j], slots, now[j], now[2 + j])
        assert all(same(a, b) for a, b in zip(cache.tensors, now))
        want = plain.attend(new[0], now, tables, [0, 1, 2], held, heads, 0, D ** -0.5)
        assert np.abs(out.double().cpu().numpy() - want).max() <= 2.0 ** -6 * float(np.abs(plain.numbers(now[1], now[3])).max())
        held = [h + 1 for h in held]


def test_the_same_call_gives_the_same_bits():
    batch, tables, pages = step([4000, 37, 900], [1, 1, 1], 16)
    cache = on_gpu(filled(pages, 8, 16, 128, torch.int8))
    q = torch.randn(3, 32 * 128, device=DEV).to(torch.bfloat16)
    first = ops.attention_cache8(q, cache, batch, 0, 32)
    assert all(same(first, ops.attention_cache8(q, cache, batch, 0, 32)) for _ in range(20))


# ------------------------------------------------------------------------------------------ copying
@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16, torch.float32, torch.float8_e4m3fn], ids=ids)
@pytest.mark.parametrize("shape", [(1, 9, 5), (3, 700, 2, 16, 64), (2, 40, 1, 8, 3), (4, 11, 2, 16, 128)])
def test_pages_are_copied(dtype, shape):
    g = torch.Generator().manual_seed(0)
    planes = [torch.randint(0, 255, shape[:-1] + (shape[-1] * dtype.itemsize,), dtype=torch.uint8, generator=g).view(dtype) for _ in range(2)]
    planes.append(torch.rand(shape[0] + 1, shape[1], 3, generator=g))               # another plane with more layers
    n = shape[1]
    order = np.random.default_rng(1).permutation(n)
    half = n // 2
    src, dst = order[:half], order[half:2 * half]
    src[half // 2:half // 2 + 2] = src[0]                                           # one page to several others
    got = [t.to(DEV) for t in planes]
    ops.copy_pages(got, src.tolist(), dst.tolist())
    for t, w in zip(got, planes):
        w = w.clone()
        x = w.view(torch.uint8) if w.dtype != torch.float32 else w
        x[:, torch.from_numpy(dst)] = x[:, torch.from_numpy(src)]
        assert same(t, w)


def test_planes_that_are_part_of_wider_ones_and_many_planes():
    g = torch.Generator().manual_seed(2)
    whole = torch.randn(4, 12, 64, generator=g).to(DEV)
    planes = [whole[i % 4:i % 4 + 1, :, 4 * i:4 * i + 3] for i in range(11)]
    want = whole.clone()
    for i in range(11):
        want[i % 4, 7, 4 * i:4 * i + 3] = whole[i % 4, 2, 4 * i:4 * i + 3]
    ops.copy_pages(planes, [2], [7])
    assert torch.equal(whole, want)
    ops.copy_pages(planes, [], [])
    assert torch.equal(whole, want)


def test_an_output_and_queries_at_odd_addresses():
    batch, tables, pages = step([200, 9, 70], [1, 3, 2], 16)
    for D in (64, 128):
        for dtype in (torch.bfloat16, torch.float32):
            cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
            wide = torch.randn(6, 8 * D + 1, device=DEV).to(dtype)
            q = wide[:, 1:]
            want = ops.attention_cache8(q.contiguous(), cache, batch, 0, 8)
            room = torch.full((6 * 8 * D + 2,), 3.0, dtype=dtype, device=DEV)
            out = room[1:-1].view(6, 8 * D)
            assert ops.attention_cache8(q, cache, batch, 0, 8, out=out) is out and same(out, want) and room[0] == room[-1] == 3.0


@pytest.mark.parametrize("group", [1, 5, 8, 9, 17, 33])
@pytest.mark.parametrize("held", [[0, 15, 16, 33], [130, 700, 1500, 64], [5000, 17, 2049, 4096]])
def test_rows_joined_over_every_number_of_blocks(group, held, monkeypatch):
    """Tiles whose keys 1 to 16 blocks share, with pairs that fill them in part."""
    from hipinfer_b200.kernels import cache8

    batch, tables, pages = step(held, [1] * len(held), 32)
    cache = filled(pages, 2, 32, 64, torch.int8)
    q = torch.randn(len(held), 2 * group * 64, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16)
    for ranks in range(1, 17):
        monkeypatch.setattr(cache8, "_ranks", lambda *a: ranks)
        batch.extra.clear()
        check(q, cache, batch, tables, 2 * group)


# ------------------------------------------------------------------------------------------ calls that differ from an engine's
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 50])
def test_places_that_no_row_of_a_portion_sees_do_not_count(D, window):
    """NaN codes and scales behind a portion's last token and, with a window, ahead of its first key."""
    held, rows, ps = [70, 300, 0], [45, 1, 133], 16
    batch, tables, pages = step(held, rows, ps)
    cache = filled(pages, 2, ps, D, torch.float8_e4m3fn)
    q = torch.randn(sum(rows), 8 * D, generator=torch.Generator().manual_seed(12)).to(torch.bfloat16)
    clean = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 8, window)
    seen = {(t[j // ps], j % ps) for t, h, n in zip(tables, held, rows) for j in range(max(0, h - window + 1) if window else 0, h + n)}
    blocks = {p for p, i in seen}
    for p in range(pages):
        for i in range(ps):
            if (p, i) not in seen:
                cache[0].view(torch.uint8)[p, :, i] = 0x7f
                cache[1].view(torch.uint8)[p, :, i] = 0xff
        if p not in blocks:
            cache[2][p, ::2], cache[3][p, ::2], cache[2][p, 1::2], cache[3][p, 1::2] = float("nan"), float("inf"), float("inf"), float("nan")
    assert same(ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 8, window), clean)


@pytest.mark.parametrize("D", [64, 128])
def test_a_portion_s_rows_with_infinities_and_nan_stay_alone(D):
    batch, tables, pages = step([100, 20], [70, 1], 16)
    q = torch.randn(71, 4 * D, generator=torch.Generator().manual_seed(13)).to(torch.bfloat16)
    cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
    want = ops.attention_cache8(q.to(DEV), cache, batch, 0, 4)
    q[3, 5], q[40, D + 1], q[70, 3 * D] = float("nan"), float("inf"), float("-inf")
    got = ops.attention_cache8(q.to(DEV), cache, batch, 0, 4)
    bad = torch.zeros(71, 4, dtype=torch.bool)
    bad[3, 0] = bad[40, 1] = bad[70, 3] = True
    assert torch.equal(got.view(71, 4, D).isnan().all(-1).cpu(), bad) and same(got.view(71, 4, D)[~bad.to(DEV)], want.view(71, 4, D)[~bad.to(DEV)])


@pytest.mark.parametrize("rows", [[1, 0, 1], [0, 1, 1], [0, 0, 0], [0, 3, 0, 1], [0, 40, 1], [40, 0, 0], [17] + [0] * 16])
@pytest.mark.parametrize("D", [64, 128, 72])
def test_requests_without_a_row(rows, D):
    held = [37 + 5 * i for i in range(len(rows))]
    batch, tables, pages = step(held, rows, 16)
    q = torch.randn(sum(rows), 8 * D, generator=torch.Generator().manual_seed(14)).to(torch.bfloat16)
    cache = filled(pages, 2, 16, D, torch.int8)
    if sum(rows):
        check(q, cache, batch, tables, 8)
    else:
        assert ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 8).shape == (0, 8 * D)


@pytest.mark.parametrize("rows", [[1, 1, 1], [2, 1, 5], [1, 90, 3]])
def test_a_batch_on_several_streams_at_once(rows):
    batch, tables, pages = step([400, 21, 1300], rows, 16)
    cache = on_gpu(filled(pages, 2, 16, 64, torch.int8))
    q = torch.randn(sum(rows), 512, device=DEV).to(torch.bfloat16)
    want = ops.attention_cache8(q, cache, step([400, 21, 1300], rows, 16)[0], 0, 8)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for s in streams:                                            # none waits for another
        with torch.cuda.stream(s):
            got += [ops.attention_cache8(q, cache, batch, 0, 8) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(same(x, want) for x in got)


@pytest.mark.parametrize("rows", [[2, 1, 5], [1, 90, 3], [64, 64, 200]])
def test_a_step_of_several_rows_is_captured_after_a_run(rows):
    batch, tables, pages = step([400, 21, 1300], rows, 16)
    cache = on_gpu(filled(pages, 2, 16, 64, torch.int8))
    q = torch.randn(sum(rows), 512, device=DEV).to(torch.bfloat16)
    with pytest.raises(ops.KernelError, match="once before it is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.attention_cache8(q, cache, batch, 0, 8)
    ops.attention_cache8(q, cache, batch, 0, 8)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.attention_cache8(q, cache, batch, 0, 8)))
    fresh = torch.randn_like(q)
    q.copy_(fresh)
    want = ops.attention_cache8(fresh, cache, step([400, 21, 1300], rows, 16)[0], 0, 8)
    for graph, out in graphs + graphs:
        graph.replay()
        assert same(out, want)
        out.zero_()


def test_a_copy_of_a_cache_has_its_own_memory():
    import copy
    cache = on_gpu(filled(5, 2, 16, 64, torch.int8))
    other = copy.deepcopy(cache)
    before = [t.clone() for t in cache.tensors]
    x = torch.randn(1, 128, device=DEV)
    ops.store_cache8(x, x, torch.tensor([16], dtype=torch.int32, device=DEV), other)
    torch.cuda.synchronize()
    assert all(same(a, b) for a, b in zip(cache.tensors, before)) and not same(other.k, cache.k)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(copy.copy(cache).tensors, cache.tensors))


def test_pages_of_an_empty_cache_are_zeros():
    cache = on_gpu(filled(0, 2, 16, 64, torch.int8))
    k, v = ops.expand_cache8(cache, torch.tensor([0, -1, 3], dtype=torch.int32, device=DEV))
    assert k.shape == v.shape == (3, 2, 16, 64) and not k.any() and not v.any()


def test_places_of_rows_are_not_made_while_a_graph_is_captured():
    ops.row_places(DEV, 1)
    n = max(t.numel() for t in cache8._rows[DEV]) + 1
    with pytest.raises(ops.KernelError, match="before it is captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.row_places(DEV, n)
    assert ops.row_places(DEV, n).tolist() == list(range(n))


@pytest.mark.parametrize("rows", [1, 16, 17, 33])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_blocks_with_numbers_that_are_not_finite_among_others(rows, dtype, codes):
    """Infinities, NaN and the type's largest numbers in rows at odd places, over blocks that hold larger numbers already."""
    heads, ps, D, pages = 2, 32, 128, 3
    cache = filled(pages, heads, ps, D, codes)
    g = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(rows, heads * D, generator=g).to(dtype) for _ in range(2))
    for t, x in ((k, float("inf")), (v, float("-inf")), (k, float("nan")), (v, float("nan"))):
        t.view(-1)[torch.randperm(t.numel(), generator=g)[:9]] = x
    if rows > 16:
        v[16, 3:9] = torch.finfo(dtype).max
    slots = [(7 + i) % (pages * ps) for i in range(rows)]
    got = on_gpu(cache)
    ops.store_cache8(k.to(DEV), v.to(DEV), torch.tensor(slots, dtype=torch.int32, device=DEV), got)
    for x, c, s, gc, gs in ((k, cache[0], cache[2], got.k, got.k_scale), (v, cache[1], cache[3], got.v, got.v_scale)):
        wc, ws = plain.store(x, slots, c, s)
        assert same(gs, ws) and same(gc, wc)


@pytest.mark.parametrize("rows", [[1, 1], [3, 1], [40, 1], [600, 1]])
@pytest.mark.parametrize("D", [64, 128, 80])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=ids)
def test_blocks_of_zeros_among_others(rows, D, dtype):
    """Values of all-zero blocks as storing leaves them (scale 1e-30 / M), blocks that nothing was stored to (scale 0), and tiny ones, in turn."""
    batch, tables, pages = step([900, 333], rows, 16)
    k, v, ks, vs = filled(pages, 2, 16, D, torch.int8)
    for at, scale in ((0, 1e-30 / 127), (2, 0.0), (3, 1e-20), (5, 1e-12)):
        vs[at::7] = scale
    v[0::7] = v[2::7] = 0
    q = torch.randn(sum(rows), 8 * D, generator=torch.Generator().manual_seed(15)).to(dtype)
    check(q, (k, v, ks, vs), batch, tables, 8)
    vs *= 1e-9
    check(q, (k, v, ks, vs), batch, tables, 8)


@pytest.mark.parametrize("rows", [[1, 1], [3, 1], [40, 1]])
@pytest.mark.parametrize("D", [64, 80])
def test_an_empty_cache_gives_zeros(rows, D):
    batch, _, _ = step([900, 333], rows, 16)
    q = torch.randn(sum(rows), 8 * D, device=DEV).to(torch.bfloat16)
    out = torch.ones_like(q)
    assert not ops.attention_cache8(q, on_gpu(filled(0, 2, 16, D, torch.int8)), batch, 0, 8, out=out).any()


@pytest.mark.parametrize("rows", [[1, 1], [5, 2], [300, 1]])
@pytest.mark.parametrize("D, ps", [(128, 16), (96, 16)])
def test_pages_beyond_32_bits_of_bytes(rows, D, ps):
    """The same pages at the end of a cache whose codes take more than 2^32 bytes: the same bits."""
    heads, dtype = 8, torch.int8
    batch, tables, pages = step([200, 41], rows, ps)
    small = on_gpu(filled(pages, heads, ps, D, dtype))
    n = 2 ** 32 // (heads * ps * D) + pages + 3
    big = ops.new_cache8(n, heads, ps, D, dtype, DEV)
    for a, b in zip(big.tensors, small.tensors):
        a[n - pages:].copy_(b)
    q = torch.randn(sum(rows), 32 * D, device=DEV).to(torch.bfloat16)
    want = ops.attention_cache8(q, small, batch, 0, 32)
    x = torch.randn(7, heads * D, device=DEV).to(torch.bfloat16)
    slots = torch.arange(3 * ps + 11, 3 * ps + 18, dtype=torch.int32, device=DEV) % (pages * ps)
    ops.store_cache8(x, x, slots, small)
    after = ops.attention_cache8(q, small, batch, 0, 32)
    high = step([200, 41], rows, ps)[0]
    high.block_tables[0] += (high.block_tables[0] >= 0) * (n - pages)
    assert same(ops.attention_cache8(q, big, high, 0, 32), want)
    ops.store_cache8(x, x, slots + (n - pages) * ps, big)
    assert same(ops.attention_cache8(q, big, high, 0, 32), after)
    which = torch.arange(pages, dtype=torch.int32, device=DEV)
    for a, b in zip(ops.expand_cache8(big, which + (n - pages)), ops.expand_cache8(small, which)):
        assert same(a, b)
    ops.copy_pages([t[None] for t in big.tensors], list(range(n - pages, n)), list(range(1, pages + 1)))
    assert all(same(a[1:pages + 1], b) for a, b in zip(big.tensors, small.tensors))


@pytest.mark.parametrize("rows", [[1, 1], [5, 2], [300, 1], [300, 200]])
@pytest.mark.parametrize("window", [0, 100])
def test_calls_through_the_interpreter_give_the_same_bits(rows, window, monkeypatch):
    """Without the binding in C++: every operator, the same launches."""
    from hipinfer_b200.kernels import library

    batch, tables, pages = step([200, 41], rows, 16, window)
    start = filled(pages, 2, 16, 128, torch.int8)
    g = torch.Generator().manual_seed(16)
    q, k = torch.randn(sum(rows), 8 * 128, generator=g).to(torch.bfloat16).to(DEV), torch.randn(9, 256, generator=g).to(torch.bfloat16).to(DEV)
    slots = torch.arange(18, 27, dtype=torch.int32, device=DEV)

    def run():
        cache, before = on_gpu(start), library.launches[0]
        attended = ops.attention_cache8(q, cache, batch, 0, 8, window)
        ops.store_cache8(k, k, slots, cache)
        read = ops.expand_cache8(cache, torch.arange(pages, dtype=torch.int32, device=DEV))
        ops.copy_pages([t[None] for t in cache.tensors], [0], [1])
        return [attended, *read, *cache.tensors], library.launches[0] - before

    bound, launches = run()
    monkeypatch.setattr(cache8, "_bound", False)
    plainly, as_many = run()
    assert all(same(a, b) for a, b in zip(bound, plainly)) and launches == as_many


@pytest.mark.parametrize("D", [64, 128])
def test_portions_of_wider_rows_and_at_odd_addresses(D):
    rows, held = [300, 1, 40], [50, 100, 7]
    batch, tables, pages = step(held, rows, 16)
    cache = filled(pages, 2, 16, D, torch.int8)
    q = torch.randn(sum(rows), 8 * D, generator=torch.Generator().manual_seed(17)).to(torch.bfloat16)
    want = check(q, cache, batch, tables, 8)
    wide = torch.zeros(sum(rows), 8 * D + 3, dtype=torch.bfloat16, device=DEV)
    wide[:, 2:-1] = q.to(DEV)
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(q.shape).copy_(q)
    room = torch.full((q.numel() + 2,), 3.0, dtype=torch.bfloat16, device=DEV)
    out = room[1:-1].view(q.shape)
    for x, to in ((wide[:, 2:-1], None), (odd, None), (q.to(DEV), out)):
        got = ops.attention_cache8(x, on_gpu(cache), batch, 0, 8, out=to)
        V = float(np.abs(plain.numbers(cache[1], cache[3])).max())
        assert (got.float() - want.float()).abs().max() <= V * 2.0 ** -7 * 8        # (each within 2^-8 (2 + A) V of the exact one, A below 6)
    assert room[0] == room[-1] == 3.0
