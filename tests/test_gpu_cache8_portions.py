"""Portions over a cache in 8 bits on the flash kernel: the limit from which on a request's rows go there is set by the tests, and every call asserts that it
was launched. Bounds: tests/cache8_bounds.py."""
import pytest
import torch

import cache8_bounds as bounds
from hipinfer_b200.engine.batch import StepEntry, build_step_batch
from hipinfer_b200.kernels import cache8, library, ops
from test_gpu_cache8 import CODES, DEV, filled, ids, on_gpu, same, step

pytestmark = pytest.mark.gpu


@pytest.fixture
def portions(monkeypatch):
    """attention_cache8 with requests of `limit` rows and more on the flash kernel (two launches, and one for other requests' rows)."""
    def attend(q, cache, batch, heads, window=0, scale=None, limit=16, **more):
        monkeypatch.setattr(cache8, "_portion_limit", lambda *a: limit)
        before = library.launches[0]
        got = ops.attention_cache8(q, cache, batch, 0, heads, window=window, scale=scale, **more)
        flash, others = (any(n > 0 and (n >= limit > 0) == there for n in batch.h_q_len) for there in (True, False))
        assert library.launches[0] - before == 2 * flash + others and flash == (limit > 0)
        return got
    return attend


def queries(n, seed=1):
    return torch.randn(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("size", [1e-30, 1e-29, 1.2e-28, 1e-20, 1e20, 1e30])
@pytest.mark.parametrize("codes", CODES, ids=ids)
@pytest.mark.parametrize("D", [64, 128])
def test_values_near_the_least_and_the_largest_numbers(D, codes, size, portions):
    """Blocks as storing leaves them for values of any size: as rows of one token read them."""
    held, rows, ps, heads = [40, 7], [33, 1], 16, 4
    batch, tables, pages = step(held, rows, ps)
    v = (queries(pages * ps * 2 * D, 2) * size).view(pages * ps, 2 * D).to(DEV)
    k = queries(pages * ps * 2 * D, 3).view(pages * ps, 2 * D).to(DEV)
    cache = ops.new_cache8(pages, 2, ps, D, codes, DEV)
    ops.store_cache8(k, v, torch.arange(pages * ps, dtype=torch.int32, device=DEV), cache)
    q = queries(sum(rows) * heads * D).view(-1, heads * D).to(torch.bfloat16)
    want, bound = bounds.attend(q, [t.cpu() for t in cache.tensors], tables, held, rows, heads)
    got = portions(q.to(DEV), cache, batch, heads)
    assert bounds.beyond(got, want, bound) <= 1
    assert float(want.abs().max()) > size / 10


STEPS = {
    "a prompt": ([0], [333]),
    "one tile": ([0], [16]),
    "behind others": ([0, 40, 1000], [70, 33, 129]),
    "mixed": ([37, 0, 250, 9, 0], [65, 17, 1, 15, 256]),
    "long": ([2900, 0], [130, 1]),
}


@pytest.mark.parametrize("name", STEPS)
@pytest.mark.parametrize("heads, kv_heads, ps, D", [(32, 8, 16, 64), (8, 2, 16, 128), (7, 1, 32, 128), (4, 4, 64, 64), (24, 1, 128, 64), (6, 2, 128, 128)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_portions_of_every_kind(name, heads, kv_heads, ps, D, codes, portions):
    held, rows = STEPS[name]
    batch, tables, pages = step(held, rows, ps)
    q, cache = queries(sum(rows) * heads * D).view(-1, heads * D).to(torch.bfloat16), filled(pages, kv_heads, ps, D, codes)
    want, bound = bounds.attend(q, cache, tables, held, rows, heads)
    assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, heads), want, bound) <= 1


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 1000])
@pytest.mark.parametrize("heads, kv_heads, ps, D", [(8, 2, 16, 64), (4, 1, 32, 128), (2, 2, 128, 64)])
@pytest.mark.parametrize("codes", CODES, ids=ids)
def test_a_window(window, heads, kv_heads, ps, D, codes, portions):
    """Pages that no row sees any more have been given back."""
    for name in ("behind others", "mixed"):
        held, rows = STEPS[name]
        batch, tables, pages = step(held, rows, ps, window)
        q, cache = queries(sum(rows) * heads * D, 2).view(-1, heads * D).to(torch.bfloat16), filled(pages, kv_heads, ps, D, codes)
        want, bound = bounds.attend(q, cache, tables, held, rows, heads, window, 0.2)
        assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, heads, window, 0.2), want, bound) <= 1


@pytest.mark.parametrize("limit", cache8.PORTION_ROWS + (0,))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 77])
def test_either_side_of_every_limit(limit, D, window, portions):
    """Requests of as many rows as a limit has, one fewer and one more: whichever kernel they go through."""
    held = [5, 0, 300, 17, 64, 0, 128, 1, 90]
    rows = [15, 16, 31, 32, 63, 64, 127, 128, 1]
    batch, tables, pages = step(held, rows, 16, window)
    q, cache = queries(sum(rows) * 8 * D, 4).view(-1, 8 * D).to(torch.bfloat16), filled(pages, 2, 16, D, torch.int8)
    want, bound = bounds.attend(q, cache, tables, held, rows, 8, window)
    assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, 8, window, limit=limit), want, bound) <= 1


@pytest.mark.parametrize("ps", [16, 32, 128])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_that_are_not_there(ps, D, portions):
    """Numbers outside of the cache in the middle of a portion's keys, at their beginning (rows that see nothing are 0), for a whole request, at a tile's places that
    keys of an item before left something in."""
    held, rows, heads = [600, 0, 40, 0, 513], [70, 300, 33, 40, 20], 4
    batch, tables, pages = step(held, rows, ps)
    table = batch.block_tables[0]
    table[0, 1], table[0, 3], table[1, 0], table[2, :], table[4, 2] = -1, pages + 2, -5, -1, 2 ** 30
    tables = [row.tolist() for row in table.cpu()]
    q, cache = queries(sum(rows) * heads * D, 5).view(-1, heads * D).to(torch.bfloat16), filled(pages, 2, ps, D, torch.float8_e4m3fn)
    want, bound = bounds.attend(q, cache, tables, held, rows, heads)
    got = portions(q.to(DEV), on_gpu(cache), batch, heads)
    assert bounds.beyond(got, want, bound) <= 1
    assert not got[70:70 + min(300, ps)].any() and not got[370:403].any() and got[70 + ps].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("ps", [16, 64])
def test_places_that_no_row_sees_do_not_count(D, window, ps, portions):
    """NaN codes and scales behind a portion's last token and, with a window, ahead of its first key: the same bits."""
    held, rows = [70, 300, 0], [45, 1, 133]
    batch, tables, pages = step(held, rows, ps)
    cache = filled(pages, 2, ps, D, torch.float8_e4m3fn)
    q = queries(sum(rows) * 8 * D, 12).view(-1, 8 * D).to(torch.bfloat16)
    clean = portions(q.to(DEV), on_gpu(cache), batch, 8, window)
    seen = {(t[j // ps], j % ps) for t, h, n in zip(tables, held, rows) for j in range(max(0, h - window + 1) if window else 0, h + n)}
    blocks = {(p, i // 16) for p, i in seen}
    for p in range(pages):
        for i in range(ps):
            if (p, i) not in seen:
                cache[0].view(torch.uint8)[p, :, i] = 0x7f
                cache[1].view(torch.uint8)[p, :, i] = 0xff
        for b in range(ps // 16):
            if (p, b) not in blocks:
                cache[2][p, ::2, b], cache[3][p, ::2, b], cache[2][p, 1::2, b], cache[3][p, 1::2, b] = float("nan"), float("inf"), float("inf"), float("nan")
    got = portions(q.to(DEV), on_gpu(cache), batch, 8, window)
    assert same(got, clean) and torch.isfinite(got.float()).all()


@pytest.mark.parametrize("D", [64, 128])
def test_rows_with_infinities_and_nan_stay_alone(D, portions):
    batch, tables, pages = step([100, 20, 0], [70, 1, 200], 16)
    q = queries(271 * 4 * D, 13).view(-1, 4 * D).to(torch.bfloat16)
    cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
    want = portions(q.to(DEV), cache, batch, 4)
    q[3, 5], q[40, D + 1], q[70, 3 * D], q[271 - 130, 2 * D] = float("nan"), float("inf"), float("-inf"), float("inf")
    got = portions(q.to(DEV), cache, batch, 4)
    bad = torch.zeros(271, 4, dtype=torch.bool)
    bad[3, 0] = bad[40, 1] = bad[70, 3] = bad[141, 2] = True
    assert torch.equal(got.view(271, 4, D).isnan().all(-1).cpu(), bad) and same(got.view(271, 4, D)[~bad.to(DEV)], want.view(271, 4, D)[~bad.to(DEV)])


@pytest.mark.parametrize("D", [64, 128])
def test_blocks_of_unlike_scales(D, portions):
    """Zeros as storing leaves them (scale 1e-30 / M), blocks that nothing was stored to (scale 0), tiny ones and ones of 10^9 in turn."""
    held, rows = [900, 333], [600, 1]
    batch, tables, pages = step(held, rows, 16)
    k, v, ks, vs = filled(pages, 2, 16, D, torch.int8)
    for at, scale in ((0, 1e-30 / 127), (2, 0.0), (3, 1e-20), (5, 1e-12), (6, 1e9)):
        vs[at::7] = scale
        if scale < 1:
            ks[(at + 1) % 7::7] *= 1e-20 if scale else 0.0
    v[0::7] = v[2::7] = 0
    q = queries(sum(rows) * 8 * D, 15).view(-1, 8 * D).to(torch.bfloat16)
    for times in (1.0, 1e-9, 1e-25, 1e20):
        cache = (k, v, ks, vs * times)
        want, bound = bounds.attend(q, cache, tables, held, rows, 8)
        assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, 8), want, bound) <= 1


@pytest.mark.parametrize("scale", [1e-30, 1e-5, 1.0, 30.0])
@pytest.mark.parametrize("D", [64, 128])
def test_softmax_scales(scale, D, portions):
    """From weights that are all alike to rows one of whose keys has nearly all of it."""
    held, rows = [100, 0], [40, 200]
    batch, tables, pages = step(held, rows, 16)
    q = queries(sum(rows) * 8 * D, 6).view(-1, 8 * D).to(torch.bfloat16)
    cache = filled(pages, 2, 16, D, torch.int8)
    cache[2][:, :, :] *= 1e-3 if scale > 1 else 1.0
    want, bound = bounds.attend(q, cache, tables, held, rows, 8, 0, scale)
    assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, 8, 0, scale), want, bound) <= 1


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("ps", [16, 32])
@pytest.mark.parametrize("window", [0, 2000])
def test_every_key_of_a_long_range_counts_once(D, ps, window, portions):
    """Scores that are all alike, and key j the value 1 in dimension j mod D alone: a result is how many of the keys that its row sees have that dimension, over their number."""
    held, rows, heads = [3000, 4975], [200, 25], 2
    batch, tables, pages = step(held, rows, ps, window)
    k, v, ks, vs = filled(pages, 1, ps, D, torch.int8)
    v.zero_()
    for t, h, n in zip(tables, held, rows):
        for j in range(max(0, h - window + 1) if window else 0, h + n):
            v[t[j // ps], 0, j % ps, j % D] = 64
    vs[:] = 1 / 64
    got = portions(torch.zeros(sum(rows), heads * D, dtype=torch.bfloat16, device=DEV), on_gpu((k, v, ks, vs)), batch, heads, window).double().cpu().view(-1, heads, D)
    at = 0
    for h, n in zip(held, rows):
        for p in range(h, h + n):
            lo = max(0, p - window + 1) if window else 0
            count = torch.bincount(torch.arange(lo, p + 1) % D, minlength=D).double()
            # (of up to 79 keys: off by 2^-8 of that for the result's rounding and nothing else, weights of one power of two being exact)
            assert ((got[at] * (p + 1 - lo) - count).abs() < 0.5).all()
            at += 1


def test_the_interpreter_s_call_has_the_same_bits(portions, monkeypatch):
    for D in (64, 128):
        for window in (0, 100):
            batch, tables, pages = step([200, 41, 0], [300, 3, 20], 16, window)
            cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
            q = queries(323 * 8 * D, 16).view(-1, 8 * D).to(torch.bfloat16).to(DEV)
            want = portions(q, cache, batch, 8, window)
            out = torch.zeros_like(q)
            with monkeypatch.context() as m:
                m.setattr(cache8, "_bound", False)
                assert same(portions(q, cache, batch, 8, window), want)
                assert portions(q, cache, batch, 8, window, out=out) is out and same(out, want)
            out.zero_()
            assert portions(q, cache, batch, 8, window, out=out) is out and same(out, want)


def test_streams_and_graphs(portions):
    """The same batch on several streams at once, and captured twice after a run: the same bits."""
    rows, held = [64, 1, 200], [400, 21, 1300]
    batch, tables, pages = step(held, rows, 16)
    for D in (64, 128):
        cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
        q = queries(265 * 8 * D, 17).view(-1, 8 * D).to(torch.bfloat16).to(DEV)
        with pytest.raises(ops.KernelError, match="once before it is captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                portions(q, cache, step(held, rows, 16)[0], 8)
        want = portions(q, cache, batch, 8)
        streams = [torch.cuda.Stream() for _ in range(4)]
        torch.cuda.synchronize()
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got += [portions(q, cache, batch, 8) for _ in range(3)]
        torch.cuda.synchronize()
        assert all(same(x, want) for x in got)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, portions(q, cache, batch, 8)))
        fresh = torch.randn_like(q)
        q.copy_(fresh)
        want = portions(fresh, cache, step(held, rows, 16)[0], 8)
        for graph, out in graphs + graphs:
            graph.replay()
            assert same(out, want)
            out.zero_()


@pytest.mark.parametrize("rows", [[0, 40, 1], [40, 0, 0], [17] + [0] * 16, [0, 0, 16]])
@pytest.mark.parametrize("D", [64, 128])
def test_requests_without_a_row(rows, D, portions):
    held = [37 + 5 * i for i in range(len(rows))]
    batch, tables, pages = step(held, rows, 16)
    q, cache = queries(sum(rows) * 8 * D, 14).view(-1, 8 * D).to(torch.bfloat16), filled(pages, 2, 16, D, torch.int8)
    want, bound = bounds.attend(q, cache, tables, held, rows, 8)
    assert bounds.beyond(portions(q.to(DEV), on_gpu(cache), batch, 8), want, bound) <= 1


@pytest.mark.parametrize("D", [64, 128])
def test_rows_behind_the_last_request_s_and_memory_around_them_stay(D, portions):
    batch, tables, pages = step([100, 20], [70, 33], 16)
    cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
    q = queries(103 * 4 * D, 18).view(-1, 4 * D).to(torch.bfloat16).to(DEV)
    room = torch.full((103 * 4 * D + 64,), 3.0, dtype=torch.bfloat16, device=DEV)
    out = room[8:-56].view(103, 4 * D)
    before = [t.clone() for t in cache.tensors]
    assert same(portions(q, cache, batch, 4, out=out), portions(q, cache, batch, 4)) and bool((room[:8] == 3).all()) and bool((room[-56:] == 3).all())
    assert all(same(a, b) for a, b in zip(before, cache.tensors))


@pytest.mark.parametrize("D", [64, 128])
def test_portions_over_pages_beyond_32_bits_of_bytes(D, portions):
    heads, ps = 8, 16
    batch, tables, pages = step([200, 41], [300, 17], ps)
    small = on_gpu(filled(pages, heads, ps, D, torch.int8))
    n = 2 ** 32 // (heads * ps * D) + pages + 3
    big = ops.new_cache8(n, heads, ps, D, torch.int8, DEV)
    for a, b in zip(big.tensors, small.tensors):
        a[n - pages:].copy_(b)
    q = queries(317 * 32 * D, 19).view(-1, 32 * D).to(torch.bfloat16).to(DEV)
    high = step([200, 41], [300, 17], ps)[0]
    high.block_tables[0] += (high.block_tables[0] >= 0) * (n - pages)
    assert same(portions(q, big, high, 32), portions(q, small, batch, 32))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 100])
def test_portions_that_are_expanded_some_at_a_time(D, window, monkeypatch):
    """The same bits, whatever part of them is expanded together, with the binding and without, captured too; memory for one part."""
    monkeypatch.setattr(cache8, "_portion_limit", lambda *a: 16)
    held, rows, heads = [0, 300, 40, 1000, 7, 100, 160], [16, 30, 1, 333, 0, 20, 15], 8
    batch, tables, pages = step(held, rows, 16, window)
    cache = on_gpu(filled(pages, 2, 16, D, torch.int8))
    q = queries(sum(rows) * heads * D, 20).view(-1, heads * D).to(torch.bfloat16).to(DEV)
    want = ops.attention_cache8(q, cache, batch, 0, heads, window=window)
    for most, groups in ((1, 4), (25, 3), (100, 1 if window else 2)):
        monkeypatch.setattr(cache8, "PORTION_BYTES", most * 4 * 2 * 16 * D)
        assert len(cache8._portion_groups(batch, cache, window, 16)) == groups
        for bound in (cache8._bound, False):
            with monkeypatch.context() as m:
                m.setattr(cache8, "_bound", bound)
                before, out = library.launches[0], torch.full_like(want, 7.0)
                assert same(ops.attention_cache8(q, cache, batch, 0, heads, window=window), want) and library.launches[0] - before == 1 + 2 * groups
                assert ops.attention_cache8(q, cache, batch, 0, heads, window=window, out=out) is out and same(out, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attention_cache8(q, cache, batch, 0, heads, window=window)
        out.zero_()
        graph.replay()
        assert same(out, want)


def test_the_memory_of_many_long_portions(monkeypatch):
    """Six portions behind 20,000 tokens: no more than the bound and one request's beside the output."""
    monkeypatch.setattr(cache8, "_portion_limit", lambda *a: 16)
    monkeypatch.setattr(cache8, "PORTION_BYTES", 1 << 24)
    held, rows, D = [20000] * 6, [16] * 6, 128
    batch, tables, pages = step(held, rows, 16)
    cache = on_gpu(filled(pages, 1, 16, D, torch.int8))
    q = queries(96 * 2 * D, 21).view(-1, 2 * D).to(torch.bfloat16).to(DEV)
    ops.attention_cache8(q, cache, batch, 0, 2)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.attention_cache8(q, cache, batch, 0, 2)
    one = 20016 * D * 4                                            # keys and values of a request in 16 bits; scales are a 32nd
    assert one < torch.cuda.max_memory_allocated() - before < (1 << 24) * 1.1 + (1 << 21)


def test_more_requests_than_a_flash_launch_has(monkeypatch):
    """65,540 requests of a token each and a portion among them: the portion stays with the others' kernel, whose tiles are more than a launch has."""
    monkeypatch.setattr(cache8, "_portion_limit", lambda *a: 16)
    R, D, at = 65540, 64, 65537
    rows = [1] * R
    rows[at] = 40
    tables = [[[r]] for r in range(R)]
    tables[at] = [[at, R, R + 1]]
    batch = build_step_batch([StepEntry(r, [0] * n) for r, n in enumerate(rows)], [0] * R, [0] * R, tables, [[[0] * n] for n in rows], 1, DEV)
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(-127, 128, (2, R + 2, 1, 16, D), dtype=torch.int8, generator=g)
    scales = torch.rand(2, R + 2, 1, 1, generator=g) * 0.02 + 0.01
    cache = (codes[0], codes[1], scales[0], scales[1])
    q = queries(batch.n_rows * D, 22).view(-1, D).to(torch.bfloat16)
    before = library.launches[0]
    got = ops.attention_cache8(q.to(DEV), on_gpu(cache), batch, 0, 1).cpu()
    assert library.launches[0] - before == 1
    single = torch.cat([got[:at], got[at + 40:]]).double()
    want = (codes[1].double() * scales[1].double()[..., None])[:R, 0, 0]
    want = torch.cat([want[:at], want[at + 1:]])
    assert ((single - want).abs() <= want.abs() * 2.0 ** -7).all()              # (2^-8 for the result, less for the weight)
    portion, bound = bounds.attend(q[at:at + 40], cache, [tables[at][0]], [0], [40], 1)
    assert bounds.beyond(got[at:at + 40], portion, bound) <= 1
