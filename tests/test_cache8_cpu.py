"""What the operators of a cache in 8 bits refuse, on the host: before anything is launched."""
import numpy as np
import pytest
import torch

from hipinfer_b200.engine.batch import StepEntry, build_step_batch
from hipinfer_b200.kernels import cache8, ops

CACHE = dict(pages=4, n_kv_heads=2, page_size=16, head_dim=64, device="cpu")


@pytest.fixture
def calls(monkeypatch):
    """The launches, with tensors of the host let through."""
    made = []
    monkeypatch.setattr(cache8, "_here", lambda what, *t: None)
    monkeypatch.setattr(ops, "_call", lambda lib, name, *a: made.append((name, a)))
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    return made


def batch_of(held, rows, ps=16):
    tables = [[list(range(-(-(h + n) // ps)))] for h, n in zip(held, rows)]
    return build_step_batch([StepEntry(i, [0] * n) for i, n in enumerate(rows)], held, list(range(len(rows))), tables, [[[0] * n] for n in rows], 1, "cpu")


def test_without_a_gpu_there_is_no_implementation():
    cache = ops.new_cache8(**CACHE)
    rows, slots = torch.zeros(1, 128), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.store_cache8(rows, rows, slots, cache), lambda: ops.expand_cache8(cache, slots),
                 lambda: ops.attention_cache8(torch.zeros(1, 256), cache, batch_of([3], [1]), 0, 4), lambda: ops.copy_pages([cache.k[None]], [0], [1])):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()


def test_tensors_on_another_device_than_the_current_one(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)

    class Elsewhere:
        is_cuda, device = True, torch.device("cuda:1")

    with pytest.raises(ops.KernelError, match="the current device is cuda:0"):
        cache8._here("x", Elsewhere())


@pytest.mark.parametrize("change", [dict(k=torch.zeros(4, 2, 16, 64)), dict(v=torch.zeros(4, 2, 16, 32, dtype=torch.int8)),
                                    dict(v=torch.zeros(4, 2, 16, 64, dtype=torch.uint8)), dict(k=torch.zeros(4, 2, 64, 16, dtype=torch.int8).transpose(2, 3)),
                                    dict(k_scale=torch.zeros(4, 2, 2)), dict(v_scale=torch.zeros(4, 2, 1, dtype=torch.float64)),
                                    dict(k_scale=torch.zeros(4, 2, 2)[:, :, :1])])
def test_a_cache_of_other_parts(change):
    c = ops.new_cache8(**CACHE)
    parts = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale)
    assert ops.Cache8(**parts).code == 2
    with pytest.raises(ops.KernelError):
        ops.Cache8(**{**parts, **change})


@pytest.mark.parametrize("change", [dict(pages=0), dict(page_size=0), dict(head_dim=0), dict(dtype=torch.bfloat16), dict(n_kv_heads=-1)])
def test_a_new_cache_of_no_size(change):
    with pytest.raises(ops.KernelError):
        ops.new_cache8(**{**CACHE, **change})


def test_blocks_of_a_page():
    assert [ops.cache8_blocks(n) for n in (1, 8, 16, 24, 32, 64)] == [1, 1, 1, 2, 2, 4]
    c = ops.new_cache8(3, 2, 24, 5, torch.float8_e4m3fn, "cpu")
    assert c.k_scale.shape == (3, 2, 2) and c.k.dtype == torch.float8_e4m3fn and not c.k.float().any()


def test_storing_refuses(calls):
    cache = ops.new_cache8(**CACHE)
    rows, slots = torch.zeros(3, 128), torch.zeros(3, dtype=torch.int32)
    ops.store_cache8(rows, rows, slots, cache)
    ops.store_cache8(rows[:0], rows[:0], slots[:0], cache)
    assert [n for n, _ in calls] == ["hb_cache8_store"]
    for k, v, s in ((rows, rows[:2], slots), (rows[:, :127], rows[:, :127], slots), (rows.half(), rows.half(), slots), (rows, rows.bfloat16(), slots),
                    (rows, rows, slots[:2]), (rows, rows, slots.long()), (rows.view(3, 2, 64), rows, slots),
                    (torch.zeros(128, 3).t(), rows, slots), (rows, rows, torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ops.KernelError):
            ops.store_cache8(k, v, s, cache)
    assert len(calls) == 1


def test_reading_back_refuses(calls):
    cache, pages = ops.new_cache8(**CACHE), torch.zeros(3, dtype=torch.int32)
    assert ops.expand_cache8(cache, pages)[0].shape == (3, 2, 16, 64) and len(calls) == 1
    assert ops.expand_cache8(cache, pages[:0])[1].shape == (0, 2, 16, 64) and len(calls) == 1
    for p, t in ((pages.long(), torch.float32), (pages[None], torch.float32), (pages, torch.float16)):
        with pytest.raises(ops.KernelError):
            ops.expand_cache8(cache, p, t)
    assert len(calls) == 1


def test_attention_refuses(calls):
    cache, batch = ops.new_cache8(**CACHE), batch_of([5, 20], [1, 2])
    q = torch.zeros(3, 4 * 64)
    assert ops.attention_cache8(q, cache, batch, 0, 4).shape == (3, 256) and len(calls) == 1
    for x, heads, kw in ((q, 3, {}), (q, 0, {}), (q[:2], 4, {}), (q.half(), 4, {}), (torch.zeros(256, 3).t(), 4, {}), (q, 4, dict(window=-1)),
                         (q, 4, dict(out=torch.zeros(3, 128))), (q, 4, dict(out=torch.zeros(3, 256, dtype=torch.bfloat16))),
                         (q, 4, dict(out=torch.zeros(3, 512)[:, ::2]))):
        with pytest.raises(ops.KernelError):
            ops.attention_cache8(x, cache, batch, 0, heads, **kw)
    short = batch_of([5, 20], [1, 2])
    short.block_tables[0] = short.block_tables[0][:, :1].contiguous()                     # (23 tokens in one page of 16)
    with pytest.raises(ops.KernelError, match="up to 22 tokens"):
        ops.attention_cache8(q, cache, short, 0, 4)
    batch.block_tables[0] = batch.block_tables[0].long()
    with pytest.raises(ops.KernelError):
        ops.attention_cache8(q, cache, batch, 0, 4)
    wide = ops.new_cache8(1, 1, 16, 257, device="cpu")
    with pytest.raises(ops.KernelError, match="at most 256"):
        ops.attention_cache8(torch.zeros(1, 257), wide, batch_of([3], [1]), 0, 1)
    assert len(calls) == 1


def test_copying_refuses(calls):
    plane = torch.zeros(2, 6, 3, 4)
    ops.copy_pages([plane, plane[:, :, :1]], [0, 0], [4, 5])
    assert len(calls) == 1
    for src, dst in (([0], [6]), ([6], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]), ([0, 1], [2]), ([[0]], [[1]])):
        with pytest.raises(ops.KernelError):
            ops.copy_pages([plane], src, dst)
    for bad in (torch.zeros(6), torch.zeros(2, 6, 4, 3).transpose(2, 3), torch.zeros(1, 6, 3).expand(2, 6, 3), torch.zeros(2, 1, 3).expand(2, 6, 3)):
        with pytest.raises(ops.KernelError):
            ops.copy_pages([plane, bad], [0], [1])
    ops.copy_pages([], [0], [1])
    ops.copy_pages([plane], [], [])
    ops.copy_pages([torch.zeros(0, 6, 3)], [0], [1])
    assert len(calls) == 1
    name, args = calls[0]
    assert name == "hb_copy_pages" and args[1] == 2 and args[4] == 2


def test_a_run_of_the_plain_storing_is_what_its_words_say():
    import plain_cache8 as plain

    codes, scales = torch.zeros(2, 1, 16, 2, dtype=torch.int8), torch.zeros(2, 1, 1)
    codes, scales = plain.store(torch.tensor([[1.0, -127.0], [63.5, 2.5]]), [16, 17], codes, scales)
    assert scales.tolist() == [[[0.0]], [[1.0]]] and codes[1, 0, :2].tolist() == [[1, -127], [64, 2]]
    codes, scales = plain.store(torch.tensor([[254.0, 3.0]]), [18], codes, scales)
    assert scales[1].tolist() == [[2.0]] and codes[1, 0, :3].tolist() == [[0, -64], [32, 1], [127, 2]]
    assert np.isfinite(plain.numbers(codes, scales)).all()


@pytest.mark.parametrize("change", [dict(positions=torch.zeros(3, dtype=torch.int64)), dict(positions=torch.zeros(2, dtype=torch.int32)),
                                    dict(row_request=torch.zeros(3, 1, dtype=torch.int32)), dict(positions=torch.zeros(6, dtype=torch.int32)[::2])])
def test_attention_refuses_rows_places_of_another_form(calls, change):
    cache, batch = ops.new_cache8(**CACHE), batch_of([5, 20], [1, 2])
    for name, x in change.items():
        setattr(batch, name, x)
    with pytest.raises(ops.KernelError, match=next(iter(change))):
        ops.attention_cache8(torch.zeros(3, 256), cache, batch, 0, 4)
    assert not calls


@pytest.mark.parametrize("window", [-1, 2 ** 31, 2 ** 32 + 5])
def test_attention_refuses_windows_of_more_than_31_bits(calls, window):
    with pytest.raises(ops.KernelError, match="window"):
        ops.attention_cache8(torch.zeros(3, 256), ops.new_cache8(**CACHE), batch_of([5, 20], [1, 2]), 0, 4, window)
    assert not calls


def test_a_copy_of_a_cache_names_its_own_tensors():
    import copy
    import pickle

    cache = ops.new_cache8(**CACHE)
    for other in (copy.deepcopy(cache), pickle.loads(pickle.dumps(cache))):
        assert [int(x) for x in other._native[:4]] == [t.data_ptr() for t in other.tensors] and other.native != cache.native
        assert all(a.data_ptr() != b.data_ptr() for a, b in zip(other.tensors, cache.tensors))


@pytest.mark.parametrize("rows", [[0, 20, 1], [0, 0, 17, 300], [16]])
def test_pages_of_portions_pass_requests_without_rows_over(rows):
    batch = batch_of([40] * len(rows), rows)
    index, places, base = cache8._pages_of_portions(batch, 16, batch.block_tables[0].shape[1], 0, 16)
    assert index.numel() == sum(-(-(40 + n) // 16) for n in rows if n >= 16)
    for r, n in enumerate(rows):
        assert int((places[r] >= 0).sum()) == (-(-(40 + n) // 16) if n >= 16 else 0)
