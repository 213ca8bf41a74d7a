"""The cache in 8 bits as the engine keeps it, and forks at any length: bookkeeping and refusals. No GPU."""
import pytest
import torch

import tiny
from hipinfer_b200.cache import CacheError, CacheGroupSpec, CacheManager, CacheStorage, OutOfPages, OutOfStateSlots
from hipinfer_b200.config import config_from_dict, get_architecture
from hipinfer_b200.engine.runner import cache8_dtype, check_cache8
from hipinfer_b200.kernels import ops
from hipinfer_b200.models.decoder import DecoderModel, StepCachePlan
from hipinfer_b200.parts.registry import BuildContext

FULL = CacheGroupSpec("full", "full", n_layers=2, kv_heads=2, head_dim=16)
WIN = CacheGroupSpec("win", "window", n_layers=1, kv_heads=1, head_dim=32, window=40)


def test_a_fork_at_any_length_gets_the_last_page_for_itself():
    cm = CacheManager([FULL], 16, 12, 5)
    cm.add_request("a")
    cm.append("a", 37)
    b = cm.fork("a", "b", 37)
    assert b.length == 37 and cm.block_table("b", 0) == [0, 1, 3] and b.copied == [(2, 3)]
    c = cm.fork("a", "c", 20)
    assert c.length == 20 and cm.block_table("c", 0) == [0, 4] and c.copied == [(1, 4)]
    d = cm.fork("b", "d", 32)
    assert d.length == 32 and cm.block_table("d", 0) == [0, 1] and d.copied == [None]
    e = cm.fork("a", "e", 0)
    assert e.length == 0 and cm.block_table("e", 0) == [] and e.copied == [None]
    cm.check()
    assert cm.append("b", 2) == [[53, 54]] and cm.append("a", 1) == [[37]]
    for r in "abcde":
        cm.free_request(r)
        cm.check()
    assert cm.free_pages() == [12]


def test_a_fork_at_any_length_refuses_and_leaves_everything_as_it_was():
    cm = CacheManager([FULL], 16, 3, 3)
    cm.add_request("a")
    cm.append("a", 37)
    with pytest.raises(OutOfPages):
        cm.fork("a", "b", 37)
    assert not cm.has_request("b") and cm.slots.free_count == 2 and cm.free_pages() == [0]
    assert cm.fork("a", "b", 32).length == 32
    for length in (-1, 38):
        with pytest.raises(CacheError):
            cm.fork("a", "c", length)
    with pytest.raises(CacheError):
        cm.fork("a", "b", 16)
    cm.fork("a", "c", 16)
    with pytest.raises(OutOfStateSlots):
        cm.fork("a", "d", 16)
    cm.check()


def test_a_fork_inside_a_page_of_a_window():
    cm = CacheManager([FULL, WIN], 16, 10, 4)
    cm.add_request("a")
    cm.append("a", 100)
    cm.release_behind_window("a")
    with pytest.raises(CacheError, match="gone"):
        cm.fork("a", "b", 50)
    b = cm.fork("a", "b", 100)
    assert b.copied[0] is not None and b.copied[1] is not None and cm.block_table("b", 1)[:3] == [-1, -1, -1]
    cm.check()


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("page_size, blocks", [(16, 1), (32, 2), (8, 1), (24, 2)])
def test_the_planes_of_a_layer(dtype, page_size, blocks):
    s = CacheStorage([FULL], [5], page_size, torch.bfloat16, "cpu", {}, 1, dtype)
    assert {n: (tuple(t.shape), t.dtype) for n, t in s.kv[0].items()} == {
        **{n: ((2, 5, 2, page_size, 16), dtype) for n in "kv"}, **{f"{n}_scale": ((2, 5, 2, blocks), torch.float32) for n in "kv"}}
    layer = s.layer_cache(StepCachePlan(0, 1, True))
    assert isinstance(layer.cache8, ops.Cache8) and layer.cache8.k.data_ptr() == s.kv[0]["k"][1].data_ptr() and layer is s.layer_cache(StepCachePlan(0, 1, True))
    page = 2 * 2 * 2 * (page_size * 16 + 4 * blocks)                   # layers, planes, heads
    assert s.bytes_per_token() == -(-page // page_size) and s.nbytes() == 5 * page
    assert CacheStorage([FULL], [5], page_size, torch.bfloat16, "cpu", {}, 1).layer_cache(StepCachePlan(0, 0, True)).cache8 is None


def test_planes_that_are_no_keys_and_values_of_one_shape():
    for planes in ((("latent", 1, 64),), (("k", 1, 64), ("v", 1, 32))):
        with pytest.raises(ValueError, match="8 bits"):
            CacheStorage([CacheGroupSpec("g", "full", 1, planes=planes)], [2], 16, torch.bfloat16, "cpu", {}, 1, torch.int8)


def test_names_of_the_codes():
    assert cache8_dtype(None) is None and cache8_dtype("int8") is torch.int8
    assert cache8_dtype("fp8") is cache8_dtype("float8_e4m3fn") is cache8_dtype(torch.float8_e4m3fn) is torch.float8_e4m3fn
    for name in ("int4", "bfloat16", torch.bfloat16, ""):
        with pytest.raises(ValueError):
            cache8_dtype(name)


def test_models_whose_layers_keep_something_else_are_refused():
    import torirax_models as tm

    def model(cfg):
        cfg = config_from_dict(cfg)
        return DecoderModel(get_architecture(cfg.architecture).build_spec(cfg), BuildContext.meta())

    check_cache8(model(tiny.TINY_A))
    with pytest.raises(ValueError, match="8 bits"):
        check_cache8(model(tm.P))
    with pytest.raises(ValueError, match="8 bits"):
        check_cache8(model({**tiny.TINY_A, "head_dim": 272}))
