"""What a call says that the library refuses after the binding has taken its arguments: the words of the library that refused, with its sizes."""
import pytest
import torch

from hipinfer_b200.kernels import cache8, ops
from test_gpu_cache8 import DEV, filled, on_gpu, step

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["binding", "interpreter"])
def way(request, monkeypatch):
    monkeypatch.setattr(cache8, "_bound", None if request.param == "binding" else False)


def test_storing_into_more_heads_than_a_call_has(way):
    cache = ops.new_cache8(1, 65536, 1, 1, device=DEV)
    x = torch.zeros(1, 65536, device=DEV)
    with pytest.raises(ops.KernelError, match="hb_cache8_store: 65536 kv heads"):
        ops.store_cache8(x, x, torch.zeros(1, dtype=torch.int32, device=DEV), cache)


def test_attention_of_more_heads_than_a_tile_counts(way):
    batch, _, pages = step([3], [1], 16)
    with pytest.raises(ops.KernelError, match="hb_cache8_attention_mma: 1 kv heads of 64 for 32768"):
        ops.attention_cache8(torch.zeros(1, 32768 * 64, device=DEV), on_gpu(filled(pages, 1, 16, 64, torch.int8)), batch, 0, 32768)


def test_portions_of_more_heads_than_the_flash_kernel_lists(way, monkeypatch):
    monkeypatch.setattr(cache8, "_portion_limit", lambda *a: 16)
    batch, _, pages = step([3], [16], 16)
    with pytest.raises(ops.KernelError, match="hb_flash_prefill_tc: 60000 heads"):
        ops.attention_cache8(torch.zeros(16, 60000 * 64, dtype=torch.bfloat16, device=DEV), on_gpu(filled(pages, 1, 16, 64, torch.int8)), batch, 0, 60000)


def test_copying_more_layers_than_a_launch_has(way):
    with pytest.raises(ops.KernelError, match="hb_copy_pages: 65536 layers"):
        ops.copy_pages([torch.zeros(65536, 2, 1, device=DEV)], [0], [1])


def test_calls_go_on_behind_a_refused_one(way):
    cache = ops.new_cache8(2, 65536, 1, 1, device=DEV)
    with pytest.raises(ops.KernelError):
        ops.store_cache8(torch.zeros(1, 65536, device=DEV), torch.zeros(1, 65536, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), cache)
    k, v = ops.expand_cache8(cache, torch.tensor([1], dtype=torch.int32, device=DEV))
    assert not k.any() and not v.any()
