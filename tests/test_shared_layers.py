"""Which layers read pages that requests share once for all of them, as the decoder counts them (no GPU)."""
import torch

import selovik_models
import tiny
from hipinfer_b200.config import get_architecture, load_config
from hipinfer_b200.engine.runner import ModelRunner
from hipinfer_b200.models.decoder import DecoderModel
from hipinfer_b200.parts.registry import BuildContext


def model(folder):
    config = load_config(folder)
    return DecoderModel(get_architecture(config.architecture).build_spec(config), BuildContext.meta())


class Runner:
    """What the runner's rule looks at."""

    _shared_prefixes, _saved_bytes = ModelRunner._shared_prefixes, ModelRunner._saved_bytes

    def __init__(self, folder):
        self.model = model(folder)
        self.cache = type("Cache", (), {"groups": self.model.cache_groups})
        self.page_size, self.dtype, self._forked = 16, torch.bfloat16, {"f"}


def test_layers_that_share_reads_are_counted(tmp_path):
    m = model(tiny.make_model_folder(tmp_path, "a", torch.bfloat16))
    assert [g.kind for g in m.cache_groups] == ["full"] and m.shared_layers == [len(m.spec.order)]


def test_other_attention_shares_none(tmp_path):
    m = model(selovik_models.make_folder(tmp_path, "d", seed=1, dtype=torch.float32)[0])
    assert not m.state_specs and "full" in [g.kind for g in m.cache_groups] and not any(m.shared_layers)


def test_what_is_saved(tmp_path):
    tables = [[torch.arange(4).int().numpy()] * 4 for _ in range(3)]
    (tmp_path / "a").mkdir()
    (tmp_path / "d").mkdir()
    r = Runner(tiny.make_model_folder(tmp_path / "a", "a", torch.bfloat16))
    shared = r._shared_prefixes(tables, [40, 40, 40])
    g = r.model.cache_groups[0]
    assert shared == [[(0, 3, 32)]]
    assert r._saved_bytes(shared) == 2 * 32 * 2 * sum(h * d for _, h, d in g.planes) * len(r.model.spec.order)
    r = Runner(selovik_models.make_folder(tmp_path / "d", "d", seed=1, dtype=torch.float32)[0])
    assert not any(r._shared_prefixes(tables, [40, 40, 40]))
