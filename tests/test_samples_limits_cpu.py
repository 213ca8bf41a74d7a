"""Engine.sample_many's limits, with a runner that only counts (no GPU)."""
import math
from types import SimpleNamespace

import pytest

from hipinfer_b200.engine import samples


def engine(**kw):
    return SimpleNamespace(**{**dict(vocab=100, max_seq=512, max_prefill=64, runner=None), **kw})


@pytest.mark.parametrize("temperature", [math.nan, -1.0, -math.inf])
def test_a_temperature_that_is_none_is_refused(temperature):
    with pytest.raises(ValueError, match="temperature"):
        samples.sample_many(engine(), [1, 2], 2, 4, temperature, 0, 0, (), True)
